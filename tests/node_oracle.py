"""The operators on nodes from their definitions in 64 bits on the CPU, each with a bound of the error that the kernels'
arithmetic allows.

With u the half unit of the tensors' type (2^-24, 2^-11, 2^-8 for 24, 11 and 8 bits) the kernels round an output once,
u |out|, and where operands have 16 bits they round p and ds to operands of a product, u p and u |ds| in every term of a
sum; delta = g.o of the rounded output (where its remainder is not kept), u sum |g o|. What is left are errors in 32
bits: a dot product of d terms, a sum of n, one of exp and log each, in all (d + n + 32) 2^-24 of the sums of absolute values, times 1 + S where a
score of absolute sum S stands in an exponent.
"""

import math

import torch

HALF_UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}
# numbers below this are stored with an absolute error of half the smallest one
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float64: 0.0}


def segment_views(q_ptr, k_ptr, k_len, nk, causal):
    """For each segment (first query, end, first key, keys, visible [queries, keys])."""
    out = []
    for s in range(len(q_ptr) - 1):
        q0, q1, k0, k1 = q_ptr[s], q_ptr[s + 1], k_ptr[s], min(k_ptr[s + 1], nk)
        n = max(0, k1 - k0)
        if k_len is not None:
            n = min(n, max(0, k_len[s]))
        see = torch.ones(q1 - q0, n, dtype=torch.bool)
        if causal:
            see = torch.arange(n)[None] <= torch.arange(q1 - q0)[:, None] + n - (q1 - q0)
        out.append((q0, q1, k0, n, see))
    return out


def attention(q, k, v, views, scale, grad=None):
    """({name: value}, {name: bound}) of out, lse and, with the output's gradient, dq, dk and dv."""
    u, tiny = HALF_UNIT[q.dtype], TINY[q.dtype]
    up = 0.0 if q.dtype == torch.float32 else u  # p and ds as operands
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    nq, hq, d = q.shape
    g = hq // k.shape[1]
    names = ["out", "lse"] + (["dq", "dk", "dv"] if grad is not None else [])
    like = dict(out=q, lse=q[..., 0], dq=q, dk=k, dv=v)
    val = {n: torch.zeros_like(like[n]) for n in names}
    err = {n: torch.zeros_like(like[n]) for n in names}
    val["lse"].fill_(-math.inf)
    if grad is not None:
        do = grad.detach().cpu().double()
    for q0, q1, k0, n, see in views:
        if q1 == q0 or n == 0:
            continue
        rows, keys = slice(q0, q1), slice(k0, k0 + n)
        for h in range(hq):
            kh = h // g
            qq, kk, vv = q[rows, h], k[keys, kh], v[keys, kh]

            def over(weights, x):  # sum over visible entries only, whatever hidden ones hold
                if torch.isfinite(x).all():
                    return weights @ x
                return torch.where((weights != 0)[:, :, None], weights[:, :, None] * x[None], 0.0).sum(1)

            s = torch.where(see, (qq[:, None] * kk[None]).sum(-1) * scale, -math.inf)
            size = torch.where(see, (qq[:, None] * kk[None]).abs().sum(-1) * scale, 0.0)
            any_seen = see.any(1)
            e32 = 2.0 ** -24 * (d + n + 32) * (1 + size.amax())
            lse = torch.logsumexp(s, 1)
            p = torch.where(see & any_seen[:, None], torch.exp(s - torch.where(any_seen, lse, 0.0)[:, None]), 0.0)
            o = over(p, vv)
            o_err = (up + 3 * e32) * over(p, vv.abs()) + u * o.abs()
            val["out"][rows, h], val["lse"][rows, h] = o, lse
            err["out"][rows, h] = o_err
            err["lse"][rows, h] = torch.where(any_seen, 3 * e32 + 2.0 ** -22 * (1 + lse.abs()), 0.0)
            if grad is None:
                continue
            gg = do[rows, h]
            gv = torch.where(see, (gg[:, None] * vv[None]).sum(-1), 0.0)
            gv_abs = torch.where(see, (gg[:, None] * vv[None]).abs().sum(-1), 0.0)
            delta = torch.where(any_seen, (gg * o).sum(-1), 0.0)
            delta_abs = torch.where(any_seen, (gg * o).abs().sum(-1), 0.0)
            delta_err = torch.where(any_seen, (gg.abs() * o_err).sum(-1), 0.0)
            ds = torch.where(see, p * (gv - delta[:, None]), 0.0)
            size_ds = p * (gv_abs + delta_abs[:, None])
            ds_err = torch.where(see, up * ds.abs() + 3 * e32 * size_ds + p * delta_err[:, None], 0.0)
            val["dq"][rows, h] = over(ds, kk) * scale
            err["dq"][rows, h] = over(ds_err, kk.abs()) * scale
            val["dk"][keys, kh] += over(ds.t(), qq) * scale
            err["dk"][keys, kh] += over(ds_err.t(), qq.abs()) * scale
            val["dv"][keys, kh] += over(p.t(), gg)
            err["dv"][keys, kh] += over((up + 3 * e32) * p.t(), gg.abs())
    for n in ("dq", "dk", "dv"):
        if n in val:
            err[n] += u * val[n].abs()
    if grad is not None:  # the sums over the rows of dk and dv are of one length more than scores know
        for n in ("dk", "dv"):
            err[n] += 2.0 ** -24 * nq * g * err[n] / u if u > 2.0 ** -24 else 0
    return val, {n: e + tiny for n, e in err.items()}


def check(got, val, err, what):
    got = got.detach().cpu().double()
    assert got.shape == val.shape, what
    same = (got == val) | (torch.isnan(got) & torch.isnan(val))
    bad = ~same & ~((got - val).abs() <= err)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside their bound, first at {at}: "
                             f"{got[at]} instead of {val[at]} +- {err[at]}")


def rotate(x, weight, positions, table, interleaved, eps, grad=None):
    """(out, bound[, dx, bound, dweight, bound]). An output is at most a norm (d + 8 errors of 32 bits), a weight and two
    products; a gradient adds the sums along a head."""
    u, tiny = HALF_UNIT[x.dtype], TINY[x.dtype]
    x = x.detach().cpu().double()
    d, half = x.shape[2], table.shape[2]
    e32 = 2.0 ** -24 * (d + 16)
    c, s = (table.detach().cpu().double()[positions.cpu(), i][:, None] for i in (0, 1))
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)

    def turned(y, sign, a=False):
        z = y.clone()
        cc, ss = (c.abs(), s.abs()) if a else (c, s)
        z[..., first] = y[..., first] * cc - (-1 if a else sign) * y[..., second] * ss
        z[..., second] = y[..., second] * cc + (1 if a else sign) * y[..., first] * ss
        return z

    w = weight.detach().cpu().double() if weight is not None else None
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if weight is not None else 1.0
    y = x * r * (w if w is not None else 1.0)
    out = turned(y, 1)
    result = [out, u * out.abs() + e32 * turned(y.abs(), 1, True) + tiny]
    if grad is None:
        return result
    g = grad.detach().cpu().double()
    gy, gy_abs = turned(g, -1), turned(g.abs(), 1, True)
    if w is None:
        return result + [gy, u * gy.abs() + e32 * gy_abs + tiny, None, None]
    n = x * r
    gw, gw_abs = gy * w, gy_abs * w.abs()
    along = (gw * n).mean(-1, keepdim=True)
    dx = r * (gw - n * along)
    dx_abs = r * (gw_abs + n.abs() * (gw_abs * n.abs()).mean(-1, keepdim=True))
    dw, dw_abs = (gy * n).sum((0, 1)), (gy_abs * n.abs()).sum((0, 1))
    terms = x.shape[0] * x.shape[1]
    return result + [dx, u * dx.abs() + 4 * e32 * dx_abs + tiny,
                     dw, u * dw.abs() + (3 * e32 + 2.0 ** -24 * terms) * dw_abs + tiny]


def philox(counter, key):
    """Ten rounds of Philox-4x32 on Python's whole numbers (Salmon et al., SC 2011, figure 3 and table 2)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(rows, channels, seed, p):
    """[rows, channels] of what dropout keeps."""
    low = 0xFFFFFFFF
    key, step = (int(v) & ((1 << 64) - 1) for v in seed.tolist())
    drop = round(p * 65536)
    out = torch.zeros(rows, channels, dtype=torch.bool)
    for r in range(rows):
        for group in range((channels + 7) // 8):
            words = philox((group, r, step & low, step >> 32), (key & low, key >> 32))
            for c in range(8 * group, min(channels, 8 * group + 8)):
                bits = words[c % 8 // 2] >> (16 * (c % 2)) & 0xFFFF
                out[r, c] = bits >= drop
    return out
