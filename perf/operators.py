"""What the operators on the nodes of a batch are judged by: attention among the nodes of a structure (or the tokens of a
sequence), the norm of its queries and keys with the position rotation, the form of both that reads and writes a cache
for one new token at a time, and dropout of whole irreps.

A case names the operator ("op") and how far a pass goes ("run"):

* "attention": rows of many segments one after the other, every row attending to its own segment. "forward", or "train"
  (output and the gradients of queries, keys and values).
* "decode": one new row for each segment, attending to the part of a cache that the segment fills.
* "rotary": norm of each head of queries and keys and rotation by position. "forward" or "train".
* "append": the same for a few new tokens, whose keys and values go into the rows of a cache.
* "dropout": irreps of a node dropped as a whole, added to a residual stream. "forward" or "train".

With ``own`` false a pass is computed from elementary torch operations in 32 bits and rounded once at the end, with it
true by the calls that a program makes of this package.
"""

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "float64": torch.float64}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2, "float64": 8}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------


def _attention(run, dtype, segments, shortest, longest, q_heads, k_heads, head, causal, lens_seed=0, **name):
    return dict(op="attention", run=run, dtype=dtype, segments=segments, shortest=shortest, longest=longest, spread="log",
                q_heads=q_heads, k_heads=k_heads, head=head, causal=causal, lens_seed=lens_seed, **name)


def _decode(dtype, segments, shortest, longest, slots, q_heads, k_heads, head, lens_seed=0, **name):
    return dict(op="decode", run="forward", dtype=dtype, segments=segments, shortest=shortest, longest=longest,
                spread="even", slots=slots, q_heads=q_heads, k_heads=k_heads, head=head, lens_seed=lens_seed, **name)


def _rotary(run, dtype, rows, longest, q_heads, k_heads, head, rotary, interleaved, norm, **name):
    return dict(op="rotary", run=run, dtype=dtype, rows=rows, longest=longest, q_heads=q_heads, k_heads=k_heads,
                head=head, rotary=rotary, interleaved=interleaved, norm=norm, **name)


def _append(dtype, tokens, slots, q_heads, k_heads, head, rotary, interleaved, norm, **name):
    return dict(op="append", run="forward", dtype=dtype, tokens=tokens, slots=slots, q_heads=q_heads, k_heads=k_heads,
                head=head, rotary=rotary, interleaved=interleaved, norm=norm, **name)


def _dropout(run, dtype, rows, irreps, p, residual, **name):
    return dict(op="dropout", run=run, dtype=dtype, rows=rows, irreps=irreps, p=p, residual=residual, **name)


def listed():
    return [
        # training step of a global attention layer over the atoms of each molecule of a batch, in the features' own type
        _attention("train", "float32", 512, 9, 61, 8, 8, 32, False, 1, name="molecules-train"),
        # a few packed prompts read in at once before generation begins, grouped heads: the largest call
        _attention("forward", "bfloat16", 7, 500, 8192, 32, 8, 128, True, 2, name="prompt-large"),
        # training step of a generating model on packed sequences of uneven length
        _attention("train", "bfloat16", 9, 200, 4001, 16, 4, 128, True, 3, name="sequences-train"),
        # crystals and fragments of very different sizes, half precision, heads off the powers of two
        _attention("train", "float16", 33, 1, 700, 6, 2, 72, False, 4, name="crystals-train-odd"),
        # one long sequence, one new token
        _decode("bfloat16", 1, 65537, 65537, 65600, 32, 8, 128, 5, name="token-long"),
        # serving: 64 sequences between one and 4096 tokens, a new token each
        _decode("float16", 64, 1, 4096, 4096, 16, 4, 128, 6, name="tokens-batch"),
        # the first steps of generating a handful of small molecules, where latency counts
        _decode("float32", 7, 0, 60, 64, 8, 8, 32, 7, name="tokens-small"),
        # norm and rotation of queries and keys in a training step
        _rotary("train", "bfloat16", 16411, 4001, 32, 8, 128, 128, False, True, name="rotary-train"),
        # rotation alone of a part of each head, small batch, pairs next to each other
        _rotary("forward", "float32", 333, 61, 8, 8, 32, 16, True, False, name="rotary-small"),
        # a new token of each of 64 sequences on its way into the cache
        _append("bfloat16", 64, 257, 32, 8, 128, 128, False, True, name="append"),
        # dropout with the residual of a hidden layer of 128 channels up to l = 3, training step on 20 000 atoms
        _dropout("train", "float32", 20000, "128x0e+128x1o+128x2e+128x3o", 0.1, True, name="dropout-train"),
        # scalar features of a small batch, an odd number of channels
        _dropout("forward", "bfloat16", 777, "131x0e", 0.2, False, name="dropout-small"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((1, 1), (4, 4), (8, 8), (6, 2), (8, 2), (16, 4), (32, 8), (16, 1), (5, 5))


def draw(rng):
    """One more case of the ranges above."""
    op = rng.choice(("attention", "attention", "attention", "decode", "decode", "rotary", "append", "dropout"))
    dtype = rng.choice(("float32", "bfloat16", "float16", "bfloat16"))
    q_heads, k_heads = rng.choice(_HEADS)
    head = rng.choice((32, 64, 128, 128, 24, 40, 72, 96, 112))
    seed = rng.randrange(1 << 20)
    limit = _cost(listed()[1])
    if op == "attention":
        longest = _spread(rng, 8, 1500 if dtype == "float32" else 8192)
        case = _attention(rng.choice(("forward", "train")), dtype, _spread(rng, 1, 512), _spread(rng, 1, longest), longest,
                          q_heads, k_heads, head, rng.random() < 0.5, seed)
        while case["segments"] > 1 and (_cost(case) > limit or sum(_lens(case)) > 40000):
            case["segments"] = (case["segments"] + 1) // 2
    elif op == "decode":
        longest = _spread(rng, 16, 65537)
        case = _decode(dtype, _spread(rng, 1, 300), rng.choice((0, 1, longest // 2, longest)), longest,
                       longest + rng.randrange(70), q_heads, k_heads, head, seed)
        while case["segments"] > 1 and (_cost(case) > limit or case["segments"] * case["slots"] > 600000):
            case["segments"] = (case["segments"] + 1) // 2
    elif op in ("rotary", "append"):
        rotary = rng.choice([r for r in (8, 16, 32, 64, 128, head) if r <= head])
        interleaved, norm = rng.random() < 0.4, rng.random() < 0.7
        if op == "rotary":
            case = _rotary(rng.choice(("forward", "train")), dtype, _spread(rng, 50, 16411), _spread(rng, 10, 8192),
                           q_heads, k_heads, head, rotary, interleaved, norm)
        else:
            case = _append(dtype, _spread(rng, 1, 300), _spread(rng, 20, 500), q_heads, k_heads, head, rotary,
                           interleaved, norm)
    else:
        dtype = rng.choice(("float32", "float32", "bfloat16", "float16", "float64"))
        irreps = rng.choice(("131x0e", "512x0e", "64x0e+64x1o", "128x0e+128x1o+128x2e+128x3o", "32x0e+17x1o+9x2e",
                             "7x0e+5x1e+3x3o"))
        rows = _spread(rng, 100, 20000)
        case = _dropout(rng.choice(("forward", "train")), dtype, rows, irreps,
                        rng.choice((0.05, 0.1, 0.2, 0.5)), rng.random() < 0.6)
    return case


def _lens(case):
    """Rows of each segment; the first is the longest."""
    rng = random.Random(case["lens_seed"])
    lo, hi = case["shortest"], case["longest"]
    pick = (lambda: _spread(rng, max(lo, 1), hi)) if case["spread"] == "log" else (lambda: rng.randint(lo, hi))
    return [hi] + [pick() for _ in range(case["segments"] - 1)]


def _irreps(text):
    """[(channels, components)] of "128x0e+64x1o"."""
    out = []
    for block in text.split("+"):
        mul, ir = block.split("x")
        out.append((int(mul), 2 * int(ir[:-1]) + 1))
    return out


def work(case):
    s, op = _BYTES[case["dtype"]], case["op"]
    if op == "dropout":
        n = case["rows"] * sum(m * d for m, d in _irreps(case["irreps"]))
        passes = 2 + int(case["residual"]) + (2 if case["run"] == "train" else 0)
        return {"bytes": passes * n * s, "flops": n * (2 if case["run"] == "train" else 1)}
    hq, hk, d = case["q_heads"], case["k_heads"], case["head"]
    if op == "rotary":
        n = case["rows"] * (hq + hk) * d
        per_row = 8 + case["rotary"] * 4  # its position and its row of the table
        return {"bytes": (4 if case["run"] == "train" else 2) * n * s + case["rows"] * per_row,
                "flops": n * (18 if case["run"] == "train" else 7)}
    if op == "append":
        n = case["tokens"] * (hq + 2 * hk) * d
        return {"bytes": 2 * n * s + case["tokens"] * (16 + case["rotary"] * 4), "flops": n * 7}
    lens = _lens(case)
    if op == "decode":
        keys = sum(lens)
        return {"bytes": (2 * keys * hk + 2 * len(lens) * hq) * d * s, "flops": 4 * keys * hq * d}
    rows = sum(lens)
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
    if case["run"] == "train":  # q, k, v, the output's gradient; the output and three gradients
        return {"bytes": rows * (4 * hq + 4 * hk) * d * s, "flops": 14 * pairs * hq * d}
    return {"bytes": rows * (2 * hq + 2 * hk) * d * s, "flops": 4 * pairs * hq * d}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 4e14)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------


def _rotary_table(length, rotary):
    """[length, 2, rotary / 2]: cosines and sines of position times frequency."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=1).float()


def _starts(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device="cuda")


def _groups(lens):
    """Segments by similar length, for the plain form's padded products: [(first rows, lengths, longest)]."""
    starts = np.concatenate([[0], np.cumsum(lens)])
    by_size = {}
    for i, n in enumerate(lens):
        if n:
            by_size.setdefault(max(4, int(math.ceil(math.log2(n)))), []).append(i)
    return [(torch.tensor([int(starts[i]) for i in ids], device="cuda"), torch.tensor([lens[i] for i in ids], device="cuda"),
             max(lens[i] for i in ids)) for ids in by_size.values()]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    train = case["run"] == "train"

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int64)

    st = {"case": case}
    if case["op"] == "dropout":
        dim = sum(m * d for m, d in _irreps(case["irreps"]))
        st["x"] = normal(case["rows"], dim).requires_grad_(train)
        st["residual"] = normal(case["rows"], dim) if case["residual"] else None
        st["grad"] = normal(case["rows"], dim) if train else None
        st["seed"] = whole(-(1 << 62), 1 << 62, 2)
        blocks, channel, first = _irreps(case["irreps"]), [], 0
        for mul, d in blocks:
            channel.append(first + np.repeat(np.arange(mul), d))
            first += mul
        st["channel"] = torch.tensor(np.concatenate(channel), device="cuda")
        if own:
            import openequivariance_amd as oeq
            st["module"] = oeq.IrrepDropout(case["irreps"], case["p"])
        return st
    hq, hk, d = case["q_heads"], case["k_heads"], case["head"]
    if case["op"] in ("rotary", "append"):
        n = case["rows"] if case["op"] == "rotary" else case["tokens"]
        # queries, keys and values as one projection gives them: views into its rows
        qkv = normal(n, (hq + 2 * hk) * d)
        q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
        st["q"], st["k"], st["v"] = (t.view(n, -1, d) for t in (q, k, v))
        for name in ("q_weight", "k_weight"):
            st[name] = (1 + 0.1 * normal(d).float()).to(dt) if case["norm"] else None
        if case["op"] == "rotary":
            longest = case["longest"]
            st["positions"] = (torch.arange(n, device="cuda") + whole(0, longest, 1)) % longest
            st["table"] = _rotary_table(longest, case["rotary"])
            if train:
                st["q_grad"], st["k_grad"] = normal(n, hq, d), normal(n, hk, d)
                for name in ("q", "k", "q_weight", "k_weight"):
                    if st[name] is not None:
                        st[name] = st[name].detach().requires_grad_()
        else:
            slots = case["slots"]
            st["positions"] = whole(0, slots, n)
            st["table"] = _rotary_table(slots, case["rotary"])
            st["k_cache"], st["v_cache"] = normal(n * slots, hk, d), normal(n * slots, hk, d)
            st["slots"] = torch.arange(n, device="cuda") * slots + st["positions"]
            if n > 3:
                st["slots"][n // 2] = -1  # a place of the batch without a sequence
        return st
    lens = _lens(case)
    if case["op"] == "attention":
        n = sum(lens)
        st["q"], st["k"], st["v"] = (normal(n, h, d).requires_grad_(train) for h in (hq, hk, hk))
        st["grad"] = normal(n, hq, d) if train else None
        st["ptr"], st["groups"], st["lens"] = _starts(lens), _groups(lens), lens
        return st
    slots = case["slots"]
    st["q"] = normal(len(lens), hq, d)
    st["k"], st["v"] = normal(len(lens) * slots, hk, d), normal(len(lens) * slots, hk, d)
    st["q_ptr"] = torch.arange(len(lens) + 1, device="cuda")
    st["k_ptr"] = st["q_ptr"] * slots
    st["k_len"] = torch.tensor(lens, device="cuda")
    st["lens"] = lens
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------


def _softmax_product(scores, visible, v):
    """softmax over the last axis of the visible scores, times v; nothing where nothing is visible."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _plain_attention(q, k, v, groups, causal):
    n, hq, d = q.shape
    hk = k.shape[1]
    out = torch.zeros_like(q)
    for first, lens, longest in groups:
        at = torch.arange(longest, device=q.device)
        inside = at < lens[:, None]
        rows = torch.where(inside, first[:, None] + at, first[:, None])
        b = rows.shape[0]
        qq = q[rows].view(b, longest, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d) / math.sqrt(d)
        kk, vv = k[rows].permute(0, 2, 1, 3), v[rows].permute(0, 2, 1, 3)
        scores = torch.matmul(qq, kk.transpose(2, 3)).view(b, hk, hq // hk, longest, longest)
        visible = inside[:, None, None, None, :]
        if causal:
            visible = visible & (at[None, :] <= at[:, None])
        o = _softmax_product(scores.view(b, hk, -1, longest),
                             visible.expand(b, 1, hq // hk, longest, longest).reshape(b, 1, -1, longest), vv)
        o = o.view(b, hk, hq // hk, longest, d).permute(0, 3, 1, 2, 4).reshape(b, longest, hq, d)
        out = out.index_put((rows[inside],), o[inside])
    return out


def _plain_decode(st):
    case = st["case"]
    b, hk, g, d = case["segments"], case["k_heads"], case["q_heads"] // case["k_heads"], case["head"]
    longest = max(1, max(st["lens"]))
    k = st["k"].view(b, -1, hk, d)[:, :longest].float().permute(0, 2, 1, 3)
    v = st["v"].view(b, -1, hk, d)[:, :longest].float().permute(0, 2, 1, 3)
    q = st["q"].float().view(b, hk, g, d) / math.sqrt(d)
    visible = torch.arange(longest, device=q.device) < st["k_len"][:, None, None, None]
    scores = torch.matmul(q, k.transpose(2, 3))
    return _softmax_product(scores, visible, v).reshape(b, hk * g, d).to(st["q"].dtype)


def _plain_rotary(x, weight, positions, table, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = table.shape[2]
    cos, sin = table[positions, 0][:, None], table[positions, 1][:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


_M32 = 0xFFFFFFFF


def _philox(c0, c1, c2, c3, k0, k1):
    """Four words of 32 bits from a counter and a key of such words (Salmon et al., SC 2011: Philox-4x32 with ten
    rounds), in whole numbers of 64 bits."""
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _M32) ^ c1 ^ k0, b & _M32, ((a >> 32) & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return c0, c1, c2, c3


def _plain_keep(case, seed, channel):
    """Which (row, channel) is kept, spread over the channels' components."""
    dev = channel.device
    n, groups = case["rows"], (sum(m for m, _ in _irreps(case["irreps"])) + 7) // 8
    row = torch.arange(n, device=dev)[:, None].expand(n, groups)
    group = torch.arange(groups, device=dev)[None].expand(n, groups)
    words = _philox(group, row, (seed[1] & _M32).expand(n, groups), ((seed[1] >> 32) & _M32).expand(n, groups),
                    seed[0] & _M32, (seed[0] >> 32) & _M32)
    draws = torch.stack([half for w in words for half in (w & 0xFFFF, w >> 16)], dim=-1).view(n, -1)
    return (draws >= int(round(case["p"] * 65536)))[:, channel]


def _run_plain(st):
    case = st["case"]
    op, dt = case["op"], _DTYPES[case["dtype"]]
    if op == "dropout":
        wide = torch.float64 if dt == torch.float64 else torch.float32
        keep = _plain_keep(case, st["seed"], st["channel"])
        scale = 65536.0 / (65536 - int(round(case["p"] * 65536)))
        out = torch.where(keep, st["x"].detach().to(wide) * scale, 0.0)
        if st["residual"] is not None:
            out = out + st["residual"].to(wide)
        if case["run"] == "forward":
            return out.to(dt)
        return out.to(dt), torch.where(keep, st["grad"].to(wide) * scale, 0.0).to(dt)
    if op == "decode":
        return _plain_decode(st)
    if op == "attention":
        if case["run"] == "forward":
            return _plain_attention(st["q"].float(), st["k"].float(), st["v"].float(), st["groups"], case["causal"]).to(dt)
        q, k, v = (st[n].detach().float().requires_grad_() for n in "qkv")
        out = _plain_attention(q, k, v, st["groups"], case["causal"])
        grads = torch.autograd.grad(out, (q, k, v), st["grad"].float())
        return (out.detach().to(dt),) + tuple(g.to(dt) for g in grads)
    table, positions, inter = st["table"], st["positions"], case["interleaved"]
    if op == "append":
        q = _plain_rotary(st["q"], st["q_weight"], positions, table, inter).to(dt)
        k = _plain_rotary(st["k"], st["k_weight"], positions, table, inter).to(dt)
        used = st["slots"] >= 0
        st["k_cache"][st["slots"][used]] = k[used]
        st["v_cache"][st["slots"][used]] = st["v"][used]
        return q, st["k_cache"], st["v_cache"]
    if case["run"] == "forward":
        return tuple(_plain_rotary(st[n], st[n + "_weight"], positions, table, inter).to(dt) for n in "qk")
    leaves = [st[n].detach().float().requires_grad_() for n in ("q", "k", "q_weight", "k_weight") if st[n] is not None]
    weights = leaves[2:] if case["norm"] else [None, None]
    out = [_plain_rotary(leaves[i], weights[i], positions, table, inter) for i in (0, 1)]
    grads = torch.autograd.grad(out, leaves, (st["q_grad"].float(), st["k_grad"].float()))
    return tuple(t.detach().to(dt) for t in out) + tuple(g.to(dt) for g in grads)


# ---------------------------------------------------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------------------------------------------------


def _run_own(st):
    import openequivariance_amd as oeq
    case = st["case"]
    op = case["op"]
    if op == "dropout":
        out = st["module"](st["x"], st["residual"], seed=st["seed"])
        if case["run"] == "forward":
            return out
        return out.detach(), torch.autograd.grad(out, st["x"], st["grad"])[0]
    if op == "decode":
        return oeq.packed_attention(st["q"], st["k"], st["v"], st["q_ptr"], st["k_ptr"], k_len=st["k_len"])
    if op == "attention":
        out = oeq.packed_attention(st["q"], st["k"], st["v"], st["ptr"], causal=case["causal"])
        if case["run"] == "forward":
            return out
        return (out.detach(),) + torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["grad"])
    weights = dict(q_weight=st["q_weight"], k_weight=st["k_weight"], interleaved=case["interleaved"])
    if op == "append":
        q = oeq.qk_norm_rotary_append(st["q"], st["k"], st["v"], st["positions"], st["table"], st["k_cache"],
                                      st["v_cache"], st["slots"], **weights)
        return q, st["k_cache"], st["v_cache"]
    out = oeq.qk_norm_rotary(st["q"], st["k"], st["positions"], st["table"], **weights)
    if case["run"] == "forward":
        return out
    leaves = [st[n] for n in ("q", "k", "q_weight", "k_weight") if st[n] is not None]
    return tuple(t.detach() for t in out) + torch.autograd.grad(out, leaves, (st["q_grad"], st["k_grad"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------


def _exact_attention(st, case):
    """One segment after the other, a few heads at a time, the gradients by their formulas."""
    q, k, v = (st[n].detach().double() for n in "qkv")
    hq, hk, d = case["q_heads"], case["k_heads"], case["head"]
    g, train = hq // hk, case["run"] == "train"
    scale = d ** -0.5
    out = torch.zeros_like(q)
    if train:
        do = st["grad"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    first = 0
    for n in case_lens(case):
        part = slice(first, first + n)
        first += n
        if not n:
            continue
        step = max(1, min(hk, int(4e8 / (n * n * g))))  # heads of keys at a time
        for h in range(0, hk, step):
            hs = slice(h, min(hk, h + step))
            qs = slice(h * g, min(hk, h + step) * g)
            kk = k[part, hs].transpose(0, 1).repeat_interleave(g, 0).contiguous()
            vv = v[part, hs].transpose(0, 1).repeat_interleave(g, 0).contiguous()
            qq = q[part, qs].transpose(0, 1).contiguous()
            s = torch.bmm(qq, kk.transpose(1, 2).contiguous()) * scale
            if case["causal"]:
                s += torch.full((n, n), -math.inf, dtype=torch.float64, device=s.device).triu(1)
            p = torch.softmax(s, dim=-1)
            o = torch.bmm(p, vv)
            out[part, qs] = o.transpose(0, 1)
            if train:
                oo = do[part, qs].transpose(0, 1).contiguous()
                ds = p * (torch.bmm(oo, vv.transpose(1, 2).contiguous()) - (oo * o).sum(-1, keepdim=True))
                dq[part, qs] = (torch.bmm(ds, kk) * scale).transpose(0, 1)
                heads = kk.shape[0] // g
                dk[part, hs] = (torch.bmm(ds.transpose(1, 2).contiguous(), qq) * scale).view(heads, g, n, d).sum(1).transpose(0, 1)
                dv[part, hs] = torch.bmm(p.transpose(1, 2).contiguous(), oo).view(heads, g, n, d).sum(1).transpose(0, 1)
    return (out, dq, dk, dv) if train else out


def case_lens(case):
    """Rows of each segment of an attention or decode case."""
    return _lens(case)


def _exact_decode(st, case):
    hk, d, slots = case["k_heads"], case["head"], case["slots"]
    q = st["q"].double().view(case["segments"], hk, -1, d)
    out = torch.zeros_like(q)
    for i, n in enumerate(case_lens(case)):
        if n:
            k = st["k"][i * slots:i * slots + n].double().permute(1, 2, 0).contiguous()
            v = st["v"][i * slots:i * slots + n].double().transpose(0, 1).contiguous()
            out[i] = torch.bmm(torch.softmax(torch.bmm(q[i], k) * d ** -0.5, dim=-1), v)
    return out.view(case["segments"], -1, d)


def _turn(half, rotary, interleaved):
    """Places of the first and second partners of the turned pairs."""
    i = torch.arange(half, device="cuda")
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def _exact_rotary(x, weight, st, case, grad):
    """(output, gradient of x, gradient of the weight), the gradients where the output's is given."""
    x = x.detach().double()
    first, second = _turn(case["rotary"] // 2, case["rotary"], case["interleaved"])
    rows = st["table"].double()[st["positions"]]
    c, s = rows[:, None, 0], rows[:, None, 1]
    r = 1.0 / torch.sqrt(torch.square(x).mean(-1, keepdim=True) + 1e-6) if weight is not None else None
    w = weight.detach().double() if weight is not None else None
    y = x * r * w if weight is not None else x
    out = y.clone()
    out[..., first] = y[..., first] * c - y[..., second] * s
    out[..., second] = y[..., first] * s + y[..., second] * c
    if grad is None:
        return out, None, None
    g = grad.double()
    gy = g.clone()
    gy[..., first] = g[..., first] * c + g[..., second] * s
    gy[..., second] = g[..., second] * c - g[..., first] * s
    if weight is None:
        return out, gy, None
    unit = x * r
    gu = gy * w
    return out, r * (gu - unit * (gu * unit).mean(-1, keepdim=True)), (gy * unit).sum((0, 1))


def _exact_draws(key, step, row, group):
    """Philox-4x32 with ten rounds in numpy's unsigned 64-bit numbers: eight 16-bit numbers for each group of channels."""
    low = np.uint64(_M32)
    c = [group, row, np.full_like(row, step & _M32), np.full_like(row, step >> 32)]
    k = [np.uint64(key & _M32), np.uint64(key >> 32)]
    for _ in range(10):
        first, second = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(second >> np.uint64(32)) ^ c[1] ^ k[0], second & low, (first >> np.uint64(32)) ^ c[3] ^ k[1], first & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return np.stack([c[0] & np.uint64(0xFFFF), c[0] >> np.uint64(16), c[1] & np.uint64(0xFFFF), c[1] >> np.uint64(16),
                     c[2] & np.uint64(0xFFFF), c[2] >> np.uint64(16), c[3] & np.uint64(0xFFFF), c[3] >> np.uint64(16)], -1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "attention":
        return _exact_attention(st, case)
    if op == "decode":
        return _exact_decode(st, case)
    if op == "dropout":
        key, step = (int(v) & ((1 << 64) - 1) for v in st["seed"].tolist())
        n, blocks = case["rows"], _irreps(case["irreps"])
        groups = (sum(m for m, _ in blocks) + 7) // 8
        row, group = np.meshgrid(np.arange(n, dtype=np.uint64), np.arange(groups, dtype=np.uint64), indexing="ij")
        drop = int(round(case["p"] * 65536))
        kept = _exact_draws(key, step, row, group).reshape(n, -1) >= drop
        channels = np.concatenate([np.repeat(np.arange(m), d) + sum(b[0] for b in blocks[:i])
                                   for i, (m, d) in enumerate(blocks)])
        factor = torch.from_numpy(kept[:, channels]).to("cuda").double() * (65536.0 / (65536 - drop))
        out = st["x"].detach().double() * factor
        if st["residual"] is not None:
            out = out + st["residual"].double()
        return out if case["run"] == "forward" else (out, st["grad"].double() * factor)
    train = case["run"] == "train"
    q, dq, dqw = _exact_rotary(st["q"], st["q_weight"], st, case, st["q_grad"] if train else None)
    k, dk, dkw = _exact_rotary(st["k"], st["k_weight"], st, case, st["k_grad"] if train else None)
    if op == "append":
        k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
        for i, at in enumerate(st["slots"].tolist()):
            if at >= 0:
                k_cache[at], v_cache[at] = k[i], st["v"][i].double()
        return q, k_cache, v_cache
    if not train:
        return q, k
    return (q, k, dq, dk) + ((dqw, dkw) if case["norm"] else ())
