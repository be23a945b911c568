"""The operators whose parameters are chosen row by row from their definitions in 64 bits on the CPU, each with a bound of the
error that the kernels' arithmetic allows.

With u the half unit of the tensors' type an output is rounded once, u |out|. A sum of n products held in 32 bits is off by at
most (n + 8) 2^-23 of the sum of absolute products: each addition, in whatever order, by a unit at most (matrix instructions
may cut instead of rounding), and the products of floats by half of one. What lies between two thin products is such a sum
itself; where operands have 16 bits it is kept to 16 bits at least, 2^-16 of it.
"""

import torch

from tests.node_oracle import HALF_UNIT, TINY


def dot_error(n, size):
    return (n + 8) * 2.0 ** -23 * size


def rounded(out, dtype):
    """What the last rounding may add."""
    return HALF_UNIT[dtype] * out.abs() + TINY[dtype]


def order_of(types, count):
    """(order, ptr) by sorting on the host."""
    keys = torch.where((types >= 0) & (types < count), types, count)
    order = torch.sort(keys, stable=True).indices
    ptr = torch.searchsorted(keys[order].contiguous(), torch.arange(count + 1))
    return order.int(), ptr.int()


def rows_of(types, count):
    return [(t, (types == t).nonzero()[:, 0]) for t in range(count)]


def linear(x, weight, types, bias=None, grad=None):
    """({name: value}, {name: bound}) of out and, with the output's gradient, dx, dw and db."""
    dt = x.dtype
    x, weight = x.detach().cpu().double(), weight.detach().cpu().double()
    types = types.cpu()
    count, outer, inner = weight.shape
    shape = x.shape
    val = {"out": torch.zeros(*shape[:-1], outer, dtype=torch.float64)}
    if grad is not None:
        grad = grad.detach().cpu().double()
        val.update(dx=torch.zeros_like(x), dw=torch.zeros_like(weight), db=torch.zeros(count, outer, dtype=torch.float64))
    err = {k: torch.zeros_like(v) for k, v in val.items()}
    for t, rows in rows_of(types, count):
        if not len(rows):
            continue
        xt, w = x[rows].reshape(-1, inner), weight[t]
        b = torch.zeros(outer, dtype=torch.float64) if bias is None else bias[t].detach().cpu().double()
        n = xt.shape[0]
        view = (len(rows), *shape[1:-1], -1)
        val["out"][rows] = (xt @ w.t() + b).view(view)
        err["out"][rows] = dot_error(inner + 1, xt.abs() @ w.abs().t() + b.abs()).view(view)
        if grad is None:
            continue
        g = grad[rows].reshape(-1, outer)
        val["dx"][rows], err["dx"][rows] = (g @ w).view(view), dot_error(outer, g.abs() @ w.abs()).view(view)
        val["dw"][t], err["dw"][t] = g.t() @ xt, dot_error(n, g.abs().t() @ xt.abs())
        val["db"][t], err["db"][t] = g.sum(0), dot_error(n, g.abs().sum(0))
    return val, {k: err[k] + rounded(val[k], dt) for k in val}


def adapters(x, weight, down, up, types, scale=None, grad=None):
    """The same of out and dx, dweight, ddown, dup."""
    dt = x.dtype
    keep = 0.0 if dt == torch.float32 else 2.0 ** -16
    x, weight, down, up = (t.detach().cpu().double() for t in (x, weight, down, up))
    types = types.cpu()
    (count, rank, inner), outer = down.shape, weight.shape[0]
    scale = torch.ones(count, dtype=torch.float64) if scale is None else scale.cpu().double()
    val = {"out": x @ weight.t()}
    size = {"out": x.abs() @ weight.abs().t()}  # sums of absolute products
    more = {"out": torch.zeros_like(val["out"])}  # errors of what lies between
    terms = {"out": inner + rank}
    if grad is not None:
        g_all = grad.detach().cpu().double()
        val.update(dx=g_all @ weight, dweight=g_all.t() @ x, ddown=torch.zeros_like(down), dup=torch.zeros_like(up))
        size.update(dx=g_all.abs() @ weight.abs(), dweight=g_all.abs().t() @ x.abs(), ddown=torch.zeros_like(down), dup=torch.zeros_like(up))
        more.update({k: torch.zeros_like(val[k]) for k in ("dx", "dweight", "ddown", "dup")})
        terms.update(dx=outer + rank, dweight=x.shape[0], ddown=x.shape[0], dup=x.shape[0])
    for t, rows in rows_of(types, count):
        if not len(rows):
            continue
        s, a, b, xt = scale[t], down[t], up[t], x[rows]
        u, u_size = s * xt @ a.t(), s.abs() * xt.abs() @ a.abs().t()
        u_err = dot_error(inner + 1, u_size) + keep * u.abs()
        val["out"][rows] += u @ b.t()
        size["out"][rows] += u.abs() @ b.abs().t()
        more["out"][rows] = u_err @ b.abs().t()
        if grad is None:
            continue
        g = g_all[rows]
        v, v_size = s * g @ b, s.abs() * g.abs() @ b.abs()
        v_err = dot_error(outer + 1, v_size) + keep * v.abs()
        val["dx"][rows] += v @ a
        size["dx"][rows] += v.abs() @ a.abs()
        more["dx"][rows] = v_err @ a.abs()
        val["ddown"][t], size["ddown"][t], more["ddown"][t] = v.t() @ xt, v.abs().t() @ xt.abs(), v_err.t() @ xt.abs()
        val["dup"][t], size["dup"][t], more["dup"][t] = g.t() @ u, g.abs().t() @ u.abs(), g.abs().t() @ u_err
    return val, {k: dot_error(terms[k], size[k]) + 2 * more[k] + rounded(val[k], dt) for k in val}


def embedding_gradient(grad, types, count, scale):
    dt = grad.dtype
    grad, types = grad.detach().cpu().double(), types.cpu()
    val = torch.zeros(count, grad.shape[1], dtype=torch.float64)
    err = torch.zeros_like(val)
    for t, rows in rows_of(types, count):
        if len(rows):
            val[t], err[t] = grad[rows].sum(0) * scale, dot_error(len(rows), grad[rows].abs().sum(0) * abs(scale))
    return val, err + rounded(val, dt)


def check(got, val, err, what=""):
    got = got.detach().cpu().double()
    assert got.shape == val.shape, (what, got.shape, val.shape)
    off = (got - val).abs() - err
    worst = off.max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {(off > 0).sum().item()} of {off.numel()} are off by up to {worst} more than allowed"
    assert torch.isfinite(got).all() or not torch.isfinite(val).all(), what
