"""What the operators whose parameters are chosen row by row are judged by: an embedding of the rows' types, a linear layer
with weights of its own for every type (species of atoms, experts of a mixture), and low-rank adapters of many requests
or data sets beside a shared projection.

A case names the operator ("op") and how far a pass goes ("run": "forward", or "train": the output and the gradients of
what is trained):

* "embedding": rows of a table by type, scaled. Trained: the table.
* "linear": a product with the weights of the row's type, on rows or on all components of an irrep of a row. Trained: the
  weights, the biases where there are any, and the layer's input.
* "adapters": the shared projection plus the two thin products of the row's adapter. Trained: the adapters and the input;
  the shared projection too where "full" is set.

Types are drawn with probabilities that fall as (1 + type) ** -skew; "outside" is the share of rows without one, and "runs"
has rows of one type next to each other, as the tokens of one request are. Whatever the operators need in order to find the rows of a
type is done within a pass.

With ``own`` false a pass is computed from elementary torch operations in 32 bits and rounded once at the end, with it
true by the calls that a program makes of this package.
"""

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------


def _embedding(run, dtype, rows, types, channels, scale, skew=0.0, outside=0.0, **name):
    return dict(op="embedding", run=run, dtype=dtype, rows=rows, types=types, channels=channels, scale=scale, skew=skew,
                outside=outside, runs=False, **name)


def _linear(run, dtype, rows, components, types, inner, outer, bias, skew=0.0, outside=0.0, **name):
    return dict(op="linear", run=run, dtype=dtype, rows=rows, components=components, types=types, inner=inner, outer=outer,
                bias=bias, skew=skew, outside=outside, runs=False, **name)


def _adapters(run, dtype, rows, types, inner, outer, rank, full, runs, skew=0.0, outside=0.0, **name):
    return dict(op="adapters", run=run, dtype=dtype, rows=rows, types=types, inner=inner, outer=outer, rank=rank, full=full,
                runs=runs, skew=skew, outside=outside, **name)


def listed():
    return [
        # the species of a few small molecules on their way into a model, where latency counts
        _embedding("forward", "float32", 61, 10, 64, 1.0, name="species-small"),
        # training step on 20 000 atoms, a few species most frequent by far
        _embedding("train", "float32", 20000, 89, 512, 0.5, skew=2.0, name="species-train"),
        # tokens that spell structures: large vocabulary, most tokens rare, some places of the batch empty
        _embedding("train", "bfloat16", 16411, 32003, 1024, 32.0, skew=1.0, outside=0.05, name="tokens-train"),
        # self connection of the vectors (l = 1) of 20 000 atoms, weights by species, the features' own type
        _linear("train", "float32", 20000, 3, 10, 128, 128, False, skew=1.0, name="species-vectors-train"),
        # a prompt through the first product of 16 experts: the largest call
        _linear("forward", "bfloat16", 32768, 0, 16, 2048, 5632, False, skew=0.5, name="experts-prompt"),
        # training step of a layer of experts on packed sequences, uneven shares
        _linear("train", "bfloat16", 16411, 0, 32, 1024, 2048, False, skew=0.7, name="experts-train"),
        # serving: one token of each of 24 sequences, most of the experts idle
        _linear("forward", "float16", 24, 0, 64, 2048, 1408, False, name="experts-tokens"),
        # readout by species with odd numbers of channels, half precision
        _linear("train", "float16", 777, 0, 7, 131, 93, True, skew=0.5, outside=0.03, name="readout-train-odd"),
        # serving: one token of each of 48 requests beside a projection they share, 32 adapters and some rows without one
        _adapters("forward", "bfloat16", 48, 32, 4096, 4096, 16, False, False, outside=0.1, name="adapters-tokens"),
        # prompts of nine requests read in at once
        _adapters("forward", "bfloat16", 8209, 9, 4096, 4096, 64, False, True, name="adapters-prompts"),
        # fine-tuning on four data sets at once, the shared projection frozen
        _adapters("train", "bfloat16", 4001, 4, 1024, 1024, 32, False, False, name="adapters-train"),
        # the same for a small readout with odd numbers of channels, shared projection trained too
        _adapters("train", "float32", 333, 5, 131, 67, 6, True, False, outside=0.1, name="adapters-train-odd"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A number of channels: most often a multiple of 8 or 64, else any."""
    n, grid = _spread(rng, lo, hi), rng.choice((1, 8, 8, 64, 64))
    return max(grid, n // grid * grid)


def draw(rng):
    """One more case of the ranges above."""
    op = rng.choice(("embedding", "linear", "linear", "adapters"))
    dtype = rng.choice(("float32", "bfloat16", "float16", "bfloat16"))
    run = rng.choice(("forward", "train"))
    skew, outside = rng.choice((0.0, 0.5, 1.0, 2.0)), rng.choice((0.0, 0.0, 0.05, 0.5))
    limit = _cost(listed()[4])
    if op == "embedding":
        case = _embedding(run, dtype, _spread(rng, 1, 32768), _spread(rng, 4, 65537), _width(rng, 8, 4096),
                          rng.choice((1.0, 0.5, 32.0)), skew, outside)
        while case["types"] * case["channels"] > 1 << 27:
            case["types"] = (case["types"] + 1) // 2
        return case
    rows, inner, outer = _spread(rng, 1, 32768), _width(rng, 16, 5632), _width(rng, 16, 5632)
    if op == "linear":
        components = rng.choice((0, 0, 0, 1, 3, 5, 7))
        case = _linear(run, dtype, rows, components, _spread(rng, 1, 128), inner, outer, rng.random() < 0.4, skew, outside)
        while case["types"] * inner * outer > 1 << 28:
            case["types"] = (case["types"] + 1) // 2
    else:
        rank = rng.choice((4, 6, 8, 16, 16, 32, 64, 128))
        case = _adapters(run, dtype, rows, _spread(rng, 1, 64), inner, outer, rank, rng.random() < 0.3, rng.random() < 0.5,
                         skew, outside)
    while case["rows"] > 1 and _cost(case) > limit:
        case["rows"] = (case["rows"] + 1) // 2
    return case


def _used(case):
    """How many types the rows have, on average over the draws of types."""
    weight = [(1 + t) ** -case["skew"] for t in range(case["types"])]
    rows = case["rows"] * (1 - case["outside"])
    return sum(-math.expm1(rows * math.log1p(-min(w / sum(weight), 1 - 1e-12))) for w in weight)


def work(case):
    s, train, n, used = _BYTES[case["dtype"]], case["run"] == "train", case["rows"], _used(case)
    some = n * (1 - case["outside"])  # rows with a type
    if case["op"] == "embedding":
        c = case["channels"]
        return {"bytes": 8 * n + (n + used) * c * s + (some + case["types"]) * c * s * train, "flops": some * c * (1 + train)}
    inner, outer = case["inner"], case["outer"]
    if case["op"] == "linear":
        k = max(1, case["components"])
        weights = used * (inner + case["bias"]) * outer
        moved = n * k * (inner + outer) * (1 + train) + weights + case["types"] * (inner + case["bias"]) * outer * train
        return {"bytes": 8 * n + moved * s, "flops": 2 * some * k * inner * outer * (1 + 2 * train)}
    thin = case["rank"] * (inner + outer)
    full = case["full"] and train
    moved = n * (inner + outer) * (1 + train) + inner * outer * (1 + full) + used * thin + case["types"] * thin * train
    return {"bytes": 8 * n + moved * s,
            "flops": 2 * n * inner * outer * (1 + train + full) + 2 * some * thin * (1 + 2 * train)}


def _cost(case):
    w, fp32 = work(case), case["dtype"] == "float32"
    return max(w["bytes"] / 4e12, w["flops"] / (8e13 if fp32 else 6e14))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, train, n, count = _DTYPES[case["dtype"]], case["run"] == "train", case["rows"], case["types"]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * by).to(dt)

    p = (1.0 + torch.arange(count, device="cuda", dtype=torch.float64)) ** -case["skew"]
    names = torch.randperm(count, generator=gen, device="cuda")  # which type is the most frequent
    ends = (p / p.sum()).cumsum(0)
    at = torch.searchsorted(ends, torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)).clamp(max=count - 1)
    at = at.sort().values if case["runs"] else at
    types = torch.where(torch.rand(n, generator=gen, device="cuda") < case["outside"], -1, names[at])
    st = {"case": case, "types": types}
    if case["op"] == "embedding":
        st["weight"] = normal(count, case["channels"]).requires_grad_(train)
        st["grad"] = normal(n, case["channels"]) if train else None
        return st
    inner, outer = case["inner"], case["outer"]
    if case["op"] == "linear":
        part = [case["components"]] if case["components"] else []
        st["x"] = normal(n, *part, inner).requires_grad_(train)
        st["weight"] = normal(count, outer, inner, by=inner ** -0.5).requires_grad_(train)
        st["bias"] = normal(count, outer).requires_grad_(train) if case["bias"] else None
        st["grad"] = normal(n, *part, outer) if train else None
        return st
    st["x"] = normal(n, inner).requires_grad_(train)
    st["weight"] = normal(outer, inner, by=inner ** -0.5).requires_grad_(train and case["full"])
    st["down"] = normal(count, case["rank"], inner, by=inner ** -0.5).requires_grad_(train)
    st["up"] = normal(count, outer, case["rank"], by=0.5 * case["rank"] ** -0.5).requires_grad_(train)
    st["scale"] = torch.tensor([2.0, 0.5, 1.0, 1.5], device="cuda")[torch.arange(count, device="cuda") % 4]
    st["grad"] = normal(n, outer) if train else None
    return st


def _trained(st):
    case = st["case"]
    if case["op"] == "embedding":
        return ["weight"]
    if case["op"] == "linear":
        return ["x", "weight"] + (["bias"] if case["bias"] else [])
    return ["x", "down", "up"] + (["weight"] if case["full"] else [])


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------


def _plain_linear(x, weight, bias, types, count):
    out = torch.zeros(*x.shape[:-1], weight.shape[1], device=x.device)
    for t in range(count):
        rows = (types == t).nonzero()[:, 0]
        y = torch.matmul(x[rows], weight[t].t())
        out = out.index_copy(0, rows, y if bias is None else y + bias[t])
    return out


def _plain_adapters(x, weight, down, up, types, scale):
    out = torch.matmul(x, weight.t())
    for a in range(down.shape[0]):
        rows = (types == a).nonzero()[:, 0]
        thin = torch.matmul(x[rows], down[a].t()) * scale[a]
        out = out.index_add(0, rows, torch.matmul(thin, up[a].t()))
    return out


def _run_plain(st):
    case, types = st["case"], st["types"]
    dt, train = _DTYPES[case["dtype"]], case["run"] == "train"
    if case["op"] == "embedding":
        known = types >= 0
        at = torch.where(known, types, 0)
        out = (st["weight"].detach()[at].float() * case["scale"]).masked_fill(~known[:, None], 0.0).to(dt)
        if not train:
            return out
        table = torch.zeros(st["weight"].shape, device="cuda")
        table.index_add_(0, at, (st["grad"].float() * case["scale"]).masked_fill(~known[:, None], 0.0))
        return out, table.to(dt)
    names = _trained(st)
    wide = {k: st[k].detach().float() for k in ("x", "weight", "bias", "down", "up") if st.get(k) is not None}
    if train:
        for k in names:
            wide[k].requires_grad_()
    if case["op"] == "linear":
        out = _plain_linear(wide["x"], wide["weight"], wide.get("bias"), types, case["types"])
    else:
        out = _plain_adapters(wide["x"], wide["weight"], wide["down"], wide["up"], types, st["scale"])
    if not train:
        return out.to(dt)
    grads = torch.autograd.grad(out, [wide[k] for k in names], st["grad"].float())
    return (out.detach().to(dt),) + tuple(g.to(dt) for g in grads)


# ---------------------------------------------------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------------------------------------------------


def _run_own(st):
    import openequivariance_amd as oeq
    case = st["case"]
    if case["op"] == "embedding":
        out = oeq.type_embedding(st["types"], st["weight"], scale=case["scale"])
    elif case["op"] == "linear":
        out = oeq.typed_linear(st["x"], st["weight"], st["types"], st["bias"])
    else:
        out = oeq.adapter_linear(st["x"], st["weight"], st["down"], st["up"], st["types"], scale=st["scale"])
    if case["run"] == "forward":
        return out
    return (out.detach(),) + torch.autograd.grad(out, [st[k] for k in _trained(st)], st["grad"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------


def _rows_by_type(types, count):
    """{type: its rows}, from the host."""
    rows = {}
    for i, t in enumerate(types.tolist()):
        if 0 <= t < count:
            rows.setdefault(t, []).append(i)
    return {t: torch.tensor(r, device="cuda") for t, r in rows.items()}


def exact(case, seed):
    st = prepare(case, seed)
    train = case["run"] == "train"
    groups = _rows_by_type(st["types"], case["types"])
    g = st["grad"].double() if train else None
    if case["op"] == "embedding":
        w = st["weight"].detach()
        out = torch.zeros(case["rows"], w.shape[1], device="cuda", dtype=torch.float64)
        dw = torch.zeros(w.shape, device="cuda", dtype=torch.float64) if train else None
        for t, rows in groups.items():
            out[rows] = w[t].double() * case["scale"]
            if train:
                dw[t] = g[rows].sum(0) * case["scale"]
        return (out, dw) if train else out
    x = st["x"].detach().double()
    if case["op"] == "linear":
        w = st["weight"].detach()
        out = torch.zeros(*x.shape[:-1], w.shape[1], device="cuda", dtype=torch.float64)
        if train:
            dx, dw = torch.zeros_like(x), torch.zeros(w.shape, device="cuda", dtype=torch.float64)
            db = torch.zeros(w.shape[:2], device="cuda", dtype=torch.float64)
        for t, rows in groups.items():
            wt, xt = w[t].double(), x[rows].reshape(-1, x.shape[-1])
            y = xt @ wt.t()
            if st["bias"] is not None:
                y += st["bias"].detach()[t].double()
            out[rows] = y.view(len(rows), *x.shape[1:-1], -1)
            if train:
                gt = g[rows].reshape(-1, g.shape[-1])
                dx[rows] = (gt @ wt).view(len(rows), *x.shape[1:])
                dw[t], db[t] = gt.t() @ xt, gt.sum(0)
        if not train:
            return out
        return (out, dx, dw) + ((db,) if case["bias"] else ())
    w, scale = st["weight"].detach().double(), st["scale"].double()
    out = x @ w.t()
    if train:
        dx = g @ w
        ddown, dup = (torch.zeros(st[k].shape, device="cuda", dtype=torch.float64) for k in ("down", "up"))
    for a, rows in groups.items():
        down, up, xa = st["down"].detach()[a].double(), st["up"].detach()[a].double(), x[rows]
        out[rows] += scale[a] * ((xa @ down.t()) @ up.t())
        if train:
            ga = scale[a] * g[rows]
            back = ga @ up
            dx[rows] += back @ down
            ddown[a], dup[a] = back.t() @ xa, ga.t() @ (xa @ down.t())
    if not train:
        return out
    return (out, dx, ddown, dup) + ((g.t() @ x,) if case["full"] else ())
