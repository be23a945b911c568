"""The operators whose parameters are chosen row by row on the GPU, against their definitions in 64 bits."""

import pytest
import torch

import openequivariance_amd as oeq
from tests import typed_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(gen, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(*shape, generator=gen) * by).to(dtype).cuda()


def draw_types(gen, rows, count, outside=0.1):
    """Uneven shares, some types without rows, some rows without a type (negative or too large)."""
    if count == 0:
        return torch.full((rows,), -1).cuda()
    types = (torch.rand(rows, generator=gen) ** 2 * count).long().clamp(max=count - 1)
    if count > 2:
        types[types == count // 2] = 0
    away = torch.rand(rows, generator=gen)
    types[away < outside] = -1
    types[away < outside / 2] = count
    return types.cuda()


# ---------------------------------------------------------------------------------------------------------------------
# the index
# ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [0, 1, 63, 65, 1023, 8191, 8192, 8193, 20000, 32769, 300001])
@pytest.mark.parametrize("count", [0, 1, 3, 255, 256, 65535, 65536, 70001])
def test_group_rows(rows, count):
    gen = torch.Generator().manual_seed(rows + count)
    for types in (draw_types(gen, rows, count), torch.full((rows,), count // 2).cuda(),
                  torch.randint(-2, count + 2, (rows,), generator=gen).cuda()):
        groups = oeq.group_rows(types, count)
        order, ptr = O.order_of(types.cpu(), count)
        assert torch.equal(groups.order.cpu(), order) and torch.equal(groups.ptr.cpu(), ptr)
        assert groups.types is types


def test_group_rows_of_far_types_and_strided_ones():
    types = torch.tensor([1 << 40, -(1 << 40), 3, (1 << 32) + 1, 1, 3], device="cuda")
    groups = oeq.group_rows(types, 4)
    assert groups.order.tolist() == [4, 2, 5, 0, 1, 3] and groups.ptr.tolist() == [0, 0, 1, 1, 3]
    wide = torch.stack([types, types.flip(0)], dim=1)
    assert torch.equal(oeq.group_rows(wide[:, 0], 4).order, groups.order)
    with pytest.raises(RuntimeError, match="Dtype mismatch"):
        oeq.group_rows(types.int(), 4)
    with pytest.raises(RuntimeError, match="Shape mismatch"):
        oeq.group_rows(wide, 4)
    with pytest.raises(RuntimeError, match="number of types"):
        oeq.group_rows(types, -1)


# ---------------------------------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,count,channels", [(0, 5, 8), (1, 1, 1), (61, 10, 64), (300, 7, 131), (1000, 2, 24), (4001, 9000, 40),
                                                 (20000, 3, 8), (257, 70000, 16), (5, 0, 8), (5, 3, 0), (700, 12, 2056)])
def test_embedding(rows, count, channels, dtype):
    gen = torch.Generator().manual_seed(rows)
    weight = normal(gen, count, channels, dtype=dtype).requires_grad_()
    types, grad = draw_types(gen, rows, count), normal(gen, rows, channels, dtype=dtype)
    out = oeq.type_embedding(types, weight, scale=0.3)
    known = (types >= 0) & (types < count)
    want = torch.zeros(rows, channels, device="cuda", dtype=dtype)
    want[known] = (weight.detach()[types[known]].float() * 0.3).to(dtype)
    assert torch.equal(out, want)
    got, = torch.autograd.grad(out, weight, grad)
    O.check(got, *O.embedding_gradient(grad, types, count, 0.3), "gradient")
    again, = torch.autograd.grad(oeq.type_embedding(oeq.group_rows(types, count), weight, scale=0.3), weight, grad)
    assert torch.equal(got, again)


def test_embedding_of_strided_tables_and_gradients():
    gen = torch.Generator().manual_seed(3)
    wide, types = normal(gen, 9, 50), draw_types(gen, 200, 9)
    for part in (wide[:, 2:34], wide[:, 1:34], wide.t()[:9, :5]):
        table = part.detach().requires_grad_()
        out = oeq.type_embedding(types, table)
        known = (types >= 0) & (types < 9)
        assert torch.equal(out[known], part[types[known]]) and not out[~known].any()
        for grad in (normal(gen, 200, 2 * part.shape[1])[:, ::2], normal(gen, 1, part.shape[1]).expand(200, -1)):
            got, = torch.autograd.grad(out, table, grad, retain_graph=True)
            O.check(got, *O.embedding_gradient(grad, types, 9, 1.0))


def test_embedding_twice_differentiable():
    gen = torch.Generator().manual_seed(4)
    weight, types = normal(gen, 4, 8).requires_grad_(), draw_types(gen, 30, 4)
    grad = normal(gen, 30, 8).requires_grad_()
    dw, = torch.autograd.grad(oeq.type_embedding(types, weight, scale=2.0), weight, grad, create_graph=True)
    cot = normal(gen, 4, 8)
    back, = torch.autograd.grad(dw, grad, cot)
    assert torch.equal(back, oeq.type_embedding(types, cot, scale=2.0))


# ---------------------------------------------------------------------------------------------------------------------
# linear layers
# ---------------------------------------------------------------------------------------------------------------------

SHAPES = [  # rows, components, types, in, out, bias
    (1, 0, 1, 1, 1, True), (1, 0, 5, 64, 64, False), (17, 0, 3, 8, 8, True), (63, 0, 64, 256, 96, False), (65, 0, 2, 72, 40, True),
    (129, 0, 1, 128, 128, False), (300, 3, 4, 64, 128, False), (200, 5, 10, 131, 93, True), (777, 0, 7, 131, 93, True),
    (1000, 0, 3, 512, 264, True), (257, 1, 2, 20, 300, False), (40, 7, 3, 136, 24, False), (2500, 0, 1, 64, 32, True),
    (1500, 2, 2, 32, 64, False), (600, 0, 40, 200, 520, True), (30, 0, 3, 4, 2, False), (2100, 0, 2, 640, 768, False),
    (300, 0, 63, 72, 40, False), (300, 0, 65, 72, 40, True), (900, 2, 300, 40, 24, False)]


def linear_case(rows, components, count, inner, outer, bias, dtype, seed=0, outside=0.1):
    gen = torch.Generator().manual_seed(seed + rows)
    part = (components,) if components else ()
    x = normal(gen, rows, *part, inner, dtype=dtype)
    weight = normal(gen, count, outer, inner, dtype=dtype, by=inner ** -0.5)
    b = normal(gen, count, outer, dtype=dtype) if bias else None
    return x, weight, draw_types(gen, rows, count, outside), b, normal(gen, rows, *part, outer, dtype=dtype)


def compare_linear(x, weight, types, bias, grad, index=None):
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    out = oeq.typed_linear(leaves[0], leaves[1], index if index is not None else types, leaves[2] if bias is not None else None)
    val, err = O.linear(x, weight, types, bias, grad)
    O.check(out, val["out"], err["out"], "out")
    grads = torch.autograd.grad(out, leaves, grad)
    for name, g in zip(("dx", "dw", "db"), grads):
        O.check(g, val[name], err[name], name)
    with torch.no_grad():  # the forms of serving
        O.check(oeq.typed_linear(x, weight, types, bias), val["out"], err["out"], "out without gradients")
    return (out.detach(), *grads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(shape, dtype):
    x, weight, types, bias, grad = linear_case(*shape, dtype)
    first = compare_linear(x, weight, types, bias, grad)
    again = compare_linear(x, weight, types, bias, grad, oeq.group_rows(types, shape[2]))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 33, 64, 65, 200])
def test_linear_of_few_rows(rows, dtype):
    for inner, outer, count, bias in ((2048, 48, 5, True), (520, 1000, 3, False), (40, 72, 30, False), (100, 33, 4, True)):
        compare_linear(*linear_case(rows, 0, count, inner, outer, bias, dtype, outside=0.2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_views(dtype):
    """Blocks of wider features, transposed and expanded weights, gradients that are views."""
    gen = torch.Generator().manual_seed(5)
    x, weight, types, bias, grad = linear_case(150, 3, 4, 64, 72, True, dtype)
    wide = torch.cat([x.flatten(1), normal(gen, 150, 40, dtype=dtype)], dim=1)
    base = compare_linear(x, weight, types, bias, grad)
    block = wide[:, :192].view(150, 3, 64)
    assert not block.is_contiguous()
    turned = weight.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(x).copy_(x)  # begins off 16 bytes
    for args in ((block, weight, grad), (x, turned, grad), (odd, weight, grad), (x.transpose(0, 1).contiguous().transpose(0, 1), weight, grad)):
        got = compare_linear(args[0], args[1], types, bias, args[2])
        assert all(torch.allclose(a.float(), b.float(), rtol=1e-2, atol=1e-2) for a, b in zip(got, base))
    compare_linear(x, weight[:1].expand(4, -1, -1), types, bias, grad[:1].expand(150, -1, -1))
    compare_linear(x[..., ::2], weight[..., ::2], types, bias, grad)
    compare_linear(x.transpose(0, 1).contiguous()[:, :3].transpose(0, 1).contiguous(), weight, types[:3], bias, grad[:3])


@pytest.mark.parametrize("rows,components,count,inner,outer", [(0, 0, 3, 8, 8), (5, 0, 0, 8, 8), (5, 0, 3, 0, 8), (5, 0, 3, 8, 0),
                                                               (5, 4, 3, 0, 4), (0, 2, 2, 3, 4)])
def test_linear_of_nothing(rows, components, count, inner, outer):
    part = (components,) if components else ()
    x, weight = torch.ones(rows, *part, inner, device="cuda"), torch.ones(count, outer, inner, device="cuda")
    types, bias = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.ones(count, outer, device="cuda")
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    out = oeq.typed_linear(x, weight, types, bias)
    assert out.shape == (rows, *part, outer)
    assert torch.equal(out, torch.full_like(out, float(inner + 1) if count else 0.0))
    dx, dw, db = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert torch.equal(dx, torch.full_like(dx, float(outer) if count else 0.0))
    if count:
        n = rows * max(1, components)
        assert (dw[0] == n).all() and not dw[1:].any() and (db[0] == n).all() and not db[1:].any()


def test_linear_of_no_components():
    x, weight = torch.ones(5, 0, 8, device="cuda", requires_grad=True), torch.ones(2, 3, 8, device="cuda", requires_grad=True)
    bias, types = torch.ones(2, 3, device="cuda", requires_grad=True), torch.zeros(5, dtype=torch.int64, device="cuda")
    out = oeq.typed_linear(x, weight, types, bias)
    assert out.shape == (5, 0, 3)
    dx, dw, db = torch.autograd.grad(out, (x, weight, bias), torch.ones_like(out))
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_rows_without_a_type_have_no_influence():
    """Whatever such rows and the matrices of types without rows hold; nor do rows of one type reach another's results."""
    for dtype in DTYPES:
        x, weight, types, bias, grad = linear_case(400, 0, 6, 96, 80, True, dtype)
        clean = compare_linear(x, weight, types, bias, grad)
        away = (types < 0) | (types >= 6)
        weight[3], bias[3] = float("nan"), float("inf")  # (no row has type 3)
        x[away], grad[away] = float("nan"), float("inf")
        assert away.any() and not (types == 3).any()
        leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
        out = oeq.typed_linear(leaves[0], leaves[1], types, leaves[2])
        got = (out.detach(),) + torch.autograd.grad(out, leaves, grad)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        x[types == 1] = float("nan")
        out = oeq.typed_linear(leaves[0].detach().copy_(x).requires_grad_(), leaves[1], types, leaves[2])
        dw, = torch.autograd.grad(out, leaves[1], grad)
        assert torch.isnan(out[types == 1]).all() and torch.equal(out[types != 1], clean[0][types != 1])
        assert torch.isnan(dw[1]).all() and torch.equal(dw[0], clean[2][0]) and torch.equal(dw[2:], clean[2][2:])


def test_linear_with_a_type_of_many_rows():
    """Sums over many shares of one type's rows."""
    for dtype in DTYPES:
        x, weight, types, bias, grad = linear_case(30001, 0, 2, 40, 24, True, dtype, outside=0.01)
        compare_linear(x, weight, types, bias, grad)
        x, weight, types, bias, grad = linear_case(3000, 3, 5, 72, 40, False, dtype)
        compare_linear(x, weight, types, bias, grad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_with_one_frequent_type_of_many(dtype):
    """Types whose tiles fill the card together, of which two have most of the rows, next to each other in the index."""
    x, weight, types, _, grad = linear_case(13001, 0, 80, 392, 392, False, dtype)
    types[:] = torch.where(torch.arange(13001, device="cuda") % 4 == 0, types, 40 + torch.arange(13001, device="cuda") % 3 % 2)
    compare_linear(x, weight, types, None, grad)
    compare_linear(x[:, :131], weight[:, :65, :131], types, None, grad[:, :65])


def test_far_offsets():
    """Rows, and matrices, that begin past 2^31 elements of their tensor."""
    table = torch.zeros(9, 1 << 28, device="cuda", dtype=torch.float16)
    table[8, :64] = torch.arange(64)
    types = torch.tensor([8, 0, 8], device="cuda")
    part = table[:, :64]
    assert torch.equal(oeq.type_embedding(types, part)[0], part[8])
    weight = table.view(9, 1 << 14, 1 << 14)[:, :8, :64]  # [types, 8, 64], 2^28 elements apart
    for rows in (3, 200):
        x = torch.ones(rows, 64, device="cuda", dtype=torch.float16)
        out = oeq.typed_linear(x, weight, torch.full((rows,), 8, device="cuda"))
        assert (out[:, 0] == 2016).all() and not out[:, 1:].any()
    out = oeq.typed_linear(table[:, :64], torch.ones(1, 8, 64, device="cuda", dtype=torch.float16), torch.zeros(9, dtype=torch.int64, device="cuda"))
    assert (out[8] == 2016).all() and not out[:8].any()
    w = torch.ones(1, 8, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    grad = torch.ones(9, 8, device="cuda", dtype=torch.float16)
    got, = torch.autograd.grad(oeq.typed_linear(table[:, :64], w, torch.zeros(9, dtype=torch.int64, device="cuda")), w, grad)
    assert torch.equal(got[0, 0], table[8, :64])


def test_linear_second_derivatives():
    """As a model trained on forces takes them, against the same in 64 bits."""
    x, weight, types, bias, grad = linear_case(90, 3, 4, 24, 40, True, torch.float32)

    def plain(x, w, b):
        at = types.cpu()
        known = (at >= 0) & (at < 4)
        safe = torch.where(known, at, 0)
        y = torch.einsum("nci,noi->nco", x, w[safe]) + b[safe][:, None]
        return y * known[:, None, None]

    def second(fn, x, w, b, g):
        leaves = [t.requires_grad_() for t in (x, w, b, g)]
        first = torch.autograd.grad(fn(x, w, b), leaves[:3], g, create_graph=True)
        return torch.autograd.grad(sum((t * t).sum() for t in first), leaves[:2] + leaves[3:])

    want = second(plain, *(t.detach().cpu().double() for t in (x, weight, bias, grad)))
    got = second(lambda a, w, b: oeq.typed_linear(a, w, types, b), *(t.detach().clone() for t in (x, weight, bias, grad)))
    for a, b in zip(got, want):
        # three sums in a row of up to 270 terms in 32 bits: 1e-4 of the largest is 800 units
        assert (a.cpu().double() - b).abs().max() <= 1e-4 * b.abs().max()


def test_gradients_against_differences():
    """Of a loss in 64 bits from outputs in 32: central differences with a step of 2^-6, exact for what is linear."""
    x, weight, types, bias, grad = linear_case(70, 0, 3, 16, 24, True, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
    grads = torch.autograd.grad(oeq.typed_linear(leaves[0], leaves[1], types, leaves[2]), leaves, grad)
    gen = torch.Generator().manual_seed(6)
    for i, g in enumerate(grads):
        way = normal(gen, *g.shape)
        sides = []
        for sign in (1, -1):
            moved = [t.detach() + sign * 2.0 ** -6 * way if j == i else t.detach() for j, t in enumerate(leaves)]
            sides.append((oeq.typed_linear(moved[0], moved[1], types, moved[2]).double() * grad.double()).sum())
        along = (g.double() * way.double()).sum()
        # 1 680 outputs of size up to 10, each off by up to 32 2^-23 10: 4e-5 each, in quadrature 2e-3, over the step 2^-5
        assert abs((sides[0] - sides[1]) * 32 - along) <= 0.1 + 1e-4 * abs(along)


# ---------------------------------------------------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------------------------------------------------


def adapter_case(rows, count, inner, outer, rank, dtype, seed=0, outside=0.2, by=1.0):
    gen = torch.Generator().manual_seed(seed + rows)
    x, weight = normal(gen, rows, inner, dtype=dtype, by=by), normal(gen, outer, inner, dtype=dtype, by=inner ** -0.5)
    down = normal(gen, count, rank, inner, dtype=dtype, by=inner ** -0.5)
    up = normal(gen, count, outer, rank, dtype=dtype, by=rank ** -0.5 if rank else 1.0)
    scale = (torch.arange(count, device="cuda") % 3 - 1.0) * 1.5  # (one third of the adapters has scale 0)
    return x, weight, down, up, draw_types(gen, rows, count, outside), scale, normal(gen, rows, outer, dtype=dtype)


def compare_adapters(x, weight, down, up, types, scale, grad, index=None):
    leaves = [t.detach().requires_grad_() for t in (x, weight, down, up)]
    out = oeq.adapter_linear(*leaves, index if index is not None else types, scale=scale)
    val, err = O.adapters(x, weight, down, up, types, scale, grad)
    O.check(out, val["out"], err["out"], "out")
    grads = torch.autograd.grad(out, leaves, grad)
    for name, g in zip(("dx", "dweight", "ddown", "dup"), grads):
        O.check(g, val[name], err[name], name)
    with torch.no_grad():
        O.check(oeq.adapter_linear(x, weight, down, up, types, scale=scale), val["out"], err["out"], "out without gradients")
    return (out.detach(), *grads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,count,inner,outer,rank", [
    (1, 1, 8, 8, 1), (5, 3, 64, 128, 8), (48, 32, 256, 192, 16), (64, 2, 100, 36, 6), (65, 4, 128, 128, 4), (333, 5, 131, 67, 6),
    (500, 3, 512, 264, 64), (150, 1, 64, 520, 128), (20, 2, 1024, 48, 130), (700, 40, 72, 80, 20), (33, 4, 40, 40, 0), (20, 0, 64, 72, 8),
    (300, 0, 64, 72, 8), (400, 63, 64, 72, 8), (400, 70, 64, 72, 8), (100, 2, 64, 72, 8), (129, 2, 64, 72, 8)])
def test_adapters(rows, count, inner, outer, rank, dtype):
    case = adapter_case(rows, count, inner, outer, rank, dtype)
    first = compare_adapters(*case)
    again = compare_adapters(*case, oeq.group_rows(case[4], count))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("by", [1e-4, 300.0])
def test_adapters_of_small_and_large_rows_in_half_precision(by):
    """What lies between the thin products leaves float16's range on either side, or its precision."""
    for rows in (40, 300):
        x, weight, down, up, types, scale, grad = adapter_case(rows, 3, 256, 64, 16, torch.float16, by=by)
        down = (down.float() * (1e-2 if by < 1 else 40.0)).half()  # u about 1e-6 or 1e4, with some past 65 504
        up = (up.float() * (1.0 if by < 1 else 1e-3)).half()
        leaves = [t.detach().requires_grad_() for t in (x, weight, down, up)]
        out = oeq.adapter_linear(*leaves, types, scale=scale * 8)
        val, err = O.adapters(x, weight, down, up, types, scale * 8, grad * 1e-3)
        O.check(out, val["out"], err["out"], "out")
        for name, g in zip(("dx", "dweight", "ddown", "dup"), torch.autograd.grad(out, leaves, grad * 1e-3)):
            if val[name].abs().max() < 6e4:
                O.check(g, val[name], err[name], name)


def test_adapters_views_and_what_is_not_asked_for():
    for dtype in DTYPES:
        x, weight, down, up, types, scale, grad = adapter_case(130, 3, 64, 72, 8, dtype)
        turned = (x.t().contiguous().t(), weight.t().contiguous().t(), down.transpose(1, 2).contiguous().transpose(1, 2),
                  up.transpose(1, 2).contiguous().transpose(1, 2))
        compare_adapters(*turned, types, scale, grad.t().contiguous().t())
        down.requires_grad_()
        out = oeq.adapter_linear(x, weight, down, up, types)
        val, err = O.adapters(x, weight, down, up, types, None, grad)
        O.check(out, val["out"], err["out"])
        out.backward(grad)
        O.check(down.grad, val["ddown"], err["ddown"])
        assert x.grad is None and weight.grad is None and up.grad is None


# ---------------------------------------------------------------------------------------------------------------------
# together, and around them
# ---------------------------------------------------------------------------------------------------------------------


class Model(torch.nn.Module):
    """Species' embedding, self connections of scalars and vectors by species, a projection with an adapter by data set."""

    def __init__(self, gen, species, sets, c):
        super().__init__()
        shapes = dict(table=(species, c), scalars=(species, c, c), vectors=(species, c, c), bias=(species, c), shared=(c, c),
                      down=(sets, 8, c), up=(sets, c, 8))
        for name, shape in shapes.items():
            self.register_parameter(name, torch.nn.Parameter(torch.randn(shape, generator=gen) * shape[-1] ** -0.5))

    def forward(self, species, sets, vectors):
        kinds = oeq.group_rows(species, self.table.shape[0])
        s = oeq.type_embedding(kinds, self.table, scale=2.0)
        s = s + torch.tanh(oeq.typed_linear(s, self.scalars, kinds, self.bias))
        v = oeq.typed_linear(vectors, self.vectors, kinds)
        return oeq.adapter_linear(s, self.shared, self.down, self.up, sets) + v.square().sum(1)


def plain_model(p, species, sets, vectors):
    known, at = (species >= 0)[:, None], species.clamp(min=0)
    s = torch.where(known, p["table"][at] * 2.0, 0.0)
    s = s + torch.tanh(torch.where(known, torch.einsum("ni,noi->no", s, p["scalars"][at]) + p["bias"][at], 0.0))
    v = torch.where(known[:, None], torch.einsum("nci,noi->nco", vectors, p["vectors"][at]), 0.0)
    thin = torch.einsum("ni,nri->nr", s, p["down"][sets.clamp(min=0)])
    delta = torch.where((sets >= 0)[:, None], torch.einsum("nr,nor->no", thin, p["up"][sets.clamp(min=0)]), 0.0)
    return s @ p["shared"].t() + delta + v.square().sum(1)


def model_case(rows=500):
    gen = torch.Generator().manual_seed(7)
    model = Model(gen, 9, 3, 64)
    species, sets = torch.randint(-1, 9, (rows,), generator=gen), torch.randint(-1, 3, (rows,), generator=gen)
    return model, species, sets, torch.randn(rows, 3, 64, generator=gen)


def test_a_model_of_them():
    model, species, sets, vectors = model_case()
    p = {n: t.detach().double().requires_grad_() for n, t in model.named_parameters()}
    loss = plain_model(p, species, sets, vectors.double()).square().sum()
    want = torch.autograd.grad(loss, list(p.values()))
    model = model.cuda()
    model(species.cuda(), sets.cuda(), vectors.cuda()).square().sum().backward()
    for (name, t), w in zip(model.named_parameters(), want):
        # five sums of up to 1 500 terms one behind the other: 2e-5 of the largest is 170 units
        assert (t.grad.cpu().double() - w).abs().max() <= 2e-5 * w.abs().max(), name


def test_training_step_in_a_graph():
    """Captured, replayed with new inputs and the program's own work between, equal to the eager step every time."""
    model, species, sets, vectors = model_case(3000)
    model = model.cuda()
    species, sets, vectors = species.cuda(), sets.cuda(), vectors.cuda()

    def step():
        out = model(species, sets, vectors)
        return (out.detach(),) + torch.autograd.grad(out, list(model.parameters()), out.detach())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        gen = torch.Generator().manual_seed(20 + i)
        species.copy_(torch.randint(-1, 9, species.shape, generator=gen))
        sets.copy_(torch.randint(-1, 3, sets.shape, generator=gen))
        vectors.copy_(torch.randn(vectors.shape, generator=gen))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), i


def test_two_graphs_and_a_side_stream():
    """Serving steps captured on two streams and replayed side by side: nothing is shared between them."""
    cases = [adapter_case(48, 8, 512, 256, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [oeq.adapter_linear(*c[:5], scale=c[5]) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(oeq.adapter_linear(*c[:5], scale=c[5]))
        graphs.append(graph)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_autocast():
    x, weight, types, bias, grad = linear_case(100, 0, 3, 64, 64, True, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = oeq.typed_linear(x, weight, types, bias)
        both = oeq.adapter_linear(x, weight[0], weight[:, :8], weight[:, :, :8], types)
    assert out.dtype == torch.bfloat16 and both.dtype == torch.bfloat16
    assert torch.equal(out, oeq.typed_linear(x.bfloat16(), weight.bfloat16(), types, bias.bfloat16()))
    leaf = weight.detach().requires_grad_()
    with torch.autocast("cuda", dtype=torch.float16):
        loss = oeq.typed_linear(x, leaf, types, bias).float().square().sum()
    assert torch.autograd.grad(loss, leaf)[0].dtype == torch.float32


def test_compiled():
    model, species, sets, vectors = model_case(100)
    model, args = model.cuda(), (species.cuda(), sets.cuda(), vectors.cuda())
    want = model(*args)
    got = torch.compile(model, backend="aot_eager", fullgraph=True)(*args)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
    got.sum().backward()
    assert model.table.grad is not None


def test_refusals():
    x, weight, types, bias, grad = linear_case(10, 0, 3, 16, 24, True, torch.float32)
    good = oeq.group_rows(types, 3)
    for args, text in (((x.double(), weight.double(), types), "float32, float16 or bfloat16"), ((x, weight.half(), types), "Dtype mismatch"),
                       ((x[0], weight, types), "Shape mismatch for tensor 'x'"), ((x, weight[0], types), "Shape mismatch for tensor 'weight'"),
                       ((x, weight[..., :8], types), "Shape mismatch for tensor 'weight'"), ((x, weight, types[:5]), "Shape mismatch for tensor 'types'"),
                       ((x, weight, types.int()), "Dtype mismatch for tensor 'types'"), ((x, weight, types.cpu()), "not on the GPU"),
                       ((x, weight, types, bias[:, :3]), "Shape mismatch for tensor 'bias'"), ((x, weight, types, bias.half()), "Dtype mismatch for tensor 'bias'"),
                       ((x, weight[:2], good), "Shape mismatch for tensor 'ptr'"), ((x, weight, good._replace(order=good.order.long())), "Dtype mismatch for tensor 'order'"),
                       ((x, weight, good._replace(order=None)), "both 'order' and 'ptr'")):
        with pytest.raises(RuntimeError, match=text):
            oeq.typed_linear(*args)
    with pytest.raises(RuntimeError, match="Shape mismatch for tensor 'weight'"):
        oeq.type_embedding(types, weight)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        oeq.type_embedding(types, weight[0].double())
    a = adapter_case(10, 3, 16, 24, 4, torch.float32)
    for change, text in ({0: a[0].half()}, "Dtype mismatch"), ({1: a[1][:, :8]}, "tensor 'weight'"), ({2: a[2][..., :8]}, "tensor 'down'"), \
            ({3: a[3][:, :8]}, "tensor 'up'"), ({3: a[3][:2]}, "tensor 'up'"), ({4: a[4][:3]}, "tensor 'adapters'"):
        args = [change.get(i, t) for i, t in enumerate(a[:5])]
        with pytest.raises(RuntimeError, match=text):
            oeq.adapter_linear(*args)
    for bad, text in ((a[5].double(), "Dtype mismatch for tensor 'scale'"), (a[5][:2], "tensor 'scale'")):
        with pytest.raises(RuntimeError, match=text):
            oeq.adapter_linear(*a[:5], scale=bad)
    with pytest.raises(RuntimeError, match="scales have no gradient"):
        oeq.adapter_linear(*a[:5], scale=a[5].clone().requires_grad_())
    down = a[2].requires_grad_()
    first, = torch.autograd.grad(oeq.adapter_linear(a[0], a[1], down, *a[3:5]).square().sum(), down, create_graph=True)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        first.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        oeq.typed_linear(fwd.make_dual(x, x), weight, types)


def test_an_index_made_by_hand_stays_inside_the_rows():
    """Numbers that are no rows and bounds that do not ascend are cut off, not followed."""
    x, weight, types, bias, grad = linear_case(50, 0, 3, 16, 24, True, torch.float32)
    order = torch.tensor([1 << 30, -5, 77] + list(range(47)), dtype=torch.int32, device="cuda")
    for ptr in ([0, 60, -3, 1 << 30], [9, 5, 2, 0], [-(1 << 31), 10, 20, 50]):
        index = oeq.RowGroups(types, order, torch.tensor(ptr, dtype=torch.int32, device="cuda"))
        w = weight.detach().requires_grad_()
        out = oeq.typed_linear(x, w, index, bias)
        assert out.shape == (50, 24) and torch.autograd.grad(out, w, grad)[0].shape == w.shape
        table = weight[:, 0].detach().requires_grad_()
        assert torch.autograd.grad(oeq.type_embedding(index, table), table, x)[0].shape == (3, 16)
