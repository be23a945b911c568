"""Calls of the operators whose parameters are chosen row by row that were once answered wrongly, against their definitions in
64 bits."""

import ctypes

import pytest
import torch

import openequivariance_amd as oeq
from openequivariance_amd import runtime as rt
from tests import typed_oracle as O
from tests.test_typed_operators_gpu import DTYPES, adapter_case, linear_case, normal

pytestmark = pytest.mark.gpu

ELEMENT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [9, 64, 65, 200])
def test_a_bias_and_a_thin_product_of_one_call_are_both_added(rows, dtype):
    """On both sides of the number of rows from which tiles are taken."""
    gen = torch.Generator().manual_seed(rows)
    count, inner, outer, rank, wide = 3, 64, 72, 6, 8
    x, w = normal(gen, rows, inner, dtype=dtype), normal(gen, count, outer, inner, dtype=dtype, by=inner ** -0.5)
    bias, up = normal(gen, count, outer, dtype=dtype), normal(gen, count, outer, rank, dtype=dtype)
    thin = torch.zeros(rows, wide, device="cuda")
    thin[:, :rank] = normal(gen, rows, rank)
    types = torch.randint(-1, count + 1, (rows,), generator=gen).cuda()
    groups, out = oeq.group_rows(types, count), torch.full((rows, outer), 7.0, device="cuda", dtype=dtype)
    a = rt._TypedRows(type=ELEMENT[dtype], rank=rank, rows=rows, parts=1, types=count, inner=inner, outer=outer, x_row_stride=inner,
                      w_type_stride=outer * inner, w_row_stride=inner, up_type_stride=outer * rank, up_outer_stride=rank, up_rank_stride=1,
                      x=x.data_ptr(), w=w.data_ptr(), bias=bias.data_ptr(), thin=thin.data_ptr(), up=up.data_ptr(),
                      type_of_row=types.data_ptr(), order=groups.order.data_ptr(), ptr=groups.ptr.data_ptr())
    rt._check(rt.load_library().oeq_typed_product(ctypes.byref(a), out.data_ptr(), torch.cuda.current_stream().cuda_stream), "product")
    val, _ = O.linear(x, w, types, bias)
    val, size = val["out"], val["out"].new_zeros(rows, outer)
    keep = 0.0 if dtype == torch.float32 else 2.0 ** -16  # (what a thin row keeps as an operand)
    err = torch.zeros_like(size)
    for t, at in O.rows_of(types.cpu(), count):
        u, b = thin[at.cuda(), :rank].cpu().double(), up[t].cpu().double()
        val[at] += u @ b.t()
        size[at] = (x[at.cuda()].cpu().double().abs() @ w[t].cpu().double().abs().t() + u.abs() @ b.abs().t()
                    + bias[t].cpu().double().abs())
        err[at] = keep * (u.abs() @ b.abs().t())
    O.check(out, val, O.dot_error(inner + rank + 1, size) + 2 * err + O.rounded(val, dtype), "out")


def plain_adapters(x, weight, down, up, types, scale):
    """The definition in 64 bits, infinities and NaN included: products one by one, so that nothing is multiplied that a row has not."""
    x, weight, down, up, scale = (t.detach().cpu().double() for t in (x, weight, down, up, scale))
    out = x @ weight.t()
    for t, at in O.rows_of(types.cpu(), down.shape[0]):
        u = scale[t] * (x[at, None, :] * down[t]).sum(-1)
        out[at] += (u[:, None, :] * up[t]).sum(-1)
    return out


def same_kind(got, want, dtype):
    """Infinities, their signs and NaN as in the definition (which is rounded to the type first)."""
    got, want = got.detach().cpu().double(), want.to(dtype).double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 300])
def test_adapters_with_infinities(rows, dtype):
    """An infinite weight of an adapter: an infinity of the product's sign, whatever is left of the operand beside it in its lower part."""
    x, weight, down, up, types, scale, grad = adapter_case(rows, 3, 64, 72, 8, dtype)
    scale = torch.tensor([1.5, -1.0, 2.0], device="cuda")
    down, up = down.clone(), up.clone()
    up[0, 5, 2], up[1, 40, 0], up[2, 71, 7], up[2, 70, 7] = float("inf"), float("-inf"), float("inf"), float("nan")
    # rows between whose products the upper part is all there is (0.5 s), or too small for float16 beside the row's largest (2^-28 s)
    x[:9], down[:, 2], types[:9] = 0, 0, torch.arange(9, device="cuda") % 3
    x[:9, 0], x[:9, 1], down[:, :, 0], down[:, 2, 1] = 0.5, 2.0 ** -14, 0.0, 2.0 ** -14
    down[:, 0, 0] = down[:, 7, 0] = 1.0
    out = oeq.adapter_linear(x, weight, down, up, types, scale=scale)
    want = plain_adapters(x, weight, down, up, types, scale)
    assert want.isinf().sum() > 20 and want[:, 70].isnan().any()
    same_kind(out, want, dtype)
    # dx: the same with the matrices of the other direction
    up = adapter_case(rows, 3, 64, 72, 8, dtype)[3]
    down[0, 3, 60], down[1, 0, 0], down[2, 1, 33] = float("-inf"), float("inf"), float("inf")
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(oeq.adapter_linear(leaf, weight, down, up, types, scale=scale), leaf, grad)
    want = plain_adapters(grad, weight.t(), up.transpose(1, 2), down.transpose(1, 2), types, scale)
    assert want.isinf().sum() > 20
    same_kind(dx, want, dtype)


@pytest.mark.parametrize("rows", [40, 300])
def test_adapters_between_whose_products_are_infinities(rows):
    """One infinite element between the thin products leaves the others as they are, past float16's range too."""
    dtype = torch.float16
    x, weight = torch.zeros(rows, 64, device="cuda", dtype=dtype), torch.zeros(72, 64, device="cuda", dtype=dtype)
    down, up = torch.zeros(1, 8, 64, device="cuda", dtype=dtype), torch.zeros(1, 72, 8, device="cuda", dtype=dtype)
    x[:] = 1000.0
    down[0, 0, 0], down[0, 1, 1:9] = float("inf"), 1000.0  # u = (inf, 8e6, 0, ..)
    up[0, :, 0], up[0, :, 1] = 1.0, -1.0
    types, scale = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.ones(1, device="cuda")
    out = oeq.adapter_linear(x, weight, down, up, types, scale=scale)
    same_kind(out, plain_adapters(x, weight, down, up, types, scale), dtype)


@pytest.mark.parametrize("rows", [40, 300])
def test_adapters_near_the_end_of_the_range(rows):
    """A sum between the thin products that is finite, but past what bfloat16 holds: 2^128 (1 - 2^-9 - 2^-10) becomes infinite when it is
    rounded to 8 bits."""
    dtype = torch.bfloat16
    x, weight = torch.zeros(rows, 64, device="cuda", dtype=dtype), torch.zeros(72, 64, device="cuda", dtype=dtype)
    down, up = torch.zeros(1, 8, 64, device="cuda", dtype=dtype), torch.zeros(1, 72, 8, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = 2.0 ** 126, 2.0 ** 118
    down[0, 0, 0], down[0, 0, 1] = 3.984375, 1.25  # 2^128 (1 - 2^-8) + 2^118 1.25
    down[0, 0, 2], x[:, 2] = 1.0, 2.0 ** 118
    up[0, :, 0] = 2.0 ** -10
    types, scale = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.ones(1, device="cuda")
    val, err = O.adapters(x, weight, down, up, types, scale)
    assert val["out"].max() < 2.0 ** 118
    O.check(oeq.adapter_linear(x, weight, down, up, types, scale=scale), val["out"], err["out"], "out")


def test_an_index_is_checked_by_the_lookup_too():
    x, weight, types, bias, grad = linear_case(10, 0, 3, 16, 24, True, torch.float32)
    table, good = weight[:, 0], oeq.group_rows(types, 3)
    for index, text in ((oeq.group_rows(types, 4), "Shape mismatch for tensor 'ptr'"), (good._replace(order=good.order[:5]), "Shape mismatch for tensor 'order'"),
                        (good._replace(order=good.order.long()), "Dtype mismatch for tensor 'order'"), (good._replace(ptr=None), "both 'order' and 'ptr'")):
        for leaf in (table, table.detach().requires_grad_()):
            with pytest.raises(RuntimeError, match=text):
                oeq.type_embedding(index, leaf)


@pytest.mark.parametrize("components", [0, 3])
def test_a_bias_gradient_differentiated_alone_has_no_other_term(components):
    """The sum of gradients by type is linear in them: its derivative is the lookup of its cotangent, whatever the rows hold."""
    x, weight, types, bias, grad = linear_case(90, components, 4, 24, 40, True, torch.float32)
    x[types == 1] = float("inf")
    leaves = [bias.detach().requires_grad_(), grad.requires_grad_()]
    db, = torch.autograd.grad(oeq.typed_linear(x, weight, types, leaves[0]), leaves[0], grad, create_graph=True)
    cot = normal(torch.Generator().manual_seed(1), 4, 40)
    back, = torch.autograd.grad(db, grad, cot)
    known = (types >= 0) & (types < 4)
    want = torch.where(known[:, None], cot[torch.where(known, types, 0)], 0.0)
    assert torch.equal(back, want[:, None].expand(-1, 3, -1) if components else want)


def test_autocast_leaves_integers_alone():
    """They are refused as without it, not computed with."""
    x, weight, types, bias, grad = linear_case(10, 0, 3, 16, 24, True, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
            oeq.typed_linear(x.long(), weight, types)
        with pytest.raises(RuntimeError, match="Dtype mismatch for tensor 'down'"):
            oeq.adapter_linear(x, weight[0], weight[:, :8].int(), weight[:, :, :8], types)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ratio", [2.0 ** 8, 2.0 ** 14, 2.0 ** 20])
@pytest.mark.parametrize("rows", [40, 300])
def test_adapters_keep_what_is_small_beside_the_rest_of_a_row(rows, ratio, dtype):
    """Between the thin products a row has an element 1 .. 2 and one `ratio` times larger; half of the columns take the small one alone."""
    gen = torch.Generator().manual_seed(rows)
    x, weight = torch.zeros(rows, 64, device="cuda", dtype=dtype), torch.zeros(72, 64, device="cuda", dtype=dtype)
    down, up = torch.zeros(1, 8, 64, device="cuda", dtype=dtype), torch.zeros(1, 72, 8, device="cuda", dtype=dtype)
    small = 1 + torch.rand(rows, generator=gen)
    x[:, 0], x[:, 1], x[:, 2] = ratio ** 0.5, small.to(dtype).cuda(), (small * 2.0 ** -9).to(dtype).cuda()
    down[0, 0, 0], down[0, 5, 1], down[0, 5, 2] = ratio ** 0.5, 1.0, 1.0
    up[0, 36:, 0], up[0, :, 5] = 1.0, normal(gen, 72, dtype=dtype)
    types, scale = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.ones(1, device="cuda")
    val, err = O.adapters(x, weight, down, up, types, scale)
    got = oeq.adapter_linear(x, weight, down, up, types, scale=scale)
    O.check(got[:, :36], val["out"][:, :36], err["out"][:, :36], "columns that take the small one")
    if ratio < 2.0 ** 16:  # (else past float16)
        O.check(got, val["out"], err["out"], "out")


@pytest.mark.parametrize("rows", [9, 300])
def test_long_sums_of_floats_are_added_up_in_parts(rows):
    """2^24 and 4 095 ones: a chain of additions in 32 bits loses every one of them (half a unit of the sum each). In parts of 512 terms at
    most the first part's ones are lost, the other parts are even numbers, which the total holds."""
    n, most = 4096, 514
    want = 2.0 ** 24 + n - 1
    x, w = torch.ones(rows, n, device="cuda"), torch.ones(1, 64, n, device="cuda")
    x[:, 0] = 2.0 ** 24
    types, leaf = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.zeros(rows, 64, device="cuda", requires_grad=True)
    assert (oeq.typed_linear(x, w, types) - want).abs().max() <= most
    dx, = torch.autograd.grad(oeq.typed_linear(leaf, w.transpose(1, 2).contiguous(), types), leaf, x)  # (n columns out, 64 in)
    assert (dx - want).abs().max() <= most
    out = oeq.adapter_linear(x, torch.zeros(64, n, device="cuda"), w[:, :4].contiguous(), torch.eye(64, 4, device="cuda")[None], types)
    assert (out[:, :4] - want).abs().max() <= most
    g, x = torch.ones(n, 64, device="cuda"), torch.ones(n, rows, device="cuda")
    x[0] = 2.0 ** 24
    w = torch.zeros(1, 64, rows, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(oeq.typed_linear(x, w, torch.zeros(n, dtype=torch.int64, device="cuda")), w, g)
    assert (dw - want).abs().max() <= most
