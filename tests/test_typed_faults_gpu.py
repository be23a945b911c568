"""Calls of the operators whose parameters are chosen row by row that were once answered wrongly, against their definitions in
64 bits."""

import ctypes

import pytest
import torch

import openequivariance_amd as oeq
from openequivariance_amd import runtime as rt
from tests import typed_oracle as O
from tests.test_typed_operators_gpu import DTYPES, normal

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
