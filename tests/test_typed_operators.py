"""What of the operators whose parameters are chosen row by row needs no GPU: the oracle's gradients against differences, shapes
of traced calls and the refusals of the C ABI."""

import ctypes

import pytest
import torch

import openequivariance_amd as oeq
from openequivariance_amd import runtime as rt
from tests import typed_oracle as O


def along(fn, tensors, i, way, grad, step=1e-5):
    sides = []
    for sign in (1, -1):
        moved = [t + sign * step * way if j == i else t for j, t in enumerate(tensors)]
        sides.append((fn(*moved) * grad).sum())
    return (sides[0] - sides[1]) / (2 * step)


def test_oracle_gradients_against_differences():
    """The formulas that the kernels' gradients are compared with, in 64 bits. (The functions are of the second degree in all
    operands together: central differences of one of them are exact but for 1e-16 / step.)"""
    gen = torch.Generator().manual_seed(1)
    x, w, b, g = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((7, 2, 5), (3, 4, 5), (3, 4), (7, 2, 4)))
    types = torch.tensor([0, 2, 2, -1, 0, 2, 3])
    val, _ = O.linear(x, w, types, b, g)
    assert not val["out"][3].any() and not val["out"][6].any() and not val["dw"][1].any()
    for i, name in enumerate(("dx", "dw", "db")):
        way = torch.randn(val[name].shape, generator=gen, dtype=torch.float64)
        got = along(lambda x, w, b: O.linear(x, w, types, b)[0]["out"], (x, w, b), i, way, g)
        assert abs(got - (val[name] * way).sum()) <= 1e-8, name
    x, w, down, up, g = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((7, 5), (4, 5), (3, 2, 5), (3, 4, 2), (7, 4)))
    scale = torch.tensor([1.0, 0.0, -2.0])
    val, _ = O.adapters(x, w, down, up, types, scale, g)
    assert torch.allclose(val["out"][3], w @ x[3])
    for i, name in enumerate(("dx", "dweight", "ddown", "dup")):
        way = torch.randn(val[name].shape, generator=gen, dtype=torch.float64)
        got = along(lambda *t: O.adapters(*t, types, scale)[0]["out"], (x, w, down, up), i, way, g)
        assert abs(got - (val[name] * way).sum()) <= 1e-8, name
    g = torch.randn(7, 4, generator=gen, dtype=torch.float64)
    dw, _ = O.embedding_gradient(g, types, 3, 0.5)
    assert torch.allclose(dw[2], 0.5 * (g[1] + g[2] + g[5])) and not dw[1].any()


def test_traced_calls_have_the_kernels_shapes():
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, device="meta", dtype=dtype)

    types = empty(7, dtype=torch.int64)
    groups = oeq.group_rows(types, 5)
    assert groups.order.shape == (7,) and groups.ptr.shape == (6,) and groups.ptr.dtype == torch.int32
    assert oeq.type_embedding(groups, empty(5, 12)).shape == (7, 12)
    assert oeq.typed_linear(empty(7, 3, 8), empty(5, 12, 8), types).shape == (7, 3, 12)
    assert oeq.typed_linear(empty(7, 8), empty(5, 12, 8), groups, empty(5, 12)).shape == (7, 12)
    out = oeq.adapter_linear(empty(7, 8), empty(12, 8), empty(5, 3, 8), empty(5, 12, 3), types)
    assert out.shape == (7, 12) and out.dtype == torch.bfloat16
    grads = torch.ops.oeq_amd.typed_linear_backward(empty(7, 12), empty(7, 8), empty(5, 12, 8), types, None, None, True, False, True)
    assert [tuple(t.shape) for t in grads] == [(7, 8), (0,), (5, 12)]
    out, thin = torch.ops.oeq_amd.adapter_linear(empty(7, 8), empty(12, 8), empty(5, 3, 8), empty(5, 12, 3), types, None, None, None)
    assert thin.shape == (7, 8) and thin.dtype == torch.float32
    grads = torch.ops.oeq_amd.adapter_linear_backward(out, empty(7, 8), empty(12, 8), empty(5, 3, 8), empty(5, 12, 3), types, None, thin,
                                                      None, None, False, True, True, True)
    assert [tuple(t.shape) for t in grads] == [(0,), (12, 8), (5, 3, 8), (5, 12, 3)]


def refused(rc, text):
    message = rt.load_library().oeq_last_error().decode()
    assert rc == -1 and text in message, (rc, message)


def test_c_abi_refuses_indices():
    """Checked on the host before anything is launched (the addresses are never read)."""
    lib = rt.load_library()
    for args, text in (((-1, 3, 16, 16, 16, None, 0, None), "rows"), ((3, -1, 16, 16, 16, None, 0, None), "types"),
                       ((3, 1 << 24, 16, 16, 16, None, 0, None), "types"), ((1 << 30, 3, 16, 16, 16, None, 0, None), "rows"),
                       ((3, 3, None, 16, 16, None, 0, None), "NULL"), ((3, 3, 16, 16, None, None, 0, None), "NULL"),
                       ((100000, 3, 16, 16, 16, None, 0, None), "workspace"), ((100000, 3, 16, 16, 16, 16, 64, None), "workspace")):
        refused(lib.oeq_group_rows(*args), text)
    assert lib.oeq_group_rows_workspace_bytes(100, 3) == 0
    assert lib.oeq_group_rows_workspace_bytes(100000, 3) < lib.oeq_group_rows_workspace_bytes(100000, 300)


def test_c_abi_refuses_tables():
    lib = rt.load_library()
    assert lib.oeq_type_lookup(0, 0, 3, 8, None, None, 8, 1.0, None, None) == 0
    for args, text in (((3, 2, 3, 8, 16, 16, 8, 1.0, 16, None), "element type"), ((0, -2, 3, 8, 16, 16, 8, 1.0, 16, None), "rows"),
                       ((0, 2, 3, -8, 16, 16, 8, 1.0, 16, None), "channels"), ((0, 2, 3, 8, None, 16, 8, 1.0, 16, None), "NULL"),
                       ((0, 2, 3, 8, 16, None, 8, 1.0, 16, None), "NULL"), ((0, 2, 3, 8, 16, 18, 8, 1.0, 16, None), "unaligned"),
                       ((0, 2, 3, 8, 16, 16, -8, 1.0, 16, None), "rows")):
        refused(lib.oeq_type_lookup(*args), text)
    need = lib.oeq_type_sum_workspace_bytes(1000, 3, 8)
    assert need > 0 and lib.oeq_type_sum_workspace_bytes(10, 3, 8) == 0
    good = [0, 1000, 1, 3, 8, 16, 16, 16, 16, 8, 0, 1.0, 16, 16, need, None]
    for changes, text in (({0: 5}, "element type"), ({1: -1}, "rows"), ({2: 0}, "parts"), ({3: -1}, "types"), ({4: -1}, "channels"),
                          ({5: None}, "NULL"), ({8: None}, "NULL"), ({9: -8}, "strides"), ({12: None}, "NULL"), ({14: need - 1}, "workspace"),
                          ({13: None}, "workspace"), ({8: 18}, "unaligned"), ({1: 1 << 29, 3: 1 << 23}, "too many")):
        refused(lib.oeq_type_sum(*[changes.get(i, a) for i, a in enumerate(good)]), text)


def test_c_abi_refuses_products():
    lib = rt.load_library()

    def rows(**changes):
        fields = dict(type=2, across=0, shared=0, rank=0, rows=1000, parts=1, types=3, inner=32, outer=16, x_row_stride=32, w_type_stride=512,
                      w_row_stride=32, x=16, w=16, type_of_row=16, order=16, ptr=16)
        fields.update(changes)
        return ctypes.byref(rt._TypedRows(**fields))

    assert lib.oeq_typed_product(rows(rows=0), None, None) == 0 and lib.oeq_typed_product(rows(outer=0), None, None) == 0
    refused(lib.oeq_typed_product(None, 16, None), "NULL")
    for changes, text in ((dict(type=3), "element type"), (dict(rows=-1), "rows"), (dict(rows=1 << 28, parts=4), "rows"), (dict(parts=0), "parts"),
                          (dict(types=-1), "types"), (dict(inner=-1), "inner"), (dict(outer=1 << 31), "outer"), (dict(rank=-1), "rank"),
                          (dict(rank=4, parts=2), "rank"), (dict(rank=4), "NULL"), (dict(x_row_stride=-1), "stride of -1"), (dict(x=0), "NULL"),
                          (dict(w=0), "NULL"), (dict(type_of_row=0), "NULL"), (dict(rows=9, type_of_row=0), "NULL"), (dict(order=0), "NULL"), (dict(ptr=0), "NULL"), (dict(shared=1, bias=16), "bias"),
                          (dict(x=17), "unaligned"), (dict(rows=1 << 28, outer=1 << 20), "too many")):
        refused(lib.oeq_typed_product(rows(**changes), 16, None), text)
    refused(lib.oeq_typed_product(rows(), None, None), "NULL")
    refused(lib.oeq_typed_product(rows(), 8, None), "unaligned")
    for changes, text in ((dict(parts=2), "parts"), (dict(shared=1), "shared"), (dict(bias=16), "bias"), (dict(rank=3, thin=16, up=16), "rank")):
        refused(lib.oeq_typed_thin_product(rows(**changes), 16, 16, None), text)
    refused(lib.oeq_typed_thin_product(rows(), 16, None, None), "NULL")
    assert lib.oeq_typed_needs_index(rows()) and not lib.oeq_typed_needs_index(rows(rows=9))
    assert lib.oeq_typed_needs_index(rows(rows=9, across=1))
    assert [lib.oeq_thin_stride(r) for r in (0, 1, 8, 9)] == [0, 8, 8, 16]


def test_c_abi_refuses_sums_of_products():
    lib = rt.load_library()

    def sums(**changes):
        fields = dict(type=2, thin=0, rows=10, parts=1, types=3, a_columns=32, b_columns=16, a_row_stride=32, b_row_stride=16, a=16, b=16,
                      order=16, ptr=16)
        fields.update(changes)
        return ctypes.byref(rt._TypedSum(**fields))

    call = lib.oeq_typed_sum_products
    assert call(sums(types=0), None, None, 0, None) == 0
    refused(call(None, 16, None, 0, None), "NULL")
    for changes, text in ((dict(type=7), "element type"), (dict(rows=-1), "rows"), (dict(parts=0), "parts"), (dict(a_columns=-1), "columns"),
                          (dict(thin=3), "thin"), (dict(b_row_stride=-1), "stride of -1"), (dict(a=0), "NULL"), (dict(order=0), "NULL"),
                          (dict(ptr=0), "NULL"), (dict(a=17), "unaligned"), (dict(thin=1, a=18), "unaligned"),
                          (dict(types=1 << 22, a_columns=1000), "too many")):
        refused(call(sums(**changes), 16, None, 0, None), text)
    refused(call(sums(), None, None, 0, None), "NULL")
    many = sums(rows=100000)
    need = lib.oeq_typed_sum_workspace_bytes(many)
    assert need > 0
    refused(call(many, 16, 16, need - 1, None), "workspace")


@pytest.mark.parametrize("type_", [0, 1, 2])
@pytest.mark.parametrize("thin", [1, 2])
def test_c_abi_refuses_a_thin_operand_of_several_parts(type_, thin):
    """A float operand beside others has one part a row: the kernel of mixed operands counts rows of the index."""
    fields = dict(type=type_, thin=thin, rows=10, parts=2, types=3, a_columns=32, b_columns=16, a_row_stride=64, a_part_stride=32,
                  b_row_stride=32, b_part_stride=16, a=16, b=16, order=16, ptr=16)
    refused(rt.load_library().oeq_typed_sum_products(ctypes.byref(rt._TypedSum(**fields)), 16, None, 0, None), "parts")


def test_c_abi_refuses_more_threads_than_a_launch_counts():
    """Threads of a launch are counted in 32 bits: blocks of 512 have half the room of blocks of 256."""
    lib = rt.load_library()
    d = rt._TypedSum(type=2, rows=10, parts=1, types=1 << 23, a_columns=16, b_columns=16, a_row_stride=16, b_row_stride=16, a=16, b=16,
                     order=16, ptr=16)
    refused(lib.oeq_typed_sum_products(ctypes.byref(d), 16, None, 0, None), "too many")
    for rows, outer in ((9, 1 << 28), (64, (1 << 31) - 512)):  # the form for few rows: 16 columns to a block of 256
        a = rt._TypedRows(type=2, rows=rows, parts=1, types=3, inner=8, outer=outer, x_row_stride=8, w_type_stride=8, w_row_stride=8,
                          x=16, w=16, type_of_row=16)
        refused(lib.oeq_typed_product(ctypes.byref(a), 16, None), "too many")


def test_no_kernel_has_scratch_memory():
    blob = rt.lib_path().read_bytes()
    names, at = {}, 0
    while (at := blob.find(b"\x7fELF", at + 1)) >= 0:
        if int.from_bytes(blob[at + 18:at + 20], "little") == 224:  # EM_AMDGPU
            names.update(rt.kernel_resources(blob[at:]))
    own = {n: r for n, r in names.items() if "typed_products" in n or "row_groups" in n}
    assert len(own) >= 30
    assert not {n: r for n, r in own.items() if r[1] > 0}


@pytest.mark.parametrize("name", ["group_rows", "type_embedding", "typed_linear", "adapter_linear", "RowGroups"])
def test_public_names(name):
    assert name in oeq.__all__ and getattr(oeq, name).__doc__
