"""The tiles of products by type that are taken for large calls: each is run at sizes off its own, by name, against the definitions in
64 bits."""

import re

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import openequivariance_amd as oeq
from tests import typed_oracle as O
from tests.test_typed_operators_gpu import adapter_case, linear_case

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def tiles_of(run):
    """[(kernel, its truth values and tile)] of the products by type that a call launches."""
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as record:
        result = run()
        torch.cuda.synchronize()
    found = []
    for event in record.events():  # (names with 16-bit types come as the compiler wrote them)
        at = re.search(r"typed_products::(row|sum)_products<.*?((?:true, |false, )+)(\d+), ", event.name)
        if not at:
            at = re.search(r"typed_products12(row|sum)_productsI.*?((?:Lb[01]E)+)Li(\d+)E", event.name)
        if at:
            found.append((at[1], *(v in ("true", "1") for v in re.findall("true|false|0|1", at[2])), int(at[3])))
    return found, result


def linear_tiles(x, weight, types, grad):
    """Checks a call and its gradients, and returns the tiles of out, dx and dw."""
    leaves = [t.detach().requires_grad_() for t in (x, weight)]

    def run():
        out = oeq.typed_linear(*leaves, types)
        return (out.detach(), *torch.autograd.grad(out, leaves, grad))

    found, got = tiles_of(run)
    val, err = O.linear(x, weight, types, None, grad)
    for name, g in zip(("out", "dx", "dw"), got):
        O.check(g, val[name], err[name], name)
    return found


# (kernel, across, direct, thin, tile) of rows, (kernel, direct, parts, tile) of sums
@pytest.mark.parametrize("dtype", HALVES)
def test_linear_in_tiles_of_256(dtype):
    x, weight, types, _, grad = linear_case(8751, 0, 2, 1288, 1288, False, dtype)
    assert linear_tiles(x, weight, types, grad) == [("row", False, True, False, 256), ("row", True, True, False, 256), ("sum", True, False, 128)]


@pytest.mark.parametrize("dtype", HALVES)
def test_linear_in_tiles_of_128(dtype):
    x, weight, types, _, grad = linear_case(6251, 0, 2, 776, 776, False, dtype)
    assert linear_tiles(x, weight, types, grad) == [("row", False, True, False, 128), ("row", True, True, False, 128), ("sum", True, False, 128)]


@pytest.mark.parametrize("dtype", HALVES)
def test_linear_in_tiles_of_128_off_16_bytes(dtype):
    x, weight, types, _, grad = linear_case(6501, 0, 2, 777, 777, False, dtype)
    assert linear_tiles(x, weight, types, grad) == [("row", False, False, False, 128), ("row", True, False, False, 128), ("sum", False, False, 64)]


def test_linear_in_tiles_of_128_in_float32():
    x, weight, types, _, grad = linear_case(19001, 3, 10, 120, 120, False, torch.float32)
    assert linear_tiles(x, weight, types, grad) == [("row", False, True, False, 128), ("row", True, True, False, 128), ("sum", True, True, 64)]


@pytest.mark.parametrize("dtype", [torch.float32] + HALVES)
def test_sums_of_components_in_tiles_of_128(dtype):
    x, weight, types, _, grad = linear_case(3001, 3, 2, 776, 520, False, dtype)
    assert linear_tiles(x, weight, types, grad)[2] == ("sum", True, True, 128)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("count", [65, 20])
def test_sums_in_tiles_of_256(count, dtype):
    """Of so many types that none is cut, and with one that is; some types have no rows."""
    x, weight, types, _, grad = linear_case(9001, 0, count, 776, 776, False, dtype)
    types[1000:6000] = 7
    assert linear_tiles(x, weight, types, grad)[2] == ("sum", True, False, 256)


def adapter_tiles(x, weight, down, up, types, scale, grad):
    leaf = x.detach().requires_grad_()

    def run():
        out = oeq.adapter_linear(leaf, weight, down, up, types, scale=scale)
        return (out.detach(), *torch.autograd.grad(out, leaf, grad))

    found, got = tiles_of(run)
    val, err = O.adapters(x, weight, down, up, types, scale, grad)
    for name, g in zip(("out", "dx"), got):
        O.check(g, val[name], err[name], name)
    return [t for t in found if t[3] is True]  # those with a thin product


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,inner,outer,tile", [(8751, 1288, 1288, 256), (6251, 776, 776, 128)])
@pytest.mark.parametrize("rank", [6, 40])
def test_adapters_in_large_tiles(rank, rows, inner, outer, tile, dtype):
    found = adapter_tiles(*adapter_case(rows, 2, inner, outer, rank, dtype))
    assert found == [("row", False, True, True, tile), ("row", True, True, True, tile)]


@pytest.mark.parametrize("rank", [6, 40])
def test_adapters_in_large_tiles_off_16_bytes(rank):
    found = adapter_tiles(*adapter_case(6501, 2, 777, 777, rank, torch.bfloat16))
    assert found == [("row", False, False, True, 128), ("row", True, False, True, 128)]


def test_adapters_in_large_tiles_in_float32():
    found = adapter_tiles(*adapter_case(30001, 2, 248, 248, 20, torch.float32))
    assert found == [("row", False, True, True, 128), ("row", True, True, True, 128)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,width,tile", [(8751, 1288, 256), (6251, 776, 128)])
def test_adapters_in_large_tiles_with_infinities(rows, width, tile, dtype):
    """Infinite weights in the last column of all, of one type."""
    x, weight, down, up, types, scale, _ = adapter_case(rows, 2, width, width, 16, dtype)
    up[1, width - 1, 3] = float("-inf")
    scale = torch.tensor([1.0, -2.0], device="cuda")
    found, out = tiles_of(lambda: oeq.adapter_linear(x, weight, down, up, types, scale=scale))
    assert ("row", False, True, True, tile) in found
    u = -2.0 * (x.double() @ down[1, 3].double())
    hit = types == 1
    assert hit.any() and (u[hit].abs() > 1e-3).float().mean() > 0.9
    sure = hit & (u.abs() > 1e-3)  # (else the sum in 32 bits might have the other sign)
    assert torch.equal(out[sure, -1].double(), torch.where(u[sure] < 0, float("inf"), float("-inf")).double())
    assert torch.isfinite(out[:, :-1]).all() and torch.isfinite(out[~hit]).all()
