"""Attention among nodes, norm and rotation of its queries and keys, the cache form of both and dropout of irreps against
their definitions in 64 bits (tests/node_oracle.py, whose bounds hold before any run)."""

import math

import pytest
import torch

import openequivariance_amd as oeq
from tests import node_oracle as N

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def normal(*shape, dtype=F32, seed=0, device="cuda"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def starts(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


def on_gpu(x):
    return None if x is None else torch.tensor(x, dtype=torch.int64, device="cuda")


def attention_case(dtype, q_ptr, k_ptr, k_len, nq, nk, hq, hk, d, causal, seed=0, scale=None, gradients=True, spoil=None):
    q, k, v = normal(nq, hq, d, dtype=dtype, seed=seed), normal(nk, hk, d, dtype=dtype, seed=seed + 1), normal(
        nk, hk, d, dtype=dtype, seed=seed + 2)
    g = normal(nq, hq, d, dtype=dtype, seed=seed + 3)
    if spoil:
        spoil(q, k, v, g)
    q, k, v = (t.requires_grad_(gradients) for t in (q, k, v))
    views = N.segment_views(q_ptr, k_ptr, k_len, nk, causal)
    val, err = N.attention(q, k, v, views, scale or d ** -0.5, g if gradients else None)
    out, lse = oeq.packed_attention(q, k, v, on_gpu(q_ptr), on_gpu(k_ptr), k_len=on_gpu(k_len), causal=causal, scale=scale,
                                    return_lse=True)
    got = dict(out=out, lse=lse)
    if gradients:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g)))
    for name, x in got.items():
        N.check(x, val[name], err[name], name)
    return got


LENGTHS = {
    "one": [1],
    "small": [5, 1, 0, 9, 31, 32, 33],
    "tile": [127, 128, 129, 3],
    "long": [700, 0, 61],
    "many": [i % 4 for i in range(330)],
    "empty-runs": [0] * 70 + [40] + [0] * 130 + [2],
}


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_segments(dtype, lens, causal):
    lens = LENGTHS[lens]
    ptr = starts(lens)
    attention_case(dtype, ptr, ptr, None, ptr[-1], ptr[-1], 4, 2, 32, causal)


@pytest.mark.parametrize("d", [8, 24, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("heads", [(1, 1), (6, 2), (8, 1)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_heads(dtype, heads, d):
    ptr = starts([70, 1, 97])
    attention_case(dtype, ptr, ptr, None, ptr[-1], ptr[-1], *heads, d, True, seed=d)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_with_other_keys(dtype, causal):
    """More and fewer keys than queries, none at all, caches filled in part, rows outside all segments."""
    q_lens, k_lens = [3, 40, 0, 17, 1, 5, 9, 2], [50, 7, 9, 0, 200, 64, 9, 33]
    q_ptr, k_ptr = starts(q_lens, 2), starts(k_lens, 5)
    nq, nk = q_ptr[-1] + 3, k_ptr[-1] + 4
    attention_case(dtype, q_ptr, k_ptr, None, nq, nk, 4, 2, 64, causal)
    attention_case(dtype, q_ptr, k_ptr, [50, 0, 3, 0, 150, 900, 1, 20], nq, nk, 4, 2, 64, causal, seed=5)
    attention_case(dtype, q_ptr, k_ptr, [-3, 7, 3, 0, 1, 2, 1, 33], nq, nk, 2, 2, 32, causal, seed=7)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads", [(1, 1, 32), (8, 2, 64), (12, 4, 128), (5, 5, 72), (32, 1, 128), (40, 1, 40), (128, 2, 16)])
def test_attention_of_single_rows(dtype, heads):
    """A new row of every segment against a partly filled cache."""
    hq, hk, d = heads
    used = [1, 0, 300, 33, 600, 599, 256, 257]
    n, slots = len(used), 600
    attention_case(dtype, starts([1] * n), [i * slots for i in range(n + 1)], used, n, n * slots, hq, hk, d, False,
                   gradients=hq < 10)


def test_attention_of_a_single_long_row():
    for dtype, nk in ((BF16, 20011), (F32, 5003)):
        attention_case(dtype, [0, 1], [0, nk], None, 1, nk, 8, 2, 128, False, gradients=False)
        attention_case(dtype, [0, 3], [0, nk], None, 3, nk, 4, 1, 64, True, gradients=False)


def test_attention_of_few_rows_with_few_or_uneven_segments():
    attention_case(BF16, starts([2, 0, 3, 1]), starts([900, 40, 0, 1200]), None, 6, 2140, 8, 2, 128, True, gradients=False)
    attention_case(F16, [1, 2], [40, 2000], None, 3, 2048, 16, 4, 96, False, gradients=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_long_segments_with_one_key_head(dtype):
    """Many tiles of queries, which are put in order, to few of keys, which are not."""
    ptr = starts([900, 0, 700])
    attention_case(dtype, ptr, ptr, None, ptr[-1], ptr[-1], 48, 1, 8, True)


@pytest.mark.parametrize("d", [32, 64, 88, 128])
@pytest.mark.parametrize("k_heads", [2, 4])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_many_tiles(dtype, k_heads, d):
    """More blocks than the compute units run at once, and (two key heads) a little more than they have units."""
    ptr = starts([i % 60 for i in range(305)])
    assert ptr[-1] > 8 * 1024
    attention_case(dtype, ptr, ptr, None, ptr[-1], ptr[-1], 8, k_heads, d, k_heads == 2)


def test_rows_far_apart():
    """140 rows 16 MiB apart: a tile of 128 spans nearly 2^31 bytes."""
    rows, apart = 140, (1 << 23) - 8
    if torch.cuda.mem_get_info()[0] < 9 << 30:
        pytest.skip("needs 9 GB")
    q, k, v = (torch.empty(rows * apart, dtype=BF16, device="cuda").as_strided((rows, 2, 16), (apart, 16, 1)) for _ in range(3))
    for n, t in enumerate((q, k, v)):
        t.copy_(normal(rows, 2, 16, dtype=BF16, seed=n))
        t.requires_grad_()
    g = normal(rows, 2, 16, dtype=BF16, seed=4)
    ptr = [0, rows]
    val, err = N.attention(q, k, v, N.segment_views(ptr, ptr, None, rows, False), 0.25, g)
    out = oeq.packed_attention(q, k, v, on_gpu(ptr))
    N.check(out, val["out"], err["out"], "out")
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g)):
        N.check(x, val[name], err[name], name)


def test_large_scores():
    """Scores of some hundreds, where every row's weight is on a few keys, and one large common part."""
    ptr = starts([200, 31])

    def spoil(q, k, v, g):
        q *= 12
        k *= 12

    for dtype in (F32, BF16):
        attention_case(dtype, ptr, ptr, None, 231, 231, 2, 2, 64, False, spoil=spoil)
    attention_case(F32, ptr, ptr, None, 231, 231, 2, 2, 64, True, scale=3.0)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_hidden_rows_have_no_influence(dtype, value, causal):
    """Rows of no segment, keys past a cache's filled part and later tokens may hold anything."""
    q_ptr, k_ptr, k_len = starts([20, 30, 9], 3), starts([20, 50, 9], 3), [20, 30, 9]

    def spoil(q, k, v, g):
        for t in (q, k, v, g):
            t[:3], t[-2:] = value, value
        k[53:73], v[53:73] = value, value  # behind the filled part of the second segment
        if causal:  # hidden from all but the segment's last row, whose results are what the formula makes of it
            pass

    got = attention_case(dtype, q_ptr, k_ptr, k_len, 64, 84, 4, 2, 40, causal, spoil=spoil)
    for name in ("out", "dq", "dk", "dv"):
        assert torch.isfinite(got[name]).all(), name
    # one query of each segment may have anything as well: the others' results stay
    q, k, v = (normal(79, 2, 32, dtype=dtype, seed=s) for s in (1, 2, 3))
    ptr = on_gpu(starts([20, 50, 9]))
    whole = oeq.packed_attention(q, k, v, ptr, causal=causal)
    q[25] = value
    part = oeq.packed_attention(q, k, v, ptr, causal=causal)
    other = torch.arange(79, device="cuda") != 25
    assert torch.equal(whole[other], part[other])


def test_a_later_token_that_is_not_finite():
    """Causal rows before it are as without it, in the output and in the gradients."""
    for dtype in (F32, BF16):
        n, bad = 150, 100
        q, k, v, g = (normal(n, 2, 64, dtype=dtype, seed=s) for s in range(4))
        k[bad], v[bad, 0, 5] = math.nan, math.inf
        g[bad:] = 0
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        out = oeq.packed_attention(q, k, v, on_gpu([0, n]), causal=True)
        ref, err = N.attention(q[:bad], k[:bad], v[:bad], N.segment_views([0, bad], [0, bad], None, bad, True), 64 ** -0.5,
                               g[:bad])
        N.check(out[:bad], ref["out"], err["out"], "out")
        dq, = torch.autograd.grad(out, q, g)
        N.check(dq[:bad], ref["dq"], err["dq"], "dq")
        assert torch.isnan(out[bad + 1:]).all()


def test_a_visible_infinity_is_passed_on():
    q, k, v = (normal(40, 1, 32, seed=s) for s in range(3))
    v[7, 0, 3] = math.inf
    out = oeq.packed_attention(q, k, v, on_gpu([0, 20, 40]))
    assert torch.isinf(out[:20, 0, 3]).all() and torch.isfinite(out[20:]).all()
    assert torch.isfinite(out[:20, 0, :3]).all() and torch.isfinite(out[:20, 0, 4:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_reads_views(dtype):
    """Parts of one projection, heads before rows, unaligned and transposed storage, gradients with strides."""
    n, hq, hk, d = 90, 4, 2, 32
    ptr = starts([50, 40])
    views = N.segment_views(ptr, ptr, None, n, False)
    qkv = normal(n, (hq + 2 * hk) * d, dtype=dtype)
    q, k, v = (t.view(n, -1, d) for t in qkv.split([hq * d, hk * d, hk * d], 1))
    g = normal(hq, n, d, dtype=dtype, seed=4).transpose(0, 1)
    plain = [t.contiguous().requires_grad_() for t in (q, k, v)]
    out = oeq.packed_attention(*plain, on_gpu(ptr))
    grads = torch.autograd.grad(out, plain, g.contiguous())
    odd = torch.empty(n * hk * d + 3, dtype=dtype, device="cuda")[3:].view(n, hk, d)
    odd.copy_(v)
    by_column = k.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for qq, kk, vv in ((q, k, v), (q.transpose(0, 1).contiguous().transpose(0, 1), by_column, odd)):
        leaves = [t.detach().requires_grad_() for t in (qq, kk, vv)]
        again = oeq.packed_attention(*leaves, on_gpu(ptr))
        assert torch.equal(again, out)
        for a, b in zip(torch.autograd.grad(again, leaves, g), grads):
            assert torch.equal(a, b)
    val, err = N.attention(q, k, v, views, d ** -0.5)
    N.check(out, val["out"], err["out"], "out")
    shared = oeq.packed_attention(q, k[:, :1].expand(n, hk, d), v, on_gpu(ptr))
    val, err = N.attention(q, k[:, :1].expand(n, hk, d), v, views, d ** -0.5)
    N.check(shared, val["out"], err["out"], "out")


def test_attention_gradient_against_differences():
    ptr = on_gpu(starts([9, 30]))
    x = [normal(39, h, 16, seed=s).requires_grad_() for s, h in enumerate((4, 2, 2))]
    g = normal(39, 4, 16, seed=9)
    grads = torch.autograd.grad(oeq.packed_attention(*x, ptr, causal=True), x, g)
    step = 1e-2
    for n in range(3):
        way = normal(*x[n].shape, seed=20 + n)
        sides = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * step * way if i == n else 0) for i, t in enumerate(x)]
            sides.append((oeq.packed_attention(*moved, ptr, causal=True) * g).double().sum())
        # central differences: an error of step^2 times a third derivative, and 2^-24 of the sum of terms over the step
        difference, along = (sides[0] - sides[1]) / (2 * step), (grads[n].double() * way).sum()
        assert abs(difference - along) <= 1e-2 * grads[n].double().norm() * way.double().norm() / math.sqrt(x[n].numel()) + 0.02


def test_attention_is_reproducible_and_runs_on_other_streams():
    ptr = on_gpu(starts([300, 5, 77]))
    x = [normal(382, h, 64, dtype=BF16, seed=s).requires_grad_() for s, h in enumerate((4, 2, 2))]
    g = normal(382, 4, 64, dtype=BF16, seed=9)

    def run():
        out = oeq.packed_attention(*x, ptr, causal=True)
        return (out,) + torch.autograd.grad(out, x, g)

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_attention_without_rows():
    for nq, nk in ((0, 0), (4, 0), (0, 4)):
        q, k, v = (normal(n, 2, 32).requires_grad_() for n in (nq, nk, nk))
        out = oeq.packed_attention(q, k, v, on_gpu([0, nq]), on_gpu([0, nk]))
        assert out.shape == q.shape and not out.any()
        for x, t in zip(torch.autograd.grad(out.sum(), (q, k, v)), (q, k, v)):
            assert x.shape == t.shape and not x.any()
    out = oeq.packed_attention(normal(4, 2, 32), normal(4, 2, 32), normal(4, 2, 32), on_gpu([0]))
    assert not out.any()


def test_attention_refuses():
    q, k = normal(8, 4, 32), normal(8, 2, 32)
    ptr = on_gpu([0, 8])
    run = oeq.packed_attention
    for bad, text in (
            (lambda: run(q.double(), k.double(), k.double(), ptr), "Dtype mismatch"),
            (lambda: run(q, k.half(), k, ptr), "Dtype mismatch for tensor 'k'"),
            (lambda: run(q, k, k.half(), ptr), "Dtype mismatch for tensor 'v'"),
            (lambda: run(q[..., :12], k[..., :12], k[..., :12], ptr), "multiple of 8"),
            (lambda: run(normal(8, 4, 136), normal(8, 2, 136), normal(8, 2, 136), ptr), "up to 128"),
            (lambda: run(normal(8, 3, 32), k, k, ptr), "divides"),
            (lambda: run(q, k, k[:7], ptr), "Shape mismatch for tensor 'v'"),
            (lambda: run(q[0], k, k, ptr), "Shape mismatch for tensor 'q'"),
            (lambda: run(q, k.cpu(), k, ptr), "not on the GPU"),
            (lambda: run(q, k, k, ptr.int()), "Dtype mismatch for tensor 'q_ptr'"),
            (lambda: run(q, k, k, ptr.cpu()), "not on the GPU"),
            (lambda: run(q, k, k, ptr, on_gpu([0, 4, 8])), "Shape mismatch for tensor 'k_ptr'"),
            (lambda: run(q, k, k, ptr, k_len=on_gpu([8, 8])), "Shape mismatch for tensor 'k_len'"),
            (lambda: run(q, k, k, ptr, scale=0.0), "scale"),
            (lambda: run(q, k, k, ptr, scale=math.nan), "scale")):
        with pytest.raises(RuntimeError, match=text):
            bad()
    x = q.clone().requires_grad_()
    g, = torch.autograd.grad(run(x, k, k, ptr).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        g.sum().backward()


def test_starts_that_point_outside_are_cut_off():
    q, k = normal(8, 2, 32), normal(8, 2, 32, seed=1)
    far = 1 << 40
    out = oeq.packed_attention(q, k, k, on_gpu([0, 4, far]), on_gpu([0, 4, far]))
    assert torch.equal(out, oeq.packed_attention(q, k, k, on_gpu([0, 4, 8])))
    assert not oeq.packed_attention(q, k, k, on_gpu([-far, -5]), on_gpu([-far, -5])).any()
    assert not oeq.packed_attention(q, k, k, on_gpu([0, 8]), on_gpu([far, far + 8])).any()


def test_long_caches_pass_32_bits():
    """More than 2^31 elements in front of the rows that are read and written."""
    hk, d, slots = 8, 128, 1 << 18
    rows = 9 * slots
    if torch.cuda.mem_get_info()[0] < 3 * rows * hk * d * 2:
        pytest.skip("needs 15 GB")
    k_cache, v_cache = (torch.empty(rows, hk, d, dtype=BF16, device="cuda") for _ in range(2))
    used, at = 700, 8 * slots + 5
    assert at * hk * d > 1 << 31
    k_cache[at:at + used] = normal(used, hk, d, dtype=BF16, seed=1)
    v_cache[at:at + used] = normal(used, hk, d, dtype=BF16, seed=2)
    q = normal(1, 16, d, dtype=BF16, seed=3)
    table = oeq.rotary_table(1024, d, device="cuda")
    k_new, v_new, where = normal(1, hk, d, dtype=BF16, seed=4), normal(1, hk, d, dtype=BF16, seed=5), on_gpu([used])
    turned = oeq.qk_norm_rotary_append(q, k_new, v_new, where, table, k_cache, v_cache, on_gpu([at + used]))
    assert torch.equal(v_cache[at + used], v_new[0])
    keys, values = k_cache[at:at + used + 1], v_cache[at:at + used + 1]
    assert torch.equal(keys[used], oeq.qk_norm_rotary(q, k_new, where, table)[1][0])
    out = oeq.packed_attention(turned, k_cache, v_cache, on_gpu([0, 1]), on_gpu([at, rows]), k_len=on_gpu([used + 1]))
    val, err = N.attention(turned, keys, values, N.segment_views([0, 1], [0, used + 1], None, used + 1, False), d ** -0.5)
    N.check(out, val["out"], err["out"], "out")
    many = oeq.packed_attention(turned.expand(40, 16, d), k_cache, v_cache, on_gpu([0, 40]), on_gpu([at, rows]),
                                k_len=on_gpu([used + 1]))
    N.check(many[39:], val["out"], err["out"], "out")


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", ["both", "q", "none"])
@pytest.mark.parametrize("d,rotary", [(8, 8), (32, 16), (72, 72), (72, 24), (128, 128), (128, 64), (96, 8)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_norm_and_rotation(dtype, d, rotary, normed, interleaved):
    for rows, hq, hk in ((1, 1, 1), (37, 6, 2), (300, 3, 1)):
        q, k = normal(rows, hq, d, dtype=dtype, seed=1), normal(rows, hk, d, dtype=dtype, seed=2)
        gq, gk = normal(rows, hq, d, dtype=dtype, seed=3), normal(rows, hk, d, dtype=dtype, seed=4)
        weights = [(1 + 0.3 * normal(d, seed=5 + i)).to(dtype) if normed == "both" or (normed == "q" and i == 0) else None
                   for i in (0, 1)]
        leaves = [t.requires_grad_() for t in [q, k] + weights if t is not None]
        positions = torch.randint(0, 500, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
        table = oeq.rotary_table(500, rotary, device="cuda")
        out = oeq.qk_norm_rotary(q, k, positions, table, *weights, eps=1e-5, interleaved=interleaved)
        grads = list(torch.autograd.grad(out, leaves, (gq, gk)))
        for n, (x, w, g) in enumerate(((q, weights[0], gq), (k, weights[1], gk))):
            y, y_err, dx, dx_err, dw, dw_err = N.rotate(x, w, positions, table, interleaved, 1e-5, g)
            N.check(out[n], y, y_err, "out")
            N.check(grads[n], dx, dx_err, "gradient")
            if w is not None:
                N.check(grads[2 + n], dw, dw_err, "weight's gradient")


def test_rotation_reads_views_and_gradients_of_one_output():
    n, hq, hk, d = 50, 4, 2, 64
    qkv = normal(n, (hq + 2 * hk) * d, dtype=BF16)
    q, k, _v = (t.view(n, -1, d) for t in qkv.split([hq * d, hk * d, hk * d], 1))
    table, positions = oeq.rotary_table(64, 32, device="cuda"), torch.arange(n, device="cuda")
    a = oeq.qk_norm_rotary(q, k, positions, table)
    b = oeq.qk_norm_rotary(q.contiguous(), k.transpose(0, 1).contiguous().transpose(0, 1), positions, table)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q, k = (t.detach().float().requires_grad_() for t in (q, k))
    g = normal(hq, n, d, seed=3).transpose(0, 1)
    out = oeq.qk_norm_rotary(q, k, positions, table)
    dq, dk = torch.autograd.grad(out[0], (q, k), g)
    N.check(dq, *N.rotate(q, None, positions, table, False, 1e-6, g)[2:4], "gradient")
    assert not dk.any()


def test_rotation_of_rows_that_are_zero_and_positions_outside():
    q, k, w = torch.zeros(4, 2, 32, device="cuda"), normal(4, 1, 32), torch.ones(32, device="cuda")
    table = oeq.rotary_table(10, 16, device="cuda")
    out, other = oeq.qk_norm_rotary(q, k, on_gpu([0, 9, 10, -1]), table, w)
    assert not out[:2].any()
    assert torch.isfinite(other[:2]).all() and torch.isnan(other[2:, :, :16]).all()
    assert torch.equal(other[:, :, 16:], k[:, :, 16:])
    empty = oeq.qk_norm_rotary(q[:0].requires_grad_(), k[:0], on_gpu([]), table, w.requires_grad_())
    grads = torch.autograd.grad(empty[0].sum(), (w,))
    assert empty[0].shape == (0, 2, 32) and not grads[0].any()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_append_writes_the_slots_it_is_given(dtype, interleaved):
    for n, hq, hk, d, rotary in ((1, 4, 4, 32, 32), (9, 6, 2, 72, 24), (130, 8, 1, 128, 128)):
        q, k, v = (normal(n, h, d, dtype=dtype, seed=s) for s, h in enumerate((hq, hk, hk)))
        w = (1 + 0.1 * normal(d, seed=7)).to(dtype)
        table, positions = oeq.rotary_table(50, rotary, device="cuda"), torch.arange(n, device="cuda") % 50
        cache = normal(3 * n, 2, hk, d, dtype=dtype, seed=8)  # keys and values of a row side by side
        k_cache, v_cache = cache[:, 0], cache[:, 1]
        before = cache.clone()
        slots = torch.randperm(3 * n, generator=torch.Generator().manual_seed(n))[:n].cuda()
        if n > 2:
            slots[1], slots[2] = -1, 3 * n
        out = oeq.qk_norm_rotary_append(q, k, v, positions, table, k_cache, v_cache, slots, w, w, interleaved=interleaved)
        want_q, want_k = oeq.qk_norm_rotary(q, k, positions, table, w, w, interleaved=interleaved)
        assert torch.equal(out, want_q)
        used = (slots >= 0) & (slots < 3 * n)
        before[slots[used], 0], before[slots[used], 1] = want_k[used], v[used]
        assert torch.equal(cache, before)


def test_rotation_refuses():
    q, k, v = normal(6, 4, 32), normal(6, 2, 32), normal(6, 2, 32)
    table, at, w = oeq.rotary_table(10, 16, device="cuda"), torch.arange(6, device="cuda"), normal(32)
    cache = normal(20, 2, 32)
    run, append = oeq.qk_norm_rotary, oeq.qk_norm_rotary_append
    for bad, text in (
            (lambda: run(q.double(), k.double(), at, table), "Dtype mismatch for tensor 'q'"),
            (lambda: run(q, k.half(), at, table), "Dtype mismatch for tensor 'k'"),
            (lambda: run(q, k[:5], at, table), "Shape mismatch for tensor 'k'"),
            (lambda: run(q[..., :20], k[..., :20], at, table), "multiple of 8"),
            (lambda: run(q, k, at.int(), table), "Dtype mismatch for tensor 'positions'"),
            (lambda: run(q, k, at[:5], table), "Shape mismatch for tensor 'positions'"),
            (lambda: run(q, k, at, table.double()), "Dtype mismatch for tensor 'table'"),
            (lambda: run(q, k, at, oeq.rotary_table(10, 40, device="cuda")), "Shape mismatch for tensor 'table'"),
            (lambda: run(q, k, at, table[:, :, :6]), "Shape mismatch for tensor 'table'"),
            (lambda: run(q, k, at, table.cpu()), "not on the GPU"),
            (lambda: run(q, k, at, table, w[:16]), "Shape mismatch for tensor 'q_weight'"),
            (lambda: run(q, k, at, table, None, w.half()), "Dtype mismatch for tensor 'k_weight'"),
            (lambda: run(q, k, at, table, w, eps=-1.0), "eps"),
            (lambda: append(q, k, v, at, table, cache, cache[:19], at), "Shape mismatch for tensor 'v_cache'"),
            (lambda: append(q, k, v, at, table, cache, cache.transpose(1, 2).contiguous().transpose(1, 2), at), "caches need"),
            (lambda: append(q, k, v, at, table, cache, cache.clone(), at[:3]), "Shape mismatch for tensor 'slots'"),
            (lambda: append(q.requires_grad_(), k, v, at, table, cache, cache.clone(), at), "no gradient")):
        with pytest.raises(RuntimeError, match=text):
            bad()
    with pytest.raises(ValueError, match="rotary_dim"):
        oeq.rotary_table(10, 12)


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["mul_ir", "ir_mul"])
@pytest.mark.parametrize("irreps", ["1x0e", "131x0e", "8x0e+4x1o", "5x0e+3x1e+2x3o", "2x2e+17x0o"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16, torch.float64])
def test_dropout_of_irreps(dtype, irreps, layout):
    module = oeq.IrrepDropout(irreps, 0.3, layout=layout)
    dim, channels = oeq.Irreps(irreps).dim, module.channels.cpu().long()
    module = module.cuda()
    for rows in (1, 7, 33):
        x = normal(rows, dim, dtype=dtype, seed=1).requires_grad_()
        base = normal(rows, dim, dtype=dtype, seed=2).requires_grad_()
        g = normal(rows, dim, dtype=dtype, seed=3)
        seed = on_gpu([-(1 << 61) + 12345, (1 << 40) + rows])
        keep = N.kept(rows, int(channels.max()) + 1, seed, 0.3)[:, channels].double() / (1 - round(0.3 * 65536) / 65536)
        u = N.HALF_UNIT[dtype]
        for residual in (None, base):
            out = module(x, residual, seed=seed)
            part = x.detach().cpu().double() * keep
            whole = part + (base.detach().cpu().double() if residual is not None else 0)
            # one product and one sum in 32 bits (64), the scale rounded to them, and the output's rounding
            e = max(2.0 ** -24, u) if dtype != torch.float64 else u
            bound = u * whole.abs() + 3 * (2.0 ** -24 if dtype != torch.float64 else u) * (part.abs() + whole.abs()) + N.TINY[dtype]
            N.check(out, whole, bound, "out")
            grads = torch.autograd.grad(out, [x] + ([residual] if residual is not None else []), g)
            want = g.cpu().double() * keep
            N.check(grads[0], want, (u + 3 * e) * want.abs() + N.TINY[dtype], "gradient")
            if residual is not None:
                assert torch.equal(grads[1], g)


def test_dropout_statistics_modes_and_seeds():
    module = oeq.IrrepDropout("64x0e+64x1o", 0.25).cuda()
    x = torch.ones(5000, 256, device="cuda")
    torch.manual_seed(3)
    a, b = module(x), module(x)
    torch.manual_seed(3)
    assert torch.equal(a, module(x)) and not torch.equal(a, b)
    kept = a != 0
    # 640 000 draws: a standard deviation of 0.00054 of the share
    assert abs(kept[:, :64].float().mean() - 0.75) < 0.004 and abs(kept[:, 64::3].float().mean() - 0.75) < 0.004
    vectors = kept[:, 64:].view(5000, 64, 3)
    assert torch.equal(vectors[..., 0], vectors[..., 1]) and torch.equal(vectors[..., 0], vectors[..., 2])
    assert torch.equal(a[kept], torch.full_like(a[kept], 1 / 0.75))
    assert not torch.equal(kept[0], kept[1]) and abs((kept[0] & kept[1]).float().mean() - 0.5625) < 0.25
    module.eval()
    assert module(x) is x and torch.equal(module(x, x), 2 * x)
    assert not oeq.IrrepDropout("256x0e", 1.0).cuda()(x).any()
    assert torch.equal(oeq.IrrepDropout("256x0e", 0.0).cuda()(x), x)
    assert module.train()(x[:0]).shape == (0, 256)


def test_dropped_values_have_no_influence_and_second_derivatives():
    module, seed = oeq.IrrepDropout("16x0e", 0.5).cuda(), on_gpu([1, 2])
    x = normal(20, 16)
    keep = module(torch.ones_like(x), seed=seed) != 0
    x[~keep] = math.nan
    assert torch.equal(module(x, seed=seed), torch.where(keep, 2 * x, 0.0))
    y = normal(20, 16, seed=4).requires_grad_()
    first, = torch.autograd.grad(module(y, seed=seed).pow(2).sum(), y, create_graph=True)
    second, = torch.autograd.grad(first.sum(), y)
    assert torch.equal(second, torch.where(keep, 8.0, 0.0))


def test_dropout_reads_views_and_long_tensors():
    module, seed = oeq.IrrepDropout("5x0e+1x1o", 0.5).cuda(), on_gpu([5, 6])
    x = normal(9, 16)[:, 3:11]
    assert torch.equal(module(x, seed=seed), module(x.contiguous(), seed=seed))
    # rows beyond 2^31 elements are numbered on: their masks are those of their rows
    rows, dim = (1 << 31) // 64 + 100, 64
    if torch.cuda.mem_get_info()[0] < 6 * rows * dim * 2:
        pytest.skip("needs 26 GB")
    module = oeq.IrrepDropout("64x0e", 0.5).cuda()
    out = module(torch.ones(rows, dim, dtype=BF16, device="cuda"), seed=seed)
    share = out[-200:].float().mean()
    assert 0.9 < share < 1.1 and not torch.equal(out[-200:-100], out[:100])
    assert not torch.equal(out[-100:], out[:100])


def test_dropout_refuses():
    module, x, seed = oeq.IrrepDropout("4x0e+1x1o", 0.1).cuda(), normal(3, 7), on_gpu([1, 2])
    for bad, text in (
            (lambda: module(x.int(), seed=seed), "Dtype mismatch for tensor 'x'"),
            (lambda: module(normal(3, 8), seed=seed), "Shape mismatch for tensor"),
            (lambda: module(x[0], seed=seed), "Shape mismatch for tensor 'x'"),
            (lambda: module(x, x.half(), seed=seed), "Dtype mismatch for tensor 'residual'"),
            (lambda: module(x, x[:2], seed=seed), "Shape mismatch for tensor 'residual'"),
            (lambda: module(x, seed=seed.int()), "Dtype mismatch for tensor 'seed'"),
            (lambda: module(x, seed=seed[:1]), "Shape mismatch for tensor 'seed'"),
            (lambda: module(x, seed=seed.cpu()), "not on the GPU")):
        with pytest.raises(RuntimeError, match=text):
            bad()
    for p in (-0.1, 1.5):
        with pytest.raises(ValueError, match="between 0 and 1"):
            oeq.IrrepDropout("4x0e", p)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def test_graph_capture_and_replay():
    """A training step's operators in a HIP graph, replayed between eager work, against the eager results."""
    n, hq, hk, d = 150, 4, 2, 32
    ptr, positions = on_gpu(starts([90, 0, 60])), torch.arange(n, device="cuda") % 90
    table, w = oeq.rotary_table(90, d, device="cuda"), torch.ones(d, device="cuda").requires_grad_()
    dropout, seed = oeq.IrrepDropout(f"{hq * d}x0e", 0.2).cuda(), on_gpu([3, 4])
    q, k, v = (normal(n, h, d, seed=s).requires_grad_() for s, h in enumerate((hq, hk, hk)))
    g = normal(n, hq * d, seed=8)

    def step():
        qq, kk = oeq.qk_norm_rotary(q, k, positions, table, w, w)
        out = dropout(oeq.packed_attention(qq, kk, v, ptr, causal=True).reshape(n, hq * d), seed=seed)
        return (out,) + torch.autograd.grad(out, (q, k, v, w), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        with torch.no_grad():
            for t in (q, k, v):
                t.add_(0.1 * i)
            seed.add_(i)
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_compiled_calls_keep_their_results():
    ptr = on_gpu([0, 20, 50])
    q, k = normal(50, 2, 32).requires_grad_(), normal(50, 2, 32, seed=1)

    def layer(q, k):
        return oeq.packed_attention(q, k, k, ptr).square()

    torch._dynamo.reset()
    compiled = torch.compile(layer, backend="aot_eager", fullgraph=True)
    for f in (layer, compiled):
        out = f(q, k)
        grad, = torch.autograd.grad(out.sum(), q)
        if f is layer:
            want = out, grad
    assert torch.equal(out, want[0]) and torch.equal(grad, want[1])


def test_autocast():
    """Projections in 16 bits beside parameters and a residual stream in 32."""
    n, ptr, positions = 40, on_gpu([0, 15, 40]), torch.arange(40, device="cuda")
    linear = torch.nn.Linear(64, 3 * 64, bias=False).cuda()
    w, table = torch.ones(32, device="cuda", requires_grad=True), oeq.rotary_table(40, 32, device="cuda")
    x, dropout = normal(n, 64), oeq.IrrepDropout("64x0e", 0.1).cuda()
    with torch.autocast("cuda", dtype=BF16):
        q, k, v = (t.view(n, 2, 32) for t in linear(x).split(64, 1))
        q, k = oeq.qk_norm_rotary(q, k, positions, table, w, w)
        out = dropout(oeq.packed_attention(q, k, v, ptr).flatten(1), x)
    assert q.dtype == BF16 and out.dtype == F32
    out.sum().backward()
    assert w.grad.dtype == F32 and linear.weight.grad.dtype == F32 and torch.isfinite(linear.weight.grad).all()


# ---------------------------------------------------------------------------
# ends of segments
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("end", [12, 1 << 40])
@pytest.mark.parametrize("rows,keys", [(8, 8), (8, 5), (150, 190)])
def test_causal_ends_past_the_tensors_have_one_diagonal(dtype, end, rows, keys):
    """A segment that is said to go on behind the tensors is the one that is cut off there: its last row sees every key,
    in the output and in all gradients."""
    end += max(rows, keys)
    leaves = [normal(n, h, 32, dtype=dtype, seed=s).requires_grad_() for s, (n, h) in enumerate(((rows, 4), (keys, 2), (keys, 2)))]
    g = normal(rows, 4, 32, dtype=dtype, seed=5)
    results = []
    for q_ptr, k_ptr in (([0, 3, rows], [0, 2, keys]), ([0, 3, end], [0, 2, end]), ([0, 3, end], [0, 2, keys])):
        out, lse = oeq.packed_attention(*leaves, on_gpu(q_ptr), on_gpu(k_ptr), causal=True, return_lse=True)
        results.append((out, lse) + torch.autograd.grad(out, leaves, g))
    for other in results[1:]:
        for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), results[0], other):
            assert torch.equal(a, b), name


def test_forward_mode_derivative_of_dropout():
    module, seed = oeq.IrrepDropout("5x0e+2x1o", 0.4).cuda(), on_gpu([7, 8])
    x, base, tx, tb = (normal(30, 11, seed=s) for s in range(4))
    want = module(tx, tb, seed=seed)
    value, tangent = torch.func.jvp(lambda a, b: module(a, b, seed=seed), (x, base), (tx, tb))
    assert torch.equal(value, module(x, base, seed=seed)) and torch.equal(tangent, want) and tangent.any()
    _, tangent = torch.func.jvp(lambda a: module(a, base, seed=seed), (x,), (tx,))
    assert torch.equal(tangent, module(tx, seed=seed))
    _, tangent = torch.func.jvp(lambda b: module(x, b, seed=seed), (base,), (tb,))
    assert torch.equal(tangent, tb)
    q, ptr = normal(11, 2, 32), on_gpu([0, 11])
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda t: oeq.packed_attention(t, q, q, ptr), (q,), (q,))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda t: oeq.qk_norm_rotary(t, q, torch.arange(11, device="cuda"), oeq.rotary_table(11, 8, device="cuda")),
                       (q,), (q,))


def test_dropout_of_a_module_that_was_not_moved():
    x, seed = normal(20, 11), on_gpu([7, 8])
    want = oeq.IrrepDropout("5x0e+2x1o", 0.4).cuda()(x, seed=seed)
    module = oeq.IrrepDropout("5x0e+2x1o", 0.4)
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y.add_(1)
        with pytest.raises(RuntimeError, match="before a graph is captured"):
            module(x, seed=seed)
    assert module.channels.device.type == "cpu"
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all()  # the capture went on
    with torch.inference_mode():
        assert torch.equal(module(x, seed=seed), want)
    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(module(leaf, seed=seed).sum(), leaf)
    assert torch.equal(grad != 0, want != 0)


# ---------------------------------------------------------------------------
# errors as a whole
# ---------------------------------------------------------------------------


def gradients_64(q, k, v, g, causal=False):
    """(values, sums of the squared terms) of out, dq, dk and dv of one segment with a head of keys for each of queries,
    in 64 bits: {name: (value, terms)}. The terms of a sum carry the roundings of its operands."""
    q, k, v, g = (t.detach().double().transpose(0, 1).contiguous() for t in (q, k, v, g))
    c = q.shape[2] ** -0.5
    kt, vt = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    s = torch.bmm(q, kt) * c
    if causal:
        s += torch.full(s.shape[1:], -math.inf, dtype=s.dtype, device=s.device).triu(1 + s.shape[2] - s.shape[1])
    p = torch.softmax(s, 2)
    out = torch.bmm(p, v)
    ds = p * (torch.bmm(g, vt) - (g * out).sum(2, keepdim=True))
    pt, dst = p.transpose(1, 2).contiguous(), ds.transpose(1, 2).contiguous()
    pairs = dict(out=(p, v, 1.0), dq=(ds, k, c), dk=(dst, q, c), dv=(pt, g, 1.0))
    return {n: ((torch.bmm(a, b) * f).transpose(0, 1), (torch.bmm(a * a, b * b) * f * f).transpose(0, 1))
            for n, (a, b, f) in pairs.items()}


def check_norm(got, value, terms, dtype, what, more=0.0):
    """The norm of the error, against that of independent roundings of one operand of each term (16-bit types) and of the
    result, every one taken at its largest and the whole twice: `more` is what 32-bit sums may add of the value's norm."""
    u, tiny = N.HALF_UNIT[dtype], N.TINY[dtype]
    allowed = ((u * u * value * value + tiny * tiny).sum() + (u * u * terms.sum() if dtype != F32 else 0.0)).sqrt()
    error = (got.double() - value).norm()
    assert error <= 2 * allowed + more * value.norm(), f"{what}: {error / value.norm():.2e} of its norm, {allowed / value.norm():.2e}"


@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-2, 1.0, 1e4])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("rows,keys", [(256, 4096), (4096, 300), (4, 3)])
def test_float16_gradients_of_any_size(rows, keys, d, size):
    """The size of the output's gradient is the caller's choice (a loss that is scaled, or is not): it costs gradients no bits."""
    q, k, v = (normal(n, 2, d, dtype=F16, seed=s).requires_grad_() for s, n in enumerate((rows, keys, keys)))
    g = (size * normal(rows, 2, d, seed=5)).to(F16)
    out = oeq.packed_attention(q, k, v, on_gpu([0, rows]), on_gpu([0, keys]))
    want = gradients_64(q, k, v, g)
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g)):
        # (32-bit sums of a few thousand terms: some 2^-24 of them each)
        check_norm(x, *want[name], F16, name, more=2.0 ** -18)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("segments,keys,hq,hk,d,few", [(1, 20011, 8, 2, 128, True), (1, 900, 4, 4, 64, True), (9, 700, 5, 1, 72, True),
                                                       (64, 60, 8, 8, 32, True), (1, 300, 4, 4, 64, False)])
def test_single_rows_lose_no_more_than_the_outputs_rounding(dtype, segments, keys, hq, hk, d, few):
    """The error is what rounding the exact result once would leave, and twice what comes before that: weights of two
    parts (the half unit squared; in one part the half unit where a call is so short that it takes the form for tiles) and
    sums of 32 bits."""
    q, k, v = (normal(segments * n, h, d, dtype=dtype, seed=s) for s, (n, h) in enumerate(((1, hq), (keys, hk), (keys, hk))))
    ptr = torch.arange(segments + 1, device="cuda")
    out = oeq.packed_attention(q, k, v, ptr, keys * ptr).double()
    qq = q.double().view(segments, hk, hq // hk, d).reshape(-1, hq // hk, d)
    kk, vv = (t.double().view(segments, keys, hk, d).transpose(1, 2).reshape(-1, keys, d) for t in (k, v))
    p = torch.softmax(torch.bmm(qq, kk.transpose(1, 2).contiguous()) * d ** -0.5, 2)
    want = torch.bmm(p, vv).view(segments, hq, d)
    before = N.HALF_UNIT[dtype] ** (2 if few else 1) * torch.bmm(p * p, vv * vv).sum().sqrt() + 2.0 ** -17 * want.norm()
    assert (out - want).norm() <= (want.to(dtype) - want).norm() + 2 * before


# ---------------------------------------------------------------------------
# results that are not finite
# ---------------------------------------------------------------------------


def all_of(leaves, q_ptr, k_ptr, k_len, causal, g):
    out, lse = oeq.packed_attention(*leaves, q_ptr, k_ptr, k_len=k_len, causal=causal, return_lse=True)
    return dict(zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + torch.autograd.grad(out, leaves, g)))


SPOILT = {
    "small": ([20, 30, 1, 9] * 5, [25, 33, 40, 9] * 5, [20, 30, 7, 9] * 5, 4, 2),
    "long": ([700, 61], [900, 200], [700, 90], 2, 1),
    "many": ([50] * 90, [70] * 90, [50] * 90, 8, 8),
    "single": ([1] * 9, [1500] * 9, [900, 3, 0, 1499, 600, 1, 256, 700, 64], 8, 2),
}


@pytest.mark.parametrize("d", [32, 72, 128])
@pytest.mark.parametrize("case", SPOILT)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_hidden_rows_change_no_bit(dtype, case, d):
    """Slots behind a cache's filled part and rows outside all segments: whatever they hold, every result is the same."""
    q_lens, k_lens, k_len, hq, hk = SPOILT[case]
    q_ptr, k_ptr = starts(q_lens, 2), starts(k_lens, 3)
    nq, nk = q_ptr[-1] + 2, k_ptr[-1] + 4
    seen_q = torch.zeros(nq, dtype=torch.bool, device="cuda")
    seen_q[2:-2] = True
    seen_k = torch.zeros(nk, dtype=torch.bool, device="cuda")
    for first, n in zip(k_ptr, k_len):
        seen_k[first:first + n] = True
    base = [normal(n, h, d, dtype=dtype, seed=s) for s, (n, h) in enumerate(((nq, hq), (nk, hk), (nk, hk), (nq, hq)))]
    want = None
    for causal in (False, True):
        for value in (0.0, math.nan, math.inf, -math.inf):
            leaves = []
            for n, t in enumerate(base):
                t = t.clone()
                t[~(seen_k if n in (1, 2) else seen_q)] = value
                leaves.append(t)
            got = all_of([t.requires_grad_() for t in leaves[:3]], on_gpu(q_ptr), on_gpu(k_ptr), on_gpu(k_len), causal, leaves[3])
            if value == 0.0:
                want = got
            for name, x in got.items():
                assert torch.equal(x, want[name]), (name, value, causal)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [150, 700])
def test_later_tokens_change_no_bit(dtype, rows):
    """Causal: what comes after a row, in the same tile or a later one."""
    bad = rows - 45
    base = [normal(rows, h, 64, dtype=dtype, seed=s) for s, h in enumerate((4, 2, 2, 4))]
    ptr, results = on_gpu([0, rows]), []
    for value in (1.0, math.nan, math.inf, -math.inf):
        leaves = [t.clone() for t in base]
        leaves[1][bad], leaves[2][bad + 1, 1, 5], leaves[2][bad] = value, value, value
        results.append(all_of([t.requires_grad_() for t in leaves[:3]], ptr, ptr, None, True, leaves[3]))
        for name in ("out", "lse", "dq"):
            assert torch.equal(results[-1][name][:bad], results[0][name][:bad]), (name, value)
            if value != 1.0 and name != "lse":
                assert not torch.isfinite(results[-1][name][bad:, 2:]).all()


@pytest.mark.parametrize("form", ["tiles", "few", "shares"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_visible_infinities_come_to_what_they_are(dtype, form):
    """A weight is above zero: an infinity of either sign stays one, both together and a NaN are NaN, columns apart."""
    segments, rows, keys = {"tiles": (3, 70, 90), "few": (40, 1, 200), "shares": (1, 1, 9000)}[form]
    q, k, v = (normal(segments * n, h, 40, dtype=dtype, seed=s) for s, (n, h) in enumerate(((rows, 4), (keys, 2), (keys, 2))))
    want = torch.zeros(segments, keys, 2, 40)
    for value, keys_at, column in ((math.inf, [3], 0), (-math.inf, [0, 88], 7), (math.inf, [5], 11), (-math.inf, [70], 11),
                                   (math.nan, [60], 39)):
        for at in keys_at:
            v.view(segments, keys, 2, 40)[-1, at, 1, column] = value
            want[-1, at, 1, column] = value
    q_ptr, k_ptr = (on_gpu([n * i for i in range(segments + 1)]) for n in (rows, keys))
    clean = v.clone()
    clean[~torch.isfinite(v)] = 0.5
    out = oeq.packed_attention(q, k, v, q_ptr, k_ptr, causal=rows > 1).view(segments, rows, 4, 40)
    other = oeq.packed_attention(q, k, clean, q_ptr, k_ptr, causal=rows > 1).view(segments, rows, 4, 40)
    for i in range(rows):
        seen = want[-1, :keys - rows + 1 + i, 1]
        expect = seen.sum(0)  # (infinities and NaN add up as they should; elsewhere zero)
        for h in (2, 3):
            got = out[-1, i, h].float().cpu()
            special = ~torch.isfinite(expect)
            assert torch.equal(got[special].nan_to_num(nan=2.0), expect[special].nan_to_num(nan=2.0)), i
            untouched = torch.isfinite(want[-1, :, 1]).all(0)
            assert torch.equal(got[untouched], other[-1, i, h].float().cpu()[untouched])
    assert torch.equal(out[..., :2, :], other[..., :2, :]) and torch.equal(out[:-1], other[:-1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients_that_are_not_finite_stay_with_what_sees_them(dtype):
    n, ptr = 300, on_gpu([0, 130, 300])
    leaves = [normal(n, h, 64, dtype=dtype, seed=s).requires_grad_() for s, h in enumerate((4, 2, 2))]
    g = normal(n, 4, 64, dtype=dtype, seed=4)
    clean = all_of(leaves, ptr, ptr, None, True, g)
    g[200, 3, 9] = -math.inf
    got = all_of(leaves, ptr, ptr, None, True, g)
    seen = torch.arange(n, device="cuda")
    seen = (seen >= 130) & (seen <= 200)
    assert torch.equal(got["dv"][:, 0], clean["dv"][:, 0]) and torch.equal(got["dv"][~seen], clean["dv"][~seen])
    assert (got["dv"][seen, 1, 9] == -math.inf).all()
    others = torch.arange(64, device="cuda") != 9
    assert torch.equal(got["dv"][..., others], clean["dv"][..., others])
    assert torch.equal(got["dk"][~seen], clean["dk"][~seen]) and torch.equal(got["dk"][:, 0], clean["dk"][:, 0])
    assert torch.isnan(got["dq"][200, 3]).all()
    row = torch.arange(n, device="cuda") != 200
    assert torch.equal(got["dq"][row], clean["dq"][row]) and torch.equal(got["dq"][200, :3], clean["dq"][200, :3])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,keys", [(90, 90), (1, 5000)])
def test_numbers_near_the_largest(dtype, rows, keys):
    """Values and output gradients whose sums stay in the type's range though raised weights times them do not."""
    q, k, v = (normal(n, 2, 64, dtype=dtype, seed=s) for s, n in enumerate((rows, keys, keys)))
    q_ptr, k_ptr = on_gpu([0, rows]), on_gpu([0, keys])
    big = (v * 5e36).requires_grad_(False)
    out = oeq.packed_attention(4 * q, k, big, q_ptr, k_ptr)
    want = gradients_64(4 * q, k, big, torch.zeros_like(q))["out"]
    assert torch.isfinite(out).all()
    check_norm(out, *want, dtype, "out", more=2.0 ** -16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    g = 1e28 * normal(rows, 2, 64, dtype=dtype, seed=6)
    want = gradients_64(q, k, v, g)
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(oeq.packed_attention(q, k, v, q_ptr, k_ptr), leaves, g)):
        check_norm(x, *want[name], dtype, name, more=2.0 ** -16)


def test_results_that_are_not_finite_take_a_few_times_as_long():
    """Uninitialised slots of a cache, and an overflow in the output's gradient, as loss scaling makes them."""
    n, slots, ptr = 4000, 512, on_gpu([0, 4000])
    leaves = [normal(n, h, 64, dtype=BF16, seed=s).requires_grad_() for s, h in enumerate((8, 2, 2))]
    q_ptr, k_ptr, k_len = on_gpu(starts([64] * 16)), on_gpu(starts([slots] * 16)), on_gpu([300] * 16)
    prompt = [normal(16 * m, h, 64, dtype=BF16, seed=s) for s, (m, h) in enumerate(((64, 8), (slots, 2), (slots, 2)))]
    g = normal(n, 8, 64, dtype=BF16, seed=5)

    def train():
        torch.autograd.grad(oeq.packed_attention(*leaves, ptr, causal=True), leaves, g)

    def read():
        oeq.packed_attention(*prompt, q_ptr, k_ptr, k_len=k_len, causal=True)

    def spoil_gradient():
        g[3990, 3, 7] = math.inf

    def spoil_slots():
        for t in prompt[1:]:
            t.view(16, slots, 2, 64)[:, 300:] = math.nan

    for call, spoil in ((train, spoil_gradient), (read, spoil_slots)):
        times = []
        for change in (None, spoil):
            if change:
                change()
            call()
            best = math.inf
            for _ in range(3):
                a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                a.record()
                call()
                call()
                b.record()
                b.synchronize()
                best = min(best, a.elapsed_time(b))
            times.append(best)
        assert times[1] <= 10 * times[0] + 0.1, times


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,d", [([5, 1, 9, 31, 32, 33], 32), ([700, 61], 32), ([70, 1, 97], 128), ([1500], 96), ([300] * 12, 64)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_errors_of_attention_as_a_whole(dtype, lens, d, causal):
    """The bounds of single elements allow for the worst of every rounding; as a whole they are far apart. float32: a weight
    is off by 2^-24 of what stands in the exponent (here up to some 8) and of the exponential itself, sums of up to
    1 500 terms by less: 2^-19 of the norm. Operands of 11 or 8 bits would show at once (2^-12 and more)."""
    ptr = starts(lens)
    leaves = [normal(ptr[-1], 3, d, dtype=dtype, seed=s).requires_grad_() for s in range(3)]
    g = normal(ptr[-1], 3, d, dtype=dtype, seed=3)
    out = oeq.packed_attention(*leaves, on_gpu(ptr), causal=causal)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + torch.autograd.grad(out, leaves, g)))
    parts = [gradients_64(*(t[a:b] for t in leaves), g[a:b], causal) for a, b in zip(ptr, ptr[1:])]
    for name, x in got.items():
        value, terms = (torch.cat([p[name][i] for p in parts]) for i in (0, 1))
        check_norm(x, value, terms, dtype, name, more=2.0 ** -19)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,d,heads", [(range(2, 14), 128, 4), (range(2, 14), 32, 4), (range(20, 60), 72, 2), (range(100, 120), 128, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_of_few_keys_lose_what_their_last_rounding_takes(dtype, lens, d, heads, causal):
    """Outputs of short segments have one rounding, their own. Gradients have a second one of that size in ds or p, so that
    the two come to the root of two of one, unless the output's error reaches them through delta. 1 000 rows and more leave the
    ratio of norms within some per cent."""
    lens = [n for n in lens for _ in range(12 if n < 14 else 1)]
    ptr = starts(lens)
    leaves = [normal(ptr[-1], heads, d, dtype=dtype, seed=s).requires_grad_() for s in range(3)]
    g = normal(ptr[-1], heads, d, dtype=dtype, seed=3)
    out = oeq.packed_attention(*leaves, on_gpu(ptr), causal=causal)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + torch.autograd.grad(out, leaves, g)))
    parts = [gradients_64(*(t[a:b] for t in leaves), g[a:b], causal) for a, b in zip(ptr, ptr[1:])]
    for name, x in got.items():
        value = torch.cat([p[name][0] for p in parts])
        once = (value.to(dtype) - value).norm()
        assert (x - value).norm() <= (1.04 if name == "out" else 1.06 * 2 ** 0.5) * once, (name, (x - value).norm() / once)
