"""What of the operators on nodes needs no GPU: the oracle's gradients against differences, tables, shapes of traced calls
and the refusals of the C ABI."""

import ctypes
import math

import pytest
import torch

import openequivariance_amd as oeq
from openequivariance_amd import runtime as rt
from tests import node_oracle as N


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


@pytest.mark.parametrize("causal", [False, True])
def test_oracle_gradients_against_differences(causal):
    """The formulas that the kernels' gradients are compared with, in 64 bits."""
    gen = torch.Generator().manual_seed(1)
    q_ptr, k_ptr, k_len = starts([4, 0, 3]), starts([6, 2, 5]), [5, 1, 2]
    q, k, v, g = (torch.randn(n, h, 8, generator=gen, dtype=torch.float64) for n, h in ((7, 4), (13, 2), (13, 2), (7, 4)))
    views = N.segment_views(q_ptr, k_ptr, k_len, 13, causal)
    val, _ = N.attention(q, k, v, views, 0.4, g)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        way, step = torch.randn(x.shape, generator=gen, dtype=torch.float64), 1e-5
        sides = []
        for sign in (1, -1):
            moved = [t + sign * step * way if t is x else t for t in (q, k, v)]
            sides.append((N.attention(*moved, views, 0.4)[0]["out"] * g).sum())
        along = (val[name] * way).sum()
        # central differences of a function of order one: step^2 and 1e-16 / step
        assert abs((sides[0] - sides[1]) / (2 * step) - along) <= 1e-8 * (1 + abs(along)), name


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation_against_differences(interleaved):
    gen = torch.Generator().manual_seed(2)
    x, g = (torch.randn(5, 2, 24, generator=gen, dtype=torch.float64) for _ in range(2))
    w, positions = 1 + 0.2 * torch.randn(24, generator=gen, dtype=torch.float64), torch.tensor([0, 3, 9, 1, 2])
    table = oeq.rotary_table(10, 16).double()
    out, _, dx, _, dw, _ = N.rotate(x, w, positions, table, interleaved, 1e-6, g)
    for t, grad in ((x, dx), (w, dw)):
        way, step = torch.randn(t.shape, generator=gen, dtype=torch.float64), 1e-5
        sides = [(N.rotate(x + (sign * step * way if t is x else 0), w + (sign * step * way if t is w else 0), positions,
                           table, interleaved, 1e-6)[0] * g).sum() for sign in (1, -1)]
        along = (grad * way).sum()
        assert abs((sides[0] - sides[1]) / (2 * step) - along) <= 1e-8 * (1 + abs(along))
    # turning keeps lengths, and products of turned heads depend on the distance of their positions alone
    plain = N.rotate(x, None, positions, table, interleaved, 0.0)[0]
    assert torch.allclose(plain.norm(dim=-1), x.norm(dim=-1), rtol=1e-6)
    y = torch.randn(1, 1, 16, generator=gen, dtype=torch.float64)
    dots = [(N.rotate(y, None, torch.tensor([a]), table, interleaved, 0.0)[0]
             * N.rotate(y.flip(-1), None, torch.tensor([a + 4]), table, interleaved, 0.0)[0]).sum() for a in (0, 5)]
    assert abs(dots[0] - dots[1]) < 1e-5


def test_rotary_tables():
    table = oeq.rotary_table(100, 32)
    angle = 73 * 10000.0 ** (-2 * 5 / 32)
    assert table.shape == (100, 2, 16) and table.dtype == torch.float32
    assert abs(table[73, 0, 5] - math.cos(angle)) < 1e-7 and abs(table[73, 1, 5] - math.sin(angle)) < 1e-7
    # stretched: positions divided throughout, or only where pairs turn slowly
    assert torch.allclose(oeq.rotary_table(100, 32, scaling=4.0)[40], table[10], atol=1e-6)
    mixed = oeq.rotary_table(100, 32, scaling=4.0, trained_length=512)
    assert torch.equal(mixed[:, :, 0], table[:, :, 0])  # 81 turns within 512 positions
    assert torch.allclose(mixed[40, :, 15], table[10, :, 15], atol=1e-6)  # less than one
    between = torch.atan2(mixed[1, 1], mixed[1, 0]) / torch.atan2(table[1, 1], table[1, 0])
    assert (between[:-1] - between[1:] >= -1e-5).all() and between[3] < 1
    for bad in (dict(rotary_dim=12), dict(rotary_dim=0), dict(rotary_dim=16, scaling=0.0), dict(rotary_dim=16, base=-1.0)):
        with pytest.raises(ValueError):
            oeq.rotary_table(10, **bad)


def test_generator_against_published_words():
    """Known answers of Philox-4x32 with ten rounds for counter and key of zeros and of ones."""
    assert N.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert N.philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_dropout_module():
    module = oeq.IrrepDropout("2x0e+2x1o", 0.5)
    assert module.channels.tolist() == [0, 1] + [2] * 3 + [3] * 3
    assert oeq.IrrepDropout("2x0e+2x1o", 0.5, layout="ir_mul").channels.tolist() == [0, 1] + [2, 3] * 3
    assert "p=0.5" in repr(module) and not module.state_dict()
    x = torch.ones(3, 8)
    module.eval()
    assert module(x) is x and torch.equal(module(x, x), 2 * x)
    with pytest.raises(ValueError):
        oeq.IrrepDropout("2x0e", 2.0)
    with pytest.raises(ValueError):
        oeq.IrrepDropout("2x0e", 0.1, layout="other")


def test_traced_calls_have_the_kernels_shapes():
    q, k = torch.empty(7, 4, 32, device="meta", dtype=torch.bfloat16), torch.empty(9, 2, 32, device="meta", dtype=torch.bfloat16)
    ptr, at = torch.empty(3, device="meta", dtype=torch.int64), torch.empty(7, device="meta", dtype=torch.int64)
    out, lse = oeq.packed_attention(q, k, k, ptr, ptr, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (7, 4) and lse.dtype == torch.float32
    table, w = torch.empty(5, 2, 8, device="meta"), torch.empty(32, device="meta", dtype=torch.bfloat16)
    turned = oeq.qk_norm_rotary(q, k[:7], at, table, w)
    assert [t.shape for t in turned] == [q.shape, k[:7].shape]
    grads = torch.ops.oeq_amd.qk_norm_rotary_backward(*turned, q, k[:7], at, table, w, None, 1e-6, False)
    assert [tuple(t.shape) for t in grads] == [(7, 4, 32), (7, 2, 32), (32,), (0,)]
    module = oeq.IrrepDropout("4x0e", 0.1).to("meta")
    assert module(torch.empty(2, 4, device="meta"), seed=at[:2]).shape == (2, 4)


def _attention(**changes):
    fields = dict(type=2, causal=0, segments=1, q_heads=4, k_heads=2, head_dim=32, scale=1.0, q_rows=8, k_rows=8,
                  q_row_stride=128, q_head_stride=32, k_row_stride=64, k_head_stride=32, v_row_stride=64, v_head_stride=32,
                  q=16, k=16, v=16, q_ptr=16, k_ptr=16)
    fields.update(changes)
    return rt._Attention(**fields)


def test_c_abi_refuses_attention_arguments():
    """Checked on the host before anything is launched (the addresses are never read)."""
    lib = rt.load_library()

    def forward(a, out=16, stats=16):
        return lib.oeq_attention_forward(ctypes.byref(a) if a is not None else None, out, None, stats, None, 0, None)

    assert lib.oeq_attention_forward(ctypes.byref(_attention(q_rows=0)), None, None, None, None, 0, None) == 0
    assert forward(None) == -1
    for changes, text in ((dict(type=3), "element type"), (dict(head_dim=12), "heads of 12"), (dict(head_dim=136), "heads of 136"),
                          (dict(head_dim=0), "heads of 0"), (dict(q_heads=3), "3 query heads"), (dict(k_heads=0), "0 key heads"),
                          (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
                          (dict(q_rows=-1), "query rows"), (dict(k_rows=1 << 31), "key rows"), (dict(segments=-1), "segments"),
                          (dict(k_row_stride=60), "stride of 60"), (dict(v_row_stride=1 << 30), "row stride"),
                          (dict(q_row_stride=-128), "row stride"), (dict(q=0), "NULL"), (dict(v=0), "NULL"),
                          (dict(q_ptr=0), "NULL"), (dict(k=8), "unaligned")):
        assert forward(_attention(**changes)) == -1, changes
        assert text in lib.oeq_last_error().decode(), changes
    assert forward(_attention(), out=None) == -1 and forward(_attention(), out=8) == -1
    backward = lib.oeq_attention_backward
    a = _attention()
    assert lib.oeq_attention_backward_workspace_bytes(ctypes.byref(a)) == 4 * 128 * 4
    assert backward(ctypes.byref(a), 16, None, 16, 16, 128, 32, 16, 16, 16, 16, 100, None) == -1
    assert "workspace" in lib.oeq_last_error().decode()
    assert backward(ctypes.byref(a), 16, None, 16, 16, 127, 32, 16, 16, 16, 16, 2048, None) == -1
    assert "strides" in lib.oeq_last_error().decode()


def test_c_abi_refuses_rotation_and_dropout_arguments():
    lib = rt.load_library()

    def rotary(**changes):
        fields = dict(type=0, interleaved=0, q_heads=4, k_heads=2, head_dim=32, rotary_dim=16, eps=1e-6, rows=3, table_rows=9,
                      q_row_stride=128, q_head_stride=32, k_row_stride=64, k_head_stride=32, q=16, k=16, positions=16, table=16)
        fields.update(changes)
        return ctypes.byref(rt._QkRotary(**fields))

    assert lib.oeq_qk_norm_rotary(rotary(rows=0), None, None, None) == 0
    for changes, text in ((dict(type=3), "element type"), (dict(head_dim=20), "heads of 20"), (dict(rotary_dim=40), "40 turned"),
                          (dict(rotary_dim=12), "12 turned"), (dict(rows=-1), "rows"), (dict(q=0), "NULL"),
                          (dict(table=0), "NULL"), (dict(k_head_stride=33), "stride of 33"), (dict(q_weight=20), "unaligned")):
        assert lib.oeq_qk_norm_rotary(rotary(**changes), 16, 16, None) == -1, changes
        assert text in lib.oeq_last_error().decode(), changes
    assert lib.oeq_qk_norm_rotary(rotary(), None, 16, None) == -1
    append = lib.oeq_qk_norm_rotary_append
    assert append(rotary(), 16, 64, 32, 16, 16, 64, 32, 16, 64, 33, 16, 5, None) == -1
    assert append(rotary(), 16, 64, 32, 16, 16, 64, 32, 16, 64, 32, 16, -5, None) == -1
    assert append(rotary(), 16, 64, 32, 16, None, 64, 32, 16, 64, 32, 16, 5, None) == -1
    a = rotary(q_weight=16)
    need = lib.oeq_qk_norm_rotary_backward_workspace_bytes(a)
    assert need > 0 and lib.oeq_qk_norm_rotary_backward_workspace_bytes(rotary()) == 0
    back = lib.oeq_qk_norm_rotary_backward
    assert back(a, 16, 128, 32, 16, 64, 32, 16, 16, 16, None, 16, need - 1, None) == -1
    assert back(a, 16, 128, 32, 16, 64, 32, 16, 16, None, None, 16, need, None) == -1
    drop = lib.oeq_irrep_dropout
    assert drop(0, 0, 8, None, None, None, None, None, 0.5, None) == 0
    for args, text in (((7, 3, 8, 16, None, 16, 16, 16, 0.5, None), "element type"), ((0, -3, 8, 16, None, 16, 16, 16, 0.5, None), "rows"),
                       ((0, 3, 8, 16, None, 16, 16, 16, 1.5, None), "p ="), ((0, 3, 8, 16, None, 16, 16, 16, math.nan, None), "p ="),
                       ((0, 3, 8, 16, None, 16, None, 16, 0.5, None), "NULL"), ((0, 3, 8, 8, None, 16, 16, 16, 0.5, None), "unaligned")):
        assert drop(*args) == -1 and text in lib.oeq_last_error().decode(), args


def test_no_kernel_of_the_library_has_scratch_memory():
    """Registers spilled in a loop cost more than any of the operators' other choices; reads back the built library."""
    blob = rt.lib_path().read_bytes()
    objects, at = [], 0
    while True:
        at = blob.find(b"\x7fELF", at + 1)
        if at < 0:
            break
        if int.from_bytes(blob[at + 18:at + 20], "little") == 224:  # EM_AMDGPU
            objects.append(blob[at:])
    names = {}
    for elf in objects:
        names.update(rt.kernel_resources(elf))
    attention = {n: r for n, r in names.items() if "packed_attention" in n}
    assert len(attention) >= 30
    assert not {n: r for n, r in attention.items() if r[1] > 0}


def test_norm_rotation_dropout_and_ordering_have_no_scratch_memory():
    blob, at, names = rt.lib_path().read_bytes(), 0, {}
    while (at := blob.find(b"\x7fELF", at + 1)) >= 0:
        if int.from_bytes(blob[at + 18:at + 20], "little") == 224:  # EM_AMDGPU
            names.update(rt.kernel_resources(blob[at:]))
    for part, least in (("qk_rotary", 9), ("irrep_dropout", 4), ("order_tiles", 1)):
        found = {n: r for n, r in names.items() if part in n}
        assert len(found) >= least, (part, len(found))
        assert not {n: r for n, r in found.items() if r[1] > 0}


def test_forward_mode_derivatives_are_right_or_refused():
    """A dual tensor need not require a gradient; its tangent must not get lost on the way."""
    import torch.autograd.forward_ad as forward_ad
    q, k = torch.empty(7, 4, 32, device="meta"), torch.empty(7, 2, 32, device="meta")
    ptr, at, seed = (torch.empty(n, device="meta", dtype=torch.int64) for n in (3, 7, 2))
    table, w, x = torch.empty(5, 2, 8, device="meta"), torch.empty(32, device="meta"), torch.empty(6, 8, device="meta")
    module = oeq.IrrepDropout("2x0e+2x1o", 0.1).to("meta")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.empty_like(t))

        for call in (lambda: oeq.packed_attention(dual(q), k, k, ptr), lambda: oeq.packed_attention(q, dual(k), k, ptr),
                     lambda: oeq.packed_attention(q, k, dual(k), ptr), lambda: oeq.qk_norm_rotary(dual(q), k, at, table),
                     lambda: oeq.qk_norm_rotary(q, dual(k), at, table, w),
                     lambda: oeq.qk_norm_rotary(q, k, at, table, None, dual(w)),
                     lambda: oeq.qk_norm_rotary(q, k, at, dual(table)),
                     lambda: oeq.qk_norm_rotary_append(dual(q), k, k, at, table, k.clone(), k.clone(), at),
                     lambda: torch.ops.oeq_amd.qk_norm_rotary_backward(dual(q), k, q, k, at, table, w, None, 1e-6, False)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        for args in ((dual(x), None), (dual(x), x), (x, dual(x)), (dual(x), dual(x)), (dual(x).requires_grad_(), x)):
            out = module(*args, seed=seed)
            tangent = forward_ad.unpack_dual(out).tangent
            assert tangent is not None and tangent.shape == x.shape
            assert out.requires_grad == args[0].requires_grad
        assert forward_ad.unpack_dual(module(x, x, seed=seed)).tangent is None
    value, tangent = torch.func.jvp(lambda t: module(t, seed=seed), (x,), (x,))
    assert value.shape == tangent.shape == x.shape


class _Elsewhere(torch.Tensor):
    """A tensor that says which GPU it is on and has no memory."""

    @staticmethod
    def __new__(cls, *shape, device=0, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=f"cuda:{device}")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(func)


def test_operands_on_another_gpu_are_refused():
    """Every operand in turn, by the GPU's code of the op itself (which ends at its checks)."""
    t, i64 = _Elsewhere, torch.int64

    def make(shape, device):
        dtype = shape[-1] if isinstance(shape[-1], torch.dtype) else torch.float32
        return t(*[n for n in shape if not isinstance(n, torch.dtype)], device=device, dtype=dtype)

    problem = oeq.TPProblem("4x0e", "1x0e", "4x0e", [(0, 0, 0, "uvu", True)], shared_weights=False, internal_weights=False)
    product, conv = oeq.TensorProduct(problem), oeq.TensorProductConv(problem)
    n, wn = 5, problem.weight_numel
    attention = dict(q=(7, 4, 32), k=(9, 2, 32), v=(9, 2, 32), q_ptr=(3, i64), k_ptr=(3, i64), k_len=(2, i64))
    rotary = dict(q=(7, 4, 32), k=(7, 2, 32), positions=(7, i64), table=(5, 2, 8), q_weight=(32,), k_weight=(32,))
    ops = torch.ops.oeq_amd
    calls = [
        (attention, lambda a: ops.packed_attention.default.redispatch(_cuda(), *a.values(), False, 0.5)),
        (dict(grad=(7, 4, 32), **{n: s for n, s in attention.items() if n in "qkv"}, out=(7, 4, 32), log2_sum=(4, 128),
              rest=(0,), q_ptr=(3, i64), k_ptr=(3, i64)),
         lambda a: ops.packed_attention_backward.default.redispatch(_cuda(), *a.values(), None, False, 0.5)),
        (rotary, lambda a: ops.qk_norm_rotary.default.redispatch(_cuda(), *a.values(), 1e-6, False)),
        (dict(q_grad=(7, 4, 32), k_grad=(7, 2, 32), **rotary),
         lambda a: ops.qk_norm_rotary_backward.default.redispatch(_cuda(), *a.values(), 1e-6, False)),
        (dict(q=(7, 4, 32), k=(7, 2, 32), v=(7, 2, 32), positions=(7, i64), table=(5, 2, 8), k_cache=(20, 2, 32),
              v_cache=(20, 2, 32), slots=(7, i64)),
         lambda a: ops.qk_norm_rotary_append.default.redispatch(_cuda(), *a.values(), None, None, 1e-6, False)),
        (dict(x=(5, 4), residual=(5, 4), channels=(4, torch.int32), seed=(2, i64)),
         lambda a: ops.irrep_dropout.default.redispatch(_cuda(), *a.values(), 0.5)),
        (dict(x=(n, 4), y=(n, 1), w=(n, wn)),
         lambda a: ops.tp_forward.default.redispatch(_cuda(), *a.values(), product.kid, None)),
        (dict(x=(6, 4), y=(n, 1), w=(n, wn), rows=(n, i64), cols=(n, i64)),
         lambda a: ops.conv_forward.default.redispatch(_cuda(), *a.values(), make((0, i64), 0), conv.kid, None)),
    ]
    for shapes, call in calls:
        for name in shapes:
            if name == "rest":  # (empty: not read)
                continue
            args = {m: make(s, int(m == name)) for m, s in shapes.items()}
            with pytest.raises(RuntimeError, match="is on cuda:"):
                call(args)


def _cuda():
    return torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)


def test_dropout_of_a_module_first_called_in_inference_mode():
    """Its table moves to the input's device with that call and stays good for training."""
    x, seed = torch.empty(3, 4, device="meta"), torch.empty(2, dtype=torch.int64, device="meta")
    for mode in (torch.inference_mode, torch.no_grad):
        module = oeq.IrrepDropout("1x0e+1x1o", 0.1)
        with mode():
            module(x, seed=seed)
        assert module.channels.device.type == "meta" and not module.channels.is_inference()
        assert module(x.clone().requires_grad_(), seed=seed).requires_grad


def test_caches_that_are_written_count_it():
    """What autograd saved of a cache is known to have changed, whatever mode wrote to it."""
    def operands():
        q, k = torch.empty(7, 4, 32, device="meta"), torch.empty(7, 2, 32, device="meta")
        at, table = torch.empty(7, device="meta", dtype=torch.int64), torch.empty(5, 2, 8, device="meta")
        return q, k, k, at, table, torch.empty(20, 2, 32, device="meta"), torch.empty(20, 2, 32, device="meta"), at

    args = operands()
    written = args[5:7]
    for n, mode in enumerate((torch.no_grad, torch.inference_mode, torch.enable_grad), 1):
        with mode():
            oeq.qk_norm_rotary_append(*args)
        assert [c._version for c in written] == [n, n] and args[0]._version == 0
    with torch.inference_mode():
        assert oeq.qk_norm_rotary_append(*operands()).shape == (7, 4, 32)  # caches without a count


def test_a_table_that_wants_a_gradient_is_refused():
    q, k = torch.empty(7, 4, 32, device="meta", requires_grad=True), torch.empty(7, 2, 32, device="meta")
    at, table = torch.empty(7, device="meta", dtype=torch.int64), torch.empty(5, 2, 8, device="meta", requires_grad=True)
    with pytest.raises(RuntimeError, match="table has no gradient"):
        oeq.qk_norm_rotary(q, k, at, table)
    assert oeq.qk_norm_rotary(q, k, at, table.detach())[0].requires_grad
    with torch.no_grad():
        oeq.qk_norm_rotary(q, k, at, table)


def test_attention_without_elements_is_the_ops_to_refuse():
    ptr = _Elsewhere(2, dtype=torch.int64)
    for shape in ((5, 2, 0), ()):
        q = _Elsewhere(*shape)
        calls = []

        def op(*args):
            calls.append(args)
            return (None, None, None)

        from openequivariance_amd._torch import nodes
        real, nodes._packed_attention = nodes._packed_attention, op
        try:
            oeq.packed_attention(q, q, q, ptr)
        finally:
            nodes._packed_attention = real
        assert calls[0][-1] == 1.0
    with pytest.raises(RuntimeError, match="multiple of 8"):
        q = _Elsewhere(5, 2, 0)
        torch.ops.oeq_amd.packed_attention.default.redispatch(_cuda(), q, q, q, ptr, ptr, None, False, 1.0)
