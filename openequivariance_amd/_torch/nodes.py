"""Operators on the nodes of a batch: attention among the nodes of a structure (or the tokens of a sequence), the norm
of its queries and keys with the rotation by position, the same for a cache that grows by one token at a time, and
dropout of whole irreps.

They stand beside the tensor products in models that mix equivariant messages with attention over all nodes of a
structure, or that generate structures token by token; the reference has no counterpart of them. Batches are laid out
as the convolution has them: the rows of all structures one after the other, ``ptr[s]`` .. ``ptr[s + 1]`` those of
structure ``s`` (int64, on the GPU; nothing is copied to the host). The kernels are part of liboeq_amd.so and take
float32, float16 and bfloat16 (dropout float64 too); sums, norms and softmax statistics are held in 32 bits.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import runtime as rt
from ..core.spec import Irreps
from . import ops

_PAIRS = "Tensor q, Tensor k, Tensor positions, Tensor table"
_SEGMENTS = "Tensor q_ptr, Tensor k_ptr, Tensor? k_len, bool causal, float scale"
_NORM = "Tensor? q_weight, Tensor? k_weight, float eps, bool interleaved"
for _schema in (
        f"packed_attention(Tensor q, Tensor k, Tensor v, {_SEGMENTS}, bool keep_rest=False) -> (Tensor, Tensor, Tensor)",
        "packed_attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor out, Tensor log2_sum, Tensor rest, "
        f"{_SEGMENTS}) -> (Tensor, Tensor, Tensor)",
        f"qk_norm_rotary({_PAIRS}, {_NORM}) -> (Tensor, Tensor)",
        f"qk_norm_rotary_backward(Tensor q_grad, Tensor k_grad, {_PAIRS}, {_NORM}) -> (Tensor, Tensor, Tensor, Tensor)",
        "qk_norm_rotary_append(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor table, Tensor(a!) k_cache, "
        f"Tensor(b!) v_cache, Tensor slots, {_NORM}) -> Tensor",
        "irrep_dropout(Tensor x, Tensor? residual, Tensor channels, Tensor seed, float p) -> Tensor"):
    ops.define_op(_schema)

_packed_attention = torch.ops.oeq_amd.packed_attention.default
_qk_norm_rotary = torch.ops.oeq_amd.qk_norm_rotary.default
_qk_norm_rotary_append = torch.ops.oeq_amd.qk_norm_rotary_append.default
_irrep_dropout = torch.ops.oeq_amd.irrep_dropout.default


def _stat_stride(rows):
    return (rows + 63) // 64 * 64 + 64


@torch.library.register_fake("oeq_amd::packed_attention")
def _(q, k, v, q_ptr, k_ptr, k_len, causal, scale, keep_rest=False):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
            q.new_empty((q.shape[1], _stat_stride(q.shape[0])), dtype=torch.float32),
            q.new_empty(q.shape if keep_rest and q.dtype.itemsize == 2 else 0))


@torch.library.register_fake("oeq_amd::packed_attention_backward")
def _(grad, q, k, v, out, log2_sum, rest, q_ptr, k_ptr, k_len, causal, scale):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))


@torch.library.register_fake("oeq_amd::qk_norm_rotary")
def _(q, k, positions, table, q_weight, k_weight, eps, interleaved):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))


@torch.library.register_fake("oeq_amd::qk_norm_rotary_backward")
def _(q_grad, k_grad, q, k, positions, table, q_weight, k_weight, eps, interleaved):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device),
            q.new_empty(0 if q_weight is None else q.shape[2]), q.new_empty(0 if k_weight is None else q.shape[2]))


@torch.library.register_fake("oeq_amd::qk_norm_rotary_append")
def _(q, k, v, positions, table, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


@torch.library.register_fake("oeq_amd::irrep_dropout")
def _(x, residual, channels, seed, p):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_ptr: torch.Tensor,
                     k_ptr: Optional[torch.Tensor] = None, *, k_len: Optional[torch.Tensor] = None, causal: bool = False,
                     scale: Optional[float] = None, return_lse: bool = False
                     ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    r"""Attention of the rows of every segment to the keys of the same segment, ``softmax(scale q k^T) v``.

    :param q: ``[rows, q_heads, head_dim]``, ``head_dim`` a multiple of 8 up to 128. Any strides; views whose heads are
        contiguous and aligned to 16 bytes (parts of one projection) are read in place.
    :param k, v: ``[key rows, k_heads, head_dim]``; query head ``h`` reads key head ``h // (q_heads // k_heads)``.
    :param q_ptr: ``[segments + 1]`` ascending starts of the segments' query rows, int64. Rows outside all segments
        return 0.
    :param k_ptr: the same for the key rows; ``q_ptr`` where left out.
    :param k_len: ``[segments]``: how many rows from ``k_ptr[s]`` on are keys (a cache that is partly filled); all up to
        ``k_ptr[s + 1]`` where left out.
    :param causal: the last row of a segment sees all its keys, the one before it all but the last, and so on.
    :param scale: positive; ``head_dim ** -0.5`` where left out.
    :param return_lse: also return the logarithm of each row's sum of exponentials, ``[rows, q_heads]`` in float32
        (without a gradient).
    :return: ``[rows, q_heads, head_dim]``. Rows that see no key are 0. What a row does not see has no influence on it
        and gets no gradient from it, infinities and NaN included. Runs and their gradients are reproducible bit by bit.
    """
    if scale is None:  # (heads without elements: the op says so)
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    out, log2_sum, _rest = _packed_attention(q, k, v, q_ptr, q_ptr if k_ptr is None else k_ptr, k_len, causal, scale)
    if return_lse:
        return out, (log2_sum[:, :q.shape[0]] * math.log(2.0)).t()
    return out


def rotary_table(length: int, rotary_dim: int, *, base: float = 10000.0, scaling: float = 1.0,
                 trained_length: Optional[int] = None, device=None) -> torch.Tensor:
    r"""Cosines and sines for :func:`qk_norm_rotary`, ``[length, 2, rotary_dim / 2]`` in float32 (computed in 64 bits):
    pair ``i`` of position ``t`` turns by ``t base ** (-2 i / rotary_dim)``.

    :param scaling: for contexts that many times longer than a model was trained on. Alone it divides all positions.
    :param trained_length: with it, a pair keeps its frequency if it turns 32 times or more within that length, takes
        the divided one if it turns once or less, and goes from one to the other linearly in between.
    """
    if rotary_dim <= 0 or rotary_dim % 8:
        raise ValueError(f"rotary_dim must be a positive multiple of 8, got {rotary_dim}")
    if length < 0 or not base > 0 or not scaling > 0:
        raise ValueError(f"rotary_table: length {length}, base {base}, scaling {scaling}")
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if trained_length is None:
        freq = freq / scaling
    else:
        turns = freq * trained_length / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / scaling)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=1).float()


def _weights(q, *weights):
    """Weights of a norm in the queries' type: under autocast projections come in 16 bits and parameters in 32."""
    if torch.is_autocast_enabled("cuda"):
        return [w if w is None else w.to(q.dtype) for w in weights]
    return weights


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""Queries and keys normed head by head and turned by position, in one pass over them.

    :param q, k: ``[rows, heads, head_dim]``, ``head_dim`` a multiple of 8 up to 128; views as in
        :func:`packed_attention`.
    :param positions: ``[rows]``, int64, each a row of ``table`` (another gives NaN).
    :param table: ``[positions, 2, rotary_dim / 2]`` cosines and sines (:func:`rotary_table`). The first ``rotary_dim``
        elements of a head are turned, the rest only normed. It has no gradient.
    :param q_weight, k_weight: ``[head_dim]``: ``x -> weight x / sqrt(mean(x^2) + eps)``; no norm where left out.
    :param interleaved: pairs are neighbours ``2 i, 2 i + 1`` instead of ``i, i + rotary_dim / 2``.
    """
    q_weight, k_weight = _weights(q, q_weight, k_weight)
    return _qk_norm_rotary(q, k, positions, table, q_weight, k_weight, eps, interleaved)


def qk_norm_rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                          k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                          eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    r"""The serving form of :func:`qk_norm_rotary`: returns the queries and writes the keys, and the values as they are, to
    the rows of the caches that ``slots`` names, in the same launch.

    :param k_cache, v_cache: ``[cache rows, k_heads, head_dim]``, written in place.
    :param slots: ``[rows]``, int64; rows whose slot is not one of the caches' (-1, say) are not written. Slots are
        different from each other.
    """
    q_weight, k_weight = _weights(q, q_weight, k_weight)
    return _qk_norm_rotary_append(q, k, v, positions, table, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved)


class IrrepDropout(torch.nn.Module):
    r"""Dropout of whole irreps: each channel of each node keeps all its components (scaled by ``1 / (1 - p)``) or none,
    so that the result turns with its input; scalars are dropped one by one. The mask is not stored: forward and
    backward take it from a counter-based generator.

    :param irreps: of the features' last dimension, e.g. ``"128x0e+128x1o"``.
    :param p: probability of a channel to be dropped, in steps of 2^-16.
    :param layout: ``"mul_ir"`` or ``"ir_mul"``, as in :class:`TPProblem`.

    A module that was not moved to the GPU moves its table there with its first call, except while a graph is captured:
    move the module before.
    """

    def __init__(self, irreps, p: float, layout: str = "mul_ir"):
        super().__init__()
        from ..core.layout import check_layouts
        check_layouts(layout, layout)
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be between 0 and 1, got {p}")
        self.irreps, self.p, self.layout = Irreps(irreps), float(p), layout
        channels, first = [], 0
        for mul, ir in self.irreps:
            one = torch.arange(first, first + mul, dtype=torch.int32)
            channels.append(one.repeat_interleave(ir.dim) if layout == "mul_ir" else one.repeat(ir.dim))
            first += mul
        self.register_buffer("channels", torch.cat(channels) if channels else torch.empty(0, dtype=torch.int32),
                             persistent=False)

    def extra_repr(self) -> str:
        return f"{self.irreps}, p={self.p}, layout={self.layout!r}"

    def _channels_on(self, x: torch.Tensor) -> torch.Tensor:
        """The table of a module that was not moved to its input's device: it moves with the first call. Not while a graph
        is captured (the copy from host memory would end the capture, and what it allocates belong to the graph), and
        not as a tensor of inference mode, which later training steps could not save."""
        if torch.compiler.is_compiling():
            return self.channels.to(x.device)
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"IrrepDropout is on {self.channels.device} and its input on {x.device}: move the module there "
                               "before a graph is captured")
        with torch.inference_mode(False):
            channels = self.channels.to(x.device)
        if type(channels) is torch.Tensor:  # (not a traced stand-in)
            self.channels = channels
        return channels

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                seed: Optional[torch.Tensor] = None) -> torch.Tensor:
        r"""
        :param x: ``[rows, irreps.dim]``
        :param residual: added to the result in the same pass.
        :param seed: two int64 on the GPU; the same seed gives the same mask. Drawn from torch's generator of the device
            where left out.
        :return: ``residual + dropout(x)``; in evaluation mode ``residual + x``.
        """
        if not self.training:
            return x if residual is None else x + residual
        if seed is None:
            seed = torch.empty(2, dtype=torch.int64, device=x.device).random_()
        channels = self.channels if self.channels.device == x.device else self._channels_on(x)
        if residual is not None and torch.is_autocast_enabled("cuda"):
            x = x.to(residual.dtype)  # (a projection in 16 bits on its way into a stream in 32)
        return _irrep_dropout(x, residual, channels, seed, self.p)
