"""Operators whose parameters are chosen row by row: an embedding of the rows' types, linear layers with a matrix for every
type, and low-rank adapters beside a projection that all rows share.

A batch has a type for every row: the species of an atom, the expert that a token is sent to, the adapter of a request or
a data set (int64, on the GPU; nothing is copied to the host). Rows whose type is not one of ``0 .. types - 1`` (-1, say) have no
parameters: they become 0 (with adapters: the shared projection alone) and leave no gradient. The reference has no counterpart of these.
The kernels are part of liboeq_amd.so and take float32, float16 and bfloat16; sums are held in 32 bits, and results and
gradients are reproducible bit by bit.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import ops

_INDEX = "Tensor? order, Tensor? ptr"
_ADAPTERS = "Tensor x, Tensor weight, Tensor down, Tensor up, Tensor types, Tensor? scale"
for _schema in (
        "group_rows(Tensor types, int count) -> (Tensor, Tensor)",
        f"type_embedding(Tensor types, Tensor weight, float scale, {_INDEX}) -> Tensor",
        f"type_embedding_backward(Tensor grad, Tensor types, int count, float scale, {_INDEX}) -> Tensor",
        f"typed_linear(Tensor x, Tensor weight, Tensor types, Tensor? bias, {_INDEX}) -> Tensor",
        f"typed_linear_backward(Tensor grad, Tensor x, Tensor weight, Tensor types, {_INDEX}, bool want_x, bool want_weight, "
        "bool want_bias) -> (Tensor, Tensor, Tensor)",
        f"adapter_linear({_ADAPTERS}, {_INDEX}) -> (Tensor, Tensor)",
        f"adapter_linear_backward(Tensor grad, {_ADAPTERS}, Tensor thin, {_INDEX}, bool want_x, bool want_weight, "
        "bool want_down, bool want_up) -> (Tensor, Tensor, Tensor, Tensor)"):
    ops.define_op(_schema)

_group_rows = torch.ops.oeq_amd.group_rows.default
_type_embedding = torch.ops.oeq_amd.type_embedding.default
_typed_linear = torch.ops.oeq_amd.typed_linear.default
_adapter_linear = torch.ops.oeq_amd.adapter_linear.default


def _like(t, *shape):
    return torch.empty(shape, dtype=t.dtype, device=t.device)


@torch.library.register_fake("oeq_amd::group_rows")
def _(types, count):
    return (types.new_empty(types.shape[0], dtype=torch.int32), types.new_empty(count + 1, dtype=torch.int32))


@torch.library.register_fake("oeq_amd::type_embedding")
def _(types, weight, scale, order, ptr):
    return _like(weight, types.shape[0], weight.shape[1])


@torch.library.register_fake("oeq_amd::type_embedding_backward")
def _(grad, types, count, scale, order, ptr):
    return _like(grad, count, grad.shape[1])


@torch.library.register_fake("oeq_amd::typed_linear")
def _(x, weight, types, bias, order, ptr):
    return _like(x, *x.shape[:-1], weight.shape[1])


@torch.library.register_fake("oeq_amd::typed_linear_backward")
def _(grad, x, weight, types, order, ptr, want_x, want_weight, want_bias):
    return (_like(x, *(x.shape if want_x else (0,))), _like(x, *(weight.shape if want_weight else (0,))),
            _like(x, *(weight.shape[:2] if want_bias else (0,))))


@torch.library.register_fake("oeq_amd::adapter_linear")
def _(x, weight, down, up, types, scale, order, ptr):
    return (_like(x, x.shape[0], weight.shape[0]),
            x.new_empty((x.shape[0], (down.shape[1] + 7) // 8 * 8), dtype=torch.float32))


@torch.library.register_fake("oeq_amd::adapter_linear_backward")
def _(grad, x, weight, down, up, types, scale, thin, order, ptr, want_x, want_weight, want_down, want_up):
    return tuple(_like(x, *(t.shape if want else (0,)))
                 for t, want in ((x, want_x), (weight, want_weight), (down, want_down), (up, want_up)))


class RowGroups(NamedTuple):
    """Rows grouped by type (:func:`group_rows`): ``order`` holds the row numbers by type, ascending within a type, those
    without a type last; type ``t`` has the places ``ptr[t]`` .. ``ptr[t + 1]`` of it (both int32)."""
    types: torch.Tensor
    order: torch.Tensor
    ptr: torch.Tensor


def group_rows(types: torch.Tensor, num_types: int) -> RowGroups:
    r"""The index that the operators of this module go by. They make it themselves from a batch's types; made here it serves
    all layers of a model that choose their parameters by the same types.

    :param types: ``[rows]``, int64.
    """
    return RowGroups(types, *_group_rows(types, num_types))


def _index(types):
    return (types.types, types.order, types.ptr) if isinstance(types, RowGroups) else (types, None, None)


def _cast(*tensors):
    """Under autocast, as torch's own linear layers."""
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        return [t.to(to) if t is not None and t.is_floating_point() and t.dtype != torch.float64 else t for t in tensors]
    return tensors


def type_embedding(types: Union[torch.Tensor, RowGroups], weight: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    r"""``scale * weight[types]``. The gradient of the table sums the rows of each type in their order.

    :param types: ``[rows]``, int64, or their index.
    :param weight: ``[types, channels]``; up to 2^19 channels have a gradient.
    """
    types, order, ptr = _index(types)
    return _type_embedding(types, weight, scale, order, ptr)


def typed_linear(x: torch.Tensor, weight: torch.Tensor, types: Union[torch.Tensor, RowGroups],
                 bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    r"""Each row times the matrix of its type: ``x[i] @ weight[types[i]].T + bias[types[i]]``. Differentiable any number of times.

    :param x: ``[rows, in]``, or ``[rows, components, in]``: all components of a row, those of an irrep in ``ir_mul`` layout,
        say, take the same matrix. Any strides; views whose last dimension is contiguous (blocks of wider features) are read
        in place.
    :param weight: ``[types, out, in]``; either of the last two dimensions may be the contiguous one.
    :param types: ``[rows]``, int64, or their index.
    :param bias: ``[types, out]``.
    """
    types, order, ptr = _index(types)
    x, weight, bias = _cast(x, weight, bias)
    return _typed_linear(x, weight, types, bias, order, ptr)


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                   adapters: Union[torch.Tensor, RowGroups], *, scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    r"""A projection that all rows share plus the low-rank one of each row's adapter ``a``:
    ``x[i] @ weight.T + scale[a] * (x[i] @ down[a].T) @ up[a].T``. What lies between the two thin products is a float32 sum, kept as
    such in memory. Next to operands of 16 bits it enters the second product as two of them together, 16 bits of it with bfloat16 and 22
    with float16 (16 at least for an element down to 2^-24 of its row's largest). It is whole with float32, and in the form for few rows (up
    to 128, of weights that are contiguous along the sum), so that 16-bit results of 128 and of 129 rows can differ in the last bit.

    :param x: ``[rows, in]``.
    :param weight: ``[out, in]``.
    :param down, up: ``[adapters, rank, in]`` and ``[adapters, out, rank]``; adapters of smaller rank are filled up with zeros.
    :param adapters: ``[rows]``, int64, or their index. Rows without one (-1) get the shared projection.
    :param scale: ``[adapters]``, float32, without a gradient; 1 where left out.

    All of ``x``, ``weight``, ``down`` and ``up`` have gradients; those that are not asked for are not computed.
    """
    types, order, ptr = _index(adapters)
    x, weight, down, up = _cast(x, weight, down, up)
    return _adapter_linear(x, weight, down, up, types, scale, order, ptr)[0]
