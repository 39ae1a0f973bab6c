"""Rotary positions with one or several axes, on the device (nq_rotation, nq_rotate).

rope.py holds the tables of consecutive positions that compression undoes and applies again;
here the angles of a step's own tokens are made once and serve every layer: rotate for prompts and
training, FourBitPagePool.append for what goes into a cache.  With several axes (time, height and
width of images and video) each frequency turns with the position of its axis.

One axis rotates as forward_rope does (nexusquant/core/rope_utils.py:75-112).
"""

from __future__ import annotations

import ctypes
import dataclasses
import struct
import threading
from typing import Dict, Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import on_device
from .rope import _scaling_key, inv_freq

_HEAD_DIMS = (64, 128, 256)
_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


@dataclasses.dataclass(frozen=True)
class Rotation:
    """Cosines and sines of some rows' positions: fp32 [rows, 2, head_dim / 2] on the device.  Made on the current stream;
    work on other streams waits for it, and keeps it, as for any tensor."""
    angles: torch.Tensor
    rows: int
    head_dim: int

    @property
    def device(self) -> torch.device:
        return self.angles.device


_tables: Dict[tuple, tuple] = {}
_lock = threading.Lock()


def frequency_axes(head_dim: int, sections: Optional[Sequence[int]], interleaved: bool) -> np.ndarray:
    """uint8 [head_dim / 2]: the axis of each frequency.  sections[a] of them belong to axis a: one axis after another,
    or, interleaved, to the axes in turn (frequency i to axis i mod axes) until an axis after the first has its number;
    the first takes what is left."""
    half = head_dim // 2
    if sections is None:
        return np.zeros(half, dtype=np.uint8)
    sections = [int(n) for n in sections]
    axes = len(sections)
    if not 1 <= axes <= 255 or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"sections must be up to 255 numbers that add up to head_dim / 2 = {half}, got {sections}")
    if not interleaved:
        return np.repeat(np.arange(axes, dtype=np.uint8), sections)
    i = np.arange(half)
    axis = np.where(i < axes * np.asarray(sections)[i % axes], i % axes, 0).astype(np.uint8)
    if np.bincount(axis, minlength=axes).tolist() != sections:
        raise ValueError(f"interleaved sections after the first must fit the frequencies in turn, got {sections}")
    return axis


def _table(head_dim: int, base: float, rope_scaling, sections, interleaved: bool) -> tuple:
    """(axes, inverse frequencies, the axis of each) as host arrays that a call passes."""
    key = (head_dim, base, _scaling_key(rope_scaling), sections, interleaved)
    got = _tables.get(key)
    if got is None:
        axis = np.ascontiguousarray(frequency_axes(head_dim, sections, interleaved))
        freq = np.ascontiguousarray(inv_freq(head_dim, base, rope_scaling).numpy(), dtype=np.float32)
        with _lock:
            if len(_tables) >= 64:
                _tables.clear()
            got = _tables[key] = (1 if sections is None else len(sections), freq, axis, freq.ctypes.data, axis.ctypes.data)
    return got


def plan_rotation(positions, head_dim: int, base: float = 10000.0, rope_scaling: Optional[dict] = None,
                  sections: Optional[Sequence[int]] = None, interleaved: bool = False, device=None) -> Rotation:
    """The rotation of tokens at `positions`, for every layer and head of a step.

    positions: int32 or int64, [rows], or [axes, rows] with `sections` (frequency_axes says which frequency
    is of which axis); on the device, or on the host (copied; not in a graph's capture).  base, rope_scaling: as
    everywhere (rope.py).  The angle is the fp32 product of position and inverse frequency, as models form it;
    its cosine and sine are exact to fp32."""
    head_dim = int(head_dim)
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} unsupported (64, 128, 256)")
    if not torch.is_tensor(positions):
        positions = torch.as_tensor(np.asarray(positions))
        if positions.numel() == 0:
            positions = positions.long()
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if not positions.is_cuda:
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise _lib.NexusQuantError(f"nexusquant_amd runs on MI355X (ROCm) devices only; the rotation is for {dev}")
        if torch.cuda.is_initialized():
            with on_device(dev):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("positions on the host cannot be copied to the device in a graph: copy them before capturing")
        positions = positions.to(dev)
    elif device is not None and torch.device(device) != positions.device and torch.device(device) != torch.device("cuda"):
        raise ValueError(f"positions are on {positions.device}, not on {device}")
    sections = None if sections is None else tuple(int(n) for n in sections)
    table = _table(head_dim, float(base), rope_scaling, sections, bool(interleaved))  # (held until the call has read its arrays)
    axes, _, _, freq, axis_of = table
    if positions.dim() == 1 and axes == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[0] != axes:
        raise ValueError(f"positions must be [rows]{'' if axes == 1 else f' of each of {axes} axes, [{axes}, rows]'}, got "
                         f"{tuple(positions.shape)}")
    rows = positions.shape[1]
    if rows > 1 and positions.stride(1) != 1:
        positions = positions.contiguous()
    dev = positions.device
    angles = torch.empty(rows, 2, head_dim // 2, dtype=torch.float32, device=dev)
    with on_device(dev):
        st = _lib.load().nq_rotation(positions.data_ptr(), int(positions.dtype == torch.int64), axes, positions.stride(0), rows,
                                     head_dim // 2, freq, axis_of, angles.data_ptr(), _lib.current_stream_handle(dev))
    _lib.check(st, "nq_rotation")
    return Rotation(angles=angles, rows=rows, head_dim=head_dim)


def empty_as(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type (1.3 us; torch.empty given those takes 2.3)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def aligned(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous, 16-byte aligned vectors: itself when they are, any strides of rows and heads."""
    row, head, one = t.stride()
    if one == 1 and not (row * t.element_size() | head * t.element_size() | t.data_ptr()) & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    (n, m, d), (row, head, one), at = t.shape, t.stride(), t.data_ptr()
    return at, at + t.element_size() * (1 + (n - 1) * row + (m - 1) * head + (d - 1) * one)


def same_or_apart(out: torch.Tensor, x: torch.Tensor) -> bool:
    """Whether out [rows, heads, d] is x, element for element, or certainly shares no memory with it."""
    if out is x or out.numel() == 0 or x.numel() == 0:
        return True
    if out.data_ptr() == x.data_ptr() and out.shape == x.shape and out.stride() == x.stride():
        return True
    (a0, a1), (b0, b1) = _extent(out), _extent(x)
    if a1 <= b0 or b1 <= a0:
        return True
    # slices of the same rows: which part of a row each takes
    size, row = out.element_size(), out.stride(0)
    if row != x.stride(0) or x.element_size() != size or row <= 0:
        return False
    span = [size * (1 + sum((n - 1) * s for n, s in zip(t.shape[1:], t.stride()[1:]))) for t in (out, x)]
    between = (b0 - a0) % (size * row)
    return between >= span[0] and between + span[1] <= size * row


def vectors_apart(t: torch.Tensor) -> bool:
    """Whether heads lie within rows, one after another, or rows within heads, so that no two vectors share memory."""
    (n, m, d), (row, head, _) = t.shape, t.stride()
    return ((m <= 1 or head >= d) and (n <= 1 or row >= (m - 1) * head + d)
            or (n <= 1 or row >= d) and (m <= 1 or head >= (n - 1) * row + d))


def check_out(out: torch.Tensor, like: torch.Tensor, name: str, align: int = 16) -> None:
    if out is not like and (out.shape != like.shape or out.dtype != like.dtype or out.device != like.device):
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    size, (row, head, one) = out.element_size(), out.stride()
    if (one != 1 and out.shape[2] > 1) or (row * size | head * size | out.data_ptr()) % align \
            or not (out.is_contiguous() or vectors_apart(out)):
        raise ValueError(f"{name} must have {align}-byte aligned head vectors of their own")


def written(*tensors: Optional[torch.Tensor]) -> None:
    """Tell autograd that a launch wrote into these: a graph that has saved one raises, as it does after torch's own writes."""
    for t in tensors:
        if t is not None:
            torch.autograd.graph.increment_version(t)


# nq_rotate_desc, packed in one go and passed as bytes
_PACK = struct.Struct("6i5P8q")


def _launch(query, key, angles: torch.Tensor, inverse: bool, q_out, k_out) -> None:
    rows = q_at = qo_at = q_heads = k_at = ko_at = k_heads = 0
    q_strides = qo_strides = k_strides = ko_strides = (0, 0)
    if query is not None:
        q = aligned(query)
        (rows, q_heads, d), q_at, q_strides, qo_at, qo_strides = q.shape, q.data_ptr(), q.stride()[:2], q_out.data_ptr(), q_out.stride()[:2]
    if key is not None:
        k = aligned(key)
        (rows, k_heads, d), k_at, k_strides, ko_at, ko_strides = k.shape, k.data_ptr(), k.stride()[:2], k_out.data_ptr(), k_out.stride()[:2]
    like = q_out if query is not None else k_out
    dev = like.device
    with on_device(dev):
        st = _lib.load().nq_rotate(_PACK.pack(
            rows, q_heads, k_heads, d, _lib.dtype_code(like.dtype), int(inverse), q_at, k_at, qo_at, ko_at,
            angles.data_ptr(), *q_strides, *k_strides, *qo_strides, *ko_strides), _lib.current_stream_handle(dev))
    _lib.check(st, "nq_rotate")


def _rotated(query, key, angles: torch.Tensor, inverse: bool):
    q_out, k_out = (None if t is None else empty_as(t) for t in (query, key))
    _launch(query, key, angles, inverse, q_out, k_out)
    return q_out, k_out


def has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether forward mode differentiates one of these (outside of its levels 0.06 us; unpack_dual takes 0.4 a tensor)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Rotate(torch.autograd.Function):
    """The gradient of a rotation is the rotation by the opposite angle, its derivative along a tangent the tangent's rotation."""

    @staticmethod
    def forward(ctx, query, key, angles, inverse, tangents):
        ctx.save_for_backward(angles)
        ctx.save_for_forward(angles)
        ctx.inverse = inverse
        ctx.set_materialize_grads(False)
        out = _rotated(query, key, angles, inverse)
        # of an input that needs no gradient the output needs none, and backward does not turn one for it
        ctx.moves = [t is not None and any(x) for t, *x in zip((query, key), ctx.needs_input_grad, tangents)]
        ctx.mark_non_differentiable(*(y for y, moves in zip(out, ctx.moves) if y is not None and not moves))
        ctx.shapes = [None if t is None else t.shape for t in (query, key)]
        return out

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        if grad_query is None and grad_key is None:
            return (None,) * 5
        angles, = ctx.saved_tensors
        # (derivatives of the gradient are asked for, or not)
        again = _differentiable if torch.is_grad_enabled() or has_tangent(grad_query, grad_key) else _rotated
        return (*again(grad_query, grad_key, angles, not ctx.inverse), None, None, None)

    @staticmethod
    def jvp(ctx, query, key, *_):
        angles, = ctx.saved_tensors
        again = _differentiable if torch.is_grad_enabled() else _rotated
        like = query if query is not None else key
        return tuple(y if y is not None or not moves else like.new_zeros(shape)
                     for y, moves, shape in zip(again(query, key, angles, ctx.inverse), ctx.moves, ctx.shapes))


def _differentiable(query, key, angles: torch.Tensor, inverse: bool):
    return _Rotate.apply(query, key, angles, inverse, (has_tangent(query), has_tangent(key)))  # (forward sees no tangents)


def rotate(query: torch.Tensor, key: Optional[torch.Tensor], rotation: Rotation, inverse: bool = False,
           out: Optional[Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]] = None
           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """query [rows, q_heads, head_dim] and key [rows, kv_heads, head_dim] (or None) rotated: coordinate i with
    i + head_dim / 2.

    fp16, bf16 or fp32, computed in fp32 and rounded once; any strides of rows and heads: slices of one fused projection
    are read in place.  inverse: by the opposite angles.  out: where the results go; (query, key) rotates in place.
    Differentiable (without out), in reverse and in forward mode.  As with any operator, a backward pass is captured into a
    graph only while no eager graph of the same leaves lives."""
    dtype, dev, grad = query.dtype, rotation.device, False
    for name, t in (("query", query), ("key", key)):
        if t is None and name == "key":
            continue
        if t.device != dev:
            _lib.require_device(t, name)
            raise ValueError(f"{name} is on {t.device}, the rotation on {dev}")
        shape = t.shape
        if len(shape) != 3 or shape[0] != rotation.rows or shape[2] != rotation.head_dim:
            raise ValueError(f"{name} must be [{rotation.rows} rows, heads, {rotation.head_dim}], got {tuple(shape)}")
        if t.dtype != dtype or dtype not in _DTYPES:
            raise ValueError(f"query and key must share an fp16, bf16 or fp32 dtype, got {t.dtype}")
        grad = grad or t.requires_grad
    if rotation.rows >= 1 << 31:
        raise ValueError(f"{rotation.rows} rows: a call takes less than 2^31")
    grad = grad and torch.is_grad_enabled() or has_tangent(query, key)
    if out is None:
        if grad:
            return _differentiable(query, key, rotation.angles, bool(inverse))
        q_out = empty_as(query)
        k_out = None if key is None else empty_as(key)
    else:
        q_out, k_out = out
        if grad or has_tangent(q_out, k_out) or any(t is not None and t.requires_grad and torch.is_grad_enabled() for t in (q_out, k_out)):
            raise NotImplementedError("rotate into given tensors has no backward pass; call it under torch.no_grad()")
        if q_out is None or (k_out is None) != (key is None):
            raise ValueError("out must be a pair of tensors for query and key")
        check_out(q_out, query, "out of query")
        if key is not None:
            check_out(k_out, key, "out of key")
        given = [(q_out, query), (q_out, key), (k_out, key), (k_out, query), (q_out, k_out)]
        if any(a is not None and b is not None and not same_or_apart(a, b) for a, b in given) or \
                (k_out is not None and q_out.numel() and q_out.data_ptr() == k_out.data_ptr()) or \
                (key is not None and query.numel() and (q_out.data_ptr() == key.data_ptr() or k_out.data_ptr() == query.data_ptr())):
            raise ValueError("out may be query and key themselves, and must not overlap them or each other otherwise")
    _launch(query, key, rotation.angles, bool(inverse), q_out, k_out)
    if out is not None:
        written(q_out, k_out)
    return q_out, k_out
