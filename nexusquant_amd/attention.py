"""Causal attention over packed prompts (nq_prompt_attention): the prefill's attention of a
serving batch, before its keys and values are compressed into pages.

scoring.attention_real is the padded form with transformers' eager roundings (and the column
sums of the scorer); here the softmax stays in fp32 and sequences of different lengths stand
one after another without padding.
"""

from __future__ import annotations

import dataclasses
import struct
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .ops import PlanTensor, on_device

_HEAD_DIMS = (64, 128, 256)


@dataclasses.dataclass(frozen=True)
class PromptPlan:
    """Which rows are whose: made once for a batch's lengths, used by every layer."""
    lengths: tuple
    rows: int                     # of all sequences
    n_tiles: int
    tiles: Optional[PlanTensor]   # int32 [n_tiles, 4] on the device


def prompt_tiles(lengths: Sequence[int], tile_rows: int) -> np.ndarray:
    """int32 [n_tiles, 4]: first row, length and first query of each tile, the ones that see most keys first."""
    n = np.asarray(lengths, dtype=np.int64).reshape(-1)
    count = -(-n // tile_rows)
    seq = np.repeat(np.arange(len(n)), count)
    q0 = (np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)) * tile_rows
    tiles = np.stack([(np.cumsum(n) - n)[seq], n[seq], q0, np.zeros_like(q0)], axis=1)
    return tiles[np.argsort(-q0, kind="stable")].astype(np.int32)


def plan_prompts(lengths: Sequence[int], device=None) -> PromptPlan:
    """The plan of sequences of `lengths` tokens (0 is allowed), one after another in this order.
    Made before a graph is captured, not in the capture."""
    lens = tuple(int(x) for x in (lengths.tolist() if torch.is_tensor(lengths) else lengths))
    if any(x < 0 for x in lens):
        raise ValueError(f"lengths must not be negative, got {min(lens)}")
    rows = sum(lens)
    if rows >= 1 << 31:
        raise ValueError(f"{rows} rows: a batch takes less than 2^31")
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise _lib.NexusQuantError(f"nexusquant_amd runs on MI355X (ROCm) devices only; the plan is for {dev}")
    tiles = prompt_tiles(lens, int(_lib.load().nq_prompt_tile_rows()))
    return PromptPlan(lengths=lens, rows=rows, n_tiles=len(tiles),
                      tiles=PlanTensor(tiles.reshape(-1), dev) if len(tiles) else None)


def _rows(t: torch.Tensor):
    """t with contiguous, 16-byte aligned head vectors (itself when they are), its address and strides."""
    row, head, one = t.stride()
    at = t.data_ptr()
    if one != 1 or (row | head) & 7 or row >= 1 << 24 or at & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        row, head, one = t.stride()
        at = t.data_ptr()
    return t, at, row, head


def _apart(t: torch.Tensor) -> bool:
    """Whether no two head vectors of t share memory."""
    (n, m, d), (row, head, _) = t.shape, t.stride()
    if n <= 1 or m <= 1:
        return (n <= 1 or row >= d) and (m <= 1 or head >= d)
    if row < d or head < d:
        return False
    if row >= (m - 1) * head + d or head >= (n - 1) * row + d:  # heads within rows, or rows within heads
        return True
    # interleaved: the rows nearest to each head's distance, from below and from above
    return not any((i < n and j * head - i * row < d) or (i + 1 < n and (i + 1) * row - j * head < d)
                   for j in range(1, m) for i in (j * head // row,))


# nq_prompt_desc, packed in one go and passed as bytes (a call's host time counts for short prompts)
_PACK = struct.Struct("6i5P8qfiPq")


# Few tiles and heads: several workgroups share a tile's keys, as many as run at once (two on a CU, at head_dim 256 one),
# with _SPLIT_STAGES stages of 64 keys each at least.  us without and with, one prompt: 2188 tokens of 4 heads x 256 95
# and 49, x 128 45 and 28, 8192 of one head 148 and 42, 4096 of 8 80 and 65, 2048 of 8 x 64 32 and 23, 700 13.5 and 13.8.
_SPLIT_TO = {64: 512, 128: 512, 256: 256}
_SPLIT_STAGES = 3
_STAGE = 64


def _splits(workgroups: int, keys: int, head_dim: int) -> int:
    """Workgroups that share a tile's keys when the launch has `workgroups` without and tiles see up to `keys` keys."""
    return max(1, min(_SPLIT_TO[head_dim] // workgroups, -(-keys // _STAGE) // _SPLIT_STAGES, 64))


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, plan: PromptPlan,
                     scale: Optional[float] = None, sliding_window: Optional[int] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each packed sequence over itself.

    query [rows, q_heads, head_dim], key and value [rows, kv_heads, head_dim] (fp16 or bf16, q_heads a
    multiple of kv_heads, head_dim 64, 128 or 256), any strides of rows and heads: slices of one fused
    projection are read in place.  scale: 1 / sqrt(head_dim) by default.  sliding_window: query i sees
    keys i - window < j <= i.
    Returns [rows, q_heads, head_dim].  Rows behind the plan's sequences are left as they are in `out`,
    and are zero without one; `out` may be `query`, and must not overlap key or value.  Inference only:
    tensors that require a gradient are refused."""
    lib = _lib.load()
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not t.is_cuda:
            _lib.require_device(t, name)
    shape, kv, dtype, dev = query.shape, key.shape, query.dtype, query.device
    if len(shape) != 3 or len(kv) != 3:
        raise ValueError(f"query and key must be [rows, heads, head_dim], got {tuple(shape)} and {tuple(kv)}")
    rows, hq, d = shape
    hkv = kv[1]
    if kv[0] != rows or kv[2] != d or value.shape != kv:
        raise ValueError(f"incompatible query {tuple(shape)}, key {tuple(kv)} and value {tuple(value.shape)}")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"{hq} query heads are no multiple of {hkv} kv heads")
    if dtype not in (torch.float16, torch.bfloat16) or key.dtype != dtype or value.dtype != dtype:
        raise ValueError("query, key and value must share an fp16 or bf16 dtype")
    if key.device != dev or value.device != dev:
        raise ValueError("query, key and value must be on one device")
    if d not in _HEAD_DIMS:
        raise ValueError(f"head_dim {d} unsupported (64, 128, 256)")
    if rows < plan.rows:
        raise ValueError(f"the plan's sequences have {plan.rows} rows, the tensors {rows}")
    if plan.tiles is not None and plan.tiles.device != dev:
        raise ValueError(f"the plan is on {plan.tiles.device}, the tensors on {dev}")
    if sliding_window is not None and int(sliding_window) <= 0:
        raise ValueError(f"sliding_window must be positive, got {sliding_window}")
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        raise NotImplementedError("prompt_attention has no backward pass; call it under torch.no_grad()")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"scale must be positive, got {scale}")
    if out is None:
        out = query.new_empty(shape)
        if rows > plan.rows:
            out[plan.rows:].zero_()
    elif (out.shape != shape or out.dtype != dtype or out.device != dev
          or out.stride(2) != 1 or out.stride(0) % 4 or out.stride(1) % 4 or out.data_ptr() % 8 or not _apart(out)):
        raise ValueError(f"out must be {tuple(shape)} {dtype} on {dev} with 8-byte aligned head vectors of their own")
    if plan.n_tiles == 0:
        return out
    q, q_at, q_row, q_head = _rows(query)
    k, k_at, k_row, k_head = _rows(key)
    v, v_at, v_row, v_head = _rows(value)
    o_row, o_head, _ = out.stride()
    window = 0 if sliding_window is None or int(sliding_window) >= max(plan.lengths) else int(sliding_window)
    split, ws, nbytes = 1, None, 0
    if plan.n_tiles * hq <= _SPLIT_TO[d] // 2:
        longest = max(plan.lengths)
        split = _splits(plan.n_tiles * hq, min(longest, window + 128) if window else longest, d)
        if split > 1:
            nbytes = lib.nq_prompt_workspace(plan.n_tiles, hq, d, split)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)  # of this call alone
    with on_device(dev):
        st = lib.nq_prompt_attention(_PACK.pack(
            hq, hkv, d, _lib.NQ_F16 if dtype == torch.float16 else _lib.NQ_BF16, plan.n_tiles, window, q_at, k_at, v_at,
            out.data_ptr(), plan.tiles.address(), q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, scale, split,
            0 if ws is None else ws.data_ptr(), nbytes),
            _lib.current_stream_handle(dev))
    _lib.check(st, "nq_prompt_attention")
    return out
