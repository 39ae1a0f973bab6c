"""A cache held in 4 bits: a pool of pages, what writes it, and the attentions that read it.

CompressedPagePool (page_pool.py) keeps keys without rotation, 8 bits a coordinate; its
attention turns every key it reads.  Here keys are stored rotated and both keys and values
as their Walsh-Hadamard transform in 16 levels with one fp16 scale a token and head: half the
bytes (66 of 130 at head_dim 128), and an attention that undoes nothing a token.  What that
gives up is re-rotation: compact keeps positions.

    pool = FourBitPagePool(num_pages, num_heads=8, page_tokens=16, head_dim=128, num_layers=32)
    rotation = plan_rotation(positions, 128, base=500000.0)      # once a step, for all layers
    slots = pool.plan_slots(new_slots)
    step = pool.plan_attention(tables, lengths)                  # lengths with the new tokens
    q = pool.append(slots, key, value, rotation=rotation, query=query, layer=layer)
    y = pool.attend(step, q, layer=layer)
"""

from __future__ import annotations

import heapq
import struct
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .hadamard import hadamard_constant
from .ops import PlanTensor, on_device
from .page_pool import PagePool
from .rotary import Rotation, aligned, check_out, empty_as, has_tangent, same_or_apart, written

_HEAD_DIMS = (64, 128, 256)
_DTYPES = (torch.float16, torch.bfloat16)


class SlotPlan:
    """Which slots some rows of tokens are stored in: made once a step, used by every layer."""

    def __init__(self, pool: "FourBitPagePool", slots: np.ndarray):
        self.pool = pool
        self.rows = len(slots)
        self.pages = np.unique(slots[slots >= 0] // pool.page_tokens)
        self.slots = PlanTensor(slots.astype(np.int32), pool.device) if len(slots) else None
        self.writable_at = -1  # the pool's references when its pages were found to be the sequence's own


class FourBitAttentionPlan:
    """Which tokens of a pool each query sees: valid for every layer while tables and lengths stay the same.
    The device arrays are made for a number of query heads, the first time that it is used (before a graph is captured)."""

    def __init__(self, pool: "FourBitPagePool", tables: List[np.ndarray], lengths: Sequence[int], queries: Sequence[int],
                 causal: bool, window: int):
        self.pool = pool
        self.lengths, self.queries = tuple(lengths), tuple(queries)
        self.causal, self.window = causal, window
        self.rows = sum(queries)
        self._tables = tables
        self._work: Dict[int, tuple] = {}

    def work(self, q_heads: int) -> tuple:
        """(device ints, their places in bytes, (items by kind, joins, slots, most chunks), workspace bytes) for q_heads
        query heads."""
        got = self._work.get(q_heads)
        if got is None:
            pool = self.pool
            with on_device(pool.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("attend: run the plan once before capturing it into a graph")
            if q_heads == 0 or q_heads % pool.num_heads:
                raise ValueError(f"num_heads {q_heads} is not a multiple of the pool's {pool.num_heads}")
            lib = _lib.load()
            parts, counts = attention_items([len(t) for t in self._tables], self.lengths, self.queries, self.causal, self.window,
                                            q_heads // pool.num_heads, pool.num_heads, pool.head_dim,
                                            [int(lib.nq_fourbit_rows(pool.head_dim, k)) for k in range(3)])
            parts = [parts[0], np.concatenate(self._tables) if self._tables else np.zeros(0, np.int32), parts[1]]
            places, at = [], 0
            for v in parts:
                places.append(at)
                at += 4 * len(v)
            ints = PlanTensor(np.concatenate(parts).astype(np.int32), pool.device) if at else None
            got = self._work[q_heads] = (ints, places, counts, int(lib.nq_fourbit_workspace(counts[4], q_heads, pool.head_dim)))
        return got


# Tiles of a sequence's rows (query tokens x query heads of a kv head) by kind: many, some, few.
_MANY, _SOME, _FEW = 0, 1, 2
# Where no sequence has this many rows tiles are of some: 24 sequences of up to 223 rows over 1500 tokens of 20 x 64 57 us, with
# tiles of many 78 (they leave half of the CUs idle); 2048 x 4 rows over 32768 of 8 x 128 1340 and 1204 (what is decoded
# serves twice the rows).
_MANY_ROWS = 512
# Up to so many rows of a sequence are tiles of few, 16 rows each: weights keep 22 bits there, where wider tiles round them to 11.
# Fewer rows also take less time so than as one tile of 128 rows with the rest left idle, more of them at head_dim 64 and 128 do
# not.  us as few and as some, with no other kind in the plan: 16 sequences of 4096 tokens of 8 x 128, 20 rows 32 and 44, 32 31
# and 45, 64 51 and 49, 96 64 and 62, 128 81 and 68; one of 32768, 20 rows 20 and 29, 96 42 and 41, 128 48 and 44; 64 of 8192 of
# 8 x 64, 32 rows 126 and 181, 64 238 and 184, 96 346 and 248; 24 of 1500 of 20 x 64, 20 rows 26 and 40, 48 39 and 42, 96 70 and
# 56; 8 of 8192 of 8 x 256, 64 rows 81 and 105, 96 126 and 133, 128 134 and 138.
_FEW_ROWS = 96
_FEW_STEP = 128  # tokens that a workgroup takes at a time
_ITEM_INTS = 12
_STAGE, _LEAST = 64, 256  # of wider tiles, and the least of a chunk
_AT_ONCE = ({64: 256, 128: 256, 256: 256}, {64: 512, 128: 512, 256: 256})  # workgroups of many and of some rows
_STAGE_US = {64: 1.8, 128: 2.3, 256: 3.7}
_START_STAGES = 3  # what a workgroup's start and end cost


def _even(spans: np.ndarray, most: int, step: int):
    """(chunks, tokens of a chunk) of each span: as few chunks of at most `most` tokens as it takes, all alike but for a
    multiple of `step`."""
    chunks = -(-spans // most)
    each = -(-spans // (chunks * step)) * step
    return -(-spans // each), each


def _few_chunks(spans: np.ndarray, heads: int, head_dim: int):
    """Chunks of few rows, of the least length with which the launch is so many workgroups.

    1024 run at once (at head_dim 256 512); with fewer there is less to join, or nothing, where a chunk has all of a sequence.
    us with 512, 1024 and 2048: 64 rows up to 8192 tokens of 8 x 128 84, 62, 63; 16 rows up to 30000 62, 61, 61; one row of
    131072 34, 35, 36; 24 rows up to 1500 of 20 x 64 12.8, 14.8, 17.2; 32 rows up to 8192 of 4 x 256 33, 37, 40.  Around the
    work from which on 1024 are taken: 8 rows up to 8192 of 8 x 128 (0.6 of it) 18.3, 18.7, 20.0; 32 up to 8192 of 8 x 64 (1.02)
    28.1, 25.1, 27.3; 16 up to 8192 of 8 x 128 (1.1) 23.0, 24.2, 24.7."""
    work = heads * int(spans.sum()) * head_dim // 128
    workgroups = 1024 if work >= 1024 * 512 and head_dim < 256 else 512
    lo, hi = 1, -(-int(spans.max()) // _FEW_STEP)
    while lo < hi:
        mid = (lo + hi) // 2
        if heads * int((-(-spans // (mid * _FEW_STEP))).sum()) > workgroups:
            lo = mid + 1
        else:
            hi = mid
    return _even(spans, lo * _FEW_STEP, _FEW_STEP)


def _last_end(stages: np.ndarray, places: int) -> float:
    """When the last of these ends, each begun in turn on the place that is free first."""
    if len(stages) <= places:
        return float(stages.max())
    if len(stages) > 16 * places:
        return float(stages.sum()) / places + float(stages[-1])
    ends = stages[:places].tolist()
    heapq.heapify(ends)
    for n in stages[places:].tolist():
        heapq.heapreplace(ends, ends[0] + n)
    return max(ends)


def _wide_chunks(spans: np.ndarray, rows: np.ndarray, heads: int, head_dim: int, at_once: int):
    """Chunks of many or some rows: (chunks, tokens of a chunk) of each span, by what the launch and the sums that are joined
    would take, the longest chunks begun first.

    Either all chunks of a span are alike, or a span is cut at a length that is the CUs' share or somewhat more, and its rest
    fills a place where a short span has ended.  us, alike and cut so: 4 sequences of 512 query tokens or fewer over up to
    16384 of 8 x 128, 313 and 278; 6 of 256 over up to 20000, 310 and 264; 5 of 300 over up to 12000 of 4 x 256, 351 and 342.
    (Expected: 323 and 275, with 5 us and 3.5 TB/s for the join.  A twentieth on top keeps whole what would
    gain as little: 2048 query tokens of 32768 of 8 x 64 take 851 whole, 904 cut.)"""
    places = max(1, at_once // heads)  # (a kv head's chunks run beside the other heads')
    share = float(spans.sum()) / places
    longest = int(spans.max())
    lengths = {(False, -(-longest // (cut * _STAGE))) for cut in (1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 128)}
    lengths |= {(True, -(-int(share * f) // _STAGE)) for f in (0.52, 0.56, 0.62, 1.0, 1.04, 1.08, 1.12, 1.2)}
    tries = []
    for cut_off, stages in lengths:
        length = max(_LEAST, stages * _STAGE)
        if cut_off:
            chunks, each = -(-spans // length), np.minimum(spans, length)
        else:
            chunks, each = _even(spans, length, _STAGE)
        n = int(chunks.sum())
        split = chunks > 1
        most = float(each.max()) / _STAGE + _START_STAGES
        total = float(spans.sum()) / _STAGE + n * _START_STAGES
        join = 0.0
        if split.any():
            join = 0.05 * _STAGE_US[head_dim] * total / places + 5.0 + heads * head_dim * 8.0 * float((rows * chunks)[split].sum()) / 3.5e6
        tries.append((_STAGE_US[head_dim] * max(most, total / places) + join, n, join, chunks, each))
    tries.sort(key=lambda x: x[:2])
    best = float("inf")
    for least, n, join, chunks, each in tries:
        if least >= best:
            break
        stages = np.repeat(each, chunks)
        stages[np.cumsum(chunks) - 1] = spans - (chunks - 1) * each
        us = _STAGE_US[head_dim] * _last_end(-np.sort(-stages) / _STAGE + _START_STAGES, places) + join
        if us < best:
            best, found = us, (chunks, each)
    return found


def attention_items(pages: Sequence[int], lengths: Sequence[int], queries: Sequence[int], causal: bool, window: int, group: int,
                    heads: int, head_dim: int, rows: Sequence[int]):
    """The work list of nq_fourbit_attention, (items, joins) as flat int32 arrays, and the counts of items by
    kind, joins, slots and the most chunks of a tile.

    pages[b], lengths[b], queries[b]: a sequence's pages in the list, tokens and query tokens.  rows: most rows of a
    tile by kind (many, some, few)."""
    tiles = []  # kind, sequence, first query token, one past the last, first row, rows, first token, one past the last
    joins = []
    first_row = first_page = 0
    starts, firsts = [], []
    wide = rows[_MANY if max(queries, default=0) * group >= _MANY_ROWS else _SOME]  # one kind beside few: launches follow each other
    for b, (n, q) in enumerate(zip(lengths, queries)):
        firsts.append(first_row)
        starts.append(first_page)
        if n == 0:
            joins += [(first_row + i, 0, 0, 0) for i in range(q)]
        first_row += q
        first_page += pages[b]
        if n == 0 or q == 0:
            continue
        most = rows[_FEW] if q * group <= _FEW_ROWS else wide
        per = max(1, most // group)  # query tokens of a tile
        for i0 in range(0, q, per):
            i1 = min(i0 + per, q)
            end = n - q + i1 if causal else n
            start = max(0, n - q + i0 - window + 1) if window else 0
            kind = _FEW if most == rows[_FEW] or (i1 - i0) * group <= rows[_FEW] else _MANY if wide > rows[_SOME] else _SOME
            for r0 in range(i0 * group, i1 * group, most):  # (more heads than a tile has rows: several, cut alike)
                tiles.append((kind, b, i0, i1, r0, min(most, i1 * group - r0), start, end))
    if not tiles:
        return (np.zeros(0, np.int32), np.array(joins, np.int32).reshape(-1)), (0, 0, 0, len(joins), 0, 0)
    t = np.array(tiles, dtype=np.int64)
    t = t[np.lexsort((t[:, 6] - t[:, 7], t[:, 0]))]  # by kind, long ones before short ones
    kind, span = t[:, 0], t[:, 7] - t[:, 6]
    chunks, each = np.empty(len(t), np.int64), np.empty(len(t), np.int64)
    for k in range(3):
        of = kind == k
        if of.any():
            chunks[of], each[of] = _few_chunks(span[of], heads, head_dim) if k == _FEW else \
                _wide_chunks(span[of], t[of, 5], heads, head_dim, _AT_ONCE[k][head_dim])
    _, b, i0, i1, r0, n_rows, start, end = t.T
    news = np.asarray(queries, dtype=np.int64)[b]
    last = np.asarray(lengths, dtype=np.int64)[b] - (news if causal else 1)
    starts, firsts = np.asarray(starts, dtype=np.int64)[b], np.asarray(firsts, dtype=np.int64)[b]
    # partial sums: slots for the query tokens of a tile that is split, the same ones for further tiles of their heads (which
    # follow it); a tile that is not goes to the output
    split = chunks > 1
    own = split & (r0 == i0 * group)
    need = np.where(own, (i1 - i0) * chunks, 0)
    slots = int(need.sum())
    if slots >= 1 << 31:
        raise ValueError("too many partial sums: split the queries over several plans")
    at = np.cumsum(need) - need
    at = at[np.maximum.accumulate(np.where(own | ~split, np.arange(len(t)), 0))]
    of = np.repeat(np.arange(len(t)), chunks)  # an item's tile
    j = np.arange(len(of)) - (np.cumsum(chunks) - chunks)[of]
    first = start[of] + j * each[of]
    items = np.zeros((len(of), _ITEM_INTS), dtype=np.int32)
    items[:, 0], items[:, 1], items[:, 2] = starts[of], first, np.minimum(each[of], end[of] - first)
    items[:, 3], items[:, 4], items[:, 5] = firsts[of], r0[of], n_rows[of]
    items[:, 6], items[:, 7] = np.where(split, at - i0 * chunks, 0)[of] + np.where(split[of], j, 0), np.where(split, chunks, 0)[of]
    items[:, 8] = last[of]
    tokens = np.where(own, i1 - i0, 0)
    of = np.repeat(np.arange(len(t)), tokens)  # a joined query token's tile
    i = np.arange(len(of)) - (np.cumsum(tokens) - tokens)[of]
    joined = np.zeros((len(joins) + len(of), 4), dtype=np.int32)
    joined[:len(joins)] = np.array(joins, dtype=np.int32).reshape(-1, 4)
    joined[len(joins):, 0], joined[len(joins):, 1], joined[len(joins):, 2] = (firsts + i0)[of] + i, at[of] + i * chunks[of], chunks[of]
    n_items = [int(chunks[kind == k].sum()) for k in range(3)]
    # the longest of a kind first (64 rows up to 8192 tokens 77 to 72 us)
    items = items[np.lexsort((-items[:, 2], np.repeat(np.arange(3), n_items)))]
    return (items.reshape(-1), joined.reshape(-1)), (*n_items, len(joined), slots, int(chunks.max()))


# nq_fourbit_append_desc and nq_fourbit_desc, packed in one go and passed as bytes
_APPEND_PACK = struct.Struct("P4i6P8qfi")
_ATTEND_PACK = struct.Struct("P10i2fi5P4qPq")


class FourBitPagePool(PagePool):
    """num_pages pages of page_tokens tokens for num_heads kv heads, in num_layers layers, 4 bits a coordinate.

    key_codes, value_codes    uint8 [layers, pages, heads, tokens, head_dim / 2], coordinate 2 i the low nibble of byte i
    key_scales, value_scales  fp16 [layers, pages, heads, tokens]

    A vector x is held as t = H x (H the orthonormal Walsh-Hadamard matrix): scale = fp16(max |t| / 7.5), nibble
    n = clamp(floor(t / scale + 8.5), 0, 15), which stands for H ((n - 8) scale): half a scale off at most.  A vector with
    an infinity or a NaN, or with sums past fp32, has a NaN scale; queries that see it get NaN.

    Page numbers, fork, copy_pages, free: as CompressedPagePool.  compact keeps positions (keys are stored rotated)."""

    def __init__(self, num_pages: int, num_heads: int, page_tokens: int, head_dim: int, num_layers: int = 1, device=None):
        shape = (int(num_layers), int(num_pages), int(num_heads), int(page_tokens))
        if min(shape) < 1:
            raise ValueError(f"layers, pages, heads and tokens must be positive (got {shape})")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise _lib.NexusQuantError(f"nexusquant_amd runs on MI355X (ROCm) devices only; the pool is on {dev}")
        self._check_shape(shape, int(head_dim))
        codes = shape + (int(head_dim) // 2,)
        self._adopt(*(torch.zeros(codes, dtype=torch.uint8, device=dev) for _ in range(2)),
                    *(torch.zeros(shape, dtype=torch.float16, device=dev) for _ in range(2)))

    @classmethod
    def from_tensors(cls, key_codes: torch.Tensor, value_codes: torch.Tensor, key_scales: torch.Tensor,
                     value_scales: torch.Tensor) -> "FourBitPagePool":
        """A pool over fields that exist already (used, not copied); all its pages are free."""
        for name, t, dt, dims in (("key_codes", key_codes, torch.uint8, 5), ("value_codes", value_codes, torch.uint8, 5),
                                  ("key_scales", key_scales, torch.float16, 4),
                                  ("value_scales", value_scales, torch.float16, 4)):
            if t.dtype != dt:
                raise TypeError(f"{name} must be {dt}, got {t.dtype}")
            if t.dim() != dims or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be a contiguous, 16-byte aligned {dims}-d tensor, got {tuple(t.shape)}")
            _lib.require_device(t, name)
            if t.device != key_codes.device:
                raise ValueError(f"{name} is on {t.device}, key_codes on {key_codes.device}")
        shape = tuple(key_codes.shape[:4])
        if min(shape) < 1:
            raise ValueError(f"layers, pages, heads and tokens must be positive (got {shape})")
        if value_codes.shape != key_codes.shape or tuple(key_scales.shape) != shape or tuple(value_scales.shape) != shape:
            raise ValueError("fields must be [layers, pages, heads, tokens(, head_dim / 2)] of one shape")
        cls._check_shape(shape, 2 * key_codes.shape[4])
        pool = cls.__new__(cls)
        pool._adopt(key_codes, value_codes, key_scales, value_scales)
        return pool

    @staticmethod
    def _check_shape(shape, head_dim: int) -> None:
        layers, pages, heads, tokens = shape
        if head_dim not in _HEAD_DIMS:
            raise NotImplementedError(f"head_dim {head_dim}: the gfx950 4-bit kernels take 64, 128 or 256")
        if layers > 65535 or heads * tokens * head_dim >= 1 << 31 or pages * heads * tokens >= 1 << 31:
            raise ValueError("a pool takes 65535 layers, pages of less than 2^31 coordinates and less than 2^31 "
                             f"token rows a layer (got {shape})")

    def _adopt(self, key_codes, value_codes, key_scales, value_scales) -> None:
        self.key_codes, self.value_codes = key_codes, value_codes
        self.key_scales, self.value_scales = key_scales, value_scales
        self.head_dim = 2 * key_codes.shape[4]
        self._start(key_codes, value_codes, key_scales, value_scales, None, bits=4)

    def compact(self, tables: Sequence[Sequence[int]], lengths: Sequence[int], kept_idx: torch.Tensor, n_kept,
                renumber: bool = False) -> Tuple[List[List[int]], List[int]]:
        """As CompressedPagePool.compact; tokens keep their positions."""
        if renumber:
            raise ValueError("a pool in 4 bits stores keys rotated: renumber=True cannot rotate them again")
        return super().compact(tables, lengths, kept_idx, n_kept)

    # ------------------------------------------------------------------- tokens

    def plan_slots(self, slots: Sequence[int]) -> SlotPlan:
        """A plan of token i in slots[i] (page * page_tokens + offset, as `slots` gives them; -1: nowhere, a padded
        batch).  Slots are distinct and in allocated pages.  Made before a graph is captured, not in the capture."""
        s = np.asarray(slots.tolist() if torch.is_tensor(slots) else slots).reshape(-1)
        if len(s) and s.dtype.kind not in "iu":
            raise ValueError(f"slots must be integers, got {s.dtype}")
        if len(s) and s.max() >= self.num_pages * self.page_tokens:  # (as the type they came in)
            raise ValueError(f"slots must lie below {self.num_pages * self.page_tokens}")
        s = np.maximum(s.astype(np.int64, copy=False), -1)
        used = s[s >= 0]
        if len(np.unique(used)) != len(used):
            raise ValueError("plan_slots: slots must be distinct")
        with self._lock:
            self.in_use(np.unique(used // self.page_tokens), "plan_slots")
        return SlotPlan(self, s)

    def _check_plan(self, plan, kind, what: str, layer: int) -> None:
        if not isinstance(plan, kind) or plan.pool is not self:
            raise ValueError(f"{what}: the plan is not one of this pool")
        if not 0 <= int(layer) < self.num_layers:
            raise ValueError(f"layer {layer} of a pool of {self.num_layers}")

    def append(self, plan: SlotPlan, key: torch.Tensor, value: torch.Tensor, rotation: Optional[Rotation] = None,
               query: Optional[torch.Tensor] = None, layer: int = 0, out: Optional[torch.Tensor] = None
               ) -> Optional[torch.Tensor]:
        """Rotate, encode and store tokens in one layer: key, value [rows, heads, head_dim] (fp16 or bf16, any strides of
        rows and heads) into the plan's slots, keys rotated by `rotation` (None: as they are, an encoder's states).
        query [rows, q_heads, head_dim] is rotated along and returned, into `out` where that is given (it may be query).
        The pages must have one reference.  One launch, without host work on the tokens: it can be captured into a graph;
        replays then store into the same slots."""
        self._check_plan(plan, SlotPlan, "append", layer)
        dtype, dev, rows, d = key.dtype, self.device, plan.rows, self.head_dim
        grad = torch.is_grad_enabled()
        for name, t in (("key", key), ("value", value), ("query", query)):
            if t is None and name == "query":
                continue
            if t.device != dev:
                _lib.require_device(t, name)
                raise ValueError(f"{name} is on {t.device}, the pool on {dev}")
            shape = t.shape
            if len(shape) != 3 or shape[0] != rows or shape[2] != d or (shape[1] != self.num_heads and name != "query"):
                heads = "q_heads" if name == "query" else self.num_heads
                raise ValueError(f"{name} must be ({rows} tokens, {heads}, {d}), got {tuple(shape)}")
            if t.dtype != dtype or dtype not in _DTYPES:
                raise ValueError(f"key, value and query must share an fp16 or bf16 dtype, got {t.dtype}")
            if grad and t.requires_grad:
                raise NotImplementedError("append has no backward pass; call it under torch.no_grad()")
        if out is not None and grad and out.requires_grad:
            raise NotImplementedError("append into a tensor that requires grad has no backward pass; call it under torch.no_grad()")
        if has_tangent(key, value, query, out):
            raise NotImplementedError("append has no derivative in forward mode; call it on tensors without tangents")
        if rotation is None:
            if query is not None:
                raise ValueError("append: a query is rotated along with the keys; without a rotation it is not taken")
        elif rotation.rows != rows or rotation.head_dim != d or rotation.device != dev:
            raise ValueError(f"append: a rotation of {rotation.rows} rows of {rotation.head_dim} on {rotation.device} for {rows} of "
                             f"{d} on {dev}")
        if out is not None:
            if query is None:
                raise ValueError("append: out is the query's")
            check_out(out, query, "out")
            if not same_or_apart(out, query) or not all(same_or_apart(out, t) and out.data_ptr() != t.data_ptr()
                                                        for t in (key, value) if t.numel()):
                raise ValueError("append: out may be query itself, and must not overlap query, key or value otherwise")
        with self._lock:
            if plan.writable_at != self._changes:
                if len(plan.pages):
                    refs = self._referenced(plan.pages, "append")
                    if refs.max() > 1:
                        raise ValueError(f"append: page {int(plan.pages[refs > 1][0])} is shared and cannot be written")
                plan.writable_at = self._changes
            given = out
            if query is not None and out is None:
                out = empty_as(query)
            if rows == 0:
                return out
            k, v = aligned(key), aligned(value)
            q = None if query is None else aligned(query)
            none = (0, 0)
            with on_device(dev):
                st = _lib.load().nq_fourbit_append(_APPEND_PACK.pack(
                    self.desc_at, int(layer), rows, 0 if q is None else q.shape[1], _lib.dtype_code(dtype),
                    0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if q is None else out.data_ptr(),
                    0 if rotation is None else rotation.angles.data_ptr(), plan.slots.address(),
                    *(none if q is None else q.stride()[:2]), *k.stride()[:2], *v.stride()[:2],
                    *(none if q is None else out.stride()[:2]), hadamard_constant(d), 0), _lib.current_stream_handle(dev))
            _lib.check(st, "nq_fourbit_append")
            written(given)
        return out

    def read(self, plan: SlotPlan, layer: int = 0, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """(keys, values) [rows, heads, head_dim] that the plan's slots stand for, keys rotated as they were stored; fp16,
        bf16 or fp32.  Rows of slot -1 are zero."""
        self._check_plan(plan, SlotPlan, "read", layer)
        code = _lib.dtype_code(dtype)
        keys = torch.empty(plan.rows, self.num_heads, self.head_dim, dtype=dtype, device=self.device)
        values = empty_as(keys)
        if plan.rows:
            with on_device(self.device):
                st = _lib.load().nq_fourbit_read(self.desc, int(layer), plan.slots.address(), plan.rows, code,
                                                 hadamard_constant(self.head_dim), keys.data_ptr(), values.data_ptr(),
                                                 _lib.current_stream_handle(self.device))
            _lib.check(st, "nq_fourbit_read")
        return keys, values

    # ---------------------------------------------------------------- attention

    def plan_attention(self, tables: Sequence[Sequence[int]], lengths: Sequence[int], queries: Optional[Sequence[int]] = None,
                       causal: bool = True, sliding_window: Optional[int] = None) -> FourBitAttentionPlan:
        """The plan of packed queries over sequences of this pool.

        Sequence b holds lengths[b] tokens in its pages tables[b] (entries past those are padding) and has queries[b]
        query rows (None: one each), one sequence's after another's.  causal: they are its last tokens', and query i sees
        the tokens up to its own, with sliding_window the last so many of them.  causal=False: every query sees all of the
        sequence's tokens, whatever their numbers (cross attention to an encoder's states).  A sequence without tokens:
        its queries' rows are zero."""
        lens = [int(n) for n in (lengths.tolist() if torch.is_tensor(lengths) else lengths)]
        news = [1] * len(lens) if queries is None else \
            [int(n) for n in (queries.tolist() if torch.is_tensor(queries) else queries)]
        if not len(tables) == len(lens) == len(news):
            raise ValueError(f"{len(tables)} tables, {len(lens)} lengths and {len(news)} numbers of queries")
        if sliding_window is not None and (int(sliding_window) <= 0 or not causal):
            raise ValueError(f"sliding_window must be positive, and needs causal queries, got {sliding_window}")
        flat = []
        for b, (n, q) in enumerate(zip(lens, news)):
            if not 0 <= n <= len(tables[b]) * self.page_tokens:
                raise ValueError(f"sequence {b}: {n} tokens in {len(tables[b])} pages of {self.page_tokens}")
            if q < 0 or (causal and q > n > 0):
                raise ValueError(f"sequence {b}: {q} queries of {n} tokens")
            flat.append(self.in_use(tables[b][:self.pages_for(n)], "plan_attention"))
        if sum(news) >= 1 << 31:
            raise ValueError(f"{sum(news)} query rows: a plan takes less than 2^31")
        window = 0 if sliding_window is None or int(sliding_window) >= max(lens, default=0) else int(sliding_window)
        return FourBitAttentionPlan(self, flat, lens, news, bool(causal), window)

    def attend(self, plan: FourBitAttentionPlan, query: torch.Tensor, layer: int = 0, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of query [rows, q_heads, head_dim] (fp16 or bf16, q_heads a multiple of the pool's, any strides of rows
        and heads) over the plan's tokens in one layer.  scale: 1 / sqrt(head_dim) by default.

        Returns [rows, q_heads, head_dim].  Rows behind the plan's are left as they are in `out`, and are zero without one;
        `out` may be query.  Codes are exact in the products; a transformed query is rounded to 2^-16 of its largest
        coordinate, weights to 22 bits where a kv head has up to 96 rows of a sequence (query tokens x query heads), and to 11
        where it has more, but for up to 16 rows that are left over behind full tiles.  A weight times its value's scale
        that is below 2^-30 of the largest scale that the row sees is lost.  An fp16 output is then 2.1e-4 from 64 bits, which
        is its own rounding, or 2.6e-4.  How a row's tokens are cut follows from the whole plan: outputs of one row alone and
        in a batch agree to roundings.
        A captured graph reads the plan's arrays: keep the plan while it is replayed.  Inference only."""
        self._check_plan(plan, FourBitAttentionPlan, "attend", layer)
        shape, dtype, dev = query.shape, query.dtype, self.device
        if query.device != dev:
            _lib.require_device(query, "query")
            raise ValueError(f"query is on {query.device}, the pool on {dev}")
        if len(shape) != 3 or shape[0] < plan.rows or shape[2] != self.head_dim:
            raise ValueError(f"query must be ({plan.rows} rows or more, num_heads, {self.head_dim}), got {tuple(shape)}")
        if dtype not in _DTYPES:
            raise ValueError(f"attend takes fp16 or bf16 queries, got {dtype}")
        if (query.requires_grad or out is not None and out.requires_grad) and torch.is_grad_enabled():
            raise NotImplementedError("attend has no backward pass; call it under torch.no_grad()")
        if has_tangent(query, out):
            raise NotImplementedError("attend has no derivative in forward mode; call it on a query without a tangent")
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not 0.0 < scale < 1e30:
            raise ValueError(f"scale must be positive, got {scale}")
        hq = shape[1]
        ints, places, counts, nbytes = plan._work.get(hq) or plan.work(hq)
        given = out
        if out is None:
            out = empty_as(query)
            if shape[0] > plan.rows:
                out[plan.rows:].zero_()
        else:
            check_out(out, query, "out", align=8)
            if not same_or_apart(out, query):
                raise ValueError("attend: out may be query itself, and must not overlap it otherwise")
        if ints is None or plan.rows == 0:
            return out
        q = aligned(query)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None  # of this call alone
        with on_device(dev):
            base = ints.address()
            st = _lib.load().nq_fourbit_attention(_ATTEND_PACK.pack(
                self.desc_at, int(layer), hq, _lib.NQ_F16 if dtype == torch.float16 else _lib.NQ_BF16, *counts[:5],
                int(plan.causal), plan.window, scale, hadamard_constant(self.head_dim), counts[5], q.data_ptr(), out.data_ptr(),
                base + places[0], base + places[1], base + places[2], *q.stride()[:2], *out.stride()[:2],
                0 if ws is None else ws.data_ptr(), nbytes), _lib.current_stream_handle(dev))
        _lib.check(st, "nq_fourbit_attention")
        written(given)
        return out
