"""vLLM page-granular caller and the decode-side consumer of compressed pages.

Mirrors nexusquant/integrations/vllm_backend.py (CompressedPage,
NexusQuantKVCompressor, NexusQuantPagedAttention) on the gfx950 library:

- compress_page        -> nq_page_encode  (vllm_backend.py:344-392)
- decompress_page      -> nq_page_decode  (:394-429)
- decompress_for_attention -> nq_page_logits (:431-467)
- pack/unpack_codes_nibble -> nq_nibble_pack / nq_nibble_unpack (:475-536)
- NexusQuantPagedAttention.forward -> nq_paged_attention (:692-765): decode
  attention read straight from the int8 pages, without materialising fp16
  keys or values.

Page format, arguments, return values and error messages are the reference's.
Every call needs the HIP library and device tensors; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import dataclasses
import math
import struct
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .hadamard import hadamard_constant
from .ops import PlanTensor, _addr, _PtrArrays, on_device
from .rope import device_merged_table, device_table

_FP16_BYTES = 2
_KERNEL_HEAD_DIMS = (64, 128, 256)


@dataclasses.dataclass
class CompressedPage:
    """A single compressed KV block (vllm_backend.py:75-125).

    key_codes / value_codes: (num_heads, num_valid, head_dim) int8, 2 * lattice point
    key_scales / value_scales: (num_heads, num_valid) fp16 per-(head, token) scale
    positions: (num_valid,) int32 absolute token positions (RoPE of keys)
    num_valid: number of tokens stored
    max_position: largest stored position when known (set by compress_page;
    lets decoding size the RoPE table without reading the positions back).
    """

    key_codes: torch.Tensor
    value_codes: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor
    positions: torch.Tensor
    num_valid: int
    max_position: Optional[int] = dataclasses.field(default=None, compare=False, repr=False)

    @property
    def compressed_bytes(self) -> int:
        n = self.num_valid
        h = self.key_codes.shape[0]
        d = self.key_codes.shape[2]
        return 2 * h * n * d + 2 * h * n * _FP16_BYTES + n * 4

    @property
    def uncompressed_bytes(self) -> int:
        n = self.num_valid
        h = self.key_codes.shape[0]
        d = self.key_codes.shape[2]
        return 2 * h * n * d * _FP16_BYTES


def _stream(dev) -> ctypes.c_void_p:
    return ctypes.c_void_p(_lib.current_stream_handle(dev))


def _page_max_position(page: CompressedPage) -> int:
    if page.max_position is None:
        pos = page.positions
        page.max_position = int(pos.max()) if pos.numel() else 0
        if pos.numel() and int(pos.min()) < 0:
            raise ValueError("page positions must be non-negative")
    return page.max_position


def _check_page(page: CompressedPage, head_dim: int) -> None:
    kc, vc = page.key_codes, page.value_codes
    for name, t, dt in (("key_codes", kc, torch.int8), ("value_codes", vc, torch.int8),
                        ("key_scales", page.key_scales, torch.float16),
                        ("value_scales", page.value_scales, torch.float16),
                        ("positions", page.positions, torch.int32)):
        _lib.require_device(t, f"CompressedPage.{name}")
        if t.dtype != dt:
            raise TypeError(f"CompressedPage.{name} must be {dt}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"CompressedPage.{name} must be contiguous")
    if kc.dim() != 3 or kc.shape[2] != head_dim or vc.shape != kc.shape:
        raise ValueError(f"page codes must be (num_heads, tokens, {head_dim}), got {tuple(kc.shape)} / "
                         f"{tuple(vc.shape)}")
    h, n, _ = kc.shape
    if tuple(page.key_scales.shape) != (h, n) or tuple(page.value_scales.shape) != (h, n):
        raise ValueError("page scales must be (num_heads, tokens)")
    if tuple(page.positions.shape) != (n,):
        raise ValueError("page positions must be (tokens,)")
    if kc.data_ptr() % 8 or vc.data_ptr() % 8:
        raise ValueError("page codes must be 8-byte aligned")


class NexusQuantKVCompressor:
    """Compression backend for vLLM paged KV cache (vllm_backend.py:132-170).

    Keys: inverse RoPE at each token's absolute position -> Hadamard -> E8;
    values: Hadamard -> E8; int8 codes 2p and fp16 per-(head, token) scales.
    """

    def __init__(self, head_dim: int = 128, bits: int = 2, eviction_rate: float = 0.0,
                 rope_base: float = 10000.0):
        if bits not in (2, 3, 4):
            raise ValueError(f"bits must be 2, 3, or 4 (got {bits})")
        if head_dim & (head_dim - 1) != 0:
            raise ValueError(f"head_dim must be a power of 2 (got {head_dim})")
        if head_dim not in _KERNEL_HEAD_DIMS:
            raise NotImplementedError(f"head_dim {head_dim}: the gfx950 page kernels take 64, 128 or 256")
        self.head_dim = head_dim
        self.bits = bits
        self.levels = 2 ** bits
        self.eviction_rate = eviction_rate  # stored as the reference does; pages keep every token
        self.rope_base = rope_base

    # ------------------------------------------------------------------ tables

    def _tables(self, max_position: int, device):
        cos, sin = device_table(max_position + 1, self.head_dim, self.rope_base, None, device)
        dm, dp = device_merged_table(cos.shape[0], self.head_dim, self.rope_base, None, device)
        return cos, sin, dm, dp

    def _desc(self, n_pages: int, heads: int, tokens: int, is_key: bool, arrays: dict, tables,
              dtype_code: int = _lib.NQ_F16) -> _lib.PageDesc:
        cos = sin = dm = dp = None
        n_pos = 0
        if is_key:
            cos, sin, dm, dp = tables
            n_pos = cos.shape[0]
        return _lib.PageDesc(
            n_pages=n_pages, heads=heads, tokens=tokens, head_dim=self.head_dim, dtype=dtype_code,
            levels=self.levels, is_key=int(is_key), src=_addr(arrays.get("src")),
            positions=_addr(arrays.get("positions")), codes=_addr(arrays.get("codes")),
            scales=_addr(arrays.get("scales")), out=_addr(arrays.get("out")),
            rope_cos=_addr(cos), rope_sin=_addr(sin), rope_sin_minus_cos=_addr(dm), rope_cos_plus_sin=_addr(dp),
            rope_n_pos=n_pos, hadamard_scale=hadamard_constant(self.head_dim))

    # ------------------------------------------------------------- public API

    def compress_page(self, key_page: torch.Tensor, value_page: torch.Tensor,
                      page_positions: torch.Tensor) -> CompressedPage:
        """Compress one KV page (num_heads, block_size, head_dim) at absolute positions."""
        return self.compress_pages([(key_page, value_page, page_positions)])[0]

    def compress_pages(self, pages: Sequence[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]
                       ) -> List[CompressedPage]:
        """compress_page over many pages; pages of equal shape share one launch per role."""
        lib = _lib.load()
        out: List[Optional[CompressedPage]] = [None] * len(pages)
        groups: Dict[tuple, List[int]] = {}
        prepared = []
        host_pos: Dict[torch.device, list] = {}  # positions given on the host, copied once per device
        for i, (k, v, pos) in enumerate(pages):
            _lib.require_device(k, "key_page")
            if k.dim() != 3 or v.shape != k.shape:
                raise ValueError(f"key/value pages must be (num_heads, block_size, head_dim) of equal shape, "
                                 f"got {tuple(k.shape)} / {tuple(v.shape)}")
            h, n, d = k.shape
            if d != self.head_dim:
                raise ValueError(f"page head_dim {d} != compressor head_dim {self.head_dim}")
            dev = k.device
            pos_list = torch.as_tensor(pos)
            if pos_list.numel() != n:
                raise ValueError(f"page_positions has {pos_list.numel()} entries for {n} tokens")
            pos_d = None
            if n and pos_list.device.type == "cpu":
                pos_np = (pos_list.to(torch.int64) if pos_list.is_floating_point() else pos_list).numpy()
                lo, hi = int(pos_np.min()), int(pos_np.max())
                host_pos.setdefault(dev, []).append((i, pos_np))
            elif n:
                lo, hi = (int(x) for x in torch.stack([pos_list.min(), pos_list.max()]).tolist())
            else:
                lo = hi = 0
            if lo < 0:
                raise ValueError("page positions must be non-negative")
            if not n or pos_list.device.type != "cpu":
                pos_d = pos_list.to(device=dev, dtype=torch.int32).contiguous()
            _lib.require_device(v, "value_page")
            kk = k.contiguous()
            vv = v.contiguous()
            kk = kk if kk.data_ptr() % 16 == 0 else kk.clone()
            vv = vv if vv.data_ptr() % 16 == 0 else vv.clone()
            prepared.append([kk, vv, pos_d, hi])
            groups.setdefault((h, n, k.dtype, v.dtype, dev), []).append(i)
        for dev, items in host_pos.items():
            flat = torch.from_numpy(np.concatenate([p.reshape(-1).astype(np.int32) for _, p in items])).to(dev)
            for (i, _), part in zip(items, flat.split([p.size for _, p in items])):
                prepared[i][2] = part.reshape(torch.as_tensor(pages[i][2]).shape)
        for (h, n, kdt, vdt, dev), idx in groups.items():
            m = len(idx)
            kc = torch.empty(m, h, n, self.head_dim, dtype=torch.int8, device=dev).unbind(0)
            vc = torch.empty(m, h, n, self.head_dim, dtype=torch.int8, device=dev).unbind(0)
            ks = torch.empty(m, h, n, dtype=torch.float16, device=dev).unbind(0)
            vs = torch.empty(m, h, n, dtype=torch.float16, device=dev).unbind(0)
            max_pos = max(prepared[i][3] for i in idx)
            tables = self._tables(max_pos, dev)
            for role, is_key in (("k", True), ("v", False)):
                src = [prepared[i][0 if is_key else 1] for i in idx]
                codes = kc if is_key else vc
                scales = ks if is_key else vs
                groups_t = [src, [prepared[i][2] for i in idx] if is_key else None, list(codes), list(scales)]
                staged = _PtrArrays(groups_t, dev, host=True)
                arrays = dict(zip(("src", "positions", "codes", "scales"), staged.arrays))
                desc = self._desc(m, h, n, is_key, arrays, tables, _lib.dtype_code(kdt if is_key else vdt))
                with torch.cuda.device(dev):
                    try:
                        st = lib.nq_page_encode(ctypes.byref(desc), _stream(dev))
                    finally:
                        staged.release()
                _lib.check(st, "nq_page_encode")
            for j, i in enumerate(idx):
                out[i] = CompressedPage(key_codes=kc[j], value_codes=vc[j], key_scales=ks[j], value_scales=vs[j],
                                        positions=prepared[i][2], num_valid=n, max_position=prepared[i][3])
        return out  # type: ignore[return-value]

    def decompress_page(self, compressed_page: CompressedPage) -> Tuple[torch.Tensor, torch.Tensor]:
        """(keys, values) (num_heads, tokens, head_dim) fp16 of one page."""
        return self.decompress_pages([compressed_page])[0]

    def decompress_pages(self, pages: Sequence[CompressedPage]) -> List[Tuple[torch.Tensor, torch.Tensor]]:
        lib = _lib.load()
        out: List[Optional[Tuple[torch.Tensor, torch.Tensor]]] = [None] * len(pages)
        groups: Dict[tuple, List[int]] = {}
        for i, p in enumerate(pages):
            _check_page(p, self.head_dim)
            h, n, _ = p.key_codes.shape
            groups.setdefault((h, n, p.key_codes.device), []).append(i)
        for (h, n, dev), idx in groups.items():
            m = len(idx)
            ko = torch.empty(m, h, n, self.head_dim, dtype=torch.float16, device=dev).unbind(0)
            vo = torch.empty(m, h, n, self.head_dim, dtype=torch.float16, device=dev).unbind(0)
            if n:
                tables = self._tables(max(_page_max_position(pages[i]) for i in idx), dev)
                for is_key in (True, False):
                    pg = [pages[i] for i in idx]
                    groups_t = [[p.key_codes if is_key else p.value_codes for p in pg],
                                [p.key_scales if is_key else p.value_scales for p in pg],
                                [p.positions for p in pg] if is_key else None,
                                list(ko if is_key else vo)]
                    staged = _PtrArrays(groups_t, dev, host=True)
                    arrays = dict(zip(("codes", "scales", "positions", "out"), staged.arrays))
                    desc = self._desc(m, h, n, is_key, arrays, tables)
                    with torch.cuda.device(dev):
                        try:
                            st = lib.nq_page_decode(ctypes.byref(desc), _stream(dev))
                        finally:
                            staged.release()
                    _lib.check(st, "nq_page_decode")
            for j, i in enumerate(idx):
                out[i] = (ko[j], vo[j])
        return out  # type: ignore[return-value]

    def decompress_for_attention(self, compressed_page: CompressedPage, query: torch.Tensor) -> torch.Tensor:
        """Logits (num_heads, q_len, tokens) fp32 = q . k / sqrt(head_dim) against the page's keys."""
        lib = _lib.load()
        p = compressed_page
        _check_page(p, self.head_dim)
        _lib.require_device(query, "query")
        h, n, d = p.key_codes.shape
        if query.dim() != 3 or query.shape[0] != h or query.shape[2] != d:
            raise ValueError(f"query must be (num_heads={h}, q_len, head_dim={d}), got {tuple(query.shape)}")
        dev = p.key_codes.device
        q = query.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        q_len = q.shape[1]
        logits = torch.empty(h, q_len, n, dtype=torch.float32, device=dev)
        if n == 0 or q_len == 0:
            return logits
        tables = self._tables(_page_max_position(p), dev)
        staged = _PtrArrays([[p.key_codes], [p.key_scales], [p.positions]], dev, host=True)
        arrays = dict(zip(("codes", "scales", "positions"), staged.arrays))
        desc = self._desc(1, h, n, True, arrays, tables)
        with torch.cuda.device(dev):
            try:
                st = lib.nq_page_logits(ctypes.byref(desc), _addr(q), _lib.dtype_code(q.dtype), q_len,
                                        ctypes.c_float(float(np.float32(math.sqrt(self.head_dim)))),
                                        _addr(logits), _stream(dev))
            finally:
                staged.release()
        _lib.check(st, "nq_page_logits")
        return logits

    @staticmethod
    def pack_codes_nibble(codes: torch.Tensor) -> torch.Tensor:
        """(..., d) int8 -> (..., ceil(d/2)) uint8: clamp(code + 8, 0, 15) nibbles, low nibble first."""
        lib = _lib.load()
        _lib.require_device(codes, "codes")
        if codes.dtype != torch.int8:
            raise TypeError(f"codes must be int8, got {codes.dtype}")
        d = codes.shape[-1]
        c = codes.contiguous()
        rows = c.numel() // d if d else 0
        out = torch.empty(*codes.shape[:-1], (d + 1) // 2, dtype=torch.uint8, device=codes.device)
        if rows and d:
            with torch.cuda.device(codes.device):
                st = lib.nq_nibble_pack(_addr(c), rows, d, _addr(out), _stream(codes.device))
            _lib.check(st, "nq_nibble_pack")
        return out

    @staticmethod
    def unpack_codes_nibble(packed: torch.Tensor, original_d: int) -> torch.Tensor:
        """Inverse of pack_codes_nibble: (..., ceil(d/2)) uint8 -> (..., original_d) int8."""
        lib = _lib.load()
        _lib.require_device(packed, "packed")
        if packed.dtype != torch.uint8:
            raise TypeError(f"packed codes must be uint8, got {packed.dtype}")
        pc = packed.shape[-1]
        d = min(int(original_d), 2 * pc)
        p = packed.contiguous()
        rows = p.numel() // pc if pc else 0
        out = torch.empty(*packed.shape[:-1], max(d, 0), dtype=torch.int8, device=packed.device)
        if rows and d > 0:
            with torch.cuda.device(packed.device):
                st = lib.nq_nibble_unpack(_addr(p), rows, pc, d, _addr(out), _stream(packed.device))
            _lib.check(st, "nq_nibble_unpack")
        return out

    def compression_ratio(self, page: CompressedPage) -> float:
        if page.uncompressed_bytes == 0:
            return 1.0
        return page.uncompressed_bytes / page.compressed_bytes


# ---------------------------------------------------------------------------
# Decode attention over compressed pages
# ---------------------------------------------------------------------------

# Workgroups (chunk, kv head) a plan should have before its chunks stay at the
# kernel's full length: two per CU.  32 query / 8 kv heads x 1000 tokens: 27 us with
# 512-token chunks, 15 with 64; a threshold of 1024 cost 2 us on ragged batches of 8
# and 32 rows, whose combine pass then adds twice the chunks.
_MIN_WORKGROUPS = 512
_MIN_CHUNK = 64  # one 16-token unit for each of a workgroup's four waves


def _tokens_used(row: Sequence[Tuple[int, int]], ctx: int) -> int:
    """Tokens a row attends to: the first ctx of its pages' tokens (a Python slice's
    semantics: a negative length drops tokens from the end, 0 none)."""
    avail = sum(n for _, n in row)
    use = 0 if ctx == 0 else (ctx if ctx > 0 else avail + ctx)
    return max(0, min(use, avail))


def chunk_length(used: Sequence[int], kv_heads: int, cap: int) -> int:
    """Chunk length for rows of `used` tokens: cap, halved while the plan would have
    fewer than _MIN_WORKGROUPS workgroups and a half still is _MIN_CHUNK tokens.

    One length for the whole plan, so where a row is cut, and with it the order of its
    fp32 sums, depends on the rows beside it: its output may differ by one rounding of
    its type between batches.  A length from the row alone gives that up for time:
    8 rows up to 4096 tokens, 32/8 heads, bf16, and 32 rows of 2000 take 21.2 and 47.2 us
    so, 32.8 and 50.2 with 64 workgroups wanted per row, 24.7 and 58.7 with 128."""
    while cap >= 2 * _MIN_CHUNK and sum(-(-n // cap) for n in used) * kv_heads < _MIN_WORKGROUPS:
        cap //= 2
    return cap


def build_chunk_plan(rows: Sequence[Sequence[Tuple[int, int]]], context_lens: Sequence[int], chunk_cap: int):
    """Cut each row's token stream into chunks of at most chunk_cap tokens.

    rows[b] lists (slot, tokens) of the pages row b reads, in order; row b
    attends to the first context_lens[b] tokens of their concatenation (Python
    slice semantics: a negative length drops tokens from the end, 0 none).
    Returns the int32 arrays of nq_attn_desc (segs, units, chunk_units,
    chunk_row, chunk_tokens, row_chunks) and the total token count.
    """
    segs: List[Tuple[int, int, int, int]] = []
    units: List[Tuple[int, int]] = []
    chunk_units: List[int] = []
    chunk_row: List[int] = []
    chunk_tokens: List[int] = []
    row_chunks = [0]
    total = 0
    for b, row in enumerate(rows):
        use = _tokens_used(row, int(context_lens[b]))
        fill = None  # tokens in the row's open chunk (None: none open)
        for slot, n_page in row:
            if use == 0:
                break
            n = min(n_page, use)
            use -= n
            t = 0
            while t < n:
                if fill is None or fill == chunk_cap:
                    chunk_units.append(len(units))
                    chunk_row.append(b)
                    chunk_tokens.append(0)
                    fill = 0
                take = min(n - t, chunk_cap - fill)
                seg = len(segs)
                segs.append((slot, t, take, fill))
                units.extend((seg, u) for u in range(0, take, 16))
                fill += take
                chunk_tokens[-1] += take
                total += take
                t += take
        row_chunks.append(len(chunk_row))
    chunk_units.append(len(units))
    parts = {
        "segs": np.array(segs, dtype=np.int32).reshape(-1),
        "units": np.array(units, dtype=np.int32).reshape(-1),
        "chunk_units": np.array(chunk_units, dtype=np.int32),
        "chunk_row": np.array(chunk_row, dtype=np.int32),
        "chunk_tokens": np.array(chunk_tokens, dtype=np.int32),
        "row_chunks": np.array(row_chunks, dtype=np.int32),
    }
    return parts, total


def unit_records(parts: dict, slot_pages: Sequence[CompressedPage], head_dim: int) -> np.ndarray:
    """The 16-int32 unit records of nq_attn_desc from a chunk plan's segments
    and units: absolute addresses of each unit's first token in its page."""
    segs = parts["segs"].reshape(-1, 4).astype(np.int64)
    units = parts["units"].reshape(-1, 2).astype(np.int64)
    rec = np.zeros((len(units), 16), dtype=np.int64)
    if len(units):
        base = np.array([[p.key_codes.data_ptr(), p.value_codes.data_ptr(), p.key_scales.data_ptr(),
                          p.value_scales.data_ptr(), p.positions.data_ptr(), p.key_codes.shape[1]]
                         for p in slot_pages], dtype=np.int64).reshape(-1, 6)
        sg = segs[units[:, 0]]
        slot, first, n, off = sg[:, 0], sg[:, 1], sg[:, 2], sg[:, 3]
        t0 = first + units[:, 1]
        b = base[slot]
        addr = np.stack([b[:, 0] + t0 * head_dim, b[:, 1] + t0 * head_dim, b[:, 2] + 2 * t0,
                         b[:, 3] + 2 * t0, b[:, 4] + 4 * t0], axis=1)
        rec[:, 0:10:2] = addr & 0xFFFFFFFF
        rec[:, 1:10:2] = addr >> 32
        rec[:, 10] = b[:, 5]
        rec[:, 11] = np.minimum(16, n - units[:, 1])
        rec[:, 12] = off + units[:, 1]
    return rec.astype(np.uint32).view(np.int32).reshape(-1)


@dataclasses.dataclass
class PagedAttentionPlan:
    """Device description of which page tokens each batch row attends to
    (the chunk plan of nq_paged_attention), reusable across decode steps while
    the pages, block tables and context lengths stay the same."""
    batch: int
    kv_heads: int
    head_dim: int
    n_chunks: int
    ints: Optional[torch.Tensor]       # int32: unit records and index arrays, see offsets
    offsets: Dict[str, int]
    max_position: int
    keepalive: list                    # the pages whose memory the plan points at
    tokens: int                        # tokens attended over all rows


# What pays to share: sharing that saves this many tokens' decoding, counted in every kv head (a segment's tokens, once
# for every row but one).  us shared and apart: 8 kv heads x 4, 32 rows x 256 tokens 15.6 and 13.4, x 512 15.9 and
# 17.1, 8 rows x 1024 13.3 and 13.2, x 2048 14.1 and 18.6; 32 x 1, 16 rows x 128 11.2 and 12.6, x 256 11.9 and 15.7.
_MIN_SAVED = 1 << 16


def shared_segments(tables: Sequence[np.ndarray], lengths: Sequence[int], page_tokens: int,
                    min_saved: int) -> List[Tuple[List[int], np.ndarray, int]]:
    """Cut the rows' tokens into segments (rows, pages, tokens) that their rows see whole.

    tables[b]: row b's pages, lengths[b]: its tokens.  Rows that begin with the same full pages
    share a segment of these, and those among them that go on alike another one, and so on; a
    segment of one row is what it has for itself.  Sharing that would save less than min_saved
    tokens is left to what follows it."""
    full = [int(n) // page_tokens for n in lengths]
    out: List[Tuple[List[int], np.ndarray, int]] = []

    # (rows, start, depth): the rows agree on their pages before `depth`; those from `start` on are in no segment yet
    todo = [([b for b in range(len(tables)) if lengths[b] > 0], 0, 0)]
    while todo:
        rows, start, depth = todo.pop()
        groups: Dict[int, List[int]] = {}
        for b in rows:
            if full[b] > depth:
                groups.setdefault(int(tables[b][depth]), []).append(b)
            elif lengths[b] > start * page_tokens:
                out.append(([b], tables[b][start:], int(lengths[b]) - start * page_tokens))
        for same in groups.values():
            if len(same) == 1:
                b = same[0]
                out.append((same, tables[b][start:], int(lengths[b]) - start * page_tokens))
                continue
            most = min(full[b] for b in same)
            stack = np.stack([tables[b][depth:most] for b in same])
            differ = np.flatnonzero((stack != stack[0]).any(axis=0))
            end = depth + int(differ[0]) if len(differ) else most
            tokens = (end - start) * page_tokens
            if (len(same) - 1) * tokens >= min_saved:
                out.append((same, tables[same[0]][start:end], tokens))
                todo.append((same, end, end))
            else:
                todo.append((same, start, end))
    return out


# Tokens that a workgroup takes at a time, by kind, and the least of a chunk: 4 rows of 4 heads over 992 tokens in
# chunks of 64 11.2 us, of 128 11.8.
_SHARED_STAGE = (128, 128, 64)
_SHARED_LEAST = (256, 128, 64)
# The kinds of segments, by query rows (batch rows x query heads of a kv head): many (wide workgroups), some, few.
# Few are up to nq_shared_attention_rows(d, 2) of them: 8 kv heads x 128, us few and some: 64 rows x 8 heads over 512
# own tokens 27.4 and 33.4, 3 x 8 over 9184 at head_dim 256 38.3 and 66.2, 8 x 1 over 8192 at 64 24.4 and 31.4.
# Segments of more than _MANY_ROWS count as many when there are at least _MANY_TOKENS tokens for each of 256 CUs
# (some are up to nq_shared_attention_rows(d, 1)): 8 kv heads x 128, us many and some: 128 query rows over 16384 shared
# tokens 31.1 and 34.4, over 4096 21.7 and 24.0, but with 256 own tokens a row, which go along with some, 32.4 and 25.1;
# 64 query rows over 4096 19.5 and 18.1.
_MANY, _SOME, _FEW = 0, 1, 2
_MANY_ROWS = 32
_MANY_TOKENS = 512
# Few go into the launch of some, where there are any, as long as they have less than this many tokens for each CU (each
# segment counted as 128 at least).  A shared 4096 tokens of 128 query rows and own ones, us together and with a launch
# for the own ones: 8 kv heads x 128, 512 a CU 35.1 and 38.7, 1024 57.8 and 44.2; x 64, 768 23.5 and 29.2, 1536 34.3 and
# 34.9; 4 x 256, 128 38.0 and 43.7, 256 59.3 and 47.2.  32 rows of 4 heads and 256 own tokens: 25.7 us together, 26.3
# with the own ones as some, 36 with a launch of their own.
_FEW_TOKENS = {64: 1536, 128: 768, 256: 192}


def _shared_chunk(lengths, tiles, kv_heads: int, cap: int, least: int, stage: int, workgroups: int) -> int:
    """Chunk length of segments: the least multiple of `stage` with which the launch is one round of
    `workgroups`.  16 rows x 4 heads over 8192 tokens, us: 512 workgroups 32.3, 256 (chunks of 256) 23.4,
    128 27.3; 64 rows' own 512 tokens: 512 workgroups 28.8, 1024 31.9."""
    length = min(least, cap)
    while length < cap and kv_heads * sum(t * -(-n // length) for t, n in zip(tiles, lengths)) > workgroups:
        length += stage
    return length


def shared_items(segments, batch: int, group: int, kv_heads: int, head_dim: int, cap: Sequence[int],
                 rows: Sequence[int]):
    """The work list of nq_shared_attention: int32 arrays items, pages, seg_rows, row_slots, and the counts of
    items, of those of segments of many rows (they come first), of few (last) and of slots.  cap, rows: most
    tokens of a chunk and most query rows of a workgroup, by kind."""
    queries = [len(r) * group for r, _, _ in segments]
    kind = [_FEW if q <= rows[_FEW] else _MANY if q > _MANY_ROWS else _SOME for q in queries]
    work = kv_heads * sum(s[2] * -(-q // rows[_MANY]) for s, q, k in zip(segments, queries, kind) if k == _MANY)
    if work < 256 * _MANY_TOKENS:
        kind = [_SOME if k == _MANY and q <= rows[_SOME] else k for k, q in zip(kind, queries)]
    launch = kind
    few_tokens = kv_heads * sum(max(s[2], 128) for s, k in zip(segments, kind) if k == _FEW)
    if _SOME in kind and few_tokens < 256 * _FEW_TOKENS[head_dim]:
        launch = [_SOME if k == _FEW else k for k in kind]
    per_tile = [max(1, n // group) for n in rows]  # batch rows of a workgroup
    tiles = [-(-len(s[0]) // per_tile[k]) for s, k in zip(segments, kind)]
    # as many workgroups as run at once: LDS leaves one of the wide ones on a CU, LDS or registers those of the others
    at_once = (1, {64: 3, 128: 2}.get(head_dim, 1), {64: 4, 128: 3}.get(head_dim, 2))
    step = []
    for k in (_MANY, _SOME, _FEW):
        of = [i for i in range(len(segments)) if launch[i] == k]
        step.append(_shared_chunk([segments[i][2] for i in of], [tiles[i] for i in of], kv_heads, cap[k],
                                  _SHARED_LEAST[k], _SHARED_STAGE[k], 256 * at_once[k]))
    chunks = [-(-s[2] // step[k]) for s, k in zip(segments, launch)]
    per_row = [0] * (batch + 1)
    for (r, _, _), c in zip(segments, chunks):
        for b in r:
            per_row[b + 1] += c
    row_slots = np.cumsum(per_row)
    nxt = row_slots[:-1].tolist()
    records, seg_rows, pages = [], [], []
    at_pages = 0
    # by kind, long ones before short ones
    for i in sorted(range(len(segments)), key=lambda i: (launch[i], -segments[i][2])):
        r, seg_pages, n = segments[i]
        at_rows = len(seg_rows)
        for b in r:
            seg_rows.append((b, nxt[b]))
            nxt[b] += chunks[i]
        # chunks in eights (one for each XCD), a chunk's row tiles one eight after another
        length, per, few = step[launch[i]], per_tile[kind[i]], int(launch[i] != kind[i])
        for c0 in range(0, chunks[i], 8):
            for r0 in range(0, len(r), per):
                for c in range(c0, min(c0 + 8, chunks[i])):
                    records.append((at_pages, c * length, min(n - c * length, length), at_rows + r0,
                                    min(len(r) - r0, per), c, few, 0))
        pages.append(np.asarray(seg_pages, dtype=np.int32))
        at_pages += len(seg_pages)
    n_kind = [sum(t * c for t, c, x in zip(tiles, chunks, launch) if x == k) for k in (_MANY, _FEW)]
    parts = {"items": np.array(records, dtype=np.int32).reshape(-1),
             "pages": np.concatenate(pages) if pages else np.zeros(0, dtype=np.int32),
             "seg_rows": np.array(seg_rows, dtype=np.int32).reshape(-1), "row_slots": row_slots.astype(np.int32)}
    return parts, len(records), n_kind[0], n_kind[1], int(row_slots[-1])


# nq_shared_desc, packed in one go and passed as bytes
_SHARED_PACK = struct.Struct("P8i8Pq2fPq")


class _SharedTables:
    """Merged rotation tables, and their addresses and length."""

    def __init__(self, dm: torch.Tensor, dp: torch.Tensor):
        self.tensors = (dm, dp)
        self.args = (dm.data_ptr(), dp.data_ptr(), dm.shape[0])
        self._streams: set = set()

    def read_on(self, device) -> int:
        """The device's current stream's handle, for a launch that reads the tables: their memory, once dropped, is not
        given to others before what this stream had queued until then has run.  (A captured graph's plan keeps them.)"""
        handle = _lib.current_stream_handle(device)
        if handle not in self._streams and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(device)
            for t in self.tensors:
                t.record_stream(stream)
            self._streams.add(handle)
        return handle


class SharedAttentionPlan:
    """Which tokens of a pool each batch row attends to, and which of them rows share: valid for every
    layer of the pool while the rows' tables and lengths stay the same.  The device arrays are made for a
    number of query heads, the first time that it is used (before a graph is captured)."""

    def __init__(self, pool, batch: int, segments):
        self.pool = pool
        self.batch = batch
        self.segments = segments
        self._work: Dict[int, tuple] = {}
        self._tables: Dict[int, _SharedTables] = {}  # by id, each once, however many attentions use the plan in turn

    def work(self, q_heads: int):
        """(device ints, what nq_shared_desc holds that all calls share: counts, the arrays' places in the ints, factors
        and workspace bytes) for q_heads query heads."""
        got = self._work.get(q_heads)
        if got is None:
            with on_device(self.pool.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("run_shared: run the plan once before capturing it into a graph")
            lib = _lib.load()
            heads, d = self.pool.num_heads, self.pool.head_dim
            most = [int(lib.nq_shared_attention_rows(d, k)) for k in range(3)]
            if q_heads == 0 or q_heads % heads or q_heads // heads > most[_MANY]:
                raise ValueError(f"num_heads {q_heads} is not a multiple (up to {most[_MANY]}) of the pool's {heads}")
            parts, *counts = shared_items(self.segments, self.batch, q_heads // heads, heads, d,
                                          [int(lib.nq_shared_attention_chunk_tokens(k)) for k in range(3)], most)
            places, at = [], 0
            for v in parts.values():
                places.append(at)  # bytes
                at += 4 * len(v)
            ints = PlanTensor(np.concatenate(list(parts.values())), self.pool.device)
            got = self._work[q_heads] = (ints, counts, places, (hadamard_constant(d), float(np.float32(math.sqrt(d)))),
                                         int(lib.nq_shared_attention_workspace(counts[-1], q_heads, d)))
        return got

    def reads(self, tables: _SharedTables):
        """Arguments of a call that reads these tables.  They are kept with the plan: a captured graph goes on reading them."""
        self._tables[id(tables)] = tables
        return tables.args


class NexusQuantPagedAttention:
    """Paged attention over compressed pages (vllm_backend.py:543-775)."""

    def __init__(self, compressor: NexusQuantKVCompressor):
        self.compressor = compressor
        self._block_pool: dict = {}
        self._next_block_id: int = 0
        self._tables: Dict[tuple, _SharedTables] = {}  # of run_shared, by (device, head_dim, rope_base)

    def allocate_block(self) -> int:
        block_id = self._next_block_id
        self._next_block_id += 1
        return block_id

    def free_block(self, block_id: int) -> None:
        self._block_pool.pop(block_id, None)

    def is_block_compressed(self, block_id: int) -> bool:
        return block_id in self._block_pool

    def compress_and_cache(self, key: torch.Tensor, value: torch.Tensor, key_cache: dict, value_cache: dict,
                           slot_mapping: torch.Tensor) -> None:
        """reshape_and_cache for compressed storage (vllm_backend.py:622-688): the new tokens of each
        block become that block's page, at positions = their slot offsets."""
        if key.shape[0] == 0:
            return
        block_size = self._infer_block_size(slot_mapping)
        device = key.device
        block_ids = (slot_mapping // block_size).tolist()
        offsets = (slot_mapping % block_size).tolist()
        tok_idx: Dict[int, list] = {}
        tok_off: Dict[int, list] = {}
        for i, (bid, off) in enumerate(zip(block_ids, offsets)):
            tok_idx.setdefault(bid, []).append(i)
            tok_off.setdefault(bid, []).append(off)
        work = []
        for bid, idx in tok_idx.items():
            t = torch.tensor(idx, dtype=torch.long, device=device)
            work.append((key[t].permute(1, 0, 2), value[t].permute(1, 0, 2),
                         torch.tensor(tok_off[bid], dtype=torch.int32)))
        pages = self.compressor.compress_pages(work)
        for bid, page in zip(tok_idx.keys(), pages):
            key_cache[bid] = page
            value_cache[bid] = page

    # --------------------------------------------------------------- forward

    def plan(self, compressed_key_cache: dict, block_tables: List[List[int]], context_lens) -> PagedAttentionPlan:
        """Chunk plan of the tokens each row attends to: the pages of block_tables[b]
        present in the cache, concatenated, first context_lens[b] tokens (Python
        slice semantics, as the reference slices the concatenation).

        The chunk length follows from all rows together (chunk_length): outputs of one
        row planned alone and in a batch agree to one rounding, not bit for bit."""
        chunk_cap = int(_lib.load().nq_paged_attention_chunk_tokens())
        ctx = [int(x) for x in (context_lens.tolist() if torch.is_tensor(context_lens) else context_lens)]
        slot_of: Dict[int, int] = {}
        slot_pages: List[CompressedPage] = []
        rows = []
        kv_heads = head_dim = None
        for b in range(len(ctx)):
            row = []
            if ctx[b] != 0:
                for bid in block_tables[b]:
                    p = compressed_key_cache.get(bid) if bid in compressed_key_cache else None
                    if p is None:
                        continue
                    if kv_heads is None:
                        kv_heads, head_dim = p.key_codes.shape[0], p.key_codes.shape[2]
                        if head_dim != self.compressor.head_dim:
                            raise ValueError(f"page head_dim {head_dim} != compressor head_dim "
                                             f"{self.compressor.head_dim}")
                    if p.key_codes.shape[0] != kv_heads or p.key_codes.shape[2] != head_dim:
                        raise ValueError("all pages must share (num_heads, head_dim)")
                    if id(p) not in slot_of:
                        _check_page(p, head_dim)
                        slot_of[id(p)] = len(slot_pages)
                        slot_pages.append(p)
                    row.append((slot_of[id(p)], p.key_codes.shape[1]))
            rows.append(row)
        used = [_tokens_used(row, c) for row, c in zip(rows, ctx)]
        chunk_cap = chunk_length(used, kv_heads or 1, chunk_cap)
        parts, total = build_chunk_plan(rows, ctx, chunk_cap)
        n_chunks = len(parts["chunk_row"])
        dev = None
        max_pos = 0
        if slot_pages:
            dev = slot_pages[0].key_codes.device
            for p in slot_pages:
                max_pos = max(max_pos, _page_max_position(p))
        parts["units"] = unit_records(parts, slot_pages, head_dim or self.compressor.head_dim)
        offsets: Dict[str, int] = {}
        buf = []
        at = 0
        for k in ("units", "chunk_units", "chunk_row", "chunk_tokens", "row_chunks"):
            v = parts[k]
            offsets[k] = at
            pad = (-len(v)) % 4  # 16-byte aligned starts
            buf.append(v)
            if pad:
                buf.append(np.zeros(pad, dtype=np.int32))
            at += len(v) + pad
        if dev is None and torch.cuda.is_available():
            dev = torch.device("cuda", torch.cuda.current_device())
        ints = torch.tensor(np.concatenate(buf), device=dev) if dev is not None else None
        return PagedAttentionPlan(batch=len(ctx), kv_heads=kv_heads or 0,
                                  head_dim=head_dim or self.compressor.head_dim, n_chunks=n_chunks,
                                  ints=ints, offsets=offsets, max_position=max_pos,
                                  keepalive=slot_pages, tokens=total)

    def run(self, plan: PagedAttentionPlan, query: torch.Tensor, out: Optional[torch.Tensor] = None,
            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of query (batch, num_heads, head_dim) over a plan's tokens."""
        lib = _lib.load()
        _lib.require_device(query, "query")
        if query.dim() != 3 or query.shape[0] != plan.batch:
            raise ValueError(f"query must be (batch={plan.batch}, num_heads, head_dim), got {tuple(query.shape)}")
        b, hq, d = query.shape
        if d != self.compressor.head_dim:
            raise ValueError(f"query head_dim {d} != compressor head_dim {self.compressor.head_dim}")
        dev = query.device
        q = query.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        if out is None:
            out = torch.empty_like(q)
        kv = plan.kv_heads if plan.n_chunks else hq
        if hq % kv:
            raise ValueError(f"num_heads {hq} is not a multiple of the pages' num_heads {kv}")
        ws_bytes = lib.nq_paged_attention_workspace(plan.n_chunks, hq, d)
        if workspace is None or workspace.numel() < ws_bytes:
            from .ops import workspace as stream_workspace
            workspace = stream_workspace(dev, ws_bytes)
        cos = sin = dm = dp = None
        n_pos = 0
        if plan.n_chunks:
            cos, sin, dm, dp = self.compressor._tables(plan.max_position, dev)
            n_pos = cos.shape[0]
        ints = plan.ints
        base = ints.data_ptr() if ints is not None else 0

        def at(name):
            return ctypes.c_void_p(base + 4 * plan.offsets[name]) if ints is not None else None

        desc = _lib.AttnDesc(
            batch=b, q_heads=hq, kv_heads=kv, head_dim=d, q_dtype=_lib.dtype_code(q.dtype),
            n_chunks=plan.n_chunks, query=_addr(q), out=_addr(out), units=at("units"),
            chunk_units=at("chunk_units"),
            chunk_row=at("chunk_row"), chunk_tokens=at("chunk_tokens"), row_chunks=at("row_chunks"),
            rope_cos=_addr(cos), rope_sin=_addr(sin), rope_sin_minus_cos=_addr(dm), rope_cos_plus_sin=_addr(dp),
            rope_n_pos=n_pos, hadamard_scale=hadamard_constant(d),
            scale_divisor=float(np.float32(math.sqrt(d))), workspace=_addr(workspace), workspace_bytes=ws_bytes)
        with torch.cuda.device(dev):
            st = lib.nq_paged_attention(ctypes.byref(desc), _stream(dev))
        _lib.check(st, "nq_paged_attention")
        return out

    # ----------------------------------------------------- rows that share pages

    def plan_shared(self, pool, block_tables: Sequence[Sequence[int]], context_lens,
                    min_saved: Optional[int] = None) -> SharedAttentionPlan:
        """The plan of rows over a CompressedPagePool: row b attends to the first context_lens[b] tokens of
        its pages block_tables[b] (0: none; entries past those tokens are padding).  Full pages that several
        rows begin with, as forks do, are read and decoded once for all of them, where that saves min_saved
        tokens' decoding (None: what pays, 65536 over the pool's heads)."""
        if pool.head_dim != self.compressor.head_dim:
            raise ValueError(f"pool head_dim {pool.head_dim} != compressor head_dim {self.compressor.head_dim}")
        ctx = [int(x) for x in (context_lens.tolist() if torch.is_tensor(context_lens) else context_lens)]
        if len(ctx) != len(block_tables):
            raise ValueError(f"{len(block_tables)} block tables for {len(ctx)} context lengths")
        tables = []
        for b, n in enumerate(ctx):
            table = block_tables[b]
            if not 0 <= n <= len(table) * pool.page_tokens:
                raise ValueError(f"row {b}: {n} tokens in {len(table)} pages of {pool.page_tokens}")
            tables.append(pool.in_use(table[:pool.pages_for(n)], "plan_shared"))  # what follows is padding
        if min_saved is None:
            min_saved = -(-_MIN_SAVED // pool.num_heads)
        return SharedAttentionPlan(pool, len(ctx), shared_segments(tables, ctx, pool.page_tokens, min_saved))

    def _shared_tables(self, max_position: int, dev) -> _SharedTables:
        """A device's merged rotation tables, kept here until a larger position needs longer ones."""
        comp = self.compressor  # may be another one, or of another base, than in the call before
        key = dev, comp.head_dim, comp.rope_base
        got = self._tables.get(key)
        if got is None or got.args[2] <= max_position:
            _, _, dm, dp = comp._tables(max_position, dev)
            got = self._tables[key] = _SharedTables(dm, dp)
        return got

    def run_shared(self, plan: SharedAttentionPlan, query: torch.Tensor, layer: int = 0,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of query (batch, num_heads, head_dim; fp16 or bf16) over a shared plan's tokens in one
        layer of its pool.  num_heads is a multiple of the pool's heads.  Rows without tokens are zero.

        What a row sees is cut by all rows of the plan: outputs of one row alone and in a batch agree to
        roundings, not bit for bit.  Values are exact codes, as in run(); weights keep 22 bits there and for segments of
        up to 16 query rows here, fp16's 11 for wider ones.
        A captured graph reads the plan's arrays and the rotation tables of the positions up to
        pool.max_position as they were: keep the plan while it is replayed, and capture again, after a call
        outside of a capture, once a token of a larger position is stored."""
        lib = _lib.load()
        pool = plan.pool
        if not query.is_cuda:
            _lib.require_device(query, "query")
        shape, dtype, dev = query.shape, query.dtype, pool.device
        if query.device != dev:
            raise ValueError(f"query is on {query.device}, the pool on {dev}")
        if len(shape) != 3 or shape[0] != plan.batch or shape[2] != pool.head_dim:
            raise ValueError(f"query must be (batch={plan.batch}, num_heads, head_dim={pool.head_dim}), got "
                             f"{tuple(shape)}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"run_shared takes fp16 or bf16 queries, got {dtype}; run() takes fp32 ones")
        if query.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("run_shared has no backward pass; call it under torch.no_grad()")
        hq = shape[1]
        ints, counts, places, factors, nbytes = plan._work.get(hq) or plan.work(hq)
        if not 0 <= int(layer) < pool.num_layers:
            raise ValueError(f"layer {layer} of a pool of {pool.num_layers}")
        if pool.head_dim != self.compressor.head_dim:
            raise ValueError(f"pool head_dim {pool.head_dim} != compressor head_dim {self.compressor.head_dim}")
        q = query.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != shape or out.dtype != dtype or out.device != dev or not out.is_contiguous() or out.data_ptr() % 8:
            raise ValueError(f"out must be a contiguous, 8-byte aligned {dtype} tensor {tuple(shape)} on {dev}")
        # of this call alone: calls on other streams and captured graphs have their own
        ws = torch.empty(nbytes or 16, dtype=torch.uint8, device=dev)
        tables = self._shared_tables(pool.max_position, dev)
        dm, dp, n_pos = plan.reads(tables)
        items, pages, seg_rows, row_slots = places
        with on_device(dev):
            base = ints.address()
            st = lib.nq_shared_attention(_SHARED_PACK.pack(
                pool.desc_at, int(layer), shape[0], hq, _lib.NQ_F16 if dtype == torch.float16 else _lib.NQ_BF16, *counts,
                q.data_ptr(), out.data_ptr(), base + items, base + pages, base + seg_rows, base + row_slots, dm, dp, n_pos,
                *factors, ws.data_ptr(), nbytes), tables.read_on(dev))
        _lib.check(st, "nq_shared_attention")
        return out

    def forward(self, query: torch.Tensor, compressed_key_cache: dict, compressed_value_cache: dict,
                block_tables: List[List[int]], context_lens: torch.Tensor) -> torch.Tensor:
        """(batch, num_heads, head_dim) attended output, the query's dtype (fp16-rounded values)."""
        plan = self.plan(compressed_key_cache, block_tables, context_lens)
        return self.run(plan, query)

    @staticmethod
    def _infer_block_size(slot_mapping: torch.Tensor) -> int:
        """The reference's heuristic (vllm_backend.py:775-786), kept as is: the first
        candidate always passes, so it returns 4 for any non-empty mapping."""
        if slot_mapping.numel() == 0:
            return 16
        for bs in [4, 8, 16, 32]:
            if (slot_mapping % bs).max() < bs:
                return bs
        return 16
