"""A pool of equally sized compressed pages: allocated, shared, copied, compacted and freed.

The pages of vllm_backend.py (int8 codes 2p, fp16 scales, int32 positions; keys stored
without rotation) in one allocation a field, for all layers of a model, with a reference
count a page.  A sequence is a list of page numbers and a length; the same numbers hold in
every layer.

- fork: branches of a sequence share its full pages, a part-filled last page is copied
- copy_pages: whole pages, in every layer (nq_pool_copy_pages)
- compact: the tokens that a keep mask leaves, moved into fewer pages (nq_pool_compact);
  with renumber=True keys move to their new positions, as truncation re-rotates them
- write: new tokens encoded into their slots (nq_page_encode, nq_pool_write)
- free: references dropped; a page without any can be allocated again

Page numbers and counts are kept on the host (under a lock).  The device work runs on the
current stream of the pool's device: calls on one stream are in order, a user of several
streams orders them.  Decode attention over a pool: NexusQuantPagedAttention.plan_shared.
"""

from __future__ import annotations

import array
import ctypes
import struct
import threading
from typing import List, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .ops import _addr, on_device, to_device
from .vllm_backend import CompressedPage

_HEAD_DIMS = (64, 128, 256)
_FIELDS = ("key_codes", "value_codes", "key_scales", "value_scales", "positions")


def _refuse_capture(what: str, device: torch.device) -> None:
    if torch.cuda.is_initialized():
        with on_device(device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{what} changes the pool's host state and cannot be captured into a graph")


class PagePool:
    """The page numbers of a pool, their references, and its whole pages and tokens moved.

    What a page holds is the subclass's: it sets head_dim and calls _start with its fields, codes
    [layers, pages, heads, tokens, bytes] and scales [layers, pages, heads, tokens]."""

    def _start(self, key_codes, value_codes, key_scales, value_scales, positions, bits: int = 0) -> None:
        self.num_layers, self.num_pages, self.num_heads, self.page_tokens = key_codes.shape[:4]
        self.device = key_codes.device
        self._refs = np.zeros(self.num_pages, dtype=np.int32)
        self._changes = 0  # of the references
        self._stack = np.arange(self.num_pages - 1, -1, -1, dtype=np.int32)  # free pages, the next one last
        self._free = self.num_pages
        self._lock = threading.RLock()
        self.desc = _lib.Pool(layers=self.num_layers, pages=self.num_pages, heads=self.num_heads,
                              tokens=self.page_tokens, head_dim=self.head_dim, reserved=bits, key_codes=_addr(key_codes),
                              value_codes=_addr(value_codes), key_scales=_addr(key_scales),
                              value_scales=_addr(value_scales), positions=_addr(positions))
        self.desc_at = ctypes.addressof(self.desc)

    # ------------------------------------------------------------- page numbers

    @property
    def free_pages(self) -> int:
        return self._free

    def ref_count(self, page: int) -> int:
        return int(self._refs[self._pages([page])[0]])

    def pages_for(self, length: int) -> int:
        """Pages that `length` tokens take."""
        return -(-int(length) // self.page_tokens)

    def _pages(self, pages) -> np.ndarray:
        # a list of ints by way of struct: a third of numpy's own conversion time
        if type(pages) is list:
            try:
                p = np.frombuffer(struct.pack(f"{len(pages)}i", *pages), dtype=np.int32)
            except struct.error:
                raise ValueError(f"page numbers must be integers in [0, {self.num_pages})") from None
        else:
            p = np.asarray(pages).reshape(-1)
            if len(p) and p.dtype.kind not in "iu":
                raise ValueError(f"page numbers must be integers, got {p.dtype}")
            if len(p) and (p.min() < 0 or p.max() >= self.num_pages):
                raise ValueError(f"page numbers must lie in [0, {self.num_pages})")
            return p.astype(np.int32, copy=False)
        if len(p) and p.view(np.uint32).max() >= self.num_pages:  # a negative number is a large one as unsigned
            raise ValueError(f"page numbers must lie in [0, {self.num_pages})")
        return p

    def _referenced(self, p: np.ndarray, what: str) -> np.ndarray:
        refs = self._refs[p]
        if len(p) and refs.min() < 1:
            raise ValueError(f"{what}: page {int(p[refs < 1][0])} is not allocated")
        return refs

    def in_use(self, pages, what: str = "pages") -> np.ndarray:
        """The page numbers as an array; raises unless all are allocated."""
        p = self._pages(pages)
        self._referenced(p, what)
        return p

    def _tally(self, p: np.ndarray):
        """The pages in p, ascending and each once, and how often each is there."""
        if 8 * len(p) < self.num_pages:
            p, n = np.unique(p, return_counts=True)
            return p, n.astype(np.int32)
        n = np.bincount(p, minlength=self.num_pages)  # 7 us where sorting 6000 pages takes 53
        p = n.nonzero()[0]
        return p, n[p].astype(np.int32)

    def allocate(self, n: int) -> List[int]:
        """n pages with one reference each.  Their contents are whatever they last held."""
        n = int(n)
        if n < 0:
            raise ValueError(f"cannot allocate {n} pages")
        with self._lock:
            if n > self._free:
                raise _lib.NexusQuantError(f"{n} pages wanted, {self._free} of {self.num_pages} free")
            return self._take(n).tolist()

    def _take(self, n: int) -> np.ndarray:
        got = self._stack[self._free - n:self._free][::-1].copy()
        self._free -= n
        self._refs[got] = 1
        self._changes += 1
        return got

    def _drop(self, p: np.ndarray, n: np.ndarray) -> None:
        left = self._refs[p] - n
        if len(p) and left.min() < 0:
            raise ValueError(f"free: page {int(p[left < 0][0])} is not allocated, or freed more often than referenced")
        self._refs[p] = left
        self._changes += 1
        gone = p[left == 0][::-1]  # the lowest is allocated next
        self._stack[self._free:self._free + len(gone)] = gone
        self._free += len(gone)

    def retain(self, pages: Sequence[int]) -> None:
        """One more reference to each page (to a page listed twice: two)."""
        with self._lock:
            p, n = self._tally(self._pages(pages))
            self._refs[p] = self._referenced(p, "retain") + n
            self._changes += 1

    def free(self, pages: Sequence[int]) -> None:
        """Drop one reference of each page (of a page listed twice: two); pages without any can be
        allocated again.  Work already queued on the pool's stream still sees them as they were."""
        with self._lock:
            self._drop(*self._tally(self._pages(pages)))

    # --------------------------------------------------------------- page moves

    def _copy(self, src, dst) -> None:
        s, d = array.array("i", src), array.array("i", dst)  # read during the call
        lib = _lib.load()
        with on_device(self.device):
            st = lib.nq_pool_copy_pages(ctypes.byref(self.desc), s.buffer_info()[0], d.buffer_info()[0], len(s),
                                        ctypes.c_void_p(_lib.current_stream_handle(self.device)))
        _lib.check(st, "nq_pool_copy_pages")

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Page dst[i] becomes a copy of page src[i] in every layer, its positions too.

        A page may be read any number of times, written once, and not both; a page with more
        than one reference is not written (its other holders would see it change)."""
        with self._lock:
            s, d = self.in_use(src, "copy_pages"), self.in_use(dst, "copy_pages")
            if len(s) != len(d):
                raise ValueError(f"{len(s)} source pages for {len(d)} destinations")
            if len(d) and self._refs[d].max() > 1:
                raise ValueError(f"copy_pages: page {int(d[self._refs[d] > 1][0])} is shared and cannot be written")
            self._copy(s.tolist(), d.tolist())

    def fork(self, pages: Sequence[int], length: int, n: int = 1) -> List[List[int]]:
        """Page lists of n branches of the sequence (`pages` holding `length` tokens).

        Full pages are shared (one more reference a branch); a part-filled last page is copied
        for each branch, so that the sequence and its branches can all go on writing."""
        _refuse_capture("fork", self.device)
        with self._lock:
            n, length = int(n), int(length)
            if n < 0:
                raise ValueError(f"cannot fork {n} branches")
            p = self.in_use(pages, "fork")
            if length < 0 or self.pages_for(length) != len(p):
                raise ValueError(f"fork: {length} tokens take {self.pages_for(max(length, 0))} pages, got {len(p)}")
            table = p.tolist()  # plain integers, whatever the list held (a 0-d tensor equals no other in a set)
            if len(set(table)) != len(table):
                raise ValueError("fork: a page stands twice in one sequence")
            if length % self.page_tokens == 0:
                self._refs[p] += n
                self._changes += 1
                return [list(table) for _ in range(n)]
            last = self.allocate(n)
            try:
                self._copy([table[-1]] * n, last)
            except Exception:
                self.free(last)
                raise
            self._refs[p[:-1]] += n
            self._changes += 1
            return [table[:-1] + [x] for x in last]

    def compact(self, tables: Sequence[Sequence[int]], lengths: Sequence[int], kept_idx: torch.Tensor, n_kept,
                renumber: bool = False) -> Tuple[List[List[int]], List[int]]:
        """The kept tokens of each sequence in new pages; its old pages lose a reference.

        tables[b], lengths[b]: a sequence's pages and tokens.  kept_idx int32 [batch, >= most
        kept] and n_kept [batch] as ops.keep_mask returns them: row b starts with the n_kept[b]
        kept positions in their order (what follows is not read).  n_kept on the device is read
        back, since it says how many pages are needed; a list of ints is taken as it is.
        renumber=False: a token keeps its position (mask eviction); True: token j moves to
        position j, keys re-rotated (truncation).  Positions in the list must lie in their
        sequence (the kernel clamps them).  Needs the new pages free beside the old ones.
        Returns the new tables and lengths."""
        _refuse_capture("compact", self.device)
        lib = _lib.load()
        _lib.require_device(kept_idx, "kept_idx")
        if kept_idx.dtype != torch.int32 or kept_idx.dim() != 2:
            raise ValueError(f"kept_idx must be int32 [batch, tokens], got {kept_idx.dtype} {tuple(kept_idx.shape)}")
        if kept_idx.device != self.device:
            raise ValueError(f"kept_idx is on {kept_idx.device}, the pool on {self.device}")
        batch = len(tables)
        idx = kept_idx.contiguous()
        step = int(lib.nq_pool_move_tokens())
        with self._lock:
            # everything that does not need the counts comes before they are read back: the device is
            # busy with what was queued before
            had = [int(n) for n in lengths]
            sizes = [len(t) for t in tables]
            if not (len(had) == kept_idx.shape[0] == batch):
                raise ValueError(f"{batch} tables, {len(had)} lengths and {kept_idx.shape[0]} rows of kept_idx")
            for b in range(batch):
                if had[b] < 0 or self.pages_for(had[b]) != sizes[b]:
                    raise ValueError(f"compact: {had[b]} tokens take {self.pages_for(max(had[b], 0))} pages, "
                                     f"got {sizes[b]}")
            flat = self._pages([p for t in tables for p in t] if batch != 1 else tables[0])
            held, times = self._tally(flat)
            if (self._referenced(held, "compact") < times).any():
                raise ValueError("compact: a page stands in more tables than it has references")
            counts = [int(x) for x in (n_kept.tolist() if torch.is_tensor(n_kept) else n_kept)]
            if len(counts) != batch:
                raise ValueError(f"{len(counts)} counts for {batch} sequences")
            seq, tiles, ends = [], [], [0]
            n_tiles = start = 0
            for b, k in enumerate(counts):
                if not 0 <= k <= had[b] or k > idx.shape[1]:
                    raise ValueError(f"sequence {b} keeps {k} of {had[b]} tokens by a list of {idx.shape[1]}")
                seq += (n_tiles, k, had[b], start, len(flat) + ends[-1])
                tiles.append(-(-k // step))
                n_tiles += tiles[-1]
                start += sizes[b]
                ends.append(ends[-1] + self.pages_for(k))
            if ends[-1] > self._free:
                raise _lib.NexusQuantError(f"{ends[-1]} pages wanted, {self._free} of {self.num_pages} free")
            new = self._take(ends[-1])
            try:
                if n_tiles:
                    plan = np.concatenate([np.repeat(np.arange(batch, dtype=np.int32), tiles),
                                           np.array(seq, dtype=np.int32), flat, new])
                    host = len(plan) <= lib.nq_pool_host_ints()
                    if not host:
                        plan = to_device(plan, self.device)
                    with on_device(self.device):
                        st = lib.nq_pool_compact(ctypes.byref(self.desc), plan.ctypes.data if host else plan.data_ptr(),
                                                 len(plan), host, n_tiles, batch, _addr(idx), idx.shape[1],
                                                 int(bool(renumber)),
                                                 ctypes.c_void_p(_lib.current_stream_handle(self.device)))
                    _lib.check(st, "nq_pool_compact")
            except Exception:
                self._drop(*self._tally(new))
                raise
            self._drop(held, times)
            if renumber and counts:
                self.max_position = max(self.max_position, max(counts) - 1)
        got = new.tolist()
        return [got[a:b] for a, b in zip(ends, ends[1:])], counts

    def slots(self, pages: Sequence[int], start: int, stop: int) -> List[int]:
        """Slots (page * page_tokens + offset) of a sequence's tokens start .. stop - 1."""
        p = self._pages(pages)
        i = np.arange(int(start), int(stop))
        if len(i) and (i[0] < 0 or i[-1] >= len(p) * self.page_tokens):
            raise ValueError(f"tokens {start} .. {stop} do not lie in {len(p)} pages of {self.page_tokens}")
        return (p[i // self.page_tokens] * self.page_tokens + i % self.page_tokens).tolist()


class CompressedPagePool(PagePool):
    """num_pages pages of page_tokens tokens for num_heads kv heads, in num_layers layers.

    key_codes, value_codes    int8 [layers, pages, heads, tokens, head_dim]
    key_scales, value_scales  fp16 [layers, pages, heads, tokens]
    positions                 int32 [pages, tokens], shared by the layers
    max_position              no stored position is larger (write() keeps it; raise it
                              after writing into `positions` directly)
    """

    def __init__(self, num_pages: int, num_heads: int, page_tokens: int, head_dim: int, num_layers: int = 1,
                 device=None):
        shape = (int(num_layers), int(num_pages), int(num_heads), int(page_tokens))
        if min(shape) < 1:
            raise ValueError(f"layers, pages, heads and tokens must be positive (got {shape})")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise _lib.NexusQuantError(f"nexusquant_amd runs on MI355X (ROCm) devices only; the pool is on {dev}")
        self._check_shape(shape, int(head_dim))
        self._adopt(torch.zeros(shape + (int(head_dim),), dtype=torch.int8, device=dev),
                    torch.zeros(shape + (int(head_dim),), dtype=torch.int8, device=dev),
                    torch.zeros(shape, dtype=torch.float16, device=dev),
                    torch.zeros(shape, dtype=torch.float16, device=dev),
                    torch.zeros(shape[1], shape[3], dtype=torch.int32, device=dev))
        self.max_position = 0

    @classmethod
    def from_tensors(cls, key_codes: torch.Tensor, value_codes: torch.Tensor, key_scales: torch.Tensor,
                     value_scales: torch.Tensor, positions: torch.Tensor) -> "CompressedPagePool":
        """A pool over fields that exist already (used, not copied); all its pages are free.
        Reads the largest position back."""
        for name, t, dt, dims in (("key_codes", key_codes, torch.int8, 5), ("value_codes", value_codes, torch.int8, 5),
                                  ("key_scales", key_scales, torch.float16, 4),
                                  ("value_scales", value_scales, torch.float16, 4),
                                  ("positions", positions, torch.int32, 2)):
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
        if (value_codes.shape != key_codes.shape or tuple(key_scales.shape) != shape
                or tuple(value_scales.shape) != shape or tuple(positions.shape) != (shape[1], shape[3])):
            raise ValueError("fields must be [layers, pages, heads, tokens(, head_dim)] and [pages, tokens] of one shape")
        cls._check_shape(shape, key_codes.shape[4])
        lo, hi = torch.stack(torch.aminmax(positions)).tolist()
        if lo < 0:
            raise ValueError("positions must be non-negative")
        pool = cls.__new__(cls)
        pool._adopt(key_codes, value_codes, key_scales, value_scales, positions)
        pool.max_position = hi
        return pool

    @staticmethod
    def _check_shape(shape, head_dim: int) -> None:
        layers, pages, heads, tokens = shape
        if head_dim not in _HEAD_DIMS:
            raise NotImplementedError(f"head_dim {head_dim}: the gfx950 page kernels take 64, 128 or 256")
        if layers > 65535 or heads * tokens * head_dim >= 1 << 31 or pages * heads * tokens >= 1 << 31:
            raise ValueError("a pool takes 65535 layers, pages of less than 2^31 bytes of codes and less than 2^31 "
                             f"token rows a layer (got {shape})")

    def _adopt(self, key_codes, value_codes, key_scales, value_scales, positions) -> None:
        self.key_codes, self.value_codes = key_codes, value_codes
        self.key_scales, self.value_scales = key_scales, value_scales
        self.positions = positions
        self.head_dim = key_codes.shape[4]
        self._start(key_codes, value_codes, key_scales, value_scales, positions)

    # ------------------------------------------------------------------- tokens

    def write(self, compressor, slots: Sequence[int], keys: torch.Tensor, values: torch.Tensor, positions,
              layer: int = 0) -> None:
        """Encode tokens and store them in one layer: keys, values [tokens, heads, head_dim], keys rotated
        to `positions` [tokens]; token i goes to slots[i], -1 skips it (a padded batch), whatever its position.
        Slots are distinct and in pages of one reference."""
        _refuse_capture("write", self.device)
        lib = _lib.load()
        if compressor.head_dim != self.head_dim:
            raise ValueError(f"compressor head_dim {compressor.head_dim} != pool head_dim {self.head_dim}")
        if not 0 <= int(layer) < self.num_layers:
            raise ValueError(f"layer {layer} of a pool of {self.num_layers}")
        if keys.dim() != 3 or tuple(keys.shape[1:]) != (self.num_heads, self.head_dim) or values.shape != keys.shape:
            raise ValueError(f"keys and values must be (tokens, {self.num_heads}, {self.head_dim}), got "
                             f"{tuple(keys.shape)} / {tuple(values.shape)}")
        if keys.device != self.device or values.device != self.device:
            raise ValueError(f"keys are on {keys.device}, values on {values.device}, the pool on {self.device}")
        s = np.asarray(slots.tolist() if torch.is_tensor(slots) else slots).reshape(-1)
        if len(s) and s.dtype.kind not in "iu":
            raise ValueError(f"slots must be integers, got {s.dtype}")
        if len(s) and s.max() >= self.num_pages * self.page_tokens:  # (as the type they came in)
            raise ValueError(f"slots must lie below {self.num_pages * self.page_tokens}")
        s = s.astype(np.int64, copy=False)
        n = keys.shape[0]
        if len(s) != n:
            raise ValueError(f"{len(s)} slots for {n} tokens")
        used = s[s >= 0]
        if len(np.unique(used)) != len(used):
            raise ValueError("write: slots must be distinct")
        if n == 0:
            return
        if len(used) < n:  # padding: its positions, -1 or large ones among them, are nobody's
            pos = torch.as_tensor(positions).reshape(-1)
            if len(pos) == n:
                positions = pos.masked_fill(torch.from_numpy(s < 0).to(pos.device), 0)
        with self._lock:
            p = self.in_use(np.unique(used // self.page_tokens), "write")
            if len(p) and self._refs[p].max() > 1:
                raise ValueError(f"write: page {int(p[self._refs[p] > 1][0])} is shared and cannot be written")
            with torch.cuda.device(self.device):
                page = compressor.compress_page(keys.permute(1, 0, 2), values.permute(1, 0, 2), positions)
                host = n <= lib.nq_pool_host_ints()
                where = np.maximum(s, -1).astype(np.int32)
                if not host:
                    where = to_device(where, self.device)
                tokens = _lib.Pool(layers=1, pages=1, heads=self.num_heads, tokens=n, head_dim=self.head_dim,
                                   key_codes=_addr(page.key_codes), value_codes=_addr(page.value_codes),
                                   key_scales=_addr(page.key_scales), value_scales=_addr(page.value_scales),
                                   positions=_addr(page.positions))
                st = lib.nq_pool_write(ctypes.byref(self.desc), int(layer), ctypes.byref(tokens),
                                       where.ctypes.data if host else where.data_ptr(), host, n,
                                       ctypes.c_void_p(_lib.current_stream_handle(self.device)))
            _lib.check(st, "nq_pool_write")
            self.max_position = max(self.max_position, page.max_position or 0)

    def page(self, page: int, layer: int = 0) -> CompressedPage:
        """One page of a layer as a CompressedPage of page_tokens tokens (views, no copy), for
        NexusQuantKVCompressor and NexusQuantPagedAttention.plan."""
        i = int(self.in_use([page], "page")[0])
        return CompressedPage(key_codes=self.key_codes[layer, i], value_codes=self.value_codes[layer, i],
                              key_scales=self.key_scales[layer, i], value_scales=self.value_scales[layer, i],
                              positions=self.positions[i], num_valid=self.page_tokens, max_position=self.max_position)
