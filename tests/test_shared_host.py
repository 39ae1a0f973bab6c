"""Host side of decode attention over shared pages: segments, work lists and refusals, without a GPU."""

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from nexusquant_amd import _lib
from nexusquant_amd.vllm_backend import (_SHARED_PACK, NexusQuantKVCompressor, NexusQuantPagedAttention,
                                         SharedAttentionPlan, _SharedTables, shared_items, shared_segments)

from test_page_pool import c_pool, host_pool

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def pages_of(segments, batch, t):
    """Per row its (page, tokens) in order of the pages, from the segments."""
    got = [[] for _ in range(batch)]
    for rows, pages, n in segments:
        assert n > 0 and len(pages) >= -(-n // t)
        for b in rows:
            got[b] += [(int(p), min(t, n - i * t)) for i, p in enumerate(pages) if i * t < n]
    return got


def cases():
    a = list(range(100, 140))
    yield [a[:20], a[:20], a[:20]], [320, 320, 320], 16          # the same rows
    yield [a[:20] + [1], a[:20] + [2], a[:20] + [3, 4]], [323, 336, 340], 16
    yield [a[:20], a[:30], [7]], [311, 480, 5], 16               # the shared run ends in the shorter row's part page
    yield [a[:2] + [1], a[:2] + [2]], [48, 47], 16               # too little to share
    yield [a[:1] + a[10:30] + [1], a[:1] + a[10:30] + [2], a[:1] + [50, 51]], [340, 350, 40], 16  # nested
    yield [[], [3], []], [0, 1, 0], 16
    yield [a[:20] + a[20:40], a[:20] + a[20:40], a[:20] + [1], a[:20] + [2]], [640, 639, 330, 330], 16  # forks of forks
    yield [[5] * 1, [5] * 1], [1, 1], 1


@pytest.mark.parametrize("min_saved", [1, 256, 10 ** 9])
@pytest.mark.parametrize("tables,lengths,t", list(cases()))
def test_segments_hold_every_token_of_every_row_once(tables, lengths, t, min_saved):
    arr = [np.asarray(x[:-(-n // t)], dtype=np.int64) for x, n in zip(tables, lengths)]
    segs = shared_segments(arr, lengths, t, min_saved)
    got = pages_of(segs, len(tables), t)
    for b, n in enumerate(lengths):
        want = [(int(p), min(t, n - i * t)) for i, p in enumerate(arr[b])]
        assert sorted(got[b]) == sorted(want)
    for rows, pages, n in segs:
        if len(rows) > 1:
            assert n % t == 0 and (len(rows) - 1) * n >= min_saved


def test_what_is_shared_is_in_one_segment():
    a = np.arange(40)
    segs = shared_segments([np.r_[a, 50], np.r_[a, 51], np.r_[a, 52]], [650, 656, 641], 16, 256)
    assert sorted((rows, n) for rows, _, n in segs) == [([0], 10), ([0, 1, 2], 640), ([1], 16), ([2], 1)]
    # nested: a common start too short by itself goes along with what its branches share
    x, y = np.arange(100, 130), np.arange(200, 230)
    segs = shared_segments([np.r_[1, x], np.r_[1, x], np.r_[1, y], np.r_[1, y]], [496] * 4, 16, 256)
    assert sorted((rows, n) for rows, _, n in segs) == [([0, 1], 496), ([2, 3], 496)]


@pytest.mark.parametrize("heads,rows,tokens,pays", [(8, 32, 256, False), (8, 32, 272, True), (8, 9, 1024, True),
                                                    (8, 9, 1008, False), (16, 2, 4096, True), (16, 2, 4080, False)])
def test_what_pays_is_shared(monkeypatch, heads, rows, tokens, pays):
    pool = host_pool(monkeypatch, layers=1, pages=tokens // 16, heads=heads, tokens=16)
    table = pool.allocate(tokens // 16)
    attn = NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=64))
    assert len(attn.plan_shared(pool, [table] * rows, [tokens] * rows).segments) == (1 if pays else rows)
    assert len(attn.plan_shared(pool, [table] * rows, [tokens] * rows, min_saved=1).segments) == 1


def test_rows_that_end_one_after_another_are_cut_without_recursion():
    """2000 rows, each a page longer than the one before: a branch at every page."""
    pages = np.arange(2000)
    lengths = [i + 1 for i in range(2000)]
    segs = shared_segments([pages[:n] for n in lengths], lengths, 1, 1)
    seen = np.zeros(2000, dtype=int)
    for rows, seg_pages, n in segs:
        assert n == len(seg_pages)
        seen[rows] += n
    assert list(seen) == lengths and len(segs) == 2000


@pytest.mark.parametrize("group,kv_heads,d,cap,rows", [
    (1, 8, 128, 1024, (256, 128, 16)), (4, 1, 64, 1024, (256, 128, 16)), (128, 2, 256, 256, (128, 128, 16)),
    (8, 64, 128, 128, (256, 128, 16)), (2, 3, 128, 1024, (256, 128, 16)), (200, 1, 128, 2048, (256, 128, 16))])
def test_items_cover_each_rows_tokens_and_slots_once(group, kv_heads, d, cap, rows):
    r = np.random.RandomState(group)
    batch = 37
    segments = [(list(range(20)), np.arange(300), 4800), ([3, 5, 36], np.arange(400, 410), 160)]
    segments += [([b], np.arange(1000 + 10 * b, 1010 + 10 * b), int(r.randint(1, 160))) for b in range(30)]
    parts, n_items, n_many, n_few, n_slots = shared_items(segments, batch, group, kv_heads, d, [cap] * 3, rows)
    items = parts["items"].reshape(-1, 8)
    where = parts["seg_rows"].reshape(-1, 2)
    assert len(items) == n_items and parts["row_slots"][0] == 0 and parts["row_slots"][-1] == n_slots
    seen, slots = {}, []
    for i, (page0, tok0, n, row0, n_rows, chunk, few, _) in enumerate(items):
        most = rows[0 if i < n_many else 2 if few or i >= n_items - n_few else 1]
        assert 1 <= n <= cap and 1 <= n_rows and n_rows * group <= most
        for b, slot0 in where[row0:row0 + n_rows]:
            slots.append(slot0 + chunk)
            assert parts["row_slots"][b] <= slot0 + chunk < parts["row_slots"][b + 1]
            for t in range(tok0, tok0 + n):
                key = (int(b), int(parts["pages"][page0 + t // 16]), t % 16)
                assert key not in seen
                seen[key] = 1
    assert sorted(slots) == list(range(n_slots))
    assert len(seen) == sum(len(s[0]) * s[2] for s in segments)


@pytest.mark.parametrize("rows,group,tokens,kind", [(16, 8, 16384, 0), (16, 8, 4096, 1), (4, 8, 60000, 1), (32, 8, 128, 0),
                                                    (1, 200, 16, 0), (2, 8, 60000, 2), (16, 1, 16, 2), (17, 1, 16, 1)])
def test_which_kind_a_segment_is(rows, group, tokens, kind):
    segments = [(list(range(rows)), np.arange(tokens // 16), tokens)]
    _, n_items, n_many, n_few, _ = shared_items(segments, rows, group, 8, 128, (2048, 1024, 1024), (256, 128, 16))
    assert (n_many, n_items - n_many - n_few, n_few) == tuple(n_items if k == kind else 0 for k in range(3))


@pytest.mark.parametrize("rows,own,together", [(32, 256, True), (32, 1024, False), (300, 1, False)])
def test_few_go_along_with_some(rows, own, together):
    segments = [(list(range(16)), np.arange(64), 1024)]
    segments += [([b], np.arange(100, 100 + -(-own // 16)), own) for b in range(rows)]
    parts, n_items, n_many, n_few, _ = shared_items(segments, rows, 8, 8, 128, (2048, 1024, 1024), (256, 128, 16))
    flagged = parts["items"].reshape(-1, 8)[:, 6]
    assert n_many == 0 and (n_few == 0) == together
    assert flagged.sum() == (n_items - (flagged == 0).sum() if together else 0) and (flagged.any() == together)


def test_no_rows_and_no_tokens():
    parts, *counts = shared_items([], 3, 4, 8, 128, (2048, 1024, 1024), (256, 128, 16))
    assert counts == [0, 0, 0, 0] and list(parts["row_slots"]) == [0, 0, 0, 0]


def test_plan_refuses_bad_tables(monkeypatch):
    pool = host_pool(monkeypatch, d=64)
    attn = NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=64))
    a = pool.allocate(4)
    assert sorted(s[2] for s in attn.plan_shared(pool, [a, a[:1], []], [16, 3, 0]).segments) == [3, 16]
    # a rectangular table: what stands behind a row's tokens is padding
    padded = np.array([a, a[:1] + [-1, 0, 99], [-1] * 4])
    assert sorted(s[2] for s in attn.plan_shared(pool, padded, [16, 4, 0]).segments) == [4, 16]
    assert sorted(s[2] for s in attn.plan_shared(pool, torch.from_numpy(padded), torch.tensor([16, 4, 0])).segments) == [4, 16]
    for tables, ctx in ((padded, [16, 5, 0]), ([[0.5]], [1]), ([np.array([0.5])], [1])):
        with pytest.raises(ValueError):
            attn.plan_shared(pool, tables, ctx)
    for tables, ctx in (([a], [17]), ([a], [-1]), ([[9]], [1]), ([a, a], [4]), ([[99]], [1])):
        with pytest.raises(ValueError):
            attn.plan_shared(pool, tables, ctx)
    with pytest.raises(ValueError):
        NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=128)).plan_shared(pool, [a], [3])
    with pytest.raises(_lib.NexusQuantError):
        attn.run_shared(SharedAttentionPlan(pool, 1, []), torch.zeros(1, 3, 64))


def test_rotation_tables_are_kept_by_device_and_grow(monkeypatch):
    attn = NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=64))
    made = []

    def tables(max_position, dev):
        made.append((max_position, dev))
        n = -(-(max_position + 1) // 4096) * 4096
        return None, None, torch.zeros(n, 1), torch.zeros(n, 1)
    monkeypatch.setattr(attn.compressor, "_tables", tables)
    a, b = torch.device("cuda", 0), torch.device("cuda", 1)
    one, two = attn._shared_tables(100, a), attn._shared_tables(4095, b)
    for _ in range(3):  # pools on two devices in turn
        assert attn._shared_tables(4095, a) is one and attn._shared_tables(7, b) is two
    assert len(made) == 2 and one.args[2] == 4096
    assert attn._shared_tables(4096, a).args[2] == 8192 and attn._shared_tables(5000, a).args[2] == 8192
    assert len(made) == 3


def test_rotation_tables_are_the_compressors(monkeypatch):
    """Another compressor on the same attention, and another base of the same one: their tables, as run() reads them."""
    from nexusquant_amd.rope import device_merged_table
    attn = NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=64, rope_base=10000.0))
    cpu = torch.device("cpu")

    def is_of(tables, d, base):
        return all(torch.equal(a, b) for a, b in zip(tables.tensors, device_merged_table(4096, d, base, None, cpu)))
    first = attn._shared_tables(100, cpu)
    assert is_of(first, 64, 10000.0)
    attn.compressor = NexusQuantKVCompressor(head_dim=64, rope_base=500000.0)
    assert is_of(attn._shared_tables(100, cpu), 64, 500000.0)
    attn.compressor.rope_base = 1000000.0
    assert is_of(attn._shared_tables(100, cpu), 64, 1000000.0)
    attn.compressor = NexusQuantKVCompressor(head_dim=128, rope_base=10000.0)
    assert is_of(attn._shared_tables(100, cpu), 128, 10000.0)
    attn.compressor = NexusQuantKVCompressor(head_dim=64, rope_base=10000.0)
    assert attn._shared_tables(100, cpu) is first


def test_rotation_tables_are_recorded_on_the_streams_that_read_them(monkeypatch):
    """Dropped tables (longer ones took their place) must outlive what other streams had queued; once a stream will do."""
    class Table:
        shape = (4096, 32)
        seen = None

        def data_ptr(self):
            return 4096

        def record_stream(self, stream):
            self.seen = (self.seen or []) + [stream]
    now, capturing = [7], [False]
    monkeypatch.setattr(_lib, "current_stream_handle", lambda dev: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: f"stream {now[0]}")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    tables = _SharedTables(Table(), Table())
    for now[0] in (7, 9, 7, 9):
        assert tables.read_on(torch.device("cuda", 0)) == now[0]
    now[0], capturing[0] = 11, True  # a capture: the graph's plan keeps the tables
    assert tables.read_on(torch.device("cuda", 0)) == 11
    assert all(t.seen == ["stream 7", "stream 9"] for t in tables.tensors)
    capturing[0] = False
    tables.read_on(torch.device("cuda", 0))
    assert all(t.seen == ["stream 7", "stream 9", "stream 11"] for t in tables.tensors)


def test_a_plan_keeps_each_table_once():
    """Two attentions (local and global rotation bases) that use one plan in turn: a table for each, not for each call."""
    plan = SharedAttentionPlan(None, 1, [])
    one, two = (_SharedTables(torch.zeros(4096, 1), torch.zeros(4096, 1)) for _ in range(2))
    for _ in range(50):
        assert plan.reads(one) == one.args and plan.reads(two) == two.args
    assert list(plan._tables.values()) == [one, two]


def test_shared_struct_matches_the_c_compiler(tmp_path):
    names = [f[0] for f in _lib.SharedDesc._fields_]
    prog = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{ROOT}/include/nexusquant_amd.h"', "int main(void){",
            'printf("%zu\\n", sizeof(nq_shared_desc));']
    prog += [f'printf("%zu\\n", offsetof(nq_shared_desc, {f}));' for f in names] + ["return 0;}"]
    (tmp_path / "p.c").write_text("\n".join(prog))
    subprocess.check_call(["gcc", "-o", str(tmp_path / "p"), str(tmp_path / "p.c")])
    out = [int(x) for x in subprocess.check_output([str(tmp_path / "p")]).split()]
    assert _SHARED_PACK.size == ctypes.sizeof(_lib.SharedDesc)
    assert out == [ctypes.sizeof(_lib.SharedDesc)] + [getattr(_lib.SharedDesc, f).offset for f in names]


@pytest.mark.parametrize("kw,pool_kw", [
    (dict(layer=1), {}), (dict(layer=-1), {}), (dict(batch=-1), {}), (dict(q_heads=0), {}), (dict(q_heads=3), {}),
    (dict(q_heads=2 * 257), {}), (dict(q_dtype=_lib.NQ_F32), {}), (dict(n_items=-1), {}), (dict(n_slots=0), {}), (dict(n_many=2), {}), (dict(n_many=-1), {}),
    (dict(n_few=2), {}), (dict(n_few=-1), {}), (dict(n_few=1, n_many=1), {}), (dict(n_few=1, q_heads=34), {}),
    (dict(query=None), {}), (dict(query=ctypes.c_void_p(4104)), {}), (dict(out=None), {}), (dict(out=ctypes.c_void_p(4100)), {}), (dict(items=None), {}),
    (dict(row_slots=None), {}), (dict(rope_sin_minus_cos=None), {}), (dict(rope_n_pos=0), {}),
    (dict(workspace=None), {}), (dict(workspace_bytes=100), {}), (dict(workspace=ctypes.c_void_p(4100)), {}),
    (dict(scale_divisor=0.0), {}), (dict(n_items=1 << 30), {}), (dict(batch=1 << 30), {}),
    ({}, dict(head_dim=96)), ({}, dict(heads=0)), ({}, dict(pages=1 << 27)), ({}, dict(key_codes=None)),
    ({}, dict(value_codes=ctypes.c_void_p(4104)))])
def test_c_entry_refuses(kw, pool_kw):
    lib = _lib.load()
    dummy = ctypes.c_void_p(4096)
    base = dict(pool=ctypes.pointer(c_pool(**pool_kw)), layer=0, batch=2, q_heads=4, q_dtype=_lib.NQ_F16, n_items=1,
                n_slots=2, query=dummy, out=dummy, items=dummy, pages=dummy, seg_rows=dummy, row_slots=dummy,
                rope_sin_minus_cos=dummy, rope_cos_plus_sin=dummy, rope_n_pos=4096, hadamard_scale=0.1,
                scale_divisor=11.3, workspace=dummy, workspace_bytes=1 << 20)
    assert lib.nq_shared_attention(ctypes.byref(_lib.SharedDesc(**{**base, **kw})), None) == -1
    assert lib.nq_last_error().startswith(b"nq_shared_attention")
    assert lib.nq_shared_attention(ctypes.byref(_lib.SharedDesc(**{**base, "batch": 0})), None) in (0, -1)


def test_c_entry_refuses_groups_that_a_kind_does_not_take():
    lib = _lib.load()
    dummy = ctypes.c_void_p(4096)
    for n_many, n_few, group in ((1, 0, 129), (0, 2, 17), (1, 1, 17)):
        desc = dict(pool=ctypes.pointer(c_pool()), layer=0, batch=1, q_heads=c_pool().heads * group, q_dtype=_lib.NQ_F16,
                    n_items=2, n_many=n_many, n_few=n_few, n_slots=2, query=dummy, out=dummy, items=dummy, pages=dummy,
                    seg_rows=dummy, row_slots=dummy)
        assert lib.nq_shared_attention(ctypes.byref(_lib.SharedDesc(**desc)), None) == -1
        assert b"too many for items of kind" in lib.nq_last_error()
