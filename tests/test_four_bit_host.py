"""The work lists of attention over a cache in 4 bits, page numbers, and the C entry points' refusals, without a GPU."""

import ctypes
import random

import numpy as np
import pytest
import torch

from nexusquant_amd import _lib, four_bit
from oracle import four_bit as ref
from test_rotary_host import check_written_tensors_are_seen


def replay(pages, lengths, queries, causal, window, group, heads, d):
    """Every row's tokens and slots as the kernels go through the lists."""
    lib = _lib.load()
    most = [lib.nq_fourbit_rows(d, k) for k in range(3)]
    (items, joins), (*n_items, n_joins, n_slots, most_chunks) = four_bit.attention_items(pages, lengths, queries, causal, window, group,
                                                                                               heads, d, most)
    items, joins = items.reshape(-1, 12), joins.reshape(-1, 4)
    assert len(items) == sum(n_items) and len(joins) == n_joins
    kinds = np.repeat([0, 1, 2], n_items)
    first_row = np.concatenate([[0], np.cumsum(queries)])
    first_page = np.concatenate([[0], np.cumsum(pages)])
    seen = {}      # (query row, head in group): how often each token
    written = {}   # slot, head in group
    direct = set()  # (query row, head in group) without a join
    for k, it in enumerate(items):
        page, tok0, n_tok, q_row0, r0, n_rows, slot0, slots, last = it[:9].tolist()
        assert 1 <= n_rows <= most[kinds[k]] and n_tok >= 1
        b = next(b for b in range(len(lengths)) if queries[b] and first_row[b] == q_row0)
        assert first_page[b] == page and 0 <= tok0 and tok0 + n_tok <= lengths[b]
        for r in range(r0, r0 + n_rows):
            i, h = divmod(r, group)
            assert i < queries[b]
            hi = last + (i if causal else 0)
            lo = max(hi - window + 1, 0) if window else 0
            got = seen.setdefault((q_row0 + i, h), np.zeros(lengths[b], int))
            got[max(lo, tok0):min(hi + 1, tok0 + n_tok)] += 1
            if slots == 0:
                assert (q_row0 + i, h) not in direct
                direct.add((q_row0 + i, h))
                continue
            slot = slot0 + i * slots
            assert 0 <= slot < n_slots and (slot, h) not in written
            written[slot, h] = q_row0 + i
    joined = set()
    for row, at, c, _ in joins.tolist():
        assert row not in joined
        joined.add(row)
        for s in range(at, at + c):
            assert all(written[s, h] == row for h in range(group))
    assert sum(c for _, _, c, _ in joins.tolist()) * group == len(written) and all(c <= most_chunks for _, _, c, _ in joins.tolist())
    rows = {(r, h) for r in joined for h in range(group)}
    assert not rows & direct and rows | direct == {(r, h) for r in range(sum(queries)) for h in range(group)}
    for b, (n, q) in enumerate(zip(lengths, queries)):
        mask = ref.seen(n, q, causal, window).numpy() if n else None
        for i in range(q):
            for h in range(group):
                got = seen.get((first_row[b] + i, h))
                assert (got is None) if not n else np.array_equal(got, mask[i].astype(int)), (b, i, h)


@pytest.mark.parametrize("seed", range(30))
def test_every_row_sees_its_tokens_once(seed):
    r = random.Random(seed)
    group, heads, d = r.choice([1, 2, 3, 4, 8, 16, 17, 130, 300]), r.choice([1, 2, 8, 40]), r.choice([64, 128, 256])
    causal = r.random() < 0.6
    lengths = [r.choice([0, 1, r.randint(1, 60), r.randint(1, 1500)]) for _ in range(r.randint(1, 5))]
    queries = [r.choice([0, 1, 1, r.randint(1, 9), r.randint(1, 300 if group < 16 else 5)]) for _ in lengths]
    if causal:
        queries = [min(q, n) if n else q for q, n in zip(queries, lengths)]
    window = r.choice([0, 0, 1, r.randint(1, 100)]) if causal else 0
    replay([-(-n // 16) for n in lengths], lengths, queries, causal, window, group, heads, d)


def test_long_sequences_and_many():
    replay([8192], [131072], [1], True, 0, 8, 8, 128)
    replay([512] * 3, [8192] * 3, [200, 1, 3], True, 0, 2, 8, 128)
    replay([32] * 64, [500] * 64, [1] * 64, True, 0, 4, 8, 128)
    replay([], [], [], True, 0, 4, 8, 128)
    replay([0], [0], [3], True, 0, 4, 8, 128)


def test_ragged_prompts_are_cut_at_the_share():
    """Long and short sequences of many rows: some are cut, unevenly, others whole."""
    for lengths, queries, group, heads, d, causal in (([16384, 8371, 11749, 951], [51, 35, 11, 3], 40, 8, 128, True),
                                                      ([9000, 3000, 5000, 640], [130, 300, 97, 200], 2, 4, 256, False),
                                                      ([20000, 100], [70, 20], 8, 100, 64, True), ([4000] * 9, [64] * 9, 16, 400, 64, True)):
        replay([-(-n // 16) for n in lengths], lengths, queries, causal, 0, group, heads, d)


def cpu_pool(pages=6, heads=2, tokens=16, d=128, layers=1):
    """A pool without a device, for what is checked before one is needed."""
    pool = four_bit.FourBitPagePool.__new__(four_bit.FourBitPagePool)
    shape = (layers, pages, heads, tokens)
    pool._adopt(*(torch.zeros(shape + (d // 2,), dtype=torch.uint8) for _ in range(2)),
                *(torch.zeros(shape, dtype=torch.float16) for _ in range(2)))
    return pool


def test_pool_shapes():
    pool = cpu_pool()
    assert (pool.head_dim, pool.page_tokens, pool.num_heads, pool.num_pages, pool.free_pages) == (128, 16, 2, 6, 6)
    assert pool.desc.head_dim == 128 and pool.desc.reserved == 4 and not pool.desc.positions
    with pytest.raises(ValueError, match="positive"):
        four_bit.FourBitPagePool(0, 2, 16, 128)
    with pytest.raises(_lib.NexusQuantError):
        four_bit.FourBitPagePool(4, 2, 16, 128, device="cpu")
    for shape, d in (((1, 4, 2, 16), 96), ((1, 1 << 25, 8, 16), 128), ((65536, 1, 1, 1), 64), ((1, 1, 1 << 13, 1 << 13), 128)):
        with pytest.raises((ValueError, NotImplementedError)):
            four_bit.FourBitPagePool._check_shape(shape, d)
    with pytest.raises(_lib.NexusQuantError):
        z = torch.zeros(1, 2, 2, 16, 64, dtype=torch.uint8)
        s = torch.zeros(1, 2, 2, 16, dtype=torch.float16)
        four_bit.FourBitPagePool.from_tensors(z, z, s, s)
    with pytest.raises(TypeError):
        four_bit.FourBitPagePool.from_tensors(z.to(torch.int8), z, s, s)
    with pytest.raises(ValueError):
        four_bit.FourBitPagePool.from_tensors(z[..., ::2], z, s, s)


def test_plans_check_page_numbers():
    pool = cpu_pool()
    t = pool.allocate(2)
    for tables, lengths in (([t], [33]), ([t], [-1]), ([[4]], [3]), ([t], [3, 4]), ([[99]], [3])):
        with pytest.raises(ValueError):
            pool.plan_attention(tables, lengths)
    with pytest.raises(ValueError):
        pool.plan_attention([t], [20], [21])
    with pytest.raises(ValueError):
        pool.plan_attention([t], [20], causal=False, sliding_window=3)
    plan = pool.plan_attention([t + [77]], [20], [3], sliding_window=20)
    assert plan.rows == 3 and plan.window == 0 and plan._tables[0].tolist() == t
    for bad in ([0, 0], [96], [40], [0.5]):
        with pytest.raises(ValueError):
            pool.plan_slots(bad)


def test_references_are_counted_as_changes():
    pool = cpu_pool()
    seen = [pool._changes]

    def changed():
        seen.append(pool._changes)
        return seen[-1] != seen[-2]

    t = pool.allocate(2)
    assert changed()
    pool.retain(t)
    assert changed()
    pool.free(t)
    assert changed()
    pool.fork(t, 32, n=1)
    assert changed()


def test_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    at = 4096

    def c_pool(**kw):
        f = dict(layers=2, pages=4, heads=2, tokens=16, head_dim=128, reserved=4, key_codes=at, value_codes=at, key_scales=at, value_scales=at)
        return _lib.Pool(**{**f, **kw})

    def append(pool=None, layer=0, rows=3, hq=2, dtype=0, q=at, k=at, v=at, out=at, angles=at, slots=at, strides=(256, 128) * 4):
        pool = c_pool() if pool is None else pool
        return lib.nq_fourbit_append(four_bit._APPEND_PACK.pack(ctypes.addressof(pool), layer, rows, hq, dtype, q, k, v, out, angles,
                                                                slots, *strides, 1.0, 0), None)

    def read(pool=None, layer=0, slots=at, n=3, dtype=0, keys=at, values=at):
        return lib.nq_fourbit_read(c_pool() if pool is None else pool, layer, slots, n, dtype, 1.0, keys, values, None)

    def attend(pool=None, layer=0, hq=4, dtype=0, counts=(1, 1, 1, 1, 2), window=0, scale=0.1, q=at, out=at, items=at, pages=at, joins=at,
               strides=(512, 128) * 2, ws=at, nbytes=1 << 20):
        pool = c_pool() if pool is None else pool
        return lib.nq_fourbit_attention(four_bit._ATTEND_PACK.pack(
            ctypes.addressof(pool), layer, hq, dtype, *counts, 1, window, scale, 0.1, 0, q, out, items, pages, joins, *strides, ws, nbytes), None)

    assert lib.nq_fourbit_append(None, None) == lib.nq_fourbit_attention(None, None) == -1
    for kw in (dict(head_dim=96), dict(layers=0), dict(pages=0), dict(heads=-1), dict(tokens=0), dict(key_codes=None),
               dict(value_scales=None), dict(key_codes=at + 8), dict(pages=1 << 27), dict(reserved=0), dict(reserved=8)):
        for call in (append, read, attend):
            assert call(pool=c_pool(**kw)) == -1, kw
    for call in (append, read, attend):
        assert call(layer=2) == call(layer=-1) == -1
    for kw in (dict(rows=-1), dict(hq=-1), dict(dtype=2), dict(k=0), dict(v=0), dict(slots=0), dict(q=0), dict(out=0), dict(angles=0),
               dict(k=at + 2), dict(out=at + 8), dict(angles=at + 4), dict(strides=(256, 124) + (256, 128) * 3)):
        assert append(**kw) == -1, kw
    for kw in (dict(slots=0), dict(n=-1), dict(dtype=3), dict(keys=0), dict(values=0), dict(values=at + 8), dict(n=(1 << 31) - 1)):
        assert read(**kw) == -1, kw
    for kw in (dict(hq=0), dict(hq=3), dict(dtype=2), dict(counts=(-1, 1, 1, 1, 1)), dict(counts=(1, 1, -1, 1, 1)), dict(counts=(1, 1, 1, -1, 1)), dict(window=-1),
               dict(scale=0.0), dict(scale=float("nan")), dict(q=0), dict(out=0), dict(items=0), dict(pages=0), dict(joins=0), dict(q=at + 8),
               dict(out=at + 4), dict(strides=(512, 124, 512, 128)), dict(strides=(512, 128, 512, 126)), dict(ws=0), dict(nbytes=16),
               dict(ws=at + 8), dict(counts=(1 << 30, 1 << 30, 1, 1, 1)), dict(counts=(1, 1, 1, 1 << 28, 1))):
        assert attend(**kw) == -1, kw
    assert append(rows=0) == read(n=0) == attend(counts=(0, 0, 0, 0, 0)) == 0
    # pools of the other kind
    assert lib.nq_pool_compact(c_pool(), at, 100, 0, 1, 1, at, 8, 1, None) == -1 and b"renumber" in lib.nq_last_error()
    assert lib.nq_pool_write(c_pool(), 0, c_pool(), at, 0, 3, None) == -1


def test_descriptors_match_the_c_compiler(tmp_path):
    """The packed formats' sizes and the places of their last fields equal gcc's on the header."""
    import os
    import subprocess
    from nexusquant_amd import rotary
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "nexusquant_amd.h")
    fields = [("nq_rotate_desc", "k_out_stride", rotary._PACK), ("nq_fourbit_append_desc", "hadamard_scale", four_bit._APPEND_PACK),
              ("nq_fourbit_append_desc", "q_stride", None), ("nq_fourbit_desc", "query", None), ("nq_fourbit_desc", "workspace_bytes", four_bit._ATTEND_PACK)]
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{header}"\nint main(void){{' + "".join(
        f'printf("%zu %zu\\n", sizeof({s}), offsetof({s}, {f}));' for s, f, _ in fields) + "return 0;}")
    subprocess.check_call(["gcc", "-o", str(tmp_path / "layout"), str(src)])
    out = [tuple(int(x) for x in line.split()) for line in subprocess.check_output([str(tmp_path / "layout")]).decode().splitlines()]
    assert all(size == pack.size for (size, _), (_, _, pack) in zip(out, fields) if pack is not None)
    import struct
    assert out[0][1] == struct.calcsize("6i5P6q") and out[1][1] == struct.calcsize("P4i6P8q") and out[2][1] == struct.calcsize("P4i6P")
    assert out[3][1] == struct.calcsize("P10i2fi") + (-struct.calcsize("P10i2fi")) % 8 and out[4][1] == struct.calcsize("P10i2fi5P4qP")


def no_launch(monkeypatch):
    """What a pool of the host gets as far as the launch with; calls are counted."""
    import contextlib

    class Lib:
        launched = 0

        def __getattr__(self, name):
            if name.startswith("nq_fourbit_r") or name.endswith("workspace"):
                return getattr(real, name)
            return self.launch

        def launch(self, *args):
            Lib.launched += 1
            return 0

    class Ints:
        def __init__(self, values, device):
            pass

        def address(self):
            return 4096

    real = _lib.load()
    monkeypatch.setattr(_lib, "load", Lib)
    monkeypatch.setattr(_lib, "current_stream_handle", lambda dev: None)
    monkeypatch.setattr(four_bit, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(four_bit, "PlanTensor", Ints)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return Lib


def host_step(pool):
    """Plans of two tokens of a sequence of 20, their rotation, and tensors for them."""
    from nexusquant_amd.rotary import Rotation
    t = pool.allocate(2)
    rotation = Rotation(angles=torch.zeros(2, 2, 64), rows=2, head_dim=128)
    q, k, v = (torch.randn(2, h, 128).half() for h in (4, 2, 2))
    return pool.plan_slots(pool.slots(t, 18, 20)), pool.plan_attention([t], [20], [2]), rotation, q, k, v


def test_tensors_with_tangents_are_refused(monkeypatch):
    from torch.autograd import forward_ad
    lib, pool = no_launch(monkeypatch), cpu_pool()
    slots, plan, rotation, q, k, v = host_step(pool)
    for grads in (False, True):
        with torch.set_grad_enabled(grads), forward_ad.dual_level():
            pool.append(slots, k, v, rotation=rotation, query=q)
            pool.attend(plan, q)
            launched = lib.launched
            dq, dk, dv = (forward_ad.make_dual(x, torch.ones_like(x)) for x in (q, k, v))
            for args in ((dk, v, q), (k, dv, q), (k, v, dq)):
                with pytest.raises(NotImplementedError, match="forward mode"):
                    pool.append(slots, *args[:2], rotation=rotation, query=args[2])
            with pytest.raises(NotImplementedError, match="forward mode"):
                pool.attend(plan, dq)
            assert lib.launched == launched
    assert launched == 4


def test_writes_in_place_are_seen_by_autograd(monkeypatch):
    no_launch(monkeypatch)
    pool = cpu_pool()
    slots, plan, rotation, q, k, v = host_step(pool)
    into = torch.empty_like(q)
    for out in (q, into):
        check_written_tensors_are_seen(lambda: pool.append(slots, k, v, rotation=rotation, query=q, out=out), out)
        check_written_tensors_are_seen(lambda: pool.attend(plan, q, out=out), out)
    versions = [x._version for x in (q, k, v)]
    pool.append(slots, k, v, rotation=rotation, query=q)
    pool.attend(plan, q)
    assert [x._version for x in (q, k, v)] == versions
    with torch.inference_mode():
        q = q.clone()
        pool.append(slots, k, v, rotation=rotation, query=q, out=q)
        pool.attend(plan, q, out=q)


def test_outputs_that_require_grad_or_have_tangents_are_refused(monkeypatch):
    from torch.autograd import forward_ad
    lib, pool = no_launch(monkeypatch), cpu_pool()
    slots, plan, rotation, q, k, v = host_step(pool)
    with forward_ad.dual_level():
        for out in (torch.empty_like(q).requires_grad_(), forward_ad.make_dual(torch.empty_like(q), torch.ones_like(q))):
            with pytest.raises(NotImplementedError):
                pool.append(slots, k, v, rotation=rotation, query=q, out=out)
            with pytest.raises(NotImplementedError):
                pool.attend(plan, q, out=out)
    assert lib.launched == 0
    with torch.no_grad():
        out = torch.empty_like(q).requires_grad_()
        assert pool.append(slots, k, v, rotation=rotation, query=q, out=out) is out and pool.attend(plan, q, out=out) is out


@pytest.mark.parametrize("reserved", [4, 8, -1, 1 << 20])
def test_pools_with_positions_are_taken_whatever_their_reserved_field_holds(reserved):
    """The field was not read before there were pools of 4 bits, which have no positions."""
    lib, at = _lib.load(), 4096
    pool = _lib.Pool(layers=2, pages=4, heads=2, tokens=16, head_dim=128, reserved=reserved, key_codes=at, value_codes=at, key_scales=at,
                     value_scales=at, positions=at)
    tokens = _lib.Pool(layers=1, pages=1, heads=2, tokens=3, head_dim=128, reserved=reserved, key_codes=at, value_codes=at, key_scales=at,
                       value_scales=at, positions=at)
    desc = _lib.SharedDesc(pool=ctypes.pointer(pool), q_heads=4, query=at, out=at, row_slots=at)
    assert lib.nq_shared_attention(ctypes.byref(desc), None) == 0
    pages = np.array([0, 1], np.int32)
    assert lib.nq_pool_copy_pages(pool, pages.ctypes.data, pages.ctypes.data, 0, None) == 0
    # as without the field: refused by what comes after it
    assert lib.nq_pool_write(pool, 0, tokens, None, 0, 3, None) == -1 and b"slots are required" in lib.nq_last_error()
    assert lib.nq_pool_compact(pool, at, 100, 0, 1, 1, None, 8, 1, None) == -1 and b"kept list" in lib.nq_last_error()
    assert lib.nq_fourbit_read(pool, 0, at, 0, 0, 1.0, at, at, None) == -1 and b"8 bits" in lib.nq_last_error()
