"""The page pool's host side: page numbers, reference counts and refusals, without a GPU.

The pool is built over CPU tensors past its constructors (which refuse them); no call here
reaches a kernel: the C entry points refuse their arguments on the host, before the dummy
pointers are used."""

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from nexusquant_amd import _lib
from nexusquant_amd.page_pool import CompressedPagePool

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fields(layers=2, pages=10, heads=3, tokens=4, d=64):
    s = (layers, pages, heads, tokens)
    return (torch.zeros(s + (d,), dtype=torch.int8), torch.zeros(s + (d,), dtype=torch.int8),
            torch.zeros(s, dtype=torch.float16), torch.zeros(s, dtype=torch.float16),
            torch.zeros(pages, tokens, dtype=torch.int32))


def host_pool(monkeypatch, **kw):
    pool = CompressedPagePool.__new__(CompressedPagePool)
    pool._adopt(*fields(**kw))
    pool.max_position = 0
    pool.copied = []
    monkeypatch.setattr(pool, "_copy", lambda s, d: pool.copied.append((list(s), list(d))), raising=False)
    return pool


def test_pages_are_allocated_lowest_first_and_come_back(monkeypatch):
    pool = host_pool(monkeypatch)
    a = pool.allocate(3)
    assert a == [0, 1, 2] and pool.free_pages == 7
    assert pool.allocate(0) == []
    pool.free([1])
    assert pool.allocate(2) == [1, 3]
    pool.free([0, 1, 2, 3])
    assert pool.free_pages == 10 and pool.allocate(4) == [0, 1, 2, 3]


def test_references_keep_a_page(monkeypatch):
    pool = host_pool(monkeypatch)
    a = pool.allocate(2)
    pool.retain(a + [a[0]])
    assert pool.ref_count(a[0]) == 3 and pool.ref_count(a[1]) == 2
    pool.free([a[0], a[0], a[1]])
    assert pool.free_pages == 8
    pool.free(a)
    assert pool.free_pages == 10


def test_wrong_page_numbers_are_refused_and_change_nothing(monkeypatch):
    pool = host_pool(monkeypatch)
    a = pool.allocate(2)
    for call in (lambda: pool.free([a[0], a[0]]), lambda: pool.free([5]), lambda: pool.free([10]),
                 lambda: pool.free([-1]), lambda: pool.retain([7]), lambda: pool.copy_pages([0], [5]),
                 lambda: pool.copy_pages([0], [0, 1]), lambda: pool.page(9), lambda: pool.allocate(-1),
                 lambda: pool.slots(a, 0, 9), lambda: pool.slots(a, -1, 2), lambda: pool.free([1 << 40]),
                 lambda: pool.free([0.5]), lambda: pool.free(np.array([1 << 32])), lambda: pool.retain((-1,)),
                 lambda: pool.retain((0.5,)), lambda: pool.free(np.array([0.0]))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.NexusQuantError, match="8 of 10 free"):
        pool.allocate(9)
    assert pool.free_pages == 8 and pool.ref_count(0) == 1 and not pool.copied


def test_fork_shares_full_pages_and_copies_the_last(monkeypatch):
    pool = host_pool(monkeypatch)
    a = pool.allocate(3)
    assert pool.fork(a, 10, 2) == [[0, 1, 3], [0, 1, 4]]
    assert pool.copied == [([2, 2], [3, 4])]
    assert [pool.ref_count(x) for x in range(5)] == [3, 3, 1, 1, 1]
    assert pool.fork(a, 12) == [[0, 1, 2]] and pool.ref_count(2) == 2  # nothing part-filled: nothing copied
    assert len(pool.copied) == 1
    assert pool.fork([], 0, 2) == [[], []] and pool.fork(a, 10, 0) == []
    for pages, length in ((a, 8), (a, 13), (a[:2], 9), ([8], 1), (a, -1), ([0, 1, 1], 12)):
        with pytest.raises(ValueError):
            pool.fork(pages, length)
    with pytest.raises(ValueError, match="shared"):
        pool.copy_pages([4], [0])
    free = pool.free_pages
    with pytest.raises(_lib.NexusQuantError):
        pool.fork(a, 10, 6)
    assert pool.free_pages == free and pool.ref_count(0) == 4


def test_a_failed_copy_leaves_the_counts(monkeypatch):
    pool = host_pool(monkeypatch)
    a = pool.allocate(3)

    def fail(s, d):
        raise _lib.NexusQuantError("copy")
    monkeypatch.setattr(pool, "_copy", fail)
    with pytest.raises(_lib.NexusQuantError):
        pool.fork(a, 9, 2)
    assert pool.free_pages == 7 and pool.ref_count(0) == 1


def test_slots_follow_the_table(monkeypatch):
    pool = host_pool(monkeypatch)
    assert pool.slots([7, 2], 3, 6) == [31, 8, 9]
    assert pool.slots([7], 2, 2) == []


def test_constructors_refuse_what_the_kernels_do_not_take():
    with pytest.raises(_lib.NexusQuantError):
        CompressedPagePool(4, 2, 16, 128, device="cpu")
    with pytest.raises(NotImplementedError):
        CompressedPagePool(4, 2, 16, 96)
    with pytest.raises(ValueError):
        CompressedPagePool(0, 2, 16, 128)
    with pytest.raises(ValueError):
        CompressedPagePool(1 << 24, 8, 16, 128)
    with pytest.raises(_lib.NexusQuantError):
        CompressedPagePool.from_tensors(*fields())
    kc, vc, ks, vs, pos = fields()
    with pytest.raises(TypeError):
        CompressedPagePool.from_tensors(kc.int(), vc, ks, vs, pos)
    with pytest.raises(ValueError):
        CompressedPagePool.from_tensors(kc[:, ::2], vc, ks, vs, pos)


def test_pool_struct_matches_the_c_compiler(tmp_path):
    names = [f[0] for f in _lib.Pool._fields_]
    prog = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{ROOT}/include/nexusquant_amd.h"', "int main(void){",
            'printf("%zu\\n", sizeof(nq_pool));']
    prog += [f'printf("%zu\\n", offsetof(nq_pool, {f}));' for f in names] + ["return 0;}"]
    (tmp_path / "p.c").write_text("\n".join(prog))
    subprocess.check_call(["gcc", "-o", str(tmp_path / "p"), str(tmp_path / "p.c")])
    out = [int(x) for x in subprocess.check_output([str(tmp_path / "p")]).split()]
    assert out == [ctypes.sizeof(_lib.Pool)] + [getattr(_lib.Pool, f).offset for f in names]


def c_pool(**kw):
    dummy = ctypes.c_void_p(4096)
    base = dict(layers=1, pages=8, heads=2, tokens=16, head_dim=128, key_codes=dummy, value_codes=dummy,
                key_scales=dummy, value_scales=dummy, positions=dummy)
    return _lib.Pool(**{**base, **kw})


def ids(*x):
    a = np.array(x, dtype=np.int32)
    return a, a.ctypes.data


@pytest.mark.parametrize("src,dst,why", [((0,), (8,), b"not a page"), ((-1,), (1,), b"not a page"),
                                         ((0, 1), (2, 2), b"twice"), ((0, 2), (2, 3), b"reads a page"),
                                         ((1,), (1,), b"reads a page")])
def test_copy_refuses_bad_pairs_on_the_host(src, dst, why):
    lib = _lib.load()
    (_s, s), (_d, d) = ids(*src), ids(*dst)
    assert lib.nq_pool_copy_pages(ctypes.byref(c_pool()), s, d, len(src), None) == -1
    assert why in lib.nq_last_error()


def test_pool_entry_points_refuse_bad_geometry():
    lib = _lib.load()
    (_s, s) = ids(0)
    dummy = ctypes.c_void_p(4096)
    for kw in (dict(head_dim=96), dict(layers=0), dict(pages=0), dict(heads=-1), dict(tokens=0),
               dict(key_codes=None), dict(value_scales=None), dict(positions=None),
               dict(key_codes=ctypes.c_void_p(4104)), dict(layers=65536), dict(pages=1 << 27),
               dict(heads=1 << 14, tokens=1 << 14)):
        assert lib.nq_pool_copy_pages(ctypes.byref(c_pool(**kw)), s, s, 1, None) == -1, kw
        assert lib.nq_pool_compact(ctypes.byref(c_pool(**kw)), dummy, 100, 0, 1, 1, dummy, 8, 0, None) == -1, kw
        assert lib.nq_pool_write(ctypes.byref(c_pool(**kw)), 0, ctypes.byref(c_pool(pages=1)), dummy, 0, 16, None) == -1, kw
    ok = ctypes.byref(c_pool())
    assert lib.nq_pool_copy_pages(None, s, s, 1, None) == -1
    assert lib.nq_pool_copy_pages(ok, s, s, -1, None) == -1
    assert lib.nq_pool_copy_pages(ok, None, s, 1, None) == -1
    assert lib.nq_pool_copy_pages(ok, None, None, 0, None) == 0
    assert lib.nq_pool_compact(ok, None, 0, 0, 0, 0, None, 0, 0, None) == 0
    for kw in (dict(plan=None), dict(kept=None), dict(n_tiles=-1), dict(n_seq=0), dict(plan_ints=5), dict(stride=-1),
               dict(plan_ints=lib.nq_pool_host_ints() + 1, on_host=1)):
        x = {**dict(plan=dummy, plan_ints=100, on_host=0, n_tiles=1, n_seq=1, kept=dummy, stride=8), **kw}
        assert lib.nq_pool_compact(ok, *x.values(), 0, None) == -1, kw
        assert lib.nq_last_error().startswith(b"nq_pool_compact")
    one = ctypes.byref(c_pool(pages=1))
    assert lib.nq_pool_write(ok, 0, None, None, 0, 0, None) == 0
    assert lib.nq_pool_write(ok, 1, one, dummy, 0, 16, None) == -1       # no such layer
    assert lib.nq_pool_write(ok, 0, one, dummy, 0, 15, None) == -1       # not one page of n tokens
    assert lib.nq_pool_write(ok, 0, ctypes.byref(c_pool(pages=1, heads=4)), dummy, 0, 16, None) == -1
    assert lib.nq_pool_write(ok, 0, one, None, 0, 16, None) == -1


def test_write_refuses_slots_past_the_pool(monkeypatch):
    """Unsigned numbers past 2^63 among them: negative ones are skipped, and these are none."""
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor
    pool = host_pool(monkeypatch)
    pool.allocate(2)
    k = torch.zeros(2, 3, 64, dtype=torch.float16)
    for slots in (np.array([0, (1 << 64) - 1], dtype=np.uint64), [0, 40], torch.tensor([40, 0]), [0, 1 << 62]):
        with pytest.raises(ValueError, match="below 40"):
            pool.write(NexusQuantKVCompressor(head_dim=64), slots, k, k, [0, 1])
    with pytest.raises(ValueError, match="integers"):
        pool.write(NexusQuantKVCompressor(head_dim=64), [0, 1 << 64], k, k, [0, 1])


def test_fork_of_a_tables_row(monkeypatch):
    """list(block_table[b]): 0-d tensors, of which no two are equal in a set; numpy's integers."""
    pool = host_pool(monkeypatch)
    a = torch.tensor(pool.allocate(3), dtype=torch.int32)
    for row in (list(a), list(a.numpy()), a, a.numpy(), tuple(a.tolist())):
        kids = pool.fork(row, 10, 2)
        assert [x[:2] for x in kids] == [[0, 1]] * 2 and all(type(p) is int for x in kids for p in x)
        pool.free([p for x in kids for p in x])
    twice = [a[0], a[1], a[1].clone()]
    for row in (twice, [int(p) for p in twice]):
        with pytest.raises(ValueError, match="twice"):
            pool.fork(row, 12)
    assert [pool.ref_count(p) for p in range(3)] == [1, 1, 1] and pool.free_pages == 7


def test_a_capture_on_the_pools_device_is_seen_from_another_current_one(monkeypatch):
    """The launches go to the pool's device's current stream, so it is that one that may be capturing."""
    now = [0]

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.was, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.was
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)
    pool = host_pool(monkeypatch)
    a = pool.allocate(3)
    pool.device = torch.device("cuda", 1)
    for call in (lambda: pool.fork(a, 12), lambda: pool.compact([a], [12], torch.zeros(1, 12, dtype=torch.int32), [3]),
                 lambda: pool.write(None, [0], None, None, [0])):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    assert now == [0] and pool.free_pages == 7 and pool.ref_count(0) == 1
    pool.device = torch.device("cuda", 0)
    assert pool.fork(a, 12) == [a]
