"""Page moves of CompressedPagePool against numpy, byte for byte: copies, forks, compaction,
token writes, and the chain of them as a serving loop uses it.  Everything that a call does not
write must keep its bytes, so whole pools are compared."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FIELDS = ("key_codes", "value_codes", "key_scales", "value_scales", "positions")


def random_pool(layers, pages, heads, tokens, d, seed=0):
    from nexusquant_amd.page_pool import CompressedPagePool
    g = torch.Generator().manual_seed(seed)
    s = (layers, pages, heads, tokens)
    f = dict(key_codes=torch.randint(-8, 9, s + (d,), generator=g, dtype=torch.int8),
             value_codes=torch.randint(-8, 9, s + (d,), generator=g, dtype=torch.int8),
             key_scales=torch.rand(s, generator=g).half(), value_scales=torch.rand(s, generator=g).half(),
             positions=torch.randint(0, 5000, (pages, tokens), generator=g, dtype=torch.int32))
    return CompressedPagePool.from_tensors(**{k: v.to(DEV) for k, v in f.items()})


def snapshot(pool):
    torch.cuda.synchronize()
    return {k: getattr(pool, k).cpu().numpy().copy() for k in FIELDS}


def assert_same(pool, want):
    got = snapshot(pool)
    for k in FIELDS:
        assert np.array_equal(got[k].view(np.uint8), want[k].view(np.uint8)), k


def copy_np(f, src, dst):
    for k in FIELDS[:4]:
        f[k][:, dst] = f[k][:, src]
    f["positions"][dst] = f["positions"][src]


@pytest.mark.parametrize("layers,heads,tokens,d,n", [
    (1, 1, 1, 64, 1), (3, 1, 1, 64, 5),        # 2-byte scale pages
    (2, 2, 1, 64, 4), (2, 3, 24, 128, 7),      # 4- and 16-byte ones
    (1, 8, 16, 128, 1), (5, 4, 7, 256, 33),
    (2, 1, 2, 64, 449), (1, 1, 3, 64, 1000),   # past one launch's pairs
    (20, 8, 16, 128, 60), (10, 1, 25, 256, 300),  # past the caches
])
def test_copy_pages(layers, heads, tokens, d, n):
    print(f"[gpu] copy layers={layers} heads={heads} tokens={tokens} d={d} n={n}", flush=True)
    pool = random_pool(layers, 2 * n + 3, heads, tokens, d, seed=n)
    pool.allocate(2 * n + 3)
    perm = np.random.RandomState(n).permutation(2 * n + 3)
    src, dst = perm[:n].copy(), perm[n:2 * n]
    src[n // 2:] = src[:n - n // 2]  # pages that are read more than once
    want = snapshot(pool)
    copy_np(want, src, dst)
    pool.copy_pages(src.tolist(), dst.tolist())
    assert_same(pool, want)


def test_fork_and_free():
    print("[gpu] fork", flush=True)
    pool = random_pool(3, 20, 2, 16, 128)
    a = pool.allocate(4)
    want = snapshot(pool)
    kids = pool.fork(a, 50, 3)
    assert kids == [[0, 1, 2, 4], [0, 1, 2, 5], [0, 1, 2, 6]]
    copy_np(want, [3, 3, 3], [4, 5, 6])
    assert_same(pool, want)
    pool.free(a)
    assert pool.free_pages == 20 - 6 and pool.allocate(1) == [3]
    assert pool.fork(a[:3], 48, 2) == [a[:3], a[:3]]
    assert_same(pool, want)


def kept_list(lens, rate, width, seed):
    r = np.random.RandomState(seed)
    idx = np.full((len(lens), width), 1 << 30, dtype=np.int32)  # what follows the list is not read
    n_kept = []
    for b, n in enumerate(lens):
        k = int(round(n * (1 - rate)))
        idx[b, :k] = np.sort(r.permutation(n)[:k])
        n_kept.append(k)
    return idx, n_kept


def compact_np(f, tables, kept_idx, n_kept, new, t, renumber):
    old = {k: v.copy() for k, v in f.items()}
    for b, k in enumerate(n_kept):
        for j in range(k):
            i = kept_idx[b, j]
            sp, so, dp, do = tables[b][i // t], i % t, new[b][j // t], j % t
            for name in FIELDS[:4]:
                f[name][:, dp, :, do] = old[name][:, sp, :, so]
            f["positions"][dp, do] = j if renumber else old["positions"][sp, so]


@pytest.mark.parametrize("layers,heads,tokens,d,lens,rate,renumber", [
    (1, 1, 16, 64, [1], 0.0, False),
    (1, 2, 16, 128, [0, 5, 0], 0.5, False),               # empty sequences
    (2, 3, 7, 128, [63, 64, 65, 1], 0.0, True),           # pages off the tile grid, nothing evicted
    (2, 2, 16, 256, [130, 17], 1.0, True),                # nothing kept
    (3, 4, 24, 64, [200, 3, 129], 0.6, False),
    (1, 8, 64, 128, [1000], 0.75, True),
    (2, 1, 1, 64, [150, 70], 0.3, False),                 # one token a page
    (1, 1, 4, 64, [4001, 3], 0.25, True),                 # a plan past what a launch's arguments hold
])
def test_compact(layers, heads, tokens, d, lens, rate, renumber):
    print(f"[gpu] compact {lens} tokens={tokens} rate={rate}", flush=True)
    need = [-(-n // tokens) for n in lens]
    pool = random_pool(layers, 2 * sum(need) + 3, heads, tokens, d, seed=sum(lens))
    order = pool.allocate(sum(need))
    order = np.random.RandomState(1).permutation(order).tolist()  # pages in no order
    at = np.concatenate([[0], np.cumsum(need)])
    tables = [order[at[b]:at[b + 1]] for b in range(len(lens))]
    idx, n_kept = kept_list(lens, rate, max(max(lens), 1), seed=2)
    want = snapshot(pool)
    pool.retain(order)
    new, new_lens = pool.compact(tables, lens, torch.tensor(idx, device=DEV),
                                 torch.tensor(n_kept, dtype=torch.int32, device=DEV), renumber=renumber)
    assert new_lens == n_kept and [len(x) for x in new] == [-(-k // tokens) for k in n_kept]
    compact_np(want, tables, idx, n_kept, new, tokens, renumber)
    assert_same(pool, want)
    assert all(pool.ref_count(p) == 1 for p in order)
    used = sum(len(x) for x in new)
    assert pool.free_pages == pool.num_pages - sum(need) - used
    pool.free(order)
    pool.free([p for x in new for p in x])
    assert pool.free_pages == pool.num_pages


def test_compact_takes_the_keep_masks_list_and_clamps_foreign_positions():
    from nexusquant_amd.ops import keep_mask
    print("[gpu] compact by keep_mask", flush=True)
    pool = random_pool(2, 80, 2, 16, 128)
    tables = [pool.allocate(20), pool.allocate(20)]
    imp = torch.rand(2, 307, generator=torch.Generator().manual_seed(1)).to(DEV)
    keep, kept_idx, n_kept = keep_mask(imp, 0.6)
    want = snapshot(pool)
    new, lens = pool.compact(tables, [307, 307], kept_idx, n_kept)
    assert lens == n_kept.tolist() == keep.sum(1).tolist()
    compact_np(want, tables, kept_idx.cpu().numpy(), lens, new, 16, False)
    assert_same(pool, want)
    assert pool.free_pages == 80 - sum(len(x) for x in new)  # the old pages were freed
    # positions outside the sequence: clamped into it
    idx = torch.tensor([[-5, 0, 1 << 30]], dtype=torch.int32, device=DEV)
    want = snapshot(pool)
    out, _ = pool.compact([new[0]], [lens[0]], idx, [3])
    compact_np(want, [new[0]], np.array([[0, 0, lens[0] - 1]]), [3], out, 16, False)
    assert_same(pool, want)


def test_compact_of_forks_keeps_what_is_shared():
    print("[gpu] compact of forks", flush=True)
    pool = random_pool(1, 40, 2, 8, 64)
    a = pool.allocate(5)
    b, = pool.fork(a, 35)
    idx, n_kept = kept_list([35, 35], 0.5, 35, seed=3)
    want = snapshot(pool)
    new, lens = pool.compact([a, b], [35, 35], torch.tensor(idx, device=DEV), n_kept)
    compact_np(want, [a, b], idx, n_kept, new, 8, False)
    assert_same(pool, want)
    assert pool.free_pages == 40 - sum(len(x) for x in new)


def test_compact_refusals():
    print("[gpu] compact refusals", flush=True)
    pool = random_pool(1, 8, 1, 16, 64)
    a = pool.allocate(4)
    idx = torch.zeros(1, 64, dtype=torch.int32, device=DEV)
    before = snapshot(pool)
    for call in (lambda: pool.compact([a], [60], idx, [61]), lambda: pool.compact([a], [60], idx, [-1]),
                 lambda: pool.compact([a], [65], idx, [3]), lambda: pool.compact([a, a], [60, 60], idx, [1, 1]),
                 lambda: pool.compact([a], [60], idx.long(), [1]), lambda: pool.compact([a], [60], idx[0], [1]),
                 lambda: pool.compact([a], [60], idx[:, :2], [3]),
                 lambda: pool.compact([a, a], [60, 60], idx.expand(2, -1), [1, 1]),  # one reference, two tables
                 lambda: pool.compact([[5, 6, 7, 4]], [60], idx, [1])):
        with pytest.raises(ValueError):
            call()
    from nexusquant_amd._lib import NexusQuantError
    with pytest.raises(NexusQuantError):
        pool.compact([a], [60], idx.cpu(), [1])
    pool.allocate(4)
    with pytest.raises(NexusQuantError, match="0 of 8 free"):
        pool.compact([a], [60], idx, [1])
    assert_same(pool, before)
    assert all(pool.ref_count(p) == 1 for p in range(8))


@pytest.mark.parametrize("heads,tokens,d,dtype,n", [(2, 16, 128, torch.float16, 1), (1, 7, 64, torch.bfloat16, 40),
                                                    (8, 16, 128, torch.bfloat16, 130), (3, 5, 256, torch.float32, 65),
                                                    (1, 16, 64, torch.float16, 1000)])
def test_write_stores_what_the_page_encoder_makes(heads, tokens, d, dtype, n):
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor
    print(f"[gpu] write heads={heads} tokens={tokens} d={d} n={n}", flush=True)
    pages = -(-n // tokens) + 4
    pool = random_pool(3, pages, heads, tokens, d, seed=n)
    pool.allocate(pages)
    comp = NexusQuantKVCompressor(head_dim=d, bits=3, rope_base=500000.0)
    g = torch.Generator().manual_seed(n)
    k = torch.randn(n, heads, d, generator=g).to(dtype).to(DEV)
    v = torch.randn(n, heads, d, generator=g).to(dtype).to(DEV)
    pos = torch.randint(0, 90000, (n,), generator=g, dtype=torch.int32)
    slots = np.random.RandomState(n).permutation(pages * tokens)[:n]
    if n > 2:
        slots[1] = -1
    want = snapshot(pool)
    pool.write(comp, slots.tolist(), k, v, pos, layer=1)
    page = comp.compress_page(k.permute(1, 0, 2), v.permute(1, 0, 2), pos)
    new = {"key_codes": page.key_codes, "value_codes": page.value_codes, "key_scales": page.key_scales,
           "value_scales": page.value_scales}
    for i, s in enumerate(slots):
        if s >= 0:
            for name, t in new.items():
                want[name][1, s // tokens, :, s % tokens] = t[:, i].cpu().numpy()
            want["positions"][s // tokens, s % tokens] = int(pos[i])
    assert_same(pool, want)
    assert pool.max_position >= int(pos.max())


def test_write_refusals():
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor
    print("[gpu] write refusals", flush=True)
    pool = random_pool(2, 6, 2, 4, 64)
    a = pool.allocate(3)
    pool.retain(a[:1])
    comp = NexusQuantKVCompressor(head_dim=64)
    k = torch.zeros(2, 2, 64, device=DEV, dtype=torch.float16)
    before = snapshot(pool)
    for call in (lambda: pool.write(comp, [4, 4], k, k, [0, 1]),                # a slot twice
                 lambda: pool.write(comp, [0, 5], k, k, [0, 1]),                # a shared page
                 lambda: pool.write(comp, [4, 12], k, k, [0, 1]),               # a page that is free
                 lambda: pool.write(comp, [4, 99], k, k, [0, 1]),
                 lambda: pool.write(comp, [4], k, k, [0, 1]),
                 lambda: pool.write(comp, [4, 5], k, k, [0]),
                 lambda: pool.write(comp, [4, 5], k, k, [0, -1]),
                 lambda: pool.write(comp, [4, 5], k, k, [0, 1], layer=2),
                 lambda: pool.write(comp, [4, 5], k[:, :1], k[:, :1], [0, 1]),
                 lambda: pool.write(comp, [4, 5], k, k.cpu(), [0, 1]),
                 lambda: pool.write(NexusQuantKVCompressor(head_dim=128), [4, 5], k, k, [0, 1])):
        with pytest.raises(ValueError):
            call()
    pool.write(comp, [], k[:0], k[:0], [])
    pool.write(comp, [-1, -(1 << 40)], k, k, [0, 1])
    assert_same(pool, before)


def test_copies_on_another_stream_and_in_a_graph():
    print("[gpu] copies on a stream and in a graph", flush=True)
    pool = random_pool(2, 12, 2, 16, 128)
    pool.allocate(12)
    want = snapshot(pool)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.copy_pages([0, 1], [6, 7])
    side.synchronize()
    copy_np(want, [0, 1], [6, 7])
    assert_same(pool, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.copy_pages([2, 6], [9, 10])
        for call in (lambda: pool.fork([0], 16), lambda: pool.compact([[0]], [16], torch.zeros(1, 1), [1])):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert_same(pool, want)
    for i in range(3):
        pool.key_codes[:, 2] = i
        torch.cuda.synchronize()
        want["key_codes"][:, 2] = i
        graph.replay()
        copy_np(want, [2, 6], [9, 10])
        assert_same(pool, want)


def test_pages_of_a_pool_are_the_compressors_pages():
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor
    print("[gpu] pool pages decoded", flush=True)
    pool = random_pool(2, 4, 2, 16, 128)
    pool.allocate(3)
    comp = NexusQuantKVCompressor(head_dim=128, bits=3)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(16, 2, 128, generator=g).half().to(DEV) for _ in range(2))
    pool.write(comp, pool.slots([2], 0, 16), k, v, list(range(100, 116)), layer=1)
    got = comp.decompress_page(pool.page(2, layer=1))
    want = comp.decompress_page(comp.compress_page(k.permute(1, 0, 2), v.permute(1, 0, 2), range(100, 116)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("where", ["list", "cpu", "device"])
def test_positions_of_skipped_tokens_do_not_count(where):
    """A padded batch: -1 and far positions where nothing is stored are not refused and do not lengthen the tables."""
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor
    print(f"[gpu] write padding positions ({where})", flush=True)
    pool = random_pool(1, 6, 2, 4, 64, seed=3)
    pool.positions.zero_()
    pool.max_position = 0
    pool.allocate(3)
    comp = NexusQuantKVCompressor(head_dim=64)
    k = torch.randn(5, 2, 64, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    slots, pos = [3, -1, 9, -1, 4], [7, -1, 8, (1 << 31) - 1, 9]
    want = snapshot(pool)
    kept = [0, 2, 4]
    page = comp.compress_page(k[kept].permute(1, 0, 2), k[kept].permute(1, 0, 2), [7, 8, 9])
    for j, i in enumerate(kept):
        at = slots[i] // 4, slots[i] % 4
        for name in FIELDS[:4]:
            want[name][0, at[0], :, at[1]] = getattr(page, name)[:, j].cpu().numpy()
        want["positions"][at] = pos[i]
    given = pos if where == "list" else torch.tensor(pos, dtype=torch.int32, device=DEV if where == "device" else "cpu")
    pool.write(comp, slots, k, k, given)
    assert_same(pool, want)
    assert pool.max_position == 9
    if where != "list":
        assert given.tolist() == pos  # the caller's are left as they are
    with pytest.raises(ValueError):
        pool.write(comp, slots, k, k, [7, -1, -8, 0, 9])  # a stored one
    with pytest.raises(ValueError):
        pool.write(comp, slots, k, k, [7, -1, 8])
    assert_same(pool, want)
