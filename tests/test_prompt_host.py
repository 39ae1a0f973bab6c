"""Host side of packed prompt attention: the tile list and the refusals, without a GPU."""

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from nexusquant_amd import _lib
from nexusquant_amd.attention import PromptPlan, _PACK, _apart, _splits, plan_prompts, prompt_attention, prompt_tiles

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("lens", [[], [0], [1], [128], [129], [0, 5, 0, 300, 128, 0], [4096, 1, 64]])
def test_tiles_cover_every_query_once_longest_first(lens):
    tiles = prompt_tiles(lens, 128)
    starts = np.concatenate([[0], np.cumsum(lens)])
    seen = []
    for first, n, q0, _ in tiles.tolist():
        b = [i for i in range(len(lens)) if starts[i] == first and lens[i] == n and n]
        assert b and 0 <= q0 < n and q0 % 128 == 0
        seen += range(first + q0, first + min(q0 + 128, n))
    assert sorted(seen) == list(range(sum(lens)))
    assert list(tiles[:, 2]) == sorted(tiles[:, 2], reverse=True)


def test_plan_refusals():
    with pytest.raises(ValueError):
        plan_prompts([3, -1], device="cuda")
    with pytest.raises(ValueError):
        plan_prompts([1 << 30, 1 << 30], device="cuda")
    with pytest.raises(_lib.NexusQuantError):
        plan_prompts([3], device="cpu")
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(_lib.NexusQuantError):
        prompt_attention(x, x, x, PromptPlan((4,), 4, 0, None))


def test_prompt_struct_matches_the_c_compiler(tmp_path):
    names = [f[0] for f in _lib.PromptDesc._fields_]
    prog = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{ROOT}/include/nexusquant_amd.h"', "int main(void){",
            'printf("%zu\\n", sizeof(nq_prompt_desc));']
    prog += [f'printf("%zu\\n", offsetof(nq_prompt_desc, {f}));' for f in names] + ["return 0;}"]
    (tmp_path / "p.c").write_text("\n".join(prog))
    subprocess.check_call(["gcc", "-o", str(tmp_path / "p"), str(tmp_path / "p.c")])
    out = [int(x) for x in subprocess.check_output([str(tmp_path / "p")]).split()]
    assert _PACK.size == ctypes.sizeof(_lib.PromptDesc)
    assert out == [ctypes.sizeof(_lib.PromptDesc)] + [getattr(_lib.PromptDesc, f).offset for f in names]


def desc(**kw):
    dummy = ctypes.c_void_p(4096)
    two = ctypes.c_int64 * 2
    base = dict(q_heads=8, kv_heads=2, head_dim=128, dtype=_lib.NQ_F16, n_tiles=1, q=dummy, k=dummy, v=dummy, out=dummy,
                tiles=dummy, q_stride=two(1024, 128), k_stride=two(256, 128), v_stride=two(256, 128),
                out_stride=two(1024, 128), scale=0.1, n_split=1)
    return _lib.PromptDesc(**{**base, **kw})


@pytest.mark.parametrize("kw", [
    dict(head_dim=96), dict(dtype=_lib.NQ_F32), dict(q_heads=0), dict(q_heads=7), dict(kv_heads=0), dict(n_tiles=-1),
    dict(sliding_window=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None),
    dict(tiles=None), dict(out=ctypes.c_void_p(4100)), dict(v=ctypes.c_void_p(4104)),
    dict(k_stride=(ctypes.c_int64 * 2)(260, 128)), dict(out_stride=(ctypes.c_int64 * 2)(1024, 130)),
    dict(k_stride=(ctypes.c_int64 * 2)(1 << 24, 128)), dict(v_stride=(ctypes.c_int64 * 2)(-256, 128)),
    dict(n_tiles=1 << 24), dict(q_heads=1 << 30, kv_heads=1), dict(n_split=0), dict(n_split=65), dict(n_split=2),
    dict(n_split=2, workspace=ctypes.c_void_p(4096), workspace_bytes=100),
    dict(n_split=2, workspace=ctypes.c_void_p(4100), workspace_bytes=1 << 30)])
def test_c_entry_refuses(kw):
    lib = _lib.load()
    assert lib.nq_prompt_attention(ctypes.byref(desc(**kw)), None) == -1
    assert lib.nq_last_error().startswith(b"nq_prompt_attention")


@pytest.mark.parametrize("workgroups,keys,d,want", [(1, 64, 128, 1), (1, 511, 64, 2), (1, 1 << 20, 128, 64), (64, 4096, 128, 8),
                                                    (128, 4096, 64, 4), (128, 4096, 256, 2), (100, 4096, 256, 2),
                                                    (129, 4096, 256, 1), (72, 500, 128, 2), (72, 200, 128, 1)])
def test_how_many_workgroups_share_a_tiles_keys(workgroups, keys, d, want):
    assert _splits(workgroups, keys, d) == want


def test_c_entry_takes_an_empty_batch():
    lib = _lib.load()
    assert lib.nq_prompt_attention(ctypes.byref(desc(n_tiles=0, q=None, tiles=None)), None) == 0
    assert lib.nq_prompt_attention(None, None) == -1


def test_a_stages_pieces_come_from_their_rows_whatever_the_stride(tmp_path):
    """Every lane's piece of every load of a stage, replayed through the kernel's own formulas: its place in LDS holds
    the chunk that the readers' layout wants there, read at row * stride + chunk."""
    (tmp_path / "p.cpp").write_text("""
#include <stdio.h>
#include "nq_tile.h"
using namespace nq::flash;
template <int D, bool VALUES> int check(long long stride) {
    using P = StagePieces<D, VALUES>;
    int bad = 0;
    for (int i = 0; i < Tile<D>::UPR / 4; ++i)
        for (int s = 0; s < 256; ++s) {
            const int place = 256 * i + s, row = place / Tile<D>::UPR;
            const int chunk = place % Tile<D>::UPR ^ (VALUES ? Tile<D>::value_swizzle(row) : Tile<D>::key_swizzle(row));
            const long long want = 2 * stride * row + 16 * chunk;
            bad += 2 * stride * P::STEP * i + (long long)P::offset(s, i % P::PERIOD, stride) != want;  // a whole stage's
            bad += 2 * (stride * P::row(s, i) + 8 * P::chunk(s, i)) != want;                           // the last one's
        }
    return bad;
}
int main(void) {
    int bad = 0;
    const long long strides[] = {0, 64, 72, 128, 136, 256, 264, 320, 384, 832, 1032, 8200, (1 << 24) - 8};
    for (long long s : strides)
        bad += check<64, false>(s) + check<64, true>(s) + check<128, false>(s) + check<128, true>(s) + check<256, false>(s) +
               check<256, true>(s);
    printf("%d\\n", bad);
    return bad != 0;
}
""")
    subprocess.check_call(["g++", "-std=c++17", "-I", os.path.join(ROOT, "nexusquant_amd", "csrc"), "-o", str(tmp_path / "p"),
                           str(tmp_path / "p.cpp")])
    assert subprocess.run([str(tmp_path / "p")], capture_output=True, text=True).stdout == "0\n"


def test_plans_are_not_made_in_a_capture(monkeypatch):
    """The copy to the device would become part of the graph, from pinned memory that is given to others afterwards."""
    import contextlib
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        plan_prompts([3, 200], device="cuda:0")
    assert plan_prompts([0, 0], device="cuda:0").n_tiles == 0  # nothing to copy


@pytest.mark.parametrize("d,per_tile", [(64, 8), (128, 16), (256, 32)])
def test_c_entry_refuses_more_tiles_than_their_join_takes(d, per_tile):
    """The join has 128 D / 1024 workgroups of 256 threads for each tile and head: 2^32 threads at most.  (The calls within
    it end at their missing workspace.)"""
    lib = _lib.load()
    most = (2 ** 32 - 1) // 256 // per_tile // 8  # tiles of 8 heads
    for n_tiles, why in ((most, b"workspace"), (most + 1, b"grid too large")):
        x = desc(head_dim=d, n_tiles=n_tiles, n_split=2)
        assert lib.nq_prompt_attention(ctypes.byref(x), None) == -1
        assert why in lib.nq_last_error(), (n_tiles, lib.nq_last_error())


def test_c_entry_refuses_products_past_64_bits():
    lib = _lib.load()
    x = desc(n_tiles=1 << 30, q_heads=1 << 30, kv_heads=1, n_split=16)  # 2^64 workgroups
    assert lib.nq_prompt_attention(ctypes.byref(x), None) == -1
    assert b"grid too large" in lib.nq_last_error()


def test_outputs_whose_head_vectors_overlap_are_seen():
    """Against the list of all addresses."""
    def overlap(rows, heads, row, head, d=8):
        at = [r * row + h * head for r in range(rows) for h in range(heads)]
        return len({a + i for a in at for i in range(d)}) < len(at) * d
    seen = set()
    for rows in range(1, 5):
        for heads in range(1, 5):
            for row in range(0, 52, 4):
                for head in range(0, 52, 4):
                    t = torch.as_strided(torch.zeros(400), (rows, heads, 8), (row, head, 1))
                    want = not overlap(rows, heads, row, head)
                    assert _apart(t) == want, (rows, heads, row, head)
                    nested = row >= (heads - 1) * head + 8 or head >= (rows - 1) * row + 8
                    seen.add((want, nested))
    assert len(seen) == 4  # interleaved ones that are apart, too
