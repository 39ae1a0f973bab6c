"""Rotations with one and several axes against 64 bits, gradients against the formula and differences."""

import math

import numpy as np
import pytest
import torch

from nexusquant_amd import plan_rotation, rotate
from nexusquant_amd.rope import inv_freq
from nexusquant_amd.rotary import frequency_axes
from oracle import four_bit as ref
from test_rotary_host import check_forward_mode, check_gradients_of_those_that_need_one, check_written_tensors_are_seen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def grid(rows, axes, start=0):
    i = torch.arange(rows)
    return torch.stack([i // 35, i // 7 % 5, i % 7, i][:axes] if axes > 1 else [i]) + start


def limit(want, x, dtype):
    """A product's two terms, their sum, cosine and sine are rounded to 32 bits (2^-24 each of |a| + |b| at most, six of
    them), the result to its type (half a step; 2^-24 below fp16's smallest normal number)."""
    half = x.shape[-1] // 2
    big = x.abs().double()
    both = (big[..., :half] + big[..., half:]).repeat(1, 1, 2)
    return want.abs() * torch.finfo(dtype).eps / 2 + 6 * 2.0 ** -24 * both + 2.0 ** -25


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,axes,sections,interleaved", [
    (64, 1, None, False), (128, 1, None, False), (256, 1, [128], False), (128, 3, [16, 24, 24], False),
    (128, 3, [24, 20, 20], True), (64, 2, [16, 16], True), (256, 4, [128, 0, 0, 0], False), (64, 3, [32, 0, 0], True)])
@pytest.mark.parametrize("rows,hq,hk", [(1, 1, 1), (33, 6, 2), (257, 4, 4)])
def test_rotation(dtype, d, axes, sections, interleaved, rows, hq, hk):
    g = torch.Generator(device="cuda").manual_seed(rows * d)
    qkv = torch.randn(rows, hq + 2 * hk, d, device="cuda", generator=g).to(TYPES[dtype])
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    pos = grid(rows, axes, start=1021)
    r = plan_rotation(pos.cuda().int() if rows % 2 else pos.cuda(), d, base=500000.0, sections=sections, interleaved=interleaved)
    ang = ref.angles(pos, inv_freq(d, 500000.0), frequency_axes(d, sections, interleaved))
    for inverse in (False, True):
        got = rotate(q, k, r, inverse=inverse)
        for x, y in zip((q, k), got):
            want = ref.rotate(x.cpu(), ang, inverse)
            off = (y.double().cpu() - want).abs()
            assert (off <= limit(want, x.cpu(), TYPES[dtype])).all(), float(off.max())
    alone, none = rotate(q, None, r)
    assert none is None and torch.equal(alone, rotate(q, k, r)[0])


def test_cosines_and_sines_of_far_positions_are_exact_to_fp32():
    pos = torch.tensor([0, 1, -3, 131071, 1 << 20, (1 << 24) + 1, -(1 << 30), (1 << 31) - 1])
    r = plan_rotation(pos.cuda(), 64, base=10000.0)
    ang = ref.angles(pos[None], inv_freq(64, 10000.0), frequency_axes(64, None, False))
    assert (r.angles[:, 0].double().cpu() - ang.cos()).abs().max() <= 2.0 ** -24
    assert (r.angles[:, 1].double().cpu() - ang.sin()).abs().max() <= 2.0 ** -24
    scaled = plan_rotation(pos.cuda(), 64, base=10000.0, rope_scaling={"type": "linear", "factor": 4.0})
    ang = ref.angles(pos[None], inv_freq(64, 10000.0, {"type": "linear", "factor": 4.0}), frequency_axes(64, None, False))
    assert (scaled.angles[:, 1].double().cpu() - ang.sin()).abs().max() <= 2.0 ** -24


def test_positions_of_the_host_and_strided_ones():
    pos = grid(40, 3, start=5)
    a = plan_rotation(pos.cuda(), 128, sections=[24, 20, 20], interleaved=True).angles
    assert torch.equal(plan_rotation(pos.tolist(), 128, sections=[24, 20, 20], interleaved=True).angles, a)
    assert torch.equal(plan_rotation(pos.int().numpy(), 128, sections=[24, 20, 20], interleaved=True).angles, a)
    wide = torch.zeros(3, 80, dtype=torch.int64, device="cuda")
    wide[:, ::2] = pos.cuda()
    assert torch.equal(plan_rotation(wide[:, ::2], 128, sections=[24, 20, 20], interleaved=True).angles, a)
    same = pos[:1].cuda().expand(3, 40)  # text: all axes alike
    assert torch.equal(plan_rotation(same, 128, sections=[16, 24, 24]).angles, plan_rotation(pos[0].cuda(), 128).angles)
    none = plan_rotation([], 64)
    q, k = rotate(torch.empty(0, 3, 64, device="cuda"), torch.empty(0, 1, 64, device="cuda"), none)
    assert q.shape == (0, 3, 64) and k.shape == (0, 1, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_and_into_slices(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(50, 12, 128, device="cuda", generator=g).to(TYPES[dtype])
    r = plan_rotation(torch.arange(50, device="cuda"), 128)
    want = [x.clone() for x in rotate(qkv[:, :8], qkv[:, 8:10], r)]
    into = torch.full((50, 12, 128), 7.0, device="cuda", dtype=TYPES[dtype])
    rotate(qkv[:, :8], qkv[:, 8:10], r, out=(into[:, 4:], into[:, :2]))
    assert torch.equal(into[:, 4:], want[0]) and torch.equal(into[:, :2], want[1]) and (into[:, 2:4] == 7.0).all()
    rest = qkv[:, 10:].clone()
    q, k = rotate(qkv[:, :8], qkv[:, 8:10], r, out=(qkv[:, :8], qkv[:, 8:10]))
    assert q.data_ptr() == qkv.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 10:], rest)
    heads_first = torch.randn(4, 50, 128, device="cuda", generator=g).to(TYPES[dtype])
    y, _ = rotate(heads_first.transpose(0, 1), None, r)
    assert torch.equal(y, rotate(heads_first.transpose(0, 1).contiguous(), None, r)[0])
    odd = torch.randn(50 * 128 * 3 + 1, device="cuda", generator=g).to(TYPES[dtype])[1:].view(50, 3, 128)  # not 16-byte aligned
    assert torch.equal(rotate(odd, None, r)[0], rotate(odd.clone(), None, r)[0])


def test_gradients():
    """Against the formula (the rotation by the opposite angle), against differences, and of broadcast gradients."""
    rows, d = 9, 64
    pos = grid(rows, 3, start=77)
    sections = [12, 10, 10]
    r = plan_rotation(pos.cuda(), d, sections=sections, interleaved=True)
    ang = ref.angles(pos, inv_freq(d, 10000.0), frequency_axes(d, sections, True))
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in TYPES.values():
        q = torch.randn(rows, 4, d, device="cuda", generator=g).to(dtype).requires_grad_()
        k = torch.randn(rows, 2, d, device="cuda", generator=g).to(dtype).requires_grad_()
        gq, gk = torch.randn(rows, 4, d, device="cuda", generator=g).to(dtype), torch.randn(rows, 1, 1, device="cuda", generator=g).to(dtype).expand(rows, 2, d)
        got = torch.autograd.grad(rotate(q, k, r), (q, k), (gq, gk))
        for x, y in zip((gq, gk), got):
            want = ref.rotate(x.cpu(), ang, inverse=True)
            assert ((y.double().cpu() - want).abs() <= limit(want, x.cpu(), dtype)).all()
    # differences in 32 bits: the function is linear, so a step of 1 has no error but the sums' rounding (2^-24 of some
    # hundred terms of up to 10)
    q = torch.randn(rows, 2, d, device="cuda", generator=g, requires_grad=True)
    w = torch.randn(rows, 2, d, device="cuda", generator=g)
    grad, = torch.autograd.grad((rotate(q, None, r)[0] * w).sum(), q)
    with torch.no_grad():
        for at in ((0, 0, 0), (3, 1, 31), (8, 1, 63), (5, 0, 40)):
            step = torch.zeros_like(q)
            step[at] = 1.0
            diff = ((rotate(q + step, None, r)[0].double() - rotate(q - step, None, r)[0].double()) * w).sum() / 2
            assert abs(float(diff) - float(grad[at])) <= 1e-4
    # one of two, and twice
    k = torch.randn(rows, 2, d, device="cuda", generator=g)
    out = rotate(q, k, r)
    assert out[0].requires_grad
    first, = torch.autograd.grad(out[0].square().sum(), q, create_graph=True)
    assert (first - 2 * q).abs().max() < 1e-4  # a rotation keeps lengths; twice 2^-23 of numbers below 10
    second, = torch.autograd.grad(first.sum(), q)
    assert (second - 2).abs().max() < 1e-5


def test_a_graph_replays():
    rows = 64
    pos = torch.arange(rows, device="cuda")
    q = torch.randn(rows, 4, 128, device="cuda").half()
    r = plan_rotation(pos, 128)
    rotate(q, None, r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotate(q, None, plan_rotation(pos, 128))[0]
    for i in range(3):
        pos.copy_(torch.arange(rows) + 100 * i)
        q.copy_(torch.randn(rows, 4, 128))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, rotate(q, None, plan_rotation(pos, 128))[0])
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,rows,hq,hk,d", [("bf16", 5000, 70, 9, 64), ("fp32", 1500, 37, 8, 128), ("fp16", 2100, 33, 1, 256)])
def test_large_outputs_and_many_heads_are_as_small_ones(dtype, rows, hq, hk, d):
    """Past 32 MB outputs are stored in another way, and a wave takes a row's heads in several steps."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    qkv = torch.randn(rows, hq + hk, d, device="cuda", generator=g).to(TYPES[dtype])
    assert qkv.numel() * qkv.element_size() >= 32 << 20
    pos = torch.arange(rows, device="cuda") * 3
    got = rotate(qkv[:, :hq], qkv[:, hq:], plan_rotation(pos, d))
    ang = ref.angles(pos[None], inv_freq(d, 10000.0), frequency_axes(d, None, False))
    for a in range(0, rows, 613):
        part = slice(a, min(a + 613, rows))
        for h in range(0, hq, 8):
            small, _ = rotate(qkv[part, h:min(h + 8, hq)], None, plan_rotation(pos[part], d))
            assert torch.equal(got[0][part, h:h + 8], small)
        small, _ = rotate(qkv[part, hq:], None, plan_rotation(pos[part], d))
        assert torch.equal(got[1][part], small)
    x = qkv[-20:].cpu()
    want = ref.rotate(x, ang[-20:])
    y = torch.cat([got[0][-20:], got[1][-20:]], dim=1)
    assert ((y.double().cpu() - want).abs() <= limit(want, x, TYPES[dtype])).all()
    rotate(qkv[:, :hq], qkv[:, hq:], plan_rotation(pos, d), out=(qkv[:, :hq], qkv[:, hq:]))
    assert torch.equal(qkv[:, :hq], got[0]) and torch.equal(qkv[:, hq:], got[1])


def test_a_captured_gradient_replays():
    rows, d = 70, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(rows, h, d, device="cuda", generator=g).bfloat16().requires_grad_() for h in (6, 2))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    r = plan_rotation(torch.arange(rows, device="cuda"), d)

    def step():
        y = rotate(q, k, r)
        return [x.detach() for x in y] + list(torch.autograd.grad(y, (q, k), (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            for t in (q, k, gq, gk):
                t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_another_stream_and_refusals():
    r = plan_rotation(torch.arange(8, device="cuda"), 64)
    q = torch.randn(8, 2, 64, device="cuda")
    want = rotate(q, None, r)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate(q, None, r)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    k = torch.randn(8, 2, 64, device="cuda")
    bad = [(q[:7], None), (q[:, :, :32], None), (q, k.half()), (q.double(), None), (q.int(), None), (q, k[:4])]
    for a, b in bad:
        with pytest.raises(ValueError):
            rotate(a, b, r)
    with pytest.raises(Exception, match="device"):
        rotate(q.cpu(), None, r)
    both = torch.randn(8, 4, 64, device="cuda")
    for out in ((both[:, :2], both[:, 1:3]), (k, torch.empty_like(k)), (q, q), (both[:, :1], both[:, :2]),
                (torch.empty(8, 2, 64, device="cuda").half(), k), (q, None), (q[:1].expand(8, 2, 64), k)):
        with pytest.raises(ValueError):
            rotate(q, k, r, out=out)
    with pytest.raises(NotImplementedError):
        rotate(q.clone().requires_grad_(), None, r, out=(torch.empty_like(q), None))
    with pytest.raises(ValueError):
        plan_rotation(torch.arange(6, device="cuda").view(2, 3), 64)
    with pytest.raises(TypeError):
        plan_rotation(torch.arange(6, device="cuda").float(), 64)


def test_gradients_of_those_that_need_one():
    check_gradients_of_those_that_need_one(plan_rotation(torch.arange(5, device="cuda"), 64), [])


def test_forward_mode():
    check_forward_mode(plan_rotation(torch.arange(5, device="cuda"), 64))


def test_writes_in_place_are_seen_by_autograd():
    r = plan_rotation(torch.arange(5, device="cuda"), 64)
    qkv = torch.randn(5, 8, 64, device="cuda")
    q, k = qkv[:, :4], qkv[:, 4:6]
    check_written_tensors_are_seen(lambda: rotate(q, k, r, out=(q, k)), q, k, qkv)


def test_rotations_planned_by_several_threads():
    """Each with bases of its own, more than the tables that are kept."""
    import threading
    positions = torch.arange(50, device="cuda")
    bases = [[1000.0 + 7 * i + 1000 * t for i in range(40)] for t in range(4)]
    got = [[] for _ in bases]

    def plan(t):
        torch.cuda.set_device(positions.device)
        for base in bases[t]:
            got[t].append(plan_rotation(positions, 128, base=base).angles)

    threads = [threading.Thread(target=plan, args=(t,)) for t in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for t, many in enumerate(bases):
        assert len(got[t]) == len(many)
        for base, angles in zip(many, got[t]):
            ang = ref.angles(positions[None], inv_freq(128, base), frequency_axes(128, None, False))
            assert (angles[:, 0].double().cpu() - ang.cos()).abs().max() <= 2.0 ** -24
            assert (angles[:, 1].double().cpu() - ang.sin()).abs().max() <= 2.0 ** -24
