"""Packed prompt attention against the formula in 64 bits.

Tolerance: with u = eps(T) / 2 the kernel rounds each weight once (at most u of it) and each
result once (u of it, or half a step of the type's subnormal numbers, which below finfo.tiny are
tiny * eps apart whatever the result: 2^-25 for fp16); logits are fp32 sums of D products, so a weight's exponent is off by at
most D 2^-24 of the sum of |q k| scale (twice, through the denominator); sums over n keys in
fp32 and the exponential's 2^-22 are added.  Nothing else is rounded."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def oracle(q, k, v, lens, scale, window):
    """(out, tolerance) in float64 of packed [rows, heads, d] tensors."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u = torch.finfo(q.dtype).eps / 2
    g = q.shape[1] // k.shape[1]
    a = 0
    for n in (x for x in lens if x):
        i = torch.arange(n, device=q.device)
        seen = i[:, None] >= i
        if window:
            seen &= i[:, None] - i < window
        for h in range(q.shape[1]):
            qq, kk, vv = q[a:a + n, h].double(), k[a:a + n, h // g].double(), v[a:a + n, h // g].double()
            p = torch.softmax(torch.where(seen, qq @ kk.T * scale, -torch.inf), -1)
            out[a:a + n, h] = p @ vv
            big = torch.where(seen, qq.abs() @ kk.abs().T * scale, 0.0).amax(-1, keepdim=True)
            rel = u + 2 * (q.shape[2] + 2) * 2 ** -24 * big + n * 2 ** -24 + 2 ** -21
            step = torch.finfo(q.dtype).tiny * u
            tol[a:a + n, h] = rel * (p @ vv.abs()) + (u * out[a:a + n, h].abs()).clamp_min(step)
        a += n
    return out, tol


def inputs(rows, hq, hkv, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hq + 2 * hkv, d, generator=g)
    x[:, :hq] *= spread
    x = x.to(dtype).to(DEV)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]  # strided: slices of one projection


def check(q, k, v, lens, scale=None, window=None, **kw):
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    got = prompt_attention(q, k, v, plan_prompts(lens, device=DEV), scale=scale, sliding_window=window, **kw)
    want, tol = oracle(q, k, v, lens, q.shape[2] ** -0.5 if scale is None else scale, window)
    off = (got.double() - want).abs() - tol
    assert got.shape == q.shape and got.dtype == q.dtype
    assert bool((off[:sum(lens)] <= 0).all()), f"over tolerance by {off.max().item()}"
    return got


@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 2, 64, torch.float16), (4, 1, 128, torch.bfloat16),
                                            (2, 2, 256, torch.float16), (8, 1, 256, torch.bfloat16),
                                            (6, 2, 128, torch.float16), (3, 3, 64, torch.bfloat16)])
@pytest.mark.parametrize("lens", [[1], [63, 64, 65, 1, 2], [0, 31, 0, 32, 33, 0], [127, 128, 129, 300]])
def test_ragged_batches(hq, hkv, d, dtype, lens):
    print(f"[gpu] prompt {hq}/{hkv} d={d} {dtype} {lens}", flush=True)
    check(*inputs(sum(lens), hq, hkv, d, dtype, seed=sum(lens) + d), lens)


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 100, 1000])
def test_sliding_window(d, dtype, window):
    print(f"[gpu] prompt window={window} d={d}", flush=True)
    lens = [257, 5, 400]
    check(*inputs(sum(lens), 4, 2, d, dtype, seed=window), lens, window=window)


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.float16)])
def test_long_prompt_and_peaked_logits(d, dtype):
    print(f"[gpu] prompt long d={d}", flush=True)
    lens = [2111]
    check(*inputs(2111, 2, 1, d, dtype, seed=1), lens)
    check(*inputs(2111, 2, 1, d, dtype, seed=2, spread=12.0), lens)   # maxima that keep rising
    check(*inputs(300, 2, 1, d, dtype, seed=3), [300], scale=0.9)


def test_rising_maxima_rescale_every_stage():
    """Keys ordered so that each stage's logits pass the ones before by more than the slack."""
    print("[gpu] prompt rising maxima", flush=True)
    q, k, v = inputs(640, 2, 1, 128, torch.float16, seed=4)
    q, k = q.contiguous(), k.contiguous()
    q[:] = 1.0
    k[:] = (torch.arange(640, device=DEV) / 64).floor()[:, None, None] * 0.9 + 0.01 * k
    check(q, k, v, [640])
    k[:] = -k  # and falling ones
    check(q, k, v, [640])


def test_rows_behind_the_sequences_and_hidden_values_do_not_count():
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt NaN in hidden places", flush=True)
    for d, dtype in ((64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)):
        lens = [100, 77]
        q, k, v = (x.contiguous() for x in inputs(200, 4, 2, d, dtype, seed=d))
        clean = check(q, k, v, lens)
        assert bool((clean[177:] == 0).all())
        for x in (q, k, v):
            x[177:] = float("nan")
        out = torch.full_like(q, 7.0)
        got = prompt_attention(q, k, v, plan_prompts(lens, device=DEV), out=out)
        assert got is out and torch.equal(got[:177], clean[:177]) and bool((got[177:] == 7.0).all())
        # a value that only later queries see: the earlier ones keep their results
        for bad in (float("inf"), float("nan")):
            v2, k2 = v.clone(), k.clone()
            v2[90, 1], k2[50, 0] = bad, float("nan")
            got = prompt_attention(q, k2, v2, plan_prompts(lens, device=DEV), sliding_window=40)
            want, tol = oracle(q, k, v, lens, d ** -0.5, 40)
            hit = torch.zeros(177, 4, dtype=torch.bool, device=DEV)
            hit[90:100, 2:] = True   # queries 90 .. of the first sequence, heads of kv head 1
            hit[50:90, :2] = True    # a NaN key: its window's queries
            assert bool((~torch.isfinite(got[:177][hit]).any(-1)).all())
            off = ((got[:177].double() - want[:177]).abs() - tol[:177])[~hit]
            assert bool((off <= 0).all()), (d, bad, off.max().item())


def test_layouts():
    """Head-major tensors, misaligned ones (copied) and a strided output."""
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt layouts", flush=True)
    lens = [90, 10]
    q, k, v = (x.contiguous() for x in inputs(100, 4, 2, 128, torch.float16, seed=5))
    want = check(q, k, v, lens)
    plan = plan_prompts(lens, device=DEV)
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(prompt_attention(*hm, plan), want)

    def shifted(x):
        buf = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)
        buf[1:] = x.reshape(-1)
        return buf[1:].view(x.shape)
    assert torch.equal(prompt_attention(*(shifted(x) for x in (q, k, v)), plan), want)
    wide = torch.full((100, 8, 128), 3.0, dtype=torch.float16, device=DEV)
    prompt_attention(q, k, v, plan, out=wide[:, 2:6])
    assert torch.equal(wide[:, 2:6], want) and bool((wide[:, :2] == 3).all()) and bool((wide[:, 6:] == 3).all())
    one = k[:, :1].expand(-1, 2, -1)  # one stored head under two
    assert torch.equal(prompt_attention(q, one, one, plan), prompt_attention(q, one.contiguous(), one.contiguous(), plan))


@pytest.mark.parametrize("hq,hkv,d,dtype", [(1, 1, 64, torch.bfloat16), (2, 1, 128, torch.float16), (2, 2, 256, torch.bfloat16)])
@pytest.mark.parametrize("lens,window", [([513], None), ([1300, 5, 0, 129], None), ([2500], 700), ([1000, 640], 1), ([1, 3000], None)])
def test_few_tiles_share_their_keys(hq, hkv, d, dtype, lens, window):
    from nexusquant_amd.attention import _splits, plan_prompts, prompt_attention
    print(f"[gpu] prompt split {hq}/{hkv} d={d} {dtype} {lens} {window}", flush=True)
    q, k, v = inputs(sum(lens), hq, hkv, d, dtype, seed=len(lens))
    plan = plan_prompts(lens, device=DEV)
    assert window or _splits(plan.n_tiles * hq, max(lens), d) > 1
    want = check(q, k, v, lens, window=window)
    assert torch.equal(prompt_attention(q, k, v, plan, sliding_window=window), want)  # joined in a fixed order
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attention(q, k, v, plan, sliding_window=window)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # what the first half of the last sequence does not see (its last queries are summed again, in other roundings)
    at = sum(lens) - lens[-1] // 2
    if lens[-1] > 1:
        ref, tol = oracle(q, k, v, lens, d ** -0.5, window)
        v[at:, -1], k[at + 1:, -1] = float("inf"), float("nan")
        got = prompt_attention(q, k, v, plan, sliding_window=window)
        assert bool(((got.double() - ref).abs() <= tol)[:at].all()) and bool(got[at + 1:, -1].isnan().all())


def test_output_in_place_of_the_query():
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt in place", flush=True)
    lens = [200, 1, 129]
    q, k, v = inputs(330, 4, 2, 128, torch.bfloat16, seed=8)
    v[150:200] = float("nan")  # hidden from the first queries of their tile: summed again after the fast pass
    plan = plan_prompts(lens, device=DEV)
    want = prompt_attention(q, k, v, plan)
    got = prompt_attention(q, k, v, plan, out=q)
    assert got is q and torch.equal(q.isnan(), want.isnan()) and torch.equal(q.nan_to_num(), want.nan_to_num())
    assert bool(want[150:200].isnan().all()) and not bool(want[:150].isnan().any())


def test_stream_graph_and_repeat():
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt stream and graph", flush=True)
    lens = [130, 300, 1]
    q, k, v = inputs(sum(lens), 4, 2, 64, torch.bfloat16, seed=6)
    plan = plan_prompts(lens, device=DEV)
    want = prompt_attention(q, k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = prompt_attention(q, k, v, plan)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attention(q, k, v, plan)
    for i in range(3):
        q.mul_(0.75)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, prompt_attention(q, k, v, plan))


def test_refusals():
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt refusals", flush=True)
    q, k, v = inputs(20, 4, 2, 64, torch.float16, seed=7)
    plan = plan_prompts([20], device=DEV)
    for call in (lambda: prompt_attention(q[:10], k, v, plan), lambda: prompt_attention(q[:10], k[:10], v[:10], plan),
                 lambda: prompt_attention(q, k[:, :, :32], v, plan), lambda: prompt_attention(q[:, :3], k, v, plan),
                 lambda: prompt_attention(q.float(), k.float(), v.float(), plan),
                 lambda: prompt_attention(q.bfloat16(), k, v, plan),
                 lambda: prompt_attention(q[..., :32], k[..., :32], v[..., :32], plan),
                 lambda: prompt_attention(q, k, v, plan, sliding_window=0),
                 lambda: prompt_attention(q, k, v, plan, scale=-1.0),
                 lambda: prompt_attention(q, k, v, plan, scale=float("nan")),
                 lambda: prompt_attention(q[0], k, v, plan),
                 lambda: prompt_attention(q, k, v, plan, out=torch.empty_like(q[:1]).expand(20, -1, -1)),
                 lambda: prompt_attention(q, k, v, plan, out=torch.empty_like(q[:, :1]).expand(-1, 4, -1)),
                 lambda: prompt_attention(q, k, v, plan, out=torch.empty(20, 4, 64, device=DEV))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        prompt_attention(q.detach().requires_grad_(), k, v, plan)
    from nexusquant_amd._lib import NexusQuantError
    with pytest.raises(NexusQuantError):
        prompt_attention(q, k.cpu(), v, plan)
    assert prompt_attention(q[:0], k[:0], v[:0], plan_prompts([0, 0], device=DEV)).shape == (0, 4, 64)


@pytest.mark.parametrize("d,widths", [(256, (264, 320)), (256, (832, 1032)), (256, (384, 256)), (128, (136, 200)), (64, (72, 104))])
@pytest.mark.parametrize("hq,hkv,lens", [(1, 1, [513]), (2, 2, [700, 0, 65]), (34, 2, [450, 130])])
def test_row_strides_of_any_multiple_of_eight(d, widths, hq, hkv, lens):
    """Keys and values in wider rows: the same bytes read, so the same results as from rows next to one another."""
    from nexusquant_amd.attention import _SPLIT_TO, plan_prompts, prompt_attention
    print(f"[gpu] prompt strides d={d} {widths} {hq}/{hkv} {lens}", flush=True)
    q, k, v = inputs(sum(lens), hq, hkv, d, torch.float16, seed=d + hq)
    plan = plan_prompts(lens, device=DEV)
    assert (plan.n_tiles * hq <= _SPLIT_TO[d] // 2) == (hq < 34 or d < 256)
    want = check(q, k, v, lens)

    def padded(x, width, pad):
        wide = torch.full((x.shape[0], hkv * width + pad), 5.0, dtype=x.dtype, device=DEV)
        y = wide[:, :hkv * width].view(x.shape[0], hkv, width)[..., :d]
        y.copy_(x)
        assert y.stride() == (hkv * width + pad, width, 1)
        return y
    for pad in (0, 8, 40):
        for window in (None, 100):
            ref = want if window is None else prompt_attention(q, k, v, plan, sliding_window=window)
            got = prompt_attention(q, padded(k, widths[0], pad), padded(v, widths[1], pad), plan, sliding_window=window)
            assert torch.equal(got, ref), (pad, window)


def test_a_plan_is_made_before_a_capture():
    """The refusal leaves the capture as it was: its graph is whole."""
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt plan in a capture", flush=True)
    q, k, v = inputs(150, 4, 2, 64, torch.float16, seed=21)
    plan = plan_prompts([150], device=DEV)
    want = prompt_attention(q, k, v, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before capturing"):
            plan_prompts([150], device=DEV)
        out = prompt_attention(q, k, v, plan)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("hq,d,dtype", [(1, 128, torch.float16), (32, 128, torch.float16), (1, 64, torch.float16),
                                        (40, 64, torch.float16), (2, 256, torch.float16), (18, 256, torch.float16),
                                        (32, 128, torch.bfloat16)])
@pytest.mark.parametrize("logit", [-9.375, -12.1875, -14.25])
def test_many_small_weights_beside_one_large(hq, d, dtype, logit):
    """A first token that takes nearly all of the weight and has a value of zero, and many that share the rest, alike (so
    that their weights' roundings add up): a fp16 weight keeps its 11 bits down to 2^-21 of the largest, e^-14.25 among
    them, though it is 11 steps of fp16's smallest number as it stands."""
    print(f"[gpu] prompt small weights {hq} d={d} {dtype} {logit}", flush=True)
    n = 1100
    q, k, v = (x.contiguous() for x in inputs(n, hq, 1, d, dtype, seed=hq + d))
    v.add_(3.0)
    v[0] = 0
    q.zero_()
    k.zero_()
    q[..., 0] = 1.0
    k[1:, :, 0] = logit
    check(q, k, v, [n], scale=1.0)
    check(q, k, v, [n], scale=1.0, window=700)


def test_overlapping_outputs_are_refused():
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    print("[gpu] prompt overlapping outputs", flush=True)
    q, k, v = inputs(20, 4, 2, 64, torch.float16, seed=31)
    plan = plan_prompts([20], device=DEV)
    buf = torch.zeros(20 * 4 * 64 * 2, dtype=torch.float16, device=DEV)
    for row, head in ((32, 1280), (192, 64), (256, 32), (64, 64)):
        with pytest.raises(ValueError, match="of their own"):
            prompt_attention(q, k, v, plan, out=torch.as_strided(buf, (20, 4, 64), (row, head, 1)))
    assert not bool(buf.any())
    want = prompt_attention(q, k, v, plan)
    for row, head in ((256, 64), (64, 1280), (264, 64), (68, 1360)):  # rows within heads, too, and with gaps
        assert torch.equal(prompt_attention(q, k, v, plan, out=torch.as_strided(buf, (20, 4, 64), (row, head, 1))), want)
