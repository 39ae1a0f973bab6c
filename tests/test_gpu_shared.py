"""Decode attention over shared pages against the formula in 64 bits.

Tolerance (u = eps / 2 of fp16): keys are rounded to fp16, so a logit is off by a sum of independent
roundings u |q_i k_i| scale; six times its 2-norm holds but for 2e-8 of the logits (Hoeffding).  Weights
are rounded to fp16 (u of each), values in the transformed domain too (u of each coordinate: the
transform is orthonormal, so at most u times the token's 2-norm in any output), the result to its
type; fp32 sums and the exponential add 2^-20."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -11
BASE = 500000.0


def make_pool(layers, pages, heads, tokens, d, levels=8, seed=0, scale_mul=1.0):
    from nexusquant_amd.page_pool import CompressedPagePool
    g = torch.Generator().manual_seed(seed)
    s = (layers, pages, heads, tokens)

    def codes():
        return torch.randn(s + (d,), generator=g).mul_(levels / 3).round_().clamp_(-levels, levels).to(torch.int8)
    pool = CompressedPagePool.from_tensors(
        key_codes=codes().to(DEV), value_codes=codes().to(DEV),
        key_scales=((torch.rand(s, generator=g) * 4 + 2) / levels).half().to(DEV),
        value_scales=((torch.rand(s, generator=g) * 2 + 1) / levels * scale_mul).half().to(DEV),
        positions=torch.zeros(pages, tokens, dtype=torch.int32, device=DEV))
    return pool


def lay(pool, table, n, start=0):
    t = pool.page_tokens
    pos = torch.arange(start, start + len(table) * t, dtype=torch.int32)
    pos[n:] = 0
    pool.positions[torch.tensor(table, device=DEV)] = pos.view(-1, t).to(DEV)
    pool.max_position = max(pool.max_position, start + n)


def walsh(x):
    d, step = x.shape[-1], 1
    while step < d:
        y = x.reshape(*x.shape[:-1], d // (2 * step), 2, step)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).reshape(x.shape)
        step *= 2
    return x / math.sqrt(d)


def row_oracle(pool, layer, table, n, q):
    """(out, tolerance without the result's rounding) in float64 of one row."""
    d, h = pool.head_dim, pool.num_heads
    pages = torch.tensor(table, device=DEV)

    def whole(codes, scales):
        x = codes[layer, pages].double() / 2 * scales[layer, pages].double()[..., None]
        return walsh(x.transpose(0, 1).reshape(h, -1, d)[:, :n])
    k, v = whole(pool.key_codes, pool.key_scales), whole(pool.value_codes, pool.value_scales)
    f = 1.0 / (BASE ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
    ang = (pool.positions[pages].reshape(-1)[:n].float().cpu()[:, None] * f).double().to(DEV)
    a, b = k.chunk(2, -1)
    k = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    q = q.double().view(h, -1, d)
    p = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(d), -1)
    out = (p @ v)
    # fp32 angles' cosines: the tables' half ulp, and that of the products, are in the 2^-20
    big = ((q ** 2) @ (k ** 2).transpose(1, 2)).sqrt().amax(-1, keepdim=True) / math.sqrt(d)
    tol = (12 * U * big + U + 2 ** -20) * (p @ v.abs()) + (U + 2 ** -20) * (p @ v.norm(dim=-1, keepdim=True))
    return out.reshape(-1, d), tol.reshape(-1, d)


def check(attn, pool, tables, ctx, q, layer=0, min_saved=1, **kw):
    plan = attn.plan_shared(pool, tables, ctx, min_saved=min_saved)  # 1: whatever can be shared is
    got = attn.run_shared(plan, q, layer=layer, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    u = torch.finfo(q.dtype).eps / 2
    err = ref = 0.0
    for b, (table, n) in enumerate(zip(tables, ctx)):
        if n == 0:
            assert bool((got[b] == 0).all())
            continue
        want, tol = row_oracle(pool, layer, table[:pool.pages_for(n)], n, q[b])
        off = (got[b].double() - want).abs()
        assert bool((off <= tol + u * want.abs()).all()), (b, n, (off - tol - u * want.abs()).max().item())
        err, ref = err + off.square().sum().item(), ref + want.square().sum().item()
    # independent roundings: in the 2-norm each kind is below its bound, four of fp16 and the result's
    assert math.sqrt(err / ref) <= 4 * U + u if ref else True
    return plan, got


def attention(d, bits=3):
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor, NexusQuantPagedAttention
    return NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=d, bits=bits, rope_base=BASE))


def queries(rows, hq, d, dtype, seed=0):
    return torch.randn(rows, hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def forks(pool, prefix, suffixes):
    """Tables and lengths of branches of one sequence of `prefix` tokens, each grown by its suffix."""
    t = pool.page_tokens
    trunk = pool.allocate(pool.pages_for(prefix))
    lay(pool, trunk, prefix)
    tables, ctx = [], []
    for s in suffixes:
        kid, = pool.fork(trunk, prefix)
        kid = kid + pool.allocate(pool.pages_for(prefix + s) - len(kid))
        own = prefix // t
        if kid[own:]:
            lay(pool, kid[own:], prefix + s - own * t, own * t)
        tables.append(kid)
        ctx.append(prefix + s)
    return tables, ctx


@pytest.mark.parametrize("heads,group,d,tokens,dtype", [
    (2, 4, 128, 16, torch.float16), (1, 8, 64, 16, torch.bfloat16), (2, 1, 256, 16, torch.float16),
    (1, 3, 128, 7, torch.bfloat16), (2, 2, 64, 24, torch.float16), (1, 16, 256, 32, torch.bfloat16)])
@pytest.mark.parametrize("rows,prefix", [(2, 300), (9, 515), (40, 1030), (1, 200)])
def test_forked_rows(heads, group, d, tokens, dtype, rows, prefix):
    print(f"[gpu] shared {heads}x{group} d={d} T={tokens} {dtype} rows={rows} prefix={prefix}", flush=True)
    r = np.random.RandomState(rows)
    pool = make_pool(1, 400 + rows * 20 + 2 * prefix // tokens, heads, tokens, d, seed=rows)
    tables, ctx = forks(pool, prefix, [int(x) for x in r.randint(0, 130, rows)])
    tables.append([])
    ctx.append(0)  # an idle row
    q = queries(rows + 1, heads * group, d, dtype, seed=rows)
    for min_saved in (1, None, 1 << 40):
        plan, _ = check(attention(d), pool, tables, ctx, q, min_saved=min_saved)
        shared = [s for s in plan.segments if len(s[0]) > 1]
        assert shared if min_saved == 1 and rows > 1 else not shared or min_saved is None


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 1023, 1024, 1025, 2500])
def test_lengths_around_the_tiles(n):
    print(f"[gpu] shared length {n}", flush=True)
    pool = make_pool(1, 3 * 170, 2, 16, 128, seed=n)
    a = pool.allocate(pool.pages_for(n))
    lay(pool, a, n)
    # one row, and the same one three times (all full pages shared)
    check(attention(128), pool, [a], [n], queries(1, 8, 128, torch.float16, seed=n))
    check(attention(128), pool, [a, a, a], [n, n, n], queries(3, 8, 128, torch.bfloat16, seed=n))


def test_nested_prefixes_layers_and_scattered_positions():
    print("[gpu] shared nested", flush=True)
    pool = make_pool(3, 300, 2, 16, 128, seed=3)
    tables, ctx = forks(pool, 500, [40, 33])
    more = []
    for table, n in zip(tables, ctx):
        own = 500 // 16
        pool.positions[torch.tensor(table[own:], device=DEV)] += 70000  # far, and not in one run
        for kid in pool.fork(table, n, 3):
            more.append((kid + pool.allocate(1), n + 9))
    pool.max_position = 80000
    tables, ctx = [x for x, _ in more], [n for _, n in more]
    plan, _ = check(attention(128), pool, tables, ctx, queries(6, 8, 128, torch.float16), layer=2)
    assert sorted(len(s[0]) for s in plan.segments if len(s[0]) > 1) == [3, 3, 6]  # forks of forks
    attn = attention(128)
    for layer in range(3):
        check(attn, pool, tables, ctx, queries(6, 8, 128, torch.bfloat16, seed=layer), layer=layer)


@pytest.mark.parametrize("scale_mul", [2.0 ** -12, 1.0, 2000.0])
def test_value_scales_of_any_size(scale_mul):
    print(f"[gpu] shared value scales x {scale_mul}", flush=True)
    pool = make_pool(1, 120, 2, 16, 64, seed=5, scale_mul=scale_mul)
    tables, ctx = forks(pool, 400, [10, 20, 0])
    q = queries(3, 4, 64, torch.bfloat16)
    check(attention(64), pool, tables, ctx, q)


def test_query_sizes():
    """bf16 queries far outside fp16's range: a power of two is taken out of each row."""
    print("[gpu] shared query sizes", flush=True)
    pool = make_pool(1, 120, 2, 16, 128, seed=6)
    pool.key_scales.mul_(2.0 ** -6)
    tables, ctx = forks(pool, 400, [10, 20, 0, 3])
    q = queries(4, 4, 128, torch.bfloat16)
    q[1] *= 2.0 ** -60
    q[2] *= 2.0 ** 7
    q[3] = 0
    check(attention(128), pool, tables, ctx, q)


def test_agrees_with_the_unshared_paths():
    """plan() / run() over the pool's pages, and a plan whose rows share nothing."""
    print("[gpu] shared against run()", flush=True)
    pool = make_pool(1, 200, 4, 16, 128, seed=7)
    tables, ctx = forks(pool, 700, [5, 60, 17])
    attn = attention(128)
    q = queries(3, 16, 128, torch.float16)
    _, got = check(attn, pool, tables, ctx, q)
    cache = {p: pool.page(p) for x in tables for p in x}
    one = attn.run(attn.plan(cache, tables, ctx), q)
    assert (got.double() - one.double()).norm() <= 6 * U * one.double().norm()
    for b in range(3):
        alone = attn.run_shared(attn.plan_shared(pool, [tables[b]], [ctx[b]]), q[b:b + 1])
        assert (got[b:b + 1].double() - alone.double()).norm() <= 6 * U * alone.double().norm()


def test_what_lies_past_a_rows_tokens_does_not_count():
    print("[gpu] shared hidden slots", flush=True)
    pool = make_pool(1, 100, 2, 16, 128, seed=8)
    tables, ctx = forks(pool, 300, [7, 30])
    attn = attention(128)
    q = queries(2, 8, 128, torch.float16)
    plan, want = check(attn, pool, tables, ctx, q)
    for table, n in zip(tables, ctx):
        last, used = table[-1], n - (len(table) - 1) * 16
        for f in (pool.key_scales, pool.value_scales):
            f[0, last, :, used:] = float("nan")
        pool.positions[last, used:] = 1 << 30
    assert torch.equal(attn.run_shared(plan, q), want)


def test_two_streams_graph_and_repeat():
    print("[gpu] shared streams and graph", flush=True)
    pool = make_pool(1, 200, 2, 16, 128, seed=9)
    tables, ctx = forks(pool, 900, [5, 60, 17, 0])
    attn = attention(128)
    q = queries(4, 8, 128, torch.bfloat16)
    plan, want = check(attn, pool, tables, ctx, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fresh = attn.plan_shared(pool, tables, ctx, min_saved=1)
        a = attn.run_shared(fresh, q)
        b = attn.run_shared(plan, q)
    c = attn.run_shared(fresh, q)  # a plan made on the other stream
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(c, want)
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attn.run_shared(plan, q)
            with pytest.raises(RuntimeError, match="before capturing"):
                attn.run_shared(attn.plan_shared(pool, tables, ctx), q)
        graphs.append((graph, out))
    for i in range(3):
        q.mul_(0.5)
        want = attn.run_shared(plan, q)
        torch.cuda.synchronize()
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out in graphs)


def test_a_graphs_tables_outlive_longer_ones():
    """A token of a larger position makes longer rotation tables; a graph captured before reads its own."""
    from nexusquant_amd import rope
    print("[gpu] shared graph and longer tables", flush=True)
    pool = make_pool(1, 60, 2, 16, 64, seed=12)
    tables, ctx = forks(pool, 400, [5, 60])
    attn = attention(64)
    q = queries(2, 8, 64, torch.float16)
    plan, want = check(attn, pool, tables, ctx, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn.run_shared(plan, q)
    rope.clear_cache()
    pool.max_position = 9000
    again = attn.run_shared(attn.plan_shared(pool, tables, ctx, min_saved=1), q)
    fill = [torch.full((4096, 32), float("nan"), device=DEV) for _ in range(8)]  # where freed tables would have been
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)
    del fill


def test_refusals():
    print("[gpu] shared refusals", flush=True)
    pool = make_pool(2, 20, 2, 16, 64, seed=10)
    attn = attention(64)
    a = pool.allocate(4)
    plan = attn.plan_shared(pool, [a], [60])
    q = queries(1, 4, 64, torch.float16)
    for call in (lambda: attn.run_shared(plan, q.float()), lambda: attn.run_shared(plan, q[:, :3]),
                 lambda: attn.run_shared(plan, q[..., :32]), lambda: attn.run_shared(plan, q.expand(2, -1, -1)),
                 lambda: attn.run_shared(plan, q, layer=2), lambda: attn.run_shared(plan, q, layer=-1),
                 lambda: attn.run_shared(plan, q, out=torch.empty_like(q.float())),
                 lambda: attn.run_shared(plan, q, out=torch.empty(257, dtype=torch.float16, device=DEV)[1:].view(1, 4, 64)),
                 lambda: attn.run_shared(plan, queries(1, 2 * 257, 64, torch.float16))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError, match="backward"):
        attn.run_shared(plan, q.requires_grad_())
    q = q.detach()
    empty = attn.plan_shared(pool, [[], []], [0, 0])
    assert bool((attn.run_shared(empty, queries(2, 4, 64, torch.float16)) == 0).all())
    assert attn.run_shared(attn.plan_shared(pool, [], []), q[:0]).shape == (0, 4, 64)


def test_a_serving_run():
    """Prompts attended, their keys and values written to pages, branches forked and grown by decode
    steps, evicted and compacted, attended again, freed: each step against 64 bits."""
    from nexusquant_amd.attention import plan_prompts, prompt_attention
    from nexusquant_amd.ops import keep_mask
    from nexusquant_amd.page_pool import CompressedPagePool
    print("[gpu] serving run", flush=True)
    h, grp, d, t, layers = 2, 4, 128, 16, 2
    lens = [300, 77]
    g = torch.Generator().manual_seed(11)
    attn = attention(d)
    pool = CompressedPagePool(200, h, t, d, num_layers=layers, device=DEV)
    tables = [pool.allocate(pool.pages_for(n)) for n in lens]
    slots = [s for x, n in zip(tables, lens) for s in pool.slots(x, 0, n)]
    pos = np.concatenate([np.arange(n) for n in lens])
    plan = plan_prompts(lens, device=DEV)
    for layer in range(layers):
        qkv = torch.randn(sum(lens), h * (grp + 2), d, generator=g).half().to(DEV)
        q, k, v = qkv[:, :h * grp], qkv[:, h * grp:h * grp + h], qkv[:, h * grp + h:]
        prompt_attention(q, k, v, plan)
        pool.write(attn.compressor, slots, k, v, pos, layer=layer)
    # the second prompt forked into four, each branch three steps on
    branches, ctx = [tables[0]] + pool.fork(tables[1], lens[1], 4), [lens[0]] + [lens[1]] * 4
    pool.free(tables[1])
    for step in range(3):
        where = []
        for i, n in enumerate(ctx):
            if pool.pages_for(n + 1) > len(branches[i]):
                branches[i] = branches[i] + pool.allocate(1)
            where += pool.slots(branches[i], n, n + 1)
        for layer in range(layers):
            k, v = (torch.randn(5, h, d, generator=g).half().to(DEV) for _ in range(2))
            pool.write(attn.compressor, where, k, v, ctx, layer=layer)
        ctx = [n + 1 for n in ctx]
        shared = attn.plan_shared(pool, branches, ctx, min_saved=1)
        for layer in range(layers):
            check(attn, pool, branches, ctx, queries(5, h * grp, d, torch.float16, seed=step), layer=layer)
            attn.run_shared(shared, queries(5, h * grp, d, torch.float16), layer=layer)
    # half of the long sequence evicted
    imp = torch.rand(1, ctx[0], generator=g).to(DEV)
    _, kept_idx, n_kept = keep_mask(imp, 0.5)
    free = pool.free_pages
    (branches[0],), (ctx[0],) = pool.compact([branches[0]], [ctx[0]], kept_idx, n_kept, renumber=True)
    assert pool.free_pages > free and ctx[0] == int(n_kept[0])
    check(attn, pool, branches, ctx, queries(5, h * grp, d, torch.bfloat16, seed=9), layer=1)
    pool.free([p for x in branches for p in x])
    assert pool.free_pages == pool.num_pages


@pytest.mark.parametrize("heads,group,d,rows,prefix", [(8, 8, 128, 40, 4112), (8, 4, 64, 24, 17000), (4, 4, 256, 33, 9000),
                                                       (2, 32, 128, 5, 1500), (1, 200, 128, 2, 700)])
def test_wide_workgroups(heads, group, d, rows, prefix):
    """Segments of many query rows: stages decoded under the attention to the one before, several row tiles."""
    print(f"[gpu] shared wide {heads}x{group} d={d} rows={rows} prefix={prefix}", flush=True)
    pool = make_pool(1, prefix // 16 + 2 + 8 * rows, heads, 16, d, seed=rows)
    tables, ctx = forks(pool, prefix, [7 * i % 90 for i in range(rows)])
    plan, _ = check(attention(d), pool, tables, ctx, queries(rows, heads * group, d, torch.float16, seed=rows))
    assert plan.work(heads * group)[1][1] > 0  # items of many rows


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)])
@pytest.mark.parametrize("heads,group,rows,prefix", [(8, 4, 8, 1040), (2, 17, 1, 2100), (2, 16, 2, 515), (1, 32, 1, 130),
                                                     (8, 1, 31, 4100)])
def test_seventeen_to_thirty_two_query_rows(heads, group, rows, prefix, d, dtype):
    """Every wave of a workgroup has all of these rows and goes on by itself: what the others stored for it (places,
    scales in units of the chunk's largest) must be there.  (Outputs of fp16 stay clear of its subnormals.)"""
    print(f"[gpu] shared alone {heads}x{group} d={d} {dtype} rows={rows} prefix={prefix}", flush=True)
    for scale_mul in (2.0 ** -12 if dtype == torch.bfloat16 else 2000.0, 1.0):
        pool = make_pool(1, prefix // 16 + 2 + 8 * rows, heads, 16, d, seed=rows, scale_mul=scale_mul)
        tables, ctx = forks(pool, prefix, [11 * i % 70 for i in range(rows)])
        q = queries(rows, heads * group, d, dtype, seed=prefix)
        plan, want = check(attention(d), pool, tables, ctx, q)
        items = plan.work(heads * group)[1]
        assert items[1] == 0 and items[0] > items[2]  # some are of neither many rows nor few
        attn = attention(d)
        for _ in range(3):
            assert torch.equal(attn.run_shared(plan, q), want)


def test_two_attentions_over_one_plan():
    """Layers of local and global rotation: each attention reads its own tables, and the plan keeps one of each."""
    from nexusquant_amd.vllm_backend import NexusQuantKVCompressor, NexusQuantPagedAttention
    print("[gpu] shared two attentions", flush=True)
    pool = make_pool(1, 60, 2, 16, 64, seed=13)
    tables, ctx = forks(pool, 400, [5, 60])
    one, two = attention(64), NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=64, bits=3, rope_base=10000.0))
    q = queries(2, 8, 64, torch.float16)
    plan, want = check(one, pool, tables, ctx, q)
    other = two.run_shared(plan, q)
    assert not torch.equal(other, want)
    for _ in range(20):
        assert torch.equal(one.run_shared(plan, q), want) and torch.equal(two.run_shared(plan, q), other)
    assert len(plan._tables) == 2


def test_longer_tables_are_made_before_a_capture():
    """A larger position than the tables reach: refused in a capture, which stays whole; one call before it, and it is not."""
    from nexusquant_amd import rope
    print("[gpu] shared longer tables in a capture", flush=True)
    rope.clear_cache()
    pool = make_pool(1, 60, 2, 16, 64, seed=14)
    tables, ctx = forks(pool, 400, [5, 60])
    attn = attention(64)
    q = queries(2, 8, 64, torch.float16)
    plan, want = check(attn, pool, tables, ctx, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn.run_shared(plan, q)
        pool.max_position = 5000
        with pytest.raises(RuntimeError, match="before capturing"):
            attn.run_shared(plan, q)
    longer = torch.cuda.CUDAGraph()
    attn.run_shared(plan, q)
    with torch.cuda.graph(longer):
        out2 = attn.run_shared(plan, q)
    for _ in range(3):
        out.zero_()
        out2.zero_()
        graph.replay()
        longer.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group,rows,prefix,kind", [(2, 4, 3, 1500, "few"), (2, 4, 8, 1500, "some"),
                                                          (8, 4, 24, 4096, "some"), (8, 8, 40, 6000, "many")])
def test_values_are_exact_and_weights_of_few_rows_nearly(heads, group, rows, prefix, kind, d):
    """Queries of zero weigh all tokens alike, so keys' roundings do not count, and values' would be all there is to see.
    Values are exact codes: a weight times its scale is rounded (U; U^2 for few rows, which keep what that rounds off, in fp16
    too), or is off by half of fp16's smallest step where the chunk's largest is at least 2^6: 2^-31 of the largest a token, 2^-20
    for a chunk's 2048.  Sums in fp32, in the transformed domain: 2^-20 of the tokens' 2-norms."""
    print(f"[gpu] shared values {kind} {heads}x{group} d={d} rows={rows} prefix={prefix}", flush=True)
    pool = make_pool(1, prefix // 16 + 2 + 8 * rows, heads, 16, d, seed=rows + d)
    tables, ctx = forks(pool, prefix, [0] * rows)
    q = torch.zeros(rows, heads * group, d, dtype=torch.float16, device=DEV)
    attn = attention(d)
    plan = attn.plan_shared(pool, tables, ctx, min_saved=1)
    n_items, n_many, n_few, _ = plan.work(heads * group)[1]
    assert {"few": n_few == n_items, "some": n_many == 0 and n_few < n_items, "many": n_many > 0}[kind]
    got = attn.run_shared(plan, q)
    w = U ** 2 if kind == "few" else U
    for b in range(0, rows, 7):
        pages = torch.tensor(tables[b], device=DEV)
        v = pool.value_codes[0, pages].double() / 2 * pool.value_scales[0, pages].double()[..., None]
        v = walsh(v.transpose(0, 1).reshape(heads, -1, d)[:, :ctx[b]])
        want = v.mean(1)
        tol = (w + 2 ** -20) * v.abs().mean(1) + 2 ** -19 * v.norm(dim=-1).amax(-1, keepdim=True)
        want, tol = (x.repeat_interleave(group, 0) for x in (want, tol))
        off = (got[b].double() - want).abs() - tol - (U * want.abs()).clamp_min(2.0 ** -25)
        assert bool((off <= 0).all()), (b, off.max().item())
