"""The serving operators over compressed pages, as timed cases in two forms.

Families:
  fork     CompressedPagePool.fork + free: a sequence branches, sharing its full pages
  copy     CompressedPagePool.copy_pages: whole pages duplicated in every layer
  compact  CompressedPagePool.compact: the tokens that a keep mask leaves, moved into fewer pages
  shared   NexusQuantPagedAttention.run_shared: one decode step of rows that begin with the same pages
  prompt   attention.prompt_attention: causal attention over packed prompts
With `own` false each is computed in elementary torch operations in 32 bits; with `own` true through the
package's entry points.  Inputs are synthetic: lattice codes drawn from a clipped normal distribution, keys
without rotation as pages hold them, queries N(0, 1).
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BASE = 500000.0


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # A sampled sequence branches into four beams: one part-filled page a beam, all 32 layers.
        dict(name="fork_beam", family="fork", layers=32, heads=8, head_dim=128, tokens=16, length=1000, branches=3),
        # A batch of prompts branches for parallel sampling, pages of 32 tokens, head_dim 64.
        dict(name="fork_sampling", family="fork", layers=24, heads=4, head_dim=64, tokens=32, length=4099, branches=48),
        # A gigabyte of pages moved aside: a swap within the pool, every layer.
        dict(name="copy_pages_1k", family="copy", layers=16, heads=8, head_dim=128, tokens=16, pages=1024),
        # One layer's eviction after a prefill, length off the page grid.
        dict(name="compact_layer_8k", family="compact", layers=1, heads=8, head_dim=128, tokens=16, batch=1,
             longest=8191, ragged=0, rate=0.6, renumber=False),
        # A ragged batch truncated in every layer, keys at their new positions.
        dict(name="compact_batch_8k", family="compact", layers=16, heads=8, head_dim=128, tokens=16, batch=4,
             longest=8192, ragged=7, rate=0.75, renumber=True),
        # Four samples of one short prompt: launches and latency count.
        dict(name="shared_few_1k", family="shared", heads=8, group=4, head_dim=128, tokens=16, rows=4, groups=1,
             prefix=1000, suffix=40, ragged=1, idle=False, dtype="fp16", bits=2),
        # A chat service's system prompt under 32 ragged conversations, an idle row in the batch.
        dict(name="shared_chat_4k", family="shared", heads=8, group=4, head_dim=128, tokens=16, rows=32, groups=1,
             prefix=4099, suffix=512, ragged=2, idle=True, dtype="bf16", bits=3),
        # Many questions about one long document, 64 query heads over 8 kv heads.
        dict(name="shared_long_32k", family="shared", heads=8, group=8, head_dim=128, tokens=16, rows=64, groups=1,
             prefix=32768, suffix=1024, ragged=3, idle=False, dtype="fp16", bits=2),
        # Two documents, as many kv heads as query heads, head_dim 64.
        dict(name="shared_two_8k", family="shared", heads=32, group=1, head_dim=64, tokens=32, rows=16, groups=2,
             prefix=8192, suffix=300, ragged=4, idle=False, dtype="bf16", bits=4),
        # A handful of short prompts, one of a single token.
        dict(name="prompt_short", family="prompt", heads=8, group=4, head_dim=128, batch=5, longest=190, ragged=5,
             window=0, dtype="bf16"),
        # A serving prefill: eight ragged prompts of up to 4096 tokens.
        dict(name="prompt_packed_4k", family="prompt", heads=8, group=4, head_dim=128, batch=8, longest=4096, ragged=6,
             window=0, dtype="bf16"),
        # One long prompt.
        dict(name="prompt_long_16k", family="prompt", heads=8, group=4, head_dim=128, batch=1, longest=16384, ragged=0,
             window=0, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["fork", "copy", "compact", "compact", "shared", "shared", "shared", "prompt", "prompt",
                         "prompt"])
    heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    d = rng.choice([64, 128, 128, 256])
    tokens = rng.choice([8, 16, 16, 24, 32, 64])
    layers = _log_int(rng, 1, 40)
    row = heads * tokens * (2 * d + 4)  # bytes of a page in one layer
    if family == "fork":
        return dict(family=family, layers=layers, heads=heads, head_dim=d, tokens=tokens,
                    length=rng.randint(1, 5000), branches=_log_int(rng, 1, max(1, min(256, (1 << 28) // (layers * row)))))
    if family == "copy":
        return dict(family=family, layers=layers, heads=heads, head_dim=d, tokens=tokens,
                    pages=_log_int(rng, 1, max(1, min(4096, (1 << 29) // (layers * row)))))
    if family == "compact":
        batch = _log_int(rng, 1, 16)
        most = (1 << 30) // (layers * heads * (2 * d + 4) * batch)
        return dict(family=family, layers=layers, heads=heads, head_dim=d, tokens=tokens, batch=batch,
                    longest=_log_int(rng, 1, max(2, min(60000, most))), ragged=rng.randint(0, 99),
                    rate=rng.choice([0.0, 0.25, 0.5, 0.6, 0.8, 0.95]), renumber=rng.random() < 0.5)
    if family == "shared":
        dtype = rng.choice(["fp16", "bf16"])
        group = rng.choice([1, 2, 4, 8])
        while heads * group > 64:
            group //= 2
        groups = rng.choice([1, 1, 1, 2, 3])
        rows = groups * _log_int(rng, 1, 64 // groups)
        prefix = _log_int(rng, 1, 60000)
        while rows * heads * group * prefix * d > 64 * 64 * 32768 * 128:
            prefix //= 2
        while groups * heads * prefix * d > 8 * 60000 * 128:
            prefix //= 2
        suffix = _log_int(rng, 1, 1500)
        while rows * heads * group * suffix * d > 64 * 64 * 1024 * 128:
            suffix //= 2
        return dict(family=family, heads=heads, group=group, head_dim=d, tokens=tokens, rows=rows, groups=groups,
                    prefix=max(1, prefix), suffix=max(1, suffix), ragged=rng.randint(1, 99), idle=rng.random() < 0.3,
                    dtype=dtype, bits=rng.choice([2, 3, 4]))
    group = rng.choice([1, 2, 4, 4, 8])
    while heads * group > 64:
        group //= 2
    batch = _log_int(rng, 1, 24)
    longest = _log_int(rng, 1, 12000)
    while batch * heads * group * longest * longest * d > 32 * 16384 * 16384 * 128:
        longest = longest * 3 // 4
    return dict(family=family, heads=heads, group=group, head_dim=d, batch=batch, longest=max(1, longest),
                ragged=rng.randint(0, 99), window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]),
                dtype=rng.choice(["fp16", "bf16"]))


def _ragged(n, longest, ragged):
    """n lengths of 1 .. longest, the first the longest; all of them for ragged 0."""
    r = random.Random(ragged)
    return [longest] + [longest if ragged == 0 else r.randint(1, longest) for _ in range(n - 1)]


def _suffixes(case):
    """Tokens that each row has past its prefix, some none; None for an idle row, which has no prefix either."""
    lens = _ragged(case["rows"], case["suffix"], case["ragged"])
    if len(lens) > 2:
        lens[1] = 0
    return lens + [None] if case["idle"] else lens


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs --

def _codes(g, shape, bound):
    x = torch.randn(shape, device=DEV, generator=g).mul_(bound / 3.0)
    return x.round_().clamp_(-bound, bound).to(torch.int8)


def _pool_fields(g, layers, pages, heads, tokens, d, levels):
    shape = (layers, pages, heads, tokens)
    ks = (torch.rand(shape, device=DEV, generator=g) * 4.0 + 2.0) / levels
    vs = (torch.rand(shape, device=DEV, generator=g) * 2.0 + 1.0) / levels
    return dict(key_codes=_codes(g, shape + (d,), levels), value_codes=_codes(g, shape + (d,), levels),
                key_scales=ks.half(), value_scales=vs.half(),
                positions=torch.zeros(pages, tokens, dtype=torch.int32, device=DEV))


def _own_pool(f):
    from nexusquant_amd.page_pool import CompressedPagePool
    layers, pages, heads, tokens, d = f["key_codes"].shape
    return CompressedPagePool.from_tensors(**f)


def _lay_positions(positions, tables, lens, t):
    for table, n in zip(tables, lens):
        flat = torch.arange(len(table) * t, dtype=torch.int32, device=DEV)
        positions[torch.tensor(table, device=DEV)] = (flat * (flat < n)).view(-1, t)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    fam, d = case["family"], case["head_dim"]
    if fam == "prompt":
        lens = _ragged(case["batch"], case["longest"], case["ragged"])
        hq, hkv = case["heads"] * case["group"], case["heads"]
        # q, k and v as a fused projection leaves them: slices of one row a token
        qkv = torch.randn(sum(lens), hq + 2 * hkv, d, device=DEV, generator=g).to(DTYPES[case["dtype"]])
        st = dict(case=case, lens=lens, q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
        if own:
            from nexusquant_amd.attention import plan_prompts
            st["plan"] = plan_prompts(lens, device=DEV)
        else:
            starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
            st["starts"] = torch.tensor(starts, device=DEV)
            st["lengths"] = torch.tensor(lens, device=DEV)
        return st
    t = case["tokens"]
    levels = 2 ** case.get("bits", 3)
    if fam == "fork":
        n = _ceil(case["length"], t)
        f = _pool_fields(g, case["layers"], n + case["branches"] + 8, case["heads"], t, d, levels)
        _lay_positions(f["positions"], [list(range(n))], [case["length"]], t)
        st = dict(case=case, fields=f, table=list(range(n)))
        if own:
            st["pool"] = _own_pool(f)
            st["table"] = st["pool"].allocate(n)
        return st
    if fam == "copy":
        n = case["pages"]
        f = _pool_fields(g, case["layers"], 2 * n + 8, case["heads"], t, d, levels)
        _lay_positions(f["positions"], [list(range(n))], [n * t], t)
        order = torch.randperm(2 * n, generator=torch.Generator().manual_seed(int(seed))).tolist()
        st = dict(case=case, fields=f, src=order[:n], dst=order[n:])
        if own:
            st["pool"] = _own_pool(f)
            st["pool"].allocate(2 * n)
        return st
    if fam == "compact":
        lens = _ragged(case["batch"], case["longest"], case["ragged"])
        pages = [_ceil(n, t) for n in lens]
        f = _pool_fields(g, case["layers"], 2 * sum(pages) + 8, case["heads"], t, d, levels)
        at = np.concatenate([[0], np.cumsum(pages)]).tolist()
        tables = [list(range(at[i], at[i + 1])) for i in range(len(lens))]
        _lay_positions(f["positions"], tables, lens, t)
        # the list of a keep mask: kept positions ascending, then the evicted ones descending
        longest = max(lens)
        idx = torch.zeros(len(lens), longest, dtype=torch.int32, device=DEV)
        kept = []
        for i, n in enumerate(lens):
            score = torch.rand(n, device=DEV, generator=g)
            score[:1] = 2.0
            score[max(0, n - 32):] = 2.0
            k = min(n, max(min(n, 33), int(n * (1.0 - case["rate"]))))
            order = score.argsort(descending=True, stable=True)
            idx[i, :n] = torch.cat([order[:k].sort().values, order[k:].sort(descending=True).values]).int()
            kept.append(k)
        st = dict(case=case, fields=f, tables=tables, lens=lens, kept_idx=idx,
                  n_kept=torch.tensor(kept, dtype=torch.int32, device=DEV))
        if own:
            st["pool"] = _own_pool(f)
            st["tables"] = [st["pool"].allocate(n) for n in pages]
        return st
    # shared: rows 0 .. rows - 1 take the prefixes in turn, then their own pages
    suffix = _suffixes(case)
    n, groups = case["prefix"], case["groups"]
    full = n // t  # the prefix's last page is copied to each branch, so what is shared are its full pages
    own_pages = [0 if s is None else _ceil(n - full * t + s, t) for s in suffix]
    f = _pool_fields(g, 1, groups * full + sum(own_pages) + 8, case["heads"], t, d, levels)
    heads_pages = [list(range(i * full, (i + 1) * full)) for i in range(groups)]
    at = np.concatenate([[0], np.cumsum(own_pages)]) + groups * full
    tables = [[] if s is None else heads_pages[i % groups] + list(range(int(at[i]), int(at[i + 1])))
              for i, s in enumerate(suffix)]
    ctx = [0 if s is None else n + s for s in suffix]
    _lay_positions(f["positions"], [x for x in tables if x], [c for c in ctx if c], t)
    q = torch.randn(len(suffix), case["heads"] * case["group"], d, device=DEV, generator=g).to(DTYPES[case["dtype"]])
    st = dict(case=case, fields=f, q=q, tables=tables, ctx=ctx)
    if own:
        from nexusquant_amd.vllm_backend import NexusQuantKVCompressor, NexusQuantPagedAttention
        st["pool"] = _own_pool(f)
        st["pool"].allocate(groups * full + sum(own_pages))
        st["attn"] = NexusQuantPagedAttention(NexusQuantKVCompressor(head_dim=d, bits=case["bits"], rope_base=BASE))
        st["plan"] = st["attn"].plan_shared(st["pool"], tables, ctx)
    else:
        live = [x for x in tables if x]
        wide = max(len(x) for x in live) - full
        st["prefix_pages"] = torch.tensor(heads_pages, dtype=torch.long, device=DEV).view(groups, full)
        st["row_pages"] = torch.tensor([x[full:] + [0] * (wide - len(x) + full) for x in live], dtype=torch.long,
                                       device=DEV).view(len(live), wide)
        st["row_tokens"] = torch.tensor([c - full * t for c in ctx if c], device=DEV)
        st["hadamard"] = _hadamard(d, torch.float32)
        st["inv_freq"] = _inv_freq(d)
    return st


# -------------------------------------------------------------- plain forms --

def _inv_freq(d):
    return (1.0 / (BASE ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)


def _hadamard(d, dtype):
    """The orthonormal Sylvester matrix: (-1)^popcount(i & j) / sqrt(d)."""
    i = torch.arange(d, device=DEV)
    x = i[:, None] & i[None, :]
    for s in (4, 2, 1):
        x = x ^ (x >> s)
    return ((1 - 2 * (x & 1)).to(torch.float64) / math.sqrt(d)).to(dtype)


def _unrotated(codes, scales, hadamard):
    return torch.matmul(codes.float() * 0.5 * scales.float()[..., None], hadamard)


def _rotated(x, positions, inv_freq):
    ang = (positions.float()[..., None] * inv_freq).double()  # the angle is fp32, as models form it
    c, s = ang.cos().float(), ang.sin().float()
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_shared(st):
    case, f = st["case"], st["fields"]
    t, d, h, grp, groups = case["tokens"], case["head_dim"], case["heads"], case["group"], case["groups"]
    q = st["q"].float()
    rows = case["rows"]
    scale = 1.0 / math.sqrt(d)

    def tokens_of(name, pages):  # [..., pages] -> [..., heads, pages * tokens, d]
        codes, scales = f[name + "_codes"][0][pages], f[name + "_scales"][0][pages]
        x = _unrotated(codes, scales, st["hadamard"])
        if name == "key":
            x = _rotated(x, f["positions"][pages][..., None, :], st["inv_freq"])
        x = x.transpose(-4, -3)  # [..., heads, pages, tokens, d]
        return x.reshape(*x.shape[:-3], x.shape[-3] * t, d)

    pre, per = st["prefix_pages"], st["row_pages"]
    kp, vp = tokens_of("key", pre), tokens_of("value", pre)          # [groups, heads, prefix, d]
    ks, vs = tokens_of("key", per), tokens_of("value", per)          # [rows, heads, own, d]
    live = q[:rows].view(rows, h, grp, d)
    # rows of a group side by side: row r belongs to group r % groups
    each = rows // groups
    side = live.view(each, groups, h, grp, d).permute(1, 2, 0, 3, 4).reshape(groups, h, each * grp, d)
    sp = torch.matmul(side, kp.transpose(-1, -2).contiguous()) * scale
    sp = sp.reshape(groups, h, each, grp, sp.shape[-1])
    ss = torch.matmul(live, ks.transpose(-1, -2).contiguous()) * scale    # [rows, heads, group, own]
    hidden = torch.arange(ss.shape[-1], device=DEV)[None, :] >= st["row_tokens"][:, None]
    ss.masked_fill_(hidden[:, None, None, :], -math.inf)

    def by_group(x):  # [rows, heads, group, n] -> [groups, heads, rows / groups, group, n]
        return x.reshape(each, groups, h, grp, x.shape[-1]).permute(1, 2, 0, 3, 4)

    if ss.shape[-1]:
        m = by_group(ss.amax(-1, keepdim=True))
        m = torch.maximum(m, sp.amax(-1, keepdim=True)) if sp.shape[-1] else m
    else:
        m = sp.amax(-1, keepdim=True)
    m_rows = m.permute(2, 0, 1, 3, 4).reshape(rows, h, grp, 1)
    ep, es = torch.exp(sp - m), torch.exp(ss - m_rows)
    num = torch.matmul(ep.reshape(groups, h, each * grp, ep.shape[-1]), vp).reshape(groups, h, each, grp, d)
    num = num.permute(2, 0, 1, 3, 4).reshape(rows, h, grp, d) + torch.matmul(es, vs)
    den = ep.sum(-1, keepdim=True).permute(2, 0, 1, 3, 4).reshape(rows, h, grp, 1) + es.sum(-1, keepdim=True)
    out = torch.zeros_like(q)
    out[:rows] = (num / den).reshape(rows, h * grp, d)
    return out.to(st["q"].dtype)


def _plain_prompt(st):
    case = st["case"]
    h, grp, d, longest = case["heads"], case["group"], case["head_dim"], case["longest"]
    q, k, v, starts, lens = st["q"], st["k"], st["v"], st["starts"], st["lengths"]
    batch, total = len(st["lens"]), q.shape[0]
    pos = torch.arange(longest, device=DEV)
    at = (starts[:, None] + pos).clamp_(max=total - 1)               # [batch, longest] padded
    qp = q[at].float().view(batch, longest, h, grp, d).permute(0, 2, 3, 1, 4).reshape(batch, h, grp * longest, d)
    kp = k[at].float().permute(0, 2, 3, 1).contiguous()              # [batch, heads, d, longest]
    vp = v[at].float().permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(qp, kp).mul_(1.0 / math.sqrt(d)).view(batch, h, grp, longest, longest)
    hidden = pos[None, :] > pos[:, None]
    if case["window"]:
        hidden |= pos[None, :] <= pos[:, None] - case["window"]
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s.div_(s.sum(-1, keepdim=True))
    o = torch.matmul(s.view(batch, h, grp * longest, longest), vp).view(batch, h, grp, longest, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, longest, h * grp, d)
    real = pos[None, :] < lens[:, None]
    return o[real].to(q.dtype)


def _plain_copy(f, src, dst):
    src, dst = torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV)
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        f[name][:, dst] = f[name][:, src]
    f["positions"][dst] = f["positions"][src]


def _plain_compact(st):
    case, f, t = st["case"], st["fields"], st["case"]["tokens"]
    kept = st["n_kept"].tolist()
    first = sum(len(x) for x in st["tables"])
    n_pages = [_ceil(k, t) for k in kept]
    at = np.concatenate([[0], np.cumsum(n_pages)]) + first
    tables = [list(range(int(at[i]), int(at[i + 1]))) for i in range(len(kept))]
    wide = max(len(x) for x in st["tables"])
    src_tab = torch.tensor([x + [0] * (wide - len(x)) for x in st["tables"]], device=DEV)
    dst_tab = torch.tensor([x + [0] * (wide - len(x)) for x in tables], device=DEV)
    j = torch.arange(st["kept_idx"].shape[1], device=DEV)
    b, j = torch.nonzero(j[None, :] < st["n_kept"][:, None], as_tuple=True)
    i = st["kept_idx"][b, j].long()
    sp, so = src_tab[b, i // t], i % t
    dp, do = dst_tab[b, j // t], j % t
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        x = f[name]
        x[:, dp, :, do] = x[:, sp, :, so]
    f["positions"][dp, do] = j.int() if case["renumber"] else f["positions"][sp, so]
    return tables, kept


# --------------------------------------------------------------------- run --

def _fields(f):
    return [f[k] for k in ("key_codes", "value_codes", "key_scales", "value_scales", "positions")]


def run(st):
    case = st["case"]
    fam = case["family"]
    if fam == "fork":
        if own:
            kids = st["pool"].fork(st["table"], case["length"], case["branches"])
            st["pool"].free([p for kid in kids for p in kid])  # the branches end
        else:
            n, kids = len(st["table"]), [list(st["table"]) for _ in range(case["branches"])]
            if case["length"] % case["tokens"]:
                kids = [kid[:-1] + [n + i] for i, kid in enumerate(kids)]
                _plain_copy(st["fields"], [st["table"][-1]] * len(kids), [kid[-1] for kid in kids])
        return [_fields(st["fields"]), np.array(kids)]
    if fam == "copy":
        if own:
            st["pool"].copy_pages(st["src"], st["dst"])
        else:
            _plain_copy(st["fields"], st["src"], st["dst"])
        return _fields(st["fields"])
    if fam == "compact":
        if own:
            pool = st["pool"]
            pool.retain([p for x in st["tables"] for p in x])  # the whole sequences stay, under another branch
            tables, lens = pool.compact(st["tables"], st["lens"], st["kept_idx"], st["n_kept"],
                                        renumber=case["renumber"])
            pool.free([p for x in tables for p in x])
        else:
            tables, lens = _plain_compact(st)
        return [_fields(st["fields"]), np.array([p for x in tables for p in x]), np.array(lens)]
    if fam == "shared":
        return st["attn"].run_shared(st["plan"], st["q"]) if own else _plain_shared(st)
    if own:
        from nexusquant_amd.attention import prompt_attention
        return prompt_attention(st["q"], st["k"], st["v"], st["plan"], sliding_window=case["window"] or None)
    return _plain_prompt(st)


def work(case):
    fam, d, h = case["family"], case["head_dim"], case["heads"]
    row = 2 * d + 4  # bytes of a token and head in one layer
    if fam in ("fork", "copy"):
        if fam == "copy":
            src = dst = case["pages"]
        else:
            src = 1 if case["length"] % case["tokens"] else 0
            dst = src * case["branches"]
        return {"bytes": max(1, (src + dst) * case["tokens"] * (case["layers"] * h * row + 4)), "flops": 0}
    if fam == "compact":
        n = sum(min(k, max(min(k, 33), int(k * (1.0 - case["rate"]))))
                for k in _ragged(case["batch"], case["longest"], case["ragged"]))
        return {"bytes": 2 * n * (case["layers"] * h * row + 4) + 4 * n, "flops": 0}
    hq = h * case["group"]
    if fam == "shared":
        suffix = [s for s in _suffixes(case) if s is not None]
        n, t = case["prefix"], case["tokens"]
        full = n // t * t
        tokens = case["groups"] * full + sum(n - full + s for s in suffix)
        return {"bytes": tokens * (h * row + 4) + 2 * 2 * len(_suffixes(case)) * hq * d,
                "flops": 4 * hq * d * sum(n + s for s in suffix)}
    w = case["window"]
    lens = _ragged(case["batch"], case["longest"], case["ragged"])
    pairs = sum(n * (n + 1) // 2 if not w or w >= n else w * (w + 1) // 2 + (n - w) * w for n in lens)
    return {"bytes": sum(lens) * 2 * d * (2 * hq + 2 * h), "flops": 4 * hq * d * pairs}


# ------------------------------------------------------------------- exact --

def _walsh(x):
    """The orthonormal Walsh-Hadamard transform of the last axis, by butterflies."""
    d = x.shape[-1]
    step = 1
    while step < d:
        y = x.reshape(*x.shape[:-1], d // (2 * step), 2, step)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).reshape(*x.shape)
        step *= 2
    return x / math.sqrt(d)


def exact(case, seed):
    fam, d = case["family"], case["head_dim"]
    if fam not in ("shared", "prompt"):
        return None  # bytes are moved: nothing is computed
    st = prepare(case, seed)
    if fam == "prompt":
        out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
        a = 0
        for n in st["lens"]:
            i = torch.arange(n, device=DEV)
            seen = i[:, None] >= i
            if case["window"]:
                seen &= i[:, None] - i < case["window"]
            for head in range(out.shape[1]):
                q = st["q"][a:a + n, head].double()
                k, v = (st[x][a:a + n, head // case["group"]].double() for x in "kv")
                logit = torch.where(seen, q @ k.T / math.sqrt(d), -math.inf)
                out[a:a + n, head] = torch.softmax(logit, dim=-1) @ v
            a += n
        return out
    f = st["fields"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    freq = _inv_freq(d)
    for r, (table, n) in enumerate(zip(st["tables"], st["ctx"])):
        if not n:
            continue
        pages = torch.tensor(table, device=DEV)

        def whole(name):  # [heads, n, d]
            x = f[name + "_codes"][0, pages].double() / 2 * f[name + "_scales"][0, pages].double().unsqueeze(-1)
            return _walsh(x.transpose(0, 1).reshape(case["heads"], -1, d)[:, :n])

        k, v = whole("key"), whole("value")
        ang = (f["positions"][pages].reshape(-1)[:n].float().unsqueeze(-1) * freq).double()
        z = torch.complex(k[..., :d // 2], k[..., d // 2:]) * torch.polar(torch.ones_like(ang), ang)
        k = torch.cat([z.real, z.imag], dim=-1)
        q = st["q"][r].double().view(case["heads"], case["group"], d)
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2)) / math.sqrt(d), dim=-1)
        out[r] = torch.matmul(p, v).reshape(-1, d)
    return out
