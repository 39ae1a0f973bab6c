"""The operators of a cache held in 4 bits, as timed cases in two forms.

Families:
  rotate   plan_rotation + rotate: rotary positions with one or several axes, forward, or forward and gradients
  append   FourBitPagePool.append + read: new tokens rotated, transformed and encoded into their slots, queries rotated
           on the way; then what the slots stand for
  attend   FourBitPagePool.attend: decode steps, several new tokens a sequence over a cached past (causal), and queries
           that see all of another sequence's tokens (an encoder's states)
With `own` false each is computed in elementary torch operations; with `own` true through the package's entry points.

The 4-bit form of a vector x of d coordinates: t = H x (H the orthonormal Sylvester matrix), s = fp16(max|t| / 7.5),
n = clamp(floor(t / s + 8.5), 0, 15); it stands for H ((n - 8) s).  Keys are stored rotated.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BASE = 500000.0


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # The patches of one image, positions of height and width.
        dict(name="rotate_image_1k", family="rotate", axes=2, interleaved=False, rows=1024, heads=8, group=2, head_dim=64,
             dtype="fp16", grad=False),
        # A video's tokens, positions of time, height and width, the axes' frequencies in turn.
        dict(name="rotate_video_16k", family="rotate", axes=3, interleaved=True, rows=16384, heads=8, group=4, head_dim=128,
             dtype="bf16", grad=False),
        # A training step's rotation of 4 x 2047 tokens, gradients too.
        dict(name="rotate_train_8k", family="rotate", axes=3, interleaved=False, rows=8188, heads=8, group=4, head_dim=128,
             dtype="fp32", grad=True),
        # One decode step of 32 sequences: latency counts.
        dict(name="append_step_32", family="append", heads=8, group=4, head_dim=128, tokens=16, batch=32, new=1, ragged=0,
             axes=1, padded=1, dtype="bf16"),
        # Ragged prompts with images among them.
        dict(name="append_prompts_8k", family="append", heads=8, group=4, head_dim=128, tokens=16, batch=4, new=4099, ragged=3,
             axes=3, padded=0, dtype="fp16"),
        # Four short conversations: launches and latency count.
        dict(name="decode_few_1k", family="attend", heads=8, group=4, head_dim=128, tokens=16, batch=4, context=1000,
             queries=1, causal=True, window=0, ragged=1, idle=False, dtype="fp16"),
        # A serving batch, ragged, an idle row in it.
        dict(name="decode_batch_8k", family="attend", heads=8, group=4, head_dim=128, tokens=16, batch=64, context=8192,
             queries=1, causal=True, window=0, ragged=2, idle=True, dtype="bf16"),
        # One document of 128 K tokens.
        dict(name="decode_long_128k", family="attend", heads=8, group=8, head_dim=128, tokens=16, batch=1, context=131072,
             queries=1, causal=True, window=0, ragged=0, idle=False, dtype="fp16"),
        # Four drafted tokens and the one before them, verified at once, a sliding window.
        dict(name="verify_5_of_4k", family="attend", heads=8, group=4, head_dim=128, tokens=16, batch=16, context=4099,
             queries=5, causal=True, window=4096, ragged=4, idle=False, dtype="bf16"),
        # Chunks of 512 tokens of long prompts over what the cache holds of them.
        dict(name="chunk_512_of_16k", family="attend", heads=8, group=4, head_dim=128, tokens=16, batch=4, context=16384,
             queries=512, causal=True, window=0, ragged=5, idle=False, dtype="bf16"),
        # Decoder tokens over their encoder's states, one at a time.
        dict(name="cross_step_1500", family="attend", heads=20, group=1, head_dim=64, tokens=32, batch=24, context=1500,
             queries=1, causal=False, window=0, ragged=6, idle=False, dtype="fp16"),
        # The decoder's first tokens over the encoder's states.
        dict(name="cross_prompt_1500", family="attend", heads=20, group=1, head_dim=64, tokens=32, batch=24, context=1500,
             queries=223, causal=False, window=0, ragged=7, idle=True, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["rotate", "append", "append", "attend", "attend", "attend", "attend"])
    heads = rng.choice([1, 2, 4, 8, 8, 16, 20])
    group = rng.choice([1, 1, 2, 4, 4, 5, 8])
    d = rng.choice([64, 128, 128, 256])
    tokens = rng.choice([8, 16, 16, 24, 32, 64])
    width = heads * (group + 2) * d
    if family == "rotate":
        grad = rng.random() < 0.4
        return dict(family=family, axes=rng.choice([1, 2, 3, 3, 4]), interleaved=rng.random() < 0.5,
                    rows=_log_int(rng, 1, max(2, min(20000, (1 << 25) // (width * (2 if grad else 1))))), heads=heads,
                    group=group, head_dim=d, dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]), grad=grad)
    if family == "append":
        batch = _log_int(rng, 1, 64)
        return dict(family=family, heads=heads, group=group, head_dim=d, tokens=tokens, batch=batch,
                    new=_log_int(rng, 1, max(2, min(9000, (1 << 25) // (width * batch)))), ragged=rng.randint(1, 99),
                    axes=rng.choice([0, 1, 1, 3]), padded=rng.choice([0, 0, 3]), dtype=rng.choice(["fp16", "bf16"]))
    batch = _log_int(rng, 1, 64)
    context = _log_int(rng, 1, 130000)
    while batch * heads * context * d > 64 * 8 * 8192 * 128:
        context = context * 3 // 4
    queries = rng.choice([1, 1, 1, rng.randint(2, 9), _log_int(rng, 10, 600)])
    causal = rng.random() < 0.7
    if causal:
        queries = min(queries, context)
    while queries > 1 and batch * heads * group * queries * context * d > 4 * 32 * 512 * 16384 * 128:
        queries = (queries + 1) // 2
    return dict(family=family, heads=heads, group=group, head_dim=d, tokens=tokens, batch=batch, context=max(1, context),
                queries=queries, causal=causal, window=rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]) if causal else 0,
                ragged=rng.randint(1, 99), idle=rng.random() < 0.3, dtype=rng.choice(["fp16", "bf16"]))


def _ragged(n, longest, ragged):
    """n lengths of 1 .. longest, the first the longest; all of them for ragged 0."""
    r = random.Random(ragged)
    return [longest] + [longest if ragged == 0 else r.randint(1, longest) for _ in range(n - 1)]


def _attended(case):
    """(tokens, queries) of each sequence; an idle one has queries but no tokens, or nothing where it would be causal."""
    lens = _ragged(case["batch"], case["context"], case["ragged"])
    new = _ragged(case["batch"], case["queries"], case["ragged"] + 100)
    got = [(n, min(q, n) if case["causal"] else q) for n, q in zip(lens, new)]
    return got + [(0, 0 if case["causal"] else case["queries"])] if case["idle"] else got


def _ceil(a, b):
    return -(-a // b)


def _sections(d, axes):
    """How many of the d / 2 frequencies each axis has."""
    rest = [15 * d // (32 * axes)] * (axes - 1)
    return [d // 2 - sum(rest)] + rest


def _axis_of(d, axes, interleaved):
    """The axis of each frequency."""
    sections = _sections(d, axes)
    if not interleaved:
        return np.repeat(np.arange(axes), sections)
    i = np.arange(d // 2)
    return np.where(i < axes * np.array(sections)[i % axes], i % axes, 0)


# ------------------------------------------------------------------ inputs --

def _inv_freq(d):
    return (1.0 / (BASE ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)


def _positions(rows, axes, start):
    """int32 [axes, rows]: a line of tokens for one axis, a grid of 24 x 32 patches a frame for several."""
    i = torch.arange(rows, device=DEV)
    w, h, t = i % 32, i // 32 % 24, i // 768
    return (torch.stack([i] if axes == 1 else ([t, h, w, i] if axes > 2 else [h, w])[:axes]) + start).to(torch.int32)


def _fields(g, pages, heads, tokens, d):
    """A layer's pages as past tokens leave them: codes of normal variates, their scales."""
    shape = (1, pages, heads, tokens)
    out = {}
    for name in ("key", "value"):
        byte = torch.zeros(shape + (d // 2,), dtype=torch.uint8, device=DEV)
        for shift in (0, 4):
            n = torch.empty(byte.shape, dtype=torch.float16, device=DEV).normal_(8.5, 2.6, generator=g)
            byte |= n.floor_().clamp_(0, 15).to(torch.uint8) << shift
        out[name + "_codes"] = byte
        out[name + "_scales"] = (torch.rand(shape, device=DEV, generator=g) * 0.2 + 0.3).half()
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    host = random.Random(int(seed))
    fam, d, dtype = case["family"], case["head_dim"], DTYPES[case["dtype"]]
    h, hq = case["heads"], case["heads"] * case["group"]
    st = dict(case=case)
    if fam in ("rotate", "append"):
        rows = case["rows"] if fam == "rotate" else sum(_ragged(case["batch"], case["new"], case["ragged"])) + case["padded"]
        axes = case["axes"]
        # a fused projection's rows: q, k and v are slices of it
        qkv = torch.randn(rows, hq + 2 * h, d, device=DEV, generator=g).to(dtype)
        st.update(q=qkv[:, :hq], k=qkv[:, hq:hq + h], v=qkv[:, hq + h:])
        if axes:
            st.update(positions=_positions(rows, axes, host.randint(0, 30000)), inv_freq=_inv_freq(d),
                      axis=torch.tensor(_axis_of(d, axes, case.get("interleaved", True)), device=DEV))
    if fam == "rotate":
        if case["grad"]:
            st["q"] = st["q"].contiguous().requires_grad_(own)
            st["k"] = st["k"].contiguous().requires_grad_(own)
            st["grads"] = tuple(torch.randn(x.shape, device=DEV, generator=g).to(dtype) for x in (st["q"], st["k"]))
        return st
    t = case["tokens"]
    if fam == "append":
        # each sequence goes on within a page that holds some tokens already; pages are where the pool had them
        new = _ragged(case["batch"], case["new"], case["ragged"])
        begin = [host.randrange(t) for _ in new]
        need = [_ceil(b + n, t) for b, n in zip(begin, new)]
        order = list(range(sum(need)))
        host.shuffle(order)
        slots = []
        for b, n, p in zip(begin, new, need):
            table, order = order[:p], order[p:]
            slots += [table[i // t] * t + i % t for i in range(b, b + n)]
        live = len(slots)
        slots += [-1] * case["padded"]
        shape = (1, sum(need) + 2, h, t)
        f = {x + "_codes": torch.zeros(shape + (d // 2,), dtype=torch.uint8, device=DEV) for x in ("key", "value")}
        f |= {x + "_scales": torch.zeros(shape, dtype=torch.float16, device=DEV) for x in ("key", "value")}
        st.update(fields=f, live=live)
        if own:
            from nexusquant_amd import FourBitPagePool, plan_rotation
            st["pool"] = FourBitPagePool.from_tensors(**f)
            st["pool"].allocate(sum(need))
            st["plan"] = st["pool"].plan_slots(slots)
            st["rotation"] = plan_rotation(st["positions"], d, BASE, sections=_sections(d, case["axes"]),
                                           interleaved=True) if case["axes"] else None
        else:
            st["slots"] = torch.tensor(slots[:live], device=DEV)
            st["hadamard"] = _hadamard(d, torch.float64)
            if case["axes"]:
                st["cos"], st["sin"] = _angles(st)
        return st
    seqs = _attended(case)
    need = [_ceil(n, t) for n, _ in seqs]
    f = _fields(g, sum(need) + 2, h, t, d)
    order = list(range(sum(need)))
    host.shuffle(order)
    at = np.concatenate([[0], np.cumsum(need)]).tolist()
    tables = [order[a:b] for a, b in zip(at, at[1:])]
    st.update(fields=f, tables=tables, seqs=seqs,
              q=torch.randn(sum(q for _, q in seqs), hq, d, device=DEV, generator=g).to(dtype))
    if own:
        from nexusquant_amd import FourBitPagePool
        st["pool"] = FourBitPagePool.from_tensors(**f)
        st["pool"].allocate(sum(need))
        st["plan"] = st["pool"].plan_attention(tables, [n for n, _ in seqs], [q for _, q in seqs], causal=case["causal"],
                                               sliding_window=case["window"] or None)
    else:
        wide, most = max(1, max(need)), max(q for _, q in seqs)
        st["pages"] = torch.tensor([x + [0] * (wide - len(x)) for x in tables], device=DEV)
        n = torch.tensor([n for n, _ in seqs], device=DEV)
        q = torch.tensor([q for _, q in seqs], device=DEV)
        first = q.cumsum(0) - q
        i = torch.arange(most, device=DEV)
        st["from_row"] = (first[:, None] + i).clamp_(max=st["q"].shape[0] - 1)     # [batch, most], padded
        st["real"] = i < q[:, None]
        last = (n - q)[:, None] + i if case["causal"] else (n - 1)[:, None] + 0 * i  # the last token that a query sees
        st["last"] = last
        st["hadamard"] = _hadamard(d, torch.float32)
    return st


# -------------------------------------------------------------- plain forms --

def _hadamard(d, dtype):
    """The orthonormal Sylvester matrix: (-1)^popcount(i & j) / sqrt(d)."""
    i = torch.arange(d, device=DEV)
    odd = ((i[:, None, None] & i[:, None]) >> torch.arange(8, device=DEV) & 1).sum(-1) & 1
    return ((1 - 2 * odd).to(torch.float64) / math.sqrt(d)).to(dtype)


def _angles(st):
    """cos and sin [rows, 1, d / 2] in 32 bits: the angle is the product of 32-bit numbers, as models form it."""
    ang = (st["positions"].float()[st["axis"]].T * st["inv_freq"]).double()[:, None]
    return ang.cos().float(), ang.sin().float()


def _rotated(x, c, s):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_rotate(st):
    c, s = _angles(st)
    out = [_rotated(x, c, s).to(x.dtype) for x in (st["q"], st["k"])]
    if st["case"]["grad"]:  # of a rotation: the rotation by the opposite angle
        out += [_rotated(x, c, -s).to(x.dtype) for x in st["grads"]]
    return out


def _encode(x, hadamard):
    """Codes and scales of vectors; in 64 bits, since a value next to a border takes one code or the other."""
    y = torch.matmul(x.double(), hadamard)
    s = (y.abs().amax(-1, keepdim=True) / 7.5).half()
    n = torch.floor(y / torch.where(s == 0, 1.0, s.double()) + 8.5).clamp_(0, 15).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), s[..., 0]


def _decode(codes, scales, hadamard):
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    return torch.matmul((n.to(hadamard.dtype) - 8) * scales.to(hadamard.dtype)[..., None], hadamard)


def _plain_append(st):
    case, f, live, t = st["case"], st["fields"], st["live"], st["case"]["tokens"]
    k, v, out = st["k"].float(), st["v"].float(), []
    if case["axes"]:
        out.append(_rotated(st["q"], st["cos"], st["sin"]).to(st["q"].dtype))
        k = _rotated(k, st["cos"], st["sin"])
    page, off = st["slots"] // t, st["slots"] % t
    for name, x in (("key", k), ("value", v)):
        f[name + "_codes"][0, page, :, off], f[name + "_scales"][0, page, :, off] = _encode(x[:live], st["hadamard"])
        stored = _decode(f[name + "_codes"][0, page, :, off], f[name + "_scales"][0, page, :, off], st["hadamard"].float())
        out.append(stored.to(st["q"].dtype))
    return out


def _plain_attend(st):
    case, f = st["case"], st["fields"]
    h, grp, d, t = case["heads"], case["group"], case["head_dim"], case["tokens"]

    def tokens_of(name):  # [batch, heads, tokens, d]
        x = _decode(f[name + "_codes"][0][st["pages"]], f[name + "_scales"][0][st["pages"]], st["hadamard"])
        return x.transpose(1, 2).reshape(x.shape[0], h, -1, d)

    k, v = tokens_of("key"), tokens_of("value")
    batch, most = st["from_row"].shape
    q = st["q"].float()[st["from_row"]].view(batch, most, h, grp, d).permute(0, 2, 3, 1, 4).reshape(batch, h, grp * most, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(d)).view(batch, h, grp, most, -1)
    i = torch.arange(s.shape[-1], device=DEV)
    hidden = i > st["last"][..., None]
    if case["window"]:
        hidden |= i <= st["last"][..., None] - case["window"]
    s.masked_fill_(hidden[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-30))  # nothing seen: zero
    o = torch.matmul(s.view(batch, h, grp * most, -1), v).view(batch, h, grp, most, d)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, most, h * grp, d)[st["real"]].to(st["q"].dtype)


# --------------------------------------------------------------------- run --

def run(st):
    case = st["case"]
    fam, d = case["family"], case["head_dim"]
    if fam == "rotate":
        if not own:
            return _plain_rotate(st)
        from nexusquant_amd import plan_rotation, rotate
        rotation = plan_rotation(st["positions"], d, BASE, sections=_sections(d, case["axes"]),
                                 interleaved=case["interleaved"])
        q, k = rotate(st["q"], st["k"], rotation)
        if case["grad"]:
            return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (st["q"], st["k"]), st["grads"])]
        return [q, k]
    if fam == "append":
        if not own:
            return _plain_append(st)
        q = st["pool"].append(st["plan"], st["k"], st["v"], rotation=st["rotation"], query=st["q"] if case["axes"] else None)
        k, v = st["pool"].read(st["plan"], dtype=DTYPES[case["dtype"]])
        return ([q] if case["axes"] else []) + [k[:st["live"]], v[:st["live"]]]
    return st["pool"].attend(st["plan"], st["q"]) if own else _plain_attend(st)


def _pairs(case):
    """(query, token) pairs that are seen."""
    total = 0
    for n, q in _attended(case):
        w = case["window"] or n
        if not case["causal"]:
            total += n * q
        else:
            total += sum(min(n - q + 1 + i, w) for i in range(q))
    return total


def work(case):
    fam, d, h = case["family"], case["head_dim"], case["heads"]
    hq = h * case["group"]
    if fam == "rotate":
        size = 4 if case["dtype"] == "fp32" else 2
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * 2 * case["rows"] * (hq + h) * d * size + 4 * case["rows"] * case["axes"],
                "flops": passes * 3 * case["rows"] * (hq + h) * d}
    if fam == "append":
        live = sum(_ragged(case["batch"], case["new"], case["ragged"]))
        rows = live + case["padded"]
        stored = live * h * 2 * (d // 2 + 2)
        angles = rows * d * 4 if case["axes"] else 0
        # queries read and written, keys and values read, written in 4 bits, read there and written back
        return {"bytes": (rows * 2 * hq * d * 2 if case["axes"] else 0) + live * 2 * h * d * 2 + 2 * stored + live * 2 * h * d * 2 + angles + 4 * rows,
                "flops": 2 * live * h * 2 * d * int(math.log2(d)) + (3 * rows * (hq + h) * d if case["axes"] else 0)}
    tokens = 0
    for n, q in _attended(case):
        if q:
            tokens += n if not case["window"] else min(n, case["window"] + q - 1)
    rows = sum(q for _, q in _attended(case))
    return {"bytes": max(1, tokens * h * 2 * (d // 2 + 2) + 2 * 2 * rows * hq * d), "flops": 4 * hq * d * _pairs(case)}


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


def _turned(x, st, sign):
    """x rotated as complex numbers of its two halves."""
    pos = st["positions"].float()
    ang = torch.stack([pos[int(a)] * f for a, f in zip(st["axis"].tolist(), st["inv_freq"])], dim=-1).double()[:, None]
    z = torch.complex(x[..., :x.shape[-1] // 2].double(), x[..., x.shape[-1] // 2:].double())
    z = z * torch.polar(torch.ones_like(ang), sign * ang)
    return torch.cat([z.real, z.imag], dim=-1)


def exact(case, seed):
    fam, d = case["family"], case["head_dim"]
    st = prepare(case, seed)
    if fam == "rotate":
        out = [_turned(st[x].detach(), st, 1) for x in "qk"]
        return out + [_turned(x, st, -1) for x in st["grads"]] if case["grad"] else out
    if fam == "append":
        out = [_turned(st["q"], st, 1)] if case["axes"] else []
        for x in (_turned(st["k"], st, 1) if case["axes"] else st["k"].double(), st["v"].double()):
            t = _walsh(x[:st["live"]])
            s = (t.abs().amax(-1, keepdim=True) / 7.5).half().double()
            level = torch.floor(t / s + 0.5).clamp(-8, 7)
            out.append(_walsh(torch.where(s > 0, level * s, 0.0)))
        return out
    f = st["fields"]
    if len(st["seqs"]) * case["heads"] * case["group"] > 4000:
        return None
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for table, (n, m) in zip(st["tables"], st["seqs"]):
        if n and m:
            pages = torch.tensor(table, device=DEV)

            def whole(name):  # [heads, n, d]
                codes = f[name + "_codes"][0, pages].transpose(0, 1).flatten(1, 2)[:, :n]
                x = torch.empty(*codes.shape[:2], d, dtype=torch.float64, device=DEV)
                x[..., 0::2], x[..., 1::2] = codes % 16, codes // 16
                return _walsh((x - 8) * f[name + "_scales"][0, pages].transpose(0, 1).flatten(1)[:, :n, None].double())

            k, v = whole("key"), whole("value")
            j = torch.arange(n, device=DEV)
            at = (n - m + torch.arange(m, device=DEV))[:, None] if case["causal"] else torch.full((m, 1), n, device=DEV)
            seen = j <= at
            if case["window"]:
                seen &= j > at - case["window"]
            for head in range(case["heads"]):
                for one in range(head * case["group"], (head + 1) * case["group"]):
                    logit = torch.where(seen, st["q"][row:row + m, one].double() @ k[head].T / math.sqrt(d), -math.inf)
                    out[row:row + m, one] = torch.softmax(logit, dim=-1) @ v[head]
        row += m
    return out
