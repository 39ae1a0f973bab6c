"""A cache held in 4 bits against 64 bits: what is stored, what is read, and attention over it."""

import math

import pytest
import torch

from nexusquant_amd import FourBitPagePool, _lib, four_bit, plan_rotation, rotate
from nexusquant_amd.rope import inv_freq
from nexusquant_amd.rotary import frequency_axes
from oracle import four_bit as ref
from test_rotary_host import check_written_tensors_are_seen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def fill(pool, seed):
    """Random codes and scales in all of a pool."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for c in (pool.key_codes, pool.value_codes):
        c.copy_(torch.randint(0, 256, c.shape, device="cuda", generator=g, dtype=torch.uint8))
    for s in (pool.key_scales, pool.value_scales):
        s.copy_(torch.rand(s.shape, device="cuda", generator=g) * 0.3 + 0.05)


def sequences(pool, lens, seed):
    """Allocated, shuffled tables."""
    need = [pool.pages_for(n) for n in lens]
    pages = torch.tensor(pool.allocate(sum(need)))
    pages = pages[torch.randperm(len(pages), generator=torch.Generator().manual_seed(seed))].tolist()
    tables = []
    for n in need:
        tables.append(pages[:n])
        pages = pages[n:]
    return tables


# ----------------------------------------------------------- append and read --

def check_stored(codes, scales, t, terms):
    """Stored levels of t = H x, as 64 bits have it.  32 bits are off by at most `terms` 2^-24 of |x| sums over sqrt(d) (a
    butterfly's sums, one rounding a stage, the rotation's and two products), the scale by half a step of fp16 more."""
    d = t.shape[-1]
    off = terms * 2.0 ** -24 * ref.walsh(t).abs().sum(-1) / math.sqrt(d) + 1e-30
    m = t.abs().amax(-1) / 7.5
    s = scales.double()
    half = torch.where(m < 2.0 ** -14, 2.0 ** -25, m * 2.0 ** -11)
    assert ((s - m.clamp(max=65504.0)).abs() <= half + off).all()
    y = t / torch.where(s == 0, 1.0, s)[..., None]
    # levels end at 7: with s >= (m / 7.5) (1 - 2^-11), or held at 65504, what lies past 7.5 s is still held as 7 (the format's
    # own bound there is 0.5 + 7.5 2^-11)
    clipped = y.clamp(-8.0, 7.5)
    good = (ref.unpack(codes) - clipped).abs() <= 0.5 + (off / torch.where(s == 0, 1.0, s))[..., None] + 2.0 ** -20
    assert (good | (s == 0)[..., None]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,hq,tokens,rows,axes", [
    (64, 1, 1, 16, 1, 1), (128, 8, 32, 16, 33, 3), (256, 3, 6, 8, 17, 1), (128, 5, 0, 24, 40, 0), (64, 20, 20, 32, 100, 1),
    (128, 2, 14, 16, 7, 1), (256, 8, 0, 16, 130, 0), (128, 16, 64, 64, 300, 2)])
def test_append_and_read(dtype, d, heads, hq, tokens, rows, axes):
    T = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(d + rows)
    pool = FourBitPagePool(rows // tokens + 5, heads, tokens, d, num_layers=3)
    fill(pool, 1)
    before = [x.clone() for x in (pool.key_codes, pool.value_codes, pool.key_scales, pool.value_scales)]
    pages = pool.allocate(rows // tokens + 3)
    order = torch.randperm(len(pages) * tokens, generator=torch.Generator().manual_seed(rows)).tolist()
    slots = [pages[i // tokens] * tokens + i % tokens for i in order[:rows]]
    if rows > 5:
        slots[3] = slots[rows - 1] = -1
    qkv = torch.randn(rows, hq + 2 * heads, d, device="cuda", generator=g).to(T)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + heads], qkv[:, hq + heads:]
    rotation, turned_q, turned_k = None, q.cpu().double(), k.cpu().double()
    if axes:
        sections = [d // 2 - (axes - 1) * (d // 8)] + [d // 8] * (axes - 1)
        pos = torch.stack([torch.arange(rows) * (a + 1) + 17 for a in range(axes)])
        rotation = plan_rotation(pos.cuda(), d, base=500000.0, sections=sections)
        ang = ref.angles(pos, inv_freq(d, 500000.0), frequency_axes(d, sections, False))
        turned_q, turned_k = ref.rotate(turned_q, ang), ref.rotate(turned_k, ang)
    plan = pool.plan_slots(slots)
    got = pool.append(plan, k, v, rotation=rotation, query=q if hq else None, layer=1)
    if hq:
        assert torch.equal(got, rotate(q, None, rotation)[0])
    else:
        assert got is None
    live = torch.tensor([i for i, s in enumerate(slots) if s >= 0])
    at = torch.tensor(slots)[live]
    kc, vc, ks, vs = (x.cpu() for x in (pool.key_codes, pool.value_codes, pool.key_scales, pool.value_scales))
    for c, s, x in ((kc, ks, turned_k), (vc, vs, v.cpu().double())):
        check_stored(c[1, at // tokens, :, at % tokens], s[1, at // tokens, :, at % tokens], ref.walsh(x[live]), 16)
    # nothing else was written
    for now, was in zip((kc, vc, ks, vs), before):
        was = was.cpu()
        was[1, at // tokens, :, at % tokens] = now[1, at // tokens, :, at % tokens]
        assert torch.equal(now, was)
    for out_type in (torch.float16, torch.bfloat16, torch.float32):
        keys, values = pool.read(plan, layer=1, dtype=out_type)
        for y, c, s in ((keys, kc, ks), (values, vc, vs)):
            want = ref.decode(c[1, at // tokens, :, at % tokens], s[1, at // tokens, :, at % tokens])
            off = (y.cpu().double()[live] - want).abs()
            # its type's rounding, the product of scale and 1 / sqrt(d) and that with a whole number
            assert (off <= want.abs() * (torch.finfo(out_type).eps / 2 + 4 * 2.0 ** -24) + 2.0 ** -25).all()
            assert (y.cpu()[[i for i, p in enumerate(slots) if p < 0]] == 0).all()


@pytest.mark.parametrize("dtype,d,heads,hq,rows", [("fp16", 128, 4, 40, 3400), ("bf16", 64, 16, 16, 3000), ("fp16", 256, 2, 18, 4000)])
def test_large_steps_are_stored_as_small_ones(dtype, d, heads, hq, rows):
    """Past 32 MB queries and values read are written in another way; a wave takes a token's heads in several steps."""
    T = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows)
    pools = [FourBitPagePool(rows // 16 + 1, heads, 16, d) for _ in range(2)]
    slots = [p * 16 + i for p in pools[0].allocate(rows // 16 + 1) for i in range(16)][:rows]
    assert pools[1].allocate(rows // 16 + 1)[0] == slots[0] // 16
    qkv = torch.randn(rows, hq + 2 * heads, d, device="cuda", generator=g).to(T)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + heads], qkv[:, hq + heads:]
    pos = torch.arange(rows, device="cuda")
    whole = pools[0].append(pools[0].plan_slots(slots), k, v, rotation=plan_rotation(pos, d), query=q)
    for a in range(0, rows, 501):
        part = slice(a, min(a + 501, rows))
        small = pools[1].append(pools[1].plan_slots(slots[part]), k[part], v[part], rotation=plan_rotation(pos[part], d), query=q[part])
        assert torch.equal(whole[part], small)
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        used = torch.tensor(slots, device="cuda")
        a, b = (getattr(p, name)[0][used // 16, :, used % 16] for p in pools)
        assert torch.equal(a, b)
    for out in (T, torch.float32):
        whole = pools[0].read(pools[0].plan_slots(slots), dtype=out)
        for a in range(0, rows, 501):
            small = pools[0].read(pools[0].plan_slots(slots[a:a + 501]), dtype=out)
            assert all(torch.equal(x[a:a + 501], y) for x, y in zip(whole, small))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_levels_next_to_a_border_are_decided_in_64_bits(dtype, d):
    """Values (nothing is rotated) are stored as 64 bits have them, bit for bit: sums of few-bit numbers, whose transforms lie
    on borders at d = 64 and 256, and random rows, whose sums in 32 bits are off by some 2^-24 of them (independent roundings
    in 6 to 8 stages; six times their spread is 2^-21 of the largest, 2^-18 of a step, and closer than 2^-17 is done again)."""
    T = TYPES[dtype]
    pool = FourBitPagePool(70, 2, 16, d)
    pages = pool.allocate(70)
    slots = [p * 16 + i for p in pages for i in range(16)]
    g = torch.Generator().manual_seed(d)
    x = torch.randn(len(slots), 2, d, generator=g)
    x[:300] = torch.randint(-2, 3, (300, 2, d), generator=g).float()
    x[300] = 1.0
    x[301] = -0.75
    x[302, :, 1:] = 0.0
    x = x.to(T)
    pool.append(pool.plan_slots(slots), torch.zeros_like(x).cuda(), x.cuda())
    codes, scales = ref.encode(x)
    at = torch.tensor(slots)
    assert torch.equal(pool.value_scales[0].cpu()[at // 16, :, at % 16], scales)
    assert torch.equal(pool.value_codes[0].cpu()[at // 16, :, at % 16], codes)


def test_rows_that_are_zero_tiny_huge_or_not_finite():
    d = 128
    pool = FourBitPagePool(2, 1, 16, d)
    pages = pool.allocate(1)
    for T, tiny, huge in ((torch.float16, 2.0 ** -24, 65504.0), (torch.bfloat16, 1e-30, 1e30)):
        x = torch.zeros(16, 1, d, dtype=T)
        g = torch.Generator().manual_seed(1)
        x[1] = torch.randn(1, d, generator=g)
        x[2, 0, 5] = tiny
        x[3] = huge
        x[4, 0, 7] = math.inf
        x[5, 0, 9] = math.nan
        x[6, 0, :2] = torch.tensor([math.inf, -math.inf])
        x[7] = torch.randn(1, d, generator=g) * 3e-5
        plan = pool.plan_slots([pages[0] * 16 + i for i in range(16)])
        pool.append(plan, x.cuda(), x.cuda())
        codes, scales = pool.key_codes[0, pages[0], 0].cpu(), pool.key_scales[0, pages[0], 0].cpu()
        assert torch.equal(pool.value_codes[0, pages[0], 0].cpu(), codes)
        assert scales[0] == 0 and scales[4:7].isnan().all() and scales[[0, 1, 2, 3, 7]].isfinite().all()
        keys, values = (y.cpu() for y in pool.read(plan, dtype=torch.float32))
        assert (keys[0] == 0).all() and (keys[8:] == 0).all() and keys[4:7].isnan().all() and values[4:7].isnan().all()
        check_stored(codes[[1, 7]], scales[[1, 7]], ref.walsh(x[[1, 7], 0].double()), 16)
        assert keys[2].abs().max() <= 2 * tiny + 2.0 ** -24 and keys[3].isfinite().all()
        # A constant row is one coordinate of its transform, huge sqrt(d), and 65504 sqrt(128) / 7.5 = 98813 is past fp16 for
        # both types: the scale is held at 65504, the level at 7, and the other 127 levels at zero.
        assert scales[3] == 65504
        assert (keys[3] - 7 * 65504.0 / math.sqrt(d)).abs().max() <= 7 * 65504.0 / math.sqrt(d) * 4 * 2.0 ** -24


# ----------------------------------------------------------------- attention --

def step(few):
    """Relative errors of a query's coordinate and of a weight: few rows' queries have 16 bits below the largest coordinate
    (2^-16 of it: what counts of smaller ones is within the sum's bound) and weights 22; wider tiles round weights to fp16."""
    return 2.0 ** -15 if few else 2.0 ** -11


def check_attention(pool, tables, lens, queries, q, got, dtype, causal=True, window=0, scale=None, layer=0, few=None):
    """Every row against 64 bits, by the bound of what the kernels round (oracle/four_bit.py) plus half a step of the output."""
    d = pool.head_dim
    fields = [x[layer].cpu() for x in (pool.key_codes, pool.key_scales, pool.value_codes, pool.value_scales)]
    row = 0
    for table, n, m in zip(tables, lens, queries):
        if m and n:
            kl, ks = ref.sequence(fields[0], fields[1], table, n)
            vl, vs = ref.sequence(fields[2], fields[3], table, n)
            mask = ref.seen(n, m, causal, window)
            want, bound = ref.attend(q[row:row + m].cpu(), kl, ks, vl, vs, mask, d ** -0.5 if scale is None else scale)
            narrow = m * (q.shape[1] // pool.num_heads) <= 16 if few is None else few
            u = step(narrow)
            off = (got[row:row + m].cpu().double() - want).abs()
            lim = bound(u, u) + want.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25
            assert (off <= lim).all(), (n, m, float((off - lim).max()))
            # and as a whole much nearer: roundings are independent, a norm's is eps / 2 / sqrt(3) for the output's
            rel = float(off.norm() / want.norm())
            assert rel <= (torch.finfo(dtype).eps / 2 if narrow else torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -11), rel
        else:
            assert (got[row:row + m] == 0).all()
        row += m


CASES = [
    # heads, group, d, tokens a page, lengths, queries, causal, window
    (1, 1, 64, 16, [1], [1], True, 0),
    (8, 4, 128, 16, [1, 15, 16, 17, 33, 0, 255], None, True, 0),
    (2, 8, 256, 8, [7, 100, 1025], None, True, 0),
    (4, 1, 64, 32, [2049, 31, 700], None, True, 0),
    (2, 16, 128, 24, [513, 64], None, True, 0),
    (1, 24, 128, 16, [300, 5], None, True, 0),            # more heads than a few tile has rows
    (1, 160, 64, 16, [77, 130], None, True, 0),           # more than a wide tile has
    (8, 4, 128, 16, [40, 129, 1000], [4, 4, 3], True, 0),
    (2, 4, 128, 16, [40, 129, 1000], [5, 33, 40], True, 0),
    (2, 4, 256, 16, [64, 129, 400], [64, 1, 100], True, 0),
    (4, 2, 64, 64, [1000, 200, 64], [130, 200, 64], True, 0),
    (2, 5, 128, 16, [333, 50], [27, 50], True, 0),        # a group that divides no tile
    (8, 4, 128, 16, [1000, 64, 3], None, True, 17),
    (2, 4, 128, 16, [1000, 300], [100, 300], True, 70),
    (2, 2, 64, 16, [500, 65], [30, 65], True, 1),
    (20, 1, 64, 32, [1500, 3, 0, 64], [1, 1, 1, 1], False, 0),
    (4, 1, 64, 32, [150, 3, 0, 64], [223, 2, 5, 17], False, 0),
    (2, 4, 128, 16, [100, 1], [60, 0], False, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,d,tokens,lens,queries,causal,window", CASES)
def test_attention(dtype, heads, group, d, tokens, lens, queries, causal, window):
    T = TYPES[dtype]
    pool = FourBitPagePool(sum(-(-n // tokens) for n in lens) + 3, heads, tokens, d, num_layers=2)
    fill(pool, d + len(lens))
    tables = sequences(pool, lens, 5)
    new = queries or [1] * len(lens)
    g = torch.Generator(device="cuda").manual_seed(11)
    q = torch.randn(sum(new), heads * group, d, device="cuda", generator=g).to(T)
    plan = pool.plan_attention(tables, lens, queries, causal=causal, sliding_window=window or None)
    got = pool.attend(plan, q, layer=1)
    check_attention(pool, tables, lens, new, q, got, T, causal, window, layer=1)
    # what no query sees changes nothing, whatever it holds: slots behind a sequence, other pages, tokens before a window
    hidden = torch.ones(pool.key_scales.shape[1:], dtype=torch.bool)
    for table, n, m in zip(tables, lens, new):
        if n and m:
            some = ref.seen(n, m, causal, window).any(0)
            for i in some.nonzero().flatten().tolist():
                hidden[table[i // tokens], :, i % tokens] = False
    for s in (pool.key_scales, pool.value_scales):
        s[1][hidden.cuda()] = math.nan
        s[0] = math.nan
    assert torch.equal(pool.attend(plan, q, layer=1), got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,d,tokens,lens,queries,window", [
    (2, 8, 256, 8, [70, 100, 1025], [1, 12, 13], 0),      # 96 rows of a sequence and 104
    (1, 24, 128, 16, [300, 130, 3000], [5, 4, 1], 0),     # a token's heads in two tiles, over several chunks
    (4, 3, 64, 16, [900, 40], [32, 33], 0),
    (1, 96, 128, 16, [5000, 70], [1, 1], 0),
    (2, 4, 128, 16, [2000, 900], [24, 25], 300),
])
def test_rows_up_to_and_past_several_small_tiles(dtype, heads, group, d, tokens, lens, queries, window):
    T = TYPES[dtype]
    pool = FourBitPagePool(sum(-(-n // tokens) for n in lens) + 3, heads, tokens, d)
    fill(pool, d + heads)
    tables = sequences(pool, lens, 5)
    q = torch.randn(sum(queries), heads * group, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(12)).to(T)
    plan = pool.plan_attention(tables, lens, queries, sliding_window=window or None)
    check_attention(pool, tables, lens, queries, q, pool.attend(plan, q), T, True, window)
    for b, (n, m) in enumerate(zip(lens, queries)):  # up to 96 rows weights and queries are not rounded to 11 bits, alone or in a batch
        if m * group <= 96:
            alone = pool.plan_attention([tables[b]], [n], [m], sliding_window=window or None)
            rows = q[sum(queries[:b]):sum(queries[:b + 1])]
            check_attention(pool, [tables[b]], [n], [m], rows, pool.attend(alone, rows), T, True, window, few=True)


@pytest.mark.parametrize("d,group,n,queries", [(128, 8, 131072, 1), (64, 2, 50000, 40), (128, 4, 40000, 40)])
def test_sums_over_long_sequences_keep_their_bits(d, group, n, queries):
    """Many values whose weighted sum is near zero: what the sums' additions lose counts hundreds of times."""
    pool = FourBitPagePool(n // 64 + 3, 1, 64, d)
    fill(pool, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    low, high = (torch.randint(1, 16, pool.value_codes.shape, device="cuda", generator=g, dtype=torch.uint8) for _ in range(2))
    pool.value_codes.copy_(low | high << 4)  # levels -7 .. 7
    tables = sequences(pool, [n], 9)
    q = torch.randn(queries, group, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    check_attention(pool, tables, [n], [queries], q, pool.attend(pool.plan_attention(tables, [n], [queries]), q), torch.float16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 4, 40])
def test_what_some_queries_do_not_see_may_be_anything(dtype, queries):
    """A NaN or infinite scale at a sequence's last token reaches the last query alone."""
    T = TYPES[dtype]
    n = 150
    pool = FourBitPagePool(12, 2, 16, 128)
    fill(pool, 2)
    tables = sequences(pool, [n], 1)
    q = torch.randn(queries, 8, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(T)
    plan = pool.plan_attention(tables, [n], [queries])
    want = pool.attend(plan, q)
    for field in (pool.key_scales, pool.value_scales):
        for bad in (math.nan, math.inf):
            slot = tables[0][(n - 1) // 16], (n - 1) % 16
            was = field[0, slot[0], 1, slot[1]].clone()
            field[0, slot[0], 1, slot[1]] = bad
            got = pool.attend(plan, q)
            # (when a row's maximum rises the rows beside it are rescaled too, so theirs may be rounded in another place)
            check_attention(pool, tables, [n - 1], [queries - 1], q[:-1], got[:-1], T, few=4 * queries <= 16)
            assert torch.equal(got[-1, :4], want[-1, :4])
            # (a key's infinite scale times a negative sum is a logit of -inf, and a weight of zero)
            assert not got[-1, 4:].isfinite().all() or (field is pool.key_scales and bad == math.inf)
            field[0, slot[0], 1, slot[1]] = was


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_and_queries_of_all_sizes(dtype):
    """A first token that takes nearly all weight with small values beside later ones with large ones; large and small queries."""
    T = TYPES[dtype]
    for queries in (1, 40):
        n = 700
        pool = FourBitPagePool(50, 1, 16, 128)
        fill(pool, 3)
        tables = sequences(pool, [n], 1)
        first, later = tables[0][0], tables[0][20]
        pool.value_scales[0, first, 0, 0] = 2.0 ** -14
        pool.value_scales[0, later] *= 1000.0
        pool.key_scales[0, first, 0, 0] = 4.0
        g = torch.Generator(device="cuda").manual_seed(1)
        for factor in (1.0, 2.0 ** -12, 30.0):
            q = (torch.randn(queries, 4, 128, device="cuda", generator=g) * factor).to(T)
            plan = pool.plan_attention(tables, [n], [queries])
            got = pool.attend(plan, q)
            kl, ks = ref.sequence(pool.key_codes[0].cpu(), pool.key_scales[0].cpu(), tables[0], n)
            vl, vs = ref.sequence(pool.value_codes[0].cpu(), pool.value_scales[0].cpu(), tables[0], n)
            want, bound = ref.attend(q.cpu(), kl, ks, vl, vs, ref.seen(n, queries, True, 0), 128 ** -0.5)
            u = step(queries == 1)
            assert ((got.cpu().double() - want).abs() <= bound(u, u) + want.abs() * torch.finfo(T).eps / 2 + 2.0 ** -25).all()


def test_scale_window_strides_and_rows_behind():
    pool = FourBitPagePool(20, 2, 16, 128)
    fill(pool, 4)
    lens, new = [100, 150], [3, 30]
    tables = sequences(pool, lens, 2)
    qkv = torch.randn(40, 12, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).half()
    plan = pool.plan_attention([t + [999] for t in tables], lens, new)  # (entries past a sequence's tokens are padding)
    got = pool.attend(plan, qkv[:, :8], scale=0.11)
    check_attention(pool, tables, lens, new, qkv[:, :8], got, torch.float16, scale=0.11)
    assert (got[33:] == 0).all()
    out = torch.full((40, 10, 128), 5.0, device="cuda").half()
    assert pool.attend(plan, qkv[:, :8], scale=0.11, out=out[:, 1:9]).data_ptr() == out[:, 1:9].data_ptr()
    assert torch.equal(out[:33, 1:9], got[:33]) and (out[33:] == 5.0).all() and (out[:, 0] == 5.0).all() and (out[:, 9] == 5.0).all()
    heads_first = qkv[:, :8].transpose(0, 1).contiguous()
    assert torch.equal(pool.attend(plan, heads_first.transpose(0, 1), scale=0.11), got)
    odd = torch.empty(40 * 8 * 128 + 1, device="cuda", dtype=torch.float16)[1:].view(40, 8, 128).copy_(qkv[:, :8])
    assert torch.equal(pool.attend(plan, odd, scale=0.11), got)
    own = qkv[:, :8].clone()
    assert pool.attend(plan, own, scale=0.11, out=own) is own and torch.equal(own[:33], got[:33]) and torch.equal(own[33:], qkv[33:, :8])
    assert torch.equal(pool.attend(pool.plan_attention(tables, lens, new, sliding_window=150), qkv[:, :8], scale=0.11), got)
    empty = pool.plan_attention([], [])
    assert pool.attend(empty, qkv[:0, :8]).shape == (0, 8, 128) and (pool.attend(empty, qkv[:4, :8]) == 0).all()


def test_decode_steps_as_they_are_used():
    """Prompts appended at once, then tokens one at a time, with positions of three axes; forks, eviction."""
    d, heads, hq, T = 128, 2, 8, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(9)
    pool = FourBitPagePool(64, heads, 16, d, num_layers=2)
    lens = [37, 64]
    tables = [pool.allocate(pool.pages_for(n)) for n in lens]
    sections = [24, 20, 20]

    def step(tables, start, stop):
        """Tokens start[b] .. stop[b] of every sequence through both layers: outputs of the last."""
        rows = [b - a for a, b in zip(start, stop)]
        pos = torch.cat([torch.stack([torch.arange(a, b), torch.arange(a, b) // 2, torch.arange(a, b) % 7]) for a, b in zip(start, stop)], dim=1)
        rotation = plan_rotation(pos.cuda(), d, sections=sections, interleaved=True)
        slots = pool.plan_slots([s for t, a, b in zip(tables, start, stop) for s in pool.slots(t, a, b)])
        plan = pool.plan_attention(tables, stop, rows)
        for layer in range(2):
            qkv = torch.randn(sum(rows), hq + 2 * heads, d, device="cuda", generator=g).to(T)
            q = pool.append(slots, qkv[:, hq:hq + heads], qkv[:, hq + heads:], rotation=rotation, query=qkv[:, :hq], layer=layer)
            out = pool.attend(plan, q, layer=layer)
            check_attention(pool, tables, stop, rows, q, out, T, layer=layer)
        return out

    step(tables, [0, 0], lens)
    for i in range(3):
        for b in range(2):
            if pool.pages_for(lens[b] + 1) > len(tables[b]):
                tables[b] += pool.allocate(1)
        step(tables, lens, [n + 1 for n in lens])
        lens = [n + 1 for n in lens]
    kids = pool.fork(tables[0], lens[0], n=2)
    assert pool.ref_count(tables[0][0]) == 3 and pool.ref_count(tables[0][-1]) == 1
    with pytest.raises(ValueError, match="shared"):
        pool.append(pool.plan_slots(pool.slots(kids[0], 0, 1)), torch.zeros(1, heads, d, device="cuda", dtype=T),
                    torch.zeros(1, heads, d, device="cuda", dtype=T))
    for now in (pool.key_codes, pool.value_codes, pool.key_scales, pool.value_scales):
        assert torch.equal(now[:, kids[1][-1]], now[:, tables[0][-1]])
    step(kids, [lens[0]] * 2, [lens[0] + 1] * 2)
    pool.free(kids[0])
    pool.free(kids[1])
    # every third token leaves
    kept = torch.arange(lens[1])[torch.arange(lens[1]) % 3 != 1].int()
    old = pool.read(pool.plan_slots(pool.slots(tables[1], 0, lens[1])), layer=1)
    (new,), (count,) = pool.compact([tables[1]], [lens[1]], kept[None].cuda(), [len(kept)])
    assert count == len(kept)
    now = pool.read(pool.plan_slots(pool.slots(new, 0, count)), layer=1)
    assert all(torch.equal(a[kept.long().cuda()], b) for a, b in zip(old, now))
    with pytest.raises(ValueError, match="rotated"):
        pool.compact([new], [count], kept[None].cuda(), [1], renumber=True)
    free = pool.free_pages
    pool.free(new)
    pool.free(tables[0])
    assert pool.free_pages == 64 and free < 64


@pytest.mark.parametrize("d", [64, 128, 256])
def test_whole_pages_copied_and_compacted_in_every_layer(d):
    pool = FourBitPagePool(12, 3, 8, d, num_layers=3)
    fill(pool, 7)
    pages = pool.allocate(8)
    fields = (pool.key_codes, pool.value_codes, pool.key_scales, pool.value_scales)
    was = [x.clone() for x in fields]
    pool.copy_pages([pages[0], pages[0], pages[3]], [pages[5], pages[1], pages[7]])
    for now, old in zip(fields, was):
        old[:, [pages[5], pages[1], pages[7]]] = old[:, [pages[0], pages[0], pages[3]]]
        assert torch.equal(now, old)
    table, n = pages[:4], 29
    kept = torch.tensor([0, 2, 3, 9, 11, 12, 20, 27, 28], dtype=torch.int32)
    (new,), _ = pool.compact([table], [n], kept[None].cuda(), torch.tensor([9], device="cuda"))
    for now, old in zip(fields, was):
        for j, i in enumerate(kept.tolist()):
            assert torch.equal(now[:, new[j // 8], :, j % 8], old[:, table[i // 8], :, i % 8])


def test_graphs_and_streams():
    d, heads, hq = 128, 2, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = FourBitPagePool(40, heads, 16, d)
    fill(pool, 5)
    lens = [200, 77, 130]
    tables = sequences(pool, lens, 1)
    slots = pool.plan_slots([pool.slots(t, n - 1, n)[0] for t, n in zip(tables, lens)])
    plan = pool.plan_attention(tables, lens)
    wide = pool.plan_attention(tables, lens, [40, 30, 50])
    pos = torch.tensor([n - 1 for n in lens], device="cuda")
    qkv = torch.randn(3, hq + 2 * heads, d, device="cuda", generator=g).half()
    many = torch.randn(120, hq, d, device="cuda", generator=g).half()

    def step():
        rotation = plan_rotation(pos, d)
        q = pool.append(slots, qkv[:, hq:hq + heads], qkv[:, hq + heads:], rotation=rotation, query=qkv[:, :hq])
        return q, pool.attend(plan, q), pool.attend(wide, many), *pool.read(slots)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs at a time have workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g))
        pos.add_(3)
        many.copy_(torch.randn(many.shape, device="cuda", generator=g))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        for x in (pool.key_codes, pool.value_codes):
            x[0, tables[0][-1]].zero_()  # the replay writes its slots again
        pool.append(slots, qkv[:, hq:hq + heads], qkv[:, hq + heads:], rotation=plan_rotation(pos, d))
        want = [x.clone() for x in step()]
        for graph, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    fresh = pool.plan_attention(tables, lens)
    with torch.cuda.stream(side):
        got = pool.attend(fresh, qkv[:, :hq]), pool.attend(plan, qkv[:, :hq])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], pool.attend(plan, qkv[:, :hq]))
    new = pool.plan_attention(tables, lens)
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            pool.attend(new, qkv[:, :hq])
    torch.cuda.synchronize()


def test_offsets_past_32_bits():
    """Pages whose codes lie past 4 GiB of their field."""
    d, heads, tokens = 256, 8, 16
    pages = 300000  # 4.9 GB of keys' codes
    shape = (1, pages, heads, tokens)
    codes = [torch.empty(shape + (d // 2,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2)]
    pool = FourBitPagePool.from_tensors(*codes, *scales)
    pool.allocate(pages)
    tables = [[pages - 1, 3, pages - 2, pages - 7], [pages - 4, pages - 9]]
    lens = [60, 23]
    g = torch.Generator(device="cuda").manual_seed(1)
    slots = pool.plan_slots([s for t, n in zip(tables, lens) for s in pool.slots(t, 0, n)])
    k, v = (torch.randn(83, heads, d, device="cuda", generator=g).half() for _ in range(2))
    pool.append(slots, k, v)
    keys, values = pool.read(slots)
    assert (keys - k).float().norm() < 0.2 * k.float().norm() and (values - v).float().norm() < 0.2 * v.float().norm()
    for new in ([1, 1], [50, 23]):
        q = torch.randn(sum(new), heads * 2, d, device="cuda", generator=g).half()
        got = pool.attend(pool.plan_attention(tables, lens, new), q)
        row = 0
        for t, n, m in zip(tables, lens, new):
            at = torch.tensor(t, device="cuda")
            kl, ks, vl, vs = (x for c, s in ((codes[0], scales[0]), (codes[1], scales[1]))
                              for x in ref.sequence(c[0][at].cpu(), s[0][at].cpu(), range(len(t)), n))
            want, bound = ref.attend(q[row:row + m].cpu(), kl, ks, vl, vs, ref.seen(n, m, True, 0), d ** -0.5)
            off = (got[row:row + m].cpu().double() - want).abs()
            assert (off <= bound(2.0 ** -11, 2.0 ** -11) + want.abs() * 2.0 ** -11 + 2.0 ** -25).all()
            row += m


def test_one_call_does_not_change_with_the_next():
    """Outputs twice on the same inputs are the same bits: sums have one order."""
    pool = FourBitPagePool(300, 4, 16, 128)
    fill(pool, 8)
    lens = [2000, 31, 900]
    tables = sequences(pool, lens, 3)
    for new in ([1, 1, 1], [40, 31, 50]):
        plan = pool.plan_attention(tables, lens, new)
        q = torch.randn(sum(new), 16, 128, device="cuda").bfloat16()
        first = pool.attend(plan, q)
        for _ in range(5):
            assert torch.equal(pool.attend(plan, q), first)


def test_refusals():
    pool = FourBitPagePool(8, 2, 16, 128, num_layers=2)
    other = FourBitPagePool(8, 2, 16, 128)
    t = pool.allocate(3)
    other.allocate(3)
    plan = pool.plan_slots([t[0] * 16, t[1] * 16 + 3])
    k = torch.randn(2, 2, 128, device="cuda").half()
    q = torch.randn(2, 4, 128, device="cuda").half()
    r = plan_rotation([0, 1], 128)
    for bad in ([t[0] * 16, t[0] * 16], [8 * 16], [1.5], [t[2] * 16 + 16], [(1 << 40)]):
        with pytest.raises(ValueError):
            pool.plan_slots(bad)
    with pytest.raises(ValueError, match="not one of this pool"):
        other.append(plan, k, k)
    for args in ((k[:1], k), (k, k[:, :1]), (k.bfloat16(), k), (k.float(), k.float()), (k[:, :, :64], k[:, :, :64])):
        with pytest.raises(ValueError):
            pool.append(plan, *args)
    for kw in (dict(query=q), dict(rotation=plan_rotation([0], 128)), dict(rotation=plan_rotation([0, 1], 64)),
               dict(layer=2), dict(layer=-1), dict(rotation=r, query=q.bfloat16()), dict(rotation=r, query=q[:1]),
               dict(rotation=r, out=q), dict(rotation=r, query=q, out=q[:, :2]), dict(rotation=r, query=q[:, :2], out=k)):
        with pytest.raises(ValueError):
            pool.append(plan, k, k, **kw)
    with pytest.raises(NotImplementedError):
        pool.append(plan, k.clone().requires_grad_(), k)
    with pytest.raises(Exception, match="device"):
        pool.append(plan, k.cpu(), k)
    pool.free([t[1]])
    with pytest.raises(ValueError, match="not allocated"):
        pool.append(plan, k, k)
    for args in (([t[:1]], [17]), ([t[:1]], [-1]), ([[5]], [3]), ([t[:1]], [3, 4])):
        with pytest.raises(ValueError):
            pool.plan_attention(*args)
    for kw in (dict(queries=[9]), dict(queries=[-1]), dict(sliding_window=0), dict(causal=False, sliding_window=4), dict(queries=[1, 1])):
        with pytest.raises(ValueError):
            pool.plan_attention([t[:1]], [8], **kw)
    step = pool.plan_attention([t[:1]], [8])
    for bad in (q[:1].float(), q[:1, :3], q[:0], q[:1, :, :64], q[:1, :0]):
        with pytest.raises(ValueError):
            pool.attend(step, bad)
    for kw in (dict(scale=0.0), dict(scale=math.nan), dict(layer=2), dict(out=q), dict(out=q[1:].bfloat16()), dict(out=q[:1, :4, ::2])):
        with pytest.raises(ValueError):
            pool.attend(step, q[:1], **kw)
    with pytest.raises(ValueError):
        pool.attend(step, q, out=torch.empty(1, device="cuda").half().expand(2, 4, 128))
    with pytest.raises(ValueError):
        other.attend(step, q[:1])
    with pytest.raises(NotImplementedError):
        pool.attend(step, q[:1].clone().requires_grad_())


def test_writes_in_place_are_seen_by_autograd():
    pool = FourBitPagePool(4, 2, 16, 128)
    t = pool.allocate(2)
    slots, plan, rotation = pool.plan_slots(pool.slots(t, 18, 20)), pool.plan_attention([t], [20], [2]), plan_rotation([18, 19], 128)
    q, k, v = (torch.randn(2, h, 128, device="cuda").half() for h in (4, 2, 2))
    check_written_tensors_are_seen(lambda: pool.append(slots, k, v, rotation=rotation, query=q, out=q), q)
    check_written_tensors_are_seen(lambda: pool.attend(plan, q, out=q), q)


def planned(pool, tables, lens, queries, q_heads, causal=True, window=0):
    """The plan's items [n, 12] and their kinds (0: many, 1: some, 2: few)."""
    rows = [int(_lib.load().nq_fourbit_rows(pool.head_dim, k)) for k in range(3)]
    (items, _), counts = four_bit.attention_items([len(t) for t in tables], lens, queries, causal, window, q_heads // pool.num_heads,
                                                  pool.num_heads, pool.head_dim, rows)
    return items.reshape(-1, 12), torch.repeat_interleave(torch.arange(3), torch.tensor(counts[:3]))


@pytest.mark.parametrize("d,group,n", [(128, 4, 131072), (64, 8, 131072), (256, 2, 131072), (128, 16, 32768)])
def test_one_workgroup_over_a_long_sequence_keeps_its_bits(d, group, n):
    """So many rows that a workgroup has all of a sequence (one table here, for all of them): levels -7 .. 7, whose sums are
    small beside the sums of what the codes stand in the products as."""
    seqs = 1024 if d < 256 else 512
    pool = FourBitPagePool(n // 64 + 3, 1, 64, d)
    fill(pool, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    low, high = (torch.randint(1, 16, pool.value_codes.shape, device="cuda", generator=g, dtype=torch.uint8) for _ in range(2))
    pool.value_codes.copy_(low | high << 4)
    tables = sequences(pool, [n], 9) * seqs
    items, kinds = planned(pool, tables, [n] * seqs, [1] * seqs, group)
    assert (kinds == 2).all() and (items[:, 2] == n).all()
    q = torch.randn(seqs, group, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    got = pool.attend(pool.plan_attention(tables, [n] * seqs), q)
    fields = [x[0].cpu() for x in (pool.key_codes, pool.key_scales, pool.value_codes, pool.value_scales)]
    kl, ks = ref.sequence(fields[0], fields[1], tables[0], n)
    vl, vs = ref.sequence(fields[2], fields[3], tables[0], n)
    mask = torch.ones(1, n, dtype=torch.bool)
    for row in (0, seqs // 2, seqs - 1):
        want, _ = ref.attend(q[row:row + 1].cpu(), kl, ks, vl, vs, mask, d ** -0.5)
        rel = float((got[row:row + 1].cpu().double() - want).norm() / want.norm())
        # An output's rounding is uniform within half a step, 2^-11 of it at most: a norm of 2^-11 / sqrt(3) at most, and of 512
        # numbers one that is 1 / sqrt(1024) of that off by chance (four times that: 1.125).  Queries' and weights' roundings, one
        # in 2^16 and 2^22, are some 3e-5, and add in squares.
        assert rel <= ((2.0 ** -11 / math.sqrt(3) * 1.125) ** 2 + 3e-5 ** 2) ** 0.5, (row, rel)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,d,tokens,lens,queries,causal,window", [
    (1, 4, 64, 16, [3000], [200], True, 0),
    (1, 4, 64, 16, [3000, 100], [200, 3], True, 700),      # chunks that some rows see none of
    (2, 2, 64, 32, [1500, 40, 0], [300, 17, 3], False, 0),
    (1, 4, 128, 16, [2000], [300], False, 0),
    (2, 4, 128, 16, [1500, 240], [300, 200], True, 0),
    (1, 8, 128, 24, [901, 130], [130, 77], True, 333),
])
def test_tiles_of_many_rows_over_several_chunks(dtype, heads, group, d, tokens, lens, queries, causal, window):
    """Eight waves a workgroup, whose sums are joined."""
    T = TYPES[dtype]
    pool = FourBitPagePool(sum(-(-n // tokens) for n in lens) + 3, heads, tokens, d)
    fill(pool, d + len(lens))
    tables = sequences(pool, lens, 5)
    items, kinds = planned(pool, tables, lens, queries, heads * group, causal, window)
    assert (items[kinds == 0, 7] > 1).any()
    q = torch.randn(sum(queries), heads * group, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(13)).to(T)
    plan = pool.plan_attention(tables, lens, queries, causal=causal, sliding_window=window or None)
    check_attention(pool, tables, lens, queries, q, pool.attend(plan, q), T, causal, window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,d,lens,queries,causal", [(4, 64, [300, 512], [300, 140], True), (4, 128, [256, 40], [256, 200], False)])
def test_tiles_of_many_rows_over_one_chunk(dtype, group, d, lens, queries, causal):
    """Outputs written by the tiles themselves: many kv heads, so that nothing is cut."""
    T, heads = TYPES[dtype], 64
    pool = FourBitPagePool(sum(-(-n // 16) for n in lens), heads, 16, d)
    fill(pool, d)
    tables = sequences(pool, lens, 5)
    items, kinds = planned(pool, tables, lens, queries, heads * group, causal)
    assert (kinds == 0).all() and (items[:, 7] == 0).any()
    q = torch.randn(sum(queries), heads * group, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(13)).to(T)
    got = pool.attend(pool.plan_attention(tables, lens, queries, causal=causal), q)
    for head in (0, 41):  # (its kv head alone against 64 bits)
        one = FourBitPagePool(pool.num_pages, 1, 16, d)
        for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
            getattr(one, name).copy_(getattr(pool, name)[:, :, head:head + 1])
        part = slice(head * group, (head + 1) * group)
        check_attention(one, tables, lens, queries, q[:, part], got[:, part], T, causal)


@pytest.mark.parametrize("d,group,n,queries", [(64, 2, 50000, 40), (128, 4, 9000, 24), (256, 4, 5000, 21)])
def test_up_to_96_rows_of_long_sequences_keep_their_bits(d, group, n, queries):
    """Values' sums near zero, with the tolerance of few rows."""
    pool = FourBitPagePool(n // 64 + 3, 1, 64, d)
    fill(pool, 4)
    tables = sequences(pool, [n], 9)
    assert (planned(pool, tables, [n], [queries], group)[1] == 2).all()
    q = torch.randn(queries, group, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    got = pool.attend(pool.plan_attention(tables, [n], [queries]), q)
    check_attention(pool, tables, [n], [queries], q, got, torch.float16, few=True)


@pytest.mark.parametrize("d,pages", [
    (256, (1 << 32) // (8 * 16 * 128)),      # 4 GiB to the byte: offsets of 32 bits up to their last
    (128, (1 << 32) // (8 * 16 * 64)),
    (64, (1 << 32) // (8 * 16 * 32)),
    (128, (1 << 32) // (8 * 16 * 64) + 40),  # and one page and more past it: of 64 bits
    (64, (1 << 32) // (8 * 16 * 32) + 40),
])
def test_few_rows_at_the_end_of_fields_of_4_gib(d, pages):
    heads, tokens = 8, 16
    shape = (1, pages, heads, tokens)
    codes = [torch.zeros(shape + (d // 2,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2)]
    pool = FourBitPagePool.from_tensors(*codes, *scales)
    pool.allocate(pages)
    half = pages // 2  # on either side of 2 GiB
    tables, lens = [[pages - 1, 0, half, pages - 2, half - 1], [half + 1, pages - 3]], [70, 23]
    g = torch.Generator(device="cuda").manual_seed(1)
    for t in tables:
        for page in t:
            for c, s in zip(codes, scales):
                c[0, page] = torch.randint(0, 256, c.shape[2:], device="cuda", generator=g, dtype=torch.uint8)
                s[0, page] = torch.rand(s.shape[2:], device="cuda", generator=g) * 0.3 + 0.05
    for new in ([1, 1], [7, 4]):
        assert (planned(pool, tables, lens, new, heads * 2)[1] == 2).all()
        q = torch.randn(sum(new), heads * 2, d, device="cuda", generator=g).half()
        got = pool.attend(pool.plan_attention(tables, lens, new), q)
        row = 0
        for t, n, m in zip(tables, lens, new):
            at = torch.tensor(t, device="cuda")
            kl, ks, vl, vs = (x for c, s in zip(codes, scales) for x in ref.sequence(c[0][at].cpu(), s[0][at].cpu(), range(len(t)), n))
            want, bound = ref.attend(q[row:row + m].cpu(), kl, ks, vl, vs, ref.seen(n, m, True, 0), d ** -0.5)
            off = (got[row:row + m].cpu().double() - want).abs()
            assert (off <= bound(2.0 ** -15, 2.0 ** -15) + want.abs() * 2.0 ** -11 + 2.0 ** -25).all()
            row += m


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("queries,window,at", [(4, 0, 159), (40, 0, 159), (150, 0, 159), (150, 0, 100), (4, 20, 159), (4, 20, 137),
                                               (40, 20, 159), (40, 20, 101), (150, 20, 159), (150, 20, 60)])
def test_a_large_scale_takes_no_bits_from_rows_that_do_not_see_it(d, queries, window, at):
    """fp16's largest scale at one token beside others of some 2^-12: later tokens, and tokens before a window."""
    n = 160
    pool = FourBitPagePool(12, 2, 16, d)
    fill(pool, 2)
    pool.value_scales.mul_(2.0 ** -10)
    tables = sequences(pool, [n], 1)
    q = torch.randn(queries, 8, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    pool.value_scales[0, tables[0][at // 16], 1, at % 16] = 65504.0
    got = pool.attend(pool.plan_attention(tables, [n], [queries], sliding_window=window or None), q).cpu().double()
    kl, ks = ref.sequence(pool.key_codes[0].cpu(), pool.key_scales[0].cpu(), tables[0], n)
    vl, vs = ref.sequence(pool.value_codes[0].cpu(), pool.value_scales[0].cpu(), tables[0], n)
    mask = ref.seen(n, queries, True, window)
    want, bound = ref.attend(q.cpu(), kl, ks, vl, vs, mask, d ** -0.5)
    few = 4 * queries <= 96
    # (rounded to fp16 below its smallest normal number, which values of 2^-12 come near to: 2^-25)
    lim = bound(step(few), step(few)) + want.abs() * 2.0 ** -11 + 2.0 ** -25
    # An output of 65504 p |n - 8| sqrt(d) at most: numbers of 65520, half a step past fp16's largest, and more are infinite.
    finite = want.abs() + lim < 65520.0
    assert ((got - want).abs() <= lim)[finite].all()
    infinite = want.abs() - lim >= 65520.0
    assert (got == torch.sign(want) * math.inf)[infinite].all()
    rows = ~mask[:, at]
    assert rows.any() and not rows.all()
    off, size = (got - want)[rows], want[rows]
    below = 2.0 ** -25 * off.numel() ** 0.5
    assert off.norm() <= size.norm() * (2.0 ** -11 + (0.0 if few else 3 * 2.0 ** -11)) + below, float(off.norm() / size.norm())
