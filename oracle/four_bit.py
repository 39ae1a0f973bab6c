"""A cache held in 4 bits, its rotations and its attention, in 64 bits.  Test infrastructure only."""

from __future__ import annotations

import math

import torch


def walsh(x: torch.Tensor) -> torch.Tensor:
    """The orthonormal Walsh-Hadamard transform of the last axis."""
    d = x.shape[-1]
    step = 1
    while step < d:
        y = x.reshape(*x.shape[:-1], d // (2 * step), 2, step)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).reshape(x.shape)
        step *= 2
    return x / math.sqrt(d)


def angles(positions: torch.Tensor, inv_freq: torch.Tensor, axis_of) -> torch.Tensor:
    """float64 [rows, d / 2]: the fp32 products of positions [axes, rows] and inverse frequencies."""
    pos = positions.cpu().to(torch.float32)
    return torch.stack([pos[int(a)] * f for a, f in zip(axis_of, inv_freq.float())], dim=-1).double()


def rotate(x: torch.Tensor, ang: torch.Tensor, inverse: bool = False) -> torch.Tensor:
    """x [rows, heads, d] in float64, coordinate i turned with i + d / 2."""
    x = x.double()
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = ang.cos()[:, None], ang.sin()[:, None] * (-1.0 if inverse else 1.0)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def unpack(codes: torch.Tensor) -> torch.Tensor:
    """Levels n - 8 in float64 of uint8 codes [..., d / 2]."""
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    return n.double() - 8


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return walsh(unpack(codes) * scales.double()[..., None])


def encode(x: torch.Tensor):
    """(codes, scales) of float64 vectors."""
    t = walsh(x.double())
    s = torch.clamp(t.abs().amax(-1) / 7.5, max=65504.0).to(torch.float16)
    n = torch.floor(t / torch.where(s == 0, 1.0, s.double())[..., None] + 8.5).clamp(0, 15).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), s


def sequence(codes: torch.Tensor, scales: torch.Tensor, table, n: int):
    """A sequence's first n tokens of a layer's fields [pages, heads, tokens, ...]: levels [heads, n, d], scales [heads, n]."""
    pages = torch.as_tensor(table, dtype=torch.long)
    c = codes[pages].transpose(0, 1).flatten(1, 2)[:, :n]
    s = scales[pages].transpose(0, 1).flatten(1)[:, :n]
    return unpack(c), s.double()


def seen(n: int, q: int, causal: bool, window: int) -> torch.Tensor:
    """bool [q, n]: which tokens each query sees."""
    j = torch.arange(n)
    if not causal:
        return torch.ones(q, n, dtype=torch.bool)
    at = (n - q + torch.arange(q))[:, None]
    mask = j <= at
    return mask & (j > at - window) if window else mask


def attend(query: torch.Tensor, key_levels, key_scales, value_levels, value_scales, mask: torch.Tensor, scale: float):
    """Outputs [q, heads, d] of queries [q, q_heads, d] over one sequence, and how far a kernel's may be off by the numbers
    that it rounds: with u the relative error of a (transformed) query's coordinate and w of a weight, the error of an output
    coordinate is at most bound(u, w).

    A logit is off by delta <= scale s_k (u sum |q~| |n - 8| + acc sum |q~|), acc the rounding of sums in 32 bits whose
    terms are up to 31 times a coordinate; softmax weights then by a factor within e^(2 delta); values' sums by w and by the
    same rounding of sums; the last transform spreads what coordinates are off by, at most sqrt(d) times."""
    m, hq, d = query.shape
    h = key_levels.shape[0]
    out = torch.zeros(m, hq, d, dtype=torch.float64)
    lim = []
    for head in range(hq):
        kv = head // (hq // h)
        qt = walsh(query[:, head].double())
        k, v = key_levels[kv] * key_scales[kv][:, None], value_levels[kv] * value_scales[kv][:, None]
        logit = torch.where(mask, qt @ k.T * scale, -math.inf)
        some = mask.any(-1, keepdim=True)
        p = torch.where(some, torch.softmax(logit, dim=-1), 0.0)
        p = torch.where(mask, p, 0.0)
        vz = torch.where(mask.any(0)[:, None], v, 0.0)
        out[:, head] = walsh(p @ vz)
        acc = 64 * 2.0 ** -24
        a_q = torch.where(mask, qt.abs() @ k.abs().T, 0.0).amax(-1) if k.shape[0] else torch.zeros(m, dtype=torch.float64)
        a_s = (qt.abs().sum(-1)[:, None] * torch.where(mask, key_scales[kv], 0.0)).amax(-1) if k.shape[0] else a_q
        big = p @ vz.abs()
        sums = p @ torch.where(mask.any(0), value_scales[kv], 0.0) if k.shape[0] else a_q
        most = torch.where(mask, value_scales[kv], 0.0).amax(-1) if k.shape[0] else a_q
        lim.append((a_q, a_s, big, sums, most, acc, k.shape[0]))

    def bound(u, w):
        got = torch.zeros(m, hq, d, dtype=torch.float64)
        for head, (a_q, a_s, big, sums, most, acc, n) in enumerate(lim):
            delta = scale * (u * a_q + acc * 31 * a_s)
            level = (torch.expm1(2 * delta) + w)[:, None] * big + (acc * 31 * sums + n * 2.0 ** -28 * most)[:, None]
            # each output coordinate is a sum of d levels, +-1 / sqrt(d) each
            got[:, head] = level.sum(-1, keepdim=True) / math.sqrt(d) + 2.0 ** -20 * big.sum(-1, keepdim=True) / math.sqrt(d)
        return got

    return out, bound
