"""The operators of kvsnap_amd.attention from their definitions: 64-bit torch on the CPU, one sequence at a time."""
import math

import torch

E4M3 = torch.float8_e4m3fn
#: Half a step of each type relative to the value, and half its least step: what one rounding may be off by.
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, E4M3: 2.0 ** -4}
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0, E4M3: 2.0 ** -10}


def table64(width, rows, base=10000.0):
    """The angles' cosines and sines as fp32 tables hold them, in 64 bits."""
    turns = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, width, 2, dtype=torch.float64) / width)
    return torch.stack([turns.cos(), turns.sin()], -1).float().double()


def rotate64(x, positions, table, axes=None, interleaved=False, inverse=False):
    """x [tokens, heads, width]; positions [tokens] or [axes, tokens]; NaN where a position has no angle."""
    x = x.double().clone()
    pairs = table.shape[1]
    positions = positions.reshape(-1, x.shape[0])
    for j in range(pairs):
        at = positions[axes[j] if axes is not None else 0].long()
        known = (at >= 0) & (at < table.shape[0])
        turn = torch.where(known[:, None], table[at.clamp(0, table.shape[0] - 1), j].double(), math.nan)
        cos, sin = turn[:, :1], turn[:, 1:] * (-1 if inverse else 1)
        low, high = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
        a, b = x[..., low].clone(), x[..., high].clone()
        x[..., low], x[..., high] = a * cos - b * sin, b * cos + a * sin
    return x


def rotation_bound(x, turned, dtype):
    """How far a rotation in fp32, rounded once to ``dtype``, may be from ``turned``: the rounding's half step, and
    for the two products and their sum in fp32 three half steps (2^-24 each) of the pair's sizes, |a| + |b| being at
    most twice the head's largest value."""
    return turned.abs() * HALF_STEP[dtype] * (1 + 2 ** -8) + 3 * 2 * 2.0 ** -24 * x.double().abs().amax(
        -1, keepdim=True) * (1 + HALF_STEP[dtype]) + LEAST[dtype]


def sides(cache):
    """K and V, each [blocks, tokens, heads, width], of a cache in either layout (views)."""
    if cache.ndim == 5:
        return cache[0], cache[1]
    both = cache.permute(0, 2, 1, 3)
    width = both.shape[-1] // 2
    return both[..., :width], both[..., width:]


def rows_of(lengths, starts, s):
    """The step's rows of sequence s, and the position of its first."""
    first, end = (s, s + 1) if starts is None else (int(starts[s]), int(starts[s + 1]))
    return first, end, int(lengths[s]) - (end - first)


def slots_of(tables, lengths, starts, size, blocks):
    """(row, sequence, position, block, slot) of every row that has a place."""
    found = []
    for s in range(len(lengths)):
        first, end, at = rows_of(lengths, starts, s)
        for row in range(first, end):
            position = at + row - first
            page = position // size
            if position >= 0 and page < tables.shape[1] and 0 <= int(tables[s, page]) < blocks:
                found.append((row, s, position, int(tables[s, page]), position % size))
    return found


def scale_of(top):
    """The e8m0 byte of the least power of two s with top <= 448 s, at least 2^-126."""
    e = -126
    while 448 * 2.0 ** e < top:
        e += 1
    return e + 127


def dequantised(cache, scales):
    """K and V in 64 bits, each [blocks, tokens, heads, width]."""
    out = []
    for c, side in enumerate(sides(cache)):
        side = side.float().double()
        if scales is not None:
            byte = scales[..., c].view(torch.uint8).double()
            side = side * torch.where(byte == 255, math.nan, 2 ** (byte - 127))[
                :, None, :, None]
        out.append(side)
    return out


def attend64(query, keys, values, tables, lengths, starts=None, *, scale=None, window=None, causal=True):
    """(out, lse) for K and V [blocks, tokens, heads, width] in 64 bits; rows that see nothing: zeros and -inf."""
    tokens, heads, width = query.shape
    blocks, size, kv, _ = keys.shape
    out = torch.zeros(query.shape, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    for s in range(len(lengths)):
        first, end, at = rows_of(lengths, starts, s)
        reach = min(int(lengths[s]), tables.shape[1] * size)
        places = torch.tensor([int(tables[s, p // size]) * size + p % size for p in range(reach)
                               ]).long().reshape(-1)
        known = (places >= 0) & (places < blocks * size)
        for row in range(first, end):
            position = at + row - first
            see = known.clone()
            line = torch.arange(reach)
            if causal:
                see &= line <= position
            if window is not None:
                see &= line > position - window
            if position < 0 or not see.any():
                continue
            where = places[see]
            k, v = keys.reshape(blocks * size, kv, width)[where], values.reshape(blocks * size, kv, width)[where]
            for h in range(heads):
                g = h // (heads // kv)
                scores = (k[:, g] @ query[row, h].double()) * (width ** -0.5 if scale is None else scale)
                top = scores.max()
                weights = (scores - top).exp()
                lse[row, h] = top + weights.sum().log()
                out[row, h] = weights @ v[:, g] / weights.sum()
    return out, lse
