"""The operators beside the snapshot dataplane, measured: rotating positions in, filling a layer's paged cache, and
attending over it.

A case is one call a serving program makes for one layer: ``rotate`` turns a tensor's heads by the positions of its
tokens (one axis for text, several for images and video), ``append`` rotates a step's queries and keys and puts keys
and values into the blocks that the block tables name, ``attend`` reads them back as attention, for single tokens and
for prompts.  Caches are the layouts that the dataplane registers (vLLM's ``[blocks, heads, tokens, 2 * width]`` view
and the K/V-split ``[2, blocks, tokens, heads, width]``), in 16 bits or in e4m3 with a power-of-two scale (e8m0) for
each block of tokens and head.  Geometries are the models that this repository's benchmark and tests use (Qwen3-8B:
8 KV heads of 128 with 32 query heads, whole or one of eight ranks; Qwen3-1.7B: 16 query heads) and generic odd ones.

The plain forms compute in 32 bits from the same tensors and round once.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "fp32": torch.float32}
QWEN3_8B = dict(heads=32, kv_heads=8, head_dim=128, block_size=16, dtype="bf16")
QWEN3_8B_TP8 = dict(QWEN3_8B, heads=4, kv_heads=1)
QWEN3_1_7B = dict(QWEN3_8B, heads=16)
#: A generic model whose rows are neither whole KiB nor powers of two.
ODD = dict(heads=6, kv_heads=3, head_dim=80, dtype="fp16")

#: ``new``: tokens a sequence adds, at most; ``length``: tokens it has then, at most; ``ragged``: 0 for every sequence
#: at those, else the seed of their spread.  ``window``: 0 for none.
ROTATE = dict(kind="rotate", ragged=0, interleaved=False, inverse=False)
APPEND = dict(kind="append", axes=1, interleaved=False)
ATTEND = dict(kind="attend", window=0, lse=False)

#: Floating operations and bytes of the largest listed cases: no drawn one passes them.
MOST_FLOPS = 4 * 128 * 32 * (8192 * 8193 // 2)
MOST_BYTES = 512 << 20
#: Rows of the tables of angles.
FARTHEST = 40960


def listed():
    return [
        # Latency: one image's patches, rotated by height and width.
        dict(ROTATE, name="rotate-image", dtype="bf16", heads=16, head_dim=80, tokens=256, axes=2),
        # A long video prompt by time, height and width: the largest rotation.
        dict(ROTATE, name="rotate-video", dtype="bf16", heads=32, head_dim=128, tokens=16384, axes=3),
        # Latency: the token that one session adds in a decode step.
        dict(APPEND, **QWEN3_8B, name="append-one", layout="vllm", cache="e4m3", seqs=1, new=1, length=4095, ragged=0),
        # A decode step of a full batch, blocks filled to every extent.
        dict(APPEND, **QWEN3_8B, name="append-batch", layout="kv_split", cache="e4m3", seqs=64, new=1, length=8192,
             ragged=3),
        # Whole prompts into a 16-bit cache: the largest append.
        dict(APPEND, **QWEN3_8B, name="append-prompt", layout="vllm", cache="bf16", seqs=2, new=8185, length=8185,
             ragged=0),
        # Ragged chunks behind partly filled 8-bit blocks, adjacent pairs, three axes, rows of 80.
        dict(APPEND, **ODD, name="append-chunks-odd", block_size=32, layout="kv_split", cache="e4m3", seqs=7, new=700,
             length=2500, ragged=5, axes=3, interleaved=True),
        # Latency: a short reply on one of eight ranks.
        dict(ATTEND, **QWEN3_8B_TP8, name="attend-one-short", layout="vllm", cache="bf16", seqs=1, new=1, length=75,
             ragged=0),
        # One long session alone: few rows, a long axis.
        dict(ATTEND, **QWEN3_8B, name="attend-one-long", layout="vllm", cache="e4m3", seqs=1, new=1, length=32768,
             ragged=0, lse=True),
        # A decode step of a full batch of ragged sessions: the largest single-token case.
        dict(ATTEND, **QWEN3_8B, name="attend-batch", layout="kv_split", cache="e4m3", seqs=64, new=1, length=8192,
             ragged=7),
        # The same for a generic model: rows of 80, a sliding window, batch padding (lengths of 0) among the sequences.
        dict(ATTEND, **ODD, name="attend-batch-odd", block_size=32, layout="vllm", cache="fp16", seqs=24, new=1,
             length=3000, ragged=9, window=1000),
        # Prompt chunks and single tokens in one step over an 8-bit cache.
        dict(ATTEND, **QWEN3_1_7B, name="attend-chunks", layout="vllm", cache="e4m3", seqs=12, new=512, length=7700,
             ragged=11),
        # A whole 8k-token prompt: the largest case.
        dict(ATTEND, **QWEN3_8B, name="attend-prompt", layout="kv_split", cache="bf16", seqs=1, new=8192, length=8192,
             ragged=0),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    while True:
        kind = rng.choice(["rotate", "append", "append", "attend", "attend", "attend"])
        kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 4, 8])
        case = dict(dtype=rng.choice(["bf16", "bf16", "fp16"]), heads=kv_heads * group,
                    head_dim=rng.choice([64, 80, 96, 112, 128, 128, 256]))
        if kind == "rotate":
            case = dict(ROTATE, **case, tokens=spread(rng, 1, 16384), axes=rng.choice([1, 2, 3]),
                        interleaved=rng.random() < 0.3, inverse=rng.random() < 0.3)
        else:
            length = spread(rng, 1, 32768)
            case.update(kv_heads=kv_heads, block_size=rng.choice([16, 16, 32, 64, 24]), length=length,
                        layout=rng.choice(["vllm", "kv_split"]), cache=rng.choice([case["dtype"], "e4m3", "e4m3"]),
                        seqs=spread(rng, 1, 96), ragged=rng.randrange(1, 1 << 20),
                        new=1 if rng.random() < 0.5 else spread(rng, 1, length))
            if kind == "append":
                case = dict(APPEND, **case)
                case.update(axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.3)
            else:
                case = dict(ATTEND, **case)
                case.update(window=rng.choice([0, 0, 0, spread(rng, 1, 2 * length)]), lse=rng.random() < 0.3)
        need = work(case)
        if need["bytes"] <= MOST_BYTES and need["flops"] <= MOST_FLOPS and room(case) <= 24 << 30:
            return case


def extents(case):
    """Tokens that each sequence adds, and has then."""
    seqs, new, length = case["seqs"], case["new"], case["length"]
    if not case["ragged"]:
        return [new] * seqs, [length] * seqs
    rng, added, lengths = random.Random(case["ragged"]), [], []
    for s in range(seqs):
        n = new if s == 0 else 1 if new == 1 or rng.random() < 0.3 else spread(rng, 1, new)
        added.append(n)
        total = length if s == 0 else max(n, spread(rng, max(1, length // 16), length))
        # Single rows that pad a captured batch: a sequence of no tokens.
        lengths.append(0 if case["kind"] == "attend" and n == 1 and s and rng.random() < 0.05 else total)
    return added, lengths


def seen(n, length, window):
    """(query, key) pairs of a sequence's n last tokens, and the keys that any of them sees."""
    if not window or window >= length:
        # max(0, ...): the query rows ahead of position 0 of a padded sequence see nothing
        first = max(0, length - n)
        return (length * (length + 1) - first * (first + 1)) // 2, length
    pairs = sum(min(p + 1, window) for p in range(max(0, length - n), length))
    low = max(0, max(0, length - n) - window + 1)
    return pairs, length - low


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    width = case["head_dim"]
    if case["kind"] == "rotate":
        turned = case["tokens"] * case["heads"] * width
        return {"bytes": 2 * size * turned + case["tokens"] * (width * 4 + 8 * case["axes"]), "flops": 3 * turned}
    added, lengths = extents(case)
    tokens, kv, heads = sum(added), case["kv_heads"], case["heads"]
    held = 1 if case["cache"] == "e4m3" else 2
    if case["kind"] == "append":
        moved = tokens * width * (2 * heads * size + 2 * kv * (size + held))
        tables = tokens * (width * 4 + 8 * case["axes"])
        return {"bytes": moved + tables, "flops": 3 * tokens * width * (heads + kv)}
    sights = [seen(n, length, case["window"]) for n, length in zip(added, lengths)]
    keys = sum(k for _, k in sights)
    moved = 2 * tokens * heads * width * size + 2 * keys * kv * width * held
    if case["cache"] == "e4m3":
        moved += 2 * keys * kv // case["block_size"]
    return {"bytes": moved + 4 * keys // case["block_size"], "flops": 4 * width * heads * sum(p for p, _ in sights)}


def room(case):
    """Bytes of the plain form's largest intermediates."""
    if case["kind"] != "attend":
        return work(case)["bytes"] * 8
    added, lengths = extents(case)
    return 4 * case["seqs"] * (max(added) * max(lengths) * case["heads"]
                               + 2 * max(lengths) * case["kv_heads"] * case["head_dim"])


def blocks_of(lengths, size):
    return [-(-length // size) for length in lengths]


def angles(case, device):
    """The cosines and sines of every position's angles, one pair of values a rotated pair, computed in 64 bits."""
    half = case["head_dim"] // 2
    frequencies = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    turns = torch.arange(FARTHEST, dtype=torch.float64, device=device)[:, None] * frequencies
    return torch.stack([turns.cos(), turns.sin()], -1).float()


def axes_of(case):
    """Which axis turns which pair: time takes the first quarter, height and width share the rest."""
    half, axes = case["head_dim"] // 2, case["axes"]
    if axes == 1:
        return None
    first = 0 if axes == 2 else half // 4
    return tuple([0] * first + [axes - 2] * ((half - first + 1) // 2) + [axes - 1] * ((half - first) // 2))


def place(case, tokens, gen, device):
    """Positions: the text's count for one axis, a grid's rows and columns for the others."""
    at = torch.randint(0, FARTHEST - tokens, (1,), generator=gen, device=device)
    line = at + torch.arange(tokens, device=device)
    if case["axes"] == 1:
        return line
    return torch.stack([line // 64, line % 64 // 8, line % 8][3 - case["axes"]:]) + at // 2


def normal(shape, dtype, gen, device):
    return torch.randn(shape, dtype=torch.float32, generator=gen, device=device).to(dtype)


def split(cache, layout):
    """K and V of a layer's cache, each [blocks, tokens, heads, width], as views."""
    if layout == "vllm":
        both = cache.permute(0, 2, 1, 3)
        return both.chunk(2, -1)
    return cache[0], cache[1]


def prepare(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype, width, heads = TYPES[case["dtype"]], case["head_dim"], case["heads"]
    if case["kind"] == "rotate":
        tokens = case["tokens"]
        return {"case": case, "x": normal((tokens, heads, width), dtype, gen, device), "table": angles(case, device),
                "positions": place(case, tokens, gen, device), "axes": axes_of(case)}
    added, lengths = extents(case)
    tokens, size, kv = sum(added), case["block_size"], case["kv_heads"]
    counts = blocks_of(lengths, size)
    # An append touches few of its sequences' blocks: the rest of the tables name blocks of a small pool.
    touched = counts if case["kind"] == "attend" else [
        c - (length - n) // size for c, length, n in zip(counts, lengths, added)]
    blocks = sum(touched) + sum(touched) // 4 + 2
    ids = torch.randperm(blocks - 1, generator=gen, device=device) + 1
    table = torch.randint(1, blocks, (case["seqs"], max(max(counts), 1)), generator=gen, device=device)
    at = 0
    for s, (count, some) in enumerate(zip(counts, touched)):
        table[s, count - some:count] = ids[at:at + some]
        at += some
    held = TYPES[case["cache"]]
    shape = (blocks, size, kv, 2 * width) if case["layout"] == "vllm" else (2, blocks, size, kv, width)
    state = {"case": case, "tables": table.to(torch.int32), "most": max(lengths),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=device), "added": max(added),
             "starts": None if max(added) == 1 else torch.tensor(
                 [sum(added[:s]) for s in range(case["seqs"] + 1)], dtype=torch.int32, device=device)}
    # A cache that has been in use: stale blocks and slots among the sequences' own; a few channels are large.
    loud = torch.where(torch.rand((width,), generator=gen, device=device) < 0.03, 8.0, 1.0)
    stored = torch.randn(shape, generator=gen, device=device) * loud.repeat(shape[-1] // width)
    state["scales"] = None
    if case["cache"] == "e4m3":
        keys, values = split(stored if case["layout"] == "kv_split" else stored.permute(0, 2, 1, 3), case["layout"])
        exponents = torch.stack([127 + power(half.abs().amax((1, 3))) for half in (keys, values)], -1)
        state["scales"] = exponents.to(torch.uint8).view(torch.float8_e8m0fnu)
        for c, half in enumerate((keys, values)):
            half /= torch.exp2(exponents[:, None, :, c, None].float() - 127)
    stored = stored.to(held)
    state["cache"] = stored.permute(0, 2, 1, 3) if case["layout"] == "vllm" else stored
    if case["kind"] == "append":
        # One projection's output, cut into queries, keys and values.
        fused = normal((tokens, heads + 2 * kv, width), dtype, gen, device)
        state["query"], state["key"], state["value"] = fused.split([heads, kv, kv], 1)
        state["table"], state["axes"] = angles(case, device), axes_of(case)
        state["positions"] = None if case["axes"] == 1 else place(case, tokens, gen, device)
    else:
        state["query"] = normal((tokens, heads, width), dtype, gen, device)
    if own:
        from kvsnap_amd.attention import PagedCache
        state["layer"] = PagedCache(state["cache"], size, scales=state["scales"])
    return state


def run(state):
    case = state["case"]
    if own:
        from kvsnap_amd.attention import rotate
        if case["kind"] == "rotate":
            return rotate(state["x"], state["positions"], state["table"], axes=state["axes"],
                          interleaved=case["interleaved"], inverse=case["inverse"])
        layer = state["layer"]
        if case["kind"] == "append":
            query = layer.append(state["key"], state["value"], state["tables"], state["lengths"],
                                 query_starts=state["starts"], query=state["query"], positions=state["positions"],
                                 rotary=state["table"], axes=state["axes"], interleaved=case["interleaved"])
            return appended(state, query)
        return layer.attend(state["query"], state["tables"], state["lengths"], query_starts=state["starts"],
                            max_length=state["most"], window=case["window"] or None, return_lse=case["lse"])
    if case["kind"] == "rotate":
        return rotated(state["x"], state["positions"], state, case["inverse"]).to(state["x"].dtype)
    return plain_append(state) if case["kind"] == "append" else plain_attend(state)


def appended(state, query):
    out = {"query": query, "cache": state["cache"]}
    if state["scales"] is not None:
        out["scales"] = state["scales"]
    return out


# ---- the plain forms


def power(top):
    """The least e for which 448 * 2**e is at least ``top`` (e4m3's largest value is 448), within e8m0's range."""
    mantissa, exponent = torch.frexp(top.float().clamp_min(448 * 2.0 ** -126) / 448)
    return exponent - (mantissa == 0.5).to(exponent.dtype)


def rotated(x, positions, state, inverse=False):
    """x [tokens, heads, width] in 32 bits, each pair (a, b) turned to (a cos - b sin, b cos + a sin)."""
    half, axes = x.shape[-1] // 2, state["axes"]
    pairs = torch.arange(half, device=x.device)
    where = positions[:, None] if axes is None else positions.T[:, torch.tensor(axes, device=x.device)]
    turn = state["table"][where, pairs]
    cos, sin = turn[:, None, :, 0], turn[:, None, :, 1]
    if inverse:
        sin = -sin
    x = x.float()
    if state["case"]["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def owners(state, tokens):
    """Each new token's sequence, and its position there."""
    lengths, device = state["lengths"].long(), state["lengths"].device
    if state["starts"] is None:
        return torch.arange(tokens, device=device), lengths - 1
    starts, rows = state["starts"].long(), torch.arange(tokens, device=device)
    of = torch.searchsorted(starts, rows, right=True) - 1
    return of, lengths[of] - starts[of + 1] + rows


def plain_append(state):
    case, size = state["case"], state["case"]["block_size"]
    of, at = owners(state, state["key"].shape[0])
    positions = at if state["positions"] is None else state["positions"]
    query = rotated(state["query"], positions, state).to(state["query"].dtype)
    new = torch.stack([rotated(state["key"], positions, state), state["value"].float()], 1)  # [tokens, 2, heads, width]
    block, slot = state["tables"].long()[of, at // size], at % size
    keys, values = split(state["cache"], case["layout"])
    if state["scales"] is None:
        keys[block, slot] = new[:, 0].to(keys.dtype)
        values[block, slot] = new[:, 1].to(keys.dtype)
        return appended(state, query)
    count, heads, device = keys.shape[0], keys.shape[2], keys.device
    finite = new.isfinite()
    top = torch.where(finite, new.abs(), 0).amax(-1).transpose(1, 2)                       # [tokens, heads, 2]
    tops = torch.zeros((count, heads, 2), device=device).scatter_reduce_(
        0, block[:, None, None].expand_as(top), top, "amax")
    first = torch.full((count,), size, device=device).scatter_reduce_(0, block, slot, "amin")
    before = state["scales"].view(torch.uint8).int()
    after = 127 + power(tops)
    after = torch.where((first > 0)[:, None, None], torch.maximum(after, before), after)
    after = torch.where((first < size)[:, None, None], after, before)
    kept = torch.arange(size, device=device) < torch.where(first < size, first, 0)[:, None]  # slots filled before
    shrink = torch.exp2((before - after).float())
    for c, half in enumerate((keys, values)):
        stored = half.float()
        lesser = (stored * shrink[:, None, :, c, None]).to(half.dtype).view(torch.uint8)
        raw = half.view(torch.uint8)
        raw.copy_(torch.where(kept[:, :, None, None], lesser, raw))
        scaled = new[:, c] * torch.exp2(127.0 - after[block, :, c].float())[..., None]
        raw[block, slot] = torch.where(finite[:, c], scaled, math.nan).to(half.dtype).view(torch.uint8)
    state["scales"].view(torch.uint8).copy_(after.to(torch.uint8))
    return appended(state, query)


def plain_attend(state):
    case, size, query = state["case"], state["case"]["block_size"], state["query"]
    tokens, heads, width = query.shape
    of, at = owners(state, tokens)
    kv, most, added = case["kv_heads"], max(state["most"], 1), state["added"]
    seqs, lengths, device = state["lengths"].shape[0], state["lengths"].long(), query.device
    line = torch.arange(most, device=device)
    pages = state["tables"].long()[:, line // size]                                        # [seqs, most]
    sides = []
    for c, half in enumerate(split(state["cache"], case["layout"])):
        raw = half if state["scales"] is None else half.view(torch.uint8)
        side = raw[pages, line % size].view(half.dtype).float()                            # [seqs, most, kv, width]
        if state["scales"] is not None:
            side = side * torch.exp2(state["scales"].view(torch.uint8)[..., c].float() - 127)[pages][..., None]
        sides.append(side.transpose(1, 2))
    # Each sequence's query rows behind one another, padded to the longest: [seqs, kv, group * added, width]
    row = torch.zeros_like(of) if state["starts"] is None else (
        torch.arange(tokens, device=device) - state["starts"].long()[of])
    padded = torch.zeros((seqs, added, heads, width), device=device)
    padded[of, row] = query.float()
    place_of = torch.full((seqs, added), -1, device=device)
    place_of[of, row] = at
    padded = padded.view(seqs, added, kv, heads // kv, width).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, width)
    scores = (padded @ sides[0].transpose(2, 3)) * width ** -0.5
    open_ = (line <= place_of[..., None]) & (line < lengths[:, None, None])                # [seqs, added, most]
    if case["window"]:
        open_ &= line > place_of[..., None] - case["window"]
    scores = scores.view(seqs, kv, heads // kv, added, most).masked_fill_(~open_[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(seqs, kv, -1, most) @ sides[1]).view(seqs, kv, heads // kv, added, width)
    out = torch.where(total > 0, out / total, 0)
    out = out.permute(0, 3, 1, 2, 4)[of, row].reshape(tokens, heads, width).to(query.dtype)
    if not case["lse"]:
        return out
    lse = (total.log() + top)[..., 0].permute(0, 3, 1, 2)[of, row].reshape(tokens, heads)
    return out, lse


# ---- the definitions, in 64 bits


def turned_exactly(x, positions, state, inverse=False):
    """Each pair as a complex number times e^(i angle)."""
    table = state["table"].double()
    axes = state["axes"] or (0,) * (x.shape[-1] // 2)
    positions = positions.reshape(-1, x.shape[0])
    turn = torch.stack([torch.view_as_complex(table[:, pair].contiguous())[positions[axis]]
                        for pair, axis in enumerate(axes)], -1)[:, None]
    if inverse:
        turn = turn.conj()
    x = x.double()
    if state["case"]["interleaved"]:
        return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    low, high = x.chunk(2, -1)
    both = torch.complex(low.contiguous(), high.contiguous()) * turn
    return torch.cat([both.real, both.imag], -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotate":
        return turned_exactly(state["x"], state["positions"], state, case["inverse"])
    return exact_append(state) if case["kind"] == "append" else exact_attend(state)


def exact_append(state):
    case, size = state["case"], state["case"]["block_size"]
    added, lengths = extents(case)
    positions = state["positions"]
    if positions is None:
        positions = torch.cat([torch.arange(length - n, length) for n, length in zip(added, lengths)])
        positions = positions.to(state["key"].device)
    query = turned_exactly(state["query"], positions, state)
    key, value = turned_exactly(state["key"], positions, state), state["value"].double()
    cache = state["cache"].double()
    sides = [(half, fresh) for half, fresh in zip(split(cache, case["layout"]), (key, value))]
    tables = state["tables"].tolist()
    exponents = None if state["scales"] is None else state["scales"].view(torch.uint8).long()
    at = 0
    for s, (n, length) in enumerate(zip(added, lengths)):
        first = length - n
        for page in range(first // size, -(-length // size)):
            low, high = max(first, page * size), min(length, (page + 1) * size)
            block, slots = tables[s][page], slice(low - page * size, high - page * size)
            rows = slice(at + low - first, at + high - first)
            for c, (half, fresh) in enumerate(sides):
                if exponents is None:
                    half[block, slots] = fresh[rows]
                    continue
                top = fresh[rows].abs().amax((0, 2)) / 448
                power_of = torch.ceil(torch.log2(top.clamp_min(2.0 ** -126))).long() + 127
                if slots.start:
                    power_of = torch.maximum(power_of, exponents[block, :, c])
                    half[block, :slots.start] *= torch.exp2((exponents[block, :, c] - power_of).double())[:, None]
                exponents[block, :, c] = power_of
                half[block, slots] = fresh[rows] * torch.exp2((127 - power_of).double())[:, None]
        at += n
    out = {"query": query, "cache": cache}
    if exponents is not None:
        out["scales"] = torch.exp2((exponents - 127).double())
    return out


def exact_attend(state):
    case, query = state["case"], state["query"]
    added, lengths = extents(case)
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    lse = torch.full(query.shape[:2], -math.inf, dtype=torch.float64, device=query.device)
    group, start = case["heads"] // case["kv_heads"], 0
    keys, values = split(state["cache"], case["layout"])
    for s, (n, length) in enumerate(zip(added, lengths)):
        rows, start = slice(start, start + n), start + n
        if not length:
            continue
        pages = state["tables"][s, :-(-length // case["block_size"])].tolist()
        queries = torch.arange(length - n, length, device=query.device)[:, None]
        line = torch.arange(length, device=query.device)
        hidden = line > queries
        if case["window"]:
            hidden |= line <= queries - case["window"]
        for h in range(case["kv_heads"]):
            held = []
            for c, half in enumerate((keys, values)):
                side = half.view(torch.uint8)[pages, :, h].view(half.dtype) if state["scales"] is not None else (
                    half[pages, :, h])
                side = side.double()
                if state["scales"] is not None:
                    exponents = state["scales"].view(torch.uint8)[pages, h, c].double() - 127
                    side = side * torch.exp2(exponents)[:, None, None]
                held.append(side.flatten(0, 1)[:length])
            for g in range(h * group, (h + 1) * group):
                scores = (query[rows, g].double() @ held[0].T) / math.sqrt(case["head_dim"])
                scores.masked_fill_(hidden, -math.inf)
                lse[rows, g] = torch.logsumexp(scores, -1)
                out[rows, g] = torch.softmax(scores, -1).nan_to_num(0.0) @ held[1]
    return (out, lse) if case["lse"] else out
