"""rotate and PagedCache.append against their definitions in 64 bits, on the GPU."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from kvsnap_amd.attention import PagedCache, block_scales, rotary_table, rotate
from paged_reference import (E4M3, HALF_STEP, rotate64, rotation_bound, scale_of, sides, slots_of, table64)

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip_library")]

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def made(shape, dtype, seed, loud=1.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * loud
    return x.to(dtype)


def close(got, want, bound):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    off = torch.where(want.isnan(), torch.zeros(()).double(), (got - want).abs() - bound)
    assert off.max() <= 0, f"off by up to {off.max():.3g} more than a rounding"


# ---------------------------------------------------------------- rotate


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("tokens,heads,width,pairs,interleaved,inverse", [
    (1, 1, 16, 8, False, False),
    (1, 1, 16, 8, True, False),
    (37, 3, 80, 40, False, False),
    (37, 3, 80, 40, True, True),
    (5, 32, 128, 64, False, True),
    (64, 4, 128, 16, False, False),        # a quarter of the values turned
    (64, 4, 128, 16, True, False),
    (9, 5, 256, 128, False, False),
    (300, 2, 64, 24, False, False),
])
def test_rotate_is_its_definition(dtype, tokens, heads, width, pairs, interleaved, inverse):
    table = table64(2 * pairs, 5000)
    x = made((tokens, heads, width), dtype, tokens + width)
    positions = torch.randint(0, 5000, (tokens,), generator=torch.Generator().manual_seed(1))
    want = rotate64(x, positions, table, None, interleaved, inverse)
    got = rotate(x.cuda(), positions.cuda(), table.float().cuda(), interleaved=interleaved, inverse=inverse)
    assert got.dtype == dtype
    close(got, want, rotation_bound(x, want, dtype))


@pytest.mark.parametrize("narrow", [False, True])
@pytest.mark.parametrize("sections", ["runs", "turns", "within-a-unit"])
def test_rotate_by_several_axes(sections, narrow):
    tokens, pairs = 50, 64
    axes = {"runs": [0] * 16 + [1] * 24 + [2] * 24, "turns": [j % 3 for j in range(pairs)],
            "within-a-unit": [0] * 13 + [1] * 30 + [2] * 21}[sections]
    table = table64(128, 300)
    positions = torch.randint(0, 300, (3, tokens), generator=torch.Generator().manual_seed(3))
    x = made((tokens, 6, 128), BF16, 4)
    want = rotate64(x, positions, table, axes)
    on_gpu = positions.cuda().to(torch.int32 if narrow else torch.int64)
    close(rotate(x.cuda(), on_gpu, table.float().cuda(), axes=axes), want, rotation_bound(x, want, BF16))


def test_rotate_strided_rows_in_place_and_back():
    """Heads cut from a wider projection, turned in place (its other columns untouched) and turned back."""
    fused = made((33, 10, 64), FP32, 5).cuda()
    before = fused.clone()
    table = rotary_table(64, 100, device="cuda")
    positions = torch.arange(33, device="cuda")
    part = fused[:, 2:7]
    assert rotate(part, positions, table, out=part) is part
    assert torch.equal(fused[:, :2], before[:, :2]) and torch.equal(fused[:, 7:], before[:, 7:])
    want = rotate64(before[:, 2:7].cpu(), positions.cpu(), table.cpu().double())
    close(part, want, rotation_bound(before[:, 2:7].cpu(), want, FP32))
    back = rotate(part, positions, table, inverse=True)
    # Two rotations, each within its bound, and the tables' fp32 cosines and sines: cos^2 + sin^2 is 1 within 2^-23.
    bound = 3 * rotation_bound(before[:, 2:7].cpu(), want.abs() + before[:, 2:7].cpu().abs(), FP32) + (
        2.0 ** -22 * before[:, 2:7].cpu().double().abs())
    close(back, before[:, 2:7].cpu().double(), bound)


def test_rotate_gives_nan_where_a_position_has_no_angle():
    table = table64(64, 10)
    x = made((4, 2, 80), BF16, 6)
    positions = torch.tensor([-1, 0, 9, 10])
    want = rotate64(x, positions, table)
    assert want[0, :, :64].isnan().all() and not want[0, :, 64:].isnan().any()
    close(rotate(x.cuda(), positions.cuda(), table.float().cuda()), want, rotation_bound(x, want, BF16))


def test_rotate_of_nothing():
    table = rotary_table(64, 10, device="cuda")
    assert rotate(torch.empty((0, 2, 64), device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"),
                  table).shape == (0, 2, 64)


def test_the_rotary_table_is_exact_far_out():
    table = rotary_table(128, 40000, base=1e6, device="cuda").cpu()
    pairs = torch.arange(64, dtype=torch.float64)
    want = 39999 * 1e6 ** (-pairs / 64)
    assert (table[39999, :, 0].double() - want.cos()).abs().max() <= 2.0 ** -24
    assert (table[39999, :, 1].double() - want.sin()).abs().max() <= 2.0 ** -24


def test_the_gradient_of_a_rotation_is_the_turn_back():
    """d/dx of sum(w * rotate(x)) is rotate(w, inverse): against central differences of the definition in 64 bits."""
    tokens, heads, width = 3, 2, 32
    table, positions = table64(width, 50), torch.tensor([0, 7, 49])
    x, w = made((tokens, heads, width), FP32, 7), made((tokens, heads, width), FP32, 8)
    got = rotate(w.cuda(), positions.cuda(), table.float().cuda(), inverse=True).cpu().double()
    step = 2.0 ** -10
    for index in range(0, x.numel(), 5):
        moved = torch.zeros(x.numel(), dtype=torch.float64)
        moved[index] = step
        moved = moved.reshape(x.shape)
        up, down = (rotate64(x.double() + sign * moved, positions, table) for sign in (1, -1))
        slope = ((up - down) * w.double()).sum() / (2 * step)
        # A rotation is linear: the differences are exact but for 64-bit rounding of values below 10 over 2^-9.
        assert abs(got.flatten()[index] - slope) <= 2.0 ** -20 * (1 + abs(slope))


# ---------------------------------------------------------------- append


def make_cache(layout, blocks, size, kv, width, dtype, seed, device="cuda"):
    """(cache, scales) of stale values, as a cache in use holds."""
    shape = (blocks, size, kv, 2 * width) if layout != "kv_split" else (2, blocks, size, kv, width)
    if layout == "vllm-hnd":
        shape = (blocks, kv, size, 2 * width)
    backing = made(shape, torch.float32, seed, 3.0).to(dtype).to(device)
    cache = backing if layout in ("kv_split", "vllm-hnd") else backing.permute(0, 2, 1, 3)
    scales = None
    if dtype == E4M3:
        rows, views = block_scales(blocks, 3, kv, device=device)
        rows.view(torch.uint8).copy_(torch.randint(118, 130, rows.shape, generator=torch.Generator().manual_seed(seed)))
        scales = views[1]
    return cache, scales


def plan(added, lengths, size, blocks, seed, spare=0):
    """int32 tables of distinct blocks, lengths and starts on the CPU."""
    rng = random.Random(seed)
    ids = rng.sample(range(blocks), blocks)
    wide = max([-(-n // size) for n in lengths] + [1]) + spare
    tables = torch.full((len(lengths), wide), -7, dtype=torch.int32)
    for s, n in enumerate(lengths):
        for page in range(-(-n // size)):
            tables[s, page] = ids.pop()
    starts = [sum(added[:s]) for s in range(len(added) + 1)]
    return tables, torch.tensor(lengths, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32)


def expect_append(cache, scales, key, value, turned, tables, lengths, starts, size, slack):
    """The cache in 64 bits after an append, how far each value may be off, and the scales' bytes: the values are
    those stored (an e4m3 cache's in its blocks' scales)."""
    dtype = cache.dtype
    want = [side.float().double() for side in sides(cache)]
    bound = [torch.zeros_like(side) for side in want]
    bytes_ = None if scales is None else scales.view(torch.uint8).int().clone()
    placed = slots_of(tables, lengths, starts, size, want[0].shape[0])
    for c, new in enumerate((turned, value.double())):
        if scales is None:
            for row, _, _, block, slot in placed:
                want[c][block, slot] = new[row]
                bound[c][block, slot] = new[row].abs() * HALF_STEP[dtype] * (1 + 2 ** -8) * (c == 0) + slack[c][row]
            continue
        by_block = {}
        for row, _, _, block, slot in placed:
            by_block.setdefault(block, []).append((row, slot))
        for block, rows in by_block.items():
            first = min(slot for _, slot in rows)
            for h in range(new.shape[1]):
                top = max(float(torch.where(new[row, h].isfinite(), new[row, h].abs(), 0.0).max()) for row, _ in rows)
                e = scale_of(top)
                before = int(bytes_[block, h, c])
                if first:
                    e = max(e, before)
                    old = want[c][block, :first, h] * 2.0 ** (before - e)
                    want[c][block, :first, h] = old.float().to(dtype).double()       # exact, then one rounding
                bytes_[block, h, c] = e
                for row, slot in rows:
                    stored = new[row, h] * 2.0 ** (127 - e)
                    stored = torch.where(stored.isfinite(), stored, math.nan)
                    want[c][block, slot, h] = stored
                    bound[c][block, slot, h] = stored.abs() * HALF_STEP[dtype] * (1 + 2 ** -8) + 2.0 ** -10 + (
                        slack[c][row, h] * 2.0 ** (127 - e))
    return want, bound, bytes_


APPENDS = [
    # added, lengths, block size, kv heads, query heads, width
    ([1], [1], 16, 1, 1, 16),
    ([1], [4096], 16, 8, 32, 128),
    ([1, 1, 1, 1, 1], [1, 16, 17, 31, 33], 16, 2, 4, 64),
    ([40, 1, 0, 17, 3], [40, 100, 50, 33, 35], 16, 3, 6, 80),
    ([7, 65, 1], [9, 65, 24], 24, 2, 2, 112),
    ([130], [150], 64, 1, 8, 256),
    ([33, 5], [33, 6], 1, 2, 2, 32),              # a token a block
    ([3] * 70, [3 + 2 * s for s in range(70)], 16, 1, 2, 64),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("layout", ["vllm", "vllm-hnd", "kv_split"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_is_its_definition(case, layout, held, dtype):
    added, lengths, size, kv, heads, width = APPENDS[case]
    blocks = sum(-(-n // size) for n in lengths) + 5
    cache, scales = make_cache(layout, blocks, size, kv, width, E4M3 if held == "e4m3" else dtype, case)
    tables, lengths, starts = plan(added, lengths, size, blocks, case, spare=1)
    tokens = sum(added)
    fused = made((tokens + 2, heads + 2 * kv, width), dtype, 10 + case)       # two rows of padding behind
    table = table64(width, 5000)
    interleaved = case % 2 == 1
    layer = PagedCache(cache, size, scales=scales)
    before, before_scales = cache.clone().cpu(), None if scales is None else scales.clone().cpu()
    q, k, v = fused.cuda().split([heads, kv, kv], 1)
    out = torch.full(q.shape, -5.0, dtype=dtype, device="cuda")
    got = layer.append(k, v, tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), query=q,
                       rotary=table.float().cuda(), interleaved=interleaved, query_out=out)
    assert got is out and (out[tokens:] == -5).all()
    at = torch.cat([torch.arange(int(n) - a, int(n)) for a, n in zip(added, lengths)])
    q, k, v = (t.cpu()[:tokens] for t in (q, k, v))
    turned = rotate64(q, at, table, None, interleaved)
    close(out[:tokens], turned, rotation_bound(q, turned, dtype))
    turned = rotate64(k, at, table, None, interleaved)
    slack = [rotation_bound(k, torch.zeros_like(turned), FP32).expand(turned.shape), torch.zeros(v.shape).double()]
    want, bound, bytes_ = expect_append(before, before_scales, k, v, turned, tables, lengths, starts, size, slack)
    for side, wanted, off in zip(sides(cache.cpu()), want, bound):
        close(side.float(), wanted, off)
    if scales is not None:
        assert torch.equal(scales.view(torch.uint8).cpu().int(), bytes_)


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
def test_append_without_starts_or_rotation_puts_one_row_a_sequence(held):
    lengths, size, kv, width = [1, 5, 16, 17, 0], 16, 2, 64
    cache, scales = make_cache("vllm", 9, size, kv, width, E4M3 if held == "e4m3" else BF16, 3)
    tables, lengths, _ = plan([1] * 5, lengths, size, 9, 3)
    key, value = made((5, kv, width), BF16, 1), made((5, kv, width), BF16, 2)
    before, before_scales = cache.clone().cpu(), None if scales is None else scales.clone().cpu()
    assert PagedCache(cache, size, scales=scales).append(key.cuda(), value.cuda(), tables.cuda(),
                                                         lengths.cuda()) is None
    want, bound, bytes_ = expect_append(before, before_scales, key, value, key.double(), tables, lengths, None, size,
                                        [torch.zeros(key.shape).double()] * 2)
    for side, wanted, off in zip(sides(cache.cpu()), want, bound):
        close(side.float(), wanted, off)
    if scales is not None:
        assert torch.equal(scales.view(torch.uint8).cpu().int(), bytes_)


def test_append_skips_pages_that_name_no_block():
    """Entries outside the cache, a table too narrow for the length, rows ahead of position 0: nothing is written."""
    size, kv, width, blocks = 16, 1, 32, 6
    for dtype in (BF16, E4M3):
        cache, scales = make_cache("kv_split", blocks, size, kv, width, dtype, 5)
        before, before_scales = cache.clone().cpu(), None if scales is None else scales.clone().cpu()
        tables = torch.tensor([[-1, 2], [blocks, 3], [4, 1 << 30], [0, 5]], dtype=torch.int32)
        lengths = torch.tensor([18, 18, 18, 40], dtype=torch.int32)          # the last: past its table
        starts = torch.tensor([0, 18, 36, 54, 94], dtype=torch.int32)
        key, value = made((94, kv, width), BF16, 1), made((94, kv, width), BF16, 2)
        PagedCache(cache, size, scales=scales).append(key.cuda(), value.cuda(), tables.cuda(), lengths.cuda(),
                                                      query_starts=starts.cuda())
        want, bound, _ = expect_append(before, before_scales, key, value, key.double(), tables, lengths, starts, size,
                                       [torch.zeros(key.shape).double()] * 2)
        for side, wanted, off in zip(sides(cache.cpu()), want, bound):
            close(side.float(), wanted, off)
        cache, scales = make_cache("kv_split", blocks, size, kv, width, dtype, 5)
        before = cache.clone()
        PagedCache(cache, size, scales=scales).append(
            key[:5].cuda(), value[:5].cuda(), tables[2:3].cuda(), torch.tensor([3], dtype=torch.int32).cuda(),
            query_starts=torch.tensor([0, 5], dtype=torch.int32).cuda())
        for side, old in zip(sides(cache.cpu().float()), sides(before.cpu().float())):
            old[4, :3] = side[4, :3]
            assert torch.equal(side, old)


def test_an_e4m3_block_grows_its_scale_and_keeps_it():
    """Token after token into one block: quiet, loud, quiet, a zero row, then values that are not finite."""
    size, kv, width = 16, 1, 32
    cache, scales = make_cache("vllm", 2, size, kv, width, E4M3, 6)
    scales.view(torch.uint8).fill_(200)                  # stale: a fresh block does not look at it
    layer = PagedCache(cache, size, scales=scales)
    rows = [made((1, kv, width), BF16, 20 + i, loud) for i, loud in enumerate((0.01, 30.0, 1.0, 0.0, 3000.0))]
    rows[2][0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan]).to(BF16)
    tables = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    top = 0.0
    for i, row in enumerate(rows):
        layer.append(row.cuda(), row.cuda(), tables, torch.tensor([i + 1], dtype=torch.int32, device="cuda"))
        finite = torch.where(row.isfinite(), row.abs(), 0).max().item()
        top = max(top, finite)
        assert (scales.view(torch.uint8)[1].cpu() == scale_of(top)).all(), i
    scale = 2.0 ** (scale_of(top) - 127)
    for side in sides(cache.cpu().float()):
        for i, row in enumerate(rows):
            wanted = torch.where(row[0, 0].isfinite(), row[0, 0].double(), math.nan)
            # Up to three roundings on the way: each half a step of the value, or half the least step of the scale then.
            close(side[1, i, 0].double() * scale, wanted, wanted.abs().nan_to_num() * 3.2 * 2.0 ** -4 + 1.2 * scale * 2.0 ** -9)


def test_append_on_a_side_stream_and_captured():
    size, kv, width, heads = 16, 2, 64, 4
    cache, scales = make_cache("kv_split", 8, size, kv, width, E4M3, 8)
    layer = PagedCache(cache, size, scales=scales)
    table = rotary_table(width, 200, device="cuda")
    tables = torch.tensor([[1, 2], [3, 4]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([1, 5], dtype=torch.int32, device="cuda")
    fused = made((2, heads + 2 * kv, width), FP16, 9).cuda()
    q, k, v = fused.split([heads, kv, kv], 1)
    start = cache.clone(), scales.view(torch.uint8).clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer.append(k, v, tables, lengths, query=q, rotary=table)
    stream.synchronize()
    cache.view(torch.uint8).copy_(start[0].view(torch.uint8))
    scales.view(torch.uint8).copy_(start[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer.append(k, v, tables, lengths, query=q, rotary=table)
    for step in range(4):
        fused.copy_(made(fused.shape, FP16, 30 + step, 2.0 ** step))
        graph.replay()
        torch.cuda.synchronize()
        replayed = cache.view(torch.uint8).clone(), scales.view(torch.uint8).clone(), captured.clone()
        cache.view(torch.uint8).copy_(start[0].view(torch.uint8))
        scales.view(torch.uint8).copy_(start[1])
        eager = layer.append(k, v, tables, lengths, query=q, rotary=table)
        assert torch.equal(eager, replayed[2])
        assert torch.equal(cache.view(torch.uint8), replayed[0])
        assert torch.equal(scales.view(torch.uint8), replayed[1])
        lengths += 1
        start = cache.clone(), scales.view(torch.uint8).clone()


def padded_batch(live, seqs, held, width=64, heads=3):
    """A step of ``seqs`` rows and sequences of which ``live``, spread among the others, have a row each (at most two)."""
    rng = random.Random(live)
    added = [0] * seqs
    for s in rng.sample(range(seqs), live):
        added[s] = rng.choice([1, 1, 2])
    blocks = seqs + 1
    cache, scales = make_cache("kv_split", blocks, 16, 1, width, E4M3 if held == "e4m3" else BF16, live)
    lengths = [n + rng.randrange(12) if n else 0 for n in added]
    tables, lengths, starts = plan(added, lengths, 16, blocks, live)
    fused = made((seqs + live, heads + 2, width), BF16, live)
    return cache, scales, tables, lengths, starts, fused, sum(added)


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("live,seqs", [(1, 600), (10, 600), (64, 600), (600, 600), (0, 600)])
def test_append_of_a_padded_batch_is_its_definition(live, seqs, held):
    cache, scales, tables, lengths, starts, fused, tokens = padded_batch(live, seqs, held)
    layer = PagedCache(cache, 16, scales=scales)
    before, before_scales = cache.clone().cpu(), None if scales is None else scales.clone().cpu()
    table = table64(64, 40)
    q, k, v = fused.cuda().split([3, 1, 1], 1)
    out = torch.full(q.shape, -5.0, dtype=BF16, device="cuda")
    layer.append(k, v, tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), query=q, rotary=table.float().cuda(),
                 query_out=out)
    assert (out[tokens:] == -5).all()
    added = (starts[1:] - starts[:-1]).tolist()
    at = torch.cat([torch.arange(int(n) - a, int(n)) for a, n in zip(added, lengths)])
    q, k, v = (t.cpu()[:tokens] for t in (q, k, v))
    if tokens:
        turned = rotate64(q, at, table)
        close(out[:tokens], turned, rotation_bound(q, turned, BF16))
    turned = rotate64(k, at, table) if tokens else k.double()
    slack = [rotation_bound(k, torch.zeros_like(turned), FP32).expand(turned.shape) if tokens else turned,
             torch.zeros(v.shape).double()]
    want, bound, bytes_ = expect_append(before, before_scales, k, v, turned, tables, lengths, starts, 16, slack)
    for side, wanted, off in zip(sides(cache.cpu()), want, bound):
        close(side.float(), wanted, off)
    if scales is not None:
        assert torch.equal(scales.view(torch.uint8).cpu().int(), bytes_)


def test_a_padded_batch_takes_no_longer_than_a_full_one():
    """Ten rows among 4096 sequences: a wave that holds the last of them and padding passes 4000 sequences in a few
    steps (a walk took 60 times a full batch's time)."""
    took = []
    for live in (4096, 10):
        cache, scales, tables, lengths, starts, fused, _ = padded_batch(live, 4096, "16-bit")
        if live == 10:              # the ten at the front, as a captured batch has them
            starts = torch.arange(4097, dtype=torch.int32).clamp(max=10)
        layer = PagedCache(cache, 16)
        tables, lengths, starts, (q, k, v) = tables.cuda(), lengths.cuda(), starts.cuda(), fused.cuda().split([3, 1, 1], 1)
        layer.append(k, v, tables, lengths, query_starts=starts, query=q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                layer.append(k, v, tables, lengths, query_starts=starts, query=q)
        times = []
        for _ in range(7):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        took.append(sorted(times)[3])
    assert took[1] < 8 * took[0], took
