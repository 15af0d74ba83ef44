"""PagedCache.attend against softmax attention in 64 bits, on the GPU."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from kvsnap_amd.attention import PagedCache, block_scales, rotary_table
from paged_reference import E4M3, attend64, dequantised, sides

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip_library")]

BF16, FP16 = torch.bfloat16, torch.float16


def made(shape, dtype, seed, loud=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * loud).to(dtype)


def make(layout, blocks, size, kv, width, dtype, seed, loud=1.0):
    """(layer, K and V in 64 bits): a cache of random values, e4m3 ones at scales of 1/16 to 2 with full mantissas."""
    shape = (blocks, size, kv, 2 * width) if layout == "vllm" else (2, blocks, size, kv, width)
    if layout == "vllm-hnd":
        shape = (blocks, kv, size, 2 * width)
    backing = made(shape, torch.float32, seed, loud)
    scales = None
    if dtype == E4M3:
        backing = backing * 4
        scales = block_scales(blocks, 2, kv)[1][1]
        scales.view(torch.uint8).copy_(torch.randint(123, 128, scales.shape,
                                                     generator=torch.Generator().manual_seed(seed + 1)))
    backing = backing.to(dtype)
    view = backing.permute(0, 2, 1, 3) if layout == "vllm" else backing
    exact = dequantised(view, scales)
    on_gpu = backing.cuda()
    cache = on_gpu.permute(0, 2, 1, 3) if layout == "vllm" else on_gpu
    if scales is not None:
        gpu_scales = block_scales(blocks, 2, kv, device="cuda")[1][1]
        gpu_scales.view(torch.uint8).copy_(scales.view(torch.uint8).cuda())
        scales = gpu_scales
    return PagedCache(cache, size, scales=scales), exact


def tables_for(lengths, size, blocks, seed, spare=1):
    rng = random.Random(seed)
    ids = rng.sample(range(blocks), blocks)
    wide = max([-(-n // size) for n in lengths] + [1]) + spare
    tables = torch.full((len(lengths), wide), -3, dtype=torch.int32)
    for s, n in enumerate(lengths):
        for page in range(-(-n // size)):
            tables[s, page] = ids.pop()
    return tables


def check(got, query, exact, tables, lengths, starts=None, *, lse=None, window=None, scale=None, rows=None):
    """Within what the kernels' roundings allow.

    A weight p (at most 1, relative to the largest) is rounded to 16 bits: half a step of it, HALF = 2^-8 for bf16
    and 2^-11 for fp16 (fp16's least steps, 2^-25 absolute, and two bf16 terms, 2^-16, are less), so the output moves
    by at most HALF * sum(p |v|) / sum(p); the output's own rounding is another half step of its value.  Scores'
    fp32 sums of w products and the exponentials' arguments move each weight by a relative e^d - 1 with
    d <= (w + 8) * 2^-24 * scale * |q||k| + 2^-22, well below 2^-12 for the sizes here, and V's fp32 sums add
    n * 2^-24, which 2^-9 * HALF_bf16 covers for the n below 4096 here."""
    keys, values = exact
    want, want_lse = attend64(query, keys, values, tables, lengths, starts, window=window, scale=scale)
    spread, _ = attend64(query, keys, values.abs().nan_to_num(0, 0, 0), tables, lengths, starts, window=window,
                         scale=scale)
    half = 2.0 ** -8 if query.dtype == BF16 else 2.0 ** -11
    bound = (half + 2.0 ** -12) * spread + half * want.abs().nan_to_num(0, 0, 0) * (1 + 2 ** -7) + (
        2.0 ** -24 if query.dtype == FP16 else 0)
    rows = slice(None) if rows is None else rows
    got, want, bound = got.cpu().double()[rows], want[rows], bound[rows]
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    off = torch.where(want.isfinite(), (got - want).abs() - bound, 0.0)
    assert off.max() <= 0, f"off by {off.max():.3g} more than the roundings"
    if lse is not None:
        lse, want_lse = lse.cpu().double()[rows], want_lse[rows]
        empty = want_lse.isinf()
        assert torch.equal(lse[empty], want_lse[empty])
        # d as above, and fp32's half step of the value, twice (the product with the scale, and the sum)
        assert ((lse - want_lse)[~empty].abs() <= 2.0 ** -12 + 2.0 ** -22 * want_lse[~empty].abs()).all()


SINGLE = [
    # lengths, block size, kv heads, group, width, window
    ([1], 16, 1, 1, 16, None),
    ([75], 16, 1, 4, 128, None),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 0], 16, 2, 4, 64, None),
    ([700, 3, 1029, 512, 513], 16, 2, 2, 128, None),
    ([300, 77], 32, 3, 2, 80, 100),
    ([300, 77, 1], 24, 1, 3, 112, 31),
    ([90, 65, 64], 64, 2, 8, 96, 1),
    ([130, 257], 16, 1, 16, 256, None),
    ([130, 257], 1, 1, 5, 32, None),
    ([513], 16, 1, 40, 48, None),                # more query heads than a product's rows
    ([4000], 16, 1, 2, 64, None),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("layout", ["vllm", "vllm-hnd", "kv_split"])
@pytest.mark.parametrize("case", range(len(SINGLE)))
def test_single_rows_are_their_definition(case, layout, held, dtype):
    lengths, size, kv, group, width, window = SINGLE[case]
    blocks = sum(-(-n // size) for n in lengths) + 3
    layer, exact = make(layout, blocks, size, kv, width, E4M3 if held == "e4m3" else dtype, case)
    tables = tables_for(lengths, size, blocks, case)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    query = made((len(lengths), kv * group, width), dtype, 50 + case)
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), window=window, return_lse=True)
    assert out.dtype == dtype
    check(out, query, exact, tables, lengths, lse=lse, window=window)


RAGGED = [
    # added, lengths, block size, kv heads, group, width, window
    ([1, 3], [1, 3], 16, 1, 1, 16, None),
    ([5, 1, 0, 40, 2], [75, 9, 33, 40, 2], 16, 2, 4, 64, None),
    ([65, 64, 63], [65, 100, 200], 16, 2, 2, 128, None),
    ([33, 7], [150, 7], 24, 1, 3, 80, None),
    ([50, 20], [90, 20], 32, 1, 2, 112, 17),
    ([130], [300], 64, 1, 1, 96, 128),
    ([20, 3], [37, 260], 16, 1, 6, 256, None),
    ([6, 2], [4, 2], 16, 1, 2, 32, None),        # two rows ahead of position 0
    ([2, 70, 1], [600, 70, 1000], 16, 1, 40, 64, None),
    ([150], [1300], 16, 1, 1, 64, 500),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("layout", ["vllm", "kv_split"])
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_prompts_and_chunks_are_their_definition(case, layout, held, dtype):
    added, lengths, size, kv, group, width, window = RAGGED[case]
    blocks = sum(-(-n // size) for n in lengths) + 3
    layer, exact = make(layout, blocks, size, kv, width, E4M3 if held == "e4m3" else dtype, case)
    tables = tables_for(lengths, size, blocks, case)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    starts = torch.tensor([sum(added[:s]) for s in range(len(added) + 1)], dtype=torch.int32)
    tokens = sum(added)
    query = made((tokens + 3, kv * group, width), dtype, 70 + case)          # three rows of padding behind
    out = torch.full(query.shape, 7.0, dtype=dtype, device="cuda")
    got, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), window=window,
                            out=out, return_lse=True)
    assert got is out and (out[tokens:] == 7).all()
    check(out, query, exact, tables, lengths, starts, lse=lse, window=window, rows=slice(0, tokens))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
def test_what_a_row_does_not_see_may_hold_anything(held, rows):
    """NaN and infinities in slots past the length, before the window and, for chunks, after a row's own position;
    and blocks that the tables do not name."""
    size, kv, width, blocks = 16, 2, 64, 20
    dtype = E4M3 if held == "e4m3" else BF16
    length, window = 133, 60
    layer, exact = make("kv_split", blocks, size, kv, width, dtype, 1)
    tables = tables_for([length], size, blocks, 1)
    query = made((rows, 4, width), BF16, 2)
    lengths = torch.tensor([length], dtype=torch.int32)
    starts = torch.tensor([0, rows], dtype=torch.int32)
    args = [t.cuda() for t in (query, tables, lengths)]
    clean = layer.attend(*args, query_starts=starts.cuda(), window=window)
    k, v = sides(layer.cache)
    bad = [math.nan, math.nan] if held == "e4m3" else [math.nan, math.inf]
    for block in range(blocks):
        for side, value in zip((k, v), bad):
            filled = side[block].float()
            page = (tables[0] == block).nonzero().flatten().tolist()
            for slot in range(size):
                position = page[0] * size + slot if page else None
                # the first row sees back to length - rows + 1 - window, the last up to length - 1
                if position is None or position >= length or position < length - rows + 1 - window:
                    filled[slot] = value
            side[block] = filled.to(dtype)
    assert torch.equal(layer.attend(*args, query_starts=starts.cuda(), window=window), clean)
    if rows > 1:
        # The last five tokens: seen by the last rows alone.
        for position in range(length - 5, length):
            v[int(tables[0, position // size]), position % size] = torch.full((kv, width), math.nan).to(dtype).cuda()
        got = layer.attend(*args, query_starts=starts.cuda(), window=window)
        assert got[rows - 5:].isnan().all() and not got[:rows - 5].isnan().any()
        assert torch.equal(got[:rows - 5], clean[:rows - 5])


def test_an_infinite_value_reaches_the_rows_that_see_it():
    layer, exact = make("vllm", 4, 16, 1, 32, BF16, 3)
    tables = tables_for([40], 16, 4, 3)
    lengths, starts = torch.tensor([40], dtype=torch.int32), torch.tensor([0, 20], dtype=torch.int32)
    block = int(tables[0, 30 // 16])
    for side, held in zip(sides(layer.cache)[1:], exact[1:]):
        side[block, 30 % 16, 0, 5] = math.inf
        held[block, 30 % 16, 0, 5] = math.inf
    query = made((20, 2, 32), BF16, 4)
    got = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda())
    want, _ = attend64(query, *exact, tables, lengths, starts)
    assert want[10:, :, 5].isinf().all() and torch.equal(got.cpu().isinf(), want.isinf())
    assert not got.isnan().any()


@pytest.mark.parametrize("rows", [1, 30])
def test_pages_that_name_no_block_are_seen_by_nobody(rows):
    for held, size in ((BF16, 16), (E4M3, 16), (BF16, 24)):
        layer, exact = make("vllm", 14, size, 1, 64, held, 5)
        tables = tables_for([100, 90], size, 14, 5, spare=0)
        tables[0, 1], tables[0, 3], tables[1, 0] = -1, 14, 1 << 30
        tables = tables[:, :4]                           # and tables too narrow for their lengths
        lengths = torch.tensor([100, 90], dtype=torch.int32)
        starts = torch.tensor([0, rows, 2 * rows], dtype=torch.int32)
        query = made((2 * rows, 2, 64), BF16, 6)
        out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(),
                                return_lse=True)
        check(out, query, exact, tables, lengths, starts, lse=lse)
        tables[:] = -1
        out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(),
                                return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_wrong_row_starts_stay_inside_the_tensors():
    """Starts that fall, or pass the rows that there are, give rows of no meaning, but no access outside."""
    layer, _ = make("vllm", 12, 16, 1, 64, BF16, 5)
    tables = tables_for([100, 60], 16, 12, 5)
    lengths = torch.tensor([100, 60], dtype=torch.int32)
    query = made((8, 2, 64), BF16, 6).cuda()
    for starts in ([0, 1 << 30, 1 << 30], [5, 3, 1], [-9, -5, 4], [0, 0, 0], [1 << 30, 0, 8]):
        layer.attend(query, tables.cuda(), lengths.cuda(), query_starts=torch.tensor(starts, dtype=torch.int32).cuda())
        layer.append(query[:, :1], query[:, :1], tables.cuda(), lengths.cuda(),
                     query_starts=torch.tensor(starts, dtype=torch.int32).cuda())
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [1, 50])
def test_scores_of_every_size(rows):
    """Scores far apart (one token takes all), all alike, and far from zero."""
    layer, exact = make("vllm", 12, 16, 1, 64, BF16, 7)
    tables = tables_for([150], 16, 12, 7)
    lengths, starts = torch.tensor([150], dtype=torch.int32), torch.tensor([0, rows], dtype=torch.int32)
    for loud in (0.0, 1e-3, 8.0, 64.0):
        # |score| <= 64 * loud * |q||k| / 8; fp32 moves it by about 2^-20 of that, which the check's 2^-12 covers to
        # loud = 8; at 64 one token's weight is all but 1.
        query = made((rows, 4, 64), BF16, 8, loud)
        out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(),
                                return_lse=True)
        check(out, query, exact, tables, lengths, starts, lse=lse if loud <= 8 else None)
    query = made((rows, 4, 64), BF16, 8)
    out = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), softmax_scale=0.02)
    check(out, query, exact, tables, lengths, starts, scale=0.02)


def test_e8m0_bytes_at_their_ends():
    """2^-127, 2^-126, and the byte that is NaN."""
    layer, _ = make("kv_split", 3, 16, 1, 64, E4M3, 9)
    held = layer.scales.view(torch.uint8)
    held[:, :, 0] = 127
    tables = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([48], dtype=torch.int32, device="cuda")
    query = made((1, 1, 64), BF16, 1, 0.0)                    # weights all alike
    mean = sides(layer.cache)[1].float().double().mean((0, 1, 2)).cpu()
    for byte in (0, 1, 240):
        held[:, :, 1] = byte
        got = layer.attend(query.cuda(), tables, lengths)[0, 0].cpu().double()
        # the mean of 48 exact values, fp32 sums, one rounding; near the type's end what is under 2^-133 may vanish
        assert ((got - mean * 2.0 ** (byte - 127)).abs() <= (2.0 ** -8 + 2.0 ** -12) * mean.abs() * 2.0 ** (byte - 127)
                + 2.0 ** -126).all()
    held[1, :, 1] = 255
    assert layer.attend(query.cuda(), tables, lengths).isnan().all()
    held[:, :, 1] = 127
    held[1, :, 0] = 255
    assert layer.attend(query.cuda(), tables, lengths).isnan().all()


def test_the_length_hint_changes_no_token():
    layer, exact = make("vllm", 80, 16, 1, 64, BF16, 10)
    tables = tables_for([1200, 7], 16, 80, 10)
    lengths = torch.tensor([1200, 7], dtype=torch.int32)
    for rows in (1, 33):
        starts = torch.tensor([0, rows, rows + 1], dtype=torch.int32)
        query = made((rows + 1, 2, 64), BF16, 11)
        for hint in (0, 1, 500, 1200, 1 << 40, None):
            out = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(),
                               max_length=hint)
            check(out, query, exact, tables, lengths, starts)


def test_strided_queries_and_outputs():
    layer, exact = make("kv_split", 8, 16, 2, 64, FP16, 12)
    tables = tables_for([60, 33], 16, 8, 12)
    lengths = torch.tensor([60, 33], dtype=torch.int32)
    fused = made((2, 9, 64), FP16, 13).cuda()
    wide = torch.zeros((2, 6, 128), dtype=FP16, device="cuda")
    out = layer.attend(fused[:, 3:7], tables.cuda(), lengths.cuda(), out=wide[:, 1:5, :64])
    check(out, fused[:, 3:7].cpu(), exact, tables, lengths)
    assert (wide[:, 0] == 0).all() and (wide[:, 5] == 0).all() and (wide[..., 64:] == 0).all()


def test_offsets_past_32_bits():
    """A cache of 5 GiB for K and V each: its last blocks."""
    size, kv, width = 16, 8, 128
    blocks = 5 * (1 << 30) // (size * kv * width * 2) + 3
    cache = torch.empty((2, blocks, size, kv, width), dtype=BF16, device="cuda")
    some = made((2, 3, size, kv, width), BF16, 14)
    cache[:, -3:] = some.cuda()
    layer = PagedCache(cache, size)
    key, value = made((1, kv, width), BF16, 16), made((1, kv, width), BF16, 17)
    lengths = torch.tensor([45], dtype=torch.int32)
    tables = torch.tensor([[blocks - 2, blocks - 1, blocks - 3]], dtype=torch.int32)
    layer.append(key.cuda(), value.cuda(), tables.cuda(), lengths.cuda())
    some[0, 0, 44 - 32], some[1, 0, 44 - 32] = key[0], value[0]
    assert torch.equal(cache[:, -3:].cpu(), some)
    for rows in (1, 20):
        query = made((rows, 8, width), BF16, 15)
        starts = torch.tensor([0, rows], dtype=torch.int32)
        out = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda())
        check(out, query, [side.double() for side in some], tables - (blocks - 3), lengths, starts)


@pytest.mark.parametrize("rows", [1, 24])
def test_captured_attention_follows_its_tables(rows):
    """A graph replayed over changed lengths, tables and values, beside another that shares nothing with it."""
    layer, exact = make("vllm", 200, 16, 1, 64, BF16, 18)
    tables = tables_for([1500, 1400], 16, 200, 18).cuda()
    lengths = torch.tensor([1500, 900], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, rows, rows + 1], dtype=torch.int32, device="cuda")
    query = made((rows + 1, 4, 64), BF16, 19).cuda()
    other = query.clone()
    layer.attend(query, tables, lengths, query_starts=starts)
    graphs, outs = [], []
    for q in (query, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer.attend(q, tables, lengths, query_starts=starts))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        query.copy_(made(query.shape, BF16, 20 + step))
        other.copy_(made(query.shape, BF16, 40 + step))
        lengths.copy_(torch.tensor([1500 - 300 * step, 900 + step], dtype=torch.int32))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for q, out in zip((query, other), outs):
            eager = layer.attend(q, tables, lengths, query_starts=starts)
            assert torch.equal(out, eager)


def test_the_same_call_gives_the_same_bits():
    layer, _ = make("kv_split", 300, 16, 2, 128, E4M3, 21)
    tables = tables_for([4000, 333], 16, 300, 21).cuda()
    lengths = torch.tensor([4000, 333], dtype=torch.int32, device="cuda")
    for rows in (1, 64):
        starts = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
        query = made((2 * rows, 8, 128), BF16, 22).cuda()
        first = layer.attend(query, tables, lengths, query_starts=starts)
        for _ in range(5):
            assert torch.equal(layer.attend(query, tables, lengths, query_starts=starts), first)


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("count", [70, 130, 300])
def test_many_sequences_of_every_length(count, held):
    """More sequences than a wave looks at at a time (64), and than are cut evenly (256); a few long ones."""
    rng = random.Random(count)
    lengths = [rng.choice([0, 1, 15, 16, 40, 100]) for _ in range(count)]
    for s, n in ((0, 2000), (count // 2, 1700), (count - 1, 2600)):
        lengths[s] = n
    blocks = sum(-(-n // 16) for n in lengths) + 1
    layer, exact = make("kv_split", blocks, 16, 2, 32, E4M3 if held == "e4m3" else BF16, count)
    tables = tables_for(lengths, 16, blocks, count)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    query = made((count, 2, 32), BF16, 3)
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), return_lse=True)
    check(out, query, exact, tables, lengths, lse=lse)
    # ragged: every fifth sequence has no row, every seventh three
    added = [0 if s % 5 == 1 else 3 if s % 7 == 0 else 1 for s in range(count)]
    starts = torch.tensor([sum(added[:s]) for s in range(count + 1)], dtype=torch.int32)
    query = made((sum(added), 2, 32), BF16, 4)
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), return_lse=True)
    check(out, query, exact, tables, lengths, starts, lse=lse)


@pytest.mark.parametrize("rows", [1, 40])
def test_a_scale_near_the_least_float_weighs_all_tokens_alike(rows):
    layer, exact = make("vllm", 10, 16, 2, 64, BF16, 3)
    lengths = torch.tensor([150], dtype=torch.int32)
    tables = tables_for([150], 16, 10, 3)
    starts = torch.tensor([0, rows], dtype=torch.int32)
    query = made((rows, 4, 64), BF16, 4)
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), return_lse=True,
                            softmax_scale=1.2e-38)
    check(out, query, exact, tables, lengths, starts, lse=lse, scale=1.2e-38)


@pytest.mark.parametrize("rows", [1, 40])
def test_a_length_that_no_table_names_sees_what_its_window_names(rows):
    """Lengths up to int32's largest, far past the tables: with a window nobody sees a token, without one a row sees
    all that is named, and every launch ends."""
    layer, exact = make("vllm", 10, 16, 2, 64, BF16, 5)
    named = tables_for([150], 16, 10, 5, spare=0)
    starts = torch.tensor([0, rows], dtype=torch.int32).cuda()
    query = made((rows, 4, 64), BF16, 6)
    for length in (2 ** 30, 2 ** 31 - 1):
        lengths = torch.tensor([length], dtype=torch.int32).cuda()
        out, lse = layer.attend(query.cuda(), named.cuda(), lengths, query_starts=starts, window=100, return_lse=True)
        assert not out.any() and lse.isneginf().all()
        out = layer.attend(query.cuda(), named.cuda(), lengths, query_starts=starts)
        # as the last rows of a sequence of all 160 named tokens and 1000 more, which no table names
        check(out, query, exact, named, torch.tensor([1160], dtype=torch.int32), starts.cpu())


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("count,window", [(3, None), (90, None), (300, None), (90, 700)])
def test_chunks_over_long_contexts_are_cut_by_their_lengths(count, window, held):
    """Tiles of rows in parts of equal length: few sequences and many (300, where a wave goes over five times 64), some
    of one row or none, contexts from none to 2800 tokens."""
    rng = random.Random(count)
    added = [rng.choice([0, 1, 1, 2, 3]) for _ in range(count)]
    lengths = [max(n, rng.choice([5, 40, 90])) for n in added]
    for s, n, length in ((0, 70, 2800), (count // 2, 2, 1500), (count - 1, 40, 900)):
        added[s], lengths[s] = n, length
    blocks = sum(-(-n // 16) for n in lengths) + 1
    layer, exact = make("vllm", blocks, 16, 1, 64, E4M3 if held == "e4m3" else FP16, count)
    tables = tables_for(lengths, 16, blocks, count)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    starts = torch.tensor([sum(added[:s]) for s in range(count + 1)], dtype=torch.int32)
    query = made((sum(added), 3, 64), FP16, 7)
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), window=window,
                            return_lse=True)
    check(out, query, exact, tables, lengths, starts, lse=lse, window=window)


def test_wrong_row_starts_over_long_contexts_stay_inside_the_tensors():
    """As above, where tiles are cut: a sequence that no workgroup takes is not joined."""
    layer, _ = make("vllm", 200, 16, 1, 64, BF16, 5)
    tables = tables_for([1500, 900, 700], 16, 200, 5)
    lengths = torch.tensor([1500, 900, 700], dtype=torch.int32)
    query = made((300, 2, 64), BF16, 6).cuda()
    for starts in ([0, 300, 0, 300], [0, 1 << 30, 0, 1 << 30], [299, 0, 300, 1], [-9, 200, 100, 300]):
        layer.attend(query, tables.cuda(), lengths.cuda(), query_starts=torch.tensor(starts, dtype=torch.int32).cuda())
    torch.cuda.synchronize()


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
def test_few_rows_of_many_sequences_are_cut_by_their_lengths(held):
    """Two to five rows of each of 80 sequences, 8 key heads: more tiles than the chip holds workgroups, none full."""
    rng = random.Random(1)
    added = [rng.randrange(2, 6) for _ in range(80)]
    lengths = [rng.choice([5, 30, 70, 200]) for _ in added]
    lengths[3], lengths[40] = 2000, 1300
    blocks = sum(-(-n // 16) for n in lengths) + 1
    layer, exact = make("kv_split", blocks, 16, 8, 32, E4M3 if held == "e4m3" else BF16, 2)
    tables = tables_for(lengths, 16, blocks, 2)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    starts = torch.tensor([sum(added[:s]) for s in range(81)], dtype=torch.int32)
    query = made((sum(added), 8, 32), BF16, 7)
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), return_lse=True)
    check(out, query, exact, tables, lengths, starts, lse=lse)


@pytest.mark.parametrize("length", [40, 1000])
@pytest.mark.parametrize("added", [0, 1, 3])
def test_one_sequence_of_few_rows_among_padding(added, length):
    """A step of four rows for one sequence that adds fewer, one among them: the rest are padding, and stay."""
    layer, exact = make("vllm", 70, 16, 2, 64, BF16, 8)
    tables = tables_for([length], 16, 70, 8)
    lengths = torch.tensor([length], dtype=torch.int32)
    starts = torch.tensor([0, added], dtype=torch.int32)
    query = made((4, 4, 64), BF16, 9)
    out = torch.full((4, 4, 64), 7.0, dtype=BF16, device="cuda")
    _, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), out=out,
                          return_lse=True)
    assert (out[added:] == 7).all()
    if added:
        check(out, query, exact, tables, lengths, starts, lse=lse, rows=slice(0, added))


@pytest.mark.parametrize("captured", [False, True])
def test_calls_at_once_on_two_streams_do_not_meet(captured):
    """Split rows and cut tiles on two streams at a time, eager or as two captured graphs: each call has a workspace of
    its own."""
    layer, exact = make("kv_split", 300, 16, 2, 64, BF16, 11)
    steps = []
    for seed, added, lengths in ((1, [1, 40, 1], [3000, 900, 17]), (2, [70, 1], [1400, 2500])):
        tables = tables_for(lengths, 16, 300, seed)
        lengths = torch.tensor(lengths, dtype=torch.int32)
        starts = torch.tensor([sum(added[:s]) for s in range(len(added) + 1)], dtype=torch.int32)
        query = made((sum(added), 8, 64), BF16, seed)
        steps.append((query, tables, lengths, starts))
    on_gpu = [[t.cuda() for t in step] for step in steps]
    call = lambda q, tables, lengths, starts: layer.attend(q, tables, lengths, query_starts=starts)
    alone = [call(*step) for step in on_gpu]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    if captured:
        graphs, outs = [torch.cuda.CUDAGraph() for _ in steps], []
        for graph, step in zip(graphs, on_gpu):
            with torch.cuda.graph(graph):
                outs.append(call(*step))
    for _ in range(5):
        if captured:
            for out in outs:
                out.zero_()
            torch.cuda.synchronize()
        else:
            outs = [None, None]
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                if captured:
                    graphs[i].replay()
                else:
                    outs[i] = call(*on_gpu[i])
        torch.cuda.synchronize()
        for out, want in zip(outs, alone):
            assert torch.equal(out, want)
    for out, (query, tables, lengths, starts) in zip(outs, steps):
        check(out, query, exact, tables, lengths, starts)
