"""PagedCache at the ends of what its callers may ask: far blocks, far scores, small weights, odd ways of cutting."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from kvsnap_amd.attention import PagedCache, rotary_table, rotate
from paged_reference import E4M3, attend64, dequantised
from test_gpu_attend import check, made, make, tables_for

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip_library")]

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("held,size", [("16-bit", 16), ("e4m3", 64), ("16-bit", 24)])
def test_blocks_past_32_gib(held, size):
    """A cache whose last blocks lie 32 GiB from its first: appends to them and attention over them, rows alone and
    chunks long enough that whole stages of 64 tokens are seen by every row."""
    width, dtype = 64, E4M3 if held == "e4m3" else BF16
    block_bytes = size * 2 * width * dtype.itemsize
    near, last = 2 ** 35 // block_bytes, 20
    blocks = near + 1 + last                        # all of the last 20 start at or past 32 GiB
    cache = torch.empty((blocks, 1, size, 2 * width), dtype=dtype, device="cuda")
    assert (blocks - last) * block_bytes >= 2 ** 35
    some = made((last, 1, size, 2 * width), torch.float32, 1).to(dtype)
    cache[-last:].view(torch.uint8).copy_(some.view(torch.uint8))
    scales = some_scales = None
    if held == "e4m3":
        scales = torch.full((blocks, 1, 2), 127, dtype=torch.uint8, device="cuda")
        some_scales = torch.randint(124, 129, (last, 1, 2), generator=torch.Generator().manual_seed(2)).to(torch.uint8)
        scales[-last:] = some_scales.cuda()
    layer = PagedCache(cache, size, scales=scales)
    exact = dequantised(some, some_scales)
    length = last * size - 5
    ids = random.Random(3).sample(range(last), last)
    tables, lengths = torch.tensor([ids], dtype=torch.int32), torch.tensor([length], dtype=torch.int32)
    far = (tables + (blocks - last)).cuda()
    for rows in (1, 70):
        query = made((rows, 2, width), BF16, 4)
        starts = torch.tensor([0, rows], dtype=torch.int32)
        out = layer.attend(query.cuda(), far, lengths.cuda(), query_starts=starts.cuda())
        check(out, query, exact, tables, lengths, starts)
    if held == "16-bit":
        key, value = made((1, 1, width), BF16, 5), made((1, 1, width), BF16, 6)
        layer.append(key.cuda(), value.cuda(), far, lengths.cuda())
        some[ids[-1], 0, (length - 1) % size] = torch.cat([key[0, 0], value[0, 0]])
        assert torch.equal(cache[-last:].cpu(), some)


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("dtype,power", [(FP16, 15), (BF16, 15), (BF16, 45)])
def test_scores_far_beyond_the_exponentials_range(dtype, power, held, rows):
    """Queries and keys of 2^power: scores of 2^33 and more, all alike but for every third token's, which are less by
    far more than any exponent.  Every product and sum is exact, so weights are 0 or alike, and the check's bound
    holds as it is."""
    size, kv, width, length = 16, 1, 64, 1500
    blocks = -(-length // size)
    shape = (2, blocks, size, kv, width)
    cache, scales = made(shape, torch.float32, 1), None
    cache[0] = 1.0
    cache[0, :, ::3] = 0.875
    if held == "e4m3":
        cache, scales = cache.to(E4M3), torch.full((blocks, kv, 2), 127, dtype=torch.uint8)
        scales[..., 0] += power
    else:
        cache[0] *= 2.0 ** power
        cache = cache.to(dtype)
    exact = dequantised(cache, scales)
    layer = PagedCache(cache.cuda(), size, scales=None if scales is None else scales.cuda())
    tables, lengths = torch.randperm(blocks, dtype=torch.int32)[None], torch.tensor([length], dtype=torch.int32)
    starts = torch.tensor([0, rows], dtype=torch.int32)
    query = torch.full((rows, 2, width), 2.0 ** power, dtype=dtype)
    query[:, 1] = -query[:, 1]
    out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda(), return_lse=True)
    check(out, query, exact, tables, lengths, starts, lse=lse)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("sink", ["first", "middle", "last seen by all"])
def test_small_weights_behind_one_that_takes_all_in_fp16(sink, rows):
    """One token's weight is 2^14 to 2^30 times any other's and its value 0, so the output is the others' alone.

    The check's roundings, and fp16's least steps: a weight beside the large one, in the same 64 tokens, is rounded by
    up to 2^-25 of 2^-5 of that one, and 64 of those, over a sum that is at least the large one, move the output by at
    most 2^-24 of the largest value."""
    size, kv, width, length = 16, 1, 64, 3000
    blocks = -(-length // size)
    at = {"first": 0, "middle": 1333, "last seen by all": length - rows}[sink]
    tables = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None]
    cache = torch.zeros((2, blocks, size, kv, width))
    cache[1] = 0.5 + torch.rand(cache[1].shape, generator=torch.Generator().manual_seed(2))
    block, slot = int(tables[0, at // size]), at % size
    cache[0, block, slot], cache[1, block, slot] = 1.0, 0.0
    cache = cache.to(FP16)
    keys, values = (side.double() for side in cache)
    times = torch.tensor([14.5, 22.0, 25.2, 30.0])           # in binary logarithms: 64 q / 8 = times * ln 2
    query = (times * math.log(2) / 8)[None, :, None].expand(rows, 4, width).to(FP16).contiguous()
    lengths, starts = torch.tensor([length], dtype=torch.int32), torch.tensor([0, rows], dtype=torch.int32)
    got, lse = PagedCache(cache.cuda(), size).attend(query.cuda(), tables.cuda(), lengths.cuda(),
                                                     query_starts=starts.cuda(), return_lse=True)
    want, want_lse = attend64(query, keys, values, tables, lengths, starts)      # values are not negative: the spread too
    bound = (2.0 ** -10 + 2.0 ** -11) * want + 2.0 ** -24 + 2.0 ** -24 * 1.5
    off = (got.cpu().double() - want).abs() - bound
    assert off.max() <= 0, (off.amax((0, 2)) / want.amin((0, 2))).tolist()
    assert ((lse.cpu().double() - want_lse).abs() <= 2.0 ** -12 + 2.0 ** -22 * want_lse.abs()).all()


@pytest.mark.parametrize("added,lengths", [([1, 1, 1], [40, 0, 300]), ([1, 1, 1], [3000, 17, 900]), ([300], [300]),
                                           ([3, 1, 40, 1], [2800, 1500, 90, 7])])
def test_queries_that_become_their_own_output(added, lengths):
    """Whole and cut, rows alone and in tiles: ``out`` is ``query``, heads of a projection."""
    blocks = sum(-(-n // 16) for n in lengths) + 2
    layer, _ = make("kv_split", blocks, 16, 2, 64, BF16, 3)
    tables = tables_for(lengths, 16, blocks, 3).cuda()
    lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
    starts = torch.tensor([sum(added[:s]) for s in range(len(added) + 1)], dtype=torch.int32).cuda()
    fused = made((sum(added), 12, 64), BF16, 4).cuda()
    query = fused[:, 2:10]
    starts = None if max(added) == 1 else starts
    want = layer.attend(query, tables, lengths, query_starts=starts)
    before = fused.clone()
    assert layer.attend(query, tables, lengths, query_starts=starts, out=query) is query
    assert torch.equal(query, want)
    assert torch.equal(fused[:, :2], before[:, :2]) and torch.equal(fused[:, 10:], before[:, 10:])


def test_a_graph_that_saved_what_a_call_writes_does_not_use_it():
    """Backward through a tensor that was written since raises, as after torch's own in-place operators; inference
    tensors, which have no version, are written all the same."""
    layer, _ = make("kv_split", 4, 16, 2, 64, BF16, 1)
    tables = torch.tensor([[1, 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([20], dtype=torch.int32, device="cuda")
    angles = rotary_table(64, 30, device="cuda")
    at = torch.tensor([3], device="cuda")
    query, key = made((1, 4, 64), BF16, 2).cuda(), made((1, 2, 64), BF16, 3).cuda()
    calls = [(lambda out: rotate(query, at, angles, out=out), torch.empty_like(query)),
             (lambda out: layer.append(key, key, tables, lengths, query=query, query_out=out), torch.empty_like(query)),
             (lambda out: layer.attend(query, tables, lengths, out=out), torch.empty_like(query)),
             (lambda out: layer.append(key, key, tables, lengths), layer.cache)]
    for call, out in calls:
        weight = torch.ones((), dtype=BF16, device="cuda", requires_grad=True)
        product = (weight * out).sum()
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
        if out is not layer.cache:
            want = out.clone()
            with torch.inference_mode():
                again = torch.zeros_like(out)
                call(again)
            assert torch.equal(again, want)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("size", [16, 24])
@pytest.mark.parametrize("byte", [0, 1, 240])
def test_e8m0_bytes_at_their_ends_in_rows_and_tiles(byte, size, rows):
    """V's scales at 2^-127, 2^-126 and 2^113, weights all alike: the mean of what a row sees, one rounding of the
    weights and one of the output, and what is under bf16's least normal number may vanish."""
    layer, _ = make("kv_split", 12, size, 1, 64, E4M3, 9)
    held = layer.scales.view(torch.uint8)
    held[..., 0], held[..., 1] = 127, byte
    exact = dequantised(layer.cache.cpu(), layer.scales.cpu())
    length = 12 * size - 5
    tables, lengths = tables_for([length], size, 12, 4, spare=0), torch.tensor([length], dtype=torch.int32)
    starts = torch.tensor([0, rows], dtype=torch.int32)
    query = torch.zeros((rows, 2, 64), dtype=BF16)
    got = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda()).cpu().double()
    want, _ = attend64(query, *exact, tables, lengths, starts)
    spread, _ = attend64(query, exact[0], exact[1].abs(), tables, lengths, starts)
    assert ((got - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * spread + 2.0 ** -8 * want.abs() + 2.0 ** -126).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("size", [16, 24])
def test_a_scale_that_is_nan_reaches_the_rows_that_see_its_block(size, side, dtype):
    """The byte 255, of K or of V, in the last block, which the last 11 of 60 rows see, and in a block in the middle
    that only a window's first rows do."""
    layer, _ = make("kv_split", 14, size, 2, 64, E4M3, 9)
    length, rows = 12 * size + 11, 60
    tables = tables_for([length], size, 14, 4).cuda()
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    query = made((rows, 4, 64), dtype, 5).cuda()
    held = layer.scales.view(torch.uint8)
    clean = layer.attend(query, tables, lengths, query_starts=starts)
    block = int(tables[0, 12])
    before = held[block, 0, side].clone()
    held[block, 0, side] = 255                                  # head 0's; head 1's is as it was
    got = layer.attend(query, tables, lengths, query_starts=starts)
    assert got[rows - 11:, :2].isnan().all()
    assert torch.equal(got[:rows - 11], clean[:rows - 11]) and torch.equal(got[:, 2:], clean[:, 2:])
    assert layer.attend(query[-1:], tables, lengths)[:, :2].isnan().all()
    held[block, 0, side] = before
    # a window of 50: the first row sees from length - 60 - 49 on, and the block of that token to its end
    window, first = 50, length - rows + 1 - 50
    clean = layer.attend(query, tables, lengths, query_starts=starts, window=window)
    page = first // size
    held[int(tables[0, page]), 1, side] = 255
    got = layer.attend(query, tables, lengths, query_starts=starts, window=window)
    seen = (page + 1) * size - first                            # rows that see its last token
    assert got[:seen, 2:].isnan().all()
    assert torch.equal(got[seen:], clean[seen:]) and torch.equal(got[:, :2], clean[:, :2])


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("size", [16, 24, 1])
@pytest.mark.parametrize("width", [80, 96, 112, 128, 192, 256])
def test_cut_rows_and_tiles_of_every_width(width, size, held):
    """Parts joined where a head's quarter does not divide a workgroup, at the widest, and over blocks that are no whole
    groups of 16 tokens: single rows and chunks over long contexts, in one step and each alone, with a window too."""
    lengths = [2900, 33, 1500, 700]
    blocks = sum(-(-n // size) for n in lengths) + 1
    layer, exact = make("kv_split", blocks, size, 2, width, E4M3 if held == "e4m3" else FP16, width)
    tables, dtype = tables_for(lengths, size, blocks, width), FP16
    lengths = torch.tensor(lengths, dtype=torch.int32)
    for added, window in (([1, 1, 1, 1], None), ([1, 3, 30, 1], None), ([2, 1, 5, 40], 1400)):
        starts = torch.tensor([sum(added[:s]) for s in range(5)], dtype=torch.int32)
        if max(added) == 1:
            starts = None
        query = made((sum(added), 6, width), dtype, 7)
        out, lse = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), window=window, return_lse=True,
                                query_starts=None if starts is None else starts.cuda())
        check(out, query, exact, tables, lengths, starts, lse=lse, window=window)


@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
@pytest.mark.parametrize("width", [16, 32, 48, 80, 112, 176, 208, 240])
def test_tiles_read_no_further_than_a_heads_width(width, held):
    """Whole stages of 64 tokens that every row sees, at widths that are less than the kernels' own: what lies behind a
    head's row (another head's of NaN, and behind the cache's last row a tail of NaN) does not reach the head."""
    size, kv, blocks, length, rows = 16, 2, 20, 320, 40
    dtype = E4M3 if held == "e4m3" else BF16
    shape = (2, blocks, size, kv, width)
    some = made(shape, torch.float32, width).to(dtype)
    backing = torch.full((some.numel() + 512,), math.nan).to(dtype)
    cache = backing[:some.numel()].view(shape)
    cache[:, :, :, 0] = some[:, :, :, 0]
    on_gpu = backing.cuda()[:some.numel()].view(shape)
    scales = torch.full((blocks, kv, 2), 127, dtype=torch.uint8) if held == "e4m3" else None
    layer = PagedCache(on_gpu, size, scales=None if scales is None else scales.cuda())
    tables = tables_for([length], size, blocks, width, spare=0)
    lengths, starts = torch.tensor([length], dtype=torch.int32), torch.tensor([0, rows], dtype=torch.int32)
    query = made((rows, 4, width), BF16, 5)
    out = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda())
    assert out[:, 2:].isnan().all()
    check(out[:, :2], query[:, :2], [side[:, :, :1] for side in dequantised(cache, scales)], tables, lengths, starts)
    # the other head is the last of its rows
    cache[:, :, :, 0], cache[:, :, :, 1] = math.nan, some[:, :, :, 1]
    on_gpu.view(torch.uint8).copy_(cache.view(torch.uint8))
    out = layer.attend(query.cuda(), tables.cuda(), lengths.cuda(), query_starts=starts.cuda())
    check(out[:, 2:], query[:, 2:], [side[:, :, 1:] for side in dequantised(cache, scales)], tables, lengths, starts)
