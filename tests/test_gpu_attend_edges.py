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
