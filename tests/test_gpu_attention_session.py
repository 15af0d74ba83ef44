"""The operators together, as a serving step uses them, over caches that a plane saves and restores.

A session's prompt is appended and attended, its blocks are saved, restored into other blocks and read there: the
attention over them has to give the same bits, and the session goes on in them, token by token, as the one that was
never moved does.  e4m3 blocks take their scales with them.
"""
import random

import pytest

torch = pytest.importorskip("torch")

from kvsnap_amd import synth
from kvsnap_amd.attention import PagedCache, block_scales, rotary_table
from kvsnap_amd.dataplane import TorchBlockDataPlane
from kvsnap_amd.host_tier import HostTier
from paged_reference import attend64, rotate64, table64

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("copy_routes")]

LAYERS, BLOCKS, SIZE, KV, HEADS, WIDTH = 3, 40, 16, 2, 4, 64


def make(layout, held):
    dtype = torch.float8_e4m3fn if held == "e4m3" else torch.bfloat16
    caches, _ = synth.make_caches(LAYERS, BLOCKS, block_size=SIZE, heads=KV, head_dim=WIDTH, dtype=dtype, layout=layout)
    rows, views = block_scales(BLOCKS, LAYERS, KV, device="cuda") if held == "e4m3" else (None, [None] * LAYERS)
    for cache in caches.values():
        cache.view(torch.uint8).random_(0, 256) if held == "e4m3" else cache.normal_()
    if rows is not None:
        rows.view(torch.uint8).random_(100, 140)
    return caches, rows, views


def table_of(ids, tokens):
    return torch.tensor([ids[:-(-tokens // SIZE)]], dtype=torch.int32, device="cuda")


class Session:
    """One session's steps through every layer: queries, keys and values from a seed."""

    def __init__(self, layers, ids):
        self.layers, self.ids, self.length = layers, ids, 0
        self.angles = rotary_table(WIDTH, 1000, device="cuda")

    def step(self, tokens, seed):
        gen = torch.Generator().manual_seed(seed)
        self.length += tokens
        tables = table_of(self.ids, self.length)
        lengths = torch.tensor([self.length], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
        outs = []
        for layer in self.layers:
            fused = (torch.randn((tokens, HEADS + 2 * KV, WIDTH), generator=gen) * 2).to(torch.bfloat16).cuda()
            q, k, v = fused.split([HEADS, KV, KV], 1)
            q = layer.append(k, v, tables, lengths, query_starts=starts, query=q, rotary=self.angles)
            outs.append(layer.attend(q, tables, lengths, query_starts=starts))
        return outs


@pytest.mark.parametrize("save_mode,restore_mode", [("staged", "dma"), ("direct", "kernel")])
@pytest.mark.parametrize("layout", ["vllm", "kv_split"])
@pytest.mark.parametrize("held", ["16-bit", "e4m3"])
def test_a_session_goes_on_where_its_blocks_are_restored(held, layout, save_mode, restore_mode, hip_library):
    caches, rows, views = make(layout, held)
    plane = TorchBlockDataPlane(caches, SIZE, 16 << 20, save_mode=save_mode, restore_mode=restore_mode, scales=rows)
    try:
        plane.warm_up()
        assert plane.block_bytes == LAYERS * 2 * SIZE * KV * WIDTH * (1 if held == "e4m3" else 2) + (
            16 if held == "e4m3" else 0)
        layers = [plane.paged_cache(name, scales=view) for name, view in zip(plane.caches, views)]
        ids = random.Random(1).sample(range(1, BLOCKS), 24)
        here, there = Session(layers, ids[:12]), Session(layers, ids[12:])
        here.step(93, 5)                        # five whole blocks and 13 slots of the sixth
        here.step(1, 6)
        used = -(-here.length // SIZE)
        with plane.staging(used) as staged:
            targets = [(staged, i * plane.block_bytes) for i in range(used)]
            plane.save_gather(here.ids[:used], targets, here.length)
            torch.cuda.synchronize()
            plane.load_scatter(there.ids[:used], targets)
        there.length = here.length
        torch.cuda.synchronize()
        # a question over what is there, then token by token, a chunk, and a token into a fresh block
        for tokens, seed in ((1, 7), (1, 8), (1, 9), (30, 10), (1, 11)):
            for moved, stayed in zip(there.step(tokens, seed), here.step(tokens, seed)):
                assert torch.equal(moved, stayed)
    finally:
        torch.cuda.synchronize()
        plane.close()


def test_the_host_tier_keeps_a_blocks_scales_with_it(hip_library):
    """A delta save and a verified restore of an e4m3 session."""
    caches, rows, views = make("kv_split", "e4m3")
    plane = TorchBlockDataPlane(caches, SIZE, 16 << 20, scales=rows)
    try:
        plane.warm_up()
        tier = HostTier(plane, 8 << 20)
        layers = [plane.paged_cache(name, scales=view) for name, view in zip(plane.caches, views)]
        ids = random.Random(2).sample(range(1, BLOCKS), 20)
        here, there = Session(layers, ids[:10]), Session(layers, ids[10:])
        here.step(40, 1)
        snapshot = tier.save(here.ids[:3], here.length)
        here.step(20, 2)
        snapshot = tier.save(here.ids[:4], here.length, previous=snapshot)
        tier.restore(there.ids[:4], snapshot, verify=True)
        torch.cuda.synchronize()
        there.length = here.length
        for moved, stayed in zip(there.step(1, 3), here.step(1, 3)):
            assert torch.equal(moved, stayed)
    finally:
        torch.cuda.synchronize()
        plane.close()


def test_a_decode_step_of_many_sessions_is_its_definition_in_a_graph(hip_library):
    """append and attend of three sessions captured once and replayed token after token, against 64-bit attention over
    exactly what was appended (a 16-bit cache)."""
    caches, _, _ = make("vllm", "16-bit")
    layer = PagedCache(next(iter(caches.values())), SIZE)
    angles = rotary_table(WIDTH, 200, device="cuda")
    exact_angles = table64(WIDTH, 200)
    ids = random.Random(3).sample(range(1, BLOCKS), 12)
    tables = torch.tensor([ids[0:4], ids[4:8], ids[8:12]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([0, 15, 31], dtype=torch.int32, device="cuda")
    fused = torch.zeros((3, HEADS + 2 * KV, WIDTH), dtype=torch.bfloat16, device="cuda")
    q, k, v = fused.split([HEADS, KV, KV], 1)

    def step():
        turned = layer.append(k, v, tables, lengths, query=q, rotary=angles)
        return turned, layer.attend(turned, tables, lengths)

    keys = [layer.cache[..., :WIDTH], layer.cache[..., WIDTH:]]
    lengths += 1
    step()
    lengths -= 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = step()
    for token in range(20):
        fused.copy_(torch.randn(fused.shape, generator=torch.Generator().manual_seed(token)).to(torch.bfloat16))
        lengths += 1
        graph.replay()
        torch.cuda.synchronize()
        exact = rotate64(q.cpu(), lengths.cpu() - 1, exact_angles)
        assert ((turned.cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -20).all()
        held = [side.permute(0, 2, 1, 3).cpu().double() for side in keys]
        want, _ = attend64(turned.cpu(), *held, tables.cpu(), lengths.cpu())
        spread, _ = attend64(turned.cpu(), held[0], held[1].abs(), tables.cpu(), lengths.cpu())
        # weights and the output in bf16: half a step each, and fp32's errors below 2^-12
        assert ((out.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * spread + 1.01 * 2.0 ** -8 * want.abs()).all()
