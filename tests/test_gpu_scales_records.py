"""Records that end with their blocks' scales, on every route that saves and restores them: rows of any whole 8-byte
words, apart by more than their length; hashed, verified, from disk."""
import ctypes as C
import hashlib
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from kvsnap_amd import synth
from kvsnap_amd.blobs import BlobDirectory, CorruptSnapshotError
from kvsnap_amd.dataplane import TorchBlockDataPlane

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("copy_routes")]

BLOCKS, SIZE, N = 90, 16, 40


def contents(caches, rows, ids):
    """What the blocks ``ids`` hold, as bytes on the host, scales last."""
    held = []
    for cache in caches.values():
        axis = 1 if cache.ndim == 5 else 0
        held.append(cache.view(torch.uint8).index_select(axis, torch.tensor(ids, device="cuda")).cpu())
    return held + [rows.view(torch.uint8)[torch.tensor(ids, device="cuda")].cpu()]


@pytest.mark.parametrize("save_mode,restore_mode", [("staged", "dma"), ("direct", "kernel")])
@pytest.mark.parametrize("layout", ["vllm", "kv_split"])
@pytest.mark.parametrize("row,apart", [(8, 8), (24, 40), (32, 32)])
def test_scales_travel_with_their_blocks_on_every_route(row, apart, layout, save_mode, restore_mode, hip_library,
                                                        oracle_lib, tmp_path):
    caches, _ = synth.make_caches(2, BLOCKS, block_size=SIZE, heads=2, head_dim=64, dtype=torch.float8_e4m3fn,
                                  layout=layout)
    gen = torch.Generator(device="cuda").manual_seed(row)
    for cache in caches.values():
        cache.view(torch.uint8).random_(0, 256, generator=gen)
    backing = torch.empty((BLOCKS, apart), dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
    rows = backing[:, :row]
    plane = TorchBlockDataPlane(caches, SIZE, 16 << 20, save_mode=save_mode, restore_mode=restore_mode, scales=rows)
    try:
        plane.warm_up()
        size = plane.block_bytes
        ids = random.Random(row).sample(range(BLOCKS), 2 * N)
        saved, into = ids[:N], ids[N:]
        want, around = contents(caches, rows, saved), backing[:, row:].clone()
        with plane.staging(N) as staged:
            targets = [(staged, i * size) for i in range(N)]
            digests = []
            plane.save_gather(saved, targets, N * SIZE, digests=digests)
            got = digests[0].result()
            records = np.ctypeslib.as_array(C.cast(staged.pointer, C.POINTER(C.c_uint8)), (N, size)).copy()
            assert (records[:, -row:] == want[-1].numpy()).all()
            for record, (hexdigest, crc) in zip(records, got):
                assert crc == oracle_lib.crc32c(record.tobytes())
                assert hexdigest == hashlib.sha256(record.tobytes()).hexdigest()
            crcs = [crc for _, crc in got]

            def cleared():
                for cache in caches.values():
                    axis = 1 if cache.ndim == 5 else 0
                    cache.view(torch.uint8).index_fill_(axis, torch.tensor(into, device="cuda"), 0)
                rows[torch.tensor(into, device="cuda")] = 0
                torch.cuda.synchronize()

            def arrived():
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(contents(caches, rows, into), want))
                assert all(torch.equal(a, b) for a, b in zip(contents(caches, rows, saved), want))
                assert torch.equal(backing[:, row:], around)

            for restore in (lambda: plane.load_scatter(into, targets),
                            lambda: plane.load_scatter_checked(into, targets, crcs),
                            lambda: plane.load_scatter_verified(into, targets, crcs)):
                cleared()
                restore()
                arrived()
            # a flipped bit of a scale is found
            at = staged.pointer + 7 * size + size - 1
            C.memmove(at, bytes([C.string_at(at, 1)[0] ^ 1]), 1)
            with pytest.raises(CorruptSnapshotError, match="block 7"):
                plane.load_scatter_verified(into, targets, crcs)
        store = BlobDirectory(tmp_path)
        snapshot = store.save(plane, saved, N * SIZE, durable=True)
        cleared()
        plane.load_from_disk(into, store, snapshot["segments"], chunk_bytes=7 * size)
        arrived()
    finally:
        torch.cuda.synchronize()
        plane.close()
