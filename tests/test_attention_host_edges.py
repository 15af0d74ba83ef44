"""What kvsnap_amd.attention refuses at its edges, without a GPU."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as forward_ad

from kvsnap_amd.attention import PagedCache, block_scales, rotate
from kvsnap_amd.native import kernel_library
from test_attention_host import (ON_CPU, Sequences, append, attend, built, c_layer, layer,  # noqa: F401  (a fixture)
                                 step)


class Rotation(C.Structure):
    _fields_ = [("angles", C.c_void_p), ("positions", C.c_void_p), ("rows", C.c_int64), ("axis_stride", C.c_int64),
                *((name, C.c_int32) for name in ("pairs", "interleaved", "narrow", "inverse")), ("axes", C.c_uint16 * 16)]


@pytest.mark.parametrize("name", ["query", "key", "value", "query_out"])
def test_a_forward_mode_tangent_is_refused_not_dropped(name):
    given = step()
    given.setdefault("query_out", torch.zeros_like(given["query"]))
    with forward_ad.dual_level():
        given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
        with pytest.raises(ValueError, match=f"^{name} carries a forward-mode tangent"):
            append(layer(), given)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode tangent"):
            append(layer(), given)
        with torch.inference_mode(), pytest.raises(ValueError, match=ON_CPU):       # which turns both modes off
            append(layer(), given)
        if name == "query":
            given.pop("query_out")
            with pytest.raises(ValueError, match="query carries a forward-mode tangent"):
                attend(layer(), given)
        x = forward_ad.make_dual(torch.zeros((3, 2, 64)), torch.ones((3, 2, 64)))
        with pytest.raises(ValueError, match="x carries a forward-mode tangent"):
            rotate(x, torch.zeros(3, dtype=torch.int64), torch.zeros((5, 32, 2)))


def test_a_gradient_of_the_cache_or_of_the_table_is_refused_not_dropped():
    cache = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, requires_grad=True)
    learned = torch.zeros((5, 32, 2), requires_grad=True)
    for call in (append, attend):
        with pytest.raises(ValueError, match="the cache requires a gradient"):
            call(PagedCache(cache, 16), step())
        with torch.no_grad(), pytest.raises(ValueError, match=ON_CPU):
            call(PagedCache(cache, 16), step())
    for call in (lambda: append(layer(), step(), rotary=learned),
                 lambda: rotate(torch.zeros((3, 2, 64)), torch.zeros(3, dtype=torch.int64), learned)):
        with pytest.raises(ValueError, match="a rotary table requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match=ON_CPU):
            call()


def test_a_plane_refuses_scales_that_it_does_not_save():
    """Its blocks would come back with the scales that some other block had."""
    from kvsnap_amd.dataplane import TorchBlockDataPlane
    plane = object.__new__(TorchBlockDataPlane)
    plane.block_size = 16
    plane.caches = {f"layer.{i}": torch.zeros((2, 4, 16, 2, 64)).to(torch.float8_e4m3fn) for i in range(3)}
    plane.scales, views = block_scales(5, 3, 2)
    views = [view[:4] for view in views]            # more rows than the caches have blocks
    for name, view in zip(plane.caches, views):
        assert plane.paged_cache(name, scales=view).scales is view
    wide, wide_views = block_scales(4, 9, 2)
    for other in (block_scales(4, 3, 2)[1][0], torch.zeros((4, 2, 2), dtype=torch.uint8), wide_views[8],
                  plane.scales[0].view(torch.uint8).view(4, 2, 2),              # all of one block's row
                  plane.scales.view(torch.uint8).flatten().as_strided((4, 2, 2), (16, 2, 1), 14)):      # into the next
        with pytest.raises(ValueError, match="no view of the plane's own"):
            plane.paged_cache("layer.0", scales=other)
    plane.scales = wide
    assert plane.paged_cache("layer.0", scales=wide_views[8]).scales is wide_views[8]
    plane.scales = None
    with pytest.raises(ValueError, match="registered without scales"):
        plane.paged_cache("layer.0", scales=views[0])
    plane.caches["plain"] = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16)
    assert plane.paged_cache("plain").scales is None


def test_the_workspace_of_heads_that_share_no_key_head_ends_no_process():
    """Fewer query heads than key heads, from C: a division by zero would be the whole process's end, so in its own."""
    program = """
import ctypes as C
from test_attention_host import c_layer
from kvsnap_amd.native import kernel_library
size = kernel_library().kvsnap_attend_workspace_bytes
for heads in (1, 3, 7, 9, 12):
    for ragged in (0, 1):
        assert size(C.addressof(c_layer(kv_heads=8)), 64, 2, ragged, heads, 1 << 20, 0) == 0
assert size(C.addressof(c_layer(kv_heads=8)), 64, 2, 1, 16, 1 << 20, 0) > 0
"""
    here = Path(__file__).resolve().parent
    done = subprocess.run([sys.executable, "-c", program], cwd=here, env={**os.environ, "PYTHONPATH": f"{here}:{here.parent}"},
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_the_c_entry_points_refuse_counts_whose_product_passes_64_bits():
    """2^40 + 1 rows of 2^24 heads in units of 16 values: 2^64 + 2^24 units for one launch."""
    lib = kernel_library()
    turns = Rotation(angles=4096, positions=4096, rows=10, pairs=8)
    assert lib.kvsnap_rotate(4096, 16, 16, 4096, 16, 16, (1 << 40) + 1, 1 << 24, 16, 0, C.addressof(turns), 0) == -1
    assert "too many values" in lib.kvsnap_cuda_error().decode()
    sequences = Sequences(4096, 4096, 4096, 2, 2, 1)
    assert lib.kvsnap_append(C.addressof(c_layer(width=16)), C.addressof(sequences), None, 4096, 16, 16, 4096, 16, 16, 4096,
                             16, 16, 4096, 16, 16, (1 << 31) - 1, (1 << 31) - 1, 0, 0) == -1
    assert "too many values" in lib.kvsnap_cuda_error().decode()


def test_a_rotary_table_of_no_positions_is_refused():
    """Its address is none, which to the library means that nothing is turned."""
    none = torch.zeros((0, 32, 2))
    with pytest.raises(ValueError, match="of one position or more"):
        append(layer(), step(), rotary=none)
    with pytest.raises(ValueError, match="of one position or more"):
        rotate(torch.zeros((3, 2, 64)), torch.zeros(3, dtype=torch.int64), none)


FUSED = torch.zeros((5, 12, 64), dtype=torch.bfloat16)
WIDE = torch.zeros((5, 4, 3, 64), dtype=torch.bfloat16)             # a head's query, key and value side by side


@pytest.mark.parametrize("out,overlaps", [
    (FUSED[:3, 0:4], False),                    # query itself
    (FUSED[:3, 4:8], False), (FUSED[:3, 8:12], False), (FUSED[3:5].reshape(-1)[:768].view(3, 4, 64), False),
    (FUSED[:3, 1:5], True), (FUSED[:3, 3:7], True), (FUSED[1:4, 0:4], True), (FUSED[2:5, 0:4], True),
    (FUSED.view(-1)[:768].view(3, 4, 64), True), (FUSED.view(-1)[512:1280].view(3, 4, 64), True),
    (FUSED.view(-1)[8:].as_strided((3, 4, 64), (768, 64, 1), 8), True),
    (FUSED.view(-1).as_strided((3, 4, 64), (64, 192, 1), 0), True),
    (torch.zeros((3, 4, 64), dtype=torch.bfloat16), False),
])
def test_an_output_over_other_rows_of_its_input_is_refused(out, overlaps):
    query = FUSED[:3, 0:4]
    why = "itself or not overlap it" if overlaps else ON_CPU
    positions, table = torch.zeros(3, dtype=torch.int64), torch.zeros((5, 32, 2))
    with pytest.raises(ValueError, match=why):
        rotate(query, positions, table, out=out)
    with pytest.raises(ValueError, match=why):
        append(layer(), step(), query=query, query_out=out)
    with pytest.raises(ValueError, match=why):
        attend(layer(), step(), query=query, out=out)


def test_an_output_over_keys_or_values_is_refused():
    q, k, v = FUSED[:3].split([4, 4, 4], 1)
    append_to = layer(kv=4)
    for out, why in ((q, ON_CPU), (k, "query_out must not overlap key"), (v, "query_out must not overlap value"),
                     (FUSED[:3, 2:6], "query itself or not overlap it"), (FUSED[:3, 6:10], "must not overlap key")):
        with pytest.raises(ValueError, match=why):
            append(append_to, step(kv=4), query=q, key=k, value=v, query_out=out)
    q, k, v = WIDE[:3].unbind(2)
    for out, why in ((q, ON_CPU), (k, "query_out must not overlap key"), (v, "query_out must not overlap value"),
                     (WIDE[2:5, :, 0], "query itself or not overlap it"), (WIDE[2:5, :, 1], "must not overlap key")):
        with pytest.raises(ValueError, match=why):
            append(append_to, step(kv=4), query=q, key=k, value=v, query_out=out)


@pytest.mark.parametrize("scales,shared", [
    (torch.zeros((4, 1, 1), dtype=torch.uint8).expand(4, 2, 2), True),           # one a block, broadcast
    (torch.zeros((1, 2, 2), dtype=torch.uint8).expand(4, 2, 2), True),
    (torch.zeros((4, 2, 1), dtype=torch.uint8).expand(4, 2, 2), True),
    (torch.zeros((20,), dtype=torch.uint8).as_strided((4, 2, 2), (2, 1, 1)), True),
    (torch.zeros((20,), dtype=torch.uint8).as_strided((4, 2, 2), (3, 2, 1)), True),
    (torch.zeros((2, 4, 2), dtype=torch.uint8).transpose(0, 1), False),
    (torch.zeros((2, 2, 4), dtype=torch.uint8).permute(2, 1, 0), False),
    (block_scales(4, 3, 2)[1][1], False),
])
def test_scales_that_share_bytes_are_read_but_not_appended_to(scales, shared):
    held = PagedCache(torch.zeros((2, 4, 16, 2, 64)).to(torch.float8_e4m3fn), 16, scales=scales)
    with pytest.raises(ValueError, match="share bytes" if shared else ON_CPU):
        append(held, step())
    with pytest.raises(ValueError, match=ON_CPU):
        attend(held, step())
