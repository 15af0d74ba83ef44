"""What kvsnap_amd.attention refuses, and its helpers, without a GPU: everything but the device is checked first."""
import ctypes as C
import math
import re
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from kvsnap_amd import attention
from kvsnap_amd.attention import PagedCache, block_scales, rotary_table, rotate
from kvsnap_amd.native import kernel_library
from paged_reference import attend64, rotate64, scale_of, table64

ROOT = Path(__file__).resolve().parents[1]
BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def built():
    from kvsnap_amd import build
    if not (build.HIP_LIBRARY.is_file() and build.BINDING.is_file()):
        build.build_all()


def layer(dtype=BF16, kv=2, width=64, size=16, blocks=4):
    scales = block_scales(blocks, 1, kv)[1][0] if dtype == E4M3 else None
    return PagedCache(torch.zeros((2, blocks, size, kv, width)).to(dtype), size, scales=scales)


def step(tokens=3, heads=4, kv=2, width=64, dtype=BF16, seqs=3):
    return dict(query=torch.zeros((tokens, heads, width), dtype=dtype), key=torch.zeros((tokens, kv, width), dtype=dtype),
                value=torch.zeros((tokens, kv, width), dtype=dtype),
                block_tables=torch.zeros((seqs, 2), dtype=torch.int32), lengths=torch.ones(seqs, dtype=torch.int32))


def append(to, given, **changes):
    given = {**given, **changes}
    return to.append(given.pop("key"), given.pop("value"), given.pop("block_tables"), given.pop("lengths"), **given)


def attend(over, given, **changes):
    given = {**given, **changes}
    given.pop("key", None), given.pop("value", None)
    return over.attend(given.pop("query"), given.pop("block_tables"), given.pop("lengths"), **given)


ON_CPU = "on one and the same CUDA device"


def test_calls_that_are_right_but_for_the_device():
    for dtype in (BF16, FP16):
        for held in (dtype, E4M3):
            with pytest.raises(ValueError, match=ON_CPU):
                append(layer(held), step(dtype=dtype))
            with pytest.raises(ValueError, match=ON_CPU):
                attend(layer(held), step(dtype=dtype))
    table = rotary_table(64, 10)
    with pytest.raises(ValueError, match=ON_CPU):
        append(layer(), step(), rotary=table, positions=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match=ON_CPU):
        attend(layer(), step(tokens=5), query_starts=torch.zeros(4, dtype=torch.int32), window=3, max_length=9,
               softmax_scale=1, return_lse=True)
    for dtype in (BF16, FP16, torch.float32):
        with pytest.raises(ValueError, match=ON_CPU):
            rotate(torch.zeros((3, 2, 64), dtype=dtype), torch.zeros(3, dtype=torch.int32), table)


@pytest.mark.parametrize("changes,why", [
    (dict(key=torch.zeros((3, 2, 64))), "both be bfloat16 or float16"),
    (dict(key=torch.zeros((3, 2, 64), dtype=FP16), value=torch.zeros((3, 2, 64), dtype=FP16)), "a 16-bit cache's own"),
    (dict(value=torch.zeros((3, 2, 64), dtype=FP16)), "both be bfloat16 or float16"),
    (dict(key=torch.zeros((3, 1, 64), dtype=BF16)), r"key must be \[any, 2, 64\]"),
    (dict(key=torch.zeros((3, 128), dtype=BF16)), "key must be"),
    (dict(value=torch.zeros((2, 2, 64), dtype=BF16)), r"value must be \[3, 2, 64\]"),
    (dict(key=torch.zeros((3, 2, 128), dtype=BF16)[..., ::2]), "last axis must be contiguous"),
    (dict(query=torch.zeros((2, 4, 64), dtype=BF16)), "query must be"),
    (dict(query=torch.zeros((3, 4, 64), dtype=FP16)), "query must have the keys' type"),
    (dict(query=None, query_out=torch.zeros((3, 4, 64), dtype=BF16)), "query_out needs a query"),
    (dict(query_out=torch.zeros((3, 3, 64), dtype=BF16)), "query_out must be"),
    (dict(query_out=torch.zeros((3, 4, 64), dtype=FP16)), "query_out must have the type"),
    (dict(key=3), "key must be a tensor"),
    (dict(lengths=None), "lengths must be a tensor"),
    (dict(lengths=torch.ones(2, dtype=torch.int32)), "block_tables must be"),
    (dict(lengths=torch.ones(3, dtype=torch.int64)), "must be int32"),
    (dict(block_tables=torch.zeros((3, 2), dtype=torch.int64)), "must be int32"),
    (dict(block_tables=torch.zeros((3, 4), dtype=torch.int32)[:, ::2]), "contiguous along their last"),
    (dict(block_tables=torch.zeros((2, 2), dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32)),
     "query_starts is needed"),
    (dict(query_starts=torch.zeros(3, dtype=torch.int32)), r"query_starts must be \[4\]"),
    (dict(query_starts=torch.zeros((), dtype=torch.int32)), "contiguous along their last"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "need a rotary table"),
    (dict(axes=[0]), "need a rotary table"),
    (dict(rotary=torch.zeros((5, 32, 2), dtype=torch.float64)), "a rotary table is"),
    (dict(rotary=torch.zeros((5, 64))), "a rotary table is"),
    (dict(rotary=torch.zeros((5, 12, 2))), "multiple of 8"),
    (dict(rotary=torch.zeros((5, 40, 2))), "multiple of 8 and at most 32"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros(2, dtype=torch.int64)), "positions must be"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros(3)), "int64 or int32"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros((2, 3), dtype=torch.int64)), "need axes"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros((5, 3), dtype=torch.int64), axes=[4] * 32), "4 at most"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros((2, 3), dtype=torch.int64), axes=[2] * 32), "axes must"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros((2, 3), dtype=torch.int64), axes=[0] * 31), "axes must"),
    (dict(rotary=torch.zeros((5, 32, 2)), positions=torch.zeros((2, 3), dtype=torch.int64), axes=[-1] * 32), "axes must"),
    (dict(key=torch.zeros((3, 2, 64), dtype=BF16, requires_grad=True)), "no gradient is recorded"),
])
def test_append_refuses(changes, why):
    with pytest.raises(ValueError, match=why):
        append(layer(), step(), **changes)


@pytest.mark.parametrize("changes,why", [
    (dict(query=torch.zeros((3, 4, 64))), "bfloat16 or float16"),
    (dict(query=torch.zeros((3, 4, 64), dtype=FP16)), "a 16-bit cache's own type"),
    (dict(query=torch.zeros((3, 4, 80), dtype=BF16)), "query must be"),
    (dict(query=torch.zeros((3, 3, 64), dtype=BF16)), "3 query heads do not share"),
    (dict(query=torch.zeros((3, 0, 64), dtype=BF16)), "0 query heads do not share"),
    (dict(query=torch.zeros((3, 4, 64), dtype=BF16, requires_grad=True)), "no gradient is recorded"),
    (dict(window=0), "a window holds"),
    (dict(window=-5), "a window holds"),
    (dict(max_length=-1), "max_length must not be negative"),
    (dict(softmax_scale=0.0), "softmax_scale must be positive"),
    (dict(softmax_scale=-1.0), "softmax_scale must be positive"),
    (dict(softmax_scale=math.nan), "softmax_scale must be positive"),
    (dict(softmax_scale=math.inf), "softmax_scale must be positive"),
    (dict(out=torch.zeros((3, 4, 64), dtype=FP16)), "out must have the type"),
    (dict(out=torch.zeros((2, 4, 64), dtype=BF16)), "out must be"),
    (dict(query=torch.zeros((4, 4, 64), dtype=BF16)), "query_starts is needed"),
    (dict(lengths=torch.ones((3, 1), dtype=torch.int32)), "block_tables must be"),
])
def test_attend_refuses(changes, why):
    with pytest.raises(ValueError, match=why):
        attend(layer(), step(), **changes)


def test_attend_refuses_what_is_no_number():
    for changes in (dict(window="3"), dict(max_length=2.5), dict(softmax_scale="x")):
        with pytest.raises(TypeError):
            attend(layer(), step(), **changes)


@pytest.mark.parametrize("x,changes,why", [
    (torch.zeros((3, 64)), {}, "x must be"),
    (torch.zeros((3, 2, 64), dtype=torch.float64), {}, "bfloat16, float16 or float32"),
    (torch.zeros((3, 2, 64)).to(E4M3), {}, "bfloat16, float16 or float32"),
    (torch.zeros((3, 2, 72)), {}, "multiple of 16 up to 256, not 72"),
    (torch.zeros((3, 2, 272)), {}, "multiple of 16 up to 256, not 272"),
    (torch.zeros((3, 2, 32)), {}, "at most 16"),
    (torch.zeros((3, 2, 64)), dict(positions=None), "needs positions"),
    (torch.zeros((3, 2, 64)), dict(rotary=None), "needs positions and a rotary table"),
    (torch.zeros((3, 2, 64)), dict(out=torch.zeros((3, 2, 64), dtype=BF16)), "out must have the type"),
    (torch.zeros((4, 2, 64)), {}, "positions must be"),
])
def test_rotate_refuses(x, changes, why):
    given = dict(positions=torch.zeros(3, dtype=torch.int64), rotary=torch.zeros((5, 32, 2)))
    given.update(changes)
    with pytest.raises(ValueError, match=why):
        rotate(x, given["positions"], given["rotary"], out=given.get("out"))


@pytest.mark.parametrize("cache,scales,why", [
    (torch.zeros((2, 4, 16, 2, 64)), None, "must be bfloat16, float16 or float8_e4m3fn"),
    (torch.zeros((2, 4, 16, 2, 72), dtype=BF16), None, "multiple of 16"),
    (torch.zeros((2, 4, 16, 2, 272), dtype=BF16), None, "multiple of 16"),
    (torch.zeros((4, 2, 16, 33), dtype=BF16), None, "a key and a value"),
    (torch.zeros((2, 4, 8, 2, 64), dtype=BF16), None, "8 token slots"),
    (torch.zeros((4, 16, 2, 128), dtype=BF16), None, "2 token slots"),
    (torch.zeros((2, 0, 16, 2, 64), dtype=BF16), None, "not empty"),
    (torch.zeros((2, 4, 16, 2, 64), dtype=BF16), torch.zeros((4, 2, 2), dtype=torch.uint8), "no other takes them"),
    (torch.zeros((2, 4, 16, 2, 64)).to(E4M3), None, "needs scales"),
    (torch.zeros((2, 4, 16, 2, 64)).to(E4M3), torch.zeros((4, 2), dtype=torch.uint8), "scales must be"),
    (torch.zeros((2, 4, 16, 2, 64)).to(E4M3), torch.zeros((4, 2, 2)), "scales must be"),
    (torch.zeros((2 * 4 * 16 * 2 * 64 + 4,), dtype=BF16)[4:].view(2, 4, 16, 2, 64), None, "16-byte aligned"),
])
def test_a_cache_that_is_no_paged_cache_is_refused(cache, scales, why):
    with pytest.raises(ValueError, match=why):
        PagedCache(cache, 16, scales=scales)


def test_block_scales_are_whole_words_a_block():
    rows, views = block_scales(5, 3, 3)
    assert rows.shape == (5, 32) and rows.dtype == torch.float8_e8m0fnu and len(views) == 3
    for i, view in enumerate(views):
        assert view.shape == (5, 3, 2) and view.data_ptr() == rows.data_ptr() + 6 * i and view.stride() == (32, 2, 1)


def test_rotary_table():
    assert torch.equal(rotary_table(32, 7, base=500.0).double(), table64(32, 7, 500.0))
    for width, positions in ((0, 5), (24, 5), (32, 0), (-16, 5)):
        with pytest.raises(ValueError):
            rotary_table(width, positions)


def test_the_references_agree_with_torch():
    """The 64-bit definitions the GPU tests use, against torch's own attention and complex products."""
    torch.manual_seed(0)
    keys, values = torch.randn((2, 5, 4, 2, 16), dtype=torch.float64)
    query = torch.randn((9, 6, 16), dtype=torch.float64)
    tables, lengths = torch.tensor([[3, 1, 4]], dtype=torch.int32), torch.tensor([11])
    out, lse = attend64(query, keys, values, tables, lengths, torch.tensor([0, 9]))
    line = [keys[[3, 1, 4]].flatten(0, 1)[:11], values[[3, 1, 4]].flatten(0, 1)[:11]]
    k, v = (side.repeat_interleave(3, 1).transpose(0, 1) for side in line)
    mask = torch.arange(11)[None] <= torch.arange(2, 11)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(query.transpose(0, 1), k, v, attn_mask=mask)
    assert torch.allclose(out, want.transpose(0, 1), atol=1e-12)
    scores = (query.transpose(0, 1) @ k.transpose(1, 2) / 4).masked_fill(~mask, -math.inf)
    assert torch.allclose(lse, scores.logsumexp(-1).T, atol=1e-12)
    x, positions, table = torch.randn((4, 1, 16), dtype=torch.float64), torch.tensor([0, 5, 2, 9]), table64(16, 10)
    turn = torch.view_as_complex(table[positions])[:, None]
    want = torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (8, 2)).contiguous()) * turn).flatten(-2)
    assert torch.allclose(rotate64(x, positions, table, interleaved=True), want, atol=1e-12)
    assert [scale_of(x) for x in (0.0, 448.0, 448.1, 447.9, 1.75, 1.8, 896.0)] == [1, 127, 128, 127, 119, 120, 128]


# ---- the C entry points, on the host


def test_the_library_exports_the_operators():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "kvsnap_attention.h").read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(kvsnap_\w+)\s*\(", text)))
    assert names == ["kvsnap_append", "kvsnap_attend", "kvsnap_attend_workspace_bytes", "kvsnap_rotate"]
    library = ROOT / "kvsnap_amd" / "_native" / "libkvsnap_hip.so"
    exported = subprocess.run(["nm", "-D", "--defined-only", str(library)], check=True, capture_output=True, text=True)
    assert set(names) <= set(exported.stdout.split())


class Sequences(C.Structure):
    _fields_ = [("block_tables", C.c_void_p), ("lengths", C.c_void_p), ("query_starts", C.c_void_p),
                ("table_stride", C.c_int64), ("table_width", C.c_int32), ("n_seqs", C.c_int32)]


def c_layer(**changes):
    given = dict(key=4096, value=8192, scales=None, block_stride=2048, token_stride=128, head_stride=64,
                 scale_block_stride=4, scale_head_stride=2, scale_side_stride=1, blocks=4, block_size=16, kv_heads=2,
                 width=64, type=0)
    given.update(changes)
    return attention._Layer(*(given[name] for name, _ in attention._Layer._fields_))


def c_attend(layer, *, sequences=None, query=4096, strides=(256, 64), tokens=3, heads=4, kind=0, scale=0.1, window=0,
             longest=32, workspace=None, room=0):
    sequences = sequences or Sequences(4096, 4096, None, 2, 2, 3)
    lib = kernel_library()
    rc = lib.kvsnap_attend(C.addressof(layer), C.addressof(sequences), query, *strides, 4096, 256, 64, None, tokens,
                           heads, kind, scale, window, longest, workspace, room, 0)
    return rc, lib.kvsnap_cuda_error().decode()


@pytest.mark.parametrize("changes,why", [
    (dict(width=72), "multiple of 16"), (dict(width=272), "multiple of 16"), (dict(blocks=0), "not be empty"),
    (dict(block_size=0), "not be empty"), (dict(key=4100), "16-byte aligned"), (dict(token_stride=12), "16-byte"),
    (dict(type=3), "bf16, fp16 or e4m3"), (dict(type=2), "has scales"), (dict(scales=4096), "has scales"),
    (dict(key=None), "device pointers"), (dict(block_stride=1 << 40), "under 64 GiB"),
    (dict(block_stride=-2048), "under 64 GiB"), (dict(block_size=1 << 21), "too many or long"),
])
def test_the_c_entry_points_refuse_a_bad_layer_before_any_gpu_call(changes, why):
    rc, message = c_attend(c_layer(**changes))
    assert rc == -1 and why in message


@pytest.mark.parametrize("changes,why", [
    (dict(tokens=-1), "bad size"), (dict(tokens=2), "one row"), (dict(heads=3), "multiple of the cache's"),
    (dict(kind=1), "16-bit cache"), (dict(kind=3), "bf16 or fp16"), (dict(query=None), "device pointers"),
    (dict(query=4104), "16-byte aligned"), (dict(strides=(256, 68)), "16-byte aligned"), (dict(scale=0.0), "positive"),
    (dict(window=-1), "negative window"), (dict(longest=-1), "negative window"),
    (dict(sequences=Sequences(4096, None, None, 2, 2, 3)), "device pointers"),
    (dict(sequences=Sequences(4096, 4096, None, 2, -2, 3)), "negative table"),
    (dict(sequences=Sequences(4096, 4096, None, 2, 1 << 27, 3)), "2^30 tokens"),
    (dict(sequences=Sequences(4096, 4096, None, 4096, 4096, 3), longest=1 << 16), "workspace is too small"),
    (dict(sequences=Sequences(4096, 4096, None, 4096, 4096, 3), longest=1 << 16, room=1 << 40, workspace=4100),
     "16-byte aligned device memory"),
])
def test_the_c_attend_refuses_bad_sizes_before_any_gpu_call(changes, why):
    rc, message = c_attend(c_layer(), **changes)
    assert rc == -1 and why in message


def test_calls_of_nothing_launch_nothing():
    assert c_attend(c_layer(), tokens=0, sequences=Sequences(None, None, None, 0, 0, 0))[0] == 0
    assert c_attend(c_layer(), heads=0)[0] == 0
    lib = kernel_library()
    assert lib.kvsnap_rotate(None, 0, 0, None, 0, 0, 0, 4, 64, 0, None, 0) == 0
    empty = Sequences(None, None, None, 0, 0, 0)
    assert lib.kvsnap_append(C.addressof(c_layer()), C.addressof(empty), None, None, 0, 0, None, 0, 0, None, 0, 0, None,
                             0, 0, 0, 0, 0, 0) == 0


def test_the_workspace_grows_with_what_is_split_and_is_none_for_short_rows():
    held = c_layer(kv_heads=8, width=128, token_stride=1024, head_stride=128, block_stride=16384)
    one = c_layer(kv_heads=1, width=128, token_stride=128, head_stride=128, block_stride=2048)
    size = kernel_library().kvsnap_attend_workspace_bytes
    assert size(C.addressof(one), 1, 1, 0, 4, 75, 0) == 0 and size(C.addressof(one), 0, 1, 0, 4, 1 << 20, 0) == 0
    # a prompt's tiles are whole; beside another sequence there is room for the parts of a row alone
    assert size(C.addressof(held), 8192, 1, 1, 32, 8192, 0) == 0 < size(C.addressof(held), 8192, 2, 1, 32, 8192, 0)
    assert size(C.addressof(held), 8192, 1, 1, 32, 8192, 0) <= 32 << 20
    assert 0 < size(C.addressof(held), 1, 1, 0, 32, 32768, 0) <= 32 << 20
    assert size(C.addressof(held), 1, 1, 0, 32, 32768, 100) == 0


# ---- a plane with scales


class Rows:
    """A row of bytes a block, as a scales tensor describes itself."""

    dtype, ndim = "torch.float8_e8m0fnu", 2

    def __init__(self, shape=(6, 32), strides=None, address=4096, device=None):
        from types import SimpleNamespace
        self.shape, self.strides, self.address = shape, strides or (shape[1], 1), address
        self.device = device or SimpleNamespace(type="cuda", index=0)

    def stride(self, axis):
        return self.strides[axis]

    def element_size(self):
        return 1

    def data_ptr(self):
        return self.address


def plane_with(scales):
    import sys
    from types import SimpleNamespace
    from unittest.mock import MagicMock, patch
    from kvsnap_amd import dataplane

    class Cache:
        dtype, ndim, shape, strides = "torch.float8_e4m3fn", 4, (8, 2, 16, 128), (4096, 128, 256, 1)
        device = scales.device

        def stride(self, axis):
            return self.strides[axis]

        def element_size(self):
            return 1

        def data_ptr(self):
            return 1 << 20

    with patch.dict(sys.modules, {"torch": SimpleNamespace()}), \
         patch.object(dataplane, "CudaPool", return_value=MagicMock()):
        return dataplane.TorchBlockDataPlane({"layer.0": Cache()}, 16, 4096, scales=scales)


def test_a_planes_record_ends_with_the_blocks_scales():
    plane = plane_with(Rows())
    assert plane.block_bytes == 4096 + 32 and plane.spans() == [(0, 1 << 20, 4096, 4096), (4096, 4096, 32, 32)]
    assert plane.min_span_bytes == 4096 and '"block scales"' in plane.layout_identity
    # the token slots past the last one are zeroed, the scales are not; and the front of every span is no filled block
    assert plane._tail_regions(15) == [(15 * 256, 256)] and not plane._token_bytes_divide()
    plane._validate_ids([0, 5])
    with pytest.raises(ValueError, match="out of range"):
        plane._validate_ids([6])


@pytest.mark.parametrize("scales,why", [
    (dict(shape=(6, 12)), "whole 8-byte words"), (dict(shape=(6, 0)), "whole 8-byte words"),
    (dict(strides=(32, 2)), "contiguous"), (dict(strides=(24, 1)), "contiguous"), (dict(strides=(36, 1)), "contiguous"),
])
def test_scales_that_a_plane_cannot_save_are_refused(scales, why):
    with pytest.raises(ValueError, match=why):
        plane_with(Rows(**scales))
    with pytest.raises(ValueError, match="8-byte aligned"):
        plane_with(Rows(address=4100)).spans()


@pytest.mark.parametrize("out,overlaps", [
    (torch.zeros((4, 64)).as_strided((3, 2, 64), (64, 32, 1)), True),           # heads run into one another
    (torch.zeros((1, 2, 64)).expand(3, 2, 64), True),
    (torch.zeros((3, 1, 64)).expand(3, 2, 64), True),
    (torch.zeros((2, 128)).as_strided((3, 2, 64), (64, 64, 1)), True),          # a row's second head is the next's first
    (torch.zeros((2, 3, 64)).transpose(0, 1), False),
    (torch.zeros((3, 2, 96))[..., :64], False),
])
def test_an_output_that_overlaps_itself_is_refused(out, overlaps):
    with pytest.raises(ValueError, match="must not overlap itself" if overlaps else ON_CPU):
        rotate(torch.zeros((3, 2, 64)), torch.zeros(3, dtype=torch.int64), torch.zeros((5, 32, 2)), out=out)


@pytest.mark.parametrize("changes", [dict(token_stride=1 << 27), dict(block_stride=(1 << 60)),
                                     dict(block_size=1 << 20, token_stride=1 << 20)])
def test_the_c_entry_points_refuse_caches_whose_places_pass_32_bits(changes):
    rc, message = c_attend(c_layer(**changes))
    assert rc == -1 and "under 64 GiB" in message
