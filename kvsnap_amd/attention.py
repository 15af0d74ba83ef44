"""Operators over a layer's paged KV cache: rotary positions, appends and attention.

What a serving step does between its projections and a layer's output, over the caches that
``TorchBlockDataPlane`` registers, saves and restores:

* :func:`rotate` turns a tensor's heads by their tokens' positions (one axis, or several for images and video);
  ``inverse`` turns them back, which is its gradient too.
* :meth:`PagedCache.append` puts a step's keys, turned, and values into the blocks that the block tables name, in
  the cache's 16 bits or in e4m3 with a power-of-two scale for each block of tokens and head.
* :meth:`PagedCache.attend` is attention over what the cache holds, for single tokens and for prompts.

Tables of blocks, lengths and row starts are read on the GPU: no call synchronizes, allocates anything but its
outputs and workspace (from torch's allocator, on the current stream), or keeps anything for a later call, so all of
them may be captured in a graph and replayed over changed tables.  Launches go to the current stream of the cache's
device.  There is no CPU fallback: without the HIP library every call raises.

The kernels' contract is in ``include/kvsnap_attention.h``.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
import struct

from .layout import describe_layer
from .native import check as _check, kernel_library

__all__ = ["PagedCache", "block_scales", "rotary_table", "rotate"]

#: Type codes of include/kvsnap_attention.h by torch type name.
_TYPES = {"torch.bfloat16": 0, "torch.float16": 1, "torch.float8_e4m3fn": 2, "torch.float32": 3}
_SEQUENCES = struct.Struct("=QQQqii").pack
_ROTATION = struct.Struct("=QQqqiiii32s").pack


class _Layer(C.Structure):
    _fields_ = [("key", C.c_void_p), ("value", C.c_void_p), ("scales", C.c_void_p),
                *((name, C.c_int64) for name in ("block_stride", "token_stride", "head_stride", "scale_block_stride",
                                                 "scale_head_stride", "scale_side_stride", "blocks")),
                *((name, C.c_int32) for name in ("block_size", "kv_heads", "width", "type"))]


def rotary_table(width, positions, *, base=10000.0, device=None):
    """The angles' cosines and sines that rotations take: fp32 ``[positions, width / 2, 2]``, pair j of position p at
    ``p * base ** (-2 j / width)``, computed in 64 bits (an angle of 40,000 radians has no fraction left in 32)."""
    import torch
    if width <= 0 or width % 16 or positions <= 0:
        raise ValueError("a rotary table needs positions, and a width that is a multiple of 16")
    pairs = torch.arange(width // 2, dtype=torch.float64, device=device)
    turns = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * pairs / width)
    return torch.stack([turns.cos(), turns.sin()], -1).float()


def block_scales(blocks, layers, heads, *, device=None):
    """Scales of e4m3 caches of ``layers`` layers: one tensor whose rows are whole 8-byte words, so that a plane can
    save them with their blocks (``TorchBlockDataPlane(..., scales=...)``), and its ``[blocks, heads, 2]`` view for
    each layer's :class:`PagedCache`."""
    import torch
    used = layers * heads * 2
    rows = torch.zeros((blocks, -(-used // 8) * 8), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    return rows, [rows[:, at:at + 2 * heads].unflatten(1, (heads, 2)) for at in range(0, used, 2 * heads)]


@lru_cache(maxsize=64)
def _packed_axes(axes):
    """Two bits a pair, 16 words of eight pairs."""
    words = [0] * 16
    for pair, axis in enumerate(axes):
        words[pair // 8] |= axis << (2 * (pair % 8))
    return struct.pack("=16H", *words)


_ONE_AXIS = bytes(32)


def _on_gpu(device, *tensors):
    """The caller's device must be one GPU for all of a call's tensors (checked last: everything else can be found
    wrong without one)."""
    if device.type != "cuda" or any(t.device != device for t in tensors):
        raise ValueError("every tensor of a call must be on one and the same CUDA device")


def _rows(what, tensor, tokens, heads, width):
    """A ``[tokens, heads, width]`` tensor (None: any) whose last axis is contiguous."""
    if tensor.ndim != 3 or any(want is not None and have != want
                               for have, want in zip(tensor.shape, (tokens, heads, width))):
        want = ", ".join("any" if n is None else str(n) for n in (tokens, heads, width))
        raise ValueError(f"{what} must be [{want}], not {list(tensor.shape)}")
    if tensor.stride(2) != 1 and tensor.shape[2] > 1:
        raise ValueError(f"{what}: the last axis must be contiguous")


def _rotation(rotary, positions, tokens, width, axes, interleaved, inverse):
    """The kernels' description of a rotation, and the tensors it reads; None without one."""
    if rotary is None:
        if positions is not None or axes is not None:
            raise ValueError("positions and axes need a rotary table")
        return None, ()
    if rotary.ndim != 3 or rotary.shape[2] != 2 or str(rotary.dtype) != "torch.float32" or not rotary.is_contiguous():
        raise ValueError("a rotary table is a contiguous float32 [positions, pairs, 2] tensor")
    rows, pairs, _ = rotary.shape
    if not pairs or pairs % 8 or 2 * pairs > width:
        raise ValueError(f"a rotary table's pairs must be a multiple of 8 and at most {width // 2}, not {pairs}")
    count, pointer, stride, narrow, tensors = 1, 0, 0, 0, (rotary,)
    if positions is not None:
        dtype = str(positions.dtype)
        if dtype not in ("torch.int64", "torch.int32"):
            raise ValueError("positions must be int64 or int32")
        if positions.ndim not in (1, 2) or positions.shape[-1] != tokens or (
                positions.stride(-1) != 1 and tokens > 1):
            raise ValueError(f"positions must be [{tokens}] or [axes, {tokens}], the last axis contiguous")
        if positions.ndim == 2:
            count, stride = positions.shape[0], positions.stride(0)
        pointer, narrow, tensors = positions.data_ptr(), dtype == "torch.int32", (rotary, positions)
    packed = _ONE_AXIS
    if axes is not None:
        axes = tuple(axes)
        if len(axes) != pairs or not 1 <= count <= 4 or not set(axes) <= set(range(count)):
            raise ValueError(f"axes must name, for each of {pairs} pairs, one of the positions' {count} axes (4 at most)")
        packed = _packed_axes(axes)
    elif count != 1:
        raise ValueError("positions of several axes need axes: the axis of each pair")
    return _ROTATION(rotary.data_ptr(), pointer, rows, stride, pairs, bool(interleaved), narrow, bool(inverse),
                     packed), tensors


def _launch(device, launch):
    """``launch(stream handle)`` with ``device`` current (the calling thread may have another)."""
    import torch
    if torch.cuda.current_device() == device.index:
        return launch(torch.cuda.current_stream(device).cuda_stream)
    with torch.cuda.device(device):
        return launch(torch.cuda.current_stream(device).cuda_stream)


def rotate(x, positions, rotary, *, axes=None, interleaved=False, inverse=False, out=None):
    """``x`` ([tokens, heads, width], bf16, fp16 or fp32) with each pair of a head's values turned by the angle of its
    token's position: (a, b) becomes (a cos - b sin, b cos + a sin), in fp32 and rounded once.

    Pair j is values j and j + pairs of a head, or with ``interleaved`` 2j and 2j + 1; values past the table's pairs
    are copied.  ``positions`` (int64 or int32) is ``[tokens]``, or ``[axes, tokens]`` for positions of several axes
    (time, height and width, say), where ``axes`` names the axis of each pair.  A position outside ``rotary``'s rows
    has no angle and gives NaN.  ``inverse`` turns the other way: it undoes a rotation, gives its gradient, and moves
    kept keys to earlier positions.  ``out`` (a new tensor if None) may be ``x`` itself.
    """
    import torch
    _rows("x", x, None, None, None)
    tokens, heads, width = x.shape
    kind = _TYPES.get(str(x.dtype), 2)
    if kind == 2:
        raise ValueError("x must be bfloat16, float16 or float32")
    if width % 16 or not 0 < width <= 256:
        raise ValueError(f"x's width must be a multiple of 16 up to 256, not {width}")
    if positions is None or rotary is None:
        raise ValueError("a rotation needs positions and a rotary table")
    rotation, tensors = _rotation(rotary, positions, tokens, width, axes, interleaved, inverse)
    if out is None:
        out = torch.empty((tokens, heads, width), dtype=x.dtype, device=x.device)
    else:
        _rows("out", out, tokens, heads, width)
        if out.dtype != x.dtype:
            raise ValueError("out must have x's type")
    _on_gpu(x.device, out, *tensors)
    lib = kernel_library()
    _launch(x.device, lambda stream: _check(lib, lib.kvsnap_rotate(
        x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1), tokens, heads, width,
        kind, rotation, stream)))
    return out


class PagedCache:
    """One layer's paged KV cache, as a plane registers it, for the operators that fill and read it.

    ``cache`` is a ``[blocks, heads, tokens, 2 * width]`` view (each token's key, then its value: vLLM's layout) or a
    K/V-split ``[2, blocks, tokens, heads, width]`` tensor of ``block_size`` token slots a block, in bfloat16,
    float16 or float8_e4m3fn; widths are multiples of 16 up to 256.  An e4m3 cache comes with ``scales``
    (float8_e8m0fnu or uint8 ``[blocks, heads, 2]``, K's and V's, see :func:`block_scales`): a stored value stands
    for itself times its block and head's power of two.  The cache is kept, not copied.

    Every call takes the step's tables (int32, on the cache's device, read there): ``block_tables`` ``[sequences,
    most blocks]``, ``lengths`` ``[sequences]`` counting the step's own tokens, and ``query_starts`` ``[sequences +
    1]``, the first row of each sequence in the step's tensors, or None where each sequence has one row.  Rows past
    the last sequence's are padding.  A table entry that names no block of the cache is skipped: nothing is written
    for it, and nobody sees its tokens.
    """

    def __init__(self, cache, block_size, *, scales=None):
        described = describe_layer("cache", cache, block_size)
        kind = _TYPES.get(str(cache.dtype))
        if kind not in (0, 1, 2):
            raise ValueError(f"a paged cache must be bfloat16, float16 or float8_e4m3fn, not {cache.dtype}")
        size = cache.element_size()
        if cache.ndim == 5:
            _, blocks, _, heads, width = cache.shape
            strides, apart = (cache.stride(1), cache.stride(2), cache.stride(3)), cache.stride(0)
        else:
            blocks, heads, _, both = cache.shape
            if both % 2:
                raise ValueError("a cache's last axis must hold a key and a value of one width")
            width = apart = both // 2
            strides = cache.stride(0), cache.stride(2), cache.stride(1)
        if width % 16 or not 0 < width <= 256 or not blocks or not heads:
            raise ValueError(f"a cache's width must be a multiple of 16 up to 256 and its axes not empty, not "
                             f"{described['shape']} of {blocks} blocks")
        address = cache.data_ptr()
        if address % 16 or any(stride * size % 16 for stride in (*strides, apart)):
            raise ValueError("a paged cache's rows must be 16-byte aligned")
        if (scales is not None) != (kind == 2):
            raise ValueError("an e4m3 cache needs scales, and no other takes them")
        scale_strides = (0, 0, 0)
        if scales is not None:
            if str(scales.dtype) not in ("torch.float8_e8m0fnu", "torch.uint8") or (
                    tuple(scales.shape) != (blocks, heads, 2)):
                raise ValueError(f"scales must be float8_e8m0fnu [{blocks}, {heads}, 2], not {scales.dtype} "
                                 f"{list(scales.shape)}")
            if scales.device != cache.device:
                raise ValueError("a cache's scales must be on its device")
            scale_strides = scales.stride()
        self.cache, self.scales, self.block_size = cache, scales, block_size
        self.blocks, self.heads, self.width, self.device = blocks, heads, width, cache.device
        self._kind = kind
        self._layer = _Layer(address, address + apart * size, scales.data_ptr() if scales is not None else None,
                             *strides, *scale_strides, blocks, block_size, heads, width, kind)
        self._layer_at = C.addressof(self._layer)

    def _sequences(self, tokens, block_tables, lengths, query_starts):
        """The kernels' description of the step's tables, and the tables."""
        if block_tables.ndim != 2 or lengths.ndim != 1 or block_tables.shape[0] != lengths.shape[0]:
            raise ValueError(f"block_tables must be [sequences, blocks] and lengths [sequences], not "
                             f"{list(block_tables.shape)} and {list(lengths.shape)}")
        tables = (block_tables, lengths) if query_starts is None else (block_tables, lengths, query_starts)
        if any(str(t.dtype) != "torch.int32" for t in tables):
            raise ValueError("block_tables, lengths and query_starts must be int32")
        if any(t.stride(-1) != 1 and t.shape[-1] > 1 for t in tables):
            raise ValueError("block_tables, lengths and query_starts must be contiguous along their last axis")
        count, wide = block_tables.shape
        if query_starts is None:
            if tokens != count:
                raise ValueError(f"{tokens} rows for {count} sequences of one row each: query_starts is needed")
        elif query_starts.ndim != 1 or query_starts.shape[0] != count + 1:
            raise ValueError(f"query_starts must be [{count + 1}], not {list(query_starts.shape)}")
        return _SEQUENCES(block_tables.data_ptr(), lengths.data_ptr(),
                          0 if query_starts is None else query_starts.data_ptr(), block_tables.stride(0), wide,
                          count), tables

    def append(self, key, value, block_tables, lengths, *, query_starts=None, query=None, positions=None, rotary=None,
               axes=None, interleaved=False, query_out=None):
        """Put a step's ``key`` and ``value`` ([rows, heads, width], bfloat16 or float16) into the slots of their
        sequences' last tokens, in one launch, and return ``query`` ([rows, query heads, width]) turned like the keys
        (into ``query_out`` if given, which may be ``query``; None without a query).

        With ``rotary`` keys and queries are turned by ``positions`` as :func:`rotate` does; without positions a
        token's is its place in its sequence.  A 16-bit cache must have the keys' type.  Into an e4m3 cache a block's
        new values go by the least power of two that keeps them within e4m3's range, or by the block's own where
        slots filled before need more; where the new ones need more, the filled slots are rounded again.  Values that
        are not finite are stored as NaN.  Slots past the length stay as they are, and so do the rows of
        ``query_out`` that are padding.  Sequences of one call must not share a block that it writes.
        """
        import torch
        _rows("key", key, None, self.heads, self.width)
        tokens = key.shape[0]
        _rows("value", value, tokens, self.heads, self.width)
        dtype = key.dtype
        kind = _TYPES.get(str(dtype))
        if kind not in (0, 1) or value.dtype != dtype or (self._kind != 2 and kind != self._kind):
            raise ValueError(f"keys and values must both be bfloat16 or float16, a 16-bit cache's own type: "
                             f"{key.dtype} and {value.dtype} into {self.cache.dtype}")
        sequences, tensors = self._sequences(tokens, block_tables, lengths, query_starts)
        rotation, more = _rotation(rotary, positions, tokens, self.width, axes, interleaved, False)
        heads, rows = 0, (0, 0, 0)
        out = (0, 0, 0)
        if query is not None:
            _rows("query", query, tokens, None, self.width)
            if query.dtype != dtype:
                raise ValueError("query must have the keys' type")
            heads = query.shape[1]
            if query_out is None:
                query_out = torch.empty(query.shape, dtype=dtype, device=query.device)
            else:
                _rows("query_out", query_out, tokens, heads, self.width)
                if query_out.dtype != dtype:
                    raise ValueError("query_out must have the query's type")
            rows = query.data_ptr(), query.stride(0), query.stride(1)
            out = query_out.data_ptr(), query_out.stride(0), query_out.stride(1)
            tensors = (*tensors, query, query_out)
        elif query_out is not None:
            raise ValueError("query_out needs a query")
        _on_gpu(self.device, key, value, *tensors, *more)
        lib = kernel_library()
        _launch(self.device, lambda stream: _check(lib, lib.kvsnap_append(
            self._layer_at, sequences, rotation, key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
            value.stride(0), value.stride(1), *rows, *out, tokens, heads, kind, stream)))
        return query_out

    def attend(self, query, block_tables, lengths, *, query_starts=None, max_length=None, softmax_scale=None,
               window=None, out=None, return_lse=False):
        """Attention of a step's ``query`` rows ([rows, query heads, width], bfloat16 or float16) over their
        sequences' tokens in the cache, the step's own included: ``[rows, query heads, width]`` of the query's type
        (``out`` if given).

        Query heads are a multiple of the cache's; consecutive ones share a key head.  A row at position p sees the
        tokens 0 to p of its sequence, with ``window`` the last ``window`` of them, itself among them; a row that
        sees none (a sequence of length 0) gets zeros.  Scores are ``softmax_scale`` (``width ** -0.5`` if None)
        times the products; softmax and sums are fp32.  A 16-bit cache must have the query's type.

        ``max_length``, the longest sequence's length if the caller knows it (the tables' width if None), only shapes
        the launch.  With ``return_lse`` the result is ``(out, lse)``: fp32 ``[rows, query heads]`` natural
        logarithms of the rows' sums of exponentials (-inf for a row that sees nothing), by which attention over
        parts of the tokens can be joined.
        """
        import torch
        _rows("query", query, None, None, self.width)
        tokens, heads, _ = query.shape
        dtype = query.dtype
        kind = _TYPES.get(str(dtype))
        if kind not in (0, 1) or (self._kind != 2 and kind != self._kind):
            raise ValueError(f"queries must be bfloat16 or float16, a 16-bit cache's own type: {dtype} over "
                             f"{self.cache.dtype}")
        if heads % self.heads or not heads:
            raise ValueError(f"{heads} query heads do not share the cache's {self.heads}")
        if window is not None and window < 1:
            raise ValueError("a window holds at least the row's own token")
        scale = self.width ** -0.5 if softmax_scale is None else softmax_scale
        if not 0 < scale < 1e30:
            raise ValueError("softmax_scale must be positive and finite")
        sequences, tensors = self._sequences(tokens, block_tables, lengths, query_starts)
        named = block_tables.shape[1] * self.block_size
        if max_length is None or max_length > named:
            max_length = named
        elif max_length < 0:
            raise ValueError("max_length must not be negative")
        if out is None:
            out = torch.empty((tokens, heads, self.width), dtype=dtype, device=query.device)
        else:
            _rows("out", out, tokens, heads, self.width)
            if out.dtype != dtype:
                raise ValueError("out must have the query's type")
        _on_gpu(self.device, query, out, *tensors)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=self.device) if return_lse else None
        lib = kernel_library()
        window = min(window or 0, 1 << 30)
        size = _workspace_bytes(lib, tokens, block_tables.shape[0], query_starts is not None, heads, self.heads,
                                self.width, max_length, window)
        scratch = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        _launch(self.device, lambda stream: _check(lib, lib.kvsnap_attend(
            self._layer_at, sequences, query.data_ptr(), query.stride(0), query.stride(1), out.data_ptr(),
            out.stride(0), out.stride(1), lse.data_ptr() if return_lse else None, tokens, heads, kind, scale, window,
            max_length, scratch.data_ptr() if size else None, size, stream)))
        return (out, lse) if return_lse else out


@lru_cache(maxsize=256)
def _workspace_bytes(lib, *sizes):
    return lib.kvsnap_attend_workspace_bytes(*sizes)
