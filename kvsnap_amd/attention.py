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

The kernels' contract is in ``include/kvsnap_attention.h``; arguments are checked in ``csrc/binding.cpp``.  No
gradient is recorded: a tensor that requires one is refused outside ``torch.no_grad()``, and one that carries a
forward-mode tangent is refused.
"""
from __future__ import annotations

import ctypes as C

from .layout import describe_layer
from .native import attention_binding

__all__ = ["PagedCache", "block_scales", "rotary_table", "rotate"]

#: Type codes of include/kvsnap_attention.h by torch type name.
_TYPES = {"torch.bfloat16": 0, "torch.float16": 1, "torch.float8_e4m3fn": 2}


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
    """Scales of e4m3 caches of ``layers`` layers: one tensor with a row of whole 16-byte words a block, which a plane
    saves with the block (``TorchBlockDataPlane(..., scales=...)``), and its ``[blocks, heads, 2]`` view for each
    layer's :class:`PagedCache`."""
    import torch
    used = layers * heads * 2
    rows = torch.zeros((blocks, -(-used // 16) * 16), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    return rows, [rows[:, at:at + 2 * heads].unflatten(1, (heads, 2)) for at in range(0, used, 2 * heads)]


def rotate(x, positions, rotary, *, axes=None, interleaved=False, inverse=False, out=None):
    """``x`` ([tokens, heads, width], bf16, fp16 or fp32) with each pair of a head's values turned by the angle of its
    token's position: (a, b) becomes (a cos - b sin, b cos + a sin), in fp32 and rounded once.

    Pair j is values j and j + pairs of a head, or with ``interleaved`` 2j and 2j + 1; values past the table's pairs
    are copied.  ``positions`` (int64 or int32) is ``[tokens]``, or ``[axes, tokens]`` for positions of several axes
    (time, height and width, say), where ``axes`` names the axis of each pair.  A position outside ``rotary``'s rows
    has no angle and gives NaN.  ``inverse`` turns the other way: it undoes a rotation, gives its gradient, and moves
    kept keys to earlier positions.  ``out`` (a new tensor if None) may be ``x`` itself, and otherwise overlaps no part
    of it.
    """
    return attention_binding().rotate(x, positions, rotary, axes, interleaved, inverse, out)


class PagedCache:
    """One layer's paged KV cache, as a plane registers it, for the operators that fill and read it.

    ``cache`` is a ``[blocks, heads, tokens, 2 * width]`` view (each token's key, then its value: vLLM's layout) or a
    K/V-split ``[2, blocks, tokens, heads, width]`` tensor of ``block_size`` token slots a block, in bfloat16,
    float16 or float8_e4m3fn; widths are multiples of 16 up to 256.  An e4m3 cache comes with ``scales``
    (float8_e8m0fnu or uint8 ``[blocks, heads, 2]``, K's and V's, see :func:`block_scales`): a stored value stands
    for itself times its block and head's power of two (to be appended to, a byte of its own).  The cache is kept,
    not copied.

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
        scale_strides, self._shared = (0, 0, 0), False
        if scales is not None:
            if str(scales.dtype) not in ("torch.float8_e8m0fnu", "torch.uint8") or (
                    tuple(scales.shape) != (blocks, heads, 2)):
                raise ValueError(f"scales must be float8_e8m0fnu [{blocks}, {heads}, 2], not {scales.dtype} "
                                 f"{list(scales.shape)}")
            if scales.device != cache.device:
                raise ValueError("a cache's scales must be on its device")
            scale_strides = scales.stride()
            covered = 0         # by the nearer axes: each block, head and side needs a byte of its own to be appended
            for stride, count in sorted(zip(scale_strides, scales.shape)):
                if count > 1:
                    self._shared = self._shared or stride <= covered
                    covered += (count - 1) * stride
        self.cache, self.scales, self.block_size = cache, scales, block_size
        self.blocks, self.heads, self.width, self.device = blocks, heads, width, cache.device
        self._kind = kind
        self._layer = _Layer(address, address + apart * size, scales.data_ptr() if scales is not None else None,
                             *strides, *scale_strides, blocks, block_size, heads, width, kind)
        self._layer_at = C.addressof(self._layer)
        self._call = attention_binding()

    def append(self, key, value, block_tables, lengths, *, query_starts=None, query=None, positions=None, rotary=None,
               axes=None, interleaved=False, query_out=None):
        """Put a step's ``key`` and ``value`` ([rows, heads, width], bfloat16 or float16) into the slots of their
        sequences' last tokens, in one launch, and return ``query`` ([rows, query heads, width]) turned like the keys
        (into ``query_out`` if given, which may be ``query`` and otherwise overlaps nothing that is read; None without a
        query).

        With ``rotary`` keys and queries are turned by ``positions`` as :func:`rotate` does; without positions a
        token's is its place in its sequence.  A 16-bit cache must have the keys' type.  Into an e4m3 cache a block's
        new values go by the least power of two that keeps them within e4m3's range, or by the block's own where
        slots filled before need more; where the new ones need more, the filled slots are rounded again.  Values that
        are not finite are stored as NaN.  Slots past the length stay as they are, and so do the rows of
        ``query_out`` that are padding (in a new tensor they hold anything).  The pages that one call writes must name
        a block only once, in one sequence and in all of them.
        """
        if self._shared:
            raise ValueError("the cache's scales share bytes among blocks, heads or K and V: none can be appended to")
        return self._call.append(self._layer_at, self.cache, key, value, block_tables, lengths, query_starts, query,
                                 positions, rotary, axes, interleaved, query_out)

    def attend(self, query, block_tables, lengths, *, query_starts=None, max_length=None, softmax_scale=None,
               window=None, out=None, return_lse=False):
        """Attention of a step's ``query`` rows ([rows, query heads, width], bfloat16 or float16) over their
        sequences' tokens in the cache, the step's own included: ``[rows, query heads, width]`` of the query's type
        (``out`` if given, which may be ``query`` and otherwise overlaps no part of it).

        Query heads are a multiple of the cache's; consecutive ones share a key head.  A row at position p sees the
        tokens 0 to p of its sequence, with ``window`` the last ``window`` of them, itself among them; a row that
        sees none (a sequence of length 0), or scores of -inf alone, gets zeros, and rows of ``out`` that are padding
        stay as they are (in a new tensor, and in ``lse``, they hold anything).  Scores are
        ``softmax_scale`` (``width ** -0.5`` if None) times the products; softmax and sums are fp32.  A 16-bit cache
        must have the query's type.

        ``max_length``, the longest sequence's length if the caller knows it (the tables' width if None), only shapes
        the launch.  With ``return_lse`` the result is ``(out, lse)``: fp32 ``[rows, query heads]`` natural
        logarithms of the rows' sums of exponentials (-inf for a row that sees nothing), by which attention over
        parts of the tokens can be joined.
        """
        return self._call.attend(self._layer_at, self.cache, query, block_tables, lengths, query_starts, max_length,
                                 softmax_scale, window, out, return_lse)
