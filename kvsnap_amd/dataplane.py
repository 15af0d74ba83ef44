"""The KV snapshot data plane on MI355X: save gather, restore scatter, and the pinned pool they use.

Drop-in for the reference's ``kvsnap/connector/dataplane.py`` (same classes,
method names, argument meaning, return values and errors), over this
package's HIP library ``_native/libkvsnap_hip.so``:

* ``CudaPool`` / ``PinnedAllocation`` (module ``pool``) bind the pinned pool
  C-ABI version 2 (reference ``dataplane.py:38-211``).
* ``copy_host_blocks`` keeps the reference restore kernel's launch contract
  (six int64 device tensors, launched on the current stream;
  ``copy_kernel.py:43-49``) and runs the HIP restore kernel.
* ``TorchBlockDataPlane`` registers the KV caches and moves records
  (reference ``dataplane.py:214-440``).  The save gathers on the GPU with one
  HIP kernel into device staging, zeroes the tail token slots there, and
  copies the records to pinned memory with the pool's DMA copies; it can also
  hand back per-record SHA-256 and CRC32C computed on the GPU from the same
  staging.  The restore reads pinned records in place with the HIP restore
  kernel, as the reference's does.

There is no CPU fallback: without the HIP library every copy path raises.
"""
from __future__ import annotations

import atexit
import ctypes as C
from collections import deque
from contextlib import contextmanager, nullcontext
import logging
import os
import threading
import time

from .native import (HIP_LIBRARY_NAME, NATIVE, HostStaging, check as _check, drain as _drain, kernel_library,
                     resolve_cuda_library)
from .layout import describe_layer, describe_scales, layout_identity
from .pool import CopyFailed, CudaPool, HipPool, PinnedAllocation, PinnedCapacityError, drop, hold, settle_readers

logger = logging.getLogger(__name__)

__all__ = ["CopyFailed", "CudaPool", "HipPool", "PinnedAllocation", "PinnedCapacityError", "TorchBlockDataPlane",
           "copy_host_blocks", "gather_blocks", "scatter_blocks", "resolve_cuda_library", "kernel_library",
           "HIP_LIBRARY_NAME", "NATIVE"]

#: Default restore grid: workgroups of 256 lanes, each with 32 KiB of 16-byte
#: reads in flight.  Twelve fill the host link (21.3 ms for 1.2 GB, as fast as
#: 32 or 64) and leave the rest of the chip alone: with 64, the 2 MiB of host
#: reads in flight held up every other kernel's memory reads behind them, and
#: a save's SHA-256 chain, whose producer waves read the records, took 52 ms
#: in the step against 47 ms with 12 or 32.
RESTORE_PROGRAMS = int(os.environ.get("KVSNAP_RESTORE_PROGRAMS", "12"))
#: Default grid of the gather and of the copy-engine restore's scatter (0: sized
#: to the work, one wave per KiB of a span; a number: that many workgroups,
#: each taking (block, span) jobs in turn).
GATHER_PROGRAMS = int(os.environ.get("KVSNAP_GATHER_PROGRAMS", "0"))
#: How a save reaches pinned memory: "staged" (device staging + DMA copies)
#: or "direct" (the gather kernel writes pinned memory itself).
SAVE_MODE = os.environ.get("KVSNAP_SAVE_MODE", "staged")
#: "shared": restores run on the pool's copy stream, serialized with saves (as
#: the reference does); "split": restores get a stream of their own, so a
#: restore's host-to-device reads overlap a save's device-to-host copies.
RESTORE_STREAM = os.environ.get("KVSNAP_RESTORE_STREAM", "shared")
#: Hash streams (each with a :class:`HashLane`) the saves rotate over.  A
#: save's SHA-256 takes as long as one record's chain (~36 ms for 2.25 MiB
#: records) however many records there are, and a lane runs every save
#: hashing on it in the same launches, so one stream keeps up with a save
#: every 26 ms (saves and restores overlapped on the link) and takes one
#: hardware queue: with HIP's default four, the engine's stream, the copy
#: stream, a restore stream and the hashes each get their own.
HASH_STREAMS = int(os.environ.get("KVSNAP_HASH_STREAMS", "1"))
#: How a restore moves records over the link: "dma" (the copy engines stage
#: each chunk into device memory, then the scatter kernel places it) or
#: "kernel" (the restore kernel reads pinned memory in place, as the
#: reference's does).  Alone the kernel is about 1 % faster (21.3 against
#: 21.55 ms for 1.2 GB); beside a decode its waves wait out the link's latency
#: on CUs the decode needs (a decode step 1.4x as long), while "dma" leaves
#: the CUs to it, and beside a save's device-to-host copies "dma" can use both
#: directions of the link at once when the runtime gives the restore stream
#: another copy engine than the copy stream's.  A serving engine decodes
#: beside its restores, so "dma" is the default.
RESTORE_MODE = os.environ.get("KVSNAP_RESTORE_MODE", "dma")
#: SHA-256 compressions per hash launch (0: a save's whole chain in one).  A
#: launch holds its hardware queue until it ends, and HIP maps a process's
#: streams onto a few hardware queues, so an unrelated stream sharing the hash
#: stream's queue would wait out a whole chain (~36 ms for 2.25 MiB records).
#: 1440 compressions take about 1.4 ms; at most two are queued at a time.
HASH_SLICE_BLOCKS = int(os.environ.get("KVSNAP_HASH_SLICE_BLOCKS", "1440"))
#: Device staging of a save without digests, per gather-and-copy round (the
#: reference stages 64 MiB at a time).  Each round's gather waits for the
#: copy before it to free the staging; with 64 MiB rounds the link idled
#: between 19 of them and an 8k-token Qwen3-8B save took 22.25 ms; 512 MiB
#: takes three rounds.  An explicit ``chunk_bytes`` still decides.
SAVE_CHUNK_BYTES = int(os.environ.get("KVSNAP_SAVE_CHUNK_BYTES", str(512 << 20)))
#: A lead-stream save's first chunk (below), at most its ``chunk_bytes``.
LEAD_FIRST_BYTES = 64 << 20
#: "1": a hashed save gathers its first chunk of records on the copy stream
#: and the rest on a stream of its own (when a hardware queue is free for it),
#: so the first device-to-host copy starts after one chunk's gather instead
#: of the whole session's.  For 1.2 GB that frees the save 0.27 ms sooner
#: (21.47-21.49 against 21.75-21.77 ms) for 4-12 us more kernel time, the first
#: chunk's launch having a fixed cost of its own.  "0" (default): one gather,
#: then the copies; under a kernel-trace profiler, which runs the copies as
#: kernels, the gather's time then stays its own.
SAVE_LEAD = os.environ.get("KVSNAP_SAVE_LEAD", "0") == "1"
#: A hashed staged save of at most this many bytes gathers with every record's
#: CRC32C folded in (kvsnap_gather_crc32c: one HBM pass, the hash stream then
#: runs SHA-256 only), where its layout allows (whole-KiB spans).  For a
#: TP = 8 shard's 151 MB it takes 65-68 us, where the gather and then the
#: CRC32C kernel take 79-84 us between them, so the ids are ready sooner; the
#: device-to-host copies wait for its end, 18 us later than for the gather
#: alone.  At full size it would hold those copies back longer (0.50 against
#: 0.37 ms at 1.2 GB), so larger saves gather and take their CRC32Cs on the
#: hash stream beside the copies.  0 turns it off.
GATHER_CRC_MAX_BYTES = int(os.environ.get("KVSNAP_GATHER_CRC_MAX_BYTES", str(384 << 20)))
#: "1" (default): a copy-engine restore places each chunk with the scatter
#: kernel on a stream of its own (when a hardware queue is free for it) while
#: the copy engine goes on to the next chunk, into a second staging slot.
#: "0": each chunk's copy and placement take turns on the restore stream,
#: and the engine idles through every placement.
PLACE_ASIDE = os.environ.get("KVSNAP_PLACE_ASIDE", "1") == "1"
#: Device memory a copy-engine plane reserves at warm_up() for its restores' staging: two slots of up to four
#: 64 MiB launches (``COPY_BATCH``), plus room for their tables and CRC32Cs.  The disk-staged restore's two
#: 128 MiB slots fit in it too.  Held until close(); 0 reserves nothing (every restore then allocates).
DEVICE_STAGING_BYTES = int(os.environ.get("KVSNAP_DEVICE_STAGING_BYTES", str(544 << 20)))
#: A copy-engine restore at the default chunking copies up to COPY_BATCH
#: launches' blocks at a time (each copy boundary costs the engine 9-15 us),
#: all but the last COPY_TAIL launches, which keep one copy each so the early
#: report still comes with at most 128 MiB left.
COPY_BATCH, COPY_TAIL = 4, 3
#: Copies of at most FEW_BLOCKS blocks (kvsnap_copy_few) go in one launch between the cache and pinned memory,
#: with no table uploaded first: unhashed direct saves and "kernel" restores of any size, and, up to FEW_BYTES,
#: staged saves and "dma" restores too.  Through the copy engine a 295 KB save took 190 us and a 4.6 MB restore
#: 157, against 5 and 80 on the link; a kernel and the engine move 4.6 MB equally fast (98 us), and a launch of
#: this size gives the CUs back within 0.15 ms, where a longer one beside a decode would hold them.  Records off
#: the 8-byte boundaries go the general way.
FEW_BLOCKS = 128
FEW_BYTES = int(os.environ.get("KVSNAP_FEW_BYTES", str(8 << 20)))
#: A hashed save of at most RECORDS_PER_HASH_THREAD records a thread hashes them on the host (kvsnap_hash_records),
#: on up to HASH_THREADS threads (and CPUs this process may use; 0 turns it off, and so does SAVE_LEAD, whose
#: gather over two streams is for GPU-hashed saves), from the pinned records as they land; the save returns when
#: they have.  A record's SHA-256 chain takes the GPU 36 ms for 2.25 MiB however few records there are; a host
#: thread with the SHA instructions hashes 3.4 GB/s of them, 26 GB/s on eight.  32 such records: the save returns
#: after 1.5 ms and the ids are there after 3.9, against 36.6; 128 of 0.9 MiB, 2.4 and 5.2 against 16.5.  Past
#: sixteen a thread the host takes a third of the chain's time or more (half at 25), and the GPU hashes beside the
#: copies without holding the host's cores.
HASH_THREADS = int(os.environ.get("KVSNAP_HASH_THREADS", "8"))
RECORDS_PER_HASH_THREAD = 16
#: Streams the plane tries, at most, while looking for hardware queues that
#: none of its other streams (nor the engine's) use.
STREAM_CANDIDATES = 12
#: Copies that keep the engines already tied to the plane's streams busy
#: while a new restore stream takes its engine (about 4.5 ms each at the
#: link's rate; 16 MiB copies, 0.3 ms, were over before the new stream's
#: first copy was issued, which then took the same engine).
ENGINE_BUSY_BYTES = 256 << 20
#: Candidate restore streams tried at most, and the pair time (a copy each way at once, as a fraction of the
#: two in turn) at which the search stops: 0.594-0.601 for the engines that carried overlapped saves and
#: restores fastest, 0.605-0.608 for one that carried them 15 % slower.
ENGINE_TRIES = 4
ENGINE_OVERLAP = 0.6
#: Copies that time a candidate restore stream's engine, each way.
ENGINE_PROBE_BYTES = 64 << 20
#: Length of the hold that tells which streams share a hardware queue, in
#: s_sleep rounds of about 3.4 us: about 3.4 ms.
HOLD_ITERS = 1000


def _source_addresses(sources, size, what="load source"):
    """The address of each ``(allocation, offset)`` source of ``size`` bytes, every allocation checked open
    (once per run of sources in one allocation) and every source inside its allocation."""
    addresses, last = [], None
    for allocation, offset in sources:
        if allocation is not last:
            allocation._open()
            last, base, end = allocation, allocation.pointer, allocation.size - size
        if offset < 0 or offset > end:
            raise ValueError(f"{what} outside its allocation")
        addresses.append(base + offset)
    return addresses


def _word_aligned(addresses):
    """Whether every record starts on the 8-byte boundary that the copy kernels' accesses want.  A reservation
    behind one of an odd size does not; the copy engine takes any address."""
    return not any(address & 7 for address in addresses)


def _runs(addresses, size, first=0):
    """(index, count) of each run of consecutive ``size``-byte records in ``addresses``."""
    runs, i = [], 0
    while i < len(addresses):
        j = i + 1
        while j < len(addresses) and addresses[j] == addresses[j - 1] + size:
            j += 1
        runs.append((first + i, j - i))
        i = j
    return runs


def _target_bounds(targets, size):
    """``(allocation, low, high)`` for each allocation of ``targets``: the bytes its records lie within."""
    bounds = {}
    for allocation, offset in targets:
        _, low, high = bounds.get(id(allocation), (allocation, offset, offset))
        bounds[id(allocation)] = (allocation, min(low, offset), max(high, offset + size))
    return list(bounds.values())


def _target_runs(targets, first, end, size):
    """``[index, count, allocation, offset]`` for each run of targets ``first..end-1`` whose records sit back
    to back in one allocation: one device-to-host copy each (reference ``dataplane.py:418-427``)."""
    runs = []
    for index in range(first, end):
        allocation, offset = targets[index]
        if runs and runs[-1][2] is allocation and runs[-1][3] + runs[-1][1] * size == offset:
            runs[-1][1] += 1
        else:
            runs.append([index, 1, allocation, offset])
    return runs


def _parts(first, end, part):
    """[first, end) in parts, each twice as long as the one before; a rest of less than half a part joins the
    last.  Hashed about half as fast as they are copied, records in such parts keep the hashes going behind the
    copies with few launches.  (A launch beside a decode waits for its CUs: in parts of 16 records the rotating
    fp8 sessions copied at 36-38 GB/s, in these at 40.)"""
    parts = []
    while first < end:
        high = min(end, first + part)
        if end - high < part // 2:
            high = end
        parts.append((first, high))
        first, part = high, 2 * part
    return parts


class StagingUnavailable(MemoryError):
    """Device staging for a copy could not be allocated.  Raised before anything was copied into a KV block or a
    pinned target: a load may be recomputed, a save fails with its blocks untouched."""


class _Progress:
    """A restore's ``progress`` list as the connector reads it (reference ``dataplane.py:369-379``):
    ``(None, total bytes)`` once the launches start, then ``(event, bytes left once it completes)`` per
    launch, the event recorded on the launch's stream right after it."""

    def __init__(self, torch, entries, total):
        self.torch, self.entries, self.total = torch, entries, total

    def start(self):
        if self.entries is not None:
            self.entries.append((None, self.total))

    def launched(self, stream, left, *, wait=False):
        if self.entries is None:
            return
        mark = self.torch.cuda.Event()
        mark.record(stream)
        if wait:
            mark.synchronize()
        self.entries.append((mark, left))


class _Landing:
    """A save's work queued on ``stream``, held on the pinned targets that its kernels write: they wait for it
    before they are released."""

    writes = True

    def __init__(self, torch, stream):
        self._event, self._held = torch.cuda.Event(), ()
        self._event.record(stream)

    def synchronize(self):
        self._event.synchronize()

    def finish(self):
        self.synchronize()
        for allocation in self._held:
            drop(self, allocation)

    def query(self):
        return self._event.query()

    def held_on(self, targets):
        self._held = {id(allocation): allocation for allocation, _ in targets}.values()
        for allocation in self._held:
            hold(self, allocation)


@contextmanager
def _drain_on_failure(*streams):
    """If queuing fails part way, wait for what was queued: its launches may still read sources or write
    targets that the caller releases as soon as the exception reaches it."""
    try:
        yield
    except BaseException:
        for stream in streams:
            if stream is not None:
                stream.synchronize()
        raise


def _int64_device_tensors(*tensors):
    """The device of launch tables that are contiguous 1-D int64 CUDA tensors on one device, else ValueError."""
    device = tensors[0].device
    for t in tensors:
        if t.device != device or t.device.type != "cuda":
            raise ValueError("restore tables must be CUDA tensors on one device")
        if str(t.dtype) != "torch.int64" or t.dim() != 1 or not t.is_contiguous():
            raise ValueError("restore tables must be contiguous 1-D int64 tensors")
    return device


def _int32_device_output(t, device, count):
    """A kernel's int32 output: a contiguous CUDA tensor on ``device`` with room for ``count``, else ValueError."""
    if t.device != device or str(t.dtype) != "torch.int32" or not t.is_contiguous() or t.numel() < count:
        raise ValueError(f"the output must be a contiguous int32 CUDA tensor on {device} of at least {count}")


def _current_stream_handle(device):
    """The handle of torch's current stream on ``device``: where the launch contract queues kernels."""
    import torch
    return torch.cuda.current_stream(device).cuda_stream


def copy_host_blocks(sources, blocks, layer_offsets, layer_bases, layer_pitches, layer_words, *, programs=None,
                     min_span_bytes=0):
    """Launch the restore kernel on the current stream.

    ``sources``: address of each packed block (pinned host or device memory);
    ``blocks``: its target block id; the ``layer_*`` tables: per span, its
    offset in a packed block, the cache's base address and block pitch in
    bytes, and its length in 8-byte words.  All int64 CUDA tensors
    (reference ``copy_kernel.py:43-49``).  ``min_span_bytes``, the shortest
    span's length when the caller knows it, only shapes the launch.
    """
    device = _int64_device_tensors(sources, blocks, layer_offsets, layer_bases, layer_pitches, layer_words)
    n_blocks, n_spans = sources.numel(), layer_offsets.numel()
    if blocks.numel() != n_blocks or not (layer_bases.numel() == layer_pitches.numel() == layer_words.numel()
                                          == n_spans):
        raise ValueError("restore table lengths disagree")
    lib = kernel_library()
    _check(lib, lib.kvsnap_restore_blocks(sources.data_ptr(), blocks.data_ptr(), n_blocks, layer_offsets.data_ptr(),
                                          layer_bases.data_ptr(), layer_pitches.data_ptr(), layer_words.data_ptr(),
                                          n_spans, min_span_bytes, RESTORE_PROGRAMS if programs is None else programs,
                                          _current_stream_handle(device)))


def gather_launcher(blocks, layer_offsets, layer_bases, layer_pitches, layer_words, records, record_pitch, *,
                    programs=None, min_span_bytes=0):
    """A zero-argument launch of the gather kernel on the current stream, with its arguments checked now:
    block ``blocks[i]`` packed at ``records + i * record_pitch``."""
    device = _int64_device_tensors(blocks, layer_offsets, layer_bases, layer_pitches, layer_words)
    lib = kernel_library()
    args = (blocks.data_ptr(), blocks.numel(), layer_offsets.data_ptr(), layer_bases.data_ptr(),
            layer_pitches.data_ptr(), layer_words.data_ptr(), layer_offsets.numel(), min_span_bytes, records,
            record_pitch, GATHER_PROGRAMS if programs is None else programs, _current_stream_handle(device))
    return lambda: _check(lib, lib.kvsnap_gather_blocks(*args))


def gather_blocks(blocks, layer_offsets, layer_bases, layer_pitches, layer_words, records, record_pitch, *,
                  programs=None, min_span_bytes=0):
    """Launch the gather kernel on the current stream: block ``blocks[i]`` packed at ``records + i * record_pitch``."""
    gather_launcher(blocks, layer_offsets, layer_bases, layer_pitches, layer_words, records, record_pitch,
                    programs=programs, min_span_bytes=min_span_bytes)()


def gather_crc32c_launcher(blocks, group_bases, group_pitches, record_bytes, records, record_pitch, crcs):
    """A zero-argument launch, on the current stream, of the gather with CRC32C: block ``blocks[i]`` packed at
    ``records + i * record_pitch`` (device memory) and its CRC32C in ``crcs[i]`` (int32 device tensor), from
    one read of the cache.  ``group_bases`` / ``group_pitches``: the source of each 1 KiB group of a record
    (:meth:`TorchBlockDataPlane.group_tables`)."""
    device = _int64_device_tensors(blocks, group_bases, group_pitches)
    _int32_device_output(crcs, device, blocks.numel())
    lib = kernel_library()
    if group_bases.numel() * 1024 != record_bytes or group_pitches.numel() != group_bases.numel():
        raise ValueError("the groups' table does not tile the record")
    args = (blocks.data_ptr(), blocks.numel(), group_bases.data_ptr(), group_pitches.data_ptr(), record_bytes,
            records, record_pitch, crcs.data_ptr(), _current_stream_handle(device))
    return lambda: _check(lib, lib.kvsnap_gather_crc32c(*args))


def scatter_blocks(records, record_pitch, blocks, layer_offsets, layer_bases, layer_pitches, layer_words, *,
                   programs=0, min_span_bytes=0):
    """Launch the scatter kernel on the current stream: the device record at ``records + i * record_pitch``
    into block ``blocks[i]``.  ``programs=0`` sizes the grid to the jobs."""
    device = _int64_device_tensors(blocks, layer_offsets, layer_bases, layer_pitches, layer_words)
    lib = kernel_library()
    _check(lib, lib.kvsnap_scatter_blocks(records, record_pitch, blocks.data_ptr(), blocks.numel(),
                                          layer_offsets.data_ptr(), layer_bases.data_ptr(), layer_pitches.data_ptr(),
                                          layer_words.data_ptr(), layer_offsets.numel(), min_span_bytes, programs,
                                          _current_stream_handle(device)))


class KernelTimer:
    """Per-kernel timing events, recorded on the stream each launch runs on.

    Set ``plane.timer = KernelTimer()`` to time the data plane's launches;
    ``summary()`` waits for the events and returns, per kernel name, the
    launch count and total and mean duration in milliseconds.  With
    ``names``, only those kernels are timed: a pair of timing events around
    every launch costs stream time of its own (about 0.15 ms in a 45 ms
    save-and-restore step with the restore's 19 launches and the hashes'
    range launches all timed).
    """

    def __init__(self, names=None):
        import torch
        self.torch = torch
        self.pairs = {}
        self.names = None if names is None else frozenset(names)

    def wants(self, name):
        return self.names is None or name in self.names

    @contextmanager
    def span(self, name, stream):
        start = self.torch.cuda.Event(enable_timing=True)
        end = self.torch.cuda.Event(enable_timing=True)
        start.record(stream)
        yield
        end.record(stream)
        self.pairs.setdefault(name, []).append((start, end))

    def add(self, name, start, end):
        """A span recorded by the caller (events with timing enabled)."""
        self.pairs.setdefault(name, []).append((start, end))

    def reset(self):
        self.pairs = {}

    def summary(self):
        result = {}
        for name, pairs in self.pairs.items():
            for _, end in pairs:            # a kernel's launches may run on several streams
                end.synchronize()
            times = [start.elapsed_time(end) for start, end in pairs]
            result[name] = {"launches": len(times), "total_ms": sum(times), "avg_ms": sum(times) / len(times)}
        return result


@contextmanager
def _timed(timer, name, stream):
    if timer is None or not timer.wants(name):
        yield
    else:
        with timer.span(name, stream):
            yield


class BlockDigests:
    """Per-block (SHA-256 hex, CRC32C) of a save, computed on the GPU from the save's device staging, or on host
    threads from its pinned records (a :class:`HostHashJob`).

    ``result()`` waits for the hashes (and raises if they failed) and returns
    the list in block order; what they read stays alive until then: the
    staging, or the targets, which close, and take another save or write
    through the pool, only once they have been read.
    """

    def __init__(self, torch, event, crc, sha, keepalive):
        self._torch, self._event, self._crc, self._sha = torch, event, crc, sha
        self._keepalive = keepalive
        self._value = None

    def ready(self):
        return self._value is not None or self._event.query()

    def result(self):
        if self._value is None:
            self._event.synchronize()
            if isinstance(self._event, HostHashJob):
                crcs, sha = self._crc.tolist(), self._sha
            else:
                import numpy as np
                crcs = (self._crc.cpu().numpy().astype(np.int64) & 0xFFFFFFFF).tolist()
                sha = self._sha.cpu().numpy()
            text = sha.tobytes().hex()                         # one pass: [n, 32] bytes -> 64 hex chars each
            self._value = [(text[64 * i:64 * i + 64], crc) for i, crc in enumerate(crcs)]
            self._keepalive = None
        return self._value


def digest_device_records(torch, records_ptr, record_bytes, record_pitch, n, device, stream, timer=None,
                          crc_stream=None):
    """Launch SHA-256 and CRC32C over ``n`` records in device (or pinned) memory.

    SHA-256 goes on ``stream`` first: it is the long one (one sequential chain
    per record) and needs only a few CUs.  CRC32C follows on ``stream``, or
    runs beside it on ``crc_stream``, which then joins back into ``stream``;
    either way work queued on ``stream`` afterwards sees both.  The CRC kernel
    takes a whole CU's LDS per workgroup, so beside copies that run as kernels
    it may wait for CUs, and the SHA chains should not wait behind it.  (A
    separate ``crc_stream`` only pays with hardware queues to spare: streams
    beyond the process's hardware queues share one and run in its order.)
    Returns (crc int32 tensor [n], sha uint8 tensor [n, 32], workspace) on the
    device; the workspace must outlive the launches.
    """
    lib = kernel_library()
    crc = torch.empty(n, dtype=torch.int32, device=device)
    sha = torch.empty((n, 32), dtype=torch.uint8, device=device)
    work_bytes = int(lib.kvsnap_crc32c_workspace_bytes(record_bytes, n))
    workspace = torch.empty(max(work_bytes, 16), dtype=torch.uint8, device=device)
    if crc_stream is not None:
        ready = torch.cuda.Event()
        ready.record(stream)
    with _timed(timer, "sha256", stream):
        _check(lib, lib.kvsnap_sha256_records(records_ptr, record_bytes, record_pitch, n, sha.data_ptr(),
                                              stream.cuda_stream))
    on = stream
    if crc_stream is not None:
        crc_stream.wait_event(ready)
        on = crc_stream
    with _timed(timer, "crc32c", on):
        _check(lib, lib.kvsnap_crc32c_records(records_ptr, record_bytes, record_pitch, n, 0, crc.data_ptr(),
                                              workspace.data_ptr(), work_bytes, on.cuda_stream))
    if crc_stream is not None:
        checked = torch.cuda.Event()
        checked.record(crc_stream)
        stream.wait_event(checked)
    return crc, sha, workspace


#: Saves whose SHA-256 ranges one launch can carry (``kvsnap_sha256_ranges``).
SHA_MAX_RANGES = 8


class HashJob:
    """One save's CRC32C and SHA-256 over ``n`` device records, fed to its stream by ``lane``.

    The lane launches the CRC32C first, then the SHA-256 chains as ranges of
    ``slice_blocks`` compressions (the chaining state carried in a device
    buffer), each launch shared with the other saves hashing on the lane.
    ``synchronize()`` / ``query()`` stand in for the completion event.  The
    lane holds ``keepalive`` (the records' owner) until the last launch that
    reads the records has finished, so their memory returns to the allocator
    only then (no ``record_stream``, whose event would be recorded on the
    hash stream whenever the records are freed, even after the stream is
    gone).
    """

    def __init__(self, torch, records_ptr, record_bytes, record_pitch, n, device, lane, slice_blocks, *,
                 timer=None, keepalive=None, crc=None):
        lib = kernel_library()
        self._torch, self._stream = torch, lane.stream
        self.records = (records_ptr, record_bytes, record_pitch, n)
        # ``crc``: the records' CRC32Cs already computed (by the checked gather) before the event the lane's
        # stream waits on; the lane then launches only the SHA-256 ranges.
        self.crc_given = crc is not None
        self.work_bytes = 0 if self.crc_given else int(lib.kvsnap_crc32c_workspace_bytes(record_bytes, n))
        with torch.cuda.stream(lane.stream):     # the buffers belong to the stream that uses them
            self.crc = crc if self.crc_given else torch.empty(n, dtype=torch.int32, device=device)
            self.sha = torch.empty((n, 32), dtype=torch.uint8, device=device)
            self.state = torch.empty((n, 8), dtype=torch.int32, device=device)
            self.workspace = None if self.crc_given else \
                torch.empty(max(self.work_bytes, 16), dtype=torch.uint8, device=device)
        self.nblocks = int(lib.kvsnap_sha256_blocks(record_bytes))
        self.slice_blocks = slice_blocks if slice_blocks > 0 else self.nblocks
        self.next_block = 0
        self.timer, self.keepalive, self.started = timer, keepalive, None
        self._event, self._error, self._done = None, None, threading.Event()
        lane.submit(self)

    def _finish(self, event=None, error=None):
        if error is None and self.timer is not None and self.started is not None:
            self.timer.add("sha256", self.started, event)
        self._event, self._error, self.keepalive = event, error, None
        self._done.set()

    def finished(self, timeout=None):
        """Whether the job is over (its launches done, or the feeding failed); waits up to ``timeout`` seconds."""
        return self._done.wait(timeout)

    def query(self):
        return self._done.is_set() and (self._error is not None or self._event.query())

    def synchronize(self):
        self._done.wait()
        if self._error is not None:
            raise self._error
        self._event.synchronize()


class HashLane:
    """A hash stream and the one thread that feeds it.

    Every save hashing on the lane shares each launch: its CRC32C goes first,
    then ``kvsnap_sha256_ranges`` carries the next ``slice_blocks``
    compressions of up to ``SHA_MAX_RANGES`` saves' chains at once, with at
    most two launches queued.  A save's SHA-256 is one sequential chain per
    record (about 36 ms for 2.25 MiB records) that needs only a few CUs, so
    saves that arrive together hash side by side on one stream, and one
    hardware queue, instead of one after another.
    """

    def __init__(self, torch, stream):
        self.torch, self.stream = torch, stream
        self._cv = threading.Condition()
        self._incoming, self._closed = [], False
        self._thread = threading.Thread(target=self._run, name="kvsnap-hash", daemon=True)
        self._thread.start()

    def submit(self, job):
        with self._cv:
            if self._closed:
                raise RuntimeError("the data plane is closed")
            self._incoming.append(job)
            self._cv.notify()

    def close(self):
        """Finish every job submitted, then stop the feeding thread."""
        with self._cv:
            self._closed = True
            self._cv.notify()
        self._thread.join()

    def _start(self, lib, job):
        records_ptr, record_bytes, record_pitch, n = job.records
        stream = self.stream
        if not job.crc_given:
            with _timed(job.timer, "crc32c", stream):
                _check(lib, lib.kvsnap_crc32c_records(records_ptr, record_bytes, record_pitch, n, 0,
                                                      job.crc.data_ptr(), job.workspace.data_ptr(), job.work_bytes,
                                                      stream.cuda_stream))
        if job.timer is not None and job.timer.wants("sha256"):
            job.started = self.torch.cuda.Event(enable_timing=True)
            job.started.record(stream)

    def _launch(self, lib, batch):
        """One launch of the next range of every job in ``batch``; returns the event recorded after it."""
        k = len(batch)
        table = [(C.c_uint64 * k)() for _ in range(8)]
        counts = (C.c_int64 * k)()
        for i, job in enumerate(batch):
            records_ptr, record_bytes, record_pitch, n = job.records
            end = min(job.next_block + job.slice_blocks, job.nblocks)
            for column, value in zip(table, (records_ptr, record_bytes, record_pitch, job.next_block, end,
                                             job.state.data_ptr(), job.sha.data_ptr(), 0)):
                column[i] = value
            counts[i] = n
            job.next_block = end
        records, record_bytes, pitches, firsts, ends, states, outs, _ = table
        _check(lib, lib.kvsnap_sha256_ranges(k, records, record_bytes, pitches, counts, firsts, ends, states, outs,
                                              self.stream.cuda_stream))
        timing = any(job.started is not None for job in batch)
        event = self.torch.cuda.Event(enable_timing=timing)
        event.record(self.stream)
        return event

    def _run(self):
        active, queued = [], []          # queued: (event, the jobs whose last launch it follows)
        while True:
            with self._cv:
                while not self._incoming and not active and not queued and not self._closed:
                    self._cv.wait()
                incoming, self._incoming = self._incoming, []
                if not incoming and not active and not queued:
                    return               # closed, and everything submitted is over
            started = []
            try:
                lib = kernel_library()   # loaded once per process; inside the try so a failure fails the jobs
                for job in incoming:
                    self._start(lib, job)
                    started.append(job)
                active += started
                while len(queued) >= 2:
                    event, ended = queued.pop(0)
                    event.synchronize()
                    for job in ended:
                        job._finish(event)
                if active:
                    batch = active[:SHA_MAX_RANGES]
                    event = self._launch(lib, batch)
                    ended = [job for job in batch if job.next_block >= job.nblocks]
                    # Jobs that did not fit this launch go first next time.
                    active = active[SHA_MAX_RANGES:] + [job for job in batch if job.next_block < job.nblocks]
                    queued.append((event, ended))
                if not active:
                    while queued:
                        event, ended = queued.pop(0)
                        event.synchronize()
                        for job in ended:
                            job._finish(event)
            except BaseException as exc:
                try:
                    self.stream.synchronize()        # launches already queued may still read the records
                except BaseException:
                    pass
                failed = [job for job in incoming if job not in started] + started + active
                failed += [job for _, ended in queued for job in ended]
                active, queued = [], []
                for job in dict.fromkeys(failed):
                    if not job.finished(timeout=0):
                        job._finish(error=exc)


class HostHashJob:
    """One save's SHA-256 and CRC32C of its pinned records, on host threads (``kvsnap_hash_records``).

    ``marks`` are ``(first, end, event)``: those records have landed once the
    event has completed.  Whoever comes first does the work: the plane's
    hashing thread (:class:`HostHashes`), for a save that lands in parts, or
    a thread that needs it done, in ``result()`` or to close or overwrite a
    target.  It is held on the targets, so their bytes stay as saved until
    they have been read, and takes no lock of the pool's meanwhile.
    """

    writes = False

    def __init__(self, lib, targets, addresses, size, marks, threads):
        import numpy as np
        n = len(targets)
        self._lib, self._addresses, self._size, self._marks, self._threads = lib, addresses, size, marks, threads
        self.sha, self.crc = np.empty((n, 32), dtype=np.uint8), np.empty(n, dtype=np.uint32)
        self._lock, self._over, self._error = threading.Lock(), False, None      # held by the thread at work
        self._held = _target_bounds(targets, size)
        for allocation, low, high in self._held:
            hold(self, allocation, low, high)

    def finish(self):
        """Hash the records, or wait for the thread that does."""
        if not self._over:
            with self._lock:
                if not self._over:
                    self._hash()

    def _hash(self):
        try:
            at = 0
            while at < len(self._marks):
                first, end, event = self._marks[at]
                event.synchronize()
                at += 1
                while at < len(self._marks) and self._marks[at][2].query():   # hashing is slower than copying:
                    end, at = self._marks[at][1], at + 1                       # take what has landed meanwhile
                records = (C.c_uint64 * (end - first))(*self._addresses[first:end])
                _check(self._lib, self._lib.kvsnap_hash_records(records, self._size, end - first,
                                                                self.sha[first:].ctypes.data,
                                                                self.crc[first:].ctypes.data, self._threads))
        except BaseException as exc:
            self._error = exc
        finally:
            for allocation, _, _ in self._held:
                drop(self, allocation)
            self._held = self._marks = ()
            self._over = True

    def query(self):
        return self._over

    def synchronize(self):
        self.finish()
        if self._error is not None:
            raise self._error


class HostHashes:
    """The thread that runs a plane's :class:`HostHashJob`s, in turn, from its first one until ``close()``.  A
    process that ends without closing its plane finishes them first (nothing may read the pinned arena while the
    runtime goes away)."""

    def __init__(self):
        self._cv, self._pid = threading.Condition(), os.getpid()
        self._jobs, self._closed = deque(), False
        self._thread = threading.Thread(target=self._run, name="kvsnap-host-hash", daemon=True)
        self._thread.start()
        atexit.register(self.close)

    def submit(self, job):
        with self._cv:
            if not self._closed:       # else it runs when its digests are asked for
                self._jobs.append(job)
                self._cv.notify()

    def close(self):
        """Finish every job submitted, then stop the thread."""
        if os.getpid() != self._pid:
            return                     # a forked child's copy: the thread is the parent's
        with self._cv:
            self._closed = True
            self._cv.notify()
        self._thread.join()
        atexit.unregister(self.close)

    def _run(self):
        while True:
            with self._cv:
                while not self._jobs and not self._closed:
                    self._cv.wait()
                if not self._jobs:
                    return
                job = self._jobs.popleft()
            job.finish()
            del job


def report_engine_pick(check):
    """Warn when no candidate restore stream paired with the copy stream's engine as the fast engines do
    (``check`` as :attr:`TorchBlockDataPlane.restore_stream_check` holds it): restores and saves at once then
    share the host link less well from this plane.  Returns whether it warned."""
    if check is None or check.get("accepted", True):
        return False
    logger.warning("copy-engine restore stream: no candidate overlapped the copy stream's engine as the fast "
                   "engines do (kept %.1f GB/s both ways; candidates %s GB/s); overlapped saves and restores "
                   "from this plane will share the host link less well.  A process's first plane has the "
                   "best chance of such a pair (restore_stream_check in stream_report()).",
                   check.get("both_ways_gbps", 0.0), check.get("tried_both_ways_gbps", []))
    return True


class TorchBlockDataPlane:
    """Packed physical blocks: layer-name order, dense per-block spans.

    Accepts the reference's layout, a [blocks, H, N, C] view per layer whose
    block is one dense span under any H/N stride permutation (reference
    ``dataplane.py:221-249``), and also a [2, blocks, N, H, C] K/V-split cache
    per layer, whose layer segment of a record is its K span followed by its
    V span.  The actual layout is recorded in ``layers`` (the snapshot
    identity); unsupported views fail closed.

    ``scales`` are the scales of e4m3 caches that :class:`kvsnap_amd.attention.PagedCache` fills: one row of bytes a
    block for all layers (``kvsnap_amd.attention.block_scales``).  A block's row is saved and restored with its block,
    behind the layers in its record, and named in the identity.
    """

    def __init__(self, caches, block_size, capacity_bytes, *, restore_programs=None, gather_programs=None,
                 save_mode=None, restore_stream=None, restore_mode=None, device_staging_bytes=None, scales=None):
        import torch
        if not caches:
            raise ValueError("empty KV cache registration")
        options = {"save_mode": (save_mode or SAVE_MODE, ("staged", "direct")),
                   "restore_stream": (restore_stream or RESTORE_STREAM, ("shared", "split")),
                   "restore_mode": (restore_mode or RESTORE_MODE, ("kernel", "dma"))}
        for option, (value, allowed) in options.items():
            if value not in allowed:
                raise ValueError(f"{option} must be one of {', '.join(allowed)}, not {value!r}")
        self.torch = torch
        self.block_size = block_size
        # Sorted by layer name: the order of the layers' spans in every record.
        self.caches = {name: caches[name] for name in sorted(caches)}
        device = next(iter(self.caches.values())).device
        if device.type != "cuda" or any(tensor.device != device for tensor in self.caches.values()):
            raise ValueError("every KV cache must be on one and the same CUDA device")
        self.layers = [describe_layer(name, tensor, block_size) for name, tensor in self.caches.items()]
        self.scales = scales
        if scales is not None:
            if scales.device != device:
                raise ValueError("the scales must be on the KV caches' device")
            self.layers.append(describe_scales(scales))
        self.block_bytes = sum(layer["bytes"] for layer in self.layers)
        self.restore_programs = RESTORE_PROGRAMS if restore_programs is None else restore_programs
        self.gather_programs = GATHER_PROGRAMS if gather_programs is None else gather_programs
        self.save_mode = options["save_mode"][0]
        self.restore_stream_mode = options["restore_stream"][0]
        self.restore_mode = options["restore_mode"][0]
        self.timer = None       # a KernelTimer, to time this plane's launches
        # Guards the lazily built streams and tables: the connector calls a plane from its save threads and
        # its loader thread at once (reference vllm.py:202-203).
        self._state_lock = threading.RLock()
        self._split_stream = None
        self.restore_stream_check = None    # what picking a copy-engine restore stream measured
        self._hash_stream_list = None
        self._hash_queues_own = None        # were the hash streams found on hardware queues of their own
        self._aside = None                  # the lead save's later gathers and the copy-engine placements
        self._aside_picked = False
        self._digest_next = 0
        self._hash_lanes = None
        self._owned_streams = []
        self._host_staging = HostStaging(torch)
        if device_staging_bytes is None:
            device_staging_bytes = DEVICE_STAGING_BYTES if self.restore_mode == "dma" else 0
        if type(device_staging_bytes) is not int or device_staging_bytes < 0:
            raise ValueError("device_staging_bytes must be a non-negative byte count")
        self.device_staging_bytes = device_staging_bytes
        self._reserved_staging = None       # allocated by warm_up(): the restores' device staging
        self._reserved_lock = threading.Lock()
        self._host_hashes = None            # the thread that hashes few-record saves' pinned records
        self._tails = {}                    # token slots kept -> the last record's tail regions
        self.pool = CudaPool(capacity_bytes, device.index)

    @property
    def _device(self):
        return next(iter(self.caches.values())).device

    def _upload(self, host, values, stream):
        """``values`` as an int64 device tensor, through the borrowed pinned buffer ``host``, on ``stream``."""
        return self._host_staging.upload_int64(host, values, self._device, stream, kernel_library())

    @property
    def layout_identity(self):
        """The registered layout as the snapshot identity string (reference ``vllm.py:236``)."""
        return layout_identity(self.layers)

    def paged_cache(self, name, *, scales=None):
        """The registered cache ``name`` for the operators that fill and read it (``kvsnap_amd.attention``); an e4m3
        one with its layer's ``scales``, a view of the rows that the plane saves with its blocks."""
        from .attention import PagedCache
        cache = PagedCache(self.caches[name], self.block_size, scales=scales)
        if scales is not None:
            rows = self.scales
            if rows is None:
                raise ValueError(f"KV cache {name!r}: the plane was registered without scales and would save its blocks "
                                 "without theirs")
            first = scales.data_ptr() - rows.data_ptr()
            used = sum((size - 1) * stride for size, stride in zip(scales.shape[1:], scales.stride()[1:])) + 1
            if (first < 0 or first + used > rows.shape[1] or scales.shape[0] > rows.shape[0]
                    or scales.stride(0) != rows.stride(0)):
                raise ValueError(f"KV cache {name!r}: the scales are no view of the plane's own: its blocks would be "
                                 "saved and restored without them")
        return cache

    def _num_blocks(self, tensor):
        return tensor.shape[1] if tensor.ndim == 5 else tensor.shape[0]

    def _validate_ids(self, ids):
        """Every id must name a block of every cache (reference dataplane.py:251-254): one pass against the
        smallest cache's block count."""
        limit = getattr(self, "_block_limit", None)
        if limit is None:
            limit = min(self._num_blocks(t) for t in self.caches.values())
            if getattr(self, "scales", None) is not None:
                limit = min(limit, self.scales.shape[0])
            self._block_limit = limit
        # C-level passes: a generator over 512 ids took 0.08 ms of a restore's 0.4 ms before its first launch.
        if ids and (not set(map(type, ids)) <= {int} or min(ids) < 0 or max(ids) >= limit):
            raise ValueError("GPU block id out of range")

    def producer_event(self):
        """An event recorded now on the engine's current stream."""
        event = self.torch.cuda.Event()
        event.record(self.torch.cuda.current_stream(next(iter(self.caches.values())).device))
        return event

    def wait_on_engine_stream(self, event):
        """Make the engine's current stream wait, on the GPU, for ``event``."""
        self.torch.cuda.current_stream(next(iter(self.caches.values())).device).wait_event(event)

    @contextmanager
    def staging(self, nblocks):
        """Pinned room for ``nblocks`` packed records, handed back to the pool (once its copies are proven
        complete) when the ``with`` block ends."""
        buffer = self.pool.reserve(nblocks * self.block_bytes)
        try:
            yield buffer
        finally:
            buffer.close()

    # ------------------------------------------------------------------ geometry

    def spans(self):
        """Per span: (record offset, base address of block 0, block pitch, bytes); 8-byte aligned."""
        if getattr(self, "_span_table", None) is None:
            spans, offset = [], 0
            for layer, tensor in zip(self.layers, self.caches.values()):
                esize = tensor.element_size()
                if tensor.ndim == 5:
                    half = layer["bytes"] // 2
                    parts = [(offset, tensor.data_ptr(), tensor.stride(1) * esize, half),
                             (offset + half, tensor.data_ptr() + tensor.stride(0) * esize,
                              tensor.stride(1) * esize, half)]
                else:
                    parts = [(offset, tensor.data_ptr(), tensor.stride(0) * esize, layer["bytes"])]
                for _, base, pitch, size in parts:
                    if base % 8 or pitch % 8 or size % 8:
                        raise ValueError(f"KV layer {layer['name']} is not 8-byte aligned for the copy kernels")
                spans.extend(parts)
                offset += layer["bytes"]
            scales = getattr(self, "scales", None)
            if scales is not None:
                if scales.data_ptr() % 8:
                    raise ValueError("the scales are not 8-byte aligned for the copy kernels")
                spans.append((offset, scales.data_ptr(), scales.stride(0), self.layers[-1]["bytes"]))
            self._span_table = spans
        return self._span_table

    @property
    def min_span_bytes(self):
        """The caches' shortest span's length: the copy launches' shape hint (short spans share a workgroup).  Found
        once: every launch asks."""
        if getattr(self, "_min_span", None) is None:
            spans = self.spans()
            self._min_span = min(span[3] for span in (spans[:-1] if getattr(self, "scales", None) is not None
                                                      else spans))
        return self._min_span

    def _copy_stream_handle(self):
        with self._state_lock:
            if getattr(self, "_copy_stream", None) is None:
                device = next(iter(self.caches.values())).device
                with self.pool.borrow_copy_stream() as handle:
                    self._copy_stream = self.torch.cuda.ExternalStream(handle, device=device)
            return self._copy_stream

    def _restore_stream(self):
        """The stream restores run on: the pool's copy stream, or (split) one of their own.

        HIP maps a process's streams onto a few hardware queues (four by
        default), and work on one queue runs in order whatever its stream.  A
        split restore stream that shares the copy stream's queue holds every
        restore launch behind the save's copy barriers (duplex save + restore
        fell from about 80 to 54 GB/s), so the plane creates its own and keeps
        one whose queue neither the copy stream nor the engine's current stream
        uses (:meth:`_pick_streams`); with copy-engine restores, one whose
        copy engine is not the copy stream's (:meth:`_pick_dma_restore_stream`).
        """
        with self._state_lock:
            copy = self._copy_stream_handle()
            if self.restore_stream_mode == "shared":
                return copy
            if self._split_stream is None:
                torch = self.torch
                device = next(iter(self.caches.values())).device
                taken = [copy, torch.cuda.current_stream(device)]
                if self.restore_mode == "dma":
                    stream = self._pick_dma_restore_stream(device, taken)
                else:
                    picked = self._pick_streams(device, 1, taken)
                    stream = picked[0] if picked else None
                self._split_stream = stream or self._own_stream(device)
            return self._split_stream

    def _hash_streams(self):
        """The streams the saves' hash kernels rotate over, on hardware queues of their own where possible.

        A hash stream sharing the copy stream's or the restore stream's queue
        would hold their copies and launches behind SHA-256 launches, so up to
        ``HASH_STREAMS`` streams are picked on queues none of those (nor the
        engine's current stream, nor each other) use.  With too few queues the
        plane makes do with one stream that shares: a save's SHA-256 is fed as
        short launches, so a shared queue is never held for a whole chain.
        """
        with self._state_lock:
            if self._hash_stream_list is None:
                torch = self.torch
                device = next(iter(self.caches.values())).device
                taken = [self._copy_stream_handle(), torch.cuda.current_stream(device)]
                if self.restore_stream_mode == "split":
                    taken.append(self._restore_stream())
                picked = self._pick_streams(device, max(1, HASH_STREAMS), taken)
                self._hash_stream_list = picked or [self._own_stream(device)]
                self._hash_queues_own = bool(picked)
            return self._hash_stream_list

    def _aside_stream(self):
        """The plane's second stream on the copy stream's side, or None: where a hashed staged save gathers
        its later records while the first chunk's device-to-host copy runs (``SAVE_LEAD``), and where a
        copy-engine restore places each chunk while the next one is copied (``PLACE_ASIDE``).

        Work on it would wait behind anything sharing its hardware queue, so
        it is picked on a queue that none of the copy, engine, restore and
        hash streams use; without one (HIP's default four queues are all
        taken when restores have a stream of their own) saves gather in one
        launch and restores copy and place in turn.
        """
        with self._state_lock:
            wanted = (SAVE_LEAD and self.save_mode == "staged") or (PLACE_ASIDE and self.restore_mode == "dma")
            if not wanted:
                return None
            if not self._aside_picked:
                self._aside_picked = True
                device = self._device
                taken = [self._copy_stream_handle(), self.torch.cuda.current_stream(device)]
                if self.restore_stream_mode == "split":
                    taken.append(self._restore_stream())
                taken += self._hash_streams()
                picked = self._pick_streams(device, 1, taken)
                self._aside = picked[0] if picked else None
            return self._aside

    def _lead_stream(self):
        """The aside stream when hashed saves may gather on it (``SAVE_LEAD``), else None."""
        return self._aside_stream() if SAVE_LEAD and self.save_mode == "staged" else None

    def _place_stream(self):
        """The aside stream when copy-engine restores may place chunks on it (``PLACE_ASIDE``), else None."""
        return self._aside_stream() if PLACE_ASIDE and self.restore_mode == "dma" else None

    def stream_report(self):
        """What the plane's streams turned out to be: the restore stream's mode and, for copy-engine
        restores, what picking it measured; how many hash streams the saves rotate over and whether they
        were found on hardware queues of their own (None before the first hashed save); whether the plane
        found its aside stream (None before it looked) and what may use it."""
        with self._state_lock:
            hashes = self._hash_stream_list
            return {"restore_stream": self.restore_stream_mode, "restore_mode": self.restore_mode,
                    "restore_stream_check": self.restore_stream_check,
                    "hash_streams": None if hashes is None else len(hashes),
                    "hash_streams_on_own_queues": self._hash_queues_own,
                    "aside_stream": None if not self._aside_picked else self._aside is not None,
                    "save_lead": SAVE_LEAD, "place_aside": PLACE_ASIDE}

    def _pick_dma_restore_stream(self, device, taken):
        """A restore stream on a hardware queue of its own whose copies run on another copy engine than
        the copy stream's, so a restore's host-to-device copies and a save's device-to-host copies share
        the link (92-97 GB/s together on MI355X's x16 link) instead of taking turns (57 GB/s).

        The HIP runtime ties a stream to one copy engine at its first copy of
        64 KiB or more, and keeps it in both directions.  Each candidate's
        first copy is issued while the copy stream and the best candidate so
        far are busy with long copies, each in its own direction; then the
        candidate's host-to-device copies are timed alone and beside a copy
        stream copy the other way.  Engines differ: beside the copy stream's,
        one candidate ran both ways at 96 GB/s and carried overlapped saves
        and restores at 86.6 GB/s, the next at 93.7 and 73.7.  So up to
        ``ENGINE_TRIES`` candidates are tried, the best pair is kept (others
        destroyed as they lose), and the search stops at one whose pair takes
        at most ``ENGINE_OVERLAP`` of the two copies in turn with host-to-device
        copies at least 85 % as fast as the copy stream's.  Every copy goes
        through the library, not torch, so no torch allocator tracks the
        streams that are destroyed here.
        """
        torch, lib = self.torch, kernel_library()
        busy_bytes, probe = ENGINE_BUSY_BYTES, ENGINE_PROBE_BYTES
        host = torch.empty(busy_bytes + 2 * probe, dtype=torch.uint8, pin_memory=True)
        dev = torch.empty(busy_bytes + 2 * probe, dtype=torch.uint8, device=device)
        host_at, dev_at = host.data_ptr(), dev.data_ptr()
        copy = self._copy_stream
        copy.wait_stream(torch.cuda.current_stream(device))

        def up(stream, nbytes, at=0):
            _check(lib, lib.kvsnap_copy_to_device(dev_at + at, host_at + at, nbytes, stream.cuda_stream))

        def down(stream, nbytes, at=0):
            _check(lib, lib.kvsnap_copy_to_host(host_at + at, dev_at + at, nbytes, stream.cuda_stream))

        def timed(*issues):
            best = float("inf")
            for _ in range(3):
                torch.cuda.synchronize(device)
                start = time.perf_counter()
                for issue in issues:
                    issue()
                torch.cuda.synchronize(device)
                best = min(best, time.perf_counter() - start)
            return best

        kept, kept_score, pairs = None, float("inf"), []
        try:
            t_down = timed(lambda: down(copy, probe))
            t_up_ref = timed(lambda: up(copy, probe))
            for tries in range(1, ENGINE_TRIES + 1):
                picked = self._pick_streams(device, 1, taken + ([kept] if kept is not None else []))
                if not picked:
                    break
                stream = picked[0]
                torch.cuda.synchronize(device)
                down(copy, busy_bytes)           # the copy stream's engine and the kept candidate's are
                if kept is not None:             # copying, each in the direction it carries, ...
                    up(kept, busy_bytes)
                up(stream, probe, busy_bytes)    # ... when the candidate takes its engine
                torch.cuda.synchronize(device)
                t_up = timed(lambda: up(stream, probe, busy_bytes))
                t_both = timed(lambda: down(copy, probe), lambda: up(stream, probe, busy_bytes + probe))
                # 0.5: both directions at full speed at once; 1: in turn.  One tied beside a busy engine has
                # run host-to-device at half the link's rate, hence the speed check.
                overlap = t_both / (t_up_ref + t_down)
                fast = t_up <= t_up_ref / 0.85
                good = fast and overlap <= ENGINE_OVERLAP
                score = overlap + (0.0 if fast else 1.0)
                measured = {"candidates": tries, "h2d_gbps": round(probe / t_up / 1e9, 1),
                            "copy_stream_h2d_gbps": round(probe / t_up_ref / 1e9, 1),
                            "both_ways_gbps": round(2 * probe / t_both / 1e9, 1), "accepted": good}
                pairs.append(measured["both_ways_gbps"])
                if score < kept_score:
                    if kept is not None:
                        self._drop_stream(kept)
                    kept, kept_score, self.restore_stream_check = stream, score, measured
                else:
                    self._drop_stream(stream)
                if good:
                    break
        finally:
            torch.cuda.synchronize(device)
            del host, dev
        if self.restore_stream_check is not None:
            self.restore_stream_check["tried_both_ways_gbps"] = pairs   # every candidate's pair, in order
            report_engine_pick(self.restore_stream_check)
        return kept

    def _pick_streams(self, device, count, taken):
        """Up to ``count`` new streams, each on a hardware queue that no stream of ``taken`` nor another
        picked one uses.  Candidates that share are kept until the end (so the next candidate lands on
        another queue) and then destroyed; four misses in a row mean every queue is taken."""
        taken, picked, rejected = list(taken), [], []
        budget, misses = STREAM_CANDIDATES, 0
        try:
            while len(picked) < count and budget > 0 and misses < 4:
                budget -= 1
                stream = self._own_stream(device)
                if any(self._shares_queue(stream, taken)):
                    rejected.append(stream)
                    misses += 1
                    continue
                picked.append(stream)
                taken.append(stream)
                misses = 0
        finally:
            for stream in rejected:
                self._drop_stream(stream)
        return picked

    def _own_stream(self, device):
        lib = kernel_library()
        handle = C.c_size_t()
        index = device.index if device.index is not None else self.torch.cuda.current_device()
        _check(lib, lib.kvsnap_stream_create(index, C.byref(handle)))
        self._owned_streams.append(handle.value)
        return self.torch.cuda.ExternalStream(handle.value, device=device)

    def _drop_stream(self, stream):
        handle = stream.cuda_stream
        self._owned_streams.remove(handle)
        _check(kernel_library(), kernel_library().kvsnap_stream_destroy(handle))

    def _shares_queue(self, held, others):
        """Per stream of ``others``: does work queued on it wait behind a hold on ``held``?

        A trivial launch on a stream with a hardware queue of its own ends
        within microseconds, while the hold lasts about 3 ms; one that shares
        ``held``'s queue ends only after the hold.  A launch counts as free
        only when it is seen finished while the hold is seen still running;
        a check whose hold ended before it could be observed is repeated, and
        anything unproven counts as shared.
        """
        torch, lib = self.torch, kernel_library()
        for _ in range(3):
            for stream in [held] + others:
                stream.synchronize()
            _check(lib, lib.kvsnap_hold_stream(held.cuda_stream, HOLD_ITERS))
            held_done = torch.cuda.Event()
            held_done.record(held)
            marks = []
            for stream in others:
                _check(lib, lib.kvsnap_hold_stream(stream.cuda_stream, 0))
                mark = torch.cuda.Event()
                mark.record(stream)
                marks.append(mark)
            free = [False] * len(others)
            conclusive = not held_done.query()
            while conclusive:
                seen = [i for i, mark in enumerate(marks) if not free[i] and mark.query()]
                if held_done.query():
                    break                       # marks first seen now may have ended after the hold
                for i in seen:
                    free[i] = True
                if all(free):
                    break
                time.sleep(50e-6)
            for stream in [held] + others:
                stream.synchronize()
            if conclusive:
                return [not f for f in free]
        return [True] * len(others)

    def _load_tables(self):
        """Per span, as int64 device tensors: its offset in a packed block, its cache's
        base address and block pitch in bytes, and its length in 8-byte words."""
        with self._state_lock:
            if getattr(self, "_tables", None) is None:
                spans = self.spans()
                self._copy_stream_handle()
                device = next(iter(self.caches.values())).device
                columns = ([s[0] for s in spans], [s[1] for s in spans], [s[2] for s in spans],
                           [s[3] // 8 for s in spans])
                self._tables = tuple(self.torch.tensor(column, dtype=self.torch.int64, device=device)
                                     for column in columns)
            return self._tables

    def group_tables(self):
        """The gather with CRC32C's table, or None where it does not apply: for each 1 KiB group of a record,
        the base address and block pitch of its source (int64 device tensors), so group g of block b is
        ``base[g] + b * pitch[g]``.  It applies when every span is whole KiB at a whole-KiB record offset,
        16-byte aligned, and the record is under 2 GiB."""
        with self._state_lock:
            if not hasattr(self, "_groups"):
                spans, size = self.spans(), self.block_bytes
                fits = bool(kernel_library().kvsnap_gather_crc32c_fits(size)) and all(
                    offset % 1024 == 0 and nbytes % 1024 == 0 and base % 16 == 0 and pitch % 16 == 0
                    for offset, base, pitch, nbytes in spans)
                self._groups = None
                if fits:
                    bases, pitches = [0] * (size // 1024), [0] * (size // 1024)
                    for offset, base, pitch, nbytes in spans:
                        for k in range(nbytes // 1024):
                            bases[offset // 1024 + k], pitches[offset // 1024 + k] = base + 1024 * k, pitch
                    device = next(iter(self.caches.values())).device
                    self._groups = tuple(self.torch.tensor(column, dtype=self.torch.int64, device=device)
                                         for column in (bases, pitches))
            return self._groups

    def _tail_regions(self, valid):
        """Byte ranges of one packed record that hold token slots >= ``valid`` (reference
        ``dataplane.py:262-272``), merged where adjacent.  Found once per ``valid`` (at most a block's token
        slots): finding them took 38 us for 36 layers of one head and 267 us for 36 layers of eight."""
        found = self._tails.get(valid)
        if found is None:
            found = self._tails[valid] = self._find_tail_regions(valid)
        return found

    def _find_tail_regions(self, valid):
        regions, offset = [], 0
        for layer in self.layers:
            if len(layer["shape"]) == 1:        # a block's scales: no token slots
                continue
            if len(layer["shape"]) == 4:       # [2, N, H, C] K/V split
                _, n, h, c = layer["shape"]
                _, sn, sh, _ = layer["stride"]
                halves = 2
            else:                               # [H, N, C]
                h, n, c = layer["shape"]
                sh, sn, _ = layer["stride"]
                halves = 1
            esize = layer["bytes"] // halves // h // n // c
            half_bytes = layer["bytes"] // halves
            for half in range(halves):
                base = offset + half * half_bytes
                for head in range(h):
                    for token in range(valid, n):
                        regions.append((base + (head * sh + token * sn) * esize, c * esize))
            offset += layer["bytes"]
        regions.sort()
        merged = []
        for start, length in regions:
            if merged and merged[-1][0] + merged[-1][1] == start:
                merged[-1] = (merged[-1][0], merged[-1][1] + length)
            else:
                merged.append((start, length))
        return merged

    def _zero_tail(self, allocation, base, valid):
        """Zero token slots past ``valid`` in one packed pinned block (host memset)."""
        for start, length in self._tail_regions(valid):
            allocation.zero(base + start, length)

    def warm_up(self):
        """Build the tables and load the kernels at registration rather than on the first restore."""
        tables = self._load_tables()
        device = next(iter(self.caches.values())).device
        # The CRC32C tables and the static array of the no-allocation entry point, set up now, outside any
        # capture or serving loop.
        _check(kernel_library(), kernel_library().kvsnap_kernels_init(device.index))
        with self.torch.cuda.stream(self._copy_stream):
            empty = self.torch.zeros(1, dtype=self.torch.int64, device=device)
            copy_host_blocks(empty[:0], empty[:0], *tables, programs=self.restore_programs,
                             min_span_bytes=self.min_span_bytes)
        self._copy_stream.synchronize()
        self._restore_stream()      # the restore, hash and aside streams are chosen while the GPU is idle
        self._hash_streams()
        self._aside_stream()
        with self._state_lock:
            if self._reserved_staging is None and self.device_staging_bytes:
                self._reserved_staging = self._allocate(self.device_staging_bytes)

    def _allocate(self, nbytes):
        """A device uint8 tensor of ``nbytes``; an allocation failure is StagingUnavailable."""
        torch = self.torch
        try:
            return torch.empty(max(1, nbytes), dtype=torch.uint8, device=self._device)[:nbytes]
        except RuntimeError as exc:        # torch's OutOfMemoryError is one
            if "out of memory" not in str(exc).lower():
                raise
            raise StagingUnavailable(f"device staging of {nbytes} bytes is unavailable: {exc}") from exc

    @contextmanager
    def _device_buffers(self, *sizes):
        """One device uint8 tensor per byte count in ``sizes`` (4 KiB aligned), for the duration of the block:
        slices of the staging reserved at warm_up() when it is free and large enough, else allocated now
        (StagingUnavailable if that fails).  Callers drain every stream that used them before the block ends."""
        spans = [-(-max(1, size) // 4096) * 4096 for size in sizes]
        reserved = self._reserved_staging
        if reserved is not None and sum(spans) <= reserved.numel() and self._reserved_lock.acquire(blocking=False):
            try:
                starts = [sum(spans[:i]) for i in range(len(spans))]
                yield [reserved[at:at + size] for at, size in zip(starts, sizes)]
            finally:
                self._reserved_lock.release()
            return
        yield [self._allocate(size) for size in sizes]

    def _token_bytes_divide(self):
        """Whether every span is its token slots one after another, each whole 8-byte words: a partly filled
        block is then the front of each of its spans."""
        if getattr(self, "_tokens_outermost", None) is None:
            outermost = getattr(self, "scales", None) is None       # a block's scales are no token slots
            for layer in self.layers if outermost else ():
                half = len(layer["shape"]) == 4           # [2, N, H, C] K/V split, else [H, N, C]
                n = layer["shape"][1]
                heads, step = (layer["shape"][2], layer["stride"][1]) if half else (layer["shape"][0],
                                                                                   layer["stride"][1])
                slot = layer["bytes"] // (2 if half else 1) // n
                outermost &= n == self.block_size and step == heads * layer["shape"][-1] and slot % 8 == 0
            self._tokens_outermost = outermost
        return self._tokens_outermost

    def _copy_few(self, lib, tables, save, addresses, block_ids, filled, stream):
        """Queue one kvsnap_copy_few launch on ``stream``, with the plane's device current (the calling thread may
        have had another): the blocks to (``save``) or from the records at ``addresses``; ``filled`` token slots
        of the last block saved, 0 for all."""
        n = len(block_ids)
        if getattr(self, "_few_columns", None) is None:
            self._few_columns = (*(t.data_ptr() for t in tables), tables[0].numel(), self.min_span_bytes)
        arguments = (1 if save else 0, (C.c_uint64 * n)(*addresses), (C.c_int64 * n)(*block_ids), n,
                     *self._few_columns, filled, self.block_size if filled else 0, self.restore_programs,
                     stream.cuda_stream)
        if self.timer is None:
            _check(lib, lib.kvsnap_copy_few(*arguments))
        else:
            with _timed(self.timer, "gather_to" if save else "restore", stream):
                _check(lib, lib.kvsnap_copy_few(*arguments))

    # ------------------------------------------------------------------ restore

    def _launch_bounds(self, n, chunk_bytes):
        """(first, end) block ranges of one launch each: ``chunk_bytes`` of records per launch."""
        step = max(1, chunk_bytes // self.block_bytes)
        return [(first, min(n, first + step)) for first in range(0, n, step)]

    @staticmethod
    def _copy_batches(launches, batched):
        """Launch indices grouped into one host-to-device copy each: up to ``COPY_BATCH`` launches while
        more than ``COPY_TAIL`` follow (a copy boundary costs the engine 9-15 us), one each for the last
        ``COPY_TAIL`` so the early report still comes within 128 MiB of the end; one each unbatched."""
        if not batched:
            return [[k] for k in range(len(launches))]
        batches, head = [], max(0, len(launches) - COPY_TAIL)
        for k in range(len(launches)):
            if k < head and batches and len(batches[-1]) < COPY_BATCH and batches[-1][-1] < head:
                batches[-1].append(k)
            else:
                batches.append([k])
        return batches

    def load_scatter(self, block_ids, sources, *, progress=None, chunk_bytes=None):
        """Copy packed pinned blocks into ``block_ids`` with the restore kernel, and wait for them.

        ``sources[i]`` is ``(allocation, offset)`` holding block i packed, in
        this pool's pinned memory.  With ``restore_mode="kernel"`` the restore
        kernel reads each (block, span) from host memory over the link and
        writes it into its place in the KV cache; with ``"dma"`` the copy
        engines stage each chunk in device memory and the scatter kernel
        places it.  One launch per ``chunk_bytes`` of blocks (64 MiB when
        None, as the reference's default, with ``"dma"`` then copying up to
        four launches' blocks at a time but for the last three), on the pool's
        copy stream (or the plane's restore stream with
        ``restore_stream="split"``).  ``progress`` receives ``(None, total
        bytes)`` and then, per launch as it is queued, ``(its completion
        event, bytes left once it completes)``.  Returns the number of
        launches (reference ``dataplane.py:334-386``).
        """
        if len(sources) != len(block_ids):
            raise ValueError("one source per block is required")
        self._validate_ids(block_ids)
        if not block_ids:
            return 0
        torch, lib = self.torch, kernel_library()
        tables = self._load_tables()
        stream = self._restore_stream()
        size, n = self.block_bytes, len(block_ids)
        launches = self._launch_bounds(n, 64 << 20 if chunk_bytes is None else chunk_bytes)
        staged = self.restore_mode == "dma"
        report = _Progress(torch, progress, n * size)
        if n <= FEW_BLOCKS and len(launches) == 1 and (
                not staged or n * size <= FEW_BYTES) and hasattr(lib, "kvsnap_copy_few"):
            with self.pool.operation():
                addresses = _source_addresses(sources, size)
                fits = _word_aligned(addresses)
                if fits:
                    report.start()
                    with torch.cuda.device(self._device.index), _drain_on_failure(stream):
                        self._copy_few(lib, tables, False, addresses, block_ids, 0, stream)
                        report.launched(stream, 0)
            if fits:
                _drain(torch, stream)
                return 1
        batches = self._copy_batches(launches, staged and chunk_bytes is None)
        # Placing on the aside stream pays from the second copy on: the copy engine then goes on to the next.
        place = self._place_stream() if staged and len(batches) > 1 else None
        per_slot = max(launches[b[-1]][1] - launches[b[0]][0] for b in batches)
        # The device slots first, before anything is uploaded or copied.
        device = self._device_buffers(*[per_slot * size] * (2 if place is not None else 1)) if staged else \
            nullcontext([])
        with self._host_staging.borrow(16 * n) as host, device as slots:
            with self.pool.operation(), torch.cuda.stream(stream):
                # Holding the pool keeps every source open, and in place, until the launches are queued.
                addresses = _source_addresses(sources, size)
                ids = self._upload(host, list(block_ids) if staged else addresses + list(block_ids), stream)
                if staged:
                    placed = [None] * len(slots)
                else:
                    ids, records = ids[n:], ids[:n]
                report.start()
                with _drain_on_failure(stream, place):
                    if not staged:
                        for first, end in launches:
                            with _timed(self.timer, "restore", stream):
                                copy_host_blocks(records[first:end], ids[first:end], *tables,
                                                 programs=self.restore_programs, min_span_bytes=self.min_span_bytes)
                            report.launched(stream, (n - end) * size)
                        batches = []
                    for b, batch in enumerate(batches):
                        slot, low, high = slots[b % len(slots)], launches[batch[0]][0], launches[batch[-1]][1]
                        if placed[b % len(slots)] is not None:
                            stream.wait_event(placed[b % len(slots)])   # the slot's last chunk is in place
                        with _timed(self.timer, "restore", stream):
                            # Without the aside stream: in stream order, behind the scatter that last read the slot.
                            for start, count in _runs(addresses[low:high], size, low):
                                _check(lib, lib.kvsnap_copy_to_device(
                                    slot.data_ptr() + (start - low) * size, addresses[start], count * size,
                                    stream.cuda_stream))
                        on = stream
                        if place is not None:
                            copied = torch.cuda.Event()
                            copied.record(stream)
                            place.wait_event(copied)
                            on = place
                        for first, end in (launches[k] for k in batch):
                            with torch.cuda.stream(on), _timed(self.timer, "place", on):
                                scatter_blocks(slot.data_ptr() + (first - low) * size, size, ids[first:end], *tables,
                                               programs=self.gather_programs, min_span_bytes=self.min_span_bytes)
                            report.launched(on, (n - end) * size)
                        if place is not None:
                            placed[b % len(slots)] = torch.cuda.Event()
                            placed[b % len(slots)].record(place)
                    if place is not None:
                        stream.wait_event(placed[(len(batches) - 1) % len(slots)])   # the restore stream's order
            _drain(torch, stream)                                                       # holds every placement
        return len(launches)

    def load_scatter_checked(self, block_ids, sources, crcs, *, progress=None, chunk_bytes=None):
        """Restore with every block's CRC32C folded from its bytes as the restore kernel copies them.

        The checks the reference makes on the host before a restore from
        pinned memory (``VolatileOwner.borrow(verify_checksums=True)``,
        reference ``kvsnap/connector/volatile.py:302-305``; the staged fetch,
        ``kvsnap/connector/vllm.py:531``) moved into the copy: each block
        crosses the host link once and its CRC32C comes out of the same pass,
        so the check adds no pass over HBM or host memory.  The blocks are
        written before the comparison: a mismatch raises
        ``CorruptSnapshotError`` once every launch has completed, and the
        caller must treat ``block_ids`` as not loaded (the worker reports them
        as load errors, which the engine recomputes).  With
        ``restore_mode="dma"`` the copy engines move each chunk into device
        memory and the same kernel, on a full grid, places and checks it from
        there, leaving the CUs to the engine while the link is busy.
        ``progress`` receives its entries only after the comparison, so a load
        is never reported early on unchecked bytes.  Returns the launch count,
        one per ``chunk_bytes`` of blocks (64 MiB when None; the copies then
        batched as :meth:`load_scatter`'s).  :meth:`load_scatter_verified`
        checks before any KV write instead.
        """
        from .blobs import CorruptSnapshotError
        self._validate_ids(block_ids)
        if not (len(sources) == len(block_ids) == len(crcs)):
            raise ValueError("one source and one CRC32C per block are required")
        if not block_ids:
            return 0
        torch, lib = self.torch, kernel_library()
        tables = self._load_tables()
        stream = self._restore_stream()
        size, n, n_spans = self.block_bytes, len(block_ids), tables[0].numel()
        launches = self._launch_bounds(n, 64 << 20 if chunk_bytes is None else chunk_bytes)
        staged = self.restore_mode == "dma"
        # As in load_scatter: copies batched, chunks placed on the aside stream while the next copy runs, two
        # slots in turn.
        batches = self._copy_batches(launches, staged and chunk_bytes is None)
        place = self._place_stream() if staged and len(batches) > 1 else None
        span_args = tuple(t.data_ptr() for t in tables)
        per_slot = max(launches[b[-1]][1] - launches[b[0]][0] for b in batches)
        slots = 2 if place is not None else 1
        # Device memory first, before anything is uploaded or copied: the per-span partial CRCs, the records'
        # CRC32Cs, and with the copy engines the chunk slots.
        device = self._device_buffers(4 * n * n_spans, 4 * n, *([per_slot * size] * slots if staged else []))
        with self._host_staging.borrow(8 * (slots * per_slot if staged else n) + 12 * n) as host, device as buffers:
            partial, crc = buffers[0].view(torch.int32), buffers[1].view(torch.int32)
            with self.pool.operation(), torch.cuda.stream(stream):
                # Holding the pool keeps every source open, and in place, until the launches are queued.
                addresses = _source_addresses(sources, size)
                if staged:
                    # The copy engines move each chunk into a device slot; the checked kernel, on a full grid,
                    # places it from there (HBM to HBM) and folds its CRC32Cs.
                    reads = [slot.data_ptr() + j * size for slot in buffers[2:] for j in range(per_slot)]
                    placed = [None] * slots
                else:
                    reads = addresses
                table = self._upload(host, reads + list(block_ids), stream)
                ids = table[len(reads):]
                with _drain_on_failure(stream, place):
                    for b, batch in enumerate(batches):
                        slot, on = b % slots, stream
                        low, high = launches[batch[0]][0], launches[batch[-1]][1]
                        if staged:
                            if placed[slot] is not None:
                                stream.wait_event(placed[slot])     # the slot's last chunk is placed
                            # Without the aside stream: in stream order, behind the kernel that last read the slot.
                            for start, count in _runs(addresses[low:high], size, low):
                                _check(lib, lib.kvsnap_copy_to_device(reads[slot * per_slot + start - low],
                                                                      addresses[start], count * size,
                                                                      stream.cuda_stream))
                            if place is not None:
                                copied = torch.cuda.Event()
                                copied.record(stream)
                                place.wait_event(copied)
                                on = place
                        for first, end in (launches[k] for k in batch):
                            with _timed(self.timer, "restore_checked", on):
                                _check(lib, lib.kvsnap_restore_blocks_checked(
                                    table.data_ptr() + 8 * (slot * per_slot + first - low if staged else first),
                                    ids.data_ptr() + 8 * first, end - first, *span_args, n_spans,
                                    0 if staged else self.restore_programs, partial.data_ptr() + 4 * first * n_spans,
                                    on.cuda_stream))
                        if place is not None:
                            placed[slot] = torch.cuda.Event()
                            placed[slot].record(place)
                    if place is not None:
                        stream.wait_event(placed[(len(batches) - 1) % slots])
                    _check(lib, lib.kvsnap_restore_checked_crc32c(partial.data_ptr(), n, span_args[0], span_args[3],
                                                                  n_spans, size, crc.data_ptr(), stream.cuda_stream))
                    # The CRC32Cs land past the table, which the upload reads earlier in stream order.
                    at = 8 * len(table)
                    _check(lib, lib.kvsnap_copy_to_host(host.data_ptr() + at, crc.data_ptr(), 4 * n,
                                                        stream.cuda_stream))
            _drain(torch, stream)
            got = host.numpy()[at:at + 4 * n].view("<u4").tolist()
        bad = [i for i, (value, want) in enumerate(zip(got, crcs)) if value != want]
        if bad:
            raise CorruptSnapshotError(f"{len(bad)} of {n} restored blocks fail their CRC32C (first: block {bad[0]})")
        report = _Progress(torch, progress, n * size)
        report.start()
        report.launched(stream, 0, wait=True)     # complete before another thread can query it
        return len(launches)

    def load_scatter_verified(self, block_ids, sources, crcs, *, progress=None, chunk_bytes=None):
        """Restore with every block's CRC32C checked on the GPU before any KV write.

        The disk-staged restore's check (reference ``kvsnap/store/store.py:
        717-718``, done there on the host in the read threads) moved to the
        GPU: the packed sources are DMA'd into device staging, CRC32C'd there
        and compared with ``crcs``; only if every block matches does the
        scatter kernel (HBM to HBM) write them into ``block_ids``.
        A mismatch raises ``CorruptSnapshotError`` and leaves the KV cache
        untouched.  ``progress`` and the return value are as for
        :meth:`load_scatter`.
        """
        from .blobs import CorruptSnapshotError
        self._validate_ids(block_ids)
        if not (len(sources) == len(block_ids) == len(crcs)):
            raise ValueError("one source and one CRC32C per block are required")
        if not block_ids:
            return 0
        torch, lib = self.torch, kernel_library()
        tables = self._load_tables()
        stream = self._copy_stream_handle()
        size, n = self.block_bytes, len(block_ids)
        launches = self._launch_bounds(n, 64 << 20 if chunk_bytes is None else chunk_bytes)
        work_bytes = int(lib.kvsnap_crc32c_workspace_bytes(size, n))
        device = self._device_buffers(n * size, 4 * n, work_bytes)
        with self._host_staging.borrow(8 * n) as host, device as (stage, crc, workspace):
            crc = crc.view(torch.int32)
            with self.pool.operation(), torch.cuda.stream(stream):
                # The pool stays held until the check has been waited for: no source may be released first.
                addresses = _source_addresses(sources, size)
                with _drain_on_failure(stream):
                    # One DMA per run of records side by side in pinned memory, across allocations (a host
                    # tier's blocks are separate allocations, reserved one after another): 512 per-record
                    # copies of 2.25 MiB cost 14 ms more than one.
                    for start, count in _runs(addresses, size):
                        _check(lib, lib.kvsnap_copy_to_device(stage.data_ptr() + start * size, addresses[start],
                                                              count * size, stream.cuda_stream))
                    with _timed(self.timer, "crc32c", stream):
                        _check(lib, lib.kvsnap_crc32c_records(stage.data_ptr(), size, size, n, 0, crc.data_ptr(),
                                                              workspace.data_ptr(), work_bytes, stream.cuda_stream))
                    _check(lib, lib.kvsnap_copy_to_host(host.data_ptr(), crc.data_ptr(), 4 * n, stream.cuda_stream))
                _drain(torch, stream)
            got = host.numpy()[:4 * n].view("<u4").tolist()
            bad = [i for i, (value, want) in enumerate(zip(got, crcs)) if value != want]
            if bad:
                raise CorruptSnapshotError(f"{len(bad)} of {n} staged blocks fail their CRC32C "
                                           f"(first: block {bad[0]})")
            report = _Progress(torch, progress, n * size)
            with torch.cuda.stream(stream):
                ids = self._upload(host, list(block_ids), stream)
                report.start()
                with _drain_on_failure(stream):
                    for first, end in launches:
                        with _timed(self.timer, "scatter", stream):
                            scatter_blocks(stage.data_ptr() + first * size, size, ids[first:end], *tables,
                                           programs=self.gather_programs, min_span_bytes=self.min_span_bytes)
                        report.launched(stream, (n - end) * size)
            _drain(torch, stream)
        return len(launches)

    def load_from_disk(self, block_ids, blobs, segments, *, first_block=0, chunk_bytes=128 << 20, workers=8,
                       verify="gpu", progress=None, ring=4):
        """Disk-staged restore with the read pipelined against the copy.

        ``blobs`` is a :class:`kvsnap_amd.blobs.BlobDirectory`; ``segments`` the
        snapshot's blocks from ``first_block`` on (reference ``store.py:
        686-723``, which reads every block into one staging buffer before the
        first copy).  ``workers`` native threads read the blocks in order into
        a ring of ``ring`` pinned chunk slots of ``chunk_bytes`` (at most
        ``ring * chunk_bytes`` pinned bytes, however large the snapshot),
        refilling a slot once its chunk's copy has completed
        (:meth:`BlobDirectory.ring_reader`).  Each chunk crosses the link in
        one copy-engine transfer into one of two device slots; with
        ``verify="gpu"`` its blocks' CRC32Cs are computed there and compared
        on the host before the scatter kernel places them, one chunk behind
        the copies, so the copy engine never waits for a comparison;
        ``verify="host"`` has the read threads check each block as it lands.
        No KV block is written before its check.  A corrupt block raises
        ``CorruptSnapshotError`` once every earlier placement has completed,
        so the error is a clean miss: the blocks already written belong to
        this request and are recomputed.  ``progress`` receives ``(None,
        total)`` and one entry per chunk placed, as for :meth:`load_scatter`.
        Returns the number of placements (one per chunk).
        """
        from .blobs import CorruptSnapshotError
        if verify not in ("gpu", "host"):
            raise ValueError("verify must be gpu or host")
        if type(ring) is not int or ring < 2:
            raise ValueError("the staging ring needs at least two slots")
        self._validate_ids(block_ids)
        n, size = len(block_ids), self.block_bytes
        if len(segments) != n:
            raise ValueError("one segment per block is required")
        if not n:
            return 0
        torch, lib = self.torch, kernel_library()
        per_chunk = max(1, min(n, chunk_bytes // size))
        bounds = [(a, min(n, a + per_chunk)) for a in range(0, n, per_chunk)]
        slots = min(ring, len(bounds))
        tables = self._load_tables()
        stream = self._restore_stream()
        place = self._place_stream() or stream      # checks and placements beside the next chunk's copy
        want = [segment["crc32c"] for segment in segments]
        checked_on_gpu = verify == "gpu"
        # Device memory first, before anything is read or copied: the CRC32Cs, the CRC workspace, two chunk slots.
        work_bytes = int(lib.kvsnap_crc32c_workspace_bytes(size, per_chunk)) if checked_on_gpu else 0
        device = self._device_buffers(4 * n if checked_on_gpu else 0, work_bytes,
                                      *[per_chunk * size] * min(2, len(bounds)))
        report = _Progress(torch, progress, n * size)
        checked = [None] * len(bounds)
        with device as buffers, self.staging(slots * per_chunk) as staged, \
                self._host_staging.borrow(12 * n) as host, \
                blobs.ring_reader(segments, staged.pointer, size, per_chunk, slots, first_block=first_block,
                                  workers=workers, verify="host" if verify == "host" else "none") as reader:
            crc, workspace, device_slots = buffers[0].view(torch.int32), buffers[1], buffers[2:]
            placed = [None] * len(device_slots)
            crcs_at = 8 * n                     # the CRC32Cs land past the block ids in the host buffer
            with torch.cuda.stream(stream), _drain_on_failure(stream, place):
                ids = self._upload(host, list(block_ids), stream)
                report.start()

                def settle(k):
                    # Chunk k's copy (and check) completed: compare, release its ring slot, place it.
                    a, b = bounds[k]
                    checked[k].synchronize()
                    if checked_on_gpu:
                        got = host.numpy()[crcs_at + 4 * a:crcs_at + 4 * b].view("<u4").tolist()
                        bad = [a + i for i, value in enumerate(got) if value != want[a + i]]
                        if bad:
                            raise CorruptSnapshotError(f"block {first_block + bad[0]} fails its checksum (CRC32C)")
                    reader.release(k)
                    slot = device_slots[k % len(device_slots)]
                    with torch.cuda.stream(place), _timed(self.timer, "place", place):
                        scatter_blocks(slot.data_ptr(), size, ids[a:b], *tables, programs=self.gather_programs,
                                       min_span_bytes=self.min_span_bytes)
                    placed[k % len(device_slots)] = torch.cuda.Event()
                    placed[k % len(device_slots)].record(place)
                    report.launched(place, (n - b) * size)

                for k, (a, b) in enumerate(bounds):
                    reader.wait(k)
                    d = k % len(device_slots)
                    if placed[d] is not None and place is not stream:
                        stream.wait_event(placed[d])          # the device slot's last chunk is placed
                    with _timed(self.timer, "disk_copy", stream):
                        _check(lib, lib.kvsnap_copy_to_device(device_slots[d].data_ptr(),
                                                              staged.pointer + (k % slots) * per_chunk * size,
                                                              (b - a) * size, stream.cuda_stream))
                    if place is not stream:
                        copied = torch.cuda.Event()
                        copied.record(stream)
                        place.wait_event(copied)
                    if checked_on_gpu:
                        with _timed(self.timer, "crc32c", place):
                            _check(lib, lib.kvsnap_crc32c_records(device_slots[d].data_ptr(), size, size, b - a, 0,
                                                                  crc.data_ptr() + 4 * a, workspace.data_ptr(),
                                                                  work_bytes, place.cuda_stream))
                        _check(lib, lib.kvsnap_copy_to_host(host.data_ptr() + crcs_at + 4 * a, crc.data_ptr() + 4 * a,
                                                            4 * (b - a), place.cuda_stream))
                    checked[k] = torch.cuda.Event()
                    checked[k].record(place)
                    if k:
                        settle(k - 1)
                settle(len(bounds) - 1)
                if place is not stream:
                    stream.wait_event(placed[(len(bounds) - 1) % len(device_slots)])
            _drain(torch, stream)
        return len(bounds)

    # ------------------------------------------------------------------ save

    def _hash_lane(self):
        """The next of the plane's hash lanes (one per hash stream, each with its feeding thread), round robin."""
        with self._state_lock:
            if self._hash_lanes is None:
                self._hash_lanes = [HashLane(self.torch, stream) for stream in self._hash_streams()]
            lane = self._hash_lanes[self._digest_next % len(self._hash_lanes)]
            self._digest_next += 1
            return lane

    def save_gather(self, block_ids, targets, num_kv_tokens, *, chunk_bytes=None, digests=None):
        """Gather ``block_ids`` on the GPU into packed records in pinned memory, and wait for them.

        ``targets[i]`` is ``(allocation, offset)``, the pinned bytes that
        receive block i's record; the caller has fenced the engine's work on
        those blocks (reference ``dataplane.py:388-437``).  Token slots from
        ``num_kv_tokens`` on in the last block are zeroed in device memory
        before the record leaves the GPU, so no snapshot carries stale KV.

        ``save_mode == "staged"`` (default): the gather kernel packs records
        into device staging, ``chunk_bytes`` at a time (``SAVE_CHUNK_BYTES``
        when None; the reference's default is 64 MiB), and the pool's copies
        take them to pinned memory, one copy per run of targets lying back to
        back in one allocation; returns the number of copies, as the
        reference does.  ``save_mode == "direct"``: the gather kernel writes
        every record straight into its pinned target over the host link, one
        launch per chunk; returns the number of launches.

        When ``digests`` is a list, one :class:`BlockDigests` is appended: the
        per-block SHA-256 and CRC32C, computed on the GPU from a device copy
        of the whole session while and after the copies run, or, for few
        records (``HASH_THREADS``), on host threads from the pinned records
        as and after they land: their bytes must then stay as saved until
        the digests are there (closing a target, or another save or write
        into it through the pool, waits for that by itself).
        """
        self._validate_ids(block_ids)
        if len(targets) != len(block_ids) or len(block_ids) != -(-num_kv_tokens // self.block_size):
            raise ValueError("block count does not cover computed tokens")
        if not block_ids:
            return 0
        torch, lib = self.torch, kernel_library()
        tables = self._load_tables()
        stream = self._copy_stream_handle()
        size, n = self.block_bytes, len(block_ids)
        chunk_bytes = SAVE_CHUNK_BYTES if chunk_bytes is None else chunk_bytes
        per_chunk = max(1, min(n, chunk_bytes // size))
        lead_first = max(1, min(chunk_bytes, LEAD_FIRST_BYTES) // size)
        filled = num_kv_tokens % self.block_size
        direct, hashed = self.save_mode == "direct", digests is not None
        for allocation, _ in targets:
            if getattr(allocation, "_uses", None):
                for held, low, high in _target_bounds(targets, size):
                    settle_readers(held, low, high)     # an earlier save's records, still being hashed there
                break
        # Few records are hashed on the host as they land; the save itself is then an unhashed one.
        threads = self._hash_threads(lib, n) if hashed else 0
        hashed = hashed and not threads
        # (A larger save hashed on the host lands in parts instead.)
        if not hashed and n <= min(FEW_BLOCKS, per_chunk) and (
                (direct and not threads) or n * size <= FEW_BYTES) and (
                not filled or self._token_bytes_divide()) and hasattr(lib, "kvsnap_copy_few"):
            with self.pool.operation():
                destinations = _source_addresses(targets, size, "save target")
                fits = _word_aligned(destinations)
                if fits:
                    with torch.cuda.device(self._device.index), _drain_on_failure(stream):
                        self._copy_few(lib, tables, True, destinations, block_ids, filled, stream)
                        landed = _Landing(torch, stream)
                        landed.held_on(targets)
                    if threads:
                        job = HostHashJob(lib, targets, destinations, size, [(0, n, landed)], threads)
            if fits:
                landed.finish()
                self._wait_targets(targets)
                if threads:           # at most 0.4 ms of hashing: no thread is woken for it
                    digests.append(BlockDigests(None, job, job.crc, job.sha, job))
                return 1 if direct else len(_target_runs(targets, 0, n, size))
        regions = self._tail_regions(filled) if filled else []
        # Looked up before the copy stream becomes current: picking the stream compares it with the engine's.
        lead = self._lead_stream() if hashed and not direct and n > lead_first else None
        # Device staging first, before anything is uploaded or copied.  A hashed save's records stay staged for
        # its hash kernels after this call returns, so they are allocated for it; the chunks of an unhashed staged
        # save come from the plane's reserved staging when it is free.
        checked = hashed and direct       # one pass: pinned records, their device copy and their CRC32Cs
        # One pass too: device records and their CRC32Cs (small sessions, whole-KiB spans).
        fused = hashed and not direct and 0 < n * size <= GATHER_CRC_MAX_BYTES and self.group_tables() is not None
        one_crc_work = max(16, int(lib.kvsnap_crc32c_workspace_bytes(size, 1))) if checked or fused else 0
        if checked:
            n_spans = tables[0].numel()
            device = nullcontext([self._allocate(n * size), self._allocate(4 * n * n_spans), self._allocate(4 * n),
                                  self._allocate(one_crc_work)])
        elif fused:
            device = nullcontext([self._allocate(n * size), self._allocate(4 * n), self._allocate(one_crc_work)])
        elif hashed:
            device = nullcontext([self._allocate(n * size)])
        elif not direct:
            device = self._device_buffers(per_chunk * size)
        elif threads:                     # the paced gather's per-span words, unused
            device = nullcontext([None, self._allocate(4 * n * tables[0].numel())])
        else:
            device = nullcontext([None])
        with self._host_staging.borrow(16 * (n + len(regions))) as host, device as (stage, *checks):
            with self.pool.operation(), torch.cuda.stream(stream):
                # Holding the pool keeps every target open until the copies are queued.
                destinations = _source_addresses(targets, size, "save target")
                values = (destinations if direct else []) + list(block_ids)
                values += [start for start, _ in regions] + [length for _, length in regions]
                table = self._upload(host, values, stream)
                ids = table[n:2 * n] if direct else table[:n]
                tail = table[len(table) - 2 * len(regions):]
                gathered, split = [], n
                marks = [] if threads else None      # (first, end, event) of the records that have landed
                part = 2 * threads                  # the first: a pair of records a thread
                with _drain_on_failure(stream, lead):
                    if checked:
                        count = self._save_direct_checked(lib, table, n, tables, tail, per_chunk, destinations[-1],
                                                          stage, *checks)
                        done = torch.cuda.Event()
                        done.record(stream)
                        gathered.append(done)
                    elif hashed:
                        # The whole session staged, for the hash kernels to read after the copies: the first
                        # chunk gathered here, the rest on the lead stream (where there is one) while that
                        # chunk's copy runs.
                        split = lead_first if lead is not None else n
                        if lead is not None:
                            begun = torch.cuda.Event()
                            begun.record(stream)
                        crcs = checks if fused else None
                        gathered.append(self._gather_part(lib, ids, tables, stage, 0, split, n, tail, stream, crcs))
                        if lead is not None:
                            lead.wait_event(begun)
                            gathered.append(self._gather_part(lib, ids, tables, stage, split, n, n, tail, lead,
                                                              crcs))
                    if checked:
                        pass
                    elif direct:
                        count = self._save_direct(lib, table, n, tables, tail, per_chunk, destinations[-1], marks,
                                                  part, *checks)
                    else:
                        count = self._save_staged(ids, targets, tables, tail, stage, per_chunk, hashed,
                                                  split, gathered[-1] if split < n else None, marks, part)
                        if threads:
                            count = len(_target_runs(targets, 0, n, size))    # as a hashed save counts them
                    landed = _Landing(torch, stream)
                    if direct:                       # copies are events of the pool's own
                        landed.held_on(targets)
                    if threads:
                        job = HostHashJob(lib, targets, destinations, size, marks, threads)
            if hashed:
                lane = self._hash_lane()
                for event in gathered:
                    lane.stream.wait_event(event)
                given = checks[1] if checked else checks[0] if fused else None
                job = HashJob(torch, stage.data_ptr(), size, size, n, self._device, lane, HASH_SLICE_BLOCKS,
                              timer=self.timer, keepalive=stage,
                              crc=None if given is None else given.view(torch.int32))
                digests.append(BlockDigests(torch, job, job.crc, job.sha, job))
            if threads:
                self._hash_on_host(job, digests)
            landed.finish()
        self._wait_targets(targets)
        return count

    def _hash_threads(self, lib, n):
        """Host threads that hash a save of ``n`` records, 0 where the GPU does."""
        if SAVE_LEAD or not hasattr(lib, "kvsnap_hash_records"):
            return 0
        threads = min(HASH_THREADS, len(os.sched_getaffinity(0)), 256)     # 256: kvsnap_hash_records' most
        if threads < 1 or n > RECORDS_PER_HASH_THREAD * threads or not lib.kvsnap_hash_records_available():
            return 0
        return threads

    def _hash_on_host(self, job, digests):
        """Start ``job`` on the plane's hashing thread; its BlockDigests go to ``digests``."""
        with self._state_lock:
            try:
                if self._host_hashes is None:
                    self._host_hashes = HostHashes()
                self._host_hashes.submit(job)
            except RuntimeError:       # no thread to be had: the job runs when its digests are asked for
                pass
        digests.append(BlockDigests(None, job, job.crc, job.sha, job))

    def _mark(self, marks, first, end):
        """Note in ``marks`` that records [first, end) have landed once the copy stream has come this far."""
        event = self.torch.cuda.Event()
        event.record(self._copy_stream)
        marks.append((first, end, event))

    @staticmethod
    def _wait_targets(targets):
        """Every copy queued on the targets' allocations, and every kernel's writes held on them, are over."""
        for allocation in {id(allocation): allocation for allocation, _ in targets}.values():
            allocation.wait()

    def _gather_part(self, lib, ids, tables, stage, first, end, n, tail, stream, crcs=None):
        """Gather records [first, end) of a whole staged session into ``stage`` on ``stream`` (zeroing the
        last record's tail when it is among them); returns an event recorded after them.  With ``crcs``
        (the CRC32C buffer, n int32 as bytes, and a one-record CRC32C workspace) the gather folds every
        record's CRC32C into the buffer as it goes, and a zeroed tail's record has its CRC32C taken again."""
        size = self.block_bytes
        with self.torch.cuda.stream(stream):
            # Built before its timing span starts, so the span holds the kernel, not the host's checks.
            if crcs is None:
                name, launch = "gather", gather_launcher(ids[first:end], *tables, stage.data_ptr() + first * size,
                                                         size, programs=self.gather_programs,
                                                         min_span_bytes=self.min_span_bytes)
            else:
                name, launch = "gather_crc", gather_crc32c_launcher(
                    ids[first:end], *self.group_tables(), size, stage.data_ptr() + first * size, size,
                    crcs[0].view(self.torch.int32)[first:end])
        with _timed(self.timer, name, stream):
            launch()
        if tail.numel() and end == n:
            last = stage.data_ptr() + (n - 1) * size
            self._zero_regions(lib, last, tail, stream)
            if crcs is not None:
                _check(lib, lib.kvsnap_crc32c_records(last, size, size, 1, 0, crcs[0].data_ptr() + 4 * (n - 1),
                                                      crcs[1].data_ptr(), crcs[1].numel(), stream.cuda_stream))
        done = self.torch.cuda.Event()
        done.record(stream)
        return done

    def _save_staged(self, ids, targets, tables, tail, stage, per_chunk, whole, split=None, rest_gathered=None,
                     marks=None, part=0):
        """Device staging to pinned memory through the pool's copies; returns the copy count: the runs of
        back-to-back targets in each chunk (with ``marks``, a chunk is copied in parts, the first of ``part``
        records, each noted in it).

        With the whole session staged (``whole``, when digests are asked for)
        nothing is recycled, so each run of back-to-back targets is one copy
        however long: one large DMA keeps the link fuller than a chunk's
        worth at a time.  The records from ``split`` on were gathered on
        another stream, and their copies wait for ``rest_gathered`` first.
        """
        size, n = self.block_bytes, len(targets)
        lib = kernel_library()
        if whole:
            copies = 0
            for first, end in ((0, split), (split, n)) if rest_gathered is not None else ((0, n),):
                if first:
                    self._copy_stream.wait_event(rest_gathered)
                for index, count, allocation, offset in _target_runs(targets, first, end, size):
                    allocation.copy(stage.data_ptr() + index * size, count * size, offset, to_host=True,
                                    producer_stream=self._copy_stream.cuda_stream)
                    copies += 1
            return copies
        copies, base = 0, stage.data_ptr()
        for first in range(0, n, per_chunk):
            end = min(n, first + per_chunk)
            launch = gather_launcher(ids[first:end], *tables, base, size, programs=self.gather_programs,
                                     min_span_bytes=self.min_span_bytes)
            with _timed(self.timer, "gather", self._copy_stream):
                launch()
            if tail.numel() and end == n:
                self._zero_regions(lib, base + (end - 1 - first) * size, tail)
            for low, high in _parts(first, end, part if marks is not None else end - first):
                for index, count, allocation, offset in _target_runs(targets, low, high, size):
                    allocation.copy(base + (index - first) * size, count * size, offset, to_host=True,
                                    producer_stream=self._copy_stream.cuda_stream)
                if marks is not None:
                    self._mark(marks, low, high)
            copies += len(_target_runs(targets, first, end, size))
        return copies

    def _save_direct(self, lib, table, n, tables, tail, per_chunk, last_record, marks=None, part=0, words=None):
        """The gather kernel writes each record into its pinned target; returns the launch count, one a chunk.
        ``table`` holds the n destinations, then the n block ids.  With ``marks``, a chunk is written in
        parts, the first of ``part`` records, each noted in it, by the checked gather, as a hashed direct save's records are:
        its paced writes leave a decode beside them alone (``words``: room for a part's per-span CRC32Cs).
        Without the device copy that a GPU-hashed save's workgroups write too, three quarters of them fill the
        link: rotating fp8 sessions beside a decode copied at 40.3 GB/s with a 0.15-0.17 ms p99 stall on 3
        workgroups, 40.0 and 0.25-0.27 on 4; the 2k session of 117 MB lands in 2.44 ms on 9, 2.42 on 12."""
        programs = self.restore_programs - self.restore_programs // 4
        columns = tuple(t.data_ptr() for t in tables)
        stream, n_spans = self._copy_stream.cuda_stream, tables[0].numel()
        for first in range(0, n, per_chunk):
            end = min(n, first + per_chunk)
            if marks is None:
                with _timed(self.timer, "gather_to", self._copy_stream):
                    _check(lib, lib.kvsnap_gather_to_records(
                        table.data_ptr() + 8 * first, table.data_ptr() + 8 * (n + first), end - first, *columns,
                        n_spans, self.min_span_bytes, self.restore_programs, stream))
            for low, high in _parts(first, end, part) if marks is not None else ():
                with _timed(self.timer, "gather_checked", self._copy_stream):
                    _check(lib, lib.kvsnap_gather_blocks_checked(
                        table.data_ptr() + 8 * low, table.data_ptr() + 8 * (n + low), high - low, *columns, n_spans,
                        0, 0, programs, words.data_ptr(), stream))
                if high == n and tail.numel():
                    self._zero_regions(lib, last_record, tail)
                self._mark(marks, low, high)
        if marks is None and tail.numel():
            self._zero_regions(lib, last_record, tail)
        return -(-n // per_chunk)

    def _save_direct_checked(self, lib, table, n, tables, tail, per_chunk, last_record, stage, partial, crc,
                             workspace):
        """A hashed direct save in one pass over the cache: the checked gather writes each record into its
        pinned target and into ``stage`` (device, for the SHA-256 kernels) and folds its CRC32C, one launch per
        chunk on the plane's small grid; the finish kernel then gives every record's CRC32C in ``crc``.  A
        zeroed tail (in both copies) changes the last record, whose CRC32C is then taken again from the stage.
        Returns the launch count.  ``table`` holds the n destinations, then the n block ids."""
        size, n_spans, stream = self.block_bytes, tables[0].numel(), self._copy_stream
        launches = 0
        for first in range(0, n, per_chunk):
            end = min(n, first + per_chunk)
            with _timed(self.timer, "gather_checked", stream):
                _check(lib, lib.kvsnap_gather_blocks_checked(
                    table.data_ptr() + 8 * first, table.data_ptr() + 8 * (n + first), end - first,
                    tables[0].data_ptr(), tables[1].data_ptr(), tables[2].data_ptr(), tables[3].data_ptr(), n_spans,
                    stage.data_ptr() + first * size, size, self.restore_programs,
                    partial.data_ptr() + 4 * first * n_spans, stream.cuda_stream))
            launches += 1
        _check(lib, lib.kvsnap_restore_checked_crc32c(partial.data_ptr(), n, tables[0].data_ptr(),
                                                      tables[3].data_ptr(), n_spans, size, crc.data_ptr(),
                                                      stream.cuda_stream))
        if tail.numel():
            self._zero_regions(lib, last_record, tail)
            self._zero_regions(lib, stage.data_ptr() + (n - 1) * size, tail)
            work_bytes = int(lib.kvsnap_crc32c_workspace_bytes(size, 1))
            _check(lib, lib.kvsnap_crc32c_records(stage.data_ptr() + (n - 1) * size, size, size, 1, 0,
                                                  crc.data_ptr() + 4 * (n - 1), workspace.data_ptr(), work_bytes,
                                                  stream.cuda_stream))
        return launches

    def _zero_regions(self, lib, record_ptr, regions, stream=None):
        """Zero the byte ranges ``regions`` (starts, then lengths) of one record, on ``stream`` (the copy
        stream by default)."""
        count = regions.numel() // 2
        stream = self._copy_stream if stream is None else stream
        _check(lib, lib.kvsnap_zero_regions(record_ptr, regions.data_ptr(), regions.data_ptr() + 8 * count, count,
                                            stream.cuda_stream))

    def close(self):
        with self._state_lock:
            lanes, self._hash_lanes = self._hash_lanes or [], None
            if self._host_hashes is not None:
                lanes.append(self._host_hashes)
                self._host_hashes = None
        for lane in lanes:
            lane.close()                # every hash job over, its records released: the streams may go
        with self._state_lock:
            lib = kernel_library() if self._owned_streams else None
            while self._owned_streams:
                _check(lib, lib.kvsnap_stream_destroy(self._owned_streams.pop()))
            self._split_stream = self._hash_stream_list = None
            # Every operation drained the streams that used the reserved staging before it let go of it.
            self._reserved_staging = None
        self.pool.close()
