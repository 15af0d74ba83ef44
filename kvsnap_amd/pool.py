"""Python side of the pinned snapshot pool: ``CudaPool`` and ``PinnedAllocation``.

The pool itself is native (``csrc/pool.cpp``, C-ABI version 2 in
``libkvsnap_hip.so``): one ``hipHostMalloc`` arena, first-fit reservations,
one copy stream and one event per reservation.  This module is the drop-in
for the reference's ctypes binding (``kvsnap/connector/dataplane.py:38-211``):
the same class and method names, arguments, return values and exceptions
(``PinnedCapacityError`` when a reservation cannot fit, ``RuntimeError`` with
the native message otherwise, "pool closed" and "pinned allocation closed"
after close, a refusal after ``fork``).

Three rules carry the reference's ownership contract:

* A kernel that writes pinned memory by itself, or host threads that hash it,
  are uses the native side does not see; they are held on their allocations
  (:func:`hold`), which wait for them before they are released or written.
* Every native call is made while the pool's re-entrant lock is held and
  the handle is checked open, so ``close`` of the pool or of an allocation
  waits for any call another thread has in flight.
* Python objects whose memory a copy may still touch (an allocation's
  ``_tensor_references``) are dropped only once the native side has proven
  the copies complete (a successful wait, release or pool close); a failure
  keeps them alive, and the pool keeps the allocation object alive too.
"""
from __future__ import annotations

import ctypes as C
from contextlib import contextmanager
import os
import threading

#: The only pool ABI this binding speaks.
POOL_ABI_VERSION = 2

# ctypes types by the short names the signature table below uses.
_TYPES = {
    "int": C.c_int, "ptr": C.c_void_p, "size": C.c_size_t, "u32": C.c_uint32, "u64": C.c_uint64,
    "i64": C.c_int64, "f32": C.c_float, "str": C.c_char_p, "stream": C.c_size_t, "u64*": C.POINTER(C.c_uint64),
    "ptr*": C.POINTER(C.c_void_p), "size*": C.POINTER(C.c_size_t), "void": None,
}

#: "result <- arguments" per pool entry point (include/kvsnap_pool.h).
POOL_SIGNATURES = {
    "kvsnap_pool_abi_version": "int <-",
    "kvsnap_cuda_error": "str <-",
    "kvsnap_pool_create": "ptr <- size int",
    "kvsnap_pool_destroy": "void <- ptr",
    "kvsnap_pool_close_checked": "int <- ptr",
    "kvsnap_pool_reserve": "int <- ptr size u64* ptr*",
    "kvsnap_pool_copy": "int <- ptr u64 size ptr size int size",
    "kvsnap_pool_copy_2d": "int <- ptr u64 size size ptr size size size int size",
    "kvsnap_pool_wait": "int <- ptr u64",
    "kvsnap_pool_ready": "int <- ptr u64",
    "kvsnap_pool_release": "int <- ptr u64",
}

#: Optional entry point (older ABI-2 builds lack it): the copy stream's handle.
COPY_STREAM_SIGNATURE = ("kvsnap_pool_copy_stream", "int <- ptr size*")


def declare(lib, name, signature):
    """Give ``lib.name`` the argument and result types of ``signature`` ("result <- arg arg ...")."""
    result, _, arguments = signature.partition("<-")
    function = getattr(lib, name)
    function.argtypes = [_TYPES[word] for word in arguments.split()]
    function.restype = _TYPES[result.strip()]
    return function


def load_pool_library(path):
    """The pool library at ``path`` with its entry points typed (no HIP call is made)."""
    lib = C.CDLL(str(path))
    for name, signature in POOL_SIGNATURES.items():
        declare(lib, name, signature)
    return lib


class PinnedCapacityError(MemoryError):
    """The pinned pool cannot fit a reservation. Nothing was copied."""


class CopyFailed(RuntimeError):
    """A save's device-to-host copy failed once it may have started: its completion cannot be proven, so
    neither the GPU blocks nor the pinned memory may be reused (the reference's ``DMAUnknown`` case,
    ``kvsnap/connector/vllm.py:602-607``)."""


# Uses of an allocation's bytes that the native pool has no event for: a kernel writing them (``writes``), or host
# threads reading them.  A use has ``finish()``, which returns once it is over, and dropped (and raises, still
# held, if that cannot be proven), and ``query()``.


def hold(use, allocation, low=0, high=None):
    """Until it is dropped, ``allocation`` and its pool close only after ``use.finish()`` has returned; waiting
    for the allocation finishes the uses that write, and writing into bytes [low, high) (to its end when None)
    those that read them.  Called with the pool held open."""
    allocation.__dict__.setdefault("_uses", {})[use] = (low, allocation.size if high is None else high)


def drop(use, allocation):
    allocation._uses.pop(use, None)


def _settle(allocation, *, writes=None):
    """Finish every use held on ``allocation`` (``writes``: those that write); one that fails stays held, to
    retry."""
    for use in list(allocation._uses):
        if writes is None or use.writes == writes:
            use.finish()


def settle_readers(allocation, low, high):
    """Finish the uses that read bytes [low, high) of ``allocation``, which are about to be overwritten."""
    for use, (first, end) in list(allocation.__dict__.get("_uses", {}).items()):
        if not use.writes and first < high and low < end:
            use.finish()


def _forget_owners(allocation):
    owners = getattr(allocation, "_tensor_references", None)
    if owners is not None:
        owners.clear()


class CudaPool:
    """The pinned arena, its copy stream and per-allocation events (C-ABI version 2)."""

    def __init__(self, capacity_bytes: int, device: int = 0, library=None):
        from .native import resolve_cuda_library
        self._pid = os.getpid()
        self._lock = threading.RLock()
        # ident -> PinnedAllocation, for every reservation the native side has not released: their Python
        # owners live as long as the memory may still be in use.
        self._allocations = {}
        self.lib = load_pool_library(resolve_cuda_library(library))
        self.abi_version = self.lib.kvsnap_pool_abi_version()
        if self.abi_version != POOL_ABI_VERSION:
            raise RuntimeError(f"unsupported kvsnap pinned pool ABI {self.abi_version} "
                               f"(this binding speaks {POOL_ABI_VERSION}); rebuild the HIP library")
        handle = self.lib.kvsnap_pool_create(capacity_bytes, device)
        if not handle:
            raise RuntimeError(self._message())
        self.handle = handle

    # -- plumbing

    def _message(self):
        text = self.lib.kvsnap_cuda_error()
        return text.decode() if text else "unknown pinned pool error"

    def _same_process(self):
        if os.getpid() != self._pid:
            raise RuntimeError("a pinned pool cannot be used in a process forked from its owner")

    def check(self, result):
        """``result`` of a native call, or RuntimeError with the native message if it is negative."""
        if result < 0:
            raise RuntimeError(self._message())
        return result

    @contextmanager
    def operation(self):
        """Hold the pool open (its lock, after the fork and closed checks) for the duration of a call."""
        self._same_process()
        with self._lock:
            if self.handle is None:
                raise RuntimeError("pool closed")
            yield self.handle

    # -- public surface

    def reserve(self, size):
        """A ``PinnedAllocation`` of ``size`` bytes; PinnedCapacityError if the arena cannot fit it."""
        ident, pointer = C.c_uint64(0), C.c_void_p(None)
        with self.operation() as handle:
            if self.lib.kvsnap_pool_reserve(handle, size, C.byref(ident), C.byref(pointer)) < 0:
                message = self._message()
                kind = PinnedCapacityError if "pinned capacity exhausted" in message else RuntimeError
                raise kind(message)
            allocation = PinnedAllocation(self, ident.value, pointer.value, size)
            self._allocations[allocation.ident] = allocation
        return allocation

    def close(self):
        """Drain the copy stream and free the arena.  On failure everything stays as it was, to retry."""
        self._same_process()
        with self._lock:
            if self.handle is None:
                return
            for allocation in self._allocations.values():
                _settle(allocation)
            self.check(self.lib.kvsnap_pool_close_checked(self.handle))
            self.handle = None
            survivors, self._allocations = self._allocations, {}
            for allocation in survivors.values():
                allocation.closed = True
                _forget_owners(allocation)

    @contextmanager
    def borrow_copy_stream(self):
        """The copy stream's handle, valid while the context is open (the pool cannot close meanwhile)."""
        with self.operation() as handle:
            name, signature = COPY_STREAM_SIGNATURE
            if not hasattr(self.lib, name):
                raise RuntimeError("this HIP library has no kvsnap_pool_copy_stream; rebuild it")
            getter = declare(self.lib, name, signature)
            stream = C.c_size_t(0)
            self.check(getter(handle, C.byref(stream)))
            if not stream.value:
                raise RuntimeError("the pool returned no copy stream")
            yield stream.value


HipPool = CudaPool


class PinnedAllocation:
    """A reservation in a pool's pinned arena: host ``pointer``, ``size`` bytes, native id ``ident``."""

    def __init__(self, pool, ident, pointer, size):
        self.pool = pool
        self.ident, self.pointer, self.size = ident, pointer, size
        self.closed = False          # released, or its pool closed
        self._uses = {}              # use -> the bytes it may touch (hold)

    def _open(self):
        if self.closed or self.pool.handle is None:
            raise RuntimeError("pinned allocation closed")

    @contextmanager
    def operation(self):
        with self.pool.operation() as handle:
            self._open()
            yield handle

    def _settled(self, offset, size, what):
        """The address of ``size`` bytes at ``offset``, once every copy queued on the allocation is over."""
        self.wait()
        if type(offset) is not int or type(size) is not int or offset < 0 or size < 0 or offset + size > self.size:
            raise ValueError(f"pinned {what} outside allocation")
        return self.pointer + offset

    def _call(self, name, *arguments):
        """A native call on this allocation, checked; the pool stays open meanwhile."""
        with self.operation() as handle:
            return self.pool.check(getattr(self.pool.lib, name)(handle, self.ident, *arguments))

    def _to_be_written(self, offset, size):
        if self._uses:
            settle_readers(self, offset, offset + size)

    def copy(self, device_ptr, size, offset=0, *, to_host, producer_stream=0):
        """Queue a copy of ``size`` bytes between ``device_ptr`` and ``offset`` of this allocation on the
        pool's stream, after the work queued on ``producer_stream`` (a stream handle, 0 for none)."""
        if any(value < 0 for value in (device_ptr, size, offset, producer_stream)):
            raise ValueError("negative copy argument")
        if to_host:
            self._to_be_written(offset, size)
        self._call("kvsnap_pool_copy", offset, device_ptr, size, 1 if to_host else 0, producer_stream)

    def copy_2d(self, device_ptr, device_pitch, host_offset, host_pitch, width, height, *,
                to_host, producer_stream=0):
        """``height`` rows of ``width`` bytes between strided device and host memory."""
        if any(value < 0 for value in (device_ptr, device_pitch, host_offset, host_pitch, width, height,
                                       producer_stream)):
            raise ValueError("negative copy argument")
        if to_host:
            self._to_be_written(host_offset, self.size - host_offset)
        self._call("kvsnap_pool_copy_2d", host_offset, host_pitch, device_ptr, device_pitch, width, height,
                   1 if to_host else 0, producer_stream)

    def wait(self):
        """Block until every copy queued on this allocation has completed."""
        if self._uses:
            with self.operation():
                _settle(self, writes=True)
        self._call("kvsnap_pool_wait")
        _forget_owners(self)

    def ready(self):
        return bool(self._call("kvsnap_pool_ready")) and all(use.query() for use in list(self._uses) if use.writes)

    def read(self):
        return self.read_range(0, self.size)

    # Host access: each waits for the allocation's copies first, with the pool held throughout.

    def read_range(self, offset, size):
        with self.operation():
            return C.string_at(self._settled(offset, size, "read"), size)

    def zero(self, offset, size):
        with self.operation():
            self._to_be_written(offset, size)
            C.memset(self._settled(offset, size, "zero"), 0, size)

    def write(self, data):
        """Replace the allocation's bytes with ``data``, which must be exactly its size."""
        if len(data) != self.size:
            raise ValueError("a pinned write must fill the whole allocation")
        with self.operation():
            self._to_be_written(0, self.size)
            C.memmove(self._settled(0, self.size, "write"), data, self.size)

    def close(self):
        """Release the reservation once its copies are proven complete; on failure it stays reserved."""
        pool = self.pool
        pool._same_process()
        with pool._lock:
            if not self.closed and pool.handle is not None:
                _settle(self)
                pool.check(pool.lib.kvsnap_pool_release(pool.handle, self.ident))
            self.closed = True
            pool._allocations.pop(self.ident, None)
            _forget_owners(self)
