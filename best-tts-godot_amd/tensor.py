"""Device tensors: a pooled device allocation plus a numpy-style view.

A :class:`DeviceTensor` is (storage, element offset, shape, element strides,
dtype).  Views (reshape of a contiguous tensor, transpose, slice, squeeze,
unsqueeze, broadcast) share storage exactly as the numpy views returned by
the reference's Reshape/Transpose/Squeeze/Unsqueeze/Slice/Split branches do
(tools/ref_runtime.py:511-549).  Storage comes from libkk's bucketed pool
(kk_alloc/kk_free) and goes back to it when the last view is dropped.
"""
import ctypes
import functools
import math
import sys

import numpy as np

from . import _lib

NP_TO_CODE = {
    np.dtype(np.float32): _lib.F32, np.dtype(np.int8): _lib.I8,
    np.dtype(np.uint8): _lib.U8, np.dtype(np.int32): _lib.I32,
    np.dtype(np.int64): _lib.I64, np.dtype(np.bool_): _lib.BOOL,
    np.dtype(np.float16): _lib.F16,
}
CODE_TO_NP = {v: k for k, v in NP_TO_CODE.items()}

# downloads: DeviceTensor.numpy calls so far; stream: the handle of libkk's stream
_state = {"device": None, "downloads": 0, "stream": None}


def init(device=0):
    """Initialise libkk on `device` (idempotent)."""
    if _state["device"] is None:
        _lib.call("kk_init", int(device))
        _state["stream"] = _stream()
        _state["device"] = int(device)
    return _state["device"]


def device_count():
    n = ctypes.c_int(0)
    _lib.call("kk_device_count", ctypes.byref(n))
    return n.value


def sync():
    init()
    _lib.call("kk_sync")


def pool_stats():
    """(live_bytes, pooled_bytes, peak_live_bytes) of the device pool."""
    vals = [ctypes.c_size_t(0) for _ in range(3)]
    _lib.call("kk_pool_stats", *[ctypes.byref(v) for v in vals])
    return tuple(v.value for v in vals)


def dispatch_count():
    """Kernels launched by libkk since init, outside graph recording."""
    n = ctypes.c_uint64(0)
    _lib.call("kk_dispatch_count", ctypes.byref(n))
    return n.value


def pool_trim(budget_bytes=0):
    init()
    _lib.call("kk_pool_trim", int(budget_bytes))


_alloc_out = ctypes.c_void_p()  # out-parameter of kk_alloc (the walk is single-threaded)
_alloc_ref = ctypes.byref(_alloc_out)
_fast = {}  # bound entry points of the allocation path


class Storage:
    """One pooled device buffer; `lent` once another library was told its
    address: then libkk's stream waits for torch's current one before the
    pool may hand the memory out again."""

    __slots__ = ("ptr", "nbytes", "lent", "__weakref__")

    def __init__(self, nbytes):
        alloc = _fast.get("kk_alloc")
        if alloc is None:
            init()
            alloc = _fast["kk_alloc"] = _lib.load().kk_alloc
        rc = alloc(nbytes if nbytes > 0 else 1, _alloc_ref)
        if rc:
            _lib.raise_error("kk_alloc", rc)
        self.ptr = _alloc_out.value
        self.nbytes = nbytes
        self.lent = False

    def __del__(self):
        ptr, self.ptr = getattr(self, "ptr", None), None
        if ptr:
            try:
                if self.lent:
                    _order("kk_stream_wait")
                if _lib._lib is not None:
                    _lib._lib.kk_free(ptr)
            except Exception:  # interpreter shutdown: the process frees it
                pass


class Borrowed:
    """Device memory of another library's array, which is kept alive.  Where
    it is torch's, torch's current stream waits for libkk's work before the
    memory goes back to torch's allocator."""

    __slots__ = ("ptr", "nbytes", "owner", "lent")

    def __init__(self, ptr, nbytes, owner):
        self.ptr = ptr
        self.nbytes = nbytes
        self.owner = owner

    def __del__(self):
        try:
            if _is_torch(self.owner):
                _order("kk_stream_signal")
        except Exception:  # interpreter shutdown
            pass


def _is_torch(arr):
    torch = sys.modules.get("torch")
    return torch is not None and isinstance(arr, torch.Tensor)


def _torch_stream(device):
    """The handle of torch's current stream; libkk's own where torch has none yet."""
    torch = sys.modules.get("torch")
    if torch is None or device is None or not torch.cuda.is_initialized():
        return _state["stream"]
    # from here on by the shortest way (the first is the second without an object for it)
    _fast["torch_stream"] = (getattr(torch._C, "_cuda_getCurrentRawStream", None) or
                             (lambda d: torch.cuda.current_stream(d).cuda_stream))
    return _fast["torch_stream"](device)


_fast["torch_stream"] = _torch_stream


def _order(which):
    """kk_stream_wait or kk_stream_signal with torch's current stream, where
    torch has one that is not libkk's.  Not while a graph is recorded: its
    replays are ordered by whoever launches them."""
    stream = _fast["torch_stream"](_state["device"])
    if stream == _state["stream"]:
        return
    try:
        _lib.call(which, stream)
    except _lib.KKError as e:
        if e.code != -4:  # KK_E_STATE
            raise


def wait_stream(stream=0):
    """Work given to libkk from here on starts after what `stream` (a HIP
    stream's handle, 0 the default stream; torch: `s.cuda_stream`) holds now."""
    init()
    _lib.call("kk_stream_wait", int(stream))


def signal_stream(stream=0):
    """Work given to `stream` from here on starts after what libkk holds now."""
    init()
    _lib.call("kk_stream_signal", int(stream))


def use_stream(stream=None):
    """libkk's work from here on goes to `stream` (a handle, see wait_stream;
    None: libkk's own stream), after what it has been given so far.  A program
    whose torch and libkk work alternate gives libkk torch's stream
    (`use_stream(torch.cuda.current_stream().cuda_stream)`): all of it is then
    in the order of the calls, and nothing waits where arrays are handed over."""
    init()
    if stream is not None and stream == _state["stream"]:
        return
    _lib.call("kk_stream_use", stream, stream is None)
    _state["stream"] = _stream()


def _stream():
    handle = ctypes.c_void_p(None)
    _lib.call("kk_stream", ctypes.byref(handle))
    return handle.value or 0


_PROTOS = {}  # (shape, strides, dtype's letter) -> KKTensor with data unset
_INTERFACES = {}  # (shape, strides, dtype's letter) -> array interface but for the address


@functools.lru_cache(maxsize=4096)
def _contig_strides(shape):
    st, acc = [], 1
    for d in reversed(shape):
        st.append(acc)
        acc *= int(d)
    return tuple(reversed(st))


class DeviceTensor:
    """A strided view of device memory (element strides, numpy semantics)."""

    __slots__ = ("storage", "offset", "shape", "strides", "dtype", "_desc", "host")

    def __init__(self, storage, shape, dtype, strides=None, offset=0):
        self.storage = storage
        self.shape = tuple(map(int, shape))
        self.dtype = dtype if isinstance(dtype, np.dtype) else np.dtype(dtype)
        if self.dtype not in NP_TO_CODE:
            raise TypeError(f"unsupported device dtype {self.dtype}")
        self.strides = tuple(map(int, strides)) if strides is not None \
            else _contig_strides(self.shape)
        self.offset = int(offset)
        self.host = None  # cached host value of a constant uploaded once
        if len(self.shape) > _lib.KK_MAX_RANK:
            raise ValueError(f"rank {len(self.shape)} exceeds {_lib.KK_MAX_RANK}")
        self._desc = None

    # ----------------------------------------------------------- creation
    @classmethod
    def empty(cls, shape, dtype=np.float32):
        shape = tuple(map(int, shape))
        dtype = dtype if isinstance(dtype, np.dtype) else np.dtype(dtype)
        if dtype not in NP_TO_CODE:
            raise TypeError(f"unsupported device dtype {dtype}")
        if len(shape) > _lib.KK_MAX_RANK:
            raise ValueError(f"rank {len(shape)} exceeds {_lib.KK_MAX_RANK}")
        return cls._fresh(shape, dtype)

    @classmethod
    def _fresh(cls, shape, dtype):
        """empty() of another tensor's shape (a tuple of int) and dtype."""
        t = object.__new__(cls)  # a fresh contiguous tensor: no view checks
        t.storage = Storage(math.prod(shape) * dtype.itemsize)
        t.shape = shape
        t.dtype = dtype
        t.strides = _contig_strides(shape)
        t.offset = 0
        t.host = None
        t._desc = None
        return t

    @classmethod
    def from_numpy(cls, arr):
        arr = np.asarray(arr)
        if not arr.flags.c_contiguous:  # (np.ascontiguousarray would make 0-d arrays 1-d)
            arr = arr.copy(order="C")
        if arr.dtype not in NP_TO_CODE:
            raise TypeError(f"unsupported dtype {arr.dtype}")
        t = cls.empty(arr.shape, arr.dtype)
        if arr.nbytes:
            _lib.call("kk_upload", ctypes.c_void_p(t.ptr),
                      arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes)
        return t

    @classmethod
    def from_array(cls, arr, stream=None):
        """A tensor over the memory of a device array of another library (one
        with `__cuda_array_interface__`, as torch's and cupy's have): no copy,
        any strides, `arr` kept alive.  libkk has a stream of its own: its
        later work waits for what `stream` (see wait_stream) holds, or the
        stream that the array names, or, for torch's arrays, torch's current
        stream; the values of other libraries' arrays that name no stream must
        be there already.  What is written to the array later needs
        wait_stream again.  A torch array's memory goes back to torch when the
        tensor and the array are dropped, in the order of torch's current
        stream; other libraries' must be kept until libkk has used it (sync
        or signal_stream).  Import torch before libkk is first used, so that
        both run on the same HIP runtime."""
        desc = arr.__cuda_array_interface__
        dtype = np.dtype(desc["typestr"])
        if dtype not in NP_TO_CODE:
            raise TypeError(f"unsupported dtype {dtype}")
        if desc.get("mask") is not None:
            raise TypeError("masked arrays are not supported")
        shape = tuple(map(int, desc["shape"]))
        strides = desc.get("strides")
        if strides is not None:
            if any(st % dtype.itemsize for st in strides):
                raise ValueError(f"strides {strides} are not whole elements of {dtype}")
            strides = [st // dtype.itemsize for st in strides]
        if stream is None and desc.get("stream") is not None:
            # the interface's names of the default and the per-thread stream are HIP's handles but for 1
            stream = 0 if desc["stream"] == 1 else desc["stream"]
        if stream is not None:
            wait_stream(stream)
        elif _is_torch(arr):
            if arr.device.index != init(arr.device.index):
                raise ValueError(f"an array on {arr.device}: libkk is on device {init()}")
            _order("kk_stream_wait")
        t = cls(Borrowed(int(desc["data"][0] or 0), math.prod(shape) * dtype.itemsize, arr), shape, dtype, strides)
        return t

    @property
    def __cuda_array_interface__(self):
        """This tensor's memory for another library (torch.as_tensor(t,
        device="cuda") makes a view that keeps it alive).  torch's current
        stream waits for what libkk has been given so far; other libraries find
        libkk's stream in the interface and wait for it themselves.  A reader
        on any other stream needs signal_stream() before it reads, and
        wait_stream() before the tensor is dropped."""
        key = (self.shape, self.strides, self.dtype.char)
        fixed = _INTERFACES.get(key)
        if fixed is None:
            item = self.dtype.itemsize
            fixed = {"shape": self.shape, "typestr": self.dtype.str, "version": 3, "strides":
                     None if self.is_contiguous() else tuple(st * item for st in self.strides)}
            if len(_INTERFACES) < 4096:
                _INTERFACES[key] = fixed
        storage = self.storage
        address = storage.ptr + self.offset * self.dtype.itemsize if 0 not in self.shape else 0
        if _state["device"] is None:
            return dict(fixed, data=(address, False))
        storage.lent = True
        _order("kk_stream_signal")
        # (1 is the interface's name of the default stream)
        return dict(fixed, data=(address, False), stream=_state["stream"] or 1)

    # ------------------------------------------------------------ queries
    @property
    def ptr(self):
        return self.storage.ptr + self.offset * self.dtype.itemsize

    @property
    def ndim(self):
        return len(self.shape)

    @property
    def size(self):
        return math.prod(self.shape)

    @property
    def code(self):
        return NP_TO_CODE[self.dtype]

    def is_contiguous(self):
        if self.strides == _contig_strides(self.shape) or self.size == 0:
            return True
        acc = 1
        for d, s in zip(reversed(self.shape), reversed(self.strides)):
            if d != 1 and s != acc:
                return False
            acc *= d
        return True

    def desc(self):
        """The kk_tensor descriptor (cached; views are immutable).  Descriptors
        of one (shape, strides, dtype) differ only in the data pointer: each
        is copied from a cached prototype."""
        ref = self._desc
        if ref is None:
            key = (self.shape, self.strides, self.dtype.char)
            proto = _PROTOS.get(key)
            if proto is None:
                proto = _lib.KKTensor()
                proto.dtype = NP_TO_CODE[self.dtype]
                proto.rank = len(self.shape)
                for i, (n, s) in enumerate(zip(self.shape, self.strides)):
                    proto.shape[i] = n
                    proto.strides[i] = s
                if len(_PROTOS) < 4096:
                    _PROTOS[key] = proto
            d = _lib.KKTensor.from_buffer_copy(proto)
            d.data = self.storage.ptr + self.offset * self.dtype.itemsize
            ref = self._desc = ctypes.byref(d)  # (which keeps d)
        return ref

    def __repr__(self):
        return f"DeviceTensor(shape={self.shape}, dtype={self.dtype}, strides={self.strides})"

    # ------------------------------------------------------------- copies
    def contiguous(self):
        if self.is_contiguous():
            return self
        out = DeviceTensor.empty(self.shape, self.dtype)
        _lib.call("kk_copy", out.desc(), self.desc())
        return out

    def astype(self, dtype):
        dtype = np.dtype(dtype)
        out = DeviceTensor.empty(self.shape, dtype)
        _lib.call("kk_copy", out.desc(), self.desc())
        return out

    def numpy(self):
        """Download (waits for all enqueued work)."""
        _state["downloads"] += 1
        src = self.contiguous()
        host = np.empty(self.shape, dtype=self.dtype)
        if host.nbytes:
            _lib.call("kk_download", host.ctypes.data_as(ctypes.c_void_p),
                      ctypes.c_void_p(src.ptr), host.nbytes)
        return host

    # -------------------------------------------------------------- views
    def _view(self, shape, strides, offset=None):
        return DeviceTensor(self.storage, shape, self.dtype, strides,
                            self.offset if offset is None else offset)

    def reshape(self, shape):
        shape = list(int(d) for d in shape)
        if -1 in shape:
            known = math.prod(d for d in shape if d != -1)
            shape[shape.index(-1)] = self.size // known if known else 0
        if math.prod(shape) != self.size:
            raise ValueError(f"cannot reshape {self.shape} into {tuple(shape)}")
        src = self if self.is_contiguous() else self.contiguous()
        return src._view(shape, _contig_strides(tuple(shape)))

    def transpose(self, perm=None):
        if perm is None:
            perm = list(range(self.ndim))[::-1]
        perm = [int(p) % self.ndim for p in perm]
        return self._view([self.shape[p] for p in perm], [self.strides[p] for p in perm])

    def expand_dims(self, axis):
        r = self.ndim + 1
        axis = int(axis) % r if axis < 0 else int(axis)
        shape = list(self.shape)
        strides = list(self.strides)
        # A unit axis is never stepped along; give it the stride a contiguous
        # layout would have.
        inner = self.strides[axis] * self.shape[axis] if axis < self.ndim else 1
        shape.insert(axis, 1)
        strides.insert(axis, inner)
        return self._view(shape, strides)

    def squeeze(self, axes=None):
        if axes is None:
            keep = [i for i, d in enumerate(self.shape) if d != 1]
        else:
            ax = {int(a) % self.ndim for a in axes}
            for a in ax:
                if self.shape[a] != 1:
                    raise ValueError(f"cannot squeeze axis {a} of extent {self.shape[a]}")
            keep = [i for i in range(self.ndim) if i not in ax]
        return self._view([self.shape[i] for i in keep], [self.strides[i] for i in keep])

    def slice_axis(self, axis, start, stop, step=1):
        """View of range(start, stop, step) along `axis` (already clamped)."""
        n = len(range(start, stop, step))
        shape = list(self.shape)
        strides = list(self.strides)
        off = self.offset + (start * self.strides[axis] if n else 0)
        shape[axis] = n
        strides[axis] = self.strides[axis] * step
        return self._view(shape, strides, off)

    def broadcast_to(self, shape):
        shape = tuple(int(d) for d in shape)
        pad = len(shape) - self.ndim
        if pad < 0:
            raise ValueError("cannot broadcast to a lower rank")
        strides = []
        for i, d in enumerate(shape):
            if i < pad:
                strides.append(0)
                continue
            sd = self.shape[i - pad]
            if sd == d:
                strides.append(self.strides[i - pad])
            elif sd == 1:
                strides.append(0)
            else:
                raise ValueError(f"cannot broadcast {self.shape} to {shape}")
        return self._view(shape, strides)
