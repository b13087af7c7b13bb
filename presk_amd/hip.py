"""Python host side of the executor: a ctypes binding of include/presk_hip.h
and `HipExec`, the mirror of the reference's `trait KernelExec`
(crates/presk-kernel/src/host.rs:28-95) over device-resident buffers.

The native library must be built (presk_amd/build.py); nothing here falls
back to a CPU path: a missing library or a device error raises.
"""
from __future__ import annotations

import ctypes
import functools
import os
import sys

import numpy as np

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "libpresk_hip.so")

EXACT, FAST = 0, 1
OK, ERR, REFUSED, OVERFLOW = 0, -1, -2, -3

STORAGE_BYTES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2, "e8m15": 3, "i64": 8}

# Every entry point include/presk_hip.h declares.
SYMBOLS = ["presk_hip_init", "presk_hip_last_error", "presk_hip_compile", "presk_hip_run", "presk_hip_run_noalloc",
           "presk_hip_kernel_info",
           "presk_hip_release", "presk_hip_kernel_text", "presk_hip_alloc", "presk_hip_free", "presk_hip_h2d", "presk_hip_d2h", "presk_hip_memset",
           "presk_hip_sync", "presk_hip_stream_create", "presk_hip_stream_destroy", "presk_hip_time",
           "presk_hip_scalar_digest", "presk_hip_batch_create", "presk_hip_batch_add", "presk_hip_batch_graph", "presk_hip_batch_graph_branches",
           "presk_hip_batch_run", "presk_hip_batch_release", "presk_hip_convert", "presk_hip_batch_add_convert",
           "presk_hip_fill_normal", "presk_hip_dropout_mask", "presk_hip_batch_add_dropout",
           "presk_hip_pskd_decode", "presk_hip_pskd_decode_idx", "presk_hip_mfma_probe",
           "presk_hip_loss_workspace", "presk_hip_head_loss", "presk_hip_distill", "presk_hip_batch_add_head_loss", "presk_hip_batch_add_distill"]


class HipError(RuntimeError):
    """An executor error, its message starting with the reference's code
    (E10001, E7005, E7007: crates/presk-rt/src/lib.rs:971-981)."""

    def __init__(self, rc: int, message: str):
        super().__init__(message)
        self.rc = rc
        self.code = message.split(":", 1)[0] if message[:1] == "E" else "E10001"


class Info(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_char * 32), ("order", ctypes.c_char * 32), ("guarded", ctypes.c_int32),
                ("n_inputs", ctypes.c_int32), ("split_bound", ctypes.c_int64), ("flops", ctypes.c_double),
                ("bytes", ctypes.c_double)]


class LossArgs(ctypes.Structure):
    """presk_hip_loss."""
    _fields_ = [("dtype", ctypes.c_char_p), ("rows", ctypes.c_int64), ("model", ctypes.c_int64), ("vocab", ctypes.c_int64),
                ("top", ctypes.c_int64), ("tied", ctypes.c_int32), ("temperature", ctypes.c_double)] + [
                    (n, ctypes.c_void_p) for n in ("x", "w", "index", "teacher", "loss", "lse", "mean", "ct", "dx", "dw", "flag", "work")] + [
                        ("work_bytes", ctypes.c_size_t)]


_lib = None


def lib():
    """The loaded executor library (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m presk_amd.build` (hipcc, gfx950)")
        L = ctypes.CDLL(LIB_PATH)
        vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
        L.presk_hip_init.argtypes = [i32]
        L.presk_hip_last_error.restype = ctypes.c_char_p
        L.presk_hip_compile.argtypes = [ctypes.c_char_p, ctypes.c_char_p, i32, i32, ctypes.POINTER(vp)]
        L.presk_hip_run.argtypes = [vp, ctypes.POINTER(vp), i64, i64, vp]
        L.presk_hip_run_noalloc.argtypes = [vp, ctypes.POINTER(vp), i64, i64, vp]
        L.presk_hip_kernel_info.argtypes = [vp, ctypes.POINTER(Info)]
        L.presk_hip_kernel_text.argtypes = [vp, ctypes.c_char_p, ctypes.c_size_t]
        L.presk_hip_kernel_text.restype = i64
        L.presk_hip_release.argtypes = [vp]
        L.presk_hip_release.restype = None
        L.presk_hip_alloc.argtypes = [ctypes.c_size_t, ctypes.POINTER(vp)]
        L.presk_hip_free.argtypes = [vp]
        L.presk_hip_h2d.argtypes = [vp, vp, ctypes.c_size_t, vp]
        L.presk_hip_d2h.argtypes = [vp, vp, ctypes.c_size_t, vp]
        L.presk_hip_memset.argtypes = [vp, i32, ctypes.c_size_t, vp]
        L.presk_hip_sync.argtypes = [vp]
        L.presk_hip_stream_create.argtypes = [ctypes.POINTER(vp)]
        L.presk_hip_stream_destroy.argtypes = [vp]
        L.presk_hip_time.argtypes = [vp, ctypes.POINTER(vp), i64, i64, vp, i32, i32, ctypes.POINTER(ctypes.c_double)]
        L.presk_hip_scalar_digest.argtypes = [i32, ctypes.c_uint64, ctypes.c_uint64, ctypes.POINTER(ctypes.c_uint64)]
        L.presk_hip_batch_create.argtypes = [ctypes.POINTER(vp)]
        L.presk_hip_batch_add.argtypes = [vp, vp, ctypes.POINTER(vp), i64, i64]
        L.presk_hip_batch_graph.argtypes = [vp]
        L.presk_hip_batch_graph_branches.argtypes = [vp, i32]
        L.presk_hip_batch_run.argtypes = [vp, vp]
        L.presk_hip_batch_release.argtypes = [vp]
        L.presk_hip_batch_release.restype = None
        L.presk_hip_convert.argtypes = [vp, ctypes.c_char_p, vp, ctypes.c_char_p, i64, vp, vp]
        L.presk_hip_fill_normal.argtypes = [vp, ctypes.c_char_p, i64, ctypes.c_uint64, ctypes.c_double, ctypes.c_double, vp]
        L.presk_hip_mfma_probe.argtypes = [ctypes.c_char_p, i64, vp, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
        L.presk_hip_pskd_decode.argtypes = [vp, ctypes.c_int, vp, i64, vp, ctypes.c_char_p, vp, vp]
        L.presk_hip_pskd_decode_idx.argtypes = [vp, ctypes.c_uint64, i64, vp, vp]
        L.presk_hip_dropout_mask.argtypes = [vp, ctypes.c_double, ctypes.c_char_p, i64, vp, vp]
        L.presk_hip_batch_add_dropout.argtypes = [vp, vp, ctypes.c_double, ctypes.c_char_p, i64, vp]
        L.presk_hip_batch_add_convert.argtypes = [vp, vp, ctypes.c_char_p, vp, ctypes.c_char_p, i64, vp]
        la = ctypes.POINTER(LossArgs)
        L.presk_hip_loss_workspace.argtypes = [la, i32, ctypes.POINTER(ctypes.c_size_t)]
        L.presk_hip_head_loss.argtypes = [la, i32, vp]
        L.presk_hip_distill.argtypes = [la, i32, vp]
        L.presk_hip_batch_add_head_loss.argtypes = [vp, la, i32]
        L.presk_hip_batch_add_distill.argtypes = [vp, la, i32]
        _lib = L
    return _lib


def check(rc: int):
    if rc != OK:
        raise HipError(rc, lib().presk_hip_last_error().decode())


_initialized = None


def init(device: int = 0):
    """presk_hip_init; device -1 takes PRESK_HIP_DEVICE (device 0 when unset)."""
    global _initialized
    if _initialized != device:
        check(lib().presk_hip_init(device))
        _initialized = device


class DeviceBuffer:
    """A device allocation holding one buffer's storage (codes for f16/e8m15)."""

    def __init__(self, nbytes: int):
        self.nbytes = int(nbytes)
        p = ctypes.c_void_p()
        check(lib().presk_hip_alloc(max(self.nbytes, 1), ctypes.byref(p)))
        self.ptr = p.value

    @classmethod
    def of(cls, a: np.ndarray) -> "DeviceBuffer":
        a = np.ascontiguousarray(a)
        d = cls(a.nbytes)
        d.upload(a)
        return d

    def upload(self, a: np.ndarray, stream=None):
        a = np.ascontiguousarray(a)
        if a.nbytes > self.nbytes:
            raise ValueError("upload larger than the buffer")
        check(lib().presk_hip_h2d(self.ptr, a.ctypes.data, a.nbytes, stream))

    def download(self, dtype, count=None, stream=None) -> np.ndarray:
        dt = np.dtype(dtype)
        n = self.nbytes // dt.itemsize if count is None else count
        out = np.empty(n, dtype=dt)
        check(lib().presk_hip_d2h(out.ctypes.data, self.ptr, out.nbytes, stream))
        return out

    def zero(self, stream=None):
        check(lib().presk_hip_memset(self.ptr, 0, self.nbytes, stream))

    def free(self):
        if self.ptr:
            lib().presk_hip_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class DeviceView(DeviceBuffer):
    """Bytes [offset, offset + nbytes) of another buffer, which it keeps alive
    and does not free."""

    def __init__(self, parent: DeviceBuffer, offset: int, nbytes: int):
        if offset < 0 or offset + nbytes > parent.nbytes:
            raise ValueError(f"view [{offset}, {offset + nbytes}) outside a buffer of {parent.nbytes} bytes")
        self.parent, self.nbytes = parent, int(nbytes)
        self.ptr = parent.ptr + int(offset)

    def free(self):
        self.ptr = None


class Compiled:
    """A compiled kernel (`KernelFn`)."""

    def __init__(self, text: str, dtype: str, lanes: int = 1, mode: int = FAST):
        h = ctypes.c_void_p()
        rc = lib().presk_hip_compile(text.encode(), dtype.encode(), lanes, mode, ctypes.byref(h))
        check(rc)
        self.handle = h.value
        self.text, self.dtype, self.lanes, self.mode = text, dtype, lanes, mode
        info = Info()
        check(lib().presk_hip_kernel_info(self.handle, ctypes.byref(info)))
        self.kind = info.kind.decode()
        self.order = info.order.decode()
        self.guarded = bool(info.guarded)
        self.n_inputs = info.n_inputs
        # integer (Quant) inputs, `int8/..` or `int4/..` in the header: each
        # has its scales' slot after the output
        head = text.split("->", 1)[0]
        self.n_quant = head.count(": int8/") + head.count(": int4/")
        self.split_bound = info.split_bound
        self.flops = info.flops
        self.bytes = info.bytes

    def read_back(self) -> str:
        """The text as the executor parsed it, printed back."""
        n = lib().presk_hip_kernel_text(self.handle, None, 0)
        buf = ctypes.create_string_buffer(n + 1)
        lib().presk_hip_kernel_text(self.handle, buf, n + 1)
        return buf.value.decode()

    def _table(self, ptrs):
        # the KernelFn table has no length: every slot the kernel reads must
        # be there (inputs, the output, a scales pointer per integer input,
        # the flag when guarded), or the launch would read a pointer past
        # the table's end
        need = self.n_inputs + 1 + self.n_quant + (1 if self.guarded else 0)
        if len(ptrs) < need or any(not p for p in ptrs):
            raise ValueError(f"a KernelFn table of {len(ptrs)} pointers for a kernel of {self.n_inputs} inputs"
                             f"{f' ({self.n_quant} integer, with scales)' if self.n_quant else ''}"
                             f"{' and a flag' if self.guarded else ''}: {need} or more non-null pointers needed")
        return (ctypes.c_void_p * len(ptrs))(*ptrs)

    def run(self, ptrs, lo=0, hi=None, stream=None):
        """One KernelFn call over device pointers [inputs..., output(, flag)]."""
        if hi is None:
            hi = max(self.split_bound, 0)
        check(lib().presk_hip_run(self.handle, self._table(ptrs), lo, hi, stream))

    def time(self, ptrs, warmup=3, reps=20, stream=None, lo=0, hi=None) -> float:
        if hi is None:
            hi = max(self.split_bound, 0)
        ms = ctypes.c_double()
        check(lib().presk_hip_time(self.handle, self._table(ptrs), lo, hi, stream, warmup, reps, ctypes.byref(ms)))
        return ms.value

    def __del__(self):
        try:
            if self.handle:
                lib().presk_hip_release(self.handle)
        except Exception:
            pass


def sync(stream=None):
    check(lib().presk_hip_sync(stream))


class HipExec:
    """The `KernelExec` of `--backend hip` (crates/presk-kernel/src/host.rs:28-95):
    runs each kernel of a launch on the device, kernels compiled once per text
    (the native backend's compile-on-first-use, crates/presk-cranelift/src/
    lib.rs:232-430), the overflow flag read after each launch (E7007,
    host.rs:140-177)."""

    def __init__(self, device: int = 0, mode: int = FAST):
        init(device)
        self.mode = mode
        self._cache: dict = {}
        self._flag = DeviceBuffer(4)

    def name(self) -> str:
        return "hip"

    def workers(self) -> int:
        return 1

    def emulates(self) -> bool:
        return False

    def codes(self) -> bool:
        return True

    def compiled(self, text: str, dtype: str, lanes: int = 1) -> Compiled:
        key = (text, dtype, lanes, self.mode)
        c = self._cache.get(key)
        if c is None:
            c = Compiled(text, dtype, lanes, self.mode)
            self._cache[key] = c
        return c

    def run(self, text: str, dtype: str, inputs: list, out: DeviceBuffer, lanes: int = 1, stream=None):
        """`KernelExec::run`: raises HipError E7007 when a narrowing store
        overflowed."""
        c = self.compiled(text, dtype, lanes)
        if len(inputs) != c.n_inputs:
            raise ValueError(f"{len(inputs)} input buffers for a kernel of {c.n_inputs} inputs")
        ptrs = [b.ptr for b in inputs] + [out.ptr]
        if c.guarded:
            self._flag.zero(stream)
            ptrs.append(self._flag.ptr)
        c.run(ptrs, stream=stream)
        if c.guarded:
            if int(self._flag.download(np.uint32, 1, stream)[0]):
                raise HipError(OVERFLOW, f"E7007: the kernel `{text.split(' (')[0][7:]}` stored a finite value past the largest "
                                         f"finite number of {dtype} (an overflow of its storage)")
        return c


# ---- the losses of a large vocabulary ---------------------------------------------

VALUE, GRAD = 1, 2
LOSS_WHAT = {"value": VALUE, "vjp": GRAD, "step": VALUE | GRAD}


_LOSS_BUFFERS = ("x", "w", "index", "teacher", "loss", "lse", "mean", "ct", "dx", "dw", "flag")


@functools.lru_cache(maxsize=1024)
def _loss_workspace(sizes: tuple, what: int, dx: bool, dw: bool) -> int:
    """presk_hip_loss_workspace (of the sizes alone: whether dx and dw are null
    is all that is looked at of the buffers)."""
    a, n = LossArgs(sizes[0].encode(), *sizes[1:]), ctypes.c_size_t()
    a.dx, a.dw = (1 if dx else None), (1 if dw else None)
    check(lib().presk_hip_loss_workspace(ctypes.byref(a), what, ctypes.byref(n)))
    return n.value


@functools.lru_cache(maxsize=1024)
def _loss_layout(sizes: tuple) -> tuple:
    """(each buffer's name, bytes, type and row length; the arguments before the
    buffers) of sizes and a type that are checked here."""
    dtype, n, model, vocab, top, tied = sizes[:6]
    _loss_workspace(sizes, VALUE, True, True)
    e = STORAGE_BYTES[dtype]
    x, w = n * (model or vocab) * e, model * vocab * e
    xr, wr, tr = model or vocab, model if tied else vocab, top or None
    return (tuple(zip(_LOSS_BUFFERS, (x, w, 8 * n * max(top, 1), e * n * top, 4 * n, 4 * n, 8, 4 * n, x, w, 4),
                      (dtype, dtype, "i64", dtype, "f32", "f32", "f32", "f32", dtype, dtype, None),
                      (xr, wr, tr, tr, None, None, None, None, xr, wr, None))),
            (dtype.encode(), *sizes[1:]))


# a torch dtype's name in the executor's terms, by the dtype object
_TORCH_TYPES: dict = {}
_TORCH_NAMES = {"torch.float32": "f32", "torch.bfloat16": "bf16", "torch.float16": "f16", "torch.int64": "i64"}


def _buffer(name: str, b, device, nbytes: int, ty: str | None = None, row: int | None = None) -> int:
    """The device pointer of a buffer of at least `nbytes` bytes: a
    DeviceBuffer, or a tensor of another library that says where and how
    large it is (torch's `data_ptr` and `nbytes`, contiguous, on `device`, any
    where that is not known, of type `ty`, its last axis `row` long where it has several)."""
    if hasattr(b, "data_ptr"):
        at = b.get_device()
        if at < 0:
            raise ValueError(f"{name} is not in device memory")
        if at != device and device not in (None, -1):
            raise ValueError(f"{name} is on device {at}, not {device}")
        have = _TORCH_TYPES.get(b.dtype)
        if have is None:
            have = _TORCH_TYPES[b.dtype] = _TORCH_NAMES.get(str(b.dtype), str(b.dtype))
        if have != ty and ty is not None:
            raise ValueError(f"{name} is {have}, not {ty}")
        if row is not None and b.ndim > 1 and b.shape[-1] != row:
            raise ValueError(f"{name} has rows of {b.shape[-1]}, not {row}")
        if not b.is_contiguous():
            raise ValueError(f"{name} is not contiguous")
        ptr, have = b.data_ptr(), b.nbytes
    else:
        ptr, have = b.ptr, b.nbytes
    if have < nbytes:
        raise ValueError(f"{name} has {have} bytes, {nbytes} needed")
    return ptr


def _place_of(bufs, stream) -> tuple:
    """(device, stream) of a call over these buffers.  With a tensor of torch's
    among them: the current device, on which the kernels run, and the caller's
    stream or, where it names none, torch's current one, on which the tensors
    were made and are read next (0 is the null stream)."""
    torch = sys.modules.get("torch")
    if torch is not None:
        for b in bufs:
            if isinstance(b, torch.Tensor) and b.is_cuda:
                now = torch.cuda.current_device()
                if now != _initialized and _initialized not in (None, -1):
                    raise ValueError(f"the current device is {now}, not {_initialized}")
                return now, torch.cuda.current_stream(now).cuda_stream if stream is None else stream
    return _initialized, stream


class Distill:
    """presk_hip_distill at fixed sizes: the divergence of given logits x
    [rows, vocab] from the softmax of a teacher's `top` logits, teacher[r, j]
    at column index[r, j] (i64; negative: unused), both at `temperature`.

    `value` writes loss, lse (f32 [rows]) and mean (f32 [2]: the counted rows'
    mean and their number), those given.  `vjp` writes the logits' cotangent
    dx from the forward's lse, for a row's cotangent ct (f32 [rows]), or for
    the mean's where mean is given in its place.  `value_and_grad` does both,
    for ct or else the mean.  Buffers are DeviceBuffers or torch tensors; a call
    with tensors that names no stream goes to torch's current one, others to
    the null stream.  `work` is workspace(kind) bytes of the caller's, or, not
    given, a buffer that this object keeps for the call's stream (with any
    smaller one outgrown, which a captured call may still use): calls that
    share a workspace, their captured graphs among them, run one after another."""

    head = False

    def __init__(self, dtype: str, rows: int, vocab: int, top: int, temperature: float = 1.0):
        self._set(dtype, rows, 0, vocab, top, False, temperature)

    def _set(self, dtype, rows, model, vocab, top, tied, temperature):
        self.dtype, self.rows, self.model, self.vocab, self.top = dtype, int(rows), int(model), int(vocab), int(top)
        self.tied, self.temperature = bool(tied), float(temperature)
        self._sizes = (self.dtype, self.rows, self.model, self.vocab, self.top, self.tied, self.temperature)
        self._work = None       # the workspace last used of the object's own
        self._works = {}        # device and stream -> those taken for it, the largest last
        self._specs, self._fixed = _loss_layout(self._sizes)

    def workspace(self, kind: str, dx: bool = True, dw: bool = True) -> int:
        """Bytes of workspace for `value`, `vjp` or `step` (value_and_grad),
        with the gradients asked for."""
        return _loss_workspace(self._sizes, LOSS_WHAT[kind], dx, dw and self.head)

    @property
    def _outgrown(self) -> list:
        return [b for own in self._works.values() for b in own if b is not self._work]

    def _own_work(self, need: int, device, stream):
        own = self._works.setdefault((device, getattr(stream, "value", stream) or 0), [])
        if not own or own[-1].nbytes < need:
            own.append(DeviceBuffer(need))
        self._work = own[-1]
        return self._work

    def args(self, kind: str, x=None, w=None, index=None, teacher=None, loss=None, lse=None, mean=None, ct=None, dx=None, dw=None,
             flag=None, work=None, stream=None, device=None) -> LossArgs:
        """The arguments of a call on `stream`, each buffer checked against its
        size and `device` (the one initialised)."""
        device = _initialized if device is None else device
        need = self.workspace(kind, dx is not None, dw is not None)
        if work is None:
            work = self._own_work(need, device, stream)
        bufs = [None if b is None else _buffer(s[0], b, device, *s[1:])
                for s, b in zip(self._specs, (x, w, index, teacher, loss, lse, mean, ct, dx, dw, flag))]
        return LossArgs(*self._fixed, *bufs, _buffer("work", work, device, need), work.nbytes)

    def _call(self, kind, stream, **bufs):
        device, stream = _place_of(bufs.values(), stream)
        a = self.args(kind, stream=stream, device=device, **bufs)
        f = lib().presk_hip_head_loss if self.head else lib().presk_hip_distill
        check(f(ctypes.byref(a), LOSS_WHAT[kind], stream))

    def value(self, x, index, teacher, loss=None, lse=None, mean=None, work=None, stream=None):
        self._call("value", stream, x=x, index=index, teacher=teacher, loss=loss, lse=lse, mean=mean, work=work)

    def vjp(self, x, index, teacher, lse, dx, ct=None, mean=None, flag=None, work=None, stream=None):
        self._call("vjp", stream, x=x, index=index, teacher=teacher, lse=lse, dx=dx, ct=ct, mean=mean, flag=flag, work=work)

    def value_and_grad(self, x, index, teacher, dx, loss=None, lse=None, mean=None, ct=None, flag=None, work=None, stream=None):
        self._call("step", stream, x=x, index=index, teacher=teacher, dx=dx, loss=loss, lse=lse, mean=mean, ct=ct, flag=flag, work=work)


class HeadLoss(Distill):
    """presk_hip_head_loss at fixed sizes: the loss of the logits x . w, which
    are the workspace's.  x [rows, model]; w [model, vocab], or [vocab, model] when
    `tied`; `top` 0: the softmax cross entropy against index[r] (negative: the
    row does not count); `top` k: Distill's loss.  The methods are Distill's,
    with w, and the gradients dx and dw, of which one may be left out."""

    head = True

    def __init__(self, dtype: str, rows: int, model: int, vocab: int, tied: bool = False, top: int = 0, temperature: float = 1.0):
        if int(model) < 1:
            raise ValueError(f"a head of model {model}")
        self._set(dtype, rows, model, vocab, top, tied, temperature)

    def value(self, x, w, index, teacher=None, loss=None, lse=None, mean=None, work=None, stream=None):
        self._call("value", stream, x=x, w=w, index=index, teacher=teacher, loss=loss, lse=lse, mean=mean, work=work)

    def vjp(self, x, w, index, lse, dx=None, dw=None, teacher=None, ct=None, mean=None, flag=None, work=None, stream=None):
        self._call("vjp", stream, x=x, w=w, index=index, teacher=teacher, lse=lse, dx=dx, dw=dw, ct=ct, mean=mean, flag=flag, work=work)

    def value_and_grad(self, x, w, index, dx=None, dw=None, teacher=None, loss=None, lse=None, mean=None, ct=None, flag=None, work=None,
                       stream=None):
        self._call("step", stream, x=x, w=w, index=index, teacher=teacher, dx=dx, dw=dw, loss=loss, lse=lse, mean=mean, ct=ct, flag=flag,
                   work=work)
