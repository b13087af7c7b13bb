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
import struct
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
           "presk_hip_loss_workspace", "presk_hip_head_loss", "presk_hip_distill", "presk_hip_batch_add_head_loss", "presk_hip_batch_add_distill",
           "presk_hip_attention_workspace", "presk_hip_attention", "presk_hip_batch_add_attention",
           "presk_hip_head_rotary_workspace", "presk_hip_head_rotary", "presk_hip_batch_add_head_rotary"]


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
        for name in ("attention", "head_rotary"):
            getattr(L, f"presk_hip_{name}_workspace").argtypes = [vp, i32, ctypes.POINTER(ctypes.c_size_t)]
            getattr(L, f"presk_hip_{name}").argtypes = [vp, i32, vp]
            getattr(L, f"presk_hip_batch_add_{name}").argtypes = [vp, vp, i32]
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
_TORCH_NAMES = {"torch.float64": "f64", "torch.float32": "f32", "torch.bfloat16": "bf16", "torch.float16": "f16", "torch.int64": "i64"}


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
    smaller one outgrown, which a captured call's graph may still use, and the
    object with it): calls that
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


# ---- a block's attention ------------------------------------------------------------


_HEADS_KINDS = {"value": 1, "vjp": 2}
_LAYOUTS = ("bshd", "bhsd")
# storage types' names where the C side finds them, for the process's life
_C_NAMES = {t: ctypes.create_string_buffer(t.encode()) for t in ("f32", "bf16", "f16")}
_NO_HEADS, _NO_MASK = (0, 0, 0, 0), (0, 0, 0)


def _c_name(dtype: str) -> int:
    if dtype not in _C_NAMES:
        _C_NAMES[dtype] = ctypes.create_string_buffer(str(dtype).encode())
    return ctypes.addressof(_C_NAMES[dtype])


@functools.lru_cache(maxsize=4096)
def _heads_sizes(cls, fixed: tuple, layout: str, batch: int, lengths: tuple, heads: tuple, d: int) -> tuple:
    """What follows from an operator's sizes, which are checked here: its
    arguments' head, its workspaces, and of queries' and of keys' tensors the axes
    and a dense one's strides of batch, row and head."""
    if layout not in _LAYOUTS:
        raise ValueError(f"a layout {layout!r}, not one of {', '.join(_LAYOUTS)}")
    head = (_c_name(fixed[0]), *fixed[1:])
    n, need = ctypes.c_size_t(), {}
    args = cls._pack(fixed, {}, 0, 0)
    for kind, what in _HEADS_KINDS.items():
        check(getattr(lib(), f"presk_hip_{cls._name}_workspace")(args, what, ctypes.byref(n)))
        need[kind] = n.value
    specs = []
    for m, h in zip(lengths, heads):
        specs.append(((batch, m, h, d), m * h * d, h * d, d) if layout == "bshd" else ((batch, h, m, d), m * h * d, d, m * d))
    return head, need, specs


class _HeadsCall:
    """What the operators over tensors of heads share: their tensors' checks,
    their workspace and their calls.  A tensor is a DeviceBuffer, dense in
    `layout`, or a torch tensor of that layout's four axes with any strides whose
    last is 1 (a slice of a packed projection, of a longer cache)."""

    _name: str                  # of the library's calls
    # a C call's arguments after the sizes: a tensor's name -> whether it is a
    # key's, then the other buffers, then the workspace
    _tensors: dict
    _plain: tuple

    def _init(self, layout: str, fixed: tuple, lengths: tuple):
        self.layout, self._fixed = layout, fixed
        self._head, self._need, self._specs = _heads_sizes(type(self), fixed, layout, self.batch, lengths, (self.heads, self.kv_heads), self.head_dim)
        self._works = {}        # device and stream -> the workspaces taken for it, the largest last

    def workspace(self, kind: str) -> int:
        """Bytes of workspace for `value` or `vjp`."""
        return self._need[kind]

    def elements(self, name: str) -> int:
        """The element count of a tensor."""
        return self.batch * self._specs[self._tensors[name]][1]

    def _heads(self, name: str, t, device) -> tuple:
        """(address, strides of batch, row and head) of a tensor that is checked here."""
        shape, *strides = self._specs[self._tensors[name]]
        if not hasattr(t, "data_ptr"):
            need = self.elements(name) * STORAGE_BYTES[self.dtype]
            if t.nbytes < need:
                raise ValueError(f"{name} has {t.nbytes} bytes, {need} needed")
            return (t.ptr, *strides)
        at = t.get_device()
        if at < 0:
            raise ValueError(f"{name} is not in device memory")
        if at != device and device not in (None, -1):
            raise ValueError(f"{name} is on device {at}, not {device}")
        if _TORCH_TYPES.get(t.dtype) != self.dtype and _type_name(t) != self.dtype:
            raise ValueError(f"{name} is {_type_name(t)}, not {self.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name} is {list(t.shape)}, not {list(shape)}")
        sb, s1, s2, one = t.stride()
        if one != 1 and shape[3] > 1 and t.numel():
            raise ValueError(f"{name}'s heads are not contiguous")
        return (t.data_ptr(), sb, s1, s2) if self.layout == "bshd" else (t.data_ptr(), sb, s2, s1)

    def _own_work(self, need: int, device, stream):
        own = self._works.setdefault((device, getattr(stream, "value", stream) or 0), [])
        if not own or own[-1].nbytes < need:
            own.append(DeviceBuffer(need))
        return own[-1]

    def args(self, kind: str, work=None, stream=None, device=None, **bufs) -> bytes:
        """The C call's arguments on `stream`, each buffer checked against its
        size and `device` (the one initialised)."""
        if unknown := sorted(set(bufs) - set(self._tensors) - set(self._plain)):
            raise TypeError(f"{self._name} has no argument {unknown[0]}")
        return self._args(kind, work, stream, _initialized if device is None else device, bufs)

    @classmethod
    def _pack(cls, fixed, got, work, work_bytes) -> bytes:
        """Those of buffers' addresses (and strides)."""
        h = [x for n in cls._tensors for x in got.get(n, _NO_HEADS)]
        for n in cls._plain:
            h += got.get(n, _NO_MASK) if n == "mask" else (got.get(n, 0),)
        return cls._struct.pack(_c_name(fixed[0]), *fixed[1:], *h, work, work_bytes)

    def _args(self, kind, work, stream, device, bufs: dict) -> bytes:
        if work is None and self._works_for(kind):
            work = self._own_work(self._need[kind], device, stream)
        given, got = bufs.get, []
        for n in self._tensors:
            b = given(n)
            got += _NO_HEADS if b is None else self._heads(n, b, device)
        for n in self._plain:
            b = given(n)
            if n == "mask":
                got += _NO_MASK if b is None else self._mask(b, device)
            else:
                got.append(0 if b is None else _buffer(n, b, device, *self._others[n]))
        if work is None:
            return self._struct.pack(*self._head, *got, 0, 0)
        return self._struct.pack(*self._head, *got, _buffer("work", work, device, self._need[kind]), work.nbytes)

    def _works_for(self, kind: str) -> bool:
        return True

    def _call(self, kind, stream, work, bufs: dict):
        device, stream = _place_of(bufs.values(), stream)
        a = self._args(kind, work, stream, device, bufs)
        check(self._launch(lib())(a, _HEADS_KINDS[kind], stream))


def _type_name(t) -> str:
    have = _TORCH_TYPES.get(t.dtype)
    if have is None:
        have = _TORCH_TYPES[t.dtype] = _TORCH_NAMES.get(str(t.dtype), str(t.dtype))
    return have


class Attention(_HeadsCall):
    """presk_hip_attention at fixed sizes: softmax(scale q k^T) v of q [batch,
    q_len, heads, head_dim] and k, v [batch, k_len, kv_heads, head_dim] (axes in that
    order, `layout` "bshd", or "bhsd"), head h with key head h // (heads //
    kv_heads), without the weights in memory; `scale` head_dim ** -0.5 unless given.

    Query i of a sequence stands at position first + i among its keys and reads
    those below `lens` (i64 [batch]; none given: k_len): all of them; with `causal`
    those up to its position, with a `window` the last so many of these; with
    `mask_cols` those before `first` and, of the next mask_cols, those whose byte
    of its row of `mask` ([batch, q_len, mask_cols] or, shared, [q_len, mask_cols];
    bool or uint8) is not 0.  `first` (i64 [batch]) not given: the queries (the
    mask's columns) are the last keys.  A query that reads no key has output 0, lse
    -inf and no gradients.

    `value` writes o and, given, lse (f32 [batch, heads, q_len]).  `vjp`, from the
    forward's o and lse and the cotangent do, writes those of dq, dk and dv that
    are given.  Buffers are DeviceBuffers or torch tensors; a call with tensors
    that names no stream goes to torch's current one, others to the null stream.
    `work` is workspace(kind) bytes of the caller's, or, not given, a buffer that
    this object keeps for the call's stream (a captured call's graph needs the object
    as long as it is replayed): calls that share a workspace, their captured graphs
    among them, run one after another."""

    _name = "attention"
    _launch = staticmethod(lambda lib: lib.presk_hip_attention)
    # presk_hip_attn
    _struct = struct.Struct("@P8qid" + "Pqqq" * 8 + "4P2qPPN")
    _tensors = {"q": False, "k": True, "v": True, "o": False, "do": False, "dq": False, "dk": True, "dv": True}
    _plain = ("lse", "lens", "first", "mask", "flag")

    def __init__(self, dtype: str, batch: int, heads: int, kv_heads: int, q_len: int, k_len: int, head_dim: int, causal: bool = False,
                 window: int = 0, mask_cols: int = 0, scale: float | None = None, layout: str = "bshd"):
        self.dtype, self.batch, self.heads, self.kv_heads = dtype, int(batch), int(heads), int(kv_heads)
        self.q_len, self.k_len, self.head_dim = int(q_len), int(k_len), int(head_dim)
        self.causal, self.window, self.mask_cols = bool(causal), int(window), int(mask_cols)
        self.scale = float(scale) if scale is not None else max(self.head_dim, 1) ** -0.5
        self._init(layout, (self.dtype, self.batch, self.heads, self.kv_heads, self.q_len, self.k_len, self.head_dim, self.window,
                            self.mask_cols, self.causal, self.scale), (self.q_len, self.k_len))
        rows = 4 * self.batch * self.heads * self.q_len
        self._others = {"lse": (rows, "f32"), "lens": (8 * self.batch, "i64"), "first": (8 * self.batch, "i64"), "flag": (4, None)}

    def _mask(self, m, device) -> tuple:
        if not self.mask_cols:
            raise ValueError("a mask of no columns (mask_cols)")
        if not hasattr(m, "data_ptr"):
            return _buffer("mask", m, device, self.batch * self.q_len * self.mask_cols), self.q_len * self.mask_cols, self.mask_cols
        at = m.get_device()
        if at < 0:
            raise ValueError("mask is not in device memory")
        if at != device and device not in (None, -1):
            raise ValueError(f"mask is on device {at}, not {device}")
        if str(m.dtype) not in ("torch.bool", "torch.uint8"):
            raise ValueError(f"mask is {m.dtype}, not bool or uint8")
        want = (self.q_len, self.mask_cols)
        if tuple(m.shape) not in (want, (self.batch,) + want):
            raise ValueError(f"mask is {list(m.shape)}, not {[self.batch, *want]} or {list(want)}")
        st = m.stride()
        if st[-1] != 1 and self.mask_cols > 1 and m.numel():
            raise ValueError("mask's rows are not contiguous")
        return m.data_ptr(), st[0] if m.ndim == 3 else 0, st[-2]

    def value(self, q, k, v, o, lse=None, lens=None, first=None, mask=None, flag=None, work=None, stream=None):
        self._call("value", stream, work, {"q": q, "k": k, "v": v, "o": o, "lse": lse, "lens": lens, "first": first, "mask": mask, "flag": flag})

    def vjp(self, q, k, v, o, lse, do, dq=None, dk=None, dv=None, lens=None, first=None, mask=None, flag=None, work=None, stream=None):
        self._call("vjp", stream, work, {"q": q, "k": k, "v": v, "o": o, "lse": lse, "do": do, "dq": dq, "dk": dk, "dv": dv, "lens": lens,
                                         "first": first, "mask": mask, "flag": flag})


def rotary_frequencies(rotary: int, base: float = 1e4) -> np.ndarray:
    """The rotation's radians a position, f64 [rotary / 2]: base ** (-2 r / rotary)."""
    return base ** (-2.0 * np.arange(rotary // 2) / max(rotary, 1))


class HeadRotary(_HeadsCall):
    """presk_hip_head_rotary at fixed sizes: each head of q [batch, seq, heads,
    head_dim] and k [batch, seq, kv_heads, head_dim] (kv_heads 0: q alone; axes by
    `layout`, as Attention's) normed, with `norm`, by its root mean square and the
    gains gq and gk ([head_dim]; not given: ones), and its first `rotary` elements
    (all, unless given) turned by the token's position: pair r by at * freq[r]
    radians, freq f64 [rotary / 2] (rotary_frequencies) and `at` i64 [batch, seq]
    (not given: 0, 1, ..).  `pairs` "half": elements r and r + rotary / 2; "even":
    2 r and 2 r + 1.

    `value` writes yq and yk, which may be q and k.  `vjp`, from the cotangents dyq
    and dyk and, with `norm`, q and k, writes dq and dk (which may be dyq and dyk)
    and those of dgq and dgk that are given.  Buffers, streams and `work` as
    Attention's; only a gradient with `norm` needs any workspace."""

    _name = "head_rotary"
    _launch = staticmethod(lambda lib: lib.presk_hip_head_rotary)
    # presk_hip_rot
    _struct = struct.Struct("@P6qiid" + "Pqqq" * 8 + "8PN")
    _tensors = {"q": False, "k": True, "yq": False, "yk": True, "dyq": False, "dyk": True, "dq": False, "dk": True}
    _plain = ("freq", "at", "gq", "gk", "dgq", "dgk", "flag")

    def __init__(self, dtype: str, batch: int, seq: int, heads: int, kv_heads: int, head_dim: int, rotary: int | None = None,
                 norm: bool = False, eps: float = 1e-6, pairs: str = "half", layout: str = "bshd"):
        if pairs not in ("half", "even"):
            raise ValueError(f"pairs {pairs!r}, not half or even")
        self.dtype, self.batch, self.seq, self.heads, self.kv_heads = dtype, int(batch), int(seq), int(heads), int(kv_heads)
        self.head_dim, self.rotary = int(head_dim), int(head_dim if rotary is None else rotary)
        self.norm, self.eps, self.pairs = bool(norm), float(eps), pairs
        self._init(layout, (self.dtype, self.batch, self.seq, self.heads, self.kv_heads, self.head_dim, self.rotary, self.norm,
                            self.pairs == "even", self.eps), (self.seq, self.seq))
        gain = (self.head_dim * STORAGE_BYTES[self.dtype], self.dtype)
        self._others = {"freq": (4 * self.rotary, "f64"), "at": (8 * self.batch * self.seq, "i64"), "flag": (4, None),
                        "gq": gain, "gk": gain, "dgq": gain, "dgk": gain}

    def _works_for(self, kind: str) -> bool:
        return self.norm and kind == "vjp"

    def value(self, q, freq, yq, k=None, yk=None, at=None, gq=None, gk=None, flag=None, work=None, stream=None):
        self._call("value", stream, work, {"q": q, "k": k, "yq": yq, "yk": yk, "freq": freq, "at": at, "gq": gq, "gk": gk, "flag": flag})

    def vjp(self, freq, dyq, dq, dyk=None, dk=None, q=None, k=None, at=None, gq=None, gk=None, dgq=None, dgk=None, flag=None, work=None,
            stream=None):
        self._call("vjp", stream, work, {"q": q, "k": k, "dyq": dyq, "dyk": dyk, "dq": dq, "dk": dk, "freq": freq, "at": at, "gq": gq, "gk": gk,
                                         "dgq": dgq, "dgk": dgk, "flag": flag})
