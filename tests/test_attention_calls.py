"""What hip.Attention and hip.HeadRotary take and refuse, without a GPU: the
library checks every call before it launches anything, and where a call that
passes would launch, the launch is recorded in its place."""
import ctypes
import struct

import pytest

torch = pytest.importorskip("torch")

from presk_amd import hip  # noqa: E402

CURRENT = 0x5000
BF = torch.bfloat16


class Tensor(torch.Tensor):
    """A tensor that says it is in device memory."""

    at = 0
    is_cuda = True

    def get_device(self):
        return Tensor.at


def dev(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Tensor)


class Memory:
    """A buffer of device memory that is never touched."""

    taken = 0

    def __init__(self, nbytes):
        Memory.taken += 1
        self.nbytes, self.ptr = nbytes, Memory.taken << 36


class Library:
    """The executor's library with the launches taken out: a call's checks run,
    those of a step of a sequence, which are the same."""

    def __init__(self, real, calls):
        self.real, self.calls, self.batch = real, calls, ctypes.c_void_p()
        hip.check(real.presk_hip_batch_create(ctypes.byref(self.batch)))

    def __getattr__(self, name):
        return getattr(self.real, name)

    def _call(self, name, a, what, stream):
        rc = getattr(self.real, "presk_hip_batch_add_" + name)(self.batch, a, what)
        if rc == hip.OK:
            self.calls.append((a, what, stream))
        return rc

    def presk_hip_attention(self, a, what, stream):
        return self._call("attention", a, what, stream)

    def presk_hip_head_rotary(self, a, what, stream):
        return self._call("head_rotary", a, what, stream)


@pytest.fixture
def calls(monkeypatch):
    got, real = [], hip.lib()
    library = Library(real, got)
    monkeypatch.setattr(hip, "lib", lambda: library)
    monkeypatch.setattr(hip, "DeviceBuffer", Memory)
    monkeypatch.setattr(hip, "_initialized", 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: type("S", (), {"cuda_stream": CURRENT + d})())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    yield got
    real.presk_hip_batch_release(library.batch)


def attention(**changed):
    sizes = dict(dtype="bf16", batch=2, heads=4, kv_heads=2, q_len=8, k_len=8, head_dim=64)
    sizes.update(changed)
    return hip.Attention(**sizes)


def buffers(kind="value", **changed):
    b = {"q": dev(2, 8, 4, 64), "k": dev(2, 8, 2, 64), "v": dev(2, 8, 2, 64), "o": dev(2, 8, 4, 64), "lse": dev(2, 4, 8, dtype=torch.float32)}
    if kind == "vjp":
        b.update(do=dev(2, 8, 4, 64), dq=dev(2, 8, 4, 64), dk=dev(2, 8, 2, 64), dv=dev(2, 8, 2, 64))
    b.update(changed)
    return {n: x for n, x in b.items() if x is not None}


def test_the_arguments_are_the_headers():
    """The packed arguments as the C structures lay them out."""
    heads = type("Heads", (ctypes.Structure,), {"_fields_": [("p", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("b", "s", "h")]})
    tail = [("work", ctypes.c_void_p), ("work_bytes", ctypes.c_size_t)]
    fields = [("dtype", ctypes.c_char_p)] + [(f"n{i}", ctypes.c_int64) for i in range(8)] + [("causal", ctypes.c_int32), ("scale", ctypes.c_double)]
    fields += [(f"h{i}", heads) for i in range(8)] + [(f"p{i}", ctypes.c_void_p) for i in range(4)]
    fields += [("mask_batch", ctypes.c_int64), ("mask_row", ctypes.c_int64), ("flag", ctypes.c_void_p)] + tail
    c = type("Attn", (ctypes.Structure,), {"_fields_": fields})
    assert hip.Attention._struct.size == ctypes.sizeof(c)
    a = attention(causal=True, scale=0.25)
    got = c.from_buffer_copy(a._pack(a._fixed, {"q": (1, 2, 3, 4), "dv": (5, 6, 7, 8), "lse": 9, "mask": (10, 11, 12), "flag": 13}, 14, 15))
    assert (got.dtype, got.n0, got.n5, got.n7, got.causal, got.scale) == (b"bf16", 2, 64, 0, 1, 0.25)
    assert (got.h0.p, got.h0.h, got.h7.p, got.h7.h, got.p0, got.p3, got.mask_batch, got.mask_row) == (1, 4, 5, 8, 9, 10, 11, 12)
    assert (got.flag, got.work, got.work_bytes) == (13, 14, 15)
    fields = [("dtype", ctypes.c_char_p)] + [(f"n{i}", ctypes.c_int64) for i in range(6)] + [("norm", ctypes.c_int32), ("even", ctypes.c_int32),
                                                                                           ("eps", ctypes.c_double)]
    fields += [(f"h{i}", heads) for i in range(8)] + [(f"p{i}", ctypes.c_void_p) for i in range(7)] + tail
    c = type("Rot", (ctypes.Structure,), {"_fields_": fields})
    assert hip.HeadRotary._struct.size == ctypes.sizeof(c)
    r = hip.HeadRotary("f16", 1, 2, 3, 4, 64, rotary=32, norm=True, eps=0.5, pairs="even")
    got = c.from_buffer_copy(r._pack(r._fixed, {"dk": (1, 2, 3, 4), "freq": 5, "dgk": 6, "flag": 7}, 8, 9))
    assert (got.dtype, got.n5, got.norm, got.even, got.eps, got.h7.p, got.p0, got.p5, got.p6) == (b"f16", 32, 1, 1, 0.5, 1, 5, 6, 7)
    assert (got.work, got.work_bytes) == (8, 9)
    assert struct.calcsize("P") == 8


@pytest.mark.parametrize("changed, text", [
    (dict(dtype="f64"), "E7005.*storage type `f64`"), (dict(dtype="e8m15"), "E7005"), (dict(dtype="f32", head_dim=130), "E7005.*in f32"),
    (dict(heads=4, kv_heads=3), "whole groups"), (dict(kv_heads=0), "whole groups"), (dict(heads=0), "heads 0"), (dict(head_dim=0), "head_dim 0"),
    (dict(head_dim=257), "head_dim 257"), (dict(batch=-1), "batch -1"), (dict(q_len=-1), "q_len -1"), (dict(k_len=1 << 28), "k_len"),
    (dict(window=4), "window without causal"), (dict(window=-1, causal=True), "window -1"), (dict(mask_cols=-2), "mask_cols"),
    (dict(mask_cols=8, causal=True), "mask and causal"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(batch=1 << 20, heads=4096, kv_heads=1), "past what a launch holds"),
])
def test_sizes_that_are_refused(changed, text):
    with pytest.raises(hip.HipError, match=text):
        attention(**changed)


def test_a_layout_that_there_is_not():
    with pytest.raises(ValueError, match="layout 'sbhd'"):
        attention(layout="sbhd")


@pytest.mark.parametrize("kind, changed, text", [
    ("value", dict(q=dev(2, 8, 4, 32)), r"q is \[2, 8, 4, 32\], not \[2, 8, 4, 64\]"),
    ("value", dict(k=dev(2, 8, 4, 64)), "k is"),
    ("value", dict(v=dev(2, 8, 2, 64, dtype=torch.float16)), "v is f16, not bf16"),
    ("value", dict(v=dev(2, 8, 64, 2).transpose(2, 3)), "v's heads are not contiguous"),
    ("value", dict(lens=dev(2, dtype=torch.int32)), "lens is torch.int32"),
    ("value", dict(first=dev(1, dtype=torch.int64)), "first has 8 bytes, 16 needed"),
    ("value", dict(lse=dev(2, 4, 7, dtype=torch.float32)), "lse has"),
    ("value", dict(lse=dev(2, 4, 8, dtype=BF)), "lse is bf16"),
    ("value", dict(mask=dev(8, 8, dtype=torch.bool)), "a mask of no columns"),
    ("value", dict(work=dev(16, dtype=torch.uint8)), "work has 16 bytes"),
    ("vjp", dict(dq=None, dk=None, dv=None), "a gradient without an output"),
])
def test_buffers_that_are_refused(calls, kind, changed, text):
    op = attention()
    b = buffers(kind, **changed)
    with pytest.raises((ValueError, hip.HipError), match=text):
        getattr(op, kind)(**b)
    assert not calls


def test_calls_that_pass(calls):
    op = attention(causal=True, window=3)
    op.value(**buffers())
    op.value(**buffers(lse=None, lens=dev(2, dtype=torch.int64), first=dev(2, dtype=torch.int64)), stream=0x7000)
    op.vjp(**buffers("vjp", dk=None, dv=None))
    m = attention(mask_cols=8)
    for mask in (dev(2, 8, 8, dtype=torch.bool), dev(8, 8, dtype=torch.uint8), dev(1, 8, 8, dtype=torch.bool).expand(2, 8, 8)):
        m.value(**buffers(mask=mask))
    assert [(what, s) for _, what, s in calls] == [(1, CURRENT), (1, 0x7000), (2, CURRENT)] + [(1, CURRENT)] * 3
    m = Memory(2 * 8 * 4 * 64 * 2)
    attention(kv_heads=4).value(m, Memory(m.nbytes), Memory(m.nbytes), Memory(m.nbytes))
    assert calls[-1][2] is None


@pytest.mark.parametrize("mask, text", [
    (dev(2, 8, 8, dtype=torch.float32), "mask is torch.float32"), (dev(8, 7, dtype=torch.bool), r"mask is \[8, 7\]"),
    (dev(2, 8, 8, dtype=torch.bool).transpose(1, 2), "mask's rows"), (None, "mask is null"),
])
def test_masks_that_are_refused(calls, mask, text):
    with pytest.raises((ValueError, hip.HipError), match=text):
        attention(mask_cols=8).value(**buffers(mask=mask))


def test_outputs_that_meet(calls):
    op = attention()
    b = buffers()
    with pytest.raises(hip.HipError, match="o meets q"):
        op.value(**{**b, "o": b["q"]})
    with pytest.raises(hip.HipError, match="o has elements that meet"):
        op.value(**{**b, "o": dev(1, 8, 4, 64).expand(2, 8, 4, 64)})
    with pytest.raises(hip.HipError, match="lse meets o"):
        op.value(**{**b, "lse": b["o"].view(torch.float32)})
    # slices side by side in one buffer's rows are apart, the same slice is not
    packed, grads = dev(2, 8, 8, 64), dev(2, 8, 8, 64)
    q, k, v = packed.split((4, 2, 2), 2)
    dq, dk, dv = grads.split((4, 2, 2), 2)
    v8 = buffers("vjp", q=q, k=k, v=v, dq=dq, dk=dk, dv=dv)
    op.vjp(**v8)
    op.vjp(**{**v8, "dq": packed.split((4, 2, 2), 2)[0], "q": b["q"]})
    for same in ({"dk": dv}, {"dv": dq[:, :, 1:3]}, {"dk": k}, {"dk": packed[:, :, 5:7]}):
        with pytest.raises(hip.HipError, match="meets"):
            op.vjp(**{**v8, **same})
    assert len(calls) == 2


def test_strides_that_are_refused(calls):
    op = attention(batch=1, heads=1, kv_heads=1)
    row = dev(64 + 7)
    lap = row.as_strided((1, 8, 1, 64), (64, 1, 64, 1))
    b = {n: dev(1, 8, 1, 64) for n in ("q", "k", "v", "o")}
    with pytest.raises(hip.HipError, match="k has rows of 64 elements 1 apart"):
        op.value(**{**b, "k": lap})
    far = torch.empty(64, dtype=BF).as_strided((1, 8, 1, 64), (0, 0, 0, 1)).as_subclass(Tensor)
    with pytest.raises(hip.HipError, match="k has rows of 64 elements 0 apart"):
        op.value(**{**b, "k": far})


def test_rows_far_apart(calls):
    """A tile's rows lie within 2^31 bytes, past which an offset stands for none."""
    op = attention(batch=1, heads=1, kv_heads=1)
    b = {n: dev(1, 8, 1, 64) for n in ("q", "k", "v", "o")}
    wide = torch.empty(7 * 2 ** 23 + 64, dtype=BF)
    op.value(**{**b, "k": wide.as_strided((1, 8, 1, 64), (0, 2 ** 23 - 8, 0, 1)).as_subclass(Tensor)})
    with pytest.raises(hip.HipError, match=r"k has rows 2\^24 bytes apart or more"):
        op.value(**{**b, "k": wide.as_strided((1, 8, 1, 64), (0, 2 ** 23, 0, 1)).as_subclass(Tensor)})


def test_the_own_workspace_is_a_streams_and_devices(calls, monkeypatch):
    op = attention()
    for s in (0x10, 0x20, 0x10, 0):
        op.value(**buffers(), stream=s)
    size = hip.Attention._struct.size
    works = [struct.unpack_from("P", a, size - 16)[0] for a, _, _ in calls]
    assert works[0] == works[2] and len(set(works)) == 3
    monkeypatch.setattr(hip, "_initialized", None)
    monkeypatch.setattr(Tensor, "at", 1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    op.value(**buffers(), stream=0)
    assert struct.unpack_from("P", calls[-1][0], size - 16)[0] not in works


def test_tensors_of_another_device_are_refused(calls, monkeypatch):
    b = buffers()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device is 1, not 0"):
        attention().value(**b)
    monkeypatch.setattr(hip, "_initialized", None)
    with pytest.raises(ValueError, match="q is on device 0, not 1"):
        attention().value(**b)


def rotary(**changed):
    sizes = dict(dtype="bf16", batch=2, seq=8, heads=4, kv_heads=2, head_dim=64)
    sizes.update(changed)
    return hip.HeadRotary(**sizes)


@pytest.mark.parametrize("changed, text", [
    (dict(dtype="f64"), "E7005"), (dict(rotary=3), "rotary 3"), (dict(rotary=66), "rotary 66"), (dict(rotary=-2), "rotary -2"),
    (dict(head_dim=300), "head_dim 300"), (dict(heads=0), "heads 0"), (dict(kv_heads=-1), "kv_heads -1"), (dict(norm=True, eps=-1.0), "eps"),
    (dict(norm=True, eps=float("nan")), "eps"), (dict(seq=-1), "seq -1"), (dict(batch=1 << 20, seq=1 << 20), "past what a launch holds"),
])
def test_rotary_sizes_that_are_refused(changed, text):
    with pytest.raises(hip.HipError, match=text):
        rotary(**changed)
    with pytest.raises(ValueError, match="pairs 'odd'"):
        rotary(pairs="odd")


def test_rotary_calls(calls):
    f = dev(32, dtype=torch.float64)
    q, k, yq, yk = dev(2, 8, 4, 64), dev(2, 8, 2, 64), dev(2, 8, 4, 64), dev(2, 8, 2, 64)
    g = dev(64)
    op, normed = rotary(), rotary(norm=True)
    op.value(q, f, yq, k=k, yk=yk)
    op.value(q, f, q, k=k, yk=k)                        # in place
    op.vjp(f, q, q, dyk=k, dk=yk)
    normed.vjp(f, yq, yq, dyk=yk, dk=yk, q=q, k=k, gq=g, dgq=dev(64))
    rotary(kv_heads=0).value(q, f, yq)
    assert len(calls) == 5
    for call, text in [(lambda: op.value(q, f, yq), "k is null"), (lambda: op.value(q, dev(32, dtype=torch.float32), yq, k=k, yk=yk), "freq is f32"),
                       (lambda: op.value(q, dev(31, dtype=torch.float64), yq, k=k, yk=yk), "freq has"),
                       (lambda: op.value(q, f, yq, k=k, yk=yk, at=dev(8, dtype=torch.int64)), "at has"),
                       (lambda: op.value(q, f, yq, k=k, yk=yk, gq=g), "gains without a norm"),
                       (lambda: op.value(q, f, yq, k=k, yk=q[:, :, :2]), "yk meets q"),
                       (lambda: op.value(q, f, q[:, :, torch.arange(4)].as_subclass(Tensor), k=k, yk=k), None),
                       (lambda: normed.vjp(f, yq, yq, dyk=yk, dk=yk), "q is null"),
                       (lambda: normed.vjp(f, yq, q, dyk=yk, dk=yk, q=q, k=k), "dq meets q")]:
        if text is None:
            call()
            continue
        with pytest.raises((ValueError, hip.HipError), match=text):
            call()


def test_workspaces_come_from_the_sizes():
    """Rows' sums, a mask's bits and splits' sums, and no more."""
    op = attention(batch=3, q_len=100, k_len=300)
    assert op.workspace("vjp") == (8 * 3 * 4 * 100 + 255) // 256 * 256
    few = attention(batch=1, q_len=1, k_len=4096, heads=32, kv_heads=8)
    splits = -(-4096 // 256)
    assert few.workspace("value") == splits * 32 * (4 * 64 + 8)
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    masked = attention(mask_cols=300, k_len=300, q_len=100)
    assert masked.workspace("vjp") == up(4 * 2 * 100 * 10) + up(4 * 2 * 300 * 4) + up(2 * 4 * 10) + up(8 * 2 * 4 * 100)


def test_buffers_between_each_other(calls):
    """Outputs whose elements lie between other tensors' are apart from them: single
    tokens of a packed projection, and heads before rows in one buffer."""
    op = attention(q_len=1, k_len=1)
    one = lambda: dev(2, 1, 8, 64).split((4, 2, 2), 2)  # noqa: E731
    (q, k, v), (dq, dk, dv) = one(), one()
    lse = dev(2, 4, 1, dtype=torch.float32)
    b = {"q": q, "k": k, "v": v, "o": dev(2, 1, 4, 64), "lse": lse, "do": dev(2, 1, 4, 64), "dq": dq, "dk": dk, "dv": dv}
    op.vjp(**b)
    rotary(seq=1).value(q, dev(32, dtype=torch.float64), q, k=k, yk=k)
    for same in ({"dk": dv}, {"dk": dq[:, :, 3:].expand(2, 1, 2, 64)}, {"dv": q[:, :, 2:]}):
        with pytest.raises(hip.HipError, match="meet"):
            op.vjp(**{**b, **same})
    (q, k, v), (dq, dk, dv) = (dev(2, 3, 4, 8, 64).unbind(1) for _ in range(2))
    op = attention(kv_heads=4, layout="bhsd")
    b = {"q": q, "k": k, "v": v, "o": dev(2, 4, 8, 64), "lse": dev(2, 4, 8, dtype=torch.float32), "do": dev(2, 4, 8, 64), "dq": dq, "dk": dk, "dv": dv}
    op.vjp(**b)
    # a cache's next row, beside those that the call reads
    cache = dev(2, 4, 9, 64)
    attention(kv_heads=4, layout="bhsd").value(**{**{n: b[n] for n in ("q", "v", "o", "lse")}, "k": cache[:, :, :8]})
    rotary(seq=1, heads=4, kv_heads=0, layout="bhsd").value(cache[:, :, 8:], dev(32, dtype=torch.float64), cache[:, :, 8:])
    assert len(calls) == 5
    for same in ({"dk": dq}, {"dk": dev(2, 4, 8, 64), "dv": q}):
        with pytest.raises(hip.HipError, match="meets"):
            op.vjp(**{**b, **same})
    flat = dev(2 * 4 * 8 * 64 + 32)
    cut = lambda at: flat[at:at + 2 * 4 * 8 * 64].view(2, 4, 8, 64)  # noqa: E731
    with pytest.raises(hip.HipError, match="dv meets dk|dk meets dv"):
        op.vjp(**{**b, "dk": cut(0), "dv": cut(32)})
