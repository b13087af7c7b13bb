"""The losses' entry points without a GPU: sizes, types, buffers and
workspaces are checked before anything is launched."""
import ctypes

import pytest

from presk_amd import hip


def rc_of(call):
    rc = call()
    return rc, hip.lib().presk_hip_last_error().decode()


def filled(head=True, **over):
    """Arguments that pass every check but the workspace's size (no pointer
    of them is read on the host)."""
    a = hip.LossArgs()
    a.dtype, a.rows, a.model, a.vocab, a.top, a.tied, a.temperature = b"bf16", 8, 64 if head else 0, 128, 0 if head else 4, 0, 1.0
    at = 1 << 30
    for n in ("x", "w", "index", "teacher", "loss", "lse", "mean", "ct", "dx", "dw", "flag", "work"):
        if not head and n in ("w", "dw"):
            continue
        setattr(a, n, at)
        at += 1 << 24
    a.work_bytes = 1 << 23
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over,text", [
    ({"dtype": b"f64"}, "E7005"), ({"dtype": b"e8m15"}, "E7005"), ({"dtype": None}, "E7005"),
    ({"rows": -1}, "rows -1"), ({"rows": 1 << 22}, "rows 4194304"),
    ({"model": 1 << 22}, "model 4194304"), ({"vocab": 0}, "vocab 0"), ({"vocab": 1 << 22}, "vocab 4194304"),
    ({"top": -1}, "top -1"), ({"top": 1025}, "top 1025"),
    ({"temperature": 0.0, "top": 2}, "temperature"), ({"temperature": float("nan"), "top": 2}, "temperature"),
    ({"temperature": 2.0}, "a temperature without a teacher"),
    ({"dtype": b"f32", "rows": 1 << 20, "model": 4096}, "not below 2^31"),
    ({"x": None}, "x is null"), ({"w": None}, "w is null"), ({"index": None}, "index is null"),
    ({"top": 3, "teacher": None}, "teacher is null"), ({"work": None}, "work is null"),
    ({"index": (1 << 30) + 4}, "index is not aligned to 8"), ({"x": (1 << 30) + 2}, "x is not aligned to 16"),
    ({"work": (1 << 29) + 8}, "work is not aligned to 16"), ({"work_bytes": 255}, "255 bytes"),
    ({"dx": 1 << 30}, "meets"), ({"loss": 1 << 30}, "meets"), ({"dw": (1 << 30) + (1 << 24)}, "meets"),
    ({"dx": None, "dw": None}, "a gradient without an output"),
])
def test_head_loss_refusals(over, text):
    a = filled(**over)
    rc, msg = rc_of(lambda: hip.lib().presk_hip_head_loss(ctypes.byref(a), hip.VALUE | hip.GRAD, None))
    assert rc in (hip.ERR, hip.REFUSED) and text in msg, msg
    assert (rc == hip.REFUSED) == msg.startswith("E7005")


def test_what_is_needed_of_a_gradient_alone():
    for over, text in (({"lse": None}, "lse is null"), ({"ct": None, "mean": None}, "mean is null")):
        a = filled(**over)
        rc, msg = rc_of(lambda: hip.lib().presk_hip_head_loss(ctypes.byref(a), hip.GRAD, None))
        assert rc == hip.ERR and text in msg
    a = filled(loss=None, lse=None, mean=None)
    rc, msg = rc_of(lambda: hip.lib().presk_hip_head_loss(ctypes.byref(a), hip.VALUE, None))
    assert rc == hip.ERR and "a value without an output" in msg
    for what in (0, 4):
        rc, msg = rc_of(lambda: hip.lib().presk_hip_head_loss(ctypes.byref(filled()), what, None))
        assert rc == hip.ERR and "what" in msg
    assert hip.lib().presk_hip_head_loss(None, hip.VALUE, None) == hip.ERR


@pytest.mark.parametrize("over,text", [
    ({"model": 64}, "model 64"), ({"top": 0}, "top 0"), ({"vocab": 1 << 30}, "vocab 1073741824"), ({"w": 1 << 28}, "w or dw"),
    ({"dx": None}, "dx is null"), ({"dx": 1 << 30}, "meets"),
])
def test_distill_refusals(over, text):
    a = filled(head=False, **over)
    rc, msg = rc_of(lambda: hip.lib().presk_hip_distill(ctypes.byref(a), hip.VALUE | hip.GRAD, None))
    assert rc == hip.ERR and text in msg, msg


def test_steps_of_a_sequence_are_checked_when_they_are_added():
    b = ctypes.c_void_p()
    assert hip.lib().presk_hip_batch_create(ctypes.byref(b)) == hip.OK
    try:
        assert hip.lib().presk_hip_batch_add_head_loss(b, ctypes.byref(filled(x=None)), 3) == hip.ERR
        assert hip.lib().presk_hip_batch_add_distill(b, ctypes.byref(filled(False, dx=None)), 3) == hip.ERR
        assert hip.lib().presk_hip_batch_add_head_loss(None, ctypes.byref(filled()), 3) == hip.ERR
        assert hip.lib().presk_hip_batch_add_head_loss(b, ctypes.byref(filled()), 3) == hip.OK
        assert hip.lib().presk_hip_batch_add_distill(b, ctypes.byref(filled(False)), 3) == hip.OK
    finally:
        hip.lib().presk_hip_batch_release(b)


def test_the_workspace_does_not_grow_with_the_vocabulary():
    """Past 4 GiB of f32 logits a head's workspace is its pieces': between a
    vocabulary of 128 Ki and one of 4 Mi it grows by the row sums' partials
    alone (12 bytes a row and column tile of at least 128).  Up to there it is
    the logits' and their 16-bit cotangent's."""
    for dt in ("bf16", "f16", "f32"):
        rows, model = 8192, 256
        sizes = [hip.HeadLoss(dt, rows, model, v).workspace("step") for v in ((1 << 17) + 64, (1 << 22) - 64)]
        tiles = (1 << 22) // 128
        assert sizes[1] - sizes[0] <= 12 * rows * tiles + (1 << 20), (dt, sizes)
        assert sizes[1] < rows * (1 << 22)     # a byte a logit
        assert hip.HeadLoss(dt, rows, model, 1 << 17).workspace("step") < 6.5 * (1 << 30)
    # a gradient that is not asked for takes none
    op = hip.HeadLoss("bf16", 65536, 4096, 50000)
    assert op.workspace("step", dx=False) < op.workspace("step")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_no_rows_and_the_smallest_sizes_have_a_workspace(dt):
    for rows in (0, 1):
        for kind in ("value", "vjp", "step"):
            assert hip.HeadLoss(dt, rows, 1, 1).workspace(kind) >= 256
            assert hip.HeadLoss(dt, rows, 7, 9, tied=True, top=3).workspace(kind) >= 256
            assert hip.Distill(dt, rows, 1, 1).workspace(kind) >= 256


def test_the_binding_checks_sizes():
    class Buf:
        def __init__(self, n, at):
            self.nbytes, self.ptr = n, at

    op = hip.HeadLoss("bf16", 4, 64, 100)
    big = [Buf(1 << 20, (i + 1) << 24) for i in range(6)]
    with pytest.raises(ValueError, match="x has 510 bytes, 512 needed"):
        op.value(Buf(510, 1 << 22), big[0], big[1], loss=big[2], work=big[3])
    with pytest.raises(ValueError, match="work has 16 bytes"):
        op.value(big[0], big[1], big[2], loss=big[3], work=Buf(16, 1 << 22))
    with pytest.raises(ValueError, match="model 0"):
        hip.HeadLoss("bf16", 4, 0, 100)
    with pytest.raises(hip.HipError, match="E7005"):
        hip.HeadLoss("f64", 4, 64, 100)
    with pytest.raises(hip.HipError, match="top 0"):
        hip.Distill("f32", 4, 100, 0)


def test_the_binding_checks_tensors_types_and_places():
    torch = pytest.importorskip("torch")

    class Tensor:
        """A tensor in device memory as far as the checks look."""

        def __init__(self, dtype, n, cuda=True, contiguous=True, device=0, shape=(1,)):
            self.shape, self.ndim = shape, len(shape)
            self.dtype, self.nbytes, self.whole, self.device = dtype, n, contiguous, device if cuda else -1

        def get_device(self):
            return self.device

        def data_ptr(self):
            return 1 << 24

        def is_contiguous(self):
            return self.whole

    op = hip.HeadLoss("bf16", 4, 64, 100)
    x, w, i, f = (Tensor(t, 1 << 20) for t in (torch.bfloat16, torch.bfloat16, torch.int64, torch.float32))
    assert op.args("value", x=x, w=w, index=i, loss=f, work=Tensor(torch.uint8, 1 << 20)).rows == 4
    for bad, why in [({"x": Tensor(torch.float16, 1 << 20)}, "x is f16, not bf16"), ({"w": f}, "w is f32, not bf16"),
                     ({"index": Tensor(torch.int32, 1 << 20)}, "index is torch.int32, not i64"), ({"loss": x}, "loss is bf16, not f32"),
                     ({"w": Tensor(torch.bfloat16, 1 << 20, shape=(100, 64))}, "w has rows of 64, not 100"),
                     ({"x": Tensor(torch.bfloat16, 1 << 20, cuda=False)}, "x is not in device memory"),
                     ({"x": Tensor(torch.bfloat16, 1 << 20, contiguous=False)}, "x is not contiguous")]:
        with pytest.raises(ValueError, match=why):
            op.args("value", **{**dict(x=x, w=w, index=i, loss=f, work=Tensor(torch.uint8, 1 << 20)), **bad})
    was, hip._initialized = hip._initialized, 0
    try:
        with pytest.raises(ValueError, match="x is on device 1, not 0"):
            op.args("value", x=Tensor(torch.bfloat16, 1 << 20, device=1), w=w, index=i, loss=f, work=x)
    finally:
        hip._initialized = was
