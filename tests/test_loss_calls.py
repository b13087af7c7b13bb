"""Which stream and which workspace a call of hip.HeadLoss or hip.Distill
takes, without a GPU: the library's call is recorded in its place."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from presk_amd import hip  # noqa: E402

CURRENT = 0x5000


class Tensor(torch.Tensor):
    """A tensor that says it is in device memory."""

    at = 0

    @staticmethod
    def of(t):
        return t.as_subclass(Tensor)

    is_cuda = True

    def get_device(self):
        return Tensor.at


class Library:
    """The executor's library with the losses' launches taken out."""

    def __init__(self, real, calls):
        self.real, self.calls = real, calls

    def __getattr__(self, name):
        return getattr(self.real, name)

    def presk_hip_distill(self, a, what, stream):
        self.calls.append((a._obj.work, stream))
        return hip.OK


class Memory:
    taken = 0

    def __init__(self, nbytes):
        Memory.taken += 1
        self.nbytes, self.ptr = nbytes, Memory.taken << 32


@pytest.fixture
def calls(monkeypatch):
    got, real = [], hip.lib()
    monkeypatch.setattr(hip, "lib", lambda: Library(real, got))
    monkeypatch.setattr(hip, "DeviceBuffer", Memory)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: type("S", (), {"cuda_stream": CURRENT + d})())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return got


def inputs(n=4, v=64, k=2):
    return {"x": Tensor.of(torch.zeros(n, v)), "index": Tensor.of(torch.zeros(n, k, dtype=torch.int64)),
            "teacher": Tensor.of(torch.zeros(n, k)), "loss": Tensor.of(torch.zeros(n))}


def test_a_call_with_tensors_goes_to_the_current_stream(calls):
    op = hip.Distill("f32", 4, 64, 2)
    op.value(**inputs())
    op.value(**inputs(), stream=0)
    op.value(**inputs(), stream=0x7000)
    assert [s for _, s in calls] == [CURRENT, 0, 0x7000]


def test_a_call_without_tensors_goes_to_the_null_stream(calls):
    op = hip.Distill("f32", 4, 64, 2)
    op.value(Memory(1024), Memory(64), Memory(32), loss=Memory(16))
    assert calls[0][1] is None


def test_the_own_workspace_is_a_streams(calls):
    """No two streams share one; a stream's calls do, until one needs more;
    what was outgrown stays (a captured call may use it)."""
    op = hip.Distill("f32", 4, 64, 2)
    for s in (0x10, 0x20, 0x10, None, 0, ctypes.c_void_p(0x20)):
        op.value(Memory(1024), Memory(64), Memory(32), loss=Memory(16), stream=s)
    w = [a for a, _ in calls]
    assert w[0] == w[2] != w[1] == w[5] and w[3] == w[4] not in (w[0], w[1])
    small, = (b for own in op._works.values() for b in own if b.ptr == w[0])
    small.nbytes = 16
    op.value(Memory(1024), Memory(64), Memory(32), loss=Memory(16), stream=0x10)
    assert calls[-1][0] not in w and small in op._outgrown and op._work not in op._outgrown


def test_tensors_of_another_device_than_the_current_one_are_refused(calls, monkeypatch):
    """Also where the executor was not initialised by device, or torch's
    current device was changed after that."""
    op = hip.Distill("f32", 4, 64, 2)
    for initialized in (None, -1, 0):
        monkeypatch.setattr(hip, "_initialized", initialized)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
        for stream in (None, 0, 0x7000):
            with pytest.raises(ValueError, match="is on device 0, not 1" if initialized != 0 else "current device is 1, not 0"):
                op.value(**inputs(), stream=stream)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        op.value(**inputs())
    assert len(calls) == 3


def test_the_own_workspace_is_a_devices(calls, monkeypatch):
    """The null streams of two devices are two."""
    op = hip.Distill("f32", 4, 64, 2)
    monkeypatch.setattr(hip, "_initialized", None)
    for at in (0, 1, 0):
        monkeypatch.setattr(Tensor, "at", at)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: at)
        op.value(**inputs(), stream=0)
    w = [a for a, _ in calls]
    assert w[0] == w[2] != w[1]
