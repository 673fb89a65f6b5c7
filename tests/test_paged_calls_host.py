"""What bnn_b200.paged does around a call, with the binding replaced by one that
records (no GPU)."""
import types

import pytest

torch = pytest.importorskip("torch")
from bnn_b200 import accel, paged  # noqa: E402


class Recorder:
    """Stands for the binding: notes what is called."""

    def __init__(self):
        self.seen = []

    def attention(self, *args):
        self.seen.append("attention")
        return args[0]

    def append(self, *args):
        self.seen.append("append")
        return args[0]


@pytest.fixture
def recorded(monkeypatch):
    """(Paged over a recorder, the recorder): every attribute that its constructor would make on a GPU."""
    recorder = Recorder()
    real = paged._paged_torch
    monkeypatch.setattr(paged, "_paged_torch", types.SimpleNamespace(
        bind=real.bind, stream=lambda d: 0, new_order=lambda d, n: (None, None), attention=recorder.attention, append=recorder.append))
    dll = types.SimpleNamespace(bnn_b200_device_ordinal=lambda h: 0, bnn_b200_paged_workspace=lambda h, n: 0)
    monkeypatch.setattr(paged, "_bind", lambda: dll)
    device = types.SimpleNamespace(handle=types.SimpleNamespace(value=1))
    return paged.Paged(device), recorder


ARGS = (None, None, None, torch.zeros(1, 1, dtype=torch.int32), None, None)


def test_order_and_launch_are_one_call(recorded):
    """No other thread gets between the ordering of the workspace's uses and the launch: both are one call of the
    binding, which the interpreter does not interrupt."""
    ops, recorder = recorded
    ops.attention(*ARGS, max_q=1)
    ops.append(*[None] * 9)
    assert recorder.seen == ["attention", "append"]


def test_a_closed_device_is_refused(recorded):
    """The handle is gone: nothing that was kept of it reaches the library."""
    ops, recorder = recorded
    ops.device.handle = None
    for call in (lambda: ops.append(*[None] * 9), lambda: ops.attention(*ARGS, max_q=1), lambda: paged.Paged(ops.device)):
        with pytest.raises(accel.BnnError) as e:
            call()
        assert e.value.status == accel.EINVAL
    assert not recorder.seen
