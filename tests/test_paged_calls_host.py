"""What bnn_b200.paged does around a call, with the binding replaced by one that
records (no GPU)."""
import sys
import threading
import time
import types

import pytest

torch = pytest.importorskip("torch")
from bnn_b200 import accel, paged  # noqa: E402


class Recorder:
    """Stands for the binding: notes who called what, slowly."""

    def __init__(self):
        self.seen = []

    def order(self, *args):
        self.seen.append((threading.get_ident(), "order"))
        time.sleep(0.001)

    def attention(self, *args):
        self.seen.append((threading.get_ident(), "attention"))
        return args[0]

    def append(self, *args):
        self.seen.append((threading.get_ident(), "append"))
        return args[0]


@pytest.fixture
def recorded(monkeypatch):
    """(Paged over a recorder, the recorder): every attribute that its constructor would make on a GPU."""
    recorder = Recorder()
    real = paged._paged_torch
    monkeypatch.setattr(paged, "_paged_torch", types.SimpleNamespace(
        bind=real.bind, stream=lambda d: 0, new_order=lambda d, n: (None, None), order=recorder.order, attention=recorder.attention, append=recorder.append))
    dll = types.SimpleNamespace(bnn_b200_device_ordinal=lambda h: 0, bnn_b200_paged_workspace=lambda h, n: 0)
    monkeypatch.setattr(paged, "_bind", lambda: dll)
    device = types.SimpleNamespace(handle=types.SimpleNamespace(value=1))
    return paged.Paged(device), recorder


ARGS = (None, None, None, torch.zeros(1, 1, dtype=torch.int32), None, None)


def test_order_and_launch_are_one_step_between_threads(recorded):
    ops, recorder = recorded
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=lambda: [ops.attention(*ARGS, max_q=1) for _ in range(20)]) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert len(recorder.seen) == 160
    for first, second in zip(recorder.seen[::2], recorder.seen[1::2]):
        assert first[0] == second[0] and (first[1], second[1]) == ("order", "attention")


def test_a_closed_device_is_refused(recorded):
    """The handle is gone: nothing that was kept of it reaches the library."""
    ops, recorder = recorded
    ops.device.handle = None
    for call in (lambda: ops.append(*[None] * 9), lambda: ops.attention(*ARGS, max_q=1), lambda: paged.Paged(ops.device)):
        with pytest.raises(accel.BnnError) as e:
            call()
        assert e.value.status == accel.EINVAL
    assert not recorder.seen
