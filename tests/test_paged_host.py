"""The paged-cache operators' boundary, checked without a GPU: the binding
loads, and calls without a device handle or with tensors of the host are
refused."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
from bnn_b200 import _lib, accel, paged  # noqa: E402


@pytest.mark.parametrize("name", ["bnn_b200_paged_append", "bnn_b200_paged_attention"])
def test_no_handle_is_refused(name):
    fn = getattr(_lib.load(), name)
    fn.restype = ctypes.c_int
    fn.argtypes = [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
    assert fn(None, bytes(512), None) == accel.EINVAL
    assert fn(None, None, None) == accel.EINVAL
    dll = paged._bind()
    assert dll.bnn_b200_paged_sync(None, None) == accel.EINVAL
    assert dll.bnn_b200_paged_workspace(None, ctypes.byref(ctypes.c_size_t())) == accel.EINVAL


def test_host_tensors_are_refused():
    paged._bind()
    ext = paged._paged_torch
    x = torch.zeros(2, 4, 128)
    pages = torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call, args in ((ext.append, (0, 0, x, x[:, :2], x[:, :2], None, None, i, i, pages, pages, None, None, 1e-6, False, None)),
                       (ext.attention, (0, 0, x, x.bfloat16(), pages, pages, i.view(2, 1), i, i, 1, None, 0, 0, None, False, False)),
                       (ext.append, (0, 0)), (ext.attention, (0,) * 16)):
        with pytest.raises(accel.BnnError) as e:
            call(*args)
        assert e.value.status == accel.EINVAL
