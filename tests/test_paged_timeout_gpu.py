"""Waits of the prompt tiles that run out after some tiles have gone through
(marked gpu): nothing faults, the next sync says so, and the call is right once
the limit is restored. With the limit at 1 ms a call ends within some of them."""
import ctypes
import time

import pytest

torch = pytest.importorskip("torch")
from test_paged_gpu import BF16, F16, check, make, ops  # noqa: E402, F401

pytestmark = pytest.mark.gpu

FORMS = {  # one stream; two streams over one tile of rows; two tiles of rows
    "single": ([(100, 500), (130, 130)], 4, 2, 128, 16, BF16),
    "single_64": ([(100, 500), (130, 130)], 4, 2, 64, 16, F16),
    "turns": ([(600, 1400)], 4, 2, 128, 16, BF16),
    "turns_64": ([(600, 1400)], 4, 2, 64, 32, F16),
    "pair": ([(2500, 2600)], 16, 8, 128, 64, BF16),
    "pair_64": ([(1300, 1300), (1400, 1500)], 16, 8, 64, 16, F16),
}


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("tiles", [0, 1, 2, 3])
def test_tiles_withheld(ops, name, tiles):  # noqa: F811
    from bnn_b200 import accel
    hook = ops.device.api.dll.bnn_b200_test_wait_limit
    hook.restype, hook.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int]
    requests, hq, hkv, d, page, dtype = FORMS[name]
    made = make(requests, hq, hkv, d, page, dtype)
    torch.cuda.synchronize()
    assert hook(ops.device.handle, 1_000_000, 1 + tiles) == accel.OK
    began = time.perf_counter()
    try:
        ops.attention(*made, max_q=max(n for n, _ in requests))
        with pytest.raises(accel.BnnError) as e:
            ops.sync()
    finally:
        torch.cuda.synchronize()
        assert hook(ops.device.handle, 0, 0) == accel.OK
    assert e.value.status == accel.ETIMEOUT
    assert time.perf_counter() - began < 1.0
    check(ops, made)
