"""One-row jobs and paged calls on one handle's stream (marked gpu): the jobs do
not read a paged call's output early, and may read early again once it is done."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_paged_gpu import BF16, F32, make, ops, rows, pool  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def may_read_early(ops):  # noqa: F811
    fn = ops.device.api.dll.bnn_b200_test_early_input
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p]
    return fn(ops.device.handle)


@pytest.mark.parametrize("operator", ["append", "attention"])
def test_a_sync_ends_the_hold(ops, operator):  # noqa: F811
    fn = ops.device.api.dll.bnn_b200_device_stream
    fn.restype, fn.argtypes = ctypes.c_void_p, [ctypes.c_void_p]
    own = torch.cuda.ExternalStream(fn(ops.device.handle))
    made = make([(1, 40)], 4, 2, 128, 16, BF16)
    kp, vp = pool(2, 2, 16, 128, BF16)
    at = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call():
        if operator == "append":
            ops.append(*rows(1, 4, 2, 128, F32), None, None, at, at, kp, vp)
        else:
            ops.attention(*made, max_q=1)

    torch.cuda.synchronize()
    ops.sync()
    call()  # another stream: the handle's is free
    assert may_read_early(ops) == 1
    torch.cuda.synchronize()
    with torch.cuda.stream(own):
        call()
        assert may_read_early(ops) == 0
    ops.sync()  # waits for this stream, not for the handle's
    assert may_read_early(ops) == 0
    with torch.cuda.stream(own):
        ops.sync()
        assert may_read_early(ops) == 1
    call()  # the workspace follows the streams while both are there
    torch.cuda.synchronize()


def test_a_job_after_a_paged_call_reads_its_output(ops):  # noqa: F811
    """attention -> one-row linear on the handle's stream, many times with changing values: each result is the
    synchronous job's on the same input."""
    from bnn_b200 import accel, synth
    dev = ops.device
    dll = dev.api.dll
    dll.bnn_b200_device_stream.restype = dll.bnn_b200_buffer_device_ptr.restype = ctypes.c_void_p
    dll.bnn_b200_device_stream.argtypes = dll.bnn_b200_buffer_device_ptr.argtypes = [ctypes.c_void_p]
    dll.bnn_b200_execute_async.restype, dll.bnn_b200_execute_async.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(accel.Job)]
    heads, width = 4, 512
    bits, scales = synth.w1_matrix(synth.rng_for(7, salt=3), width, 256)
    matrix = accel.Matrix(dev, bits, scales)
    src, dst = accel.Buffer(dev, width * 4), accel.Buffer(dev, 256 * 4)

    class View:
        def __init__(self, buffer, n):
            self.__cuda_array_interface__ = {"data": (dll.bnn_b200_buffer_device_ptr(buffer.handle), False), "shape": (n,), "typestr": "<f4",
                                             "version": 3}
    x, y = (torch.as_tensor(View(b, n), device="cuda") for b, n in ((src, width), (dst, 256)))
    job = accel.Job(operation=accel.OP_GEMV_F32, matrix=matrix.handle, input=accel.BufferView(src.handle, accel.TYPE_F32, 0, 0),
                    output=accel.BufferView(dst.handle, accel.TYPE_F32, 0, 0), rows=1)
    calls = [make([(1, 3000)], heads, 2, 128, 64, BF16, seed=s) for s in range(4)]
    torch.cuda.synchronize()
    got, inputs = [], []
    with torch.cuda.stream(torch.cuda.ExternalStream(dll.bnn_b200_device_stream(dev.handle))):
        for i in range(40):
            ops.attention(*calls[i % 4], max_q=1, out=x.view(1, heads, 128))
            assert dll.bnn_b200_execute_async(dev.handle, ctypes.byref(job)) == accel.OK
            got.append(y.clone())
            inputs.append(x.clone())
            if i % 8 == 7:
                ops.sync()
    torch.cuda.synchronize()
    for g, v in zip(got, inputs):
        assert np.array_equal(g.cpu().numpy(), accel.run_op(dev, accel.OP_GEMV_F32, bits, scales, v.cpu().numpy()[None])[0])
    ops.attention(*calls[0], max_q=1)
    torch.cuda.synchronize()
    del x, y
    src.free()
    dst.free()
    matrix.destroy()
