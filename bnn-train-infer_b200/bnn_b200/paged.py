"""The paged-cache operators (include/bnn_b200_paged.h) on torch tensors.

For programs that hold their tensors in torch: `Paged` takes CUDA tensors,
runs on torch's current stream and returns without waiting. Shapes:

  k_pages, v_pages  [pages, kv_heads, page_size, head_dim], bfloat16 or float16
  q, k, v           [tokens, heads or kv_heads, head_dim], views of any strides
                    whose last dimension is adjacent (so the q|k|v rows of one
                    linear are passed as three views)
  page_table        [batch, width] int32; kv_lens [batch], q_starts [batch + 1]
                    int32; positions, slots [tokens] int32
  cos, sin          [positions, rotary_dim / 2] float32

Like the other wrappers it raises accel.BnnError carrying the status. The
operators have no derivatives (the library serves trained weights): a tensor
that requires a gradient, trained gains among them, is refused outside
torch.no_grad(). The tensors are read and checked in binding/paged_torch.cpp, built beside this
file by the package Makefile; without it the import raises.
"""
import ctypes

import torch

from . import _lib, accel
from .accel import EINVAL, ENOTSUP, OK, BnnError

try:
    from . import _paged_torch
except ImportError as e:
    raise RuntimeError("bnn_b200/_paged_torch.so is missing or does not load; build it with "
                       "`make -C bnn-train-infer_b200` (there is no other path)") from e


def _bind():
    dll = _lib.load()
    _paged_torch.bind(*(ctypes.cast(getattr(dll, "bnn_b200_paged_" + n), ctypes.c_void_p).value for n in ("append", "attention")), BnnError)
    dll.bnn_b200_paged_sync.restype = ctypes.c_int
    dll.bnn_b200_paged_sync.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    dll.bnn_b200_paged_workspace.restype = ctypes.c_int
    dll.bnn_b200_paged_workspace.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]
    dll.bnn_b200_device_ordinal.restype = ctypes.c_int
    dll.bnn_b200_device_ordinal.argtypes = [ctypes.c_void_p]
    return dll


class Paged:
    """The paged-cache operators of one device handle (accel.Device), with their workspace.

    Calls on one stream run in order and share the workspace; an attention call
    on another stream first waits for the work that the stream of the previous
    one holds, so that stream has to exist still (BNN_EBUSY where it is being
    captured by then). Captured calls on branches of one CUDA graph are ordered
    likewise, and threads may share the object. The graph uses the workspace when it is replayed: replay it in
    order with the other calls, and keep this object as long as the graph.
    max_batch: most requests of a call, a bound of
    the program's own (calls beyond it are refused; the library's is 4096)."""

    def __init__(self, device: accel.Device, max_batch=4096):
        self._dll = _bind()
        self.device = device
        self._check_open()
        self._handle = device.handle.value
        self._index = self._dll.bnn_b200_device_ordinal(device.handle)
        self._max_batch = max_batch
        need = ctypes.c_size_t()
        st = self._dll.bnn_b200_paged_workspace(device.handle, ctypes.byref(need))
        if st != OK:
            raise BnnError(st, "bnn_b200_paged_workspace")
        self._workspace, self._order = _paged_torch.new_order(self._index, need.value)

    def _check_open(self):
        if not self.device.handle:
            raise BnnError(EINVAL, "the device is closed")

    def append(self, q, k, v, cos, sin, positions, slots, k_pages, v_pages, *, q_norm=None, k_norm=None, eps=1e-6, interleaved=False,
               out=None):
        """Normalises and rotates q and k, writes k and v to their slots; returns q
        (bnn_b200_paged_append). cos and sin None: no rotation."""
        self._check_open()
        return _paged_torch.append(self._handle, self._index, q, k, v, cos, sin, positions, slots, k_pages, v_pages, q_norm, k_norm, eps,
                                   interleaved, out)

    def attention(self, q, k_pages, v_pages, page_table, kv_lens, q_starts, *, max_q, scale=None, window=0, sinks=0, out=None,
                  out_dtype=None, return_lse=False):
        """Attention of each request's new tokens over its pages
        (bnn_b200_paged_attention); scale None: 1 / sqrt(head_dim). Returns
        [tokens, heads, head_dim] of q's type (or out_dtype float32), and with
        return_lse the float32 logarithms of the softmax sums [tokens, heads]."""
        self._check_open()
        f32 = False
        if out_dtype is not None:
            f32 = out_dtype == torch.float32
            if not f32 and out_dtype != getattr(q, "dtype", None) or out is not None and getattr(out, "dtype", None) != out_dtype:
                raise BnnError(EINVAL, "out_dtype: q's type or float32, and out's")
        if getattr(page_table, "ndim", 0) and page_table.shape[0] > self._max_batch:
            raise BnnError(ENOTSUP, f"more than {self._max_batch} requests")
        return _paged_torch.attention(self._handle, self._index, self._workspace, q, k_pages, v_pages, page_table, kv_lens, q_starts, max_q,
                                      scale, window, sinks, out, f32, return_lse, self._order)

    def sync(self):
        """Waits for the current stream; raises what the calls since the last sync recorded
        (bnn_b200_paged_sync)."""
        st = self._dll.bnn_b200_paged_sync(self.device.handle, _paged_torch.stream(self._index))
        if st != OK:
            raise BnnError(st, "bnn_b200_paged_sync")
