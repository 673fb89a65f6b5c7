"""Python binding of the paged-cache operators (include/bnn_b200_paged.h).

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
operators have no backward pass (the library serves trained weights).
"""
import ctypes
import math
import struct

import torch

from .accel import EINVAL, OK, BnnError

F32, BF16, F16 = 1, 2, 3
_TYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}

# BNN_PagedCache, BNN_PagedAppend and BNN_PagedAttention: 64-bit integers and
# pointers, the floating member last.
_CACHE = "2Q11q"
_APPEND = struct.Struct("=" + _CACHE + "10Q" + "14q" + "d")
_ATTENTION = struct.Struct("=" + _CACHE + "7Q" + "15q" + "d")


def _sizes():
    """Bytes of the packed argument blocks (the ABI test compares them with the header's)."""
    return {"BNN_PagedAppend": _APPEND.size, "BNN_PagedAttention": _ATTENTION.size}


def _bad(what):
    raise BnnError(EINVAL, what)


class Paged:
    """The paged-cache operators of one device handle, with their workspace.

    Calls on one stream run in order and share the workspace; a call on
    another stream first waits for the work the previous one had enqueued.
    A CUDA graph that captured a call uses the workspace too: replay it in
    order with the other calls."""

    def __init__(self, device, max_batch=256, max_kv_heads=32):
        dll = device.api.dll
        self.device = device
        self._append = dll.bnn_b200_paged_append
        self._attention = dll.bnn_b200_paged_attention
        for fn in (self._append, self._attention):
            fn.restype = ctypes.c_int
            fn.argtypes = [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
        self._sync = dll.bnn_b200_paged_sync
        self._sync.restype = ctypes.c_int
        self._sync.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
        size = dll.bnn_b200_paged_workspace
        size.restype = ctypes.c_int
        size.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
        ordinal = dll.bnn_b200_device_ordinal
        ordinal.restype = ctypes.c_int
        ordinal.argtypes = [ctypes.c_void_p]
        self.cuda = torch.device("cuda", ordinal(device.handle))
        need = ctypes.c_size_t()
        st = size(device.handle, max_batch, max_kv_heads, ctypes.byref(need))
        if st != OK:
            raise BnnError(st, "bnn_b200_paged_workspace")
        self._workspace = torch.zeros(need.value, dtype=torch.uint8, device=self.cuda)
        self._stream = torch.cuda.current_stream(self.cuda)
        self._raw_stream = self._stream.cuda_stream

    def _enter(self):
        """The raw current stream; the workspace's earlier work is ordered before it."""
        raw = torch.cuda.current_stream(self.cuda).cuda_stream
        if raw != self._raw_stream and not torch.cuda.is_current_stream_capturing():
            now = torch.cuda.current_stream(self.cuda)
            now.wait_stream(self._stream)
            self._stream, self._raw_stream = now, raw
        return raw

    def _cache(self, k_pages, v_pages):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            _bad("k_pages and v_pages: one shape [pages, kv_heads, page_size, head_dim] and type")
        kind = _TYPES.get(k_pages.dtype, 0)
        if kind < BF16:
            _bad("k_pages: bfloat16 or float16")
        pages, heads, page, dim = k_pages.shape
        strides = []
        for x in (k_pages, v_pages):
            if x.device != self.cuda:
                _bad(f"the cache is on {x.device}, the handle on {self.cuda}")
            s = x.stride()
            if s[3] != 1:
                _bad("the cache's last dimension has to be adjacent")
            # the stride of a dimension of one is free: nothing steps over it
            strides += [s[0] if pages > 1 else dim, s[1] if heads > 1 else dim, s[2] if page > 1 else dim]
        return (k_pages.data_ptr(), v_pages.data_ptr(), *strides, pages, heads, page, dim, kind)

    def _rows(self, x, name, tokens, heads, dim):
        if x.dim() != 3 or x.shape[0] != tokens or x.shape[1] != heads or x.shape[2] != dim or x.device != self.cuda:
            _bad(f"{name}: [{tokens}, {heads}, {dim}] on {self.cuda} is wanted, got {list(x.shape)} on {x.device}")
        s = x.stride()
        if s[2] != 1:
            _bad(f"{name}: the last dimension has to be adjacent")
        return s[0], s[1]

    def _vector(self, x, name, dtype, count):
        if x.dtype != dtype or x.dim() != 1 or x.shape[0] != count or x.device != self.cuda or (count > 1 and x.stride(0) != 1):
            _bad(f"{name}: {count} adjacent {dtype} on {self.cuda} are wanted")
        return x.data_ptr()

    def append(self, q, k, v, cos, sin, positions, slots, k_pages, v_pages, *, q_norm=None, k_norm=None, eps=1e-6, interleaved=False,
               out=None):
        """Normalises and rotates q and k, writes k and v to their slots; returns q
        (bnn_b200_paged_append). cos and sin None: no rotation."""
        cache = self._cache(k_pages, v_pages)
        heads_kv, dim = cache[9], cache[11]
        if q.dim() != 3:
            _bad("q: [tokens, heads, head_dim]")
        tokens, heads = q.shape[0], q.shape[1]
        kind = _TYPES.get(q.dtype, 0)
        if not kind or k.dtype != q.dtype or v.dtype != q.dtype:
            _bad("q, k and v: one type, float32, bfloat16 or float16")
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            _bad("append has no backward pass")
        qs, ks, vs = (self._rows(q, "q", tokens, heads, dim), self._rows(k, "k", tokens, heads_kv, dim),
                      self._rows(v, "v", tokens, heads_kv, dim))
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=k_pages.dtype, device=self.cuda)
        elif out.dtype != k_pages.dtype:
            _bad("out: the cache's type")
        os = self._rows(out, "out", tokens, heads, dim)
        if cos is None:
            rotary, rows, cos_at, sin_at = 0, 0, 0, 0
        else:
            if cos.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape or sin.dtype != torch.float32 or \
                    not cos.is_contiguous() or not sin.is_contiguous() or cos.device != self.cuda or sin.device != self.cuda:
                _bad("cos and sin: contiguous float32 [positions, rotary_dim / 2]")
            rows, rotary = cos.shape[0], 2 * cos.shape[1]
            cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
        st = self._append(self.device.handle, _APPEND.pack(
            *cache, q.data_ptr(), k.data_ptr(), v.data_ptr(),
            0 if q_norm is None else self._vector(q_norm, "q_norm", torch.float32, dim),
            0 if k_norm is None else self._vector(k_norm, "k_norm", torch.float32, dim), cos_at, sin_at,
            self._vector(positions, "positions", torch.int32, tokens), self._vector(slots, "slots", torch.int32, tokens), out.data_ptr(),
            tokens, heads, kind, *qs, *ks, *vs, *os, rotary, rows, 1 if interleaved else 0, eps),
            torch.cuda.current_stream(self.cuda).cuda_stream)
        if st != OK:
            raise BnnError(st, "bnn_b200_paged_append")
        return out

    def attention(self, q, k_pages, v_pages, page_table, kv_lens, q_starts, *, max_q, scale=None, window=0, sinks=0, out=None,
                  out_dtype=None, return_lse=False):
        """Attention of each request's new tokens over its pages
        (bnn_b200_paged_attention); scale None: 1 / sqrt(head_dim). Returns
        [tokens, heads, head_dim] of q's type (or out_dtype float32), and with
        return_lse the float32 logarithms of the softmax sums [tokens, heads]."""
        cache = self._cache(k_pages, v_pages)
        dim = cache[11]
        if q.dim() != 3 or q.dtype != k_pages.dtype:
            _bad("q: [tokens, heads, head_dim] of the cache's type")
        if torch.is_grad_enabled() and q.requires_grad:
            _bad("attention has no backward pass")
        tokens, heads = q.shape[0], q.shape[1]
        qs = self._rows(q, "q", tokens, heads, dim)
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != self.cuda or \
                (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            _bad("page_table: int32 [batch, width], rows adjacent")
        batch, width = page_table.shape
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=out_dtype or q.dtype, device=self.cuda)
        elif out_dtype not in (None, out.dtype):
            _bad("out and out_dtype differ")
        os = self._rows(out, "out", tokens, heads, dim)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=self.cuda) if return_lse else None
        st = self._attention(self.device.handle, _ATTENTION.pack(
            *cache, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, page_table.data_ptr(),
            self._vector(kv_lens, "kv_lens", torch.int32, batch), self._vector(q_starts, "q_starts", torch.int32, batch + 1),
            self._workspace.data_ptr(), self._workspace.numel(), batch, tokens, heads, max_q, *qs, *os, heads,
            page_table.stride(0) if batch > 1 else width, width, window, sinks, _TYPES.get(out.dtype, 0),
            1.0 / math.sqrt(dim) if scale is None else scale), self._enter())
        if st != OK:
            raise BnnError(st, "bnn_b200_paged_attention")
        return (out, lse) if return_lse else out

    def sync(self):
        """Waits for the current stream; raises what the calls since the last sync recorded
        (bnn_b200_paged_sync)."""
        st = self._sync(self.device.handle, torch.cuda.current_stream(self.cuda).cuda_stream)
        if st != OK:
            raise BnnError(st, "bnn_b200_paged_sync")
