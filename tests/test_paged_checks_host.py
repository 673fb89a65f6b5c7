"""Host checks of the paged operators' C entry points (no GPU: calls without
tokens, so that a description that passes its checks returns at once)."""
import ctypes
from ctypes import c_double, c_int64, c_void_p

import pytest

from bnn_b200 import _lib, accel


class Cache(ctypes.Structure):
    _fields_ = [("k", c_void_p), ("v", c_void_p)] + [(n, c_int64) for n in (
        "k_page_stride", "k_head_stride", "k_row_stride", "v_page_stride", "v_head_stride", "v_row_stride", "pages", "kv_heads", "page_size",
        "head_dim", "type")]


class Append(ctypes.Structure):
    _fields_ = [("cache", Cache)] + [(n, c_void_p) for n in ("q", "k", "v", "q_norm", "k_norm", "cos", "sin", "positions", "slots", "q_out")] + \
        [(n, c_int64) for n in ("tokens", "heads", "type", "q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride",
                                "v_token_stride", "v_head_stride", "out_token_stride", "out_head_stride", "rotary_dim", "table_rows",
                                "interleaved")] + [("eps", c_double)]


class Attention(ctypes.Structure):
    _fields_ = [("cache", Cache)] + [(n, c_void_p) for n in ("q", "out", "lse", "page_table", "kv_lens", "q_starts", "workspace")] + \
        [(n, c_int64) for n in ("workspace_bytes", "batch", "tokens", "heads", "max_q", "q_token_stride", "q_head_stride", "out_token_stride",
                                "out_head_stride", "lse_token_stride", "table_stride", "table_width", "window", "sinks", "out_type")] + \
        [("scale", c_double)]


BF16 = 2
CACHE = Cache(1 << 20, 1 << 21, 4096, 2048, 128, 4096, 2048, 128, 4, 2, 16, 128, BF16)


def status(name, desc, **fields):
    """The entry point's answer; the handle is a block of zeros that a call without tokens does not look into."""
    for k, v in fields.items():
        setattr(desc, k, v)
    fn = getattr(_lib.load(), "bnn_b200_paged_" + name)
    fn.restype, fn.argtypes = ctypes.c_int, [c_void_p, c_void_p, c_void_p]
    handle = ctypes.create_string_buffer(1 << 14)
    return fn(ctypes.addressof(handle), ctypes.addressof(desc), None)


def attention(**fields):
    return status("attention", Attention(cache=CACHE, batch=1, heads=4, max_q=1, table_width=3, table_stride=3, out_type=BF16, scale=0.1),
                  **fields)


def append(**fields):
    return status("append", Append(cache=CACHE, heads=4, type=BF16, eps=1e-6), **fields)


@pytest.mark.parametrize("scale,want", [(0.1, accel.OK), (1e-30, accel.OK), (2e38, accel.OK), (2.9e38, accel.EINVAL), (1e39, accel.EINVAL),
                                        (1e-60, accel.EINVAL), (0.0, accel.EINVAL), (float("nan"), accel.EINVAL)])
def test_scale_is_checked_as_the_kernels_use_it(scale, want):
    """They multiply by scale * log2(e) in FP32: infinite from 2.36e38 on, and zero times it NaN."""
    assert attention(scale=scale) == want


@pytest.mark.parametrize("eps,want", [(0.0, accel.OK), (1e-60, accel.OK), (3e38, accel.OK), (1e39, accel.EINVAL), (-1e-9, accel.EINVAL)])
def test_eps_is_checked_as_the_kernels_use_it(eps, want):
    assert append(eps=eps) == want


@pytest.mark.parametrize("stride,want", [(3, accel.OK), (100, accel.OK), (2, accel.OK), (0, accel.OK), (-1, accel.EINVAL)])
def test_requests_may_share_a_row_of_the_table(stride, want):
    assert attention(batch=2, table_stride=stride) == want
