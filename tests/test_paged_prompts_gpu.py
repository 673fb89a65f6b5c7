"""Prompts large enough for two row tiles in a CTA (marked gpu): both head sizes
and types, last tiles of one row to a full one, windows, hidden pages and cache
rows that hold anything. Oracle and bounds: paged_oracle.py.
"""
import math

import pytest

torch = pytest.importorskip("torch")
from test_paged_gpu import BF16, F16, check, make, ops  # noqa: E402, F401

pytestmark = pytest.mark.gpu

SHAPES = [(128, BF16, 64), (128, F16, 16), (64, BF16, 16), (64, F16, 32)]
# rows of a request's last pair of tiles: 1, 127, 128, 129, 255, 256 for one head of the group
LENGTHS = [1, 127, 128, 129, 255, 256, 257, 383, 384, 385]


def fills_the_gpu(requests, hq, hkv):
    """(row tiles in pairs) * KV heads: the prompt kernel takes pairs from one for each SM on."""
    return (sum(n for n, _ in requests) * (hq // hkv) // 256 + len(requests)) * hkv >= torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("d,dtype,page", SHAPES)
@pytest.mark.parametrize("context", [0, 77, 500])
@pytest.mark.parametrize("group", [1, 3])
def test_last_tiles(ops, d, dtype, page, context, group):  # noqa: F811
    requests = [(n, n + context * (i % 3)) for i, n in enumerate(LENGTHS + LENGTHS[::-1])]
    assert fills_the_gpu(requests, 8 * group, 8)
    check(ops, make(requests, 8 * group, 8, d, page, dtype, seed=context + group))


@pytest.mark.parametrize("d,dtype,page", SHAPES)
def test_one_long_prompt(ops, d, dtype, page):  # noqa: F811
    for requests in ([(2500, 2500)], [(2401, 3000)]):
        assert fills_the_gpu(requests, 16, 8)
        check(ops, make(requests, 16, 8, d, page, dtype, seed=page))


@pytest.mark.parametrize("d,dtype,page", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 0), (130, 5), (300, 200), (2000, 4)])
def test_windows(ops, d, dtype, page, window, sinks):  # noqa: F811
    requests = [(700, 1900), (300, 300), (129, 1500), (513, 600), (40, 2500)] * 3 + [(256, 1024)] * 4
    assert fills_the_gpu(requests, 16, 8)
    for released, junk in ((False, None), (True, math.nan)):
        made = make(requests, 16, 8, d, page, dtype, seed=window, window=window, sinks=sinks, released=released, junk=junk)
        check(ops, made, window=window, sinks=sinks)


@pytest.mark.parametrize("d,dtype,page", SHAPES)
@pytest.mark.parametrize("holes", [(0,), (1, 4, 5), tuple(range(40))])
def test_hidden_pages(ops, d, dtype, page, holes):  # noqa: F811
    requests = [(n, n + 90) for n in LENGTHS + LENGTHS[::-1]]
    check(ops, make(requests, 16, 8, d, page, dtype, holes=holes, junk=math.nan))


@pytest.mark.parametrize("d,dtype,page", SHAPES)
def test_tokens_before_the_first_position(ops, d, dtype, page):  # noqa: F811
    requests = [(n, max(0, n - 130)) for n in LENGTHS + LENGTHS[::-1]]
    assert fills_the_gpu(requests, 8, 8)
    check(ops, make(requests, 8, 8, d, page, dtype))


@pytest.mark.parametrize("d,dtype,page", SHAPES)
@pytest.mark.parametrize("gain,scale", [(30.0, None), (0.0, None), (100.0, 3.0)])
def test_peaked_and_flat(ops, d, dtype, page, gain, scale):  # noqa: F811
    requests = [(n, n + 200) for n in LENGTHS + LENGTHS[::-1]]
    check(ops, make(requests, 8, 8, d, page, dtype, gain=gain), scale=scale)


@pytest.mark.parametrize("d,dtype,page", SHAPES)
def test_a_step_of_prompts_and_single_tokens(ops, d, dtype, page):  # noqa: F811
    """Requests of every kind in one call: both kernels, pairs of tiles among them."""
    requests = [(1, 1 + 97 * i % 3000) for i in range(40)] + [(700, 1700), (300, 300)] + [(2, 900 + i) for i in range(7)] + [(1200, 1200)]
    assert fills_the_gpu(requests, 16, 8)
    check(ops, make(requests, 16, 8, d, page, dtype))
