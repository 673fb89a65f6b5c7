"""NaN and infinities that only later tokens of a request see (marked gpu).

Every form of the attention takes such values into a product with a weight of
zero and has to compute the rows that do not see them again. Here the rows are
whole, cut into a few parts, cut into more than one CTA joins at a time, in
groups of 16 behind a long cache, and tiles of the three forms of the prompt
kernel; the bounds are those of paged_oracle.py.
"""
import math

import pytest

torch = pytest.importorskip("torch")
import paged_oracle as oracle  # noqa: E402
from test_paged_gpu import BF16, F16, check, make, ops, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def poison(made, b, position, bad, which=2, dims=slice(None)):
    """`bad` in the value (which 2) or key (1) row of one position of request b, in every KV head."""
    table = made[3]
    pages = made[which]
    page = pages.shape[2]
    pages[int(table[b, position // page]), :, position % page, dims] = bad


def same_bits(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0, 1, -1), b.nan_to_num(0, 1, -1))


SPLIT = {  # (requests, query heads, KV heads, head_dim, page, type)
    "whole": ([(3, 70), (2, 300)] * 5, 4, 2, 128, 16, BF16),
    "eight_cut": ([(2, 4096)] * 8, 16, 8, 128, 64, BF16),
    "ragged_cut": ([(2 + b % 3, 1500 + 160 * b) for b in range(30)], 8, 2, 64, 32, F16),
    "many_cut": ([(2, 6400)] * 61, 8, 4, 64, 64, BF16),
    "two_levels": ([(4, 40000)], 2, 1, 128, 64, BF16),
    "two_levels_of_two": ([(2, 30001), (3, 29000)], 4, 2, 128, 16, F16),
    "groups_of_rows": ([(40, 9000)], 4, 2, 128, 64, BF16),
    "groups_of_rows_of_three": ([(33, 2500), (20, 4100), (17, 3000)], 2, 1, 64, 16, BF16),
}


@pytest.mark.parametrize("name", SPLIT)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_of_last_tokens_behind_cut_caches(ops, name, bad):  # noqa: F811
    """The value of every request's last token is not finite: all other tokens' results are, on every run."""
    requests, hq, hkv, d, page, dtype = SPLIT[name]
    made = make(requests, hq, hkv, d, page, dtype, seed=3)
    for b, (n, kv) in enumerate(requests):
        poison(made, b, kv - 1, bad)
    first, first_lse = check(ops, made)
    last = (made[5][1:] - 1).long()
    earlier = torch.ones(first.shape[0], dtype=torch.bool, device="cuda")
    earlier[last] = False
    assert torch.isfinite(first[earlier]).all() and not torch.isfinite(first[last]).any()
    assert torch.isfinite(first_lse).all()
    for _ in range(20):
        got, lse = ops.attention(*made, max_q=max(n for n, _ in requests), return_lse=True)
        assert same_bits(got, first) and torch.equal(lse, first_lse)


TILES = {  # one stream; two streams over one tile of rows; two tiles of rows
    "single": ([(100, 300), (130, 400)], 4, 2, 128, 16, BF16),
    "single_64": ([(100, 300), (130, 400)], 4, 2, 64, 16, F16),
    "turns": ([(600, 1400)], 4, 2, 128, 16, BF16),
    "turns_64": ([(600, 1400)], 4, 2, 64, 32, F16),
    "pair": ([(2500, 2600)], 16, 8, 128, 64, BF16),
    "pair_64": ([(1300, 1300), (1400, 1500)], 16, 8, 64, 16, F16),
}


@pytest.mark.parametrize("name", TILES)
@pytest.mark.parametrize("bad,which", [(math.nan, 2), (math.inf, 2), (math.nan, 1)])
def test_values_inside_prompts(ops, name, bad, which):  # noqa: F811
    """A position in the middle of a prompt: the tokens before it stay finite, the others follow the definition."""
    requests, hq, hkv, d, page, dtype = TILES[name]
    made = make(requests, hq, hkv, d, page, dtype, seed=4)
    b = len(requests) - 1
    n, kv = requests[b]
    at = kv - n // 2 - 3
    poison(made, b, at, bad, which, slice(0, None, 3))
    q, k, v, table, lens, starts = made
    got = ops.attention(*made, max_q=max(m for m, _ in requests))
    ops.sync()
    want, _, tol, _, _ = oracle.attention(*made)
    before = int(starts[b]) + at - (kv - n)  # tokens of the call that do not see the position
    assert torch.isfinite(got[:before]).all()
    finite = torch.isfinite(want)
    within(got[finite], want[finite], tol[finite])
    assert not torch.isfinite(got[~finite]).any()


@pytest.mark.parametrize("requests,dtype", [([(2048, 2048)], BF16), ([(2048, 2048)], F16), ([(2, 4096)] * 8, BF16), ([(40, 9000)], F16)])
@pytest.mark.parametrize("which,share", [(2, 0.0), (1, 0.0), (1, 0.5)])
def test_a_value_that_rows_see_costs_little(ops, requests, dtype, which, share):  # noqa: F811
    """A NaN that makes most rows NaN, and rightly: they are not computed again key by key (160 to 800 times
    the call's time). A check of the unseen values of each row is allowed: up to 64 keys' dependent loads a row of a
    warp, 32 rows, at most 1 us a batch of eight: 0.3 ms for calls of 35 us and more, so 40 times bounds it."""
    max_q = max(n for n, _ in requests)

    def spent(made):
        best = math.inf
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                ops.attention(*made, max_q=max_q)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    made = make(requests, 16, 8, 128, 64, dtype)
    plain = spent(made)
    for b, (n, kv) in enumerate(requests):
        poison(made, b, int(share * (kv - 1)), math.nan, which)
    assert spent(made) < 40 * plain
