"""The paged-cache operators against their definitions in 64 bits (marked gpu).

Bounds are derived in paged_oracle.py. Lengths of zero and one, rows whose
mask leaves nothing, released pages, infinities and NaN in rows that no token
sees or that only later tokens see, every group size and page size, strided
and transposed tensors, offsets past 2^32 bytes, other streams, graphs,
refusals.
"""
import math
import random

import pytest

torch = pytest.importorskip("torch")
import paged_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from bnn_b200 import accel, paged
    dev = accel.Device(0)
    yield paged.Paged(dev)
    torch.cuda.synchronize()
    dev.close()


def within(got, want, tol):
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs() - tol)
    off = torch.where(torch.isnan(off), math.inf, off)
    assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.numel()} outside, worst by {float(off.max()):.3g} (bound there " \
                                f"{float(tol.flatten()[off.argmax()]):.3g})"


def make(requests, hq, hkv, d, page, dtype, *, seed=0, window=0, sinks=0, released=False, holes=(), junk=None, order="hnd", spare=3,
         gain=1.0):
    """Tensors of a call with requests [(n, kv)]; `junk` fills every cache row that no token sees."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max([1] + [-(-kv // page) for _, kv in requests])
    need = sum(-(-kv // page) for _, kv in requests)
    pages = need + spare
    perm = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.full((len(requests), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (n, kv) in enumerate(requests):
        c = -(-kv // page)
        table[b, :c] = perm[at:at + c]
        at += c
        if released and window:
            low = max(0, kv - n - window + 1)
            for p in range(-(-sinks // page), low // page):
                table[b, p] = -1
        for p in holes:
            if p < c:
                table[b, p] = (-1, pages, 1 << 30)[p % 3]
    shape = (pages, hkv, page, d) if order == "hnd" else (pages, page, hkv, d)
    k, v = (torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(2))
    if order != "hnd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    if junk is not None:
        unseen = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        for b, (n, kv) in enumerate(requests):
            for j in range(kv if n else 0):
                low = kv - n - window + 1 if window else 0
                p = int(table[b, j // page])
                if 0 <= p < pages and (j >= low or j < sinks):
                    unseen[p, j % page] = False
        for x in (k, v):
            x.masked_fill_(unseen[:, None, :, None], junk)
    starts = [0]
    for n, _ in requests:
        starts.append(starts[-1] + n)
    q = (gain * torch.randn(starts[-1], hq, d, device="cuda", generator=g)).to(dtype)
    lens = torch.tensor([kv for _, kv in requests], dtype=torch.int32, device="cuda")
    return q, k, v, table, lens, torch.tensor(starts, dtype=torch.int32, device="cuda")


def check(ops, made, *, window=0, sinks=0, scale=None, out_dtype=None, max_q=None, **kw):
    q, k, v, table, lens, starts = made
    n = starts[1:] - starts[:-1]
    max_q = int(n.max()) if max_q is None else max_q
    got, lse = ops.attention(q, k, v, table, lens, starts, max_q=max_q, window=window, sinks=sinks, scale=scale, out_dtype=out_dtype,
                             return_lse=True, **kw)
    ops.sync()
    want, want_lse, tol, lse_tol, covered = oracle.attention(q, k, v, table, lens, starts, scale=scale, window=window, sinks=sinks,
                                                             out_dtype=out_dtype)
    within(got[covered], want[covered], tol[covered])
    within(lse[covered], want_lse[covered], lse_tol[covered])
    return got, lse


# (requests, window, sinks): few new tokens, then prompts, then both
DECODE = {
    "one": ([(1, 1)], 0, 0),
    "two": ([(1, 2), (1, 1)], 0, 0),
    "ends_in_pages": ([(1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 127), (1, 129)], 0, 0),
    "empty_among": ([(1, 0), (1, 5), (0, 40), (1, 300), (0, 0)], 0, 0),
    "long_and_short": ([(1, 4097), (1, 3), (1, 1500)], 0, 0),
    "one_long": ([(1, 9001)], 0, 0),
    "window": ([(1, 700), (1, 3), (1, 100), (1, 101), (1, 99)], 100, 0),
    "window_one": ([(1, 70), (1, 1)], 1, 0),
    "sinks": ([(1, 700), (1, 3), (1, 105), (1, 2050)], 100, 4),
    "many_sinks": ([(1, 700), (1, 50)], 33, 90),
}
PREFILL = {
    "prompt_17": ([(17, 17)], 0, 0),
    "prompt_128": ([(128, 128)], 0, 0),
    "prompt_257": ([(257, 257)], 0, 0),
    "ragged": ([(40, 40), (1, 1), (130, 130), (64, 64), (0, 0), (33, 33)], 0, 0),
    "chunks": ([(100, 333), (17, 1000), (256, 257), (129, 700)], 0, 0),
    "no_keys": ([(40, 13), (30, 0), (50, 60)], 0, 0),  # tokens that stand before the first position
    "window": ([(300, 700), (45, 45), (130, 1000)], 50, 0),
    "window_one": ([(150, 200)], 1, 0),
    "sinks": ([(300, 900), (40, 2000), (129, 129)], 130, 5),
    "many_sinks": ([(200, 500)], 33, 190),
    "mixed": ([(1, 777), (200, 300), (1, 5), (2, 90), (1, 0)], 0, 0),
}
CASES = {**{"decode_" + k: v for k, v in DECODE.items()}, **{"prefill_" + k: v for k, v in PREFILL.items()}}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("d,hq,hkv,page,dtype", [(128, 4, 2, 16, BF16), (64, 8, 1, 32, F16), (128, 3, 1, 64, F16), (64, 4, 4, 128, BF16)])
def test_lengths_and_masks(ops, name, d, hq, hkv, page, dtype):
    requests, window, sinks = CASES[name]
    check(ops, make(requests, hq, hkv, d, page, dtype, seed=len(name)), window=window, sinks=sinks)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, F16)])
def test_group_sizes(ops, group, d, dtype):
    check(ops, make([(1, 333), (1, 70)], 2 * group, 2, d, 16, dtype, seed=group))
    check(ops, make([(67, 300), (130, 131)], 2 * group, 2, d, 16, dtype, seed=group))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("order", ["hnd", "nhd"])
def test_page_sizes_and_orders(ops, page, order):
    for requests in ([(1, 1000), (1, page), (1, page + 1)], [(150, 601), (20, page), (19, page + 1)]):
        check(ops, make(requests, 4, 2, 128, page, BF16, order=order), window=0)
        check(ops, make(requests, 4, 2, 64, page, BF16, order=order), window=90, sinks=3)


@pytest.mark.parametrize("requests", [[(2, 2), (2, 300)], [(5, 5), (3, 200), (1, 77)], [(8, 1000)], [(4, 3), (8, 2)], [(16, 40), (16, 16)]])
@pytest.mark.parametrize("group", [1, 2, 3])
def test_a_few_new_tokens(ops, requests, group):
    check(ops, make(requests, 2 * group, 2, 128, 16, BF16))
    check(ops, make(requests, 2 * group, 2, 64, 32, F16), window=40, sinks=2)


@pytest.mark.parametrize("requests,window,sinks", [
    ([(100, 3000)], 0, 0), ([(9, 1024)], 0, 0), ([(120, 1500)], 200, 5), ([(40, 2100)], 1500, 0),  # one request: its rows in groups of 16
    ([(20, 1024), (20, 1023), (1, 4000), (300, 1500), (17, 2500)], 0, 0),  # some of each kernel's
    ([(30, 1800), (200, 1900), (64, 64), (2, 1100)], 300, 20), ([(33, 1200), (0, 0), (5, 0)], 0, 0)])
@pytest.mark.parametrize("d,hq,hkv,page,dtype", [(128, 4, 2, 16, BF16), (64, 8, 1, 64, F16), (128, 5, 1, 32, F16)])
def test_groups_of_rows_behind_a_long_cache(ops, requests, window, sinks, d, hq, hkv, page, dtype):
    check(ops, make(requests, hq, hkv, d, page, dtype), window=window, sinks=sinks)
    check(ops, make(requests, hq, hkv, d, page, dtype, junk=math.nan, window=window, sinks=sinks, released=bool(window)), window=window,
          sinks=sinks)


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("requests,window,sinks", [([(1, 37), (1, 300), (1, 129)], 0, 0), ([(1, 500), (1, 33)], 70, 3),
                                                   ([(40, 140), (130, 500)], 0, 0), ([(40, 700), (130, 400)], 70, 3)])
def test_rows_that_no_token_sees(ops, junk, requests, window, sinks):
    for d, page, dtype in ((128, 16, BF16), (64, 64, F16)):
        check(ops, make(requests, 4, 2, d, page, dtype, window=window, sinks=sinks, junk=junk), window=window, sinks=sinks)
        check(ops, make(requests, 4, 2, d, page, dtype, window=window, sinks=sinks, junk=junk, released=True), window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,kv", [(3, 70), (100, 300)])
def test_values_that_only_later_tokens_see(ops, bad, n, kv):
    """A NaN at one position reaches the tokens from that position on, and no token before it."""
    made = make([(n, kv), (n, kv)], 4, 2, 128, 16, BF16)
    _, k, v, table, _, _ = made
    for b, x, at in ((0, v, kv - 2), (1, k, kv - n // 2)):
        x[int(table[b, at // 16]), :, at % 16, 5] = bad
    q, _, _, _, lens, starts = made
    got = ops.attention(q, k, v, table, lens, starts, max_q=n)
    ops.sync()
    want, _, tol, _, _ = oracle.attention(q, k, v, table, lens, starts)
    ok = torch.isfinite(want).all(-1)
    assert ok[:n - 2].all() and not ok[n - 1].any()
    assert not torch.isnan(got[ok]).any()
    within(got[ok], want[ok], tol[ok])
    if not math.isinf(bad) or n == 3:
        assert torch.equal(torch.isfinite(got[:n]), torch.isfinite(want[:n]))


@pytest.mark.parametrize("requests", [[(1, 200), (1, 40), (1, 16)], [(100, 200), (40, 40), (16, 16)]])
def test_entries_outside_the_pool_hide_their_keys(ops, requests):
    for holes in ((0,), (1, 2), range(16)):
        check(ops, make(requests, 4, 2, 128, 16, BF16, holes=holes))


@pytest.mark.parametrize("requests", [[(1, 900), (1, 33)], [(90, 400), (33, 33)]])
@pytest.mark.parametrize("gain,scale", [(30.0, None), (1.0, 4.0), (1.0, 1e-4), (0.0, None), (100.0, 3.0)])
def test_peaked_and_flat_scores(ops, requests, gain, scale):
    for dtype in (BF16, F16):
        check(ops, make(requests, 4, 2, 128, 32, dtype, gain=gain), scale=scale)


def test_rising_scores(ops):
    """Every key outweighs all before it, so the running maximum moves at each tile."""
    for n in (1, 60):
        q, k, v, table, lens, starts = make([(n, 2000)], 2, 1, 128, 16, BF16, seed=9)
        q.fill_(1.0)
        rise = torch.arange(2000, device="cuda") / 16.0
        k[table[0].long()[torch.arange(2000, device="cuda") // 16], 0, torch.arange(2000, device="cuda") % 16] = \
            (rise / 8)[:, None].to(BF16)
        check(ops, (q, k, v, table, lens, starts))
        k.neg_()
        check(ops, (q, k, v, table, lens, starts))


def test_first_scores_far_below_the_rest(ops):
    """Weights that a first maximum fits and a later one turns to nothing."""
    for n, kv in ((1, 700), (140, 700)):
        for big in (60.0, -60.0):
            q, k, v, table, lens, starts = make([(n, kv)], 2, 1, 64, 16, F16)
            q.fill_(1.0)
            at = torch.arange(kv, device="cuda")
            k[table[0].long()[at // 16], 0, at % 16] = torch.where(at < 400, -big / 8, big / 8)[:, None].to(F16)
            check(ops, (q, k, v, table, lens, starts))


@pytest.mark.parametrize("requests", [[(1, 1), (1, 200)], [(60, 100), (1, 200)]])
def test_float32_result_and_views(ops, requests):
    q, k, v, table, lens, starts = make(requests, 6, 2, 128, 16, BF16)
    check(ops, (q, k, v, table, lens, starts), out_dtype=F32)
    # heads before tokens, a wider row, an odd element offset
    for wide in (q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat((q, q), 2)[..., :128],
                 torch.cat((q.flatten(), q.flatten()[:9]))[9:].view_as(q).copy_(q)):
        check(ops, (wide, k, v, table, lens, starts))
    out = torch.full((q.shape[0], 6, 200), 7.0, dtype=BF16, device="cuda")
    check(ops, (q, k, v, table, lens, starts), out=out[..., 3:131])
    assert (out[..., :3] == 7).all() and (out[..., 131:] == 7).all()
    table2 = torch.cat((table, torch.full((2, 5), 1 << 20, dtype=torch.int32, device="cuda")), 1)
    check(ops, (q, k, v, table2, lens, starts))


def test_tokens_of_no_request_stay(ops):
    q, k, v, table, lens, starts = make([(1, 50), (1, 60)], 4, 2, 128, 16, BF16)
    for n in (1, 40):
        q2 = torch.randn(2 * n + 10, 4, 128, device="cuda").to(BF16)
        starts2 = torch.tensor([5, 5 + n, 5 + 2 * n], dtype=torch.int32, device="cuda")
        out = torch.full_like(q2, 9.0)
        check(ops, (q2, k, v, table, lens, starts2), out=out)
        assert (out[:5] == 9).all() and (out[5 + 2 * n:] == 9).all()


def test_offsets_past_32_bits(ops):
    """A pool whose pages lie 2^26 elements apart: byte offsets up to 12 GB."""
    gap, pages, d = 1 << 26, 48, 128
    room = torch.zeros(2, (pages - 1) * gap + 2 * 16 * d, dtype=BF16, device="cuda")
    for requests in ([(1, 700), (1, 60)], [(70, 700), (20, 60)]):
        q, k, v, table, lens, starts = make(requests, 4, 2, d, 16, BF16, spare=0)
        assert k.shape[0] <= pages
        far = [room[i].as_strided(k.shape, (gap, 16 * d, d, 1)) for i in range(2)]
        far[0].copy_(k)
        far[1].copy_(v)
        near = check(ops, (q, k, v, table, lens, starts))
        got = check(ops, (q, far[0], far[1], table, lens, starts))
        assert torch.equal(near[0], got[0]) and torch.equal(near[1], got[1])


def test_same_bits_again_on_another_stream_and_in_a_graph(ops):
    for requests in ([(1, 5000), (1, 17), (1, 900)], [(200, 900), (17, 17)]):
        made = make(requests, 8, 2, 128, 16, BF16)
        max_q = max(n for n, _ in requests)
        first = ops.attention(*made, max_q=max_q)
        for _ in range(3):
            assert torch.equal(first, ops.attention(*made, max_q=max_q))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = ops.attention(*made, max_q=max_q)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, again)
        out = torch.empty_like(first)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.attention(*made, max_q=max_q, out=out)
        for scale in (1.0, 0.5):
            made[0].mul_(scale)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.attention(*made, max_q=max_q))
        del graph


def test_nothing_to_do(ops):
    q, k, v, table, lens, starts = make([(1, 20)], 4, 2, 128, 16, BF16)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ops.attention(q[:0], k, v, table[:0], none, torch.zeros(1, dtype=torch.int32, device="cuda"), max_q=0).shape == (0, 4, 128)
    assert ops.attention(q[:0], k, v, table, lens, torch.zeros(2, dtype=torch.int32, device="cuda"), max_q=1).shape == (0, 4, 128)
    ops.sync()


# ---- append

def rows(tokens, hq, hkv, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, (hq + 2 * hkv) * d, device="cuda", generator=g) * (0.1 + 5 * torch.rand(tokens, 1, device="cuda", generator=g))
    return x.to(dtype).view(tokens, hq + 2 * hkv, d).split((hq, hkv, hkv), 1)


def angles(n, rotary):
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(rotary // 2, device="cuda", dtype=torch.float64) / max(1, rotary // 2))
    return a.cos().float(), a.sin().float()


def check_append(ops, q, k, v, k_pages, v_pages, *, rotary, norms=True, interleaved=False, seed=0, eps=1e-6, slots=None, **kw):
    tokens, d, page = q.shape[0], q.shape[2], k_pages.shape[2]
    r = random.Random(seed)
    cos, sin = angles(500, rotary) if rotary else (None, None)
    positions = torch.tensor([r.randrange(500) for _ in range(tokens)], dtype=torch.int32, device="cuda")
    if slots is None:
        slots = r.sample(range(k_pages.shape[0] * page), tokens)
        for i in range(3, tokens, 7):
            slots[i] = -1 - i
    slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
    gains = [1 + 0.5 * torch.randn(d, device="cuda") for _ in range(2)] if norms else [None, None]
    args = dict(q_norm=gains[0], k_norm=gains[1], eps=eps, interleaved=interleaved)
    want = oracle.append(q, k, v, cos, sin, positions, slots, k_pages, v_pages, **args)
    got = ops.append(q, k, v, cos, sin, positions, slots, k_pages, v_pages, **args, **kw)
    ops.sync()
    within(got, *want[0])
    within(k_pages, *want[1])  # rows of other slots: bound zero
    within(v_pages, *want[2])
    return got


def pool(pages, hkv, page, d, dtype, order="hnd"):
    shape = (pages, hkv, page, d) if order == "hnd" else (pages, page, hkv, d)
    k, v = torch.randn(shape, device="cuda").to(dtype), torch.randn(shape, device="cuda").to(dtype)
    return (k, v) if order == "hnd" else (k.transpose(1, 2), v.transpose(1, 2))


@pytest.mark.parametrize("tokens", [1, 2, 33, 200])
@pytest.mark.parametrize("src", [F32, BF16, F16])
@pytest.mark.parametrize("d,hq,hkv,dtype", [(128, 16, 8, BF16), (64, 7, 1, F16), (128, 5, 5, F16), (64, 8, 2, BF16)])
def test_append(ops, tokens, src, d, hq, hkv, dtype):
    for rotary, inter, norms in ((d, False, True), (d // 2, True, True), (8, False, False), (24, False, True), (0, False, True)):
        check_append(ops, *rows(tokens, hq, hkv, d, src), *pool(20, hkv, 16, d, dtype), rotary=rotary, interleaved=inter, norms=norms)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("order", ["hnd", "nhd"])
def test_append_pages_and_orders(ops, page, order):
    check_append(ops, *rows(40, 4, 2, 128, F32), *pool(5, 2, page, 128, BF16, order), rotary=128)


def test_append_views(ops):
    for src, d in ((F32, 128), (BF16, 64), (F16, 128)):
        q, k, v = rows(9, 4, 2, d, src)
        check_append(ops, q.contiguous(), k.contiguous(), v.contiguous(), *pool(4, 2, 16, d, BF16), rotary=d)
        turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]  # heads before tokens
        check_append(ops, *turned, *pool(4, 2, 16, d, BF16), rotary=d)
        flat = torch.zeros(9 * 8 * d + 1, dtype=src, device="cuda")[1:].view(9, 8, d)  # an odd element offset
        flat.copy_(torch.cat((q, k, v), 1))
        check_append(ops, *flat.split((4, 2, 2), 1), *pool(4, 2, 16, d, BF16), rotary=d)
        out = torch.full((9, 4, d + 8), 3.0, dtype=BF16, device="cuda")
        check_append(ops, q, k, v, *pool(4, 2, 16, d, BF16), rotary=d, out=out[..., :d])
        assert (out[..., d:] == 3).all()
        layers = [torch.randn(3, 4, 2, 16, d, device="cuda").to(BF16) for _ in range(2)]
        keep = [x.clone() for x in layers]
        check_append(ops, q, k, v, layers[0][1], layers[1][1], rotary=d)
        for x, y in zip(layers, keep):
            assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])


def test_append_small_and_large_values(ops):
    q, k, v = rows(20, 4, 2, 128, F32)
    for size in (0.0, 1e-12, 1e12):
        check_append(ops, q * size, k * size, v * min(size, 1e3), *pool(4, 2, 16, 128, BF16), rotary=128, eps=1e-6)
    check_append(ops, q, k, v, *pool(4, 2, 16, 128, BF16), rotary=128, eps=0.0)


def test_append_outside_is_reported_and_not_stored(ops):
    from bnn_b200 import accel
    q, k, v = rows(4, 4, 2, 128, F32)
    cos, sin = angles(50, 128)
    for positions, slots in (([0, 50, 1, 2], [0, 1, 2, 3]), ([0, -1, 1, 2], [0, 1, 2, 3]), ([0, 1, 2, 3], [0, 64, 2, 3]),
                             ([0, 1, 2, 3], [0, 2147483647, 2, 3])):
        kp, vp = pool(4, 2, 16, 128, BF16)
        before = kp.clone(), vp.clone()
        out = ops.append(q, k, v, cos, sin, torch.tensor(positions, dtype=torch.int32, device="cuda"),
                         torch.tensor(slots, dtype=torch.int32, device="cuda"), kp, vp)
        with pytest.raises(accel.BnnError) as e:
            ops.sync()
        assert e.value.status == accel.ERANGE
        ops.sync()  # read once
        for now, was in zip((kp, vp), before):
            flat, old = (x.transpose(1, 2).reshape(64, -1) for x in (now, was))
            changed = torch.nonzero((flat != old).any(1))[:, 0].tolist()
            assert changed == [0, 2, 3]
        assert bool((out[1] == 0).all()) == (positions[1] not in range(50))


def test_prompt_then_single_tokens_agree(ops):
    """A prompt appended and attended at once, and token by token, give each token the same
    definition: both stay within the bound of the 64-bit answer."""
    tokens, hq, hkv, d, page = 45, 4, 2, 128, 16
    q, k, v = rows(tokens, hq, hkv, d, F32)
    cos, sin = angles(tokens, d)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32)
    slots = (table[0].long()[positions.long() // page] * page + positions % page).int()
    caches = [pool(3, hkv, page, d, BF16) for _ in range(2)]
    qr = ops.append(q, k, v, cos, sin, positions, slots, *caches[0])
    one = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    whole, _ = check(ops, (qr, *caches[0], table, one[1:], one))
    want, _, tol, _, _ = oracle.attention(qr, *caches[0], table, one[1:], one)
    for t in range(tokens):
        qt = ops.append(q[t:t + 1], k[t:t + 1], v[t:t + 1], cos, sin, positions[t:t + 1], slots[t:t + 1], *caches[1])
        assert torch.equal(qt, qr[t:t + 1])
        got = ops.attention(qt, *caches[1], table, one[1:] * 0 + t + 1, (one > 0).int(), max_q=1)
        within(got, want[t:t + 1], tol[t:t + 1])


# ---- refusals

def test_attention_refusals(ops):
    from bnn_b200 import accel
    q, k, v, table, lens, starts = make([(1, 20), (1, 30)], 4, 2, 128, 16, BF16)

    def refused(status, *args, **kw):
        kw = {"max_q": 1, **kw}
        with pytest.raises(accel.BnnError) as e:
            ops.attention(*args, **kw)
        assert e.value.status == status

    good = (q, k, v, table, lens, starts)
    EINVAL, ENOTSUP = accel.EINVAL, accel.ENOTSUP
    refused(EINVAL, q.float(), *good[1:])
    refused(EINVAL, q.half(), *good[1:])
    refused(EINVAL, q, k.float(), v.float(), *good[3:])
    refused(EINVAL, q, k, v.half(), *good[3:])
    refused(EINVAL, q, k, v[:1], *good[3:])
    refused(EINVAL, q[:, :3], *good[1:])  # heads no multiple of kv_heads
    refused(EINVAL, q[..., :64], *good[1:])
    refused(EINVAL, q[0], *good[1:])
    refused(EINVAL, q, k, v, table.long(), lens, starts)
    refused(EINVAL, q, k, v, table, lens.long(), starts)
    refused(EINVAL, q, k, v, table, lens[:1], starts)
    refused(EINVAL, q, k, v, table, lens, starts[:2])
    refused(EINVAL, q.cpu(), *good[1:])
    refused(EINVAL, q, k.cpu(), v.cpu(), *good[3:])
    refused(EINVAL, *good, scale=0.0)
    refused(EINVAL, *good, scale=-1.0)
    refused(EINVAL, *good, scale=math.nan)
    refused(EINVAL, *good, scale=math.inf)
    refused(EINVAL, *good, window=-1)
    refused(EINVAL, *good, sinks=-1)
    refused(EINVAL, *good, max_q=-1)
    refused(EINVAL, *good, out_dtype=F16)
    refused(EINVAL, *good, out=torch.empty(2, 4, 128, dtype=F16, device="cuda"))
    refused(EINVAL, *good, out=torch.empty(2, 4, 64, dtype=BF16, device="cuda"))
    odd = torch.empty(k.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(k)
    refused(EINVAL, q, odd, v, *good[3:])  # the cache off its 16-byte boundary
    refused(EINVAL, q.clone().requires_grad_(), *good[1:])
    refused(ENOTSUP, torch.empty(2, 4, 96, dtype=BF16, device="cuda"), k[..., :96], v[..., :96], *good[3:])
    small = torch.empty(3, 2, 8, 128, dtype=BF16, device="cuda")
    refused(ENOTSUP, q, small, small, *good[3:])
    refused(ENOTSUP, torch.empty(2, 34, 128, dtype=BF16, device="cuda"), *good[1:])
    many = 5000
    refused(ENOTSUP, q, k, v, table[:1].expand(many, -1).contiguous(), lens[:1].expand(many).contiguous(),
            torch.zeros(many + 1, dtype=torch.int32, device="cuda"))
    ops.sync()


def test_more_new_tokens_than_declared(ops):
    from bnn_b200 import accel
    for n in (40, 300):
        q, k, v, table, lens, starts = make([(n, n), (1, 30)], 4, 2, 128, 16, BF16)
        for max_q in (1, 20):
            out = torch.full_like(q, 9.0)
            ops.attention(q, k, v, table, lens, starts, max_q=max_q, out=out)
            with pytest.raises(accel.BnnError) as e:
                ops.sync()
            assert e.value.status == accel.ERANGE
            assert (out[:n] == 9).all()
            want, _, tol, _, _ = oracle.attention(q, k, v, table, lens, starts)
            within(out[n:], want[n:], tol[n:])


def test_workspace_too_small_and_too_many_requests(ops):
    from bnn_b200 import accel, paged
    made = make([(1, 20)] * 3, 4, 2, 64, 16, BF16)
    small = paged.Paged(ops.device, max_batch=3)
    check(small, made)
    small._workspace = small._workspace[:-1]
    with pytest.raises(accel.BnnError) as e:
        small.attention(*made, max_q=1)
    assert e.value.status == accel.EINVAL
    with pytest.raises(accel.BnnError) as e:
        paged.Paged(ops.device, max_batch=2).attention(*made, max_q=1)
    assert e.value.status == accel.ENOTSUP


def test_append_refusals(ops):
    from bnn_b200 import accel
    q, k, v = rows(3, 4, 2, 128, F32)
    kp, vp = pool(4, 2, 16, 128, BF16)
    cos, sin = angles(50, 128)
    p = torch.zeros(3, dtype=torch.int32, device="cuda")
    s = torch.arange(3, dtype=torch.int32, device="cuda")

    def refused(status, *args, **kw):
        with pytest.raises(accel.BnnError) as e:
            ops.append(*args, **kw)
        assert e.value.status == status

    EINVAL, ENOTSUP = accel.EINVAL, accel.ENOTSUP
    refused(EINVAL, q, k.half(), v, cos, sin, p, s, kp, vp)
    refused(EINVAL, q.double(), k.double(), v.double(), cos, sin, p, s, kp, vp)
    refused(EINVAL, q, k[:2], v, cos, sin, p, s, kp, vp)
    refused(EINVAL, q, k[:, :1], v, cos, sin, p, s, kp, vp)
    refused(EINVAL, q, k, v, cos, sin, p.long(), s, kp, vp)
    refused(EINVAL, q, k, v, cos, sin, p, s[:2], kp, vp)
    refused(EINVAL, q, k, v, cos.double(), sin.double(), p, s, kp, vp)
    refused(EINVAL, q, k, v, cos, sin[:, :10], p, s, kp, vp)
    refused(EINVAL, q, k, v, torch.cat((cos, cos), 1), torch.cat((sin, sin), 1), p, s, kp, vp)  # more than head_dim
    refused(ENOTSUP, q, k, v, cos[:, :6].contiguous(), sin[:, :6].contiguous(), p, s, kp, vp)
    refused(EINVAL, q, k, v, cos, sin, p, s, kp.float(), vp.float())
    refused(EINVAL, q, k, v, cos, sin, p, s, kp, vp.cpu())
    refused(EINVAL, q, k, v, cos, sin, p, s, kp, vp, q_norm=torch.ones(64, device="cuda"))
    refused(EINVAL, q, k, v, cos, sin, p, s, kp, vp, eps=-1.0)
    refused(EINVAL, q, k, v, cos, sin, p, s, kp, vp, eps=math.nan)
    refused(EINVAL, q, k, v, cos, sin, p, s, kp, vp, out=torch.empty(3, 4, 128, device="cuda"))
    refused(EINVAL, q.clone().requires_grad_(), k, v, cos, sin, p, s, kp, vp)
    refused(ENOTSUP, q[..., :32], k[..., :32], v[..., :32], cos[:, :16].contiguous(), sin[:, :16].contiguous(), p, s, kp[..., :32],
            vp[..., :32])
    ops.sync()


def test_starved_loads_time_out_then_recover(ops):
    """With the tiles kernel's loads withheld and the limit at 1 ms every wait of it runs
    out (nothing faults, nothing is in flight); the next sync says so, and with the limits
    restored the same call is right."""
    import ctypes
    from bnn_b200 import accel
    hook = ops.device.api.dll.bnn_b200_test_wait_limit
    hook.restype, hook.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int]
    made = make([(200, 300), (40, 40)], 4, 2, 128, 16, BF16)
    torch.cuda.synchronize()
    assert hook(ops.device.handle, 1_000_000, 1) == accel.OK
    try:
        ops.attention(*made, max_q=200)
        with pytest.raises(accel.BnnError) as e:
            ops.sync()
    finally:
        torch.cuda.synchronize()
        assert hook(ops.device.handle, 0, 0) == accel.OK
    assert e.value.status == accel.ETIMEOUT
    check(ops, made)


@pytest.mark.parametrize("batch", [127, 320, 321, 1000])
def test_many_requests(ops, batch):
    """More requests than a CTA has threads, of all sizes."""
    r = random.Random(batch)
    few = [(r.choice((0, 1, 1, 1, 2)), r.randrange(0, 90)) for _ in range(batch)]
    check(ops, make(few, 2, 1, 64, 16, BF16))
    some = [(r.choice((0, 1, 1, 9, 40)), r.randrange(0, 90)) for _ in range(batch - 1)] + [(150, 1200)]
    check(ops, make(some, 2, 1, 64, 16, BF16))
