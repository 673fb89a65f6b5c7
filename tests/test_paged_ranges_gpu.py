"""Lengths and offsets that only the device sees (marked gpu): a request whose
numbers cannot be right is reported and left alone, the others are served."""
import pytest

torch = pytest.importorskip("torch")
import paged_oracle as oracle  # noqa: E402
from test_paged_gpu import BF16, check, make, ops, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# a call of each kernel, and of both
CALLS = {"split": [(1, 100), (2, 333), (1, 50)], "tiles": [(40, 100), (130, 333), (17, 50)],
         "both": [(1, 1100), (300, 1500), (1, 2000), (40, 40), (30, 900)]}


def reported(ops, made, bad, max_q):  # noqa: F811
    """The call's status is BNN_ERANGE once; every request but `bad` is right, and nothing else is written."""
    from bnn_b200 import accel
    q, k, v, table, lens, starts = made
    out = torch.full_like(q, 9.0)
    ops.attention(q, k, v, table, lens, starts, max_q=max_q, out=out)
    with pytest.raises(accel.BnnError) as e:
        ops.sync()
    assert e.value.status == accel.ERANGE
    ops.sync()
    good = [b for b in range(len(lens)) if b != bad]
    served = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for b in good:
        n0, n1 = int(starts[b]), int(starts[b + 1])
        served[n0:n1] = True
        want, _, tol, _, _ = oracle.attention(q[n0:n1], k, v, table[b:b + 1], lens[b:b + 1],
                                              torch.tensor([0, n1 - n0], dtype=torch.int32, device="cuda"))
        within(out[n0:n1], want, tol)
    assert (out[~served] == 9).all()


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("d", [64, 128])
def test_a_table_too_narrow_for_one_request(ops, name, d):  # noqa: F811
    requests = CALLS[name]
    longest = max(range(len(requests)), key=lambda b: requests[b][1])
    q, k, v, table, lens, starts = make(requests, 4, 2, d, 16, BF16)
    second = sorted(kv for _, kv in requests)[-2]
    narrow = table[:, :-(-second // 16)].contiguous()
    reported(ops, (q, k, v, narrow, lens, starts), longest, max(n for n, _ in requests))
    check(ops, (q, k, v, table, lens, starts))


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("length", [-1, -2147483648, 2147483647])
def test_a_length_that_cannot_be(ops, name, length):  # noqa: F811
    requests = CALLS[name]
    for bad in (0, 1):
        q, k, v, table, lens, starts = make(requests, 4, 2, 128, 16, BF16)
        lens[bad] = length
        reported(ops, (q, k, v, table, lens, starts), bad, max(n for n, _ in requests))


@pytest.mark.parametrize("name", CALLS)
def test_tokens_outside_the_call(ops, name):  # noqa: F811
    requests = CALLS[name]
    q, k, v, table, lens, starts = make(requests, 4, 2, 128, 16, BF16)
    max_q = max(n for n, _ in requests) + 3
    last = len(requests) - 1
    for at, value, bad in ((last + 1, q.shape[0] + 1, last), (0, -1, 0)):
        off = starts.clone()
        off[at] = value
        # the request's own tokens stay unwritten too
        reported(ops, (q, k, v, table, lens, off), bad, max_q)


def test_requests_without_tokens_may_hold_anything(ops):  # noqa: F811
    """Padding of a batch: no new tokens, any length, offsets that go back."""
    q, k, v, table, lens, starts = make([(1, 60), (0, 20), (1, 90), (0, 0), (0, 0)], 4, 2, 128, 16, BF16)
    want, _ = check(ops, (q, k, v, table, lens, starts))
    lens[1], lens[3], lens[4] = -5, 1 << 30, 100000
    starts[4], starts[5] = 0, 0
    got = ops.attention(q, k, v, table, lens, starts, max_q=1)
    ops.sync()
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [1, 40])
def test_one_table_row_for_all_requests(ops, n):  # noqa: F811
    """Requests that continue one prompt: the same pages for each, an expanded row."""
    q, k, v, table, lens, starts = make([(n, 300)] * 4, 4, 2, 128, 16, BF16)
    shared = table[1:2].expand(4, -1)
    want = ops.attention(q, k, v, shared.contiguous(), lens, starts, max_q=n)
    got, _ = check(ops, (q, k, v, shared, lens, starts))
    assert torch.equal(got, want)
