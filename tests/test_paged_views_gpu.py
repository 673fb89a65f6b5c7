"""Tensors of unusual strides at the paged operators (marked gpu)."""
import pytest

torch = pytest.importorskip("torch")
from test_paged_gpu import BF16, F32, check, check_append, make, ops, pool, rows  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,heads,strides", [(1, 4, (513, 128, 1)), (3, 1, (132, 7, 1)), (1, 1, (3, 5, 1)), (1, 4, (0, 128, 1))])
def test_a_dimension_of_one_may_have_any_stride(ops, tokens, heads, strides):  # noqa: F811
    """Nothing steps over it."""
    buffer = torch.empty(2000, dtype=BF16, device="cuda")
    out = buffer.as_strided((tokens, heads, 128), strides)
    q, k, v = rows(tokens, heads, 1, 128, F32)
    check_append(ops, q, k, v, *pool(4, 1, 16, 128, BF16), rotary=0, out=out)
    made = make([(1, 40)] * tokens, heads, 1, 128, 16, BF16)
    check(ops, made, out=out)
    odd = buffer.as_strided((tokens, heads, 128), strides, 1000)
    odd.copy_(made[0])
    check(ops, (odd, *made[1:]))


@pytest.mark.parametrize("shape", [(1, 4, 128), (3, 1, 128)])
def test_an_expanded_result_is_refused(ops, shape):  # noqa: F811
    """Its rows share memory: whichever is written last would stay."""
    from bnn_b200 import accel
    out = torch.empty(shape, dtype=BF16, device="cuda").expand(3, 4, 128)
    made = make([(1, 40)] * 3, 4, 2, 128, 16, BF16)
    at = torch.arange(3, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.attention(*made, max_q=1, out=out),
                 lambda: ops.append(*rows(3, 4, 2, 128, F32), None, None, at, at, *pool(2, 2, 16, 128, BF16), out=out)):
        with pytest.raises(accel.BnnError) as e:
            call()
        assert e.value.status == accel.EINVAL
    ops.sync()


def test_arguments_of_another_kind_are_refused(ops):  # noqa: F811
    """With the wrappers' error, and nothing launched: the result given stays as it is."""
    from bnn_b200 import accel
    q, k, v, table, lens, starts = made = make([(1, 40)], 4, 2, 128, 16, BF16)
    at = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((1, 4, 128), 9.0, dtype=BF16, device="cuda")
    many = torch.ones(2)  # no truth value
    new = (*rows(1, 4, 2, 128, F32), None, None, at, at, *pool(2, 2, 16, 128, BF16))
    for call in (lambda: ops.append(*new, out=out, interleaved=many), lambda: ops.attention(*made, max_q=1, out=out, return_lse=many),
                 lambda: ops.attention(q, k, v, None, lens, starts, max_q=1, out=out),
                 lambda: ops.attention(q, k, v, 3, lens, starts, max_q=1, out=out),
                 lambda: ops.attention(None, k, v, table, lens, starts, max_q=1, out_dtype=BF16),
                 lambda: ops.attention(*made, max_q=1, out=7, out_dtype=F32), lambda: ops.attention(*made, max_q=1.5, out=out),
                 lambda: ops.attention(*made, max_q=1, out=out, scale="half"), lambda: ops.append(*new, out=out, eps=None)):
        with pytest.raises(accel.BnnError) as e:
            call()
        assert e.value.status == accel.EINVAL
    ops.sync()
    assert (out == 9).all()
