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
