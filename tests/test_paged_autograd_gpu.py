"""The paged operators and autograd (marked gpu): they have no derivatives, so a
tensor that wants one is refused, and what they write counts as written."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # noqa: E402
from test_paged_gpu import BF16, F32, angles, make, ops, pool, rows  # noqa: E402, F401

pytestmark = pytest.mark.gpu

APPEND = ("q", "k", "v", "cos", "sin", "positions", "slots", "k_pages", "v_pages")
ATTENTION = ("q", "k_pages", "v_pages", "page_table", "kv_lens", "q_starts")


def append_tensors():
    kp, vp = pool(4, 2, 16, 128, BF16)
    q, k, v = (x.contiguous() for x in rows(3, 4, 2, 128, F32))
    cos, sin = angles(50, 128)
    at = torch.arange(3, dtype=torch.int32, device="cuda")
    named = dict(zip(APPEND, (q, k, v, cos, sin, at, at.clone(), kp, vp)))
    return {**named, "q_norm": torch.ones(128, device="cuda"), "k_norm": torch.ones(128, device="cuda"),
            "out": torch.empty(3, 4, 128, dtype=BF16, device="cuda")}


def attention_tensors():
    named = dict(zip(ATTENTION, make([(1, 20), (1, 30)], 4, 2, 128, 16, BF16)))
    return {**named, "out": torch.empty_like(named["q"])}


CASES = [("append", n) for n in ("q", "k", "v", "cos", "sin", "k_pages", "v_pages", "q_norm", "k_norm", "out")] + \
        [("attention", n) for n in ("q", "k_pages", "v_pages", "out")]


@pytest.mark.parametrize("operator,name", CASES)
def test_wanted_gradients_are_refused(ops, operator, name):  # noqa: F811
    from bnn_b200 import accel
    tensors = append_tensors() if operator == "append" else attention_tensors()
    extra = {} if operator == "append" else {"max_q": 1}
    call = getattr(ops, operator)
    tensors[name].requires_grad_()
    with pytest.raises(accel.BnnError) as e:
        call(**tensors, **extra)
    assert e.value.status == accel.EINVAL
    with torch.no_grad():
        call(**tensors, **extra)
    ops.sync()


@pytest.mark.parametrize("operator,name", CASES)
def test_tangents_are_refused(ops, operator, name):  # noqa: F811
    from bnn_b200 import accel
    tensors = append_tensors() if operator == "append" else attention_tensors()
    extra = {} if operator == "append" else {"max_q": 1}
    call = getattr(ops, operator)
    with forward_ad.dual_level():
        dual = {**tensors, name: forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))}
        with pytest.raises(accel.BnnError) as e:
            call(**dual, **extra)
        assert e.value.status == accel.EINVAL
    call(**tensors, **extra)
    ops.sync()


@pytest.mark.parametrize("operator,names", [("append", ("k_pages", "v_pages", "out")), ("attention", ("out",))])
def test_writes_are_counted(ops, operator, names):  # noqa: F811
    """A tensor that autograd saved and an operator then wrote: backward refuses it, as after any in-place operation."""
    tensors = append_tensors() if operator == "append" else attention_tensors()
    extra = {} if operator == "append" else {"max_q": 1}
    counts = {n: t._version for n, t in tensors.items()}
    losses = []
    for n in names:
        w = torch.ones((), device="cuda", dtype=tensors[n].dtype, requires_grad=True)
        losses.append((tensors[n] * w).sum())  # saves tensors[n]
    getattr(ops, operator)(**tensors, **extra)
    ops.sync()
    assert {n for n, t in tensors.items() if t._version != counts[n]} == set(names)
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_inference_tensors_are_taken(ops):  # noqa: F811
    with torch.inference_mode():
        a, b = append_tensors(), attention_tensors()
        ops.append(**a)
        ops.attention(**b, max_q=1)
    ops.append(**a)
    ops.attention(**b, max_q=1)
    ops.sync()
