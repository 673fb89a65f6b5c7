"""The serving example as a user runs it (marked gpu): requests of unlike lengths
over W1A8 linears and one paged cache, each request's last logits against the
same layers with plain attention over the whole request.

The cache is bfloat16 (relative rounding 2^-8 per key and value) and every
linear quantises its input rows to 8 bits (relative 2^-8 of the row's largest
value), so a flipped code moves a row by no more than such a rounding: a few
roundings per layer of independent sign, 2^-8 * sqrt(6 * layers) < 5 % for the
three layers here."""
import sys
from pathlib import Path

import pytest

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.mark.parametrize("args", [
    ["--requests", "7", "--batch", "4", "--longest", "200", "--new", "12"],
    ["--requests", "3", "--batch", "1", "--longest", "40", "--new", "20"],  # one row per step: the one-kernel linears
    ["--requests", "5", "--batch", "5", "--longest", "1300", "--new", "5", "--chunk", "100"],
])
def test_requests_agree_with_plain_attention(args):
    import paged_serving
    assert paged_serving.main([*args, "--layers", "3", "--check"]) < 0.05
