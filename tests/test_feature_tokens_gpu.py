"""The example that runs the token operators together, against its float64 chain. Its fp16 tensors are rounded
five times on the way to the attention rows (2^-11 each, added at most: 2.4e-3). The steps add the 8-bit cache: a
value is off by half a step of its page's largest value, about four deviations over 127, so a deviation by
4 / 127 / sqrt(12) = 0.9%, of keys and of values, in a chain of four steps."""
import pytest

from examples import feature_tokens

pytestmark = pytest.mark.gpu


def test_feature_tokens(gpu):
    attention, last = feature_tokens.main()
    assert attention <= 2.4e-3 and last <= 4 * 2 * 9e-3
