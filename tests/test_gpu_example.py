"""The example runs the feed-forward block's operators together."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_feed_forward_example(dev, dtype):
    """It learns its batch, and one token at a time gives the batch's rows: outputs of
    norms, of order 1 to 4, after two blocks; in bf16 a rounding of h, the branch and n
    each (2^-8) may fall differently, some ten of them in all, in f32 the sums' orders."""
    import feed_forward

    losses, worst = feed_forward.main(["--dtype", dtype, "--steps", "40"])
    assert losses[-1] < 0.7 * losses[0]
    assert worst <= (10 * 4 * 2.0 ** -8 if dtype == "bf16" else 1e-4)
