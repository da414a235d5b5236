"""The example layer end to end: training, a prompt in chunks and generation agree to what the cache's type costs."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


# bf16 alone: the two paths round q, k and the output alike and sum in another order (half a unit, 2^-8, a few times);
# codes: keys and values are off by up to half a step of 1/127 (int8), or 1/16 (fp8: 4 bits of significand), of their
# row's largest value, which is about 2.5 times its mean magnitude
@pytest.mark.parametrize("codes,most", [("16bit", 2.0**-6), ("int8", 2.5 / 127), ("fp8", 2.5 / 32)])
@pytest.mark.parametrize("window,sinks", [(256, 4), (64, 0)])
def test_generation_agrees_with_training(device, codes, most, window, sinks):
    import windowed_layer

    assert windowed_layer.main(["--codes", codes, "--window", str(window), "--sinks", str(sinks)]) <= most
