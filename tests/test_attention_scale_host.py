"""A scale whose exponent (scale times log2 e) leaves the range of floats is refused on the host."""
import math

import pytest

from test_attention_host import backward, forward, net, refused, shape  # noqa: F401


@pytest.mark.parametrize("scale", [3.0e38, 2.5e38, math.inf, -0.5])
def test_scales(net, scale):  # noqa: F811
    refused(forward(net, a=shape(scale=scale)), "scale")
    refused(backward(net, a=shape(scale=scale)), "scale")
