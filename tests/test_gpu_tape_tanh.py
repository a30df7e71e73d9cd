"""The gradient of tanh that the tape forms from whole inputs."""
import numpy as np
import pytest

from test_gpu_tape import be, dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, top", [(np.float32, 40.0), (np.float64, 340.0)])
def test_tanh_slope_far_out(be, dtype, top):
    """1 - tanh^2 = 4 s(2x) s(-2x), s the sigmoid, in the type under test against 4 e / (1 + e)^2 in a wider one, relative to the value: each
    s is 1 / (1 + exp) with an exponential within 2 units in the last place of an argument that is exact (4 half steps), the sum and the
    quotient (2 each, the f64 reciprocal is within a unit), and three products: 2 * 8 + 3 < 24 half steps.  The
    loss's own gradient is 2^-k: its products are exact.  Where e comes near the smallest normal number, half of its step is added."""
    from rtensors_amd import tensor as T
    W = {np.float32: np.float64, np.float64: np.longdouble}[dtype]
    x = np.concatenate([np.linspace(-top, top, 4095), [0.0]]).astype(dtype)
    zero = np.zeros_like(x)
    _, g, _ = T.activation_step(dev(be, x), dev(be, zero), dev(be, np.full_like(x, 2)), "tanh", 0.0, seed_with_loss=False)
    got = -g.to_numpy().astype(W) * x.size
    e = np.exp(-2 * np.abs(x.astype(W)))
    want = 4 * e / (1 + e) ** 2
    off = np.abs(got - want) - np.finfo(dtype).tiny * np.finfo(dtype).eps * x.size * 4
    assert (off <= 24 * np.finfo(dtype).eps / 2 * want).all(), float((off / want).max() / (np.finfo(dtype).eps / 2))
