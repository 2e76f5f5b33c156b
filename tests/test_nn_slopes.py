"""The slopes of the activations beside F32 tensors, in the mean square, next to their formula evaluated in F32 step by step."""
import numpy as np
import pytest

from tests import nn_reference as ref
from tests.support import DT, GPU, array, from_f64, h, normal, tensor

pytestmark = pytest.mark.gpu
F = np.float32


def on_gpu(values):
    return tensor(from_f64(values, DT.F32), DT.F32, list(values.shape), GPU)


@pytest.mark.parametrize("S", [1, 70])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes_of_normal_arguments(act, S):
    """A weight of zero makes z the bias, one row with a gradient of one makes the sum the slope. The roundings of F32: the slope
    is rounded once (0.29 units of 2^-24 of a binade in the mean square, up to 0.58 relative), its last addition once more,
    and its logistic or normal part, of which it holds at most 1 + |z| slope times, a few units: 1.2 units in the mean square
    are allowed, where the formula in F32 with correctly rounded functions has 0.7 to 0.8."""
    C = 1 << 15
    z = ref.rounded(normal(8, C), DT.F32)
    x, grad = normal(9, S * C).reshape(1, S, C), np.zeros((1, S, C))
    grad[0, S // 2] = 1
    w, b = on_gpu(np.zeros(C)), on_gpu(z)
    _, mean, rstd = h.group_norm(on_gpu(x), C // 8, w, b, 1e-5, act)
    _, _, d_bias = h.grad_group_norm(on_gpu(grad), on_gpu(x), mean, rstd, C // 8, w, b, act)
    slope = ref.activate(z, act)[1]
    off = array(d_bias).astype(np.float64) - slope
    assert np.sqrt((off ** 2).mean() / (slope ** 2).mean()) <= 1.2 * 2.0 ** -24
