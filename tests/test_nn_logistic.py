"""The logistic function in both operators over its whole range, in steps of F32 that do not grow with the argument."""
import numpy as np
import pytest

from tests import nn_reference as ref
from tests.support import DT, GPU, array, from_f64, h, normal, tensor, to_f64

pytestmark = pytest.mark.gpu
U = ref.COMPUTE[DT.F32]


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


def arguments(far):
    """From -far to far, dense about zero, as F32 holds them."""
    z = np.concatenate([np.linspace(-far, far, 20001), np.linspace(-4, 4, 8001), 2.0 ** np.arange(-30, 6), -(2.0 ** np.arange(-30, 6))])
    return ref.rounded(z, DT.F32)


# Units of 2^-24 of the value. The exponential: two for the hardware's, one for its correction. The sum: one, and the
# reciprocal two: six for the logistic, for a ratio of both another one.
@pytest.mark.parametrize("T", [1, 40])
def test_a_sigmoid_gate_and_what_is_left_of_it(T):
    """With no input the state is the gate's factor times the initial one, without an initial state what is left of it times
    the input; later steps have a gate of infinity, which keeps the state."""
    z = arguments(86.0)
    C = z.size
    gate = np.full((1, T, C), np.inf)
    gate[0, 0] = z
    x = np.zeros((1, T, C))
    one = np.ones((1, C))
    _, kept = h.linear_recurrence(on_gpu(gate, DT.F32), on_gpu(x, DT.F32), on_gpu(one, DT.F32), None, True)
    a = ref.sigmoid(z)
    ref.assert_within(values(kept)[0], a, 7 * U * a, DT.F32, "a")
    x[0, 0] = 1.0
    _, left = h.linear_recurrence(on_gpu(gate, DT.F32), on_gpu(x, DT.F32), None, None, True)
    a = ref.sigmoid(-z)
    ref.assert_within(values(left)[0], a, 7 * U * a, DT.F32, "1 - a")


def test_the_ends_of_the_gate():
    z = np.array([np.inf, -np.inf, np.nan, 200.0, -200.0, 3e38, -3e38, 0.0])
    gate = z.reshape(1, 1, -1)
    x, start = np.full(gate.shape, 2.0), np.full((1, z.size), 3.0)
    out, _ = h.linear_recurrence(on_gpu(gate, DT.F32), on_gpu(x, DT.F32), on_gpu(start, DT.F32), None, True)
    assert np.array_equal(values(out)[0, 0], [3, 2, np.nan, 3, 2, 3, 2, 2.5], equal_nan=True)


@pytest.mark.parametrize("S", [1, 80])
def test_silu(S):
    """A weight of zero makes z the bias itself. Its slope is a (1 + z (1 - a)): seven units of each of the two terms, which
    cancel where it is small, three more for the product and the sum."""
    z = arguments(80.0)
    C = z.size // 8 * 8
    z = z[:C]
    w, b = on_gpu(np.zeros(C), DT.F32), on_gpu(z, DT.F32)
    x = on_gpu(normal(3, S * C).reshape(1, S, C), DT.F32)
    out, mean, rstd = h.group_norm(x, C // 8, w, b, 1e-5, "silu")
    a, rest = ref.sigmoid(z), ref.sigmoid(-z)
    want = np.broadcast_to(z * a, (1, S, C))
    ref.assert_within(values(out), want, 8 * U * np.abs(want), DT.F32, "silu")
    grad = np.zeros((1, S, C))
    grad[0, S // 2] = 1.0
    _, _, d_bias = h.grad_group_norm(on_gpu(grad, DT.F32), x, mean, rstd, C // 8, w, b, "silu")
    slope = a * (1 + z * rest)
    # 1 - a as a difference is off by a unit of one, and by a's own six units.
    bound = 10 * U * (a + np.abs(z) * a * rest) + np.abs(z) * a * (7 * U * a + U)
    ref.assert_within(values(d_bias), slope, bound, DT.F32, "the slope of silu")
