"""Factors that are not finite, from states that are not zero: no state after them is finite, in `out`, in `last` or backwards,
and other channels are as they were."""
import numpy as np
import pytest

from tests.support import DT, GPU, array, from_f64, h, normal, tensor, uniform

pytestmark = pytest.mark.gpu


def on_gpu(values):
    return tensor(from_f64(values, DT.F32), DT.F32, list(values.shape), GPU)


@pytest.mark.parametrize("gate", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T, C", [(2, 8), (16, 8), (90, 8), (700, 8), (700, 3), (700, 300), (40, 200), (3000, 72)])
def test_no_state_after_it_is_finite(T, C, gate):
    n, bad = T * C, C // 2
    x, grad = (normal(k, n).reshape(1, T, C) for k in (1, 2))
    start, grad_last = (normal(k, C).reshape(1, C) + 1 for k in (3, 4))
    for at in sorted({0, 1, T // 3, T // 2, T - 1}):
        factors = uniform(5, n, 0.6, 1.0).reshape(1, T, C)
        good = [array(t) for t in h.linear_recurrence(on_gpu(factors), on_gpu(x), on_gpu(start))]
        factors[0, at, bad] = gate
        out, last = h.linear_recurrence(on_gpu(factors), on_gpu(x), on_gpu(start))
        got = array(out).reshape(T, C)
        assert np.isfinite(got[:at, bad]).all() and not np.isfinite(got[at:, bad]).any() and not np.isfinite(array(last).reshape(C)[bad])
        others = [k for k in range(C) if k != bad]
        assert np.array_equal(got[:, others], good[0].reshape(T, C)[:, others])
        assert np.array_equal(array(last).reshape(C)[others], good[1].reshape(C)[others])
        back = h.grad_linear_recurrence(on_gpu(grad), on_gpu(grad_last), on_gpu(factors), on_gpu(x), on_gpu(x), on_gpu(start))
        d_input = array(back[1]).reshape(T, C)
        assert np.isfinite(d_input[at:, bad]).all() and not np.isfinite(d_input[:at, bad]).any()
        assert not np.isfinite(array(back[2]).reshape(C)[bad]) and np.isfinite(d_input[:, others]).all()
