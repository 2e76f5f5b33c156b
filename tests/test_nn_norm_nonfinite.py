"""Weights, biases and elements that are not finite, or far out, in one group: the other groups' gradients are the formula's."""
import numpy as np
import pytest

from tests import nn_reference as ref
from tests.support import DT, GPU, array, from_f64, h, normal, tensor, to_f64

pytestmark = pytest.mark.gpu


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


# Groups that leave lanes or vectors of lanes without elements, groups that do not, and maps of larger ones.
SIZES = [(5, 1, 160, 4), (5, 1, 40, 4), (70, 1, 96, 2), (3, 7, 160, 4), (4, 1, 8160, 2), (4, 1, 5000, 2), (2, 100, 160, 4)]


@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("which, value", [("weight", np.nan), ("weight", np.inf), ("bias", np.nan), ("bias", -np.inf)])
@pytest.mark.parametrize("N, S, C, G", SIZES)
def test_a_weight_or_bias_that_is_not_finite_stays_in_its_group(N, S, C, G, which, value, act):
    for dtype in (DT.BF16, DT.F32):
        u = ref.COMPUTE[dtype]
        x, grad = (ref.rounded(normal(k, N * S * C, 0.2).reshape(N, S, C), dtype) for k in (1, 2))
        weight, bias = (ref.rounded(normal(k, C, m, 0.3), dtype) for k, m in ((3, 1.0), (4, 0.0)))
        _, mean, rstd, _, _ = ref.group_norm(x, G, weight, bias, 1e-5, None, u)
        mean, rstd = (ref.rounded(v, DT.F32) for v in (mean, rstd))
        r, bounds = ref.group_norm_backward(grad, x, mean, rstd, G, weight, bias, act, u)
        if act == "relu":
            z, _, _, z_bound, _ = ref.group_norm(x, G, weight, bias, 1e-5, None, u)
            near = np.abs(z) <= 2 * z_bound
            if near.any():  # a slope within rounding of the corner: its gradient is taken out
                grad = np.where(near, 0.0, grad)
                r, bounds = ref.group_norm_backward(grad, x, mean, rstd, G, weight, bias, act, u)
        (weight if which == "weight" else bias)[0] = value
        got = h.grad_group_norm(on_gpu(grad, dtype), on_gpu(x, dtype), on_gpu(mean, DT.F32), on_gpu(rstd, DT.F32), G,
                                on_gpu(weight, dtype), on_gpu(bias, dtype), act)
        W = C // G
        for t, name in zip(got, ("d_x", "d_weight", "d_bias")):
            v, want, bound = (a[..., W:] for a in (values(t), r[name], np.broadcast_to(bounds[name], r[name].shape)))
            ref.assert_within(v, want, bound, dtype, f"{name} of the other groups")


@pytest.mark.parametrize("N, S, C, G", SIZES)
def test_equal_elements_far_out(N, S, C, G):
    """Every element 2^122 and rstd 2^8: hat is zero, though mean * rstd is past F32's range."""
    grad = ref.rounded(normal(2, N * S * C, 0.2).reshape(N, S, C), DT.F32)
    x, mean, rstd = (on_gpu(np.full(s, v), DT.F32) for s, v in (((N, S, C), 2.0 ** 122), ((N, G), 2.0 ** 122), ((N, G), 2.0 ** 8)))
    one, zero = (on_gpu(np.full(C, v), DT.F32) for v in (1.0, 0.0))
    d_x, d_weight, d_bias = (values(t) for t in h.grad_group_norm(on_gpu(grad, DT.F32), x, mean, rstd, G, one, zero, None))
    r, bounds = ref.group_norm_backward(grad, np.zeros((N, S, C)), np.zeros((N, G)), np.full((N, G), 2.0 ** 8), G, None, None, None,
                                        ref.COMPUTE[DT.F32])
    ref.assert_within(d_x, r["d_x"], bounds["d_x"], DT.F32, "d_x")
    ref.assert_within(d_bias, r["d_bias"], bounds["d_bias"], DT.F32, "d_bias")
    assert (d_weight == 0).all()


@pytest.mark.parametrize("N, S, C, G", SIZES)
def test_rows_that_are_not_there_add_nothing(N, S, C, G):
    """With a weight of infinity and relu the channel's own gradients are finite: those of the positive elements' half. Rows
    past the last one, whose elements would be zeros, are in no sum."""
    dtype, u = DT.F32, ref.COMPUTE[DT.F32]
    x, grad = (ref.rounded(normal(k, N * S * C, 0.2).reshape(N, S, C), dtype) for k in (11, 12))
    weight, bias = np.ones(C), np.zeros(C)
    weight[0] = np.inf
    _, mean, rstd, _, _ = ref.group_norm(x, G, None, None, 1e-5, None, u)
    mean, rstd = (ref.rounded(v, DT.F32) for v in (mean, rstd))
    _, d_weight, d_bias = h.grad_group_norm(on_gpu(grad, dtype), on_gpu(x, dtype), on_gpu(mean, DT.F32), on_gpu(rstd, DT.F32), G,
                                            on_gpu(weight, dtype), on_gpu(bias, dtype), "relu")
    hat = (x[..., 0] - mean[:, :1]) * rstd[:, :1]
    d = np.where(hat > 0, grad[..., 0], 0)
    ref.assert_within(values(d_bias)[0], d.sum(), 64 * u * np.abs(d).sum(), dtype, "d_bias")
    ref.assert_within(values(d_weight)[0], (d * hat).sum(), 70 * u * (np.abs(d * hat).sum() + np.abs(d * mean[:, :1] * rstd[:, :1]).sum()), dtype,
                      "d_weight")
