"""Group normalisation with an activation and its backward pass on the GPU against 64-bit formulas."""
import numpy as np
import pytest

from tests import nn_reference as ref
from tests.support import DT, FLOATS, GPU, array, from_f64, h, normal, tensor, to_f64

pytestmark = pytest.mark.gpu
ACTIVATIONS = [None, "relu", "silu", "gelu", "gelu_tanh"]
WIDE = {DT.F16: DT.F32, DT.BF16: DT.F32, DT.F32: DT.F32, DT.F64: DT.F64}


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


class Case:
    def __init__(self, dtype, N, S, C, G, act, seed, mean=0.3, weights=None, affine=True):
        self.dtype, self.G, self.act, self.u, self.eps = dtype, G, act, ref.COMPUTE[dtype], 1e-5
        self.w_dtype = weights or dtype
        self.x = ref.rounded(normal(seed, N * S * C, mean, 1.0).reshape(N, S, C), dtype)
        self.weight = ref.rounded(normal(seed + 1, C, 1.0, 0.3), self.w_dtype) if affine else None
        self.bias = ref.rounded(normal(seed + 2, C, 0.0, 0.3), self.w_dtype) if affine else None
        self.grad = ref.rounded(normal(seed + 3, N * S * C).reshape(N, S, C), dtype)

    def vectors(self):
        return (None, None) if self.weight is None else (on_gpu(self.weight, self.w_dtype), on_gpu(self.bias, self.w_dtype))

    def check(self, laid=None):
        laid = laid or (lambda v: on_gpu(v, self.dtype))
        w, b = self.vectors()
        x = laid(self.x)
        out, mean, rstd = h.group_norm(x, self.G, w, b, self.eps, self.act)
        want, want_mean, want_rstd, bound, rel = ref.group_norm(self.x, self.G, self.weight, self.bias, self.eps, self.act, self.u)
        centred = np.abs(self.x).mean()
        ref.assert_within(values(mean), want_mean, ref.fold(self.x[0].size // self.G) * (np.abs(want_mean) + centred), mean.dtype, "mean")
        ref.assert_within(values(rstd), want_rstd, rel * want_rstd, rstd.dtype, "rstd")
        ref.assert_within(values(out), want, bound, self.dtype, "out")
        d_x, d_weight, d_bias = h.grad_group_norm(laid(self.grad), x, mean, rstd, self.G, w, b, self.act)
        if self.act == "relu":  # no input of these seeds sits within its own rounding of the corner
            z, _, _, z_bound, _ = ref.group_norm(self.x, self.G, self.weight, self.bias, self.eps, None, self.u)
            assert (np.abs(z) > z_bound).all()
        r, bounds = ref.group_norm_backward(self.grad, self.x, values(mean), values(rstd), self.G, self.weight, self.bias, self.act, self.u)
        ref.assert_within(values(d_x), r["d_x"], bounds["d_x"], self.dtype, "d_x")
        if self.weight is not None:
            ref.assert_within(values(d_weight), r["d_weight"], bounds["d_weight"], self.w_dtype, "d_weight")
            ref.assert_within(values(d_bias), r["d_bias"], bounds["d_bias"], self.w_dtype, "d_bias")
        else:
            assert d_weight is None and d_bias is None


SIZES = [(1, 1, 1, 1), (3, 1, 8, 2), (700, 1, 512, 4), (37, 1, 96, 6), (5, 1, 130, 13), (9, 1, 4096, 1), (3, 1, 40960, 2), (2, 7, 24, 4),
         (4, 60, 20, 4), (2, 300, 10, 1), (3, 1100, 40, 4), (1, 5000, 36, 3), (2, 257, 640, 32), (70, 3, 33, 33), (1, 70000, 3, 3)]


@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("N, S, C, G", SIZES)
def test_sizes(N, S, C, G, dtype):
    Case(dtype, N, S, C, G, "silu", seed=N + S + C).check()


@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("N, S, C, G", [(50, 1, 64, 4), (2, 400, 24, 2)])
def test_activations(N, S, C, G, act, dtype):
    Case(dtype, N, S, C, G, act, seed=7).check()


@pytest.mark.parametrize("N, S, C, G", [(50, 1, 64, 4), (2, 400, 24, 2)])
def test_weights_of_another_type_or_none(N, S, C, G):
    for dtype in (DT.F16, DT.BF16):
        Case(dtype, N, S, C, G, "gelu", 17, weights=DT.F32).check()
    for dtype in FLOATS:
        Case(dtype, N, S, C, G, "silu", 19, affine=False).check()


@pytest.mark.parametrize("layout", ["channels first", "a slice", "every other channel", "positions backwards in memory", "odd start"])
@pytest.mark.parametrize("N, S, C, G", [(40, 1, 24, 3), (3, 130, 24, 3), (2, 700, 24, 3)])
def test_strided_maps(N, S, C, G, layout):
    for dtype in (DT.BF16, DT.F32):
        c = Case(dtype, N, S, C, G, "silu", 23)

        def laid(v):
            if layout == "channels first":
                return on_gpu(np.ascontiguousarray(v.transpose(0, 2, 1)), dtype).permute([0, 2, 1])
            if layout == "a slice":
                return on_gpu(np.concatenate([v, np.full_like(v, np.nan)], 2), dtype).narrow(2, 0, C)
            if layout == "odd start":
                return on_gpu(np.concatenate([np.full((N, S, 1), np.nan), v], 2), dtype).narrow(2, 1, C)
            if layout == "every other channel":
                return on_gpu(np.repeat(v, 2, axis=2), dtype).slice(2, 0, None, 2)
            return on_gpu(np.ascontiguousarray(v.transpose(1, 0, 2)), dtype).permute([1, 0, 2])

        c.check(laid)


@pytest.mark.parametrize("N, S, C, G", [(20, 1, 64, 4), (2, 500, 24, 2), (1, 20000, 8, 2)])
def test_a_mean_far_from_zero_and_an_outlying_first_element(N, S, C, G):
    """The variance does not suffer from the mean's size: f64 accumulation (F32), or centred (F64)."""
    for dtype, far in ((DT.F32, 3000.0), (DT.F64, 1e6)):
        c = Case(dtype, N, S, C, G, None, 29, mean=far, affine=False)
        out, mean, rstd = h.group_norm(on_gpu(c.x, dtype), G)
        want, want_mean, want_rstd, bound, _ = ref.group_norm(c.x, G, None, None, 1e-5, None, c.u)
        # The deviations from the mean are exact to a step of the mean's own error (2^-50 of it).
        off = 2.0 ** -50 * far
        ref.assert_within(values(rstd), want_rstd, (8 * c.u + 4 * off) * want_rstd, dtype, "rstd")
        ref.assert_within(values(out), want, bound + 4 * c.u * np.abs(want) + 4 * off, dtype, "out")
        c.x[:, 0, 0] = 1e4 * far
        out, mean, rstd = h.group_norm(on_gpu(ref.rounded(c.x, dtype), dtype), G)
        _, _, want_rstd, _, _ = ref.group_norm(ref.rounded(c.x, dtype), G, None, None, 1e-5, None, c.u)
        ref.assert_within(values(rstd), want_rstd, 16 * c.u * want_rstd, dtype, "rstd with an outlier")


@pytest.mark.parametrize("N, S, C, G", [(40, 1, 24, 3), (2, 700, 24, 3)])
def test_strided_weights(N, S, C, G):
    c = Case(DT.BF16, N, S, C, G, "silu", 27)
    vectors = c.vectors
    c.vectors = lambda: tuple(on_gpu(np.repeat(v, 2), DT.BF16).slice(0, 0, None, 2) for v in (c.weight, c.bias))
    c.check()
    c.vectors = vectors


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("N, S, C, G", [(40, 1, 24, 3), (2, 700, 24, 3)])
def test_activations_far_out(N, S, C, G, act):
    """Where the activation is z or zero and its slope one or zero, however large z is (its square is past F32's range)."""
    c = Case(DT.F32, N, S, C, G, act, 25)
    c.bias = np.where(np.arange(C) % 2 == 0, 1e25, -1e25)
    w, b = c.vectors()
    x = on_gpu(c.x, DT.F32)
    out, mean, rstd = h.group_norm(x, G, w, b, c.eps, act)
    z = np.broadcast_to(c.bias if act is None else np.maximum(c.bias, 0), c.x.shape)
    assert (values(out) == np.float32(z)).all()  # |hat * weight| is less than half a step of 1e25
    grads = h.grad_group_norm(on_gpu(c.grad, DT.F32), x, mean, rstd, G, w, b, act)
    # The gradient of such an activation is that of none, with the zeroed channels' gradients gone.
    grad = c.grad if act is None else np.where(c.bias > 0, c.grad, 0)
    r, bounds = ref.group_norm_backward(grad, c.x, values(mean), values(rstd), G, c.weight, c.bias, None, c.u)
    for got, name in zip(grads, ("d_x", "d_weight", "d_bias")):
        ref.assert_within(values(got), r[name], bounds[name], DT.F32, name)


@pytest.mark.parametrize("dtype", [DT.F32, DT.F64], ids=lambda d: d.name)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("S", [1, 80])
def test_activations_over_their_range(S, act, dtype):
    """A weight of zero makes z the bias itself: the activation and its slope, S times over, from -12 to 12."""
    C, u = 2400, ref.COMPUTE[dtype]
    z = ref.rounded(np.linspace(-12, 12, C), dtype)
    w, b = on_gpu(np.zeros(C), dtype), on_gpu(z, dtype)
    x, ones = on_gpu(normal(28, S * C).reshape(1, S, C), dtype), on_gpu(np.ones((1, S, C)), dtype)
    out, mean, rstd = h.group_norm(x, 1, w, b, 1e-5, act)
    y, slope, rel = ref.activate(z, act)
    ref.assert_within(values(out), np.broadcast_to(y, (1, S, C)), np.broadcast_to((rel + 4) * u * np.abs(y), (1, S, C)), dtype, "out")
    d_x, _, d_bias = h.grad_group_norm(ones, x, mean, rstd, 1, w, b, act)
    assert (values(d_x) == 0).all()
    ref.assert_within(values(d_bias), S * slope, S * (rel * u * (1 + np.abs(z)) + 64 * u * np.abs(slope)), dtype, "d_bias")


def test_many_groups_of_one_channel_are_maps_too():
    c = Case(DT.BF16, 1, 70, 4100, 4100, "silu", 26)
    c.check()
    Case(DT.F32, 2, 130, 2050, 1025, None, 27).check()


def test_equal_elements_and_nan():
    x = np.full((3, 4, 16), 2.5)
    x[1, 2, 5] = np.nan
    x[2, 1, 9] = np.inf
    out, mean, rstd = (values(t) for t in h.group_norm(on_gpu(x, DT.F32), 2, None, None, 1e-3))
    assert not out[0].any() and (mean[0] == 2.5).all() and np.allclose(rstd[0], 1e-3 ** -0.5, rtol=1e-6)
    assert np.isnan(out[1, :, :8]).all() and not out[1, :, 8:].any()
    assert not out[2, :, :8].any() and np.isnan(out[2, 1, 9])


def test_empty_maps():
    out, mean, rstd = h.group_norm(on_gpu(np.zeros((2, 0, 8)), DT.BF16), 4)
    assert out.shape == [2, 0, 8] and np.isnan(values(mean)).all() and np.isnan(values(rstd)).all()
    w = on_gpu(np.ones(8), DT.BF16)
    d_x, d_w, d_b = h.grad_group_norm(on_gpu(np.zeros((2, 0, 8)), DT.BF16), on_gpu(np.zeros((2, 0, 8)), DT.BF16), mean, rstd, 4, w, w)
    assert d_x.shape == [2, 0, 8] and not values(d_w).any() and not values(d_b).any()
    out, mean, rstd = h.group_norm(on_gpu(np.zeros((0, 3, 8)), DT.BF16), 4)
    assert out.shape == [0, 3, 8] and mean.shape == [0, 4]
    d_x, d_w, d_b = h.grad_group_norm(out, out, mean, rstd, 4, w, w)
    assert not values(d_w).any() and not values(d_b).any()


def test_two_dimensions_are_tokens_and_four_are_maps():
    x = normal(1, 6 * 5 * 4 * 8).reshape(6, 5, 4, 8)
    whole = values(h.group_norm(on_gpu(x, DT.F64), 2)[0])
    assert np.array_equal(whole.reshape(6, 20, 8), values(h.group_norm(on_gpu(x.reshape(6, 20, 8), DT.F64), 2)[0]))
    tokens = values(h.group_norm(on_gpu(x.reshape(120, 8), DT.F64), 2)[0])
    assert np.array_equal(tokens.reshape(120, 1, 8), values(h.group_norm(on_gpu(x.reshape(120, 1, 8), DT.F64), 2)[0]))


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("N, S, C, G", [(6, 1, 12, 3), (2, 40, 12, 3)])
def test_gradients_against_differences(N, S, C, G, act):
    """In F64, central differences along random directions: off by e^2 times a third derivative (below 1e5 here: rstd is
    of order one) and the loss's rounding over e."""
    e = 1e-5
    c = Case(DT.F64, N, S, C, G, act, 31)
    if act == "relu":  # away from its corner
        z = ref.group_norm(c.x, G, c.weight, c.bias, c.eps, None, c.u)[0]
        c.grad[np.abs(z) < 1e-3] = 0.0

    def loss(x, w, b):
        return float((values(h.group_norm(on_gpu(x, DT.F64), G, on_gpu(w, DT.F64), on_gpu(b, DT.F64), c.eps, act)[0]) * c.grad).sum())

    x, (w, b) = on_gpu(c.x, DT.F64), c.vectors()
    _, mean, rstd = h.group_norm(x, G, w, b, c.eps, act)
    got = [values(t) for t in h.grad_group_norm(on_gpu(c.grad, DT.F64), x, mean, rstd, G, w, b, act)]
    at = [c.x, c.weight, c.bias]
    for k in range(3):
        v = normal(50 + k, at[k].size).reshape(at[k].shape)
        plus, minus = ([a + s * e * v if i == k else a for i, a in enumerate(at)] for s in (1, -1))
        assert abs((loss(*plus) - loss(*minus)) / (2 * e) - (got[k] * v).sum()) < e * e * 1e5 + 1e-12 * np.abs(c.grad).sum() / e * 1e-1


def test_runs_repeat_bit_for_bit():
    for N, S, C, G in ((3000, 1, 512, 8), (2, 9000, 40, 4)):
        c = Case(DT.BF16, N, S, C, G, "silu", 41)
        x, g, (w, b) = on_gpu(c.x, DT.BF16), on_gpu(c.grad, DT.BF16), c.vectors()

        def both():
            out, mean, rstd = h.group_norm(x, G, w, b, 1e-5, "silu")
            return [array(t) for t in (out, mean, rstd, *h.grad_group_norm(g, x, mean, rstd, G, w, b, "silu"))]

        first = both()
        for _ in range(4):
            assert all(np.array_equal(p, q) for p, q in zip(first, both()))


def test_the_front_end_refuses():
    x = on_gpu(np.zeros((2, 3, 8)), DT.BF16)
    for text, call in (("multiple of the number of groups", lambda: h.group_norm(x, 3)),
                       ("unknown activation", lambda: h.group_norm(x, 2, activation="tanh")),
                       ("weight of shape", lambda: h.group_norm(x, 2, on_gpu(np.ones(7), DT.BF16))),
                       ("weight to be", lambda: h.group_norm(x, 2, on_gpu(np.ones(8), DT.F16))),
                       ("eps", lambda: h.group_norm(x, 2, None, None, -1.0)),
                       ("two dimensions", lambda: h.group_norm(on_gpu(np.zeros(8), DT.BF16), 2))):
        with pytest.raises(Exception, match=text):
            call()
