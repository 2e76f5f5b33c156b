"""Statistics where they lose digits first: means many deviations from zero, and equal elements."""
import numpy as np
import pytest

from tests import nn_reference as ref
from tests.support import DT, GPU, array, from_f64, h, normal, tensor, to_f64

pytestmark = pytest.mark.gpu


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


# Rows in lanes of a wave with one to eight vectors each, in a workgroup, and maps.
SIZES = [(21, 1, 160, 4), (9, 1, 1024, 1), (5, 1, 2048, 1), (6, 1, 1500, 1), (3, 1, 4096, 1), (40, 3, 66, 3), (2, 500, 24, 2), (1, 20000, 8, 2), (3, 70, 2100, 1)]


@pytest.mark.parametrize("far", [2.0 ** 12, 2.0 ** 16, 2.0 ** 20])
@pytest.mark.parametrize("N, S, C, G", SIZES)
def test_means_of_many_deviations(N, S, C, G, far):
    """rstd comes from deviations about the mean, or about an element of the group: the sums are off by fold() of themselves
    and by a few 2^-53 (mean / deviation)^2 squared again, nothing next to F32's rounding."""
    x = ref.rounded(normal(29, N * S * C, far, 1.0).reshape(N, S, C), DT.F32)
    out, mean, rstd = h.group_norm(on_gpu(x, DT.F32), G)
    want, want_mean, want_rstd, bound, rel = ref.group_norm(x, G, None, None, 1e-5, None, ref.COMPUTE[DT.F32])
    ref.assert_within(values(mean), want_mean, ref.fold(S * C // G) * 2 * np.abs(want_mean), DT.F32, "mean")
    ref.assert_within(values(rstd), want_rstd, rel * want_rstd, DT.F32, "rstd")
    ref.assert_within(values(out), want, bound, DT.F32, "out")


@pytest.mark.parametrize("dtype, value", [(DT.F16, 60000.0), (DT.BF16, 1e6), (DT.F32, 1234567.0), (DT.F32, 3e12), (DT.F64, 1e9 / 7)])
@pytest.mark.parametrize("N, S, C, G", SIZES)
def test_equal_elements(N, S, C, G, dtype, value):
    """The variance is zero, whatever the elements are: rstd is 1 / sqrt(eps)."""
    x = ref.rounded(np.full((N, S, C), value), dtype)
    out, mean, rstd = h.group_norm(on_gpu(x, dtype), G, None, None, 1e-5)
    u = ref.COMPUTE[dtype]
    off = ref.fold(S * C // G) * value  # of the mean; its square joins eps
    ref.assert_within(values(mean), x[0, 0, 0] * np.ones((N, G)), off, mean.dtype, "mean")
    want = np.full((N, G), 1e-5 ** -0.5)
    ref.assert_within(values(rstd), want, (4 * u + off * off / 1e-5) * want, rstd.dtype, "rstd")
    assert (np.abs(values(out)) <= 2 * (off + u * off) * 1e-5 ** -0.5 + ref.SMALLEST[dtype] + ref.TINY).all()


def test_one_element_apart():
    """A group of equal F16 elements but one, a step away: mean / deviation is past 2^16."""
    for N, S, C, G in ((4, 1, 3000, 1), (4, 100, 1500, 3)):
        x = np.full((N, S, C), 60000.0)
        x[:, S // 2, C // 2] += 32.0
        x = ref.rounded(x, DT.F16)
        _, mean, rstd = h.group_norm(on_gpu(x, DT.F16), G)
        _, want_mean, want_rstd, _, rel = ref.group_norm(x, G, None, None, 1e-5, None, ref.COMPUTE[DT.F16])
        ref.assert_within(values(mean), want_mean, ref.fold(S * C // G) * 2 * np.abs(want_mean), DT.F32, "mean")
        ref.assert_within(values(rstd), want_rstd, rel * want_rstd, DT.F32, "rstd")
