"""The weights' gradients over many rows and positions."""
from ctypes import byref, c_int64

import numpy as np
import pytest

from homura_amd import capi
from tests import nn_reference as ref
from tests.support import DT, normal

pytestmark = pytest.mark.gpu


# (N, S, C, G): a lane of the widest kernels would meet 512 rows in the first, 2048 positions in the second.
@pytest.mark.parametrize("N, S, C, G", [(66576, 1, 2016, 32), (256, 2048, 257, 1)])
def test_sums_over_many_rows_and_positions(N, S, C, G):
    """Gradients that are the same everywhere: every addition of a running sum rounds to the same side, so a run of k additions
    in F32 is off by up to k half steps. Runs of 32 and a few joins are allowed. Only d_src is memory of that size: the
    operands are one row, repeated by strides of zero."""
    ctx = capi.Context(0)
    try:
        x, grad, weight = normal(5, C), normal(6, C, 0.5, 0.2), normal(7, C, 1.0, 0.2)
        x, grad, weight = (ref.rounded(v, DT.F32) for v in (x, grad, weight))
        put = {k: ctx.upload(v.astype(np.float32)) for k, v in (("x", x), ("grad", grad), ("weight", weight), ("mean", np.zeros(G)), ("rstd", np.ones(G)))}
        put["d_src"] = ctx.malloc(4 * N * S * C)
        put["d_weight"], put["d_bias"] = ctx.malloc(4 * C), ctx.malloc(4 * C)
        d = {k: capi.make_desc(put[k].ptr, capi.F32, (N, S, C), (0, 0, 1)) for k in ("x", "grad")}
        d["d_src"] = capi.make_desc(put["d_src"].ptr, capi.F32, (N, S, C), (S * C, C, 1))
        d.update({k: capi.make_desc(put[k].ptr, capi.F32, (N, G), (0, 1)) for k in ("mean", "rstd")})
        d.update({k: capi.make_desc(put[k].ptr, capi.F32, (C,), (1,)) for k in ("weight", "d_weight", "d_bias")})
        d = {k: byref(v) for k, v in d.items()}
        need = c_int64(0)
        capi.check_nn(capi.nn.hmn_group_norm_workspace(d["d_src"], G, 1, byref(need)))
        room = ctx.malloc(max(need.value, 1))
        capi.check_nn(capi.nn.hmn_group_norm_backward(ctx.handle, d["d_src"], d["d_weight"], d["d_bias"], d["grad"], d["x"], d["mean"], d["rstd"],
                                                      d["weight"], None, G, -1, room.ptr, need.value))
        u = ref.COMPUTE[DT.F32]
        d_bias, d_weight = N * S * grad, N * S * grad * x
        got = {k: put[k].download(np.float32, C).astype(np.float64) for k in ("d_weight", "d_bias")}
        ref.assert_within(got["d_bias"], d_bias, 40 * u * np.abs(d_bias), DT.F32, "d_bias")
        ref.assert_within(got["d_weight"], d_weight, 42 * u * np.abs(d_weight), DT.F32, "d_weight")
        # Every row's gradient is the same: the first and the last one, against the formula.
        by_group = lambda v: np.repeat(v.reshape(G, -1).mean(1), C // G)  # noqa: E731
        wd = weight * grad
        want = wd - by_group(wd) - x * by_group(wd * x)
        bound = 80 * u * (np.abs(wd) + by_group(np.abs(wd)) + np.abs(x) * by_group(np.abs(wd * x)))
        row = np.empty(C, np.float32)
        for n in (0, N * S - 1):
            capi.check(capi.lib.hmr_copy_to_host(ctx.handle, row.ctypes.data, put["d_src"].ptr + 4 * n * C, row.nbytes))
            ref.assert_within(row.astype(np.float64), want, bound, DT.F32, f"d_src of row {n}")
    finally:
        ctx.close()
