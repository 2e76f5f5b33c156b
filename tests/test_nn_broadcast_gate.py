"""The gradient of a gate that is shared: summed from what the computation type holds, rounded once."""
from ctypes import byref, c_int64

import numpy as np
import pytest

from homura_amd import capi
from tests import nn_reference as ref
from tests.support import DT, FLOATS, GPU, array, from_f64, h, normal, tensor, to_f64, uniform

pytestmark = pytest.mark.gpu


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("B, T, H, D, shape", [(2, 140, 3, 16, "a head"), (3, 6, 2, 40, "a head"), (2, 300, 4, 24, "a step"), (2, 20, 3, 8, "a channel"),
                                               (4, 33, 2, 8, "all")])
def test_the_gradient_of_a_shared_gate(B, T, H, D, shape, dtype, is_sigmoid):
    u, full = ref.COMPUTE[dtype], (B, T, H, D)
    small = {"a head": (B, T, H, 1), "a step": (T, 1, 1), "a channel": (1, 1, H, D), "all": (1,)}[shape]
    n = int(np.prod(small))
    gate = ref.rounded((normal(1, n, 2.0) if is_sigmoid else uniform(1, n, 0.7, 1.0)).reshape(small), dtype)
    x, grad = (ref.rounded(normal(k, B * T * H * D).reshape(full), dtype) for k in (2, 3))
    flat = lambda v: np.broadcast_to(v, full).reshape(B, T, H * D)  # noqa: E731
    out, _ = h.linear_recurrence(on_gpu(gate, dtype), on_gpu(x, dtype), None, None, is_sigmoid)
    got = h.grad_linear_recurrence(on_gpu(grad, dtype), None, on_gpu(gate, dtype), on_gpu(x, dtype), out, None, None, is_sigmoid)
    want, bounds = ref.recurrence_backward(flat(grad), None, flat(gate), flat(x), values(out).reshape(B, T, H * D), None, None, is_sigmoid, u)
    over = tuple(k for k in range(4) if ((1,) * (4 - len(small)) + small)[k] != full[k])
    total = lambda v: v.reshape(full).sum(over, keepdims=True).reshape(small)  # noqa: E731
    # Each element's own error and its rounding to the computation type, the sum's rounding to that, and its additions (in 64
    # bits, as many as there are elements).
    each = bounds["d_gate"] + u * np.abs(want["d_gate"]) * (2 + B * T * H * D * 2.0 ** -53 / u)
    assert got[0].dtype == dtype and got[0].shape == list(small)
    ref.assert_within(values(got[0]), total(want["d_gate"]), total(each), dtype, "d_gate")
    ref.assert_within(values(got[1]).reshape(B, T, H * D), want["d_input"], bounds["d_input"], dtype, "d_input")


@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
@pytest.mark.parametrize("dtype, code", [(DT.F16, capi.F16), (DT.BF16, capi.BF16)], ids=["F16", "BF16"])
@pytest.mark.parametrize("B, T, C", [(3, 1, 40), (2, 12, 72), (2, 300, 33), (2, 700, 8), (1, 600, 259), (2, 150, 3)])
def test_a_gate_gradient_in_f32_beside_16_bits(B, T, C, dtype, code, is_sigmoid):
    """Also inside a wider tensor, whose other elements stay, and with lengths, behind which it is zero."""
    u, n = ref.COMPUTE[dtype], B * T * C
    gate = ref.rounded((normal(1, n, 2.0) if is_sigmoid else uniform(1, n, 0.7, 1.0)).reshape(B, T, C), dtype)
    x, grad = (ref.rounded(normal(k, n).reshape(B, T, C), dtype) for k in (2, 3))
    lengths = [T - b * T // 3 for b in range(B)]
    state = ref.rounded(ref.recurrence(gate, x, None, lengths, is_sigmoid, u)[0], dtype)
    want, bounds = ref.recurrence_backward(grad, None, gate, x, state, None, lengths, is_sigmoid, u)
    ctx = capi.Context(0)
    try:
        put = {k: ctx.upload(from_f64(v, dtype)) for k, v in (("gate", gate), ("x", x), ("state", state), ("grad", grad))}
        put["d_x"], put["lengths"] = ctx.malloc(2 * n), ctx.upload(np.array(lengths, dtype=np.int32))
        d = {k: capi.make_desc(b.ptr, code, (B, T, C), (T * C, C, 1)) for k, b in put.items()}
        d["lengths"] = capi.make_desc(put["lengths"].ptr, capi.I32, (B,), (1,))
        pitch = C + 5
        put["d_gate"] = ctx.upload(np.full(B * T * pitch, 77, np.float32))
        d["d_gate"] = capi.make_desc(put["d_gate"].ptr, capi.F32, (B, T, C), (T * pitch, pitch, 1), offset=3)
        d = {k: byref(v) for k, v in d.items()}
        need = c_int64(0)
        capi.check_nn(capi.nn.hmn_recurrence_workspace(d["gate"], byref(need)))
        room = ctx.malloc(max(need.value, 1))
        capi.check_nn(capi.nn.hmn_recurrence_backward(ctx.handle, int(is_sigmoid), d["d_gate"], d["d_x"], None, d["grad"], None, d["gate"],
                                                      d["x"], d["state"], None, d["lengths"], room.ptr, need.value))
        got = put["d_gate"].download(np.float32, B * T * pitch).reshape(B, T, pitch).astype(np.float64)
        assert (got[..., :3] == 77).all() and (got[..., C + 3:] == 77).all()
        ref.assert_within(got[..., 3:C + 3], want["d_gate"], bounds["d_gate"], DT.F32, "d_gate")
        ref.assert_within(to_f64(put["d_x"].download(np.uint16, n), dtype).reshape(B, T, C), want["d_input"], bounds["d_input"], dtype, "d_input")
    finally:
        ctx.close()
