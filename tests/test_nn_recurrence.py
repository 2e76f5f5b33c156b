"""The gated linear recurrence and its backward pass on the GPU against a 64-bit evaluation step by step."""
import numpy as np
import pytest

from tests import nn_reference as ref
from tests.support import DT, FLOATS, GPU, array, from_f64, h, normal, tensor, to_f64, uniform

pytestmark = pytest.mark.gpu


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


def ints(lengths, dtype=DT.I32):
    return None if lengths is None else tensor(np.asarray(lengths, dtype=np.int32 if dtype == DT.I32 else np.int64), dtype, [len(lengths)], GPU)


class Case:
    def __init__(self, dtype, B, T, C, is_sigmoid, seed, lengths=None, initial=True, state=None):
        self.dtype, self.is_sigmoid, self.u, self.lengths = dtype, is_sigmoid, ref.COMPUTE[dtype], lengths
        n = B * T * C
        gate = normal(seed, n, 2.0, 2.0) if is_sigmoid else uniform(seed, n, 0.6, 1.0) * np.where(uniform(seed + 1, n) < 0.02, -1, 1)
        if not is_sigmoid:
            gate[uniform(seed + 2, n) < 0.01] = 0.0  # a channel that forgets
            gate[uniform(seed + 3, n) < 0.01] = 1.0
        self.gate = ref.rounded(gate.reshape(B, T, C), dtype)
        self.x = ref.rounded(normal(seed + 4, n).reshape(B, T, C), dtype)
        self.state = state or (DT.F64 if dtype == DT.F64 else DT.F32)
        self.initial = ref.rounded(normal(seed + 5, B * C).reshape(B, C), self.state) if initial else None
        self.seed = seed

    def gpu_initial(self):
        return None if self.initial is None else on_gpu(self.initial, self.state)

    def check_forward(self, gate=None, x=None):
        out, last = h.linear_recurrence(gate or on_gpu(self.gate, self.dtype), x or on_gpu(self.x, self.dtype), self.gpu_initial(),
                                        ints(self.lengths), self.is_sigmoid)
        want, want_last, bound, last_bound = ref.recurrence(self.gate, self.x, self.initial, self.lengths, self.is_sigmoid, self.u)
        ref.assert_within(values(out), want, bound, self.dtype, "out")
        ref.assert_within(values(last), want_last, last_bound, last.dtype, "last")
        return out, last

    def check_backward(self, g_last=True, g=True):
        B, T, C = self.x.shape
        state = ref.recurrence(self.gate, self.x, self.initial, self.lengths, self.is_sigmoid, self.u)[0]
        state = ref.rounded(state, self.dtype)
        grad = ref.rounded(normal(self.seed + 6, B * T * C).reshape(B, T, C), self.dtype) if g else None
        grad_last = ref.rounded(normal(self.seed + 7, B * C).reshape(B, C), self.state) if g_last else None
        got = h.grad_linear_recurrence(None if grad is None else on_gpu(grad, self.dtype),
                                       None if grad_last is None else on_gpu(grad_last, self.state),
                                       on_gpu(self.gate, self.dtype), on_gpu(self.x, self.dtype), on_gpu(state, self.dtype),
                                       self.gpu_initial(), ints(self.lengths, DT.I64), self.is_sigmoid)
        want, bounds = ref.recurrence_backward(np.zeros_like(self.x) if grad is None else grad, grad_last, self.gate, self.x, state,
                                               self.initial, self.lengths, self.is_sigmoid, self.u)
        for name, t in zip(("d_gate", "d_input", "d_initial"), got):
            ref.assert_within(values(t), want[name], bounds[name], t.dtype, name)


SIZES = [(1, 1, 1), (3, 1, 130), (64, 1, 256), (2, 2, 7), (5, 7, 8), (2, 31, 65), (1, 128, 64), (2, 129, 136), (1, 300, 1003), (3, 257, 3),
         (300, 33, 40), (1, 2500, 33), (2, 1200, 72)]


@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("B, T, C", SIZES)
def test_forward_and_backward(B, T, C, dtype, is_sigmoid):
    c = Case(dtype, B, T, C, is_sigmoid, seed=B * 1000 + T + C)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("B, T, C", [(3, 60, 9), (2, 511, 8), (2, 513, 16), (4, 1100, 3), (2, 1100, 33), (2, 530, 39), (1, 1500, 64), (2, 600, 127)])
def test_few_channels(B, T, C, dtype, is_sigmoid):
    c = Case(dtype, B, T, C, is_sigmoid, seed=B * 1000 + T + C)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("dtype", [DT.BF16, DT.F64], ids=lambda d: d.name)
@pytest.mark.parametrize("B, T, C", [(256, 9, 256), (256, 32, 256), (256, 33, 256), (255, 32, 256), (3, 8, 40), (3, 9, 40), (3, 32, 40)])
def test_few_steps(B, T, C, dtype):
    c = Case(dtype, B, T, C, True, seed=B * 1000 + T + C)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32], ids=lambda d: d.name)
@pytest.mark.parametrize("T, C", [(1, 24), (9, 24), (140, 72), (700, 19), (2100, 8)])
def test_a_padded_batch(T, C, dtype, is_sigmoid):
    """Lengths of zero, one, all of it, and beyond either end; what lies behind them (NaN here) is not looked at, and the
    output and the gradients there are zero."""
    lengths = [0, 1, T, T + 5, -3, T // 2, max(0, T - 1), min(T, 129)]
    c = Case(dtype, len(lengths), T, C, is_sigmoid, seed=T, lengths=lengths)
    c.check_backward()
    for b, n in enumerate(ref.steps_of(lengths, len(lengths), T)):
        c.gate[b, n:], c.x[b, n:] = np.nan, np.inf
    out, last = c.check_forward()
    for b, n in enumerate(ref.steps_of(lengths, len(lengths), T)):
        assert not values(out)[b, n:].any()
        if n == 0:
            assert np.array_equal(values(last)[b], c.initial[b])


def test_the_gradient_behind_a_length_is_not_read():
    B, T, C, lengths = 3, 200, 40, [150, 0, 200]
    c = Case(DT.F32, B, T, C, False, 5, lengths=lengths)
    grad = normal(1, B * T * C).reshape(B, T, C)
    results = []
    for junk in (0.0, np.nan):
        for b, n in enumerate(lengths):
            grad[b, n:] = junk
        results.append([values(t) for t in h.grad_linear_recurrence(on_gpu(grad, DT.F32), None, on_gpu(c.gate, DT.F32), on_gpu(c.x, DT.F32),
                                                                    on_gpu(c.x, DT.F32), None, ints(lengths), False)])
    for a, b in zip(*results):
        assert np.array_equal(a, b) and np.isfinite(b).all()


@pytest.mark.parametrize("dtype", [DT.F16, DT.BF16], ids=lambda d: d.name)
def test_states_of_the_sequences_own_type(dtype):
    c = Case(dtype, 3, 150, 72, True, 11, state=dtype)
    out, last = c.check_forward()
    assert last.dtype == dtype
    c.check_backward()


def test_without_an_initial_state_or_one_of_the_gradients():
    c = Case(DT.F32, 2, 170, 40, False, 21, initial=False)
    c.check_forward()
    c.check_backward()
    c.check_backward(g_last=False)
    c.check_backward(g=False)


@pytest.mark.parametrize("T", [0, 1])
def test_no_steps_hand_the_state_over(T):
    x = np.zeros((2, T, 5))
    start = normal(3, 10).reshape(2, 5)
    out, last = h.linear_recurrence(on_gpu(x, DT.F64), on_gpu(x, DT.F64), on_gpu(start, DT.F64), ints([0, 0]))
    assert out.shape == [2, T, 5] and np.array_equal(values(last), start) and not values(out).any()
    d_gate, d_input, d_initial = h.grad_linear_recurrence(None, on_gpu(start, DT.F64), on_gpu(x, DT.F64), on_gpu(x, DT.F64), on_gpu(x, DT.F64),
                                                          None, ints([0, 0]))
    assert np.array_equal(values(d_initial), start) and not values(d_gate).any() and not values(d_input).any()


@pytest.mark.parametrize("shape", [(0, 4, 5), (3, 4, 0)])
def test_empty_batches(shape):
    x = np.zeros(shape)
    out, last = h.linear_recurrence(on_gpu(x, DT.BF16), on_gpu(x, DT.BF16))
    assert out.shape == list(shape) and last.shape == [shape[0], shape[2]]


def test_decoding_one_step_at_a_time_is_the_whole_sequence():
    """The state in f32 handed from call to call: the same sums, grouped otherwise."""
    c = Case(DT.BF16, 4, 40, 136, True, 31)
    whole, last = c.check_forward()
    state = c.gpu_initial()
    gate, x = on_gpu(c.gate, DT.BF16), on_gpu(c.x, DT.BF16)
    want, _, bound, _ = ref.recurrence(c.gate, c.x, c.initial, None, True, c.u)
    for t in range(40):
        out, state = h.linear_recurrence(gate.narrow(1, t, 1), x.narrow(1, t, 1), state, None, True)
        ref.assert_within(values(out), want[:, t:t + 1], bound[:, t:t + 1], DT.BF16, f"step {t}")


@pytest.mark.parametrize("layout", ["time last", "time first", "every other channel", "one buffer", "odd start"])
@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32], ids=lambda d: d.name)
def test_strided_sequences(layout, dtype):
    B, T, C = 3, 150, 41
    c = Case(dtype, B, T, C, True, 41)

    def laid(v):
        if layout == "time last":
            return on_gpu(np.ascontiguousarray(v.transpose(0, 2, 1)), dtype).permute([0, 2, 1])
        if layout == "time first":
            return on_gpu(np.ascontiguousarray(v.transpose(1, 0, 2)), dtype).permute([1, 0, 2])
        if layout == "every other channel":
            return on_gpu(np.repeat(v, 2, axis=2), dtype).slice(2, 0, None, 2)
        if layout == "odd start":
            return on_gpu(np.concatenate([np.zeros((B, T, 1)), v], 2), dtype).narrow(2, 1, C)
        return on_gpu(np.concatenate([v, np.full_like(v, np.nan)], 2), dtype).narrow(2, 0, C)

    c.check_forward(laid(c.gate), laid(c.x))
    state = ref.rounded(ref.recurrence(c.gate, c.x, c.initial, None, True, c.u)[0], dtype)
    grad = ref.rounded(normal(9, c.x.size).reshape(c.x.shape), dtype)
    got = h.grad_linear_recurrence(laid(grad), None, laid(c.gate), laid(c.x), laid(state), c.gpu_initial(), None, True)
    want, bounds = ref.recurrence_backward(grad, None, c.gate, c.x, state, c.initial, None, True, c.u)
    for name, t in zip(("d_gate", "d_input", "d_initial"), got):
        ref.assert_within(values(t), want[name], bounds[name], t.dtype, name)


def test_steps_far_apart():
    """Steps 3 million elements from each other, further than a scan's tile addresses."""
    B, T, C, step = 2, 9, 40, 3_000_000
    c = Case(DT.F32, B, T, C, True, 45)

    def laid(v):
        wide = np.zeros((T, step), np.float32)
        wide[:, :B * C] = v.transpose(1, 0, 2).reshape(T, B * C)
        return tensor(wide, DT.F32, [T, step], GPU).narrow(1, 0, B * C).as_strided([B, T, C], [C, step, 1], 0)

    c.check_forward(laid(c.gate), laid(c.x))
    state = ref.rounded(ref.recurrence(c.gate, c.x, c.initial, None, True, c.u)[0], DT.F32)
    grad = ref.rounded(normal(9, c.x.size).reshape(c.x.shape), DT.F32)
    got = h.grad_linear_recurrence(laid(grad), None, laid(c.gate), laid(c.x), laid(state), c.gpu_initial(), None, True)
    want, bounds = ref.recurrence_backward(grad, None, c.gate, c.x, state, c.initial, None, True, c.u)
    for name, t in zip(("d_gate", "d_input", "d_initial"), got):
        ref.assert_within(values(t), want[name], bounds[name], t.dtype, name)


@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32], ids=lambda d: d.name)
def test_a_gate_shared_by_a_head(dtype):
    """One gate per head, broadcast over its channels: its gradient is the sum over them."""
    B, T, H, D = 2, 140, 3, 16
    c = Case(dtype, B, T, H, False, 51)
    x = ref.rounded(normal(1, B * T * H * D).reshape(B, T, H, D), dtype)
    wide = np.repeat(c.gate, D, axis=2)
    out, last = h.linear_recurrence(on_gpu(c.gate[..., None], dtype), on_gpu(x, dtype))
    want, want_last, bound, last_bound = ref.recurrence(wide, x.reshape(B, T, H * D), None, None, False, c.u)
    ref.assert_within(values(out).reshape(B, T, H * D), want, bound, dtype, "out")
    assert last.shape == [B, H, D]
    grad = ref.rounded(normal(2, x.size).reshape(x.shape), dtype)
    d_gate, d_input, _ = h.grad_linear_recurrence(on_gpu(grad, dtype), None, on_gpu(c.gate[..., None], dtype), on_gpu(x, dtype), out)
    state = values(out).reshape(B, T, H * D)
    r, bounds = ref.recurrence_backward(grad.reshape(state.shape), None, wide, None, state, None, None, False, c.u)
    each = bounds["d_gate"] + ref.HALF_STEP[dtype] * np.abs(r["d_gate"])  # rounded element by element, then summed in f64
    assert d_gate.shape == [B, T, H, 1]
    ref.assert_within(values(d_gate)[..., 0], r["d_gate"].reshape(B, T, H, D).sum(3), each.reshape(B, T, H, D).sum(3), dtype, "d_gate")


@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
def test_gradients_against_differences(is_sigmoid):
    """In F64: the loss's central differences along random directions. A difference over 2 e is off by e^2 / 6 times a
    third derivative (the loss is a polynomial of degree at most T in the gates, with derivatives below 1e4 here) and by
    the loss's rounding over e."""
    B, T, C, e = 2, 37, 5, 1e-5
    c = Case(DT.F64, B, T, C, is_sigmoid, 61)
    grad, grad_last = normal(1, B * T * C).reshape(B, T, C), normal(2, B * C).reshape(B, C)

    def loss(gate, x, initial):
        out, last = h.linear_recurrence(on_gpu(gate, DT.F64), on_gpu(x, DT.F64), on_gpu(initial, DT.F64), None, is_sigmoid)
        return float((values(out) * grad).sum() + (values(last) * grad_last).sum())

    out, _ = h.linear_recurrence(on_gpu(c.gate, DT.F64), on_gpu(c.x, DT.F64), c.gpu_initial(), None, is_sigmoid)
    got = [values(t) for t in h.grad_linear_recurrence(on_gpu(grad, DT.F64), on_gpu(grad_last, DT.F64), on_gpu(c.gate, DT.F64),
                                                       on_gpu(c.x, DT.F64), out, c.gpu_initial(), None, is_sigmoid)]
    at = [c.gate, c.x, c.initial]
    for k in range(3):
        for trial in range(3):
            v = normal(100 + 10 * k + trial, at[k].size).reshape(at[k].shape)
            plus, minus = ([a + s * e * v if i == k else a for i, a in enumerate(at)] for s in (1, -1))
            assert abs((loss(*plus) - loss(*minus)) / (2 * e) - (got[k] * v).sum()) < e * e * 1e4 + 1e-13 * np.abs(got[k] * v).sum() / e + 1e-7


@pytest.mark.parametrize("T", [1, 3, 40, 700])
@pytest.mark.parametrize("C", [40, 259, 515, 1027])
def test_a_state_read_and_written_in_one_place(T, C):
    """last is initial, d_initial is grad_last: also where the number of channels leaves the last block of a scan a few,
    less than a vector."""
    from ctypes import byref, c_int64

    from homura_amd import capi
    B = 3
    c = Case(DT.BF16, B, T, C, True, 91)
    state = ref.rounded(ref.recurrence(c.gate, c.x, c.initial, None, True, c.u)[0], DT.BF16)
    grad = ref.rounded(normal(6, B * T * C).reshape(B, T, C), DT.BF16)
    grad_last = ref.rounded(normal(7, B * C).reshape(B, C), DT.F32)
    want = ref.recurrence(c.gate, c.x, c.initial, None, True, c.u)
    back, bounds = ref.recurrence_backward(grad, grad_last, c.gate, c.x, state, c.initial, None, True, c.u)
    ctx = capi.Context(0)
    try:
        put = {k: ctx.upload(from_f64(v, DT.BF16)) for k, v in (("gate", c.gate), ("x", c.x), ("state", state), ("grad", grad))}
        put.update({k: ctx.malloc(2 * B * T * C) for k in ("out", "d_gate", "d_x")})
        put["at"], put["g"], put["from"] = (ctx.upload(v.astype(np.float32)) for v in (c.initial, grad_last, c.initial))
        d = {k: byref(capi.make_desc(b.ptr, capi.BF16, (B, T, C), (T * C, C, 1))) for k, b in put.items()}
        d.update({k: byref(capi.make_desc(put[k].ptr, capi.F32, (B, C), (C, 1))) for k in ("at", "g", "from")})
        need = c_int64(0)
        capi.check_nn(capi.nn.hmn_recurrence_workspace(d["x"], byref(need)))
        room = ctx.malloc(need.value)
        capi.check_nn(capi.nn.hmn_recurrence(ctx.handle, 1, d["out"], d["at"], d["gate"], d["x"], d["at"], None, room.ptr, need.value))
        capi.check_nn(capi.nn.hmn_recurrence_backward(ctx.handle, 1, d["d_gate"], d["d_x"], d["g"], d["grad"], d["g"], d["gate"], d["x"],
                                                      d["state"], d["from"], None, room.ptr, need.value))
        ref.assert_within(to_f64(put["out"].download(np.uint16, B * T * C), DT.BF16).reshape(B, T, C), want[0], want[2], DT.BF16, "out")
        ref.assert_within(put["at"].download(np.float32, B * C).reshape(B, C), want[1], want[3], DT.F32, "last")
        ref.assert_within(put["g"].download(np.float32, B * C).reshape(B, C), back["d_initial"], bounds["d_initial"], DT.F32, "d_initial")
        for k, name in (("d_gate", "d_gate"), ("d_x", "d_input")):
            got = to_f64(put[k].download(np.uint16, B * T * C), DT.BF16).reshape(B, T, C)
            ref.assert_within(got, back[name], bounds[name], DT.BF16, name)
    finally:
        ctx.close()


@pytest.mark.parametrize("T", [5, 33])
def test_more_sequences_than_a_launch_has_workgroups(T):
    """2^23 of them, a workgroup of 512 threads each, would be a launch of 2^32 threads."""
    B = 1 << 23
    gate, x = (tensor(np.full(B * T, bits, dtype=np.uint16), DT.BF16, [B, T, 1], GPU) for bits in (0x3F00, 0x3F80))  # 0.5, 1
    out, last = h.linear_recurrence(gate, x)
    want = 2 - 2.0 ** -np.arange(T)
    assert (array(out).reshape(B, T) == from_f64(want, DT.BF16)).all()
    assert (array(last) == want[-1].astype(np.float32)).all()


def test_infinities_and_nan_stay_in_their_channel():
    B, T, C = 1, 300, 16
    c = Case(DT.F32, B, T, C, False, 71)
    c.x[0, 10, 3], c.x[0, 140, 5] = np.nan, np.inf
    c.gate[0, 141:, 5] = 0.5
    c.gate[0, 200, 3] = 0.0  # 0 * NaN is NaN: a zero gate forgets only what is finite
    out, last = h.linear_recurrence(on_gpu(c.gate, DT.F32), on_gpu(c.x, DT.F32))
    out = values(out)
    assert np.isnan(out[0, 10:, 3]).all() and np.isfinite(out[0, :10, 3]).all()
    assert not np.isfinite(out[0, 140:, 5]).any() and np.isfinite(out[0, :140, 5]).all()
    rest = [k for k in range(C) if k not in (3, 5)]
    want, _, bound, _ = ref.recurrence(c.gate[..., rest], c.x[..., rest], None, None, False, c.u)
    ref.assert_within(out[..., rest], want, bound, DT.F32, "the other channels")


@pytest.mark.parametrize("gate", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T", [2, 16, 90, 700])
def test_a_factor_that_is_not_finite_spoils_a_zero_state(T, gate):
    """0 * inf and 0 * NaN are NaN, and NaN stays: whether the state is zero at the start or at a later step."""
    for at in sorted({0, 1, T // 2, T - 1}):
        c = Case(DT.F32, 2, T, 8, False, 72)
        c.x[0, :at + 1, 2] = 0.0
        c.gate[0, at, 2] = gate
        out, last = (values(t) for t in h.linear_recurrence(on_gpu(c.gate, DT.F32), on_gpu(c.x, DT.F32)))
        assert np.isnan(out[0, at:, 2]).all() and np.isnan(last[0, 2]) and (out[0, :at, 2] == 0).all()
        out[0, :, 2] = 0
        assert np.isfinite(out).all()


def test_runs_repeat_bit_for_bit():
    for B, T, C in ((2, 3000, 64), (1, 5000, 13), (64, 200, 512)):
        c = Case(DT.BF16, B, T, C, True, 81)
        gate, x = on_gpu(c.gate, DT.BF16), on_gpu(c.x, DT.BF16)
        first = [array(t) for t in h.linear_recurrence(gate, x, None, None, True)]
        for _ in range(5):
            assert all(np.array_equal(a, array(b)) for a, b in zip(first, h.linear_recurrence(gate, x, None, None, True)))


@pytest.mark.parametrize("changes, text", [
    ({"gate": DT.F32}, "gate to be"), ({"lengths": [1]}, "lengths of shape"), ({"initial": (3, 4)}, "initial state of shape"),
])
def test_the_front_end_refuses(changes, text):
    x = on_gpu(np.zeros((2, 3, 4)), DT.BF16)
    gate = on_gpu(np.zeros((2, 3, 4)), changes.get("gate", DT.BF16))
    initial = on_gpu(np.zeros(changes["initial"]), DT.F32) if "initial" in changes else None
    with pytest.raises(Exception, match=text):
        h.linear_recurrence(gate, x, initial, ints(changes.get("lengths")))


def test_cpu_tensors_are_refused():
    x = tensor(np.zeros(24, dtype=np.float32), DT.F32, [2, 3, 4])
    with pytest.raises(Exception, match="ROCm tensors only"):
        h.linear_recurrence(x, x)
