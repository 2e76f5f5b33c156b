"""The operators as a recurrent block uses them - recurrence, group normalisation of the heads with silu, dropout onto the
residual, and back - and what holds for all of them: graphs, other contexts and threads, long offsets."""
import ctypes
import threading
from ctypes import byref, c_int64

import numpy as np
import pytest

from homura_amd import capi
from tests import nn_reference as ref
from tests.support import DT, GPU, array, from_f64, h, normal, tensor, to_f64

pytestmark = pytest.mark.gpu


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


def block(gate, x, w, b, residual, mask, G):
    state, last = h.linear_recurrence(gate, x, None, None, True)
    y, mean, rstd = h.group_norm(state.reshape([state.shape[0] * state.shape[1], state.shape[2]]), G, w, b, 1e-5, "silu")
    out = h.dropout_with(y.reshape(state.shape), mask, residual)
    return out, (state, y, mean, rstd)


def block_back(grad, gate, x, w, b, kept, mask, G):
    state, y, mean, rstd = kept
    d_y = h.grad_dropout(grad, mask)
    rows = [state.shape[0] * state.shape[1], state.shape[2]]
    d_state, d_w, d_b = h.grad_group_norm(d_y.reshape(rows), state.reshape(rows), mean, rstd, G, w, b, "silu")
    d_gate, d_x, _ = h.grad_linear_recurrence(d_state.reshape(state.shape), None, gate, x, state, None, None, True)
    return d_gate, d_x, d_w, d_b


B, T, C, G = 2, 300, 64, 4
MASK = (0.25, 42, 1000)


def inputs(dtype, seed=0):
    n = B * T * C
    return [on_gpu(v.reshape(s), dtype) for v, s in ((normal(seed + 1, n, 2.0), (B, T, C)), (normal(seed + 2, n), (B, T, C)),
                                                     (normal(seed + 3, C, 1.0, 0.2), (C,)), (normal(seed + 4, C, 0.0, 0.2), (C,)),
                                                     (normal(seed + 5, n), (B, T, C)), (normal(seed + 6, n), (B, T, C)))]


def test_a_block_forwards_and_backwards_against_differences():
    """In F64: the whole block's gradients along random directions, with dropout's mask held. Differences over 2 e are off
    by e^2 times a third derivative (below 1e6 for sums of this many terms) and the loss's rounding over e."""
    gate, x, w, b, residual, grad = inputs(DT.F64)
    g, e = values(grad), 1e-5

    def loss(at):
        return float((values(block(*(on_gpu(a, DT.F64) for a in at), residual, MASK, G)[0]) * g).sum())

    out, kept = block(gate, x, w, b, residual, MASK, G)
    got = [values(t) for t in block_back(grad, gate, x, w, b, kept, MASK, G)]
    at = [values(t) for t in (gate, x, w, b)]
    size = np.abs(values(out) * g).sum()
    for k in range(4):
        v = normal(60 + k, at[k].size).reshape(at[k].shape)
        plus, minus = ([a + s * e * v if i == k else a for i, a in enumerate(at)] for s in (1, -1))
        assert abs((loss(plus) - loss(minus)) / (2 * e) - (got[k] * v).sum()) < e * e * 1e6 + 2.0 ** -50 * size / e


@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32], ids=lambda d: d.name)
def test_a_block_against_64_bits(dtype):
    gate, x, w, b, residual, grad = inputs(dtype)
    out, (state, y, mean, rstd) = block(gate, x, w, b, residual, MASK, G)
    u = ref.COMPUTE[dtype]
    want, _, bound, _ = ref.recurrence(values(gate), values(x), None, None, True, u)
    ref.assert_within(values(state), want, bound, dtype, "the states")
    rows = values(state).reshape(B * T, 1, C)  # from here on, each stage from the one before it as it was rounded
    want, _, _, bound, _ = ref.group_norm(rows, G, values(w), values(b), 1e-5, "silu", u)
    ref.assert_within(values(y).reshape(rows.shape), want, bound, dtype, "the heads")
    want = ref.dropout(values(y).reshape(B, T, C), values(residual), *MASK, dtype)
    assert np.array_equal(values(out), want)


class Graph:
    """A capture of `queue()` on a context's stream."""

    def __init__(self, ctx, queue):
        self.hip = ctypes.CDLL("libamdhip64.so")
        self.stream = ctypes.c_void_p(ctx.stream())
        graph, self.executable = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0
        try:
            queue()
        finally:
            status = self.hip.hipStreamEndCapture(self.stream, byref(graph))
        assert status == 0 and graph.value
        assert self.hip.hipGraphInstantiate(byref(self.executable), graph, None, None, ctypes.c_size_t(0)) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.executable, self.stream) == 0


class Calls:
    """Every entry point over buffers of one context, sizes that need workspaces among them."""

    def __init__(self, ctx, seed, B=2, T=3000, C=48, G=3):
        self.ctx, self.shape, self.G = ctx, (B, T, C), G
        n = B * T * C
        self.buffers, self.descs = {}, {}

        def put(name, data, dtype, *sizes):
            strides = np.cumprod((1,) + sizes[:0:-1])[::-1]
            self.buffers[name] = ctx.upload(data)
            self.descs[name] = capi.make_desc(self.buffers[name].ptr, dtype, sizes, [int(s) for s in strides])

        f32 = lambda k, m, mean=0.0: normal(seed + k, m, mean).astype(np.float32)  # noqa: E731
        for k, name in enumerate(("gate", "x", "grad")):
            put(name, f32(k, n, 2.0 * (k == 0)), capi.F32, B, T, C)
        for name in ("state", "y", "z", "d_y", "d_state", "d_gate", "d_x"):
            put(name, np.zeros(n, np.float32), capi.F32, B, T, C)
        for k, name in enumerate(("w", "b")):
            put(name, f32(10 + k, C, 1.0 - k), capi.F32, C)
        for name in ("d_w", "d_b"):
            put(name, np.zeros(C, np.float32), capi.F32, C)
        for name in ("mean", "rstd"):
            put(name, np.zeros(B * G, np.float32), capi.F32, B, G)
        put("last", np.zeros(B * C, np.float32), capi.F32, B, C)
        self.base = ctx.upload(np.array([0], dtype=np.uint64))
        self.rooms = {}
        need = c_int64(0)
        capi.check_nn(capi.nn.hmn_recurrence_workspace(byref(self.descs["x"]), byref(need)))
        self.rooms["recurrence"] = (ctx.malloc(need.value), need.value)
        for back in (0, 1):
            capi.check_nn(capi.nn.hmn_group_norm_workspace(byref(self.descs["x"]), G, back, byref(need)))
            self.rooms[back] = (ctx.malloc(need.value), need.value)
        for room, size in self.rooms.values():  # what a workspace holds does not matter
            capi.check(capi.lib.hmr_memset(ctx.handle, room.ptr, 0xFF, max(size, 1)))

    OUTPUTS = ("state", "last", "y", "mean", "rstd", "z", "d_y", "d_state", "d_w", "d_b", "d_gate", "d_x")

    def queue(self):
        N, c = capi.nn, self.ctx.handle
        d = {k: byref(v) for k, v in self.descs.items()}
        room = {k: (r.ptr, s) for k, (r, s) in self.rooms.items()}
        capi.check_nn(N.hmn_recurrence(c, 1, d["state"], d["last"], d["gate"], d["x"], None, None, *room["recurrence"]))
        capi.check_nn(N.hmn_group_norm(c, d["y"], d["mean"], d["rstd"], d["state"], d["w"], d["b"], self.G, 1e-5, 15, *room[0]))
        capi.check_nn(N.hmn_dropout(c, d["z"], d["y"], d["x"], 0.3, 7, 99, self.base.ptr))
        capi.check_nn(N.hmn_dropout(c, d["d_y"], d["grad"], None, 0.3, 7, 99, self.base.ptr))
        capi.check_nn(N.hmn_group_norm_backward(c, d["d_state"], d["d_w"], d["d_b"], d["d_y"], d["state"], d["mean"], d["rstd"], d["w"],
                                                d["b"], self.G, 15, *room[1]))
        capi.check_nn(N.hmn_recurrence_backward(c, 1, d["d_gate"], d["d_x"], None, d["d_state"], None, d["gate"], d["x"], d["state"],
                                                None, None, *room["recurrence"]))

    def results(self):
        self.ctx.synchronize()
        return {k: self.buffers[k].download(np.uint32, self.buffers[k].nbytes // 4) for k in self.OUTPUTS}

    def clear(self):
        for k in self.OUTPUTS:
            capi.check(capi.lib.hmr_memset(self.ctx.handle, self.buffers[k].ptr, 0xA5, self.buffers[k].nbytes))


@pytest.fixture()
def ctx():
    c = capi.Context(0)
    yield c
    c.close()


def same(a, b):
    for k in a:
        assert np.array_equal(a[k], b[k]), k


def test_two_graphs_that_share_workspaces_replay_with_the_eager_bits(ctx):
    calls = Calls(ctx, 1)
    calls.queue()
    eager = calls.results()
    first, second = Graph(ctx, calls.queue), Graph(ctx, calls.queue)
    for k in range(4):
        calls.clear()
        first.replay()
        same(calls.results(), eager)
        calls.queue()  # the program's own work between replays
        second.replay()
        first.replay()
        same(calls.results(), eager)


def test_a_graph_that_moves_the_base_draws_new_masks(ctx):
    calls = Calls(ctx, 3, T=500)
    blocks = (np.prod(calls.shape) + 3) // 4
    graph = Graph(ctx, calls.queue)  # holds the word's address; the word itself moves
    masks = []
    for k in range(3):
        word = np.array([k * blocks], dtype=np.uint64)
        capi.check(capi.lib.hmr_copy_from_host(ctx.handle, calls.base.ptr, word.ctypes.data, 8))
        graph.replay()
        got = calls.results()["d_y"].view(np.float32)
        grad = normal(3 + 2, got.size, 0.0).astype(np.float32)
        assert np.array_equal(got, ref.dropout(grad.astype(float), None, 0.3, 7, 99 + int(k * blocks), DT.F32))
        masks.append(got != 0)
    assert not np.array_equal(masks[0], masks[1]) and not np.array_equal(masks[1], masks[2])


def test_two_contexts_at_once_from_two_threads():
    """Two streams whose kernels overlap, each with its own buffers and workspaces."""
    contexts = [capi.Context(0) for _ in range(2)]
    try:
        calls = [Calls(c, 100 * k) for k, c in enumerate(contexts)]
        alone = []
        for c in calls:
            c.queue()
            alone.append(c.results())
        for c in calls:
            c.clear()
            c.ctx.synchronize()
        failures = []

        def work(c, want):
            try:
                for _ in range(20):
                    c.queue()
                same(c.results(), want)
            except BaseException as e:  # noqa: BLE001
                failures.append(e)

        threads = [threading.Thread(target=work, args=a) for a in zip(calls, alone)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failures, failures
    finally:
        for c in contexts:
            c.close()


def test_a_read_back_does_not_take_what_the_mailbox_held_before(ctx):
    """A check's verdict travels through pinned memory that any later kernel of the context makes stale, these among
    them: the words that a dropout writes over the verdict are what is read back."""
    index = ctx.upload(np.array([5, 900], dtype=np.int64))
    slot = ctx.malloc(16)
    d = capi.make_desc(index.ptr, capi.I64, (2,), (1,))
    capi.check(capi.lib.hmr_index_check(ctx.handle, byref(d), 0, 10, 0, 0, slot.ptr))
    src = ctx.upload(np.array([1.5, 2.5], dtype=np.float64))
    o, s = (capi.make_desc(b.ptr, capi.F64, (2,), (1,)) for b in (slot, src))
    capi.check_nn(capi.nn.hmn_dropout(ctx.handle, byref(o), byref(s), None, 0.0, 0, 0, None))
    assert np.array_equal(slot.download(np.float64, 2), [1.5, 2.5])


def test_workspaces_of_exactly_the_bytes_asked_for(ctx):
    """Nothing is written past them, nor in the tensors' neighbourhood."""
    calls = Calls(ctx, 9, B=3, T=700, C=33, G=3)
    guards = {}
    for k, (room, size) in list(calls.rooms.items()):
        guarded = ctx.malloc(size + 4096)
        capi.check(capi.lib.hmr_memset(ctx.handle, guarded.ptr, 0x5A, size + 4096))
        calls.rooms[k] = (guarded, size)
        guards[k] = guarded
    calls.queue()
    ctx.synchronize()
    for k, g in guards.items():
        assert (g.download(np.uint8, g.nbytes)[calls.rooms[k][1]:] == 0x5A).all(), k


def test_outputs_inside_larger_tensors_leave_their_neighbours(ctx):
    """Rows and channels around a strided output, and behind the last sequence, stay as they were."""
    B, T, C, pad = 2, 150, 41, 7
    whole = (B + 1, T + 2, C + pad)
    n = int(np.prod(whole))
    strides = ((T + 2) * (C + pad), C + pad, 1)
    for dtype, np_dtype in ((capi.F32, np.float32), (capi.BF16, np.uint16)):
        data = (normal(1, n).astype(np.float32) if dtype == capi.F32 else from_f64(normal(1, n), DT.BF16))
        out, out2, src = (ctx.upload(v) for v in (np.full(n, 77, np_dtype), np.full(n, 77, np_dtype), data))
        d = {k: capi.make_desc(b.ptr, dtype, (B, T, C), strides, offset=strides[1] + 3) for k, b in (("o", out), ("p", out2), ("s", src))}
        d = {k: byref(v) for k, v in d.items()}
        need = c_int64(0)
        rooms = []
        for ask in (lambda: capi.nn.hmn_recurrence_workspace(d["s"], byref(need)), lambda: capi.nn.hmn_group_norm_workspace(d["s"], 1, 0, byref(need)),
                    lambda: capi.nn.hmn_group_norm_workspace(d["s"], 1, 1, byref(need))):
            capi.check_nn(ask())
            rooms.append((ctx.malloc(need.value), need.value))
        room = [(r.ptr, s) for r, s in rooms]
        stats = [ctx.malloc(4 * B) for _ in range(2)]
        m, r = (byref(capi.make_desc(b.ptr, capi.F32, (B, 1), (1, 1))) for b in stats)
        calls = {
            "recurrence": lambda: capi.nn.hmn_recurrence(ctx.handle, 1, d["o"], None, d["s"], d["s"], None, None, *room[0]),
            "recurrence_backward": lambda: capi.nn.hmn_recurrence_backward(ctx.handle, 1, d["o"], d["p"], None, d["s"], None, d["s"], d["s"],
                                                                           d["s"], None, None, *room[0]),
            "norm": lambda: capi.nn.hmn_group_norm(ctx.handle, d["o"], m, r, d["s"], None, None, 1, 1e-5, 15, *room[1]),
            "norm_backward": lambda: capi.nn.hmn_group_norm_backward(ctx.handle, d["o"], None, None, d["s"], d["s"], m, r, None, None, 1, 15, *room[2]),
            "dropout": lambda: capi.nn.hmn_dropout(ctx.handle, d["o"], d["s"], None, 0.5, 1, 2, None),
        }
        inside = np.zeros(whole, bool)
        inside[:B, 1:T + 1, 3:C + 3] = True
        for name, call in calls.items():
            capi.check_nn(call())
            for b in (out, out2):
                v = b.download(np_dtype, n).reshape(whole)
                assert (v[~inside] == 77).all(), name


def test_elements_past_four_gibibytes(ctx):
    """A tensor whose second sequence begins past byte 2^32 through every entry point: compared with the same rows on
    their own."""
    B, T, C = 2, 300, 64
    gap = (1 << 31) + 1024  # elements of 2 bytes
    data = [from_f64(normal(k, B * T * C, 1.0 * (k == 0)), DT.BF16).reshape(B, T * C) for k in range(4)]
    base = ctx.malloc(2 * (2 * gap))
    far = [gap, C, 1]

    def lay(k, at):
        for b in range(B):
            v = np.ascontiguousarray(data[k][b])
            capi.check(capi.lib.hmr_copy_from_host(ctx.handle, base.ptr + 2 * (at + b * gap), v.ctypes.data, v.nbytes))
        return byref(capi.make_desc(base.ptr, capi.BF16, (B, T, C), far, offset=at))

    step = T * C + 64
    gate, x, grad, state = (lay(k, k * step) for k in range(4))
    outs = [byref(capi.make_desc(base.ptr, capi.BF16, (B, T, C), far, offset=(4 + k) * step)) for k in range(2)]
    keep = [ctx.upload(d) for d in data]
    near = [byref(capi.make_desc(b.ptr, capi.BF16, (B, T, C), (T * C, C, 1))) for b in keep]
    near_out_b = [ctx.malloc(2 * B * T * C) for _ in range(2)]
    near_out = [byref(capi.make_desc(b.ptr, capi.BF16, (B, T, C), (T * C, C, 1))) for b in near_out_b]
    stats = [ctx.malloc(4 * B * 4) for _ in range(2)]
    m, r = (byref(capi.make_desc(b.ptr, capi.F32, (B, 4), (4, 1))) for b in stats)
    need = c_int64(0)

    def room(ask):
        capi.check_nn(ask)
        b = ctx.malloc(need.value)
        keep.append(b)
        return b.ptr, need.value

    def run(gate, x, grad, state, o):
        N = capi.nn
        ws = room(N.hmn_recurrence_workspace(gate, byref(need)))
        yield N.hmn_recurrence(ctx.handle, 1, o[0], None, gate, x, None, None, *ws)
        yield N.hmn_recurrence_backward(ctx.handle, 1, o[0], o[1], None, grad, None, gate, x, state, None, None, *ws)
        yield N.hmn_group_norm(ctx.handle, o[0], m, r, x, None, None, 4, 1e-5, 15, *room(N.hmn_group_norm_workspace(x, 4, 0, byref(need))))
        yield N.hmn_group_norm_backward(ctx.handle, o[0], None, None, grad, x, m, r, None, None, 4, 15,
                                        *room(N.hmn_group_norm_workspace(x, 4, 1, byref(need))))
        yield N.hmn_dropout(ctx.handle, o[0], x, grad, 0.5, 3, 4, None)

    for k, (a, b) in enumerate(zip(run(gate, x, grad, state, outs), run(*near, near_out))):
        capi.check_nn(a)
        capi.check_nn(b)
        for i in range(2 if k == 1 else 1):
            want = near_out_b[i].download(np.uint16, B * T * C).reshape(B, T * C)
            for s in range(B):
                got = np.empty(T * C, np.uint16)
                capi.check(capi.lib.hmr_copy_to_host(ctx.handle, got.ctypes.data, base.ptr + 2 * ((4 + i) * step + s * gap), got.nbytes))
                assert np.array_equal(got, want[s]), (k, i, s)
