"""Calls of the sizes from which the kernels load and store past the caches (112 and 224 MiB), against the same rows in smaller
calls, which go through the caches: the same arithmetic, and so the same bits."""
import numpy as np
import pytest

from tests.support import DT, FLOATS, GPU, SIZE, array, h

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def rows_past(limit_mib, per_row, operands, dtype):
    """Rows of `per_row` elements so that `operands` tensors of them are just past the limit, an even number."""
    n = limit_mib * MIB // (per_row * operands * SIZE[dtype]) + 2
    return n + n % 2


def random(seed, *shapes, dtype):
    h.manual_seed(seed)
    return [h.randn(list(s), dtype, GPU) for s in shapes]


def same(a, b, what):
    assert np.array_equal(array(a).view(np.uint8), array(b).view(np.uint8)), what


def halves(t):
    n = t.shape[0] // 2
    return t.narrow(0, 0, n), t.narrow(0, n, n)


# Whole lines (every row begins one), and rows that begin inside lines, which are loaded through the caches.
@pytest.mark.parametrize("C", [4096, 4099])
@pytest.mark.parametrize("is_sigmoid", [False, True], ids=["factor", "sigmoid"])
@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
def test_recurrence(dtype, is_sigmoid, C):
    """Two sequences: a tile's place in its sequence, and with it every fold, is the same in a call of one."""
    operands = 6 if is_sigmoid else 5
    for back in (False, True):
        T = rows_past(224, 2 * C, operands if back else 3, dtype)
        gate, x, grad = random(1, *[(2, T, C)] * 3, dtype=dtype)
        if not is_sigmoid:
            gate = gate.sigmoid()
        out, last = h.linear_recurrence(gate, x, None, None, is_sigmoid)
        assert np.isfinite(array(last)).all()
        grads = h.grad_linear_recurrence(grad, last, gate, x, out, None, None, is_sigmoid) if back else ()
        for b in range(2):
            one = [t.narrow(0, b, 1) for t in (gate, x, grad, last, out)]
            if back:
                few = h.grad_linear_recurrence(one[2], one[3], one[0], one[1], one[4], None, None, is_sigmoid)
                for name, whole, part in zip(("d_gate", "d_input", "d_initial"), grads, few):
                    same(whole.narrow(0, b, 1), part, name)
            else:
                few = h.linear_recurrence(one[0], one[1], None, None, is_sigmoid)
                same(one[4], few[0], "out"), same(one[3], few[1], "last")


def check_norm(shape, G, dtype, act):
    N, S, C = shape
    x, grad, w, b = random(2, shape, shape, (C,), (C,), dtype=dtype)
    out, mean, rstd = h.group_norm(x, G, w, b, 1e-5, act)
    d_x, d_w, d_b = h.grad_group_norm(grad, x, mean, rstd, G, w, b, act)
    sums = []
    for k, (xs, gs, ms, rs) in enumerate(zip(*(halves(t) for t in (x, grad, mean, rstd)))):
        few = h.group_norm(xs, G, w, b, 1e-5, act)
        for name, whole, part in zip(("out", "mean", "rstd"), (out, mean, rstd), few):
            same(halves(whole)[k], part, name)
        few = h.grad_group_norm(gs, xs, ms, rs, G, w, b, act)
        same(halves(d_x)[k], few[0], "d_x")
        sums.append(few[1:])
    # The weights' gradients are sums over all rows: those of the halves, each off by a rounding to the type, and by some
    # thirty of the computation type of the terms' magnitudes (sqrt(N S) for normal ones, and the sum's own size).
    u = 2.0 ** -53 if dtype == DT.F64 else 2.0 ** -24
    step = {DT.F16: 2.0 ** -11, DT.BF16: 2.0 ** -8, DT.F32: 2.0 ** -24, DT.F64: 2.0 ** -53}[dtype]
    wide = DT.F64 if dtype == DT.F64 else DT.F32
    for whole, a, c in zip((d_w, d_b), *sums):
        whole, a, c = (array(t.to(wide)).astype(np.float64) for t in (whole, a, c))
        assert (np.abs(whole - (a + c)) <= 1.5 * step * (np.abs(whole) + np.abs(a) + np.abs(c)) + 64 * u * 4 * N * S).all()


# Groups in lanes of a wave with one to eight vectors each, and in a workgroup; the widths are the 16-bit types'.
@pytest.mark.parametrize("W, C", [(64, 4096), (1024, 4096), (2048, 4096), (4096, 4096), (8192, 8192)])
@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
def test_norm_of_tokens(dtype, W, C):
    W, C = W * 2 // SIZE[dtype], C * 2 // SIZE[dtype]
    check_norm((rows_past(224, C, 2, dtype), 1, C), C // W, dtype, "silu")


@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
def test_norm_of_maps(dtype):
    """Maps and channels enough that a workgroup has a whole map's positions of its channels, in a call of half of them too."""
    C = 256 * 16 // SIZE[dtype]
    check_norm((1024, max(66, rows_past(112, 1024 * C, 2, dtype)), C), 8, dtype, "gelu_tanh")


@pytest.mark.parametrize("onto", [False, True], ids=["alone", "onto a residual"])
@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
def test_dropout(dtype, onto):
    n = 8 * rows_past(224, 8, 3 if onto else 2, dtype) + 3  # the last vector is not whole
    x, residual = random(3, (n,), (n,), dtype=dtype)
    out = h.dropout_with(x, (0.3, 11, 12345), residual if onto else None)
    half = n // 8 * 4
    for at, size in ((0, half), (half, n - half)):
        part, r, want = (t.narrow(0, at, size) for t in (x, residual, out))
        same(want, h.dropout_with(part, (0.3, 11, 12345 + at // 4), r if onto else None), "dropout")
