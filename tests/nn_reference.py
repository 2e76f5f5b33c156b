"""Plain 64-bit implementations of libhomura_nn's operators in numpy, each beside a bound on what an evaluation in the
computation type may be off by (unit `u`: half a step of f32, or of f64 for F64), to which a test adds the one rounding
to the result's type."""
import math

import numpy as np

from tests.support import DT, from_f64, to_f64

HALF_STEP = {DT.F16: 2.0 ** -11, DT.BF16: 2.0 ** -8, DT.F32: 2.0 ** -24, DT.F64: 2.0 ** -53}
SMALLEST = {DT.F16: 2.0 ** -25, DT.BF16: 2.0 ** -134, DT.F32: 2.0 ** -149, DT.F64: 2.0 ** -1074}  # half a subnormal step (and what is flushed)
COMPUTE = {DT.F16: 2.0 ** -24, DT.BF16: 2.0 ** -24, DT.F32: 2.0 ** -24, DT.F64: 2.0 ** -53}
TINY = 1e-37  # f32 values below 2^-126 may be taken for zero on their way


def rounded(values, dtype):
    """f64 values as the dtype holds them."""
    return to_f64(from_f64(np.asarray(values), dtype), dtype).reshape(np.shape(values))


def assert_within(got, want, bound, dtype, what):
    """got (f64 values of the dtype) is within `bound` and one rounding to the dtype of want; NaN and infinities agree."""
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    tiny = 0.0 if dtype == DT.F64 else TINY
    limit = np.asarray(bound) + HALF_STEP[dtype] * (np.abs(want) + bound) + SMALLEST[dtype] + tiny
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities elsewhere"
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)), 0)
    limit = np.broadcast_to(limit, want.shape)
    bad = fine & ~(off <= limit)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / limit, 0)), off.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} values off; worst at {at}: got {got[at]!r}, want {want[at]!r}, "
                             f"off {off[at]:.3g}, allowed {limit[at]:.3g}")


# ---- the recurrence ------------------------------------------------------------------------------------------------

def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-z))


def steps_of(lengths, B, T):
    return np.full(B, T) if lengths is None else np.clip(np.asarray(lengths, dtype=np.int64), 0, T)


def recurrence(gate, x, initial, lengths, is_sigmoid, u):
    """(out, last, bound on out, bound on last).

    A state is a sum of contributions b_s * a_{s+1} ... a_t. Evaluated step by step or folded in any grouping, each
    factor adds at most two roundings (its product, the sum it takes part in) and a fold at the end a few more (16 are
    allowed: slots, tiles, groups and the conversions); `size` bounds the sum of the contributions' magnitudes. A
    sigmoid's two values are off by (|gate| + 8) u relative: the exponential's argument and value, the sum, the
    reciprocal and the product (the hardware's are within one step, 2 u, each)."""
    B, T, C = x.shape
    n = steps_of(lengths, B, T)
    h = np.zeros((B, C)) if initial is None else initial.copy()
    size, err = np.abs(h), np.zeros((B, C))
    out, bound = np.zeros((B, T, C)), np.zeros((B, T, C))
    for t in range(T):
        going = (t < n)[:, None]
        a, b, rel = gate[:, t], x[:, t], 0.0
        if is_sigmoid:
            rel = (np.abs(a) + 8) * u
            a, rest = sigmoid(a), sigmoid(-a)
            b = rest * b
        with np.errstate(invalid="ignore"):
            h_new = a * h + b
            err_new = np.abs(a) * err + (2 * u + rel) * (np.abs(a) * size + np.abs(b))
            size_new = np.abs(a) * size + np.abs(b)
        h, err, size = np.where(going, h_new, h), np.where(going, err_new, err), np.where(going, size_new, size)
        out[:, t], bound[:, t] = np.where(going, h, 0), np.where(going, err + 16 * u * size, 0)
    return out, h, bound, err + 16 * u * size


def recurrence_backward(grad, grad_last, gate, x, out, initial, lengths, is_sigmoid, u):
    """({d_gate, d_input, d_initial}, their bounds), the bounds as in recurrence() along the sequence backwards."""
    B, T, C = gate.shape
    n = steps_of(lengths, B, T)
    e = np.zeros((B, C)) if grad_last is None else grad_last.copy()
    size, err = np.abs(e), np.zeros((B, C))
    r = {k: np.zeros((B, T, C)) for k in ("d_gate", "d_input")}
    bounds = {k: np.zeros((B, T, C)) for k in r}
    for t in range(T - 1, -1, -1):
        going = (t < n)[:, None]
        before = out[:, t - 1] if t else (np.zeros((B, C)) if initial is None else initial)
        with np.errstate(invalid="ignore"):
            g, g_size = e + grad[:, t], size + np.abs(grad[:, t])
            g_err = err + 16 * u * size + u * g_size
            if is_sigmoid:
                rel = (np.abs(gate[:, t]) + 8) * u
                a, rest = sigmoid(gate[:, t]), sigmoid(-gate[:, t])
                d_x, x_bound = rest * g, rest * (g_err + (rel + 2 * u) * g_size)
                inner = before - x[:, t]
                d_g = g * inner * a * rest
                g_bound = np.abs(inner) * a * rest * (g_err + (2 * rel + 6 * u) * g_size)
            else:
                rel, a = 0.0, gate[:, t]
                d_x, x_bound = g, g_err
                d_g, g_bound = g * before, np.abs(before) * (g_err + 2 * u * g_size)
            e_new, err_new, size_new = a * g, np.abs(a) * (err + (2 * u + rel) * g_size), np.abs(a) * g_size
        for k, v, b in (("d_gate", d_g, g_bound), ("d_input", d_x, x_bound)):
            r[k][:, t], bounds[k][:, t] = np.where(going, v, 0), np.where(going, b, 0)
        e, err, size = np.where(going, e_new, e), np.where(going, err_new, err), np.where(going, size_new, size)
    r["d_initial"], bounds["d_initial"] = e, err + 16 * u * size
    return r, bounds


# ---- group normalisation -----------------------------------------------------------------------------------------------

ROOT_TWO_BY_PI = math.sqrt(2 / math.pi)
_erf = np.vectorize(math.erf, otypes=[np.float64])
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def activate(z, act):
    """(act(z), act'(z), relative error of their evaluation in units of u).

    The logistic function of v is off by |v| + 8 units (its exponential's argument and value, sum, reciprocal, product),
    gelu's erfc by 2 z^2 + 16 (its argument's rounding times its condition number, and its own); the slopes add a few
    products and sums of terms no larger than 1 + |z| times theirs."""
    if act is None:
        return z, np.ones_like(z), np.zeros_like(z)
    if act == "relu":
        return np.where(z < 0, 0, z), (z > 0).astype(float), np.zeros_like(z)
    if act == "silu":
        q = sigmoid(z)
        return z * q, q * (1 + z * (1 - q)), np.abs(z) + 16
    if act == "gelu":
        q = 0.5 * _erfc(-z * math.sqrt(0.5))
        return z * q, q + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi), 2 * z * z + 16
    v = 2 * ROOT_TWO_BY_PI * (z + 0.044715 * z ** 3)
    q = sigmoid(v)
    return z * q, q * (1 + z * (1 - q) * 2 * ROOT_TWO_BY_PI * (1 + 3 * 0.044715 * z * z)), 4 * np.abs(v) + 16


def fold(m):
    """What a f64 sum of m terms may be off by, relative to the sum of their magnitudes."""
    return (m / 256 + 16) * 2.0 ** -53


def _groups(x, G):
    N, S, C = x.shape
    return x.reshape(N, S, G, C // G)


def _spread(v, C):
    """[N, G] -> [N, 1, C]"""
    return np.repeat(v, C // v.shape[1], axis=1)[:, None, :]


def group_norm(x, G, weight, bias, eps, act, u):
    """(out, mean, rstd, bound on out, relative bound on rstd). The statistics are those of f64 sums, rounded once or
    twice on their way; hat and z take one rounding a step. The mean of an f64 sum is itself off by up to a few 2^-53 of
    the elements' mean magnitude: z moves by that times rstd * weight, which is what counts in F64 where an element is
    near the mean. A run of k additions is off by at most k 2^-53 of the sum of magnitudes; fold() allows the runs of a
    workgroup of 256 lanes over the group's elements and the joins after them. The reference sums in extended precision."""
    C = x.shape[2]
    g = _groups(x, G)
    mean = g.astype(np.longdouble).mean((1, 3))
    variance = ((g - mean[:, None, :, None]) ** 2).mean((1, 3)).astype(np.float64)
    mean, rstd = mean.astype(np.float64), 1 / np.sqrt(variance + eps)
    hat = (x - _spread(mean, C)) * _spread(rstd, C)
    w = np.ones(C) if weight is None else weight
    b = np.zeros(C) if bias is None else bias
    z = hat * w + b
    y, _, rel = activate(z, act)
    mean_err = fold(g[0, :, 0].size) * (np.abs(mean) + np.abs(g).mean((1, 3)))
    z_err = 6 * u * np.abs(hat * w) + 2 * u * np.abs(b) + u * np.abs(z) + np.abs(w) * _spread(mean_err * rstd, C)
    return y, mean, rstd, 1.2 * z_err + (rel + 4) * u * np.abs(y), 4 * u + fold(g[0, :, 0].size)


def group_norm_backward(grad, x, mean, rstd, G, weight, bias, act, u):
    """({d_x, d_weight, d_bias}, their bounds) from the statistics as they were handed over. Sums over a group or a
    channel are allowed 64 roundings of the sum of their terms' magnitudes (short runs in the computation type, the
    rest in f64)."""
    N, S, C = x.shape
    mean, rstd = _spread(mean, C), _spread(rstd, C)
    w = np.ones(C) if weight is None else weight
    b = np.zeros(C) if bias is None else bias
    hat = (x - mean) * rstd
    hat_err = 3 * u * np.abs(hat) + u * np.abs(mean) * rstd  # the difference of values near the mean is exact or off by u of itself
    z = hat * w + b
    z_err = np.abs(w) * hat_err + 2 * u * np.abs(hat * w) + u * np.abs(z)
    _, slope, rel = activate(z, act)
    # |act''| is below 1.2 for all of them (relu's jump at zero is kept out of the tests' inputs).
    slope_err = (0 if act in (None, "relu") else 1.2) * z_err + rel * u * (1 + np.abs(z)) * (0 if act in (None, "relu") else 1)
    d = grad * slope
    d_err = np.abs(grad) * slope_err + 2 * u * np.abs(d)
    by_group = lambda v: _spread(_groups(v, G).mean((1, 3)), C)  # noqa: E731
    wd, wd_err = w * d, np.abs(w) * d_err + u * np.abs(w * d)
    m1, m2 = by_group(wd), by_group(wd * hat)
    m1_err = by_group(wd_err + 64 * u * np.abs(wd))
    m2_err = by_group(wd_err * np.abs(hat) + np.abs(wd) * hat_err + 64 * u * np.abs(wd * hat))
    d_x = rstd * (wd - m1 - hat * m2)
    d_x_err = rstd * (wd_err + m1_err + np.abs(hat) * m2_err + hat_err * np.abs(m2) + 6 * u * (np.abs(wd) + np.abs(m1) + np.abs(hat * m2)))
    total = lambda v: v.sum((0, 1))  # noqa: E731
    r = {"d_x": d_x, "d_weight": total(d * hat), "d_bias": total(d)}
    return r, {"d_x": d_x_err, "d_weight": total(d_err * np.abs(hat) + np.abs(d) * hat_err + 64 * u * np.abs(d * hat)),
               "d_bias": total(d_err + 64 * u * np.abs(d))}


# ---- dropout --------------------------------------------------------------------------------------------------------------

def philox_words(n, seed, offset):
    """The first n 32-bit words of the Philox4x32-10 blocks from `offset` on under `seed`."""
    mask = np.uint64(0xFFFFFFFF)
    with np.errstate(over="ignore"):
        block = np.uint64(offset) + np.arange((n + 3) // 4, dtype=np.uint64)
    c = [block & mask, block >> np.uint64(32), np.zeros_like(block), np.zeros_like(block)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & mask, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n]


def dropout(x, residual, p, seed, offset, dtype):
    """The result's very values: one rounding of the scaled element to the computation type, one of the sum, one to the
    dtype. x and residual are f64 values of the dtype, in row-major order."""
    C = np.float64 if dtype == DT.F64 else np.float32
    keep = philox_words(x.size, seed, offset).reshape(x.shape) >= round(p * 2.0 ** 32)
    scale = C(0 if p == 1 else 1 / (1 - p))
    with np.errstate(all="ignore"):
        y = np.where(keep, x.astype(C) * scale, C(0))
        if residual is not None:
            y = residual.astype(C) + y
    return rounded(y.astype(np.float64), dtype)
