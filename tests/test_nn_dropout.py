"""Dropout on the GPU: its very values, from the generator's words in numpy."""
import numpy as np
import pytest

from homura_amd import capi
from tests import nn_reference as ref
from tests.support import DT, FLOATS, GPU, array, from_f64, h, normal, tensor, to_f64, values as patterns

pytestmark = pytest.mark.gpu


def on_gpu(values, dtype):
    return tensor(from_f64(values, dtype), dtype, list(values.shape), GPU)


def values(t):
    return to_f64(array(t), t.dtype)


def check(x_gpu, x, residual_gpu, residual, mask, dtype, what=""):
    got = values(h.dropout_with(x_gpu, mask, residual_gpu))
    want = ref.dropout(x, None if residual is None else np.broadcast_to(residual, x.shape), *mask, dtype)
    assert np.array_equal(got, want, equal_nan=True), f"{what}: {(got != want).sum()} of {got.size} values differ"


@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 63, 64, 65, 1000, 1023, 4096, 33333, 262147])
def test_sizes(n, dtype):
    x, r = (ref.rounded(normal(n + k, n), dtype) for k in range(2))
    for mask in ((0.1, 67280421310721, 5), (0.5, (1 << 64) - 3, (1 << 32) - 2)):
        check(on_gpu(x, dtype), x, None, None, mask, dtype)
        check(on_gpu(x, dtype), x, on_gpu(r, dtype), r, mask, dtype)


@pytest.mark.parametrize("p", [0.0, 1.0, 2.0 ** -33, 2.0 ** -32, 1e-3, 0.9999, 1 - 2.0 ** -33, 1 - 2.0 ** -40])
def test_probabilities_to_both_ends(p):
    n = 10007
    x = ref.rounded(normal(3, n), DT.F32)
    check(on_gpu(x, DT.F32), x, None, None, (p, 11, 12), DT.F32)
    if p == 0.0:
        assert np.array_equal(values(h.dropout_with(on_gpu(x, DT.F32), (p, 11, 12))), x)


@pytest.mark.parametrize("dtype", FLOATS, ids=lambda d: d.name)
def test_every_pattern(dtype):
    """NaN, infinities, zeros of both signs and subnormals; what is dropped leaves a zero whatever it was."""
    n = 70001
    bits, more = patterns(dtype, n, 5), patterns(dtype, n, 6)
    x, r = to_f64(bits, dtype), to_f64(more, dtype)
    with np.errstate(all="ignore"):
        got = values(h.dropout_with(tensor(bits, dtype, [n], GPU), (0.4, 9, 9)))
        keep = ref.philox_words(n, 9, 9) >= round(0.4 * 2.0 ** 32)
        assert not got[~keep].any()
        assert np.array_equal(got, ref.dropout(x, None, 0.4, 9, 9, dtype), equal_nan=True)
        got = values(h.dropout_with(tensor(bits, dtype, [n], GPU), (0.4, 9, 9), tensor(more, dtype, [n], GPU)))
        assert np.array_equal(got, ref.dropout(x, r, 0.4, 9, 9, dtype), equal_nan=True)


@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32, DT.F64], ids=lambda d: d.name)
def test_the_mask_goes_by_the_position_not_by_the_layout(dtype):
    A, B, C = 6, 35, 44
    x = ref.rounded(normal(1, A * B * C).reshape(A, B, C), dtype)
    r = ref.rounded(normal(2, A * B * C).reshape(A, B, C), dtype)
    mask = (0.3, 5, 77)
    flat, onto = on_gpu(x, dtype), on_gpu(r, dtype)
    views = {
        "contiguous": flat,
        "permuted": on_gpu(np.ascontiguousarray(x.transpose(2, 0, 1)), dtype).permute([1, 2, 0]),
        "narrowed": on_gpu(np.concatenate([x, x], 2), dtype).narrow(2, C, C),
        "one off": on_gpu(np.concatenate([np.zeros(1), x.reshape(-1)]), dtype).narrow(0, 1, x.size).reshape([A, B, C]),
        "every other": on_gpu(np.repeat(x, 2, axis=1), dtype).slice(1, 1, None, 2),
    }
    for name, v in views.items():
        check(v, x, None, None, mask, dtype, name)
        check(v, x, onto, r, mask, dtype, name + " with a residual")
    for shape in ((C,), (B, 1), (A, 1, C), (1, 1, 1)):
        part = ref.rounded(normal(4, int(np.prod(shape))).reshape(shape), dtype)
        check(flat, x, on_gpu(part, dtype), part, mask, dtype, f"residual {shape}")
    one = on_gpu(x[:, :1, :], dtype).expand([A, B, C])
    check(one, np.broadcast_to(x[:, :1, :], x.shape), None, None, mask, dtype, "a broadcast x")


def test_its_gradient_is_itself_and_the_generator_moves_on():
    h.manual_seed(123)
    n = 4099
    x = ref.rounded(normal(1, n), DT.BF16)
    out, mask = h.dropout(on_gpu(x, DT.BF16), 0.25)
    assert mask == (0.25, 123, 0)
    again, later = h.dropout(on_gpu(x, DT.BF16), 0.25)
    assert later == (0.25, 123, (n + 3) // 4)
    assert not np.array_equal(values(out), values(again))
    g = ref.rounded(normal(2, n), DT.BF16)
    d = values(h.grad_dropout(on_gpu(g, DT.BF16), mask))
    assert np.array_equal(d, ref.dropout(g, None, 0.25, 123, 0, DT.BF16))
    kept = ref.philox_words(n, 123, 0) >= 1 << 30
    assert np.array_equal(d != 0, kept & (g != 0))
    # The words are those of rand: an F32 uniform below p is a word below its threshold when p has few digits.
    h.manual_seed(123)
    u = values(h.rand([n], DT.F32, GPU))
    assert np.array_equal(u >= 0.25, kept)
    # A refused call takes no blocks.
    h.manual_seed(123)
    with pytest.raises(Exception, match="probability"):
        h.dropout(on_gpu(x, DT.BF16), 1.5)
    with pytest.raises(Exception, match="broadcasts"):
        h.dropout(on_gpu(x, DT.BF16), 0.5, on_gpu(np.zeros(7), DT.BF16))
    assert h.dropout(on_gpu(x, DT.BF16), 0.5)[1] == (0.5, 123, 0)


def test_in_place_and_with_a_moved_base():
    from ctypes import byref
    ctx = capi.Context(0)
    try:
        n = 100003
        x, r = (normal(k, n).astype(np.float32) for k in (1, 2))
        base = ctx.upload(np.array([1 << 40], dtype=np.uint64))
        for same in ("src", "residual"):
            bx, br = ctx.upload(x), ctx.upload(r)
            dx, dr = (capi.make_desc(b.ptr, capi.F32, (n,), (1,)) for b in (bx, br))
            out = dx if same == "src" else dr
            capi.check_nn(capi.nn.hmn_dropout(ctx.handle, byref(out), byref(dx), byref(dr), 0.5, 7, 3, base.ptr))
            got = (bx if same == "src" else br).download(np.float32, n)
            assert np.array_equal(got, ref.dropout(x.astype(float), r.astype(float), 0.5, 7, 3 + (1 << 40), DT.F32))
    finally:
        ctx.close()


def test_more_dimensions_than_a_description_holds():
    shape = [1] * 20 + [2, 3] + [1] * 10 + [5, 1]
    x = ref.rounded(normal(9, 30), DT.F32)
    got, mask = h.dropout(on_gpu(x, DT.F32).reshape(shape), 0.5)
    assert got.shape == shape and np.array_equal(values(got).ravel(), ref.dropout(x, None, *mask, DT.F32))
    many = on_gpu(ref.rounded(normal(9, 1 << 13), DT.F32), DT.F32).reshape([2] * 13)
    turned = many.permute(list(range(12, -1, -1)))
    got, mask = h.dropout(turned, 0.5)
    assert np.array_equal(values(got), ref.dropout(values(turned), None, *mask, DT.F32))


def test_empty():
    assert h.dropout(on_gpu(np.zeros((3, 0)), DT.F32), 0.5)[0].shape == [3, 0]
