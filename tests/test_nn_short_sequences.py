"""Large batches of sequences of a few steps, which go by one tile of a scan or a thread per channel: on both sides of the choice,
every sequence as in a call of a few."""
import numpy as np
import pytest

from tests.support import DT, GPU, array, h

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [DT.BF16, DT.F32], ids=lambda d: d.name)
@pytest.mark.parametrize("T", [12, 13, 16, 17])
@pytest.mark.parametrize("C", [1003, 4096, 300])
def test_a_large_batch_is_its_sequences(T, C, dtype):
    """A tile's bits are not a thread's (their folds round apart), so a part of the batch is compared with the formula's
    accuracy: both evaluations are within 2 T + 24 units of the sum of the contributions' magnitudes, which is below 8 here."""
    size = 2 if dtype == DT.BF16 else 4
    B = -(-(64 << 20) // (T * C * size)) + 1
    h.manual_seed(T + C)
    gate, x, grad = (h.randn([B, T, C], dtype, GPU) for _ in range(3))
    out, last = h.linear_recurrence(gate, x, None, None, True)
    back = h.grad_linear_recurrence(grad, last, gate, x, out, None, None, True)
    step = 2.0 ** -24 if dtype == DT.F32 else 2.0 ** -8
    for at in (0, B // 2, B - 3):
        part = [t.narrow(0, at, 3) for t in (gate, x, grad, last, out)]
        few, few_last = h.linear_recurrence(part[0], part[1], None, None, True)
        few_back = h.grad_linear_recurrence(part[2], part[3], part[0], part[1], part[4], None, None, True)
        for name, a, b in [("out", out, few), ("last", last, few_last)] + [(n, *p) for n, *p in zip(("d_gate", "d_input", "d_initial"), back, few_back)]:
            a, b = (array(t.to(DT.F32)).astype(np.float64) for t in (a.narrow(0, at, 3), b))
            scale = np.abs(b).max()
            assert np.abs(a - b).max() <= (2 * T + 24) * 2.0 ** -24 * 8 * max(scale, 1) + 2 * step * scale, (name, at)
