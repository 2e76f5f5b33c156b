"""More of what libhomura_nn's entry points take and refuse, without a GPU (as in test_nn_cabi.py)."""
import pytest

from homura_amd import capi
from tests.test_nn_cabi import desc, recurrence_backward, refused


@pytest.mark.parametrize("dtype, text", [(capi.F16, "null context"), (capi.F32, "null context"), (capi.BF16, "d_gate has another dtype"),
                                         (capi.F64, "d_gate has another dtype")])
def test_the_gate_gradient_may_be_f32_beside_16_bits(dtype, text):
    refused(recurrence_backward(d_gate=desc(dtype, 2, 5, 24)), text)


@pytest.mark.parametrize("changes, text", [({"d_gate": desc(capi.F32, 2, 5, 25)}, "d_gate has different sizes"),
                                           ({"d_gate": desc(capi.F32, 2, 5, 24, ptr=0)}, "d_gate has no memory")])
def test_a_wide_gate_gradient_is_checked_like_the_others(changes, text):
    refused(recurrence_backward(**changes), text)
