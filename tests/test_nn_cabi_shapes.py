"""More of what libhomura_nn's entry points take and refuse, without a GPU (as in test_nn_cabi.py)."""
from ctypes import byref, c_int64

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


def test_a_workspace_query_of_any_size_is_answered():
    """Numbers of tiles that do not fit 32 bits, multiples of 2^32 among them: such sequences go without a scan."""
    need = c_int64(-1)
    for dtype in (capi.BF16, capi.F32, capi.F64):
        for sizes in ((1, 1 << 41, 1), (1, 1 << 62, 1), (1 << 40, 9, 1), (1, 1 << 40, 1 << 20), (3, (1 << 61) - 1, 1), (1, 9, 1 << 59), (1 << 32, 1 << 14, 1 << 15)):
            capi.check_nn(capi.nn.hmn_recurrence_workspace(byref(desc(dtype, *sizes, strides=[0, 0, 0])), byref(need)))
            assert need.value == 0, sizes
    refused(capi.nn.hmn_recurrence_workspace(byref(desc(capi.F32, 1 << 31, 1 << 31, 4, strides=[0, 0, 0])), byref(need)), "does not fit 64 bits")


@pytest.mark.parametrize("dtype", [capi.BF16, capi.F32, capi.F64])
def test_chained_scans_and_maps_need_a_workspace(dtype):
    need = c_int64(-1)
    for sizes in ((2, 100000, 24), (1, 5000, 24), (8, 2048, 4096)):
        capi.check_nn(capi.nn.hmn_recurrence_workspace(byref(desc(dtype, *sizes)), byref(need)))
        assert need.value > 0, sizes
    for backward in (0, 1):
        for sizes, groups in (((4, 20000, 24), 4), ((16, 4096, 320), 32), ((1, 70, 8), 1)):
            capi.check_nn(capi.nn.hmn_group_norm_workspace(byref(desc(dtype, *sizes)), groups, backward, byref(need)))
            assert need.value > 0, sizes
    # Tokens leave sums of their own for the weights' gradients, and nothing forwards.
    capi.check_nn(capi.nn.hmn_group_norm_workspace(byref(desc(dtype, 16384, 1, 4096)), 32, 1, byref(need)))
    assert need.value > 0
    capi.check_nn(capi.nn.hmn_group_norm_workspace(byref(desc(dtype, 16384, 1, 4096)), 32, 0, byref(need)))
    assert need.value == 0
