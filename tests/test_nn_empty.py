"""Calls that have nothing, or only states and statistics, to write, however many sequences or groups they name."""
from ctypes import byref

import numpy as np
import pytest

from homura_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    c = capi.Context(0)
    yield c
    c.close()


def nothing(ctx, dtype, *sizes):
    """A description of no elements: no memory of that size is there."""
    return byref(capi.make_desc(ctx.malloc(16).ptr, dtype, sizes, [0] * len(sizes)))


MANY = 1 << 40


def test_sequences_of_no_steps_without_a_state(ctx):
    d = nothing(ctx, capi.BF16, MANY, 0, 1 << 20)
    initial = byref(capi.make_desc(ctx.malloc(16).ptr, capi.F32, (MANY, 1 << 20), (0, 0)))
    for form in (capi.GATE_FACTOR, capi.GATE_SIGMOID):
        capi.check_nn(capi.nn.hmn_recurrence(ctx.handle, form, d, None, d, d, None, None, None, 0))
        capi.check_nn(capi.nn.hmn_recurrence_backward(ctx.handle, form, d, d, None, d, None, d, d, d, None, None, None, 0))
        if form == capi.GATE_FACTOR:  # 2^60 states nobody asks for
            capi.check_nn(capi.nn.hmn_recurrence(ctx.handle, form, d, None, d, d, initial, None, None, 0))
    ctx.synchronize()


def test_maps_of_no_positions_without_statistics(ctx):
    d = nothing(ctx, capi.F16, MANY, 0, 1 << 20)
    capi.check_nn(capi.nn.hmn_group_norm(ctx.handle, d, None, None, d, None, None, 1 << 20, 1e-5, -1, None, 0))
    stats = byref(capi.make_desc(ctx.malloc(16).ptr, capi.F32, (MANY, 1 << 20), (0, 0)))
    capi.check_nn(capi.nn.hmn_group_norm_backward(ctx.handle, d, None, None, d, d, stats, stats, None, None, 1 << 20, -1, None, 0))
    ctx.synchronize()


def test_no_steps_or_positions_still_hand_over_what_is_asked_for(ctx):
    B, C, G = 5, 12, 3
    state = np.arange(B * C, dtype=np.float32)
    start, last = ctx.upload(state), ctx.malloc(4 * B * C)
    d = nothing(ctx, capi.F32, B, 0, C)
    s, e = (byref(capi.make_desc(b.ptr, capi.F32, (B, C), (C, 1))) for b in (start, last))
    capi.check_nn(capi.nn.hmn_recurrence(ctx.handle, capi.GATE_FACTOR, d, e, d, d, s, None, None, 0))
    assert np.array_equal(last.download(np.float32, B * C), state)
    capi.check_nn(capi.nn.hmn_recurrence_backward(ctx.handle, capi.GATE_SIGMOID, d, d, e, d, s, d, d, d, None, None, None, 0))
    assert np.array_equal(last.download(np.float32, B * C), state)
    only = ctx.upload(np.zeros(B * G, np.float32))
    r = byref(capi.make_desc(only.ptr, capi.F32, (B, G), (G, 1)))
    capi.check_nn(capi.nn.hmn_group_norm(ctx.handle, d, None, r, d, None, None, G, 1e-5, -1, None, 0))
    assert np.isnan(only.download(np.float32, B * G)).all()
