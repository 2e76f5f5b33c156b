"""libhomura_nn as a link target, and what its entry points refuse, without a GPU: every check runs before the context
is looked at, so that a call with a NULL context that gets past them says so and queues nothing."""
import ctypes
import os
import re
import subprocess
from ctypes import byref, c_int64

import pytest

from homura_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
N = capi.nn
PTR = 0x10000  # never looked at


def test_the_library_exports_exactly_its_header():
    text = open(os.path.join(ROOT, "include", "homura_nn.h")).read()
    declared = set(re.findall(r"\b(hmn_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    out = subprocess.check_output(["nm", "-D", "--defined-only", capi.NN_PATH], text=True)
    assert {line.split()[-1] for line in out.splitlines() if line.strip()} == declared == set(capi.NN_PROTOTYPES)


def test_the_archive_holds_one_object_with_only_its_names_global():
    archive = capi.NN_PATH[:-2] + "a"
    assert subprocess.check_output(["ar", "t", archive], text=True).split() == ["homura_nn.o"]
    out = subprocess.check_output(["nm", "--defined-only", "-g", archive], text=True, stderr=subprocess.DEVNULL)
    names = {line.split()[-1] for line in out.splitlines() if len(line.split()) == 3}
    assert set(capi.NN_PROTOTYPES) <= names
    assert not {n for n in names if not n.startswith("hmn_")}


def test_a_c_program_links_against_both_archives(tmp_path):
    source = tmp_path / "both.c"
    source.write_text('#include "homura_nn.h"\n#include <stdio.h>\nint main(void) {\n'
                      '  hmr_status s = hmn_dropout(0, 0, 0, 0, 0.5, 0, 0, 0);\n'
                      '  printf("%d %s %s", (int)s, hmn_last_error(), hmr_built_archs());\n  return 0;\n}\n')
    lib = os.path.dirname(capi.NN_PATH)
    subprocess.check_call(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(source), os.path.join(lib, "libhomura_nn.a"),
                           os.path.join(lib, "libhomura_rocm.a"), "-L/opt/rocm/lib", "-lamdhip64", "-lstdc++", "-lm", "-lpthread",
                           "-Wl,-rpath,/opt/rocm/lib", "-o", str(tmp_path / "both")])
    assert subprocess.check_output([str(tmp_path / "both")], text=True) == "2 hmn_dropout: out is NULL gfx950"


def contiguous(sizes):
    strides, n = [], 1
    for s in reversed(sizes):
        strides.insert(0, n)
        n *= max(s, 1)
    return strides


def desc(dtype, *sizes, strides=None, ptr=PTR, ndim=None):
    d = capi.make_desc(ptr, dtype, sizes, strides or contiguous(sizes))
    if ndim is not None:
        d.ndim = ndim
    return d


def refused(status, text):
    assert status == capi.HMR_INVALID
    message = N.hmn_last_error().decode()
    assert text in message, message


def ref(d):
    return None if d is None else byref(d)


ROOM = (PTR, 1 << 40)


def recurrence(form=0, room=ROOM, ctx=None, **k):
    d = {"out": desc(capi.BF16, 2, 5, 24), "last": desc(capi.F32, 2, 24), "gate": desc(capi.BF16, 2, 5, 24),
         "input": desc(capi.BF16, 2, 5, 24), "initial": desc(capi.F32, 2, 24), "lengths": desc(capi.I32, 2)}
    d.update(k)
    return N.hmn_recurrence(ctx, form, *(ref(d[n]) for n in ("out", "last", "gate", "input", "initial", "lengths")), *room)


def recurrence_backward(form=1, room=ROOM, **k):
    names = ("d_gate", "d_input", "d_initial", "grad", "grad_last", "gate", "input", "out", "initial", "lengths")
    d = {n: desc(capi.F16, 2, 5, 24) for n in names}
    d.update({n: desc(capi.F32, 2, 24) for n in ("d_initial", "grad_last", "initial")}, lengths=desc(capi.I64, 2))
    d.update(k)
    return N.hmn_recurrence_backward(None, form, *(ref(d[n]) for n in names), *room)


@pytest.mark.parametrize("changes, text", [
    ({}, "null context"),
    ({"last": None, "initial": None, "lengths": None}, "null context"),
    ({"form": 2}, "unknown form 2"), ({"form": -1}, "unknown form -1"),
    ({"out": None}, "out is NULL"), ({"gate": None}, "gate is NULL"), ({"input": None}, "input is NULL"),
    ({"gate": desc(capi.BF16, 2, 5, 24, ndim=2)}, "gate has 2 dimensions"),
    ({"out": desc(capi.BF16, 2, 4, 24)}, "out has different sizes"),
    ({"input": desc(capi.F32, 2, 5, 24)}, "input has another dtype"),
    ({"out": desc(capi.BF16, 2, 5, 24, strides=[0, 24, 1])}, "out is written and has elements in one place"),
    ({"input": desc(capi.BF16, 2, 5, 24, strides=[-120, 24, 1])}, "negative stride"),
    ({"last": desc(capi.F64, 2, 24)}, "last has another dtype"), ({"initial": desc(capi.F16, 2, 24)}, "initial has another dtype"),
    ({"initial": desc(capi.F32, 24)}, "initial has 1 dimensions"),
    ({"lengths": desc(capi.F32, 2)}, "lengths are I32 or I64"), ({"lengths": desc(capi.I32, 3)}, "lengths has different sizes"),
    ({"input": desc(capi.BF16, 2, 5, 24, ptr=0)}, "input has no memory"),
    ({"gate": desc(11, 2, 5, 24)}, "invalid dtype 11"),
])
def test_recurrence_refuses(changes, text):
    refused(recurrence(**changes), text)


def test_integer_sequences_are_refused():
    i = desc(capi.I32, 2, 5, 24)
    refused(recurrence(out=i, gate=i, input=i), "floating point")


@pytest.mark.parametrize("changes, text", [
    ({}, "null context"),
    ({"form": 0, "input": None}, "null context"),
    ({"form": 1, "input": None}, "input is NULL"),
    ({"grad_last": None, "initial": None, "d_initial": None, "lengths": None}, "null context"),
    ({"d_gate": None}, "d_gate is NULL"), ({"d_input": None}, "d_input is NULL"), ({"grad": None}, "grad is NULL"),
    ({"out": None}, "out is NULL"), ({"d_gate": desc(capi.F16, 2, 5, 24, strides=[120, 0, 1])}, "elements in one place"),
    ({"d_initial": desc(capi.BF16, 2, 24)}, "d_initial has another dtype"),
    ({"grad": desc(capi.F32, 2, 5, 24)}, "grad has another dtype"),
])
def test_recurrence_backward_refuses(changes, text):
    refused(recurrence_backward(**changes), text)


def norm(groups=4, eps=1e-5, act=-1, room=ROOM, **k):
    d = {"out": desc(capi.F16, 3, 7, 24), "mean": desc(capi.F32, 3, 4), "rstd": desc(capi.F32, 3, 4), "src": desc(capi.F16, 3, 7, 24),
         "weight": desc(capi.F16, 24), "bias": desc(capi.F32, 24)}
    d.update(k)
    return N.hmn_group_norm(None, *(ref(d[n]) for n in ("out", "mean", "rstd", "src", "weight", "bias")), groups, eps, act, *room)


def norm_backward(groups=4, act=15, room=ROOM, **k):
    names = ("d_src", "d_weight", "d_bias", "grad", "src", "mean", "rstd", "weight", "bias")
    d = {n: desc(capi.BF16, 3, 7, 24) for n in names}
    d.update({n: desc(capi.F32, 3, 4) for n in ("mean", "rstd")})
    d.update({n: desc(capi.BF16, 24) for n in ("weight", "bias", "d_weight", "d_bias")})
    d.update(k)
    return N.hmn_group_norm_backward(None, *(ref(d[n]) for n in names), groups, act, *room)


@pytest.mark.parametrize("changes, text", [
    ({}, "null context"), ({"mean": None, "rstd": None, "weight": None, "bias": None}, "null context"),
    ({"groups": 0}, "24 channels do not make 0 groups"), ({"groups": 5}, "24 channels do not make 5 groups"), ({"groups": -4}, "groups"),
    ({"act": 4}, "unknown activation 4"), ({"act": 99}, "unknown activation 99"),
    ({"eps": -1e-9}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"),
    ({"src": None}, "src is NULL"), ({"out": None}, "out is NULL"), ({"out": desc(capi.F32, 3, 7, 24)}, "out has another dtype"),
    ({"mean": desc(capi.F16, 3, 4)}, "mean has to be F32"), ({"rstd": desc(capi.F32, 4, 3)}, "rstd has different sizes"),
    ({"weight": desc(capi.BF16, 24)}, "weight has another dtype"), ({"bias": desc(capi.F16, 23)}, "bias has different sizes"),
    ({"out": desc(capi.F16, 3, 7, 24, strides=[0, 24, 1])}, "elements in one place"),
])
def test_group_norm_refuses(changes, text):
    refused(norm(**changes), text)


@pytest.mark.parametrize("changes, text", [
    ({}, "null context"), ({"d_weight": None, "d_bias": None, "weight": None, "bias": None}, "null context"),
    ({"mean": None}, "mean is NULL"), ({"rstd": None}, "rstd is NULL"), ({"grad": None}, "grad is NULL"),
    ({"d_src": None}, "d_src is NULL"), ({"d_weight": desc(capi.F64, 24)}, "d_weight has another dtype"),
    ({"d_bias": desc(capi.BF16, 24, strides=[0])}, "elements in one place"), ({"groups": 7}, "do not make 7 groups"),
])
def test_group_norm_backward_refuses(changes, text):
    refused(norm_backward(**changes), text)


def dropout(p=0.5, **k):
    d = {n: desc(capi.F32, 6, 10) for n in ("out", "src", "residual")}
    d.update(k)
    return N.hmn_dropout(None, ref(d["out"]), ref(d["src"]), ref(d["residual"]), p, 1, 2, None)


@pytest.mark.parametrize("changes, text", [
    ({}, "null context"), ({"residual": None}, "null context"), ({"p": 0.0}, "null context"), ({"p": 1.0}, "null context"),
    ({"p": -0.01}, "probability"), ({"p": 1.01}, "probability"), ({"p": float("nan")}, "probability"),
    ({"src": None}, "src is NULL"), ({"src": desc(capi.F16, 6, 10)}, "different dtypes"), ({"residual": desc(capi.F32, 10)}, "dimensions"),
    ({"out": desc(capi.F32, 6, 10, strides=[0, 1])}, "elements in one place"),
    ({"src": desc(capi.F32, 6, 10, strides=[0, 1]), "residual": desc(capi.F32, 6, 10, strides=[0, 0])}, "null context"),
])
def test_dropout_refuses(changes, text):
    refused(dropout(**changes), text)


def test_integer_dropout_is_refused():
    i = desc(capi.I64, 6, 10)
    refused(dropout(out=i, src=i, residual=None), "floating point")


def test_workspaces_are_asked_for_and_checked():
    """A workspace too small, absent or misaligned is refused before the context is looked at."""
    need = c_int64(-1)
    for gate, call in ((desc(capi.BF16, 2, 100000, 24), "recurrence"), (desc(capi.F32, 1, 5000, 24), "recurrence")):
        capi.check_nn(N.hmn_recurrence_workspace(byref(gate), byref(need)))
        assert need.value >= 0
        if need.value > 0:
            state = desc(capi.F32, gate.sizes[0], gate.sizes[2])
            k = {"out": gate, "gate": gate, "input": gate, "last": state, "initial": state, "lengths": None}
            refused(recurrence(room=(PTR, need.value - 1), **k), "are needed")
            refused(recurrence(room=(None, need.value), **k), "are needed")
            refused(recurrence(room=(PTR + 8, need.value), **k), "aligned")
            refused(recurrence(room=(PTR, need.value), **k), "null context")
    src = desc(capi.F16, 4, 20000, 24)
    for backward in (0, 1):
        capi.check_nn(N.hmn_group_norm_workspace(byref(src), 4, backward, byref(need)))
        assert need.value >= 0
        if need.value > 0:
            stats = desc(capi.F32, 4, 4)
            k = {"src": src, "mean": stats, "rstd": stats}
            k.update({"d_src": src, "grad": src, "weight": None, "bias": None, "d_weight": None, "d_bias": None} if backward else {"out": src})
            call = norm_backward if backward else norm
            refused(call(room=(PTR, need.value - 1), **k), "are needed")
            refused(call(room=(PTR + 4, need.value), **k), "aligned")
            refused(call(room=(PTR, need.value), **k), "null context")
    refused(N.hmn_recurrence_workspace(None, byref(need)), "NULL")
    refused(N.hmn_group_norm_workspace(byref(src), 5, 0, byref(need)), "5 groups")


def test_workspaces_of_extreme_shapes():
    """More workgroups than a launch has go without a scan; a group for every channel needs little more than the maps do."""
    need = c_int64(-1)
    for sizes in ((1 << 23, 5, 1), (1 << 22, 700, 1), (1 << 40, 5, 1)):
        capi.check_nn(N.hmn_recurrence_workspace(byref(desc(capi.BF16, *sizes)), byref(need)))
        assert need.value == 0
    channels = 1 << 22
    capi.check_nn(N.hmn_group_norm_workspace(byref(desc(capi.BF16, 1, 65, channels)), channels, 0, byref(need)))
    assert 0 < need.value <= 48 * channels
    for sizes, groups in (((1 << 24, 65, 8), 8), ((1 << 20, 65, 32), 32)):
        for backward in (0, 1):
            capi.check_nn(N.hmn_group_norm_workspace(byref(desc(capi.BF16, *sizes)), groups, backward, byref(need)))
            assert need.value == 0


def test_the_failure_text_belongs_to_the_thread_and_the_library():
    import threading
    refused(dropout(p=2.0), "probability")
    seen = []
    t = threading.Thread(target=lambda: seen.append(N.hmn_last_error().decode()))
    t.start()
    t.join()
    assert seen == [""]
    assert "probability" in N.hmn_last_error().decode()
    assert "probability" not in capi.lib.hmr_last_error().decode()
    assert ctypes.sizeof(capi.hmr_tensor_desc) == 424
