"""The argument checks of the entry points over rows of many classes, without a GPU: every refusal comes before any
device call, returns hipErrorInvalidValue, records it and says why; and the calls that have nothing to do return 0."""
import ctypes
import math
import os
import subprocess
import sys

import pytest

from anode_amd import _lib

P = 0x7F0000001000  # a device pointer that is never dereferenced: nothing is launched
TYPES = ("f32", "bf16", "f16")
REFUSED = 1  # hipErrorInvalidValue

CALLS = {
    "top_k_rows": ("uuuufpppp", ["dim0", "dim1", "stride", "k", "temperature", "x", "value", "index", "log_norm"]),
    "softmax_distill_rows": ("uuuufppppppp", ["dim0", "dim1", "stride", "k", "temperature", "x", "teacher_value", "teacher_index",
                                              "teacher_log_norm", "loss", "row_max", "row_sum"]),
    "softmax_distill_bwd_rows": ("uuuufpppppppp", ["dim0", "dim1", "stride", "k", "temperature", "dy", "x", "teacher_value",
                                                   "teacher_index", "teacher_log_norm", "row_max", "row_sum", "dx"]),
    "softmax_distill_bwd_rows_accumulate": ("uuuufpppppppp", ["dim0", "dim1", "stride", "k", "temperature", "dy", "x",
                                                              "teacher_value", "teacher_index", "teacher_log_norm", "row_max",
                                                              "row_sum", "dx"]),
    "softmax_distill_fused_fwd_bwd_rows": ("uuuufppppppppp", ["dim0", "dim1", "stride", "k", "temperature", "x", "teacher_value",
                                                              "teacher_index", "teacher_log_norm", "dy", "loss", "row_max",
                                                              "row_sum", "dx"]),
}
VERIFY = ("uuupppppppp", ["dim0", "dim1", "dim2", "target", "draft", "draft_token", "draft_length", "accept", "pick", "token",
                          "accepted"])
_KIND = {ctypes.c_uint32: "u", ctypes.c_float: "f", ctypes.c_void_p: "p"}


def _name(call, kind):
    return f"anode_gpu_{call}_{kind}"


def _call(name, names, **change):
    lib = _lib.load()
    lib.symbol("anode_gpu_take_last_error")()
    values = {"dim0": 100, "dim1": 3, "dim2": 2, "stride": 0, "k": 5, "temperature": 1.0}
    args = [change.get(n, values.get(n, P)) for n in names]
    rc = lib.symbol(name)(*args, ctypes.byref(_lib.KernelConfig(1024, 1024)), None)
    return rc, lib.symbol("anode_gpu_take_last_error")()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("call", CALLS)
def test_parameter_lists(call, kind):
    kinds, names = CALLS[call]
    restype, argtypes, got = _lib.parse_header()[_name(call, kind)]
    assert restype is ctypes.c_int and "".join(_KIND[t] for t in argtypes) == kinds + "pp" and got == names + ["cfg", "stream"]


def test_verify_parameter_list():
    restype, argtypes, got = _lib.parse_header()["anode_gpu_verify_draft_packed_f32"]
    assert restype is ctypes.c_int and "".join(_KIND[t] for t in argtypes) == VERIFY[0] + "pp" and got == VERIFY[1] + ["cfg", "stream"]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("call", CALLS)
def test_scalars_are_checked(call, kind, capfd):
    name, names = _name(call, kind), CALLS[call][1]
    for change in ({"stride": 99}, {"stride": 1}, {"k": 1025}, {"k": 0xFFFFFFFF}, {"temperature": 0.0}, {"temperature": -1.0},
                   {"temperature": math.nan}, {"temperature": math.inf}, {"temperature": 1e-39}):
        assert _call(name, names, **change) == (REFUSED, REFUSED), change
        err = capfd.readouterr().err
        assert name in err and "nothing was enqueued" in err


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("call", CALLS)
def test_missing_and_misaligned_arrays(call, kind):
    name, names = _name(call, kind), CALLS[call][1]
    for n in names[5:]:
        if n in ("log_norm", "teacher_log_norm"):
            continue
        assert _call(name, names, **{n: None}) == (REFUSED, REFUSED), n
    for n in ("x", "dx"):
        if n in names:
            for off in (1,) if kind != "f32" else (1, 2, 3):
                assert _call(name, names, **{n: P + off}) == (REFUSED, REFUSED), (n, off)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("call", [c for c in CALLS if "dx" in CALLS[c][1]])
def test_gradients_that_lie_across_the_logits(call, kind):
    name, names = _name(call, kind), CALLS[call][1]
    size = 4 if kind == "f32" else 2
    for elements, stride, rows in ((1, 0, 3), (-1, 0, 3), (99, 0, 1), (150, 0, 3), (299, 0, 3), (100, 120, 3), (121, 200, 3),
                                   (-199, 200, 2), (301, 200, 3), (499, 200, 3), (-499, 200, 3)):
        at = P + (1 << 20) + elements * size
        assert _call(name, names, x=P + (1 << 20), dx=at, stride=stride, dim1=rows) == (REFUSED, REFUSED), (elements, stride, rows)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("call", CALLS)
def test_no_rows_is_nothing_to_do(call, kind):
    name, names = _name(call, kind), CALLS[call][1]
    nothing = {n: None for n in names[5:]}
    assert _call(name, names, dim1=0, **nothing) == (0, 0)
    # a wrong scalar is refused all the same
    assert _call(name, names, dim1=0, temperature=-1.0, **nothing) == (REFUSED, REFUSED)


def test_nothing_asked_for_is_nothing_to_do():
    for kind in TYPES:
        assert _call(_name("top_k_rows", kind), CALLS["top_k_rows"][1], k=0, log_norm=None, value=None, index=None) == (0, 0)
        for call in ("softmax_distill_bwd_rows", "softmax_distill_bwd_rows_accumulate"):
            assert _call(_name(call, kind), CALLS[call][1], dim0=0, x=None, dx=None) == (0, 0)


def test_verify_checks():
    name, names = "anode_gpu_verify_draft_packed_f32", VERIFY[1]
    for n in ("target", "draft_token", "accept", "pick", "token", "accepted"):
        assert _call(name, names, **{n: None}) == (REFUSED, REFUSED), n
    assert _call(name, names, dim1=0xFFFFFFFF) == (REFUSED, REFUSED)
    assert _call(name, names, dim2=0, target=None, token=None) == (0, 0)


def test_refusals_need_no_device():
    code = r"""
import sys
sys.path.insert(0, %r); sys.path.insert(0, %r)
import test_class_rows_refusals as t
assert t._call("anode_gpu_top_k_rows_f32", t.CALLS["top_k_rows"][1], k=2000) == (1, 1)
print("refused")
""" % (_lib.REPO_ROOT, os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0 and "refused" in r.stdout, r.stderr


def test_scratch_query():
    q = _lib.load().symbol("anode_gpu_class_rows_scratch_bytes")
    assert q(0, 0, 0) == 0 and q(131072, 0, 64) == 0 and q(0, 100, 5) == 0
    assert q(1000, 256, 10) == 0                      # short rows: one workgroup each
    assert q(131072, 4096, 64) >= 4096 * 64 * 16      # the sums of a sequence's 64 blocks
    few = q(131072, 1, 64)
    assert 0 < few <= q(131072, 8, 64) < 1 << 26
    for k in (0, 1, 64, 1024, 5000):
        assert q(0xFFFFFFFF, 1, k) < 1 << 27


def test_scratch_that_cannot_be_had_is_an_error_code():
    # no device: nothing can be allocated.  Shapes that need scratch return the code that was recorded, and enqueue nothing.
    code = r"""
import sys
sys.path.insert(0, %r); sys.path.insert(0, %r)
import test_class_rows_refusals as t
for name, names, change in (("anode_gpu_top_k_rows_f32", t.CALLS["top_k_rows"][1], {"dim0": 131072, "dim1": 2}),
                            ("anode_gpu_softmax_distill_rows_bf16", t.CALLS["softmax_distill_rows"][1], {"dim0": 131072, "dim1": 2}),
                            ("anode_gpu_softmax_distill_fused_fwd_bwd_rows_f32", t.CALLS["softmax_distill_fused_fwd_bwd_rows"][1],
                             {"dim0": 131072, "dim1": 2, "dx": t.P + (1 << 30)}),
                            ("anode_gpu_verify_draft_packed_f32", t.VERIFY[1], {"dim0": 131072})):
    rc, err = t._call(name, names, **change)
    assert rc != 0 and rc == err, (name, rc, err)
print("reported")
""" % (_lib.REPO_ROOT, os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0 and "reported" in r.stdout, r.stderr
