"""What the entry points over rows of many classes return where there is no device: the code of their own failed launch, each
time, on a machine of any kind."""
import os
import subprocess
import sys

import pytest

from anode_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
HEAD = f"""
import sys
sys.path.insert(0, {_lib.REPO_ROOT!r}); sys.path.insert(0, {HERE!r})
import test_class_rows_refusals as t
"""


def run_without_device(code):
    env = dict(os.environ, HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", HEAD + code], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr
    return r


@pytest.mark.parametrize("dim0,dim1", [(100, 3), (3000, 3), (20000, 2), (40000, 2), (80000, 40), (131072, 2)])
def test_a_launch_that_fails_is_an_error_code(dim0, dim1):
    # shapes of every kernel, with scratch and without; twice, since an error that is pending already is not a new one
    r = run_without_device(f"""
for again in range(2):
    for kind in t.TYPES:
        for call in t.CALLS:
            change = {{"dim0": {dim0}, "dim1": {dim1}, "dx": t.P + (1 << 32)}}
            rc, err = t._call(t._name(call, kind), t.CALLS[call][1], **change)
            assert rc != 0 and rc == err, (again, call, kind, rc, err)
    rc, err = t._call("anode_gpu_verify_draft_packed_f32", t.VERIFY[1], dim0={dim0}, dim2={dim1})
    assert rc != 0 and rc == err, (again, "verify", rc, err)
print("done")
""")
    assert "anode_gpu_softmax_distill_rows_f16" in r.stderr and "anode_gpu_verify_draft_packed_f32" in r.stderr


def test_a_pair_of_arrays_that_takes_two_calls_ends_at_the_first_that_fails():
    # 16-bit logits and gradient an odd number of elements apart: loss, then gradient; neither is launched twice or after a failure
    r = run_without_device("""
rc, err = t._call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_bf16", t.CALLS["softmax_distill_fused_fwd_bwd_rows"][1],
                  x=t.P + 2, dx=t.P + (1 << 20))
assert rc != 0 and rc == err, (rc, err)
print("done")
""")
    assert r.stderr.count("anode_gpu_softmax_distill_fused_fwd_bwd_rows_bf16") == 1, r.stderr


def test_scratch_that_cannot_be_had_is_the_code_of_this_call():
    # other threads' errors come and go in the process-wide record meanwhile: calls on shapes with scratch return their own
    run_without_device("""
import ctypes, threading
from anode_amd import _lib
lib = _lib.load()
cfg = ctypes.byref(_lib.KernelConfig(1024, 1024))
def call(**change):
    values = dict({"dim0": 131072, "dim1": 2, "stride": 0, "k": 5, "temperature": 1.0}, **change)
    return lib.symbol("anode_gpu_top_k_rows_f32")(*[values.get(n, t.P) for n in t.CALLS["top_k_rows"][1]], cfg, None)
want = call()
assert want not in (0, 1), want
stop = threading.Event()
def others():
    while not stop.is_set():
        call(k=2000)                                        # refused: another code
        lib.symbol("anode_gpu_take_last_error")()           # and taken
threads = [threading.Thread(target=others) for _ in range(3)]
for thread in threads:
    thread.start()
got = {call() for _ in range(4000)} | {lib.symbol("anode_gpu_reserve_scratch")(None, 1 << 20) for _ in range(4000)}
stop.set()
for thread in threads:
    thread.join()
assert got == {want}, got
print("done")
""")
