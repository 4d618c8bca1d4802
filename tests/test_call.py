"""How gpu.call() takes its arguments, without a GPU: entry points and devices are stand-ins that note what reaches them."""
import os
import subprocess
import sys

from anode_amd import _lib


def test_a_tensor_on_the_host_is_refused_as_such_without_a_device():
    code = f"""
import sys
sys.path.insert(0, {_lib.REPO_ROOT!r})
import torch
from anode_amd import gpu
assert not torch.cuda.is_available()
for name, args in (("anode_gpu_copy_flat_map_f32", (4, torch.zeros(4), torch.zeros(4))),
                   ("anode_gpu_top_k_rows_f32", (4, 1, 0, 1, 1.0, torch.zeros(4), torch.zeros(1), torch.zeros(1), None))):
    for stream in (None, 0):
        try:
            gpu.call(name, *args, stream=stream)
        except ValueError as e:
            assert "not on the GPU" in str(e), e
        else:
            raise AssertionError("not refused")
print("done")
"""
    env = dict(os.environ, HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr
