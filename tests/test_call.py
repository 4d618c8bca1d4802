"""How gpu.call() takes its arguments, without a GPU: entry points and devices are stand-ins that note what reaches them."""
import contextlib
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from anode_amd import _lib, gpu


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


class OnDevice(torch.Tensor):
    """A tensor that says that it is on a device; its data stays on the host and is never looked at."""

    @staticmethod
    def make(device, contiguous=True):
        t = torch.Tensor._make_subclass(OnDevice, torch.zeros(4))
        t.at, t.packed = device, contiguous
        return t

    def get_device(self):
        return self.at

    is_cuda = True

    def is_contiguous(self):
        return self.packed

    def data_ptr(self):
        return 1000 + self.at


@pytest.fixture
def machine(monkeypatch):
    """Two devices, of which 0 is current; device d's current stream is 70 + d.  Gives the calls: (device, arguments)."""
    calls, now = [], [0]

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d
        try:
            yield
        finally:
            now[0] = before

    def entry(*args):
        calls.append((now[0], [a for a in args if not isinstance(a, type(ctypes.byref(gpu.DEFAULT_CONFIG)))]))
        return 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(gpu, "_raw_stream", lambda d: 70 + d)
    monkeypatch.setitem(gpu._entries, "entry", (entry, 3))
    return calls


def test_a_call_goes_to_the_device_of_its_tensors(machine):
    on = OnDevice.make
    assert gpu.call("entry", 5, on(0), on(0)) == 0
    assert gpu.call("entry", 5, on(1), on(1)) == 0
    assert gpu.call("entry", 5, 6, None) == 0                      # addresses alone: the current device
    assert machine == [(0, [5, 1000, 1000, 70]), (1, [5, 1001, 1001, 71]), (0, [5, 6, None, 70])]
    assert torch.cuda.current_device() == 0
    with pytest.raises(ValueError, match="devices 0 and 1"):
        gpu.call("entry", 5, on(0), on(1))
    with pytest.raises(ValueError, match="not contiguous"):
        gpu.call("entry", 5, on(1, contiguous=False), on(1))
    assert len(machine) == 3


def test_a_stream_is_taken_as_it_is(machine):
    on = OnDevice.make
    gpu.call("entry", 5, on(1), on(1), stream=99)                  # another device's stream
    gpu.call("entry", 5, on(0), on(1), stream=98)                  # a neighbour's memory
    assert machine == [(0, [5, 1001, 1001, 99]), (0, [5, 1000, 1001, 98])]
