"""Calling the C ABI with torch-ROCm tensors.

torch is used for device memory and streams only; every computation goes
through the entry points of libanode_routines_gpu.so.  `call()` passes
arguments exactly as anode's Rust callers do (src/ops_gpu.rs:670-679): dims as
u32, device pointers, a host KernelConfig*, the stream handle.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import KernelConfig, load

# gpudevicemem's per-connection values are not visible in the reference; any
# power-of-two block size satisfies the reduction entry points' contract.
DEFAULT_CONFIG = KernelConfig(1024, 1024)


def _refuse(a: torch.Tensor):
    if not a.is_cuda:
        raise ValueError("the ABI takes device pointers: tensor is not on the GPU")
    raise ValueError("the ABI takes packed arrays: tensor is not contiguous")


_entries = {}  # name -> (function, number of arguments before (cfg, stream))


def _entry(name: str):
    lib = load()
    _, argtypes, _ = lib.prototypes[name]
    _entries[name] = entry = (lib.symbol(name), len(argtypes) - 2)
    return entry


# torch.cuda.current_stream().cuda_stream without the Stream object that it makes for every call (2.5 us of a call that
# otherwise takes 5), where this torch offers the handle by itself
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _current_stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device)


def call(name: str, *args, cfg: Optional[KernelConfig] = None, stream: Optional[int] = None):
    """Invoke entry point `name`; `args` are everything before (cfg, stream).  Returns what the entry point returns:
    None, or for those that can refuse their arguments 0 or an error code (nothing is enqueued then).

    Without a `stream` the call goes to the current stream of the device that its tensors are on, as torch's own operators
    do; they have to be on one.  A `stream` is taken as it is, and so are the tensors: the caller answers for the device that
    is current, and for what that device can reach."""
    fn, count = _entries.get(name) or _entry(name)
    if len(args) != count:
        raise TypeError(f"{name} takes {count} arguments before (cfg, stream): {load().prototypes[name][2][:-2]}")
    device = None
    values = []
    for a in args:
        if isinstance(a, torch.Tensor):
            at = a.get_device()  # -1 on the host
            if at < 0 or not a.is_contiguous():
                _refuse(a)
            if device is None:
                device = at
            elif at != device and stream is None:
                raise ValueError(f"tensors on devices {device} and {at}: the call has no stream of its own to say where it runs")
            a = a.data_ptr()
        values.append(a)
    tail = ctypes.byref(DEFAULT_CONFIG if cfg is None else cfg)
    if stream is not None:
        return fn(*values, tail, stream)
    current = torch.cuda.current_device()
    if device is None or device == current:
        return fn(*values, tail, _current_stream(current))
    with torch.cuda.device(device):
        return fn(*values, tail, _current_stream(device))


def take_last_error() -> int:
    return int(load().symbol("anode_gpu_take_last_error")())


def set_tuning(knob: int, value: int) -> int:
    return int(load().cdll.anode_gpu_set_tuning(knob, value))
