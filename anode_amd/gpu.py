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


def _refuse(a: torch.Tensor, device: int):
    if not a.is_cuda:
        raise ValueError("the ABI takes device pointers: tensor is not on the GPU")
    if a.get_device() != device:
        raise ValueError(f"the ABI works on the current device ({device}): tensor is on device {a.get_device()}")
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


def call(name: str, *args, cfg: Optional[KernelConfig] = None, stream: Optional[int] = None):
    """Invoke entry point `name`; `args` are everything before (cfg, stream).  Returns what the entry point returns:
    None, or for those that can refuse their arguments 0 or an error code (nothing is enqueued then)."""
    fn, count = _entries.get(name) or _entry(name)
    if len(args) != count:
        raise TypeError(f"{name} takes {count} arguments before (cfg, stream): {load().prototypes[name][2][:-2]}")
    device = None
    values = []
    for a in args:
        if isinstance(a, torch.Tensor):
            if device is None and a.is_cuda:  # (a tensor that is not on a GPU is refused before a device is asked for)
                device = torch.cuda.current_device()
            if a.get_device() != device or not a.is_contiguous():
                _refuse(a, device)
            a = a.data_ptr()
        values.append(a)
    if stream is None:
        device = torch.cuda.current_device() if device is None else device
        stream = torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device)
    return fn(*values, ctypes.byref(DEFAULT_CONFIG if cfg is None else cfg), stream)


def take_last_error() -> int:
    return int(load().symbol("anode_gpu_take_last_error")())


def set_tuning(knob: int, value: int) -> int:
    return int(load().cdll.anode_gpu_set_tuning(knob, value))
