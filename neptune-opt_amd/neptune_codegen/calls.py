"""What the training operators' entry points share: the key of a seen call, launches on the
tensors' own device, metadata calls and operand layouts."""
from __future__ import annotations

import contextlib

from neptune_codegen import hip

SEEN_MAX = 4096
# a launch has fewer than 2^32 work-items
MOST_THREADS = (1 << 32) - 1


class Seen(dict):
    """Launches by call key, emptied when it holds SEEN_MAX."""

    def keep(self, key, launch) -> None:
        if len(self) >= SEEN_MAX:
            self.clear()
        self[key] = launch


def tensors_key(*tensors):
    """Everything that validation and launch choice read of plain strided device tensors (None
    stands for an absent one), or None where the call takes the full path: dtypes, devices, shapes,
    strides and 16-byte alignment."""
    import torch

    if hip.recording_active():
        return None
    plain, parameter, strided, key = torch.Tensor, torch.nn.Parameter, torch.strided, []
    for t in tensors:
        if t is None:
            key.append(None)
            continue
        kind = type(t)
        if (kind is not plain and kind is not parameter) or not t.is_cuda or t.layout is not strided:
            return None
        key += (t.dtype, t.device, t.shape, t.stride(), t.data_ptr() % 16)
    return tuple(key)


def is_metadata(t) -> bool:
    from torch._subclasses.fake_tensor import FakeTensor

    return isinstance(t, FakeTensor) or t.device.type == "meta"


def device_index(t) -> int:
    import torch

    return t.device.index if t.device.index is not None else torch.cuda.current_device()


_HERE = contextlib.nullcontext()


def on_device(index: int):
    """Context in which `index` is the current device (kernels are launched on the current one)."""
    import torch

    return _HERE if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def check_tensor(t, name: str, *, metadata: bool) -> None:
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.layout != torch.strided:
        raise TypeError(f"{name} must be strided")
    if not metadata and t.device.type != "cuda":
        raise ValueError(f"{name} is on {t.device}; execution requires a ROCm (cuda) device")


def check_grid(groups: int, threads: int, name: str) -> None:
    if groups * threads > MOST_THREADS:
        raise NotImplementedError(f"{name}: the call needs {groups} workgroups of {threads} threads, "
                                  "more than one launch takes")
