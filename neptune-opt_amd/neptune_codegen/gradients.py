"""The norm of all gradients together, and their clipping to a largest norm.

There is no reference function for this path:

    norm = sqrt(sum over all tensors of the squares of their elements)       g <- g min(1, max_norm / norm)

Layout contract: a list or tuple of tensors of any shapes, each float32, bfloat16 or float16, on one device.
Clipping writes them in place, or into tensors of their sizes and their dtype or float32; what it reads and
writes fills its memory without gaps (in any order of the dimensions).  Squares and sums are fp64, the norm is
rounded to fp32 once, and each element is multiplied by the fp32 factor with one rounding.  Where the norm is
at most max_norm, an infinity or NaN, the factor is 1.  Formulas and mapping are in
csrc/kernels/nep_gradients.h.
"""
from __future__ import annotations

import threading

from neptune_codegen import calls, dispatch, hip
from neptune_codegen.emitters import BASE_OPTIONS, emit_gradients_source

TENSORS = 112            # kTensors, kMostTensors and kSumLanes of nep_gradients.h
MOST_TENSORS = 4096
LANES = 1024
WORKGROUPS = 512         # two on a CU
_HEAD = (hip.I32,) * 3
_LIST, _FAR = (hip.I64,) * (4 * TENSORS), (hip.PTR,)
_SCALE = (hip.PTR, hip.I32, hip.PTR, hip.PTR, hip.F32, hip.I32)
# in the order in which the calls are given them (GradientCalls::add)
_KERNELS = (("gradient_norm", (hip.PTR, hip.I32, hip.PTR)), ("gradient_list", _LIST + (hip.I32, hip.PTR)),
            ("gradient_sums", _LIST + _HEAD + (hip.PTR,)), ("gradient_scale", _LIST + _HEAD + _SCALE),
            ("gradient_sums_far", _FAR + _HEAD + (hip.PTR,)), ("gradient_scale_far", _FAR + _HEAD + _SCALE),
            ("gradient_one", _LIST + _HEAD + (hip.PTR, hip.F32, hip.I32, hip.I32)))
_PROGRAM = None
_CALLS = None
_OPS: dict = {}
_lock = threading.RLock()


def _program() -> hip.Program:
    global _PROGRAM
    with _lock:
        if _PROGRAM is None:
            _PROGRAM = hip.Program(emit_gradients_source(), "gradients.hip", BASE_OPTIONS)
        return _PROGRAM


def _calls(device: int | None = None):
    """The calls in C++, with the kernels of `device` among them.  (One object for all threads: kernels that one
    adds are in the object that every other one uses.)"""
    global _CALLS
    with _lock:
        if _CALLS is None:
            _CALLS = dispatch.extension().GradientCalls(TENSORS, MOST_TENSORS, LANES, WORKGROUPS)
        if device is not None and not _CALLS.has(device):
            prog = _program()
            _CALLS.add(device, [prog.kernel(name, args, LANES, device).handle for name, args in _KERNELS])
        return _CALLS


def _dense(t) -> bool:
    """Whether the tensor's elements fill its memory without gaps or overlaps."""
    want = 1
    for stride, size in sorted((t.stride(d), t.shape[d]) for d in range(t.ndim) if t.shape[d] != 1):
        if stride != want:
            return t.numel() == 0
        want *= size
    return True


def _check_list(tensors, name: str, *, metadata: bool) -> None:
    import torch

    if not isinstance(tensors, (list, tuple)) or not tensors:
        raise TypeError(f"{name} must be a list of at least one tensor")
    for t in tensors:
        calls.check_tensor(t, name, metadata=metadata, negated=True)    # (the norm resolves, clipping refuses)
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
        if t.device != tensors[0].device:
            raise ValueError(f"{name} must be on the same device")


def validate_gradient_inputs(tensors, out=None, norm=None, *, metadata: bool = False) -> None:
    import torch

    _check_list(tensors, "gradients", metadata=metadata)
    if out is not None:
        _check_list(out, "clipped gradients", metadata=metadata)
        if len(out) != len(tensors):
            raise ValueError(f"{len(tensors)} gradients need as many outputs, got {len(out)}")
        for t, o in zip(tensors, out):
            if o.shape != t.shape or o.device != t.device:
                raise ValueError(f"clipped gradient {tuple(o.shape)} must have the gradient's shape {tuple(t.shape)} "
                                 "and device")
            if o.dtype not in (t.dtype, torch.float32):
                raise TypeError(f"clipped gradients must be float32 or {t.dtype}, got {o.dtype}")
    if norm is not None:
        calls.check_tensor(norm, "gradients' norm", metadata=metadata)
        if norm.ndim or norm.dtype != torch.float32 or norm.device != tensors[0].device:
            raise ValueError("gradients' norm must be a float32 number on the gradients' device")


def _refuse_written(tensors, out) -> None:
    for t, o in zip(tensors, tensors if out is None else out):
        if o.requires_grad:
            raise ValueError("clipped gradients are written in place and must not require grad")
        if not _dense(t) or not _dense(o) or any(a != b for a, b, n in zip(t.stride(), o.stride(), t.shape)
                                                 if n != 1 and t.numel()):
            raise ValueError("clipped gradients must fill their memory without gaps, outputs in their gradient's "
                             "order")
    raise ValueError("clipped gradients must be plain tensors (and no negated views) that do not overlap one another, "
                     "what is read, or the norm")


def _refuse_recording() -> None:
    if hip.recording_active():
        raise NotImplementedError("a call with a list of tensors has no launch plan and cannot be recorded")


def _is_metadata(tensors) -> bool:
    import torch

    return isinstance(tensors, (list, tuple)) and bool(tensors) and isinstance(tensors[0], torch.Tensor) \
        and calls.is_metadata(tensors[0])


def _plain(tensors, copies: bool):
    """The tensors without their subclasses; with `copies`, those with gaps (or a sign to come) copied."""
    import torch

    return None if tensors is None else [
        ((t if _dense(t) else t.contiguous()).resolve_neg() if copies else t).as_subclass(torch.Tensor)
        for t in tensors]


def run_gradient_norm(tensors):
    """The 2-norm of all the tensors' elements together, fp32 without dimensions, on the current stream."""
    _refuse_recording()
    found = (_CALLS or _calls()).norm(tensors)
    if found is not None:
        return found
    import torch

    metadata = _is_metadata(tensors)
    validate_gradient_inputs(tensors, metadata=metadata)
    if metadata:
        return torch.empty((), dtype=torch.float32, device=tensors[0].device)
    found = _calls(calls.device_index(tensors[0])).norm(_plain(tensors, True))
    if found is None:
        raise TypeError("gradients must be plain tensors, or subclasses that are plain tensors without their class")
    return found


def _max_norm(max_norm) -> float:
    if type(max_norm) not in (int, float) or not 0.0 <= max_norm <= calls.MOST_FLOAT:
        raise ValueError("clipping needs a max_norm that is finite in fp32 and not negative")
    return float(max_norm)


def run_clip_gradients(tensors, max_norm: float, *, norm=None, out=None):
    """Scales the tensors to a common norm of at most `max_norm`, in place or into the tensors `out` (a copy,
    where the factor is 1), and returns their norm before, fp32 without dimensions.  `norm` is that norm where
    the caller has it already (from run_gradient_norm, or of the shards of several devices)."""
    _refuse_recording()
    max_norm = _max_norm(max_norm)
    found = (_CALLS or _calls()).clip(tensors, out, norm, max_norm)
    if found is not None:
        return found
    import torch

    metadata = _is_metadata(tensors)
    validate_gradient_inputs(tensors, out, norm, metadata=metadata)
    if metadata:
        return torch.empty((), dtype=torch.float32, device=tensors[0].device)
    found = _calls(calls.device_index(tensors[0])).clip(_plain(tensors, False), _plain(out, False),
                                                        None if norm is None else _plain([norm], False)[0], max_norm)
    if found is None:
        _refuse_written(tensors, out)
    return found


@dispatch.one_at_a_time
def as_gradient_norm_op(lib: str = "neptune"):
    """Custom op `(Tensor[] tensors) -> Tensor`: run_gradient_norm, without a gradient of its own."""
    import torch

    with _lock:
        if (lib, "norm") in _OPS:
            return _OPS[lib, "norm"]

    def _fake(tensors):
        validate_gradient_inputs(tensors, metadata=True)
        return torch.empty((), dtype=torch.float32, device=tensors[0].device)

    op = torch.library.custom_op(f"{lib}::gradient_norm", mutates_args=(),
                                 schema="(Tensor[] tensors) -> Tensor")(lambda tensors: run_gradient_norm(tensors))
    op.register_fake(_fake)
    with _lock:
        return _OPS.setdefault((lib, "norm"), op)


@dispatch.one_at_a_time
def as_clip_gradients_op(lib: str = "neptune"):
    """Custom op `(Tensor(a!)[] tensors, float max_norm) -> Tensor`: run_clip_gradients in place."""
    import torch

    with _lock:
        if (lib, "clip") in _OPS:
            return _OPS[lib, "clip"]

    def _clip(tensors, max_norm):
        return run_clip_gradients(tensors, max_norm)

    def _fake(tensors, max_norm):
        validate_gradient_inputs(tensors, metadata=True)
        return torch.empty((), dtype=torch.float32, device=tensors[0].device)

    op = torch.library.custom_op(f"{lib}::clip_gradients", mutates_args=("tensors",),
                                 schema="(Tensor(a!)[] tensors, float max_norm) -> Tensor")(_clip)
    op.register_fake(_fake)
    with _lock:
        return _OPS.setdefault((lib, "clip"), op)
