"""The norms after and before a block, fused with the block's gate and residual scale, and their
gradients.

There is no reference function for this path; it is run_rms_norm twice around the residual add:

    residual = x + residual_scale * gate * norm(y; gamma_after)     (the block's output y)
    normed   = norm(residual; gamma_before)                         (the next block's input)

with norm(v; gamma) = v * rsqrt(mean(v^2) + eps) * gamma over the last dimension.  gamma_after may be
None (y is added as it is), and so may the gate.  Formulas and mapping are in
csrc/kernels/nep_residual_norm.h.

Layout contract: x and y [..., n] of one shape and dtype (float32, bfloat16, float16), n up to 16384;
gammas [n] of that dtype; a gate of x's shape, or with ones in its trailing leading dimensions (a gate
[batch, 1, n] for x [batch, tokens, n]), or [n].  Outputs are fresh and contiguous.  The arithmetic is
fp32 throughout with one rounding per output; normed is the norm of the residual before its rounding.
Column sums (gradients of the gammas and of a broadcast gate) are added in one order, without atomics.
"""
from __future__ import annotations

import math
import threading

from neptune_codegen import calls, hip
from neptune_codegen.emitters import (BASE_OPTIONS, ResidualNormVariant, emit_residual_norm_source,
                                      residual_norm_kernel_name)
from neptune_codegen.template import _row_last_layout, _validate_row_last

MAX_WIDTH = 16384
CUS = 256
_PROGRAMS: dict = {}
_OPS: dict = {}
_SEEN = calls.Seen()
_lock = threading.Lock()

_FORWARD_ARGS = (hip.PTR,) * 8 + (hip.I64, hip.I32) + (hip.I64,) * 3 + (hip.F32,) * 2
_BACKWARD_ARGS = (hip.PTR,) * 14 + (hip.I64, hip.I32) + (hip.I64,) * 7 + (hip.F32,)
_JOIN_ARGS = (hip.PTR,) * 4 + (hip.I32,) + (hip.I64,) * 2


def _program(stage: str, var: ResidualNormVariant) -> hip.Program:
    with _lock:
        prog = _PROGRAMS.get((stage, var))
        if prog is None:
            prog = _PROGRAMS[stage, var] = hip.Program(
                emit_residual_norm_source(stage, var), f"{residual_norm_kernel_name(stage, var)}.hip",
                BASE_OPTIONS)
        return prog


def _gate_groups(gate, x):
    """(gate rows, rows of x per gate row) of a gate's broadcast over x, or ValueError."""
    rows = math.prod(x.shape[:-1])
    if gate is None:
        return 0, 0
    if gate.ndim == 1:
        lead = ()
    elif gate.ndim == x.ndim:
        lead = gate.shape[:-1]
    else:
        lead = None
    kept = 0
    if lead is not None:
        while kept < len(lead) and lead[kept] == x.shape[kept]:
            kept += 1
        if any(size != 1 for size in lead[kept:]):
            lead = None
    if lead is None or gate.shape[-1] != x.shape[-1]:
        raise ValueError(f"residual norm gate {tuple(gate.shape)} must have the shape of x {tuple(x.shape)}, "
                         "ones in its last leading dimensions, or be one row")
    groups = math.prod(lead)
    return groups, rows // groups if groups else 0


def validate_residual_norm_inputs(x, y, gamma_after, gamma_before, gate=None, *, metadata: bool = False):
    """(gate rows, rows of x per gate row) of a call."""
    for t, name in ((x, "x"), (y, "y"), (gamma_before, "gamma_before")):
        calls.check_tensor(t, f"residual norm {name}", metadata=metadata)
    _validate_row_last(x, metadata=metadata)
    if y.shape != x.shape:
        raise ValueError(f"residual norm y {tuple(y.shape)} must have the shape of x {tuple(x.shape)}")
    for t, name in ((gamma_after, "gamma_after"), (gamma_before, "gamma_before")):
        if t is None:
            continue
        calls.check_tensor(t, f"residual norm {name}", metadata=metadata)
        if t.ndim != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError(f"residual norm {name} must be [{x.shape[-1]}], got {tuple(t.shape)}")
    if gate is not None:
        calls.check_tensor(gate, "residual norm gate", metadata=metadata)
    for t in (y, gamma_after, gamma_before, gate):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError("residual norm tensors must share one dtype and device")
    if x.shape[-1] > MAX_WIDTH:
        raise NotImplementedError(f"residual norm rows have at most {MAX_WIDTH} columns")
    return _gate_groups(gate, x)


def _scale(residual_scale) -> float:
    if type(residual_scale) not in (int, float) or not math.isfinite(residual_scale):
        raise ValueError("residual norm needs a finite residual_scale")
    return float(residual_scale)


def _eps(eps) -> float:
    if type(eps) not in (int, float) or not math.isfinite(eps) or eps <= 0:
        raise ValueError("residual norm needs a finite positive eps")
    return float(eps)


def _rows_of(t):
    """[rows, columns] of unit column stride."""
    flat, _, cols = _row_last_layout(t)
    if cols > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    return flat


def _variant(tensors, rows, n, after, gate_kind, backward) -> ResidualNormVariant:
    """Lanes and slots of a row."""
    size = tensors[0].element_size()
    vec = 16 // size
    aligned = n % vec == 0 and all(t.data_ptr() % 16 == 0 and (t.ndim == 1 or t.stride(0) * size % 16 == 0)
                                   for t in tensors)
    slots = -(-n // vec)
    nv = 1
    if not backward and slots >= 256 and rows >= 4 * CUS:
        nv = 2
    tpr = 1 << max(0, (-(-slots // nv) - 1).bit_length())
    while tpr > 1024:
        tpr, nv = tpr // 2, nv * 2
    wg = max(512 if backward else 256, tpr)
    return ResidualNormVariant(str(tensors[0].dtype).replace("torch.", ""), not aligned, tpr, nv, wg, after,
                               gate_kind)


def _gate_kind(groups, group) -> str:
    return "none" if not groups else "rows" if group == 1 else "group"


class _Forward:
    __slots__ = ("kernel", "grid", "rest", "device", "shape", "copied")

    def __init__(self, x, y, after, before, gate, groups, group, scale, eps):
        self.shape = x.shape
        given = (x, y, after, before, gate)
        flat = [_rows_of(x), _rows_of(y)] + [t.contiguous() if t is not None else None for t in given[2:]]
        self.copied = [f if f is not None and f.data_ptr() != t.data_ptr() else None for f, t in zip(flat, given)]
        fx, fy = flat[:2]
        rows, n = fx.shape
        var = _variant([t for t in flat if t is not None], rows, n, after is not None,
                       _gate_kind(groups, group), False)
        self.device = calls.device_index(x)
        self.kernel = _program("forward", var).kernel(residual_norm_kernel_name("forward", var), _FORWARD_ARGS,
                                                      var.wg, self.device)
        self.grid = (-(-rows // (var.wg // var.tpr)),)
        calls.check_grid(self.grid[0], var.wg, "residual norm")
        self.rest = (rows, n, fx.stride(0), fy.stride(0), max(group, 1), scale, eps)

    def run(self, x, y, after, before, gate, residual, normed, stats):
        x, y, after, before, gate = (
            0 if t is None else (c if c is not None else t).data_ptr()
            for c, t in zip(self.copied, (x, y, after, before, gate)))
        with calls.on_device(self.device):
            self.kernel.launch(self.grid, (x, y, gate, after, before, residual.data_ptr(), normed.data_ptr(),
                                           0 if stats is None else stats.data_ptr()) + self.rest,
                               hip.current_stream(self.device))


def run_residual_norm(x, y, gamma_after, gamma_before, *, gate=None, residual_scale: float = 1.0,
                      eps: float = 1e-6, return_stats: bool = False):
    """(residual, normed) of the module docstring on the current stream, and with `return_stats` the fp32
    [..., 2] rates 1/root-mean-square of y (1 without gamma_after) and of the residual, which
    run_residual_norm_backward takes.  A call whose tensor layouts and numbers were seen before reuses
    that call's kernel and launch shape."""
    import torch

    key = calls.tensors_key(x, y, gamma_after, gamma_before, gate)
    call = None
    if key is not None and type(residual_scale) in (int, float) and type(eps) in (int, float):
        key += ("forward", residual_scale, eps)
        call = _SEEN.get(key)
    else:
        key = None
    if call is None:
        metadata = isinstance(x, torch.Tensor) and calls.is_metadata(x)
        groups, group = validate_residual_norm_inputs(x, y, gamma_after, gamma_before, gate, metadata=metadata)
        scale, eps = _scale(residual_scale), _eps(eps)
        if not metadata and x.numel() != 0:
            call = _Forward(x, y, gamma_after, gamma_before, gate, groups, group, scale, eps)
            if key is not None and all(c is None for c in call.copied):
                _SEEN.keep(key, call)
    residual = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    normed = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((*x.shape[:-1], 2), dtype=torch.float32, device=x.device) if return_stats else None
    if call is not None:
        call.run(x, y, gamma_after, gamma_before, gate, residual, normed, stats)
    return (residual, normed, stats) if return_stats else (residual, normed)


def _chunks(rows, groups, group, gate_kind, rpw):
    """(chunks, rows or groups per chunk, chunks per group) of the gradient's launch: about one workgroup
    per CU; chunks of whole groups (0 per group) where there are more groups than that."""
    if gate_kind != "group":
        groups, group = 1, rows
    if groups > CUS:
        chunk = -(-groups // CUS)
        return -(-groups // chunk), chunk, 0
    per_group = max(1, min(CUS // groups, -(-group // rpw)))
    chunk = -(-(-(-group // per_group)) // rpw) * rpw
    per_group = -(-group // chunk)
    return groups * per_group, chunk, per_group


class _Backward:
    __slots__ = ("kernel", "join", "grid", "join_grid", "rest", "tail", "device", "floats", "copied", "shapes")

    def __init__(self, dres, dnormed, x, y, after, before, gate, groups, group, scale):
        given = (dres, dnormed, x, y, after, before, gate)
        flat = [None if t is None else _rows_of(t) for t in given[:4]]
        flat += [None if t is None else t.contiguous() for t in given[4:]]
        self.copied = [f if f is not None and f.data_ptr() != t.data_ptr() else None for f, t in zip(flat, given)]
        rows, n = flat[2].shape
        kind = _gate_kind(groups, group)
        var = _variant([t for t in flat if t is not None], rows, n, after is not None, kind, True)
        self.device = calls.device_index(x)
        prog = _program("backward", var)
        self.kernel = prog.kernel(residual_norm_kernel_name("backward", var), _BACKWARD_ARGS, var.wg, self.device)
        self.join = prog.kernel(residual_norm_kernel_name("join", var), _JOIN_ARGS, 256, self.device)
        chunks, chunk, per_group = _chunks(rows, groups, group, kind, var.wg // var.tpr)
        split_gate = kind == "group" and per_group > 1
        self.grid = (chunks,)
        self.join_grid = (-(-n // 32), 2 + (groups if split_gate else 0)) if chunks > 1 else None
        self.floats = (2 + split_gate) * chunks * n if chunks > 1 else 0
        strides = tuple(0 if t is None else t.stride(0) for t in flat[:4])
        self.rest = (rows, n) + strides + (group if kind == "group" else rows, chunk, per_group, scale)
        self.tail = (n, chunks, per_group)

    def run(self, given, stats, dx, dy, dgate, dafter, dbefore):
        import torch

        dres, dnormed, x, y, after, before, gate = (
            0 if t is None else (c if c is not None else t).data_ptr() for c, t in zip(self.copied, given))
        pointer = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        work = torch.empty(self.floats, dtype=torch.float32, device=dx.device) if self.floats else None
        with calls.on_device(self.device):
            stream = hip.current_stream(self.device)
            self.kernel.launch(self.grid, (dres, dnormed, x, y, gate, after, before, stats.data_ptr(),
                                           dx.data_ptr(), dy.data_ptr(), pointer(dgate), pointer(dafter),
                                           dbefore.data_ptr(), pointer(work)) + self.rest, stream)
            if self.join_grid is not None:
                self.join.launch(self.join_grid, (work.data_ptr(), pointer(dafter), dbefore.data_ptr(),
                                                  pointer(dgate)) + self.tail, stream)


def run_residual_norm_backward(grad_residual, grad_normed, x, y, gamma_after, gamma_before, stats, *,
                               gate=None, residual_scale: float = 1.0):
    """(dx, dy, dgamma_after, dgamma_before, dgate) of run_residual_norm's call with these x, y, gammas and
    gate, which returned `stats`; None in the place of an absent gamma_after or gate.  `grad_residual` may
    be None (a residual that nothing else reads).  Gradients have their operand's shape and dtype."""
    import torch

    given = (grad_residual, grad_normed, x, y, gamma_after, gamma_before, gate)
    key = calls.tensors_key(*given, stats)
    call = None
    if key is not None and type(residual_scale) in (int, float):
        key += ("backward", residual_scale)
        call = _SEEN.get(key)
    else:
        key = None
    metadata = False
    if call is None:
        metadata = isinstance(x, torch.Tensor) and calls.is_metadata(x)
        groups, group = validate_residual_norm_inputs(x, y, gamma_after, gamma_before, gate, metadata=metadata)
        for t, name in ((grad_normed, "grad_normed"), (grad_residual, "grad_residual")):
            if t is None and name == "grad_residual":
                continue
            calls.check_tensor(t, f"residual norm {name}", metadata=metadata)
            if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
                raise ValueError(f"residual norm {name} must have x's shape, dtype and device")
        calls.check_tensor(stats, "residual norm stats", metadata=metadata)
        if stats.shape != (*x.shape[:-1], 2) or stats.dtype != torch.float32 or stats.device != x.device:
            raise ValueError(f"residual norm stats must be float32 {(*x.shape[:-1], 2)} on x's device")
        scale = _scale(residual_scale)
    make = torch.zeros if x.numel() == 0 else torch.empty
    dx, dy, dafter, dbefore, dgate = (
        None if t is None else make(t.shape, dtype=t.dtype, device=t.device)
        for t in (x, y, gamma_after, gamma_before, gate))
    if call is None and not metadata and x.numel() != 0:
        call = _Backward(*given, groups, group, scale)
        if key is not None and all(c is None for c in call.copied) and stats.is_contiguous():
            _SEEN.keep(key, call)
        stats = stats.contiguous()
    if call is not None:
        call.run(given, stats, dx, dy, dgate, dafter, dbefore)
    return dx, dy, dafter, dbefore, dgate


def as_residual_norm_op(residual_scale: float = 1.0, eps: float = 1e-6, lib: str = "neptune"):
    """Differentiable custom op `(Tensor x, Tensor y, Tensor? gamma_after, Tensor gamma_before, Tensor? gate)
    -> (Tensor residual, Tensor normed, Tensor stats)` with the numbers in its name."""
    import torch

    from neptune_codegen.autotune import parameter_tag

    scale, eps = _scale(residual_scale), _eps(eps)
    key = (lib, scale, eps)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = f"residual_norm{parameter_tag({'scale': scale, 'eps': eps})}"

    def _forward(x, y, gamma_after, gamma_before, gate):
        return run_residual_norm(x, y, gamma_after, gamma_before, gate=gate, residual_scale=scale, eps=eps,
                                 return_stats=True)

    def _forward_fake(x, y, gamma_after, gamma_before, gate):
        validate_residual_norm_inputs(x, y, gamma_after, gamma_before, gate, metadata=True)
        return (torch.empty(x.shape, dtype=x.dtype, device=x.device),
                torch.empty(x.shape, dtype=x.dtype, device=x.device),
                torch.empty((*x.shape[:-1], 2), dtype=torch.float32, device=x.device))

    def _absent(x):
        return torch.empty((0,), dtype=x.dtype, device=x.device)

    def _backward(grad_residual, grad_normed, x, y, gamma_after, gamma_before, gate, stats):
        grads = run_residual_norm_backward(grad_residual, grad_normed, x, y, gamma_after, gamma_before, stats,
                                           gate=gate, residual_scale=scale)
        return tuple(_absent(x) if g is None else g for g in grads)

    def _backward_fake(grad_residual, grad_normed, x, y, gamma_after, gamma_before, gate, stats):
        return tuple(_absent(x) if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
                     for t in (x, y, gamma_after, gamma_before, gate))

    define = torch.library.custom_op
    op = define(f"{lib}::{name}", mutates_args=(),
                schema="(Tensor x, Tensor y, Tensor? gamma_after, Tensor gamma_before, Tensor? gate) "
                       "-> (Tensor, Tensor, Tensor)")(_forward)
    op.register_fake(_forward_fake)
    back = define(f"{lib}::{name}_backward", mutates_args=(),
                  schema="(Tensor? grad_residual, Tensor grad_normed, Tensor x, Tensor y, Tensor? gamma_after, "
                         "Tensor gamma_before, Tensor? gate, Tensor stats) "
                         "-> (Tensor, Tensor, Tensor, Tensor, Tensor)")(_backward)
    back.register_fake(_backward_fake)

    def _setup(ctx, inputs, output):
        x, y, gamma_after, gamma_before, gate = inputs
        ctx.save_for_backward(x, y, gamma_after, gamma_before, gate, output[2])
        ctx.mark_non_differentiable(output[2])
        ctx.set_materialize_grads(False)

    def _grad(ctx, grad_residual, grad_normed, _):
        x, y, gamma_after, gamma_before, gate, stats = ctx.saved_tensors
        if grad_residual is None and grad_normed is None:
            return (None,) * 5
        if grad_normed is None:
            grad_normed = torch.zeros_like(x)
        dx, dy, dafter, dbefore, dgate = back(grad_residual, grad_normed, x, y, gamma_after, gamma_before, gate,
                                              stats)
        return dx, dy, None if gamma_after is None else dafter, dbefore, None if gate is None else dgate

    op.register_autograd(_grad, setup_context=_setup)
    with _lock:
        _OPS[key] = op
    return op
