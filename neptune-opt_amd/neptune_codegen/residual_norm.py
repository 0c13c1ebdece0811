"""The norms after and before a block, fused with the block's gate and residual scale, and their
gradients.

There is no reference function for this path; it is run_rms_norm twice around the residual add:

    residual = x + residual_scale * gate * norm(y; gamma_after)     (the block's output y)
    normed   = norm(residual; gamma_before)                         (the next block's input)

with norm(v; gamma) = v * rsqrt(mean(v^2) + eps) * gamma over the last dimension.  gamma_after may be
None (y is added as it is), and so may the gate.  run_residual_norm_quantized returns normed in 8 bits
with scales, for an 8-bit matrix product.  Formulas and mapping are in
csrc/kernels/nep_residual_norm.h.

Layout contract: x and y [..., n] of one shape and dtype (float32, bfloat16, float16), n up to 16384;
gammas [n] of that dtype; a gate of x's shape, or with ones in its trailing leading dimensions (a gate
[batch, 1, n] for x [batch, tokens, n]), or [n].  Outputs are fresh and contiguous.  The arithmetic is
fp32 throughout with one rounding per output; normed is the norm of the residual before its rounding.
Column sums (gradients of the gammas and of a broadcast gate) are added in one order, without atomics.
"""
from __future__ import annotations

import dataclasses
import math
import threading

from neptune_codegen import calls, dispatch, hip
from neptune_codegen.emitters import (BASE_OPTIONS, ResidualNormVariant, emit_residual_norm_source,
                                      residual_norm_kernel_name)
from neptune_codegen.template import _validate_row_last

MAX_WIDTH = 16384
MAX_STRIDE = 1 << 22
CUS = 256
_PROGRAMS: dict = {}
_OPS: dict = {}
_FORWARD, _QUANTIZED, _BACKWARD = calls.Table(), calls.Table(), calls.Table()
_lock = threading.Lock()

_FORWARD_ARGS = (hip.PTR,) * 8 + (hip.I64, hip.I32) + (hip.I64,) * 3 + (hip.F32,) * 2
_QUANTIZED_ARGS = _FORWARD_ARGS + (hip.PTR,)
_BACKWARD_ARGS = (hip.PTR,) * 14 + (hip.I64, hip.I32) + (hip.I64,) * 6 + (hip.F32,)
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
    if type(residual_scale) not in (int, float) or not abs(residual_scale) <= calls.MOST_FLOAT:
        raise ValueError("residual norm needs a residual_scale that is finite in fp32")
    return float(residual_scale)


def _eps(eps) -> float:
    # (a smaller one would be 0 or a denormal in fp32, and a row of zeros NaN)
    if type(eps) not in (int, float) or not calls.LEAST_FLOAT <= eps <= calls.MOST_FLOAT:
        raise ValueError("residual norm needs a positive eps that is a normal number in fp32")
    return float(eps)


def _variant(x, aligned: bool, rows: int, n: int, after: bool, gate_kind: str, backward: bool) -> ResidualNormVariant:
    """Lanes and slots of a row.  The forward pass takes two slots a lane once the rows fill the chip (bf16
    16384 x 4096 93-95 us with one, two or four; 3000 x 3001 17 us, one 20).  The gradient takes one, on
    workgroups of 512 lanes (1024 would hold its state in 128 registers: bf16 16384 x 4096 gated by sequence
    174 us, 512 lanes 145; two slots on 256 lanes 209), or of 1024 where a row needs them; a 16-bit row of
    1025 to 1536 slots takes three on 512 lanes, whose state fits their 256 registers but for rows of any alignment
    with gamma_after and a group's gate, which spill 20 (fp16) and 26 (gated 16384 x 12288 541 us, 644 by two on 1024
    lanes; 1088 x 11100 81, 116; four spill: 16384 columns 245, 240).  On 1024 lanes with 128 registers the forms
    of one 16-byte slot fit but for 8192 16-bit columns with gamma_after and a gate (up to 23 spilled); of two and
    four most gated forms spill (fp32 8192 columns up to 52, 16384 up to 138): fp32 4096 x 8192 149 us bare, 250
    with gamma_after and a gate per sequence; 16-bit 8192 x 16384 288 and 408."""
    vec = 16 // x.element_size()
    slots = -(-n // vec)
    nv = 1
    if not backward and slots >= 256 and rows >= 4 * CUS:
        nv = 2
    tpr = 1 << max(0, (-(-slots // nv) - 1).bit_length())
    while tpr > 1024:
        tpr, nv = tpr // 2, nv * 2
    if backward and vec == 8 and 1024 < slots <= 1536:
        tpr, nv = 512, 3
    wg = max(512 if backward else 256, tpr)
    access = "few" if n < vec else "words" if aligned else "any"
    return ResidualNormVariant(str(x.dtype).replace("torch.", ""), access, tpr, nv, wg, after, gate_kind)


def _operands(rows, vectors, n):
    """(tensors, row strides, whether every row is whole 16-byte words): `rows` [..., n] as they are or as
    contiguous copies, `vectors` contiguous."""
    made = [(None, 0) if t is None else calls.rows_of(t) for t in rows]
    # (a wavefront's rows are addressed with 32-bit byte offsets from its first)
    made = [(t, s) if t is None or s < MAX_STRIDE else (t.contiguous(), n) for t, s in made]
    used = [t for t, _ in made] + [None if t is None else t.contiguous() for t in vectors]
    vec = 16 // used[-2].element_size()
    aligned = (n % vec == 0 and all(s % vec == 0 for _, s in made)
               and all(t is None or t.data_ptr() % 16 == 0 for t in used))
    return tuple(used), tuple(s for _, s in made), aligned


def _gate_kind(groups, group) -> str:
    return "none" if not groups else "rows" if group == 1 else "group"


def run_residual_norm(x, y, gamma_after, gamma_before, *, gate=None, residual_scale: float = 1.0,
                      eps: float = 1e-6, return_stats: bool = False):
    """(residual, normed) of the module docstring on the current stream, and with `return_stats` the fp32
    [..., 2] rates 1/root-mean-square of y (1 without gamma_after) and of the residual, which
    run_residual_norm_backward takes.  A call whose tensor layouts and numbers were seen before reuses
    that call's kernel and launch shape."""
    import torch

    given, return_stats = (x, y, gamma_after, gamma_before, gate), bool(return_stats)
    found = _FORWARD.run(given, (residual_scale, eps, return_stats))
    if found is not None:
        return found
    metadata = isinstance(x, torch.Tensor) and calls.is_metadata(x)
    groups, group = validate_residual_norm_inputs(*given, metadata=metadata)
    numbers, scale, eps = (residual_scale, eps, return_stats), _scale(residual_scale), _eps(eps)
    outputs = [(x.shape, x.dtype)] * 2 + ([((*x.shape[:-1], 2), torch.float32)] if return_stats else [])
    if metadata or x.numel() == 0:
        return tuple(torch.empty(shape, dtype=dtype, device=x.device) for shape, dtype in outputs)
    n = x.shape[-1]
    rows = x.numel() // n
    used, strides, aligned = _operands((x, y), (gamma_after, gamma_before, gate), n)
    var = _variant(x, aligned, rows, n, gamma_after is not None, _gate_kind(groups, group), False)
    device = calls.device_index(x)
    kernel = _program("forward", var).kernel(residual_norm_kernel_name("forward", var), _FORWARD_ARGS, var.wg, device)
    tx, ty, after, before, tgate = map(calls.tensor, range(5))
    launch = (kernel, (-(-rows // (var.wg // var.tpr)),),
              (tx, ty, tgate, after, before, calls.buffer(0), calls.buffer(1),
               calls.buffer(2) if return_stats else 0, rows, n) + strides + (max(group, 1), scale, eps))
    plan = calls.Plan(device, 5, outputs, range(len(outputs)), [launch])
    if calls.same(given, used):
        _FORWARD.keep(given, numbers, plan)
    return plan.run(used)


# columns that share a scale, and the number that stands for an 8-bit type in a call's key
BLOCKS = (32, 64, 128)
_FORMATS = ("float8_e4m3fn", "float8_e5m2", "int8")


_CODES: dict = {None: 0}     # of the types seen so far


def _format(dtype) -> str:
    import torch

    name = str(dtype).replace("torch.", "")
    if not isinstance(dtype, torch.dtype) or name not in _FORMATS:
        raise TypeError(f"residual norm's 8-bit outputs are {', '.join(_FORMATS)}, got {dtype}")
    _CODES[dtype] = _FORMATS.index(name)
    return name


def _block(group) -> int:
    if group is not None and (type(group) is not int or group not in BLOCKS):
        raise ValueError(f"residual norm's scales are one per row (None) or per {BLOCKS} columns, got {group!r}")
    return group or 0


def _quantized_variant(x, aligned: bool, rows: int, n: int, after: bool, gate_kind: str, out: str, block: int,
                       power_of_two: bool) -> ResidualNormVariant:
    """The forward pass's lanes, but where the rows fill the chip, the two to five slots a lane that leave the
    fewest lanes without columns (of equal ones the most slots).  With gamma_after and a gate per group, bf16 2464 x
    8773 36.6 us by five slots, 50.2 by two; 1568 x 12544 34.1 by four, 42.7; 16384 x 4095 101 by four, 118; fp16
    5331 x 2999 25.0 by three, 30.2; bf16 16384 x 4096 82.6 by four, 82.9 by two."""
    var = _variant(x, aligned, rows, n, after, gate_kind, False)
    slots = -(-n // (16 // x.element_size()))
    if rows >= 4 * CUS and slots >= 128:
        lanes = {nv: 1 << (-(-slots // nv) - 1).bit_length() for nv in (2, 3, 4, 5)}
        nv = min((nv for nv in lanes if lanes[nv] <= 1024), key=lambda k: (lanes[k] * k, -k))
        var = dataclasses.replace(var, tpr=lanes[nv], nv=nv, wg=max(256, lanes[nv]))
    return dataclasses.replace(var, out=out, block=block, power_of_two=power_of_two)


def _quantized_outputs(x, dtype, block: int, return_stats: bool):
    import torch

    blocks = -(-x.shape[-1] // block) if block else 1
    return [(x.shape, x.dtype), (x.shape, dtype), ((*x.shape[:-1], blocks), torch.float32)] + (
        [((*x.shape[:-1], 2), torch.float32)] if return_stats else [])


def run_residual_norm_quantized(x, y, gamma_after, gamma_before, *, gate=None, residual_scale: float = 1.0,
                                eps: float = 1e-6, dtype=None, group: int | None = None,
                                power_of_two: bool = False, return_stats: bool = False):
    """(residual, values, scales) on the current stream: run_residual_norm with the second result in 8 bits,
    for an 8-bit matrix product, normed ~ values * scales, and with `return_stats` the rates as a fourth (its row
    sums run in another order for some shapes).

    `dtype` is torch.float8_e4m3fn (the default), float8_e5m2 or int8; `scales` [..., 1] in fp32 has one number
    per row, or [..., ceil(n / group)] one per `group` (32, 64 or 128) columns: the largest magnitude over the
    type's largest value, or with `power_of_two` the least power of two that is no less, at least 2^-126 (0
    stays 0); values are rounded half to even.  Where a row or group holds an infinity or NaN, its scale is not
    finite.  The gradient is straight through: run_residual_norm_backward, with the rates."""
    given, return_stats, power_of_two = (x, y, gamma_after, gamma_before, gate), bool(return_stats), bool(power_of_two)
    numbers = (residual_scale, eps, return_stats, _CODES.get(dtype, ""), group, power_of_two)   # ("" has no key)
    found = _QUANTIZED.run(given, numbers)
    if found is not None:
        return found
    import torch

    dtype = torch.float8_e4m3fn if dtype is None else dtype
    out, block = _format(dtype), _block(group)
    numbers = (residual_scale, eps, return_stats, _CODES[dtype], group, power_of_two)
    metadata = isinstance(x, torch.Tensor) and calls.is_metadata(x)
    groups, group_rows = validate_residual_norm_inputs(*given, metadata=metadata)
    scale, eps = _scale(residual_scale), _eps(eps)
    outputs = _quantized_outputs(x, dtype, block, return_stats)
    if metadata or x.numel() == 0:
        return tuple(torch.empty(shape, dtype=kind, device=x.device) for shape, kind in outputs)
    n = x.shape[-1]
    rows = x.numel() // n
    used, strides, aligned = _operands((x, y), (gamma_after, gamma_before, gate), n)
    var = _quantized_variant(x, aligned, rows, n, gamma_after is not None, _gate_kind(groups, group_rows), out, block,
                             power_of_two)
    device = calls.device_index(x)
    kernel = _program("quantized", var).kernel(residual_norm_kernel_name("quantized", var), _QUANTIZED_ARGS, var.wg,
                                               device)
    tx, ty, after, before, tgate = map(calls.tensor, range(5))
    launch = (kernel, (-(-rows // (var.wg // var.tpr)),),
              (tx, ty, tgate, after, before, calls.buffer(0), calls.buffer(1),
               calls.buffer(3) if return_stats else 0, rows, n) + strides
              + (max(group_rows, 1), scale, eps, calls.buffer(2)))
    plan = calls.Plan(device, 5, outputs, range(len(outputs)), [launch])
    if calls.same(given, used):
        _QUANTIZED.keep(given, numbers, plan)
    return plan.run(used)


@dispatch.one_at_a_time
def as_residual_norm_quantized_op(residual_scale: float = 1.0, eps: float = 1e-6, dtype=None,
                                  group: int | None = None, power_of_two: bool = False, lib: str = "neptune"):
    """Custom op `(Tensor x, Tensor y, Tensor? gamma_after, Tensor gamma_before, Tensor? gate) -> (Tensor
    residual, Tensor values, Tensor scales, Tensor stats)` with the numbers in its name.  Its 8-bit results have
    no gradient in torch: a differentiable product calls run_residual_norm_backward with the stats."""
    import torch

    from neptune_codegen.autotune import parameter_tag

    scale, eps, block, power_of_two = _scale(residual_scale), _eps(eps), _block(group), bool(power_of_two)
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    out = _format(dtype)
    key = (lib, scale, eps, out, block, power_of_two)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = (f"residual_norm_{out}_{f'blocks{block}' if block else 'rows'}{'_powers' if power_of_two else ''}"
            f"{parameter_tag({'scale': scale, 'eps': eps})}")

    def _forward(x, y, gamma_after, gamma_before, gate):
        return run_residual_norm_quantized(x, y, gamma_after, gamma_before, gate=gate, residual_scale=scale, eps=eps,
                                           dtype=dtype, group=group, power_of_two=power_of_two, return_stats=True)

    def _forward_fake(x, y, gamma_after, gamma_before, gate):
        validate_residual_norm_inputs(x, y, gamma_after, gamma_before, gate, metadata=True)
        return tuple(torch.empty(shape, dtype=kind, device=x.device)
                     for shape, kind in _quantized_outputs(x, dtype, block, True))

    op = torch.library.custom_op(
        f"{lib}::{name}", mutates_args=(),
        schema="(Tensor x, Tensor y, Tensor? gamma_after, Tensor gamma_before, Tensor? gate) "
               "-> (Tensor, Tensor, Tensor, Tensor)")(_forward)
    op.register_fake(_forward_fake)
    with _lock:
        _OPS[key] = op
    return op


def _chunks(rows, groups, group, gate_kind, rpw):
    """(workgroups, workgroups per group) of the gradient's launch: one per CU, or fewer where their partial
    sums would cost more than the rows (a row takes a workgroup about 1.7 us, a partial row 0.03 us to write and
    join: bf16 256 x 4096 18 us with 256 workgroups, 15 with 128; 16384 x 4096 148 with 256, 157-176 with 512); 0 per group
    where there are more groups than workgroups and each takes whole ones."""
    if gate_kind != "group":
        groups, group = 1, rows
    most = min(CUS, math.isqrt(64 * -(-rows // rpw)) + 1)
    if groups > most:
        return most, 0
    per_group = max(1, min(most // groups, -(-group // rpw)))
    return groups * per_group, per_group


def run_residual_norm_backward(grad_residual, grad_normed, x, y, gamma_after, gamma_before, stats, *,
                               gate=None, residual_scale: float = 1.0):
    """(dx, dy, dgamma_after, dgamma_before, dgate) of run_residual_norm's call with these x, y, gammas and
    gate, which returned `stats`; None in the place of an absent gamma_after or gate.  `grad_residual` may
    be None (a residual that nothing else reads).  Gradients have their operand's shape and dtype."""
    import torch

    given = (grad_residual, grad_normed, x, y, gamma_after, gamma_before, gate, stats)
    found = _BACKWARD.run(given, (residual_scale,))
    if found is not None:
        return found
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
    wanted = (x, y, gamma_after, gamma_before, gate)
    if metadata or x.numel() == 0:
        return tuple(None if t is None else torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in wanted)
    n = x.shape[-1]
    rows = x.numel() // n
    used, strides, aligned = _operands((grad_residual, grad_normed, x, y), (gamma_after, gamma_before, gate), n)
    used += (stats.contiguous(),)
    kind = _gate_kind(groups, group)
    var = _variant(x, aligned, rows, n, gamma_after is not None, kind, True)
    device, prog = calls.device_index(x), _program("backward", var)
    chunks, per_group = _chunks(rows, groups, group, kind, var.wg // var.tpr)
    split_gate = kind == "group" and per_group > 1
    buffers, returns = [], []
    for t in wanted:
        returns.append(None if t is None else len(buffers))
        if t is not None:
            buffers.append((t.shape, t.dtype))
    dx, dy, dafter, dbefore, dgate = (0 if r is None else calls.buffer(r) for r in returns)
    work = 0
    if chunks > 1:
        work = calls.buffer(len(buffers))
        buffers.append((((2 + split_gate) * chunks * n,), torch.float32))
    dres, dnormed, tx, ty, after, before, tgate, tstats = map(calls.tensor, range(8))
    launches = [(prog.kernel(residual_norm_kernel_name("backward", var), _BACKWARD_ARGS, var.wg, device), (chunks,),
                 (dres, dnormed, tx, ty, tgate, after, before, tstats, dx, dy, dgate, dafter, dbefore, work, rows, n)
                 + strides + (group if kind == "group" else rows, per_group, scale))]
    if chunks > 1:
        launches.append((prog.kernel(residual_norm_kernel_name("join", var), _JOIN_ARGS, 256, device),
                         (-(-n // 32), 2 + (groups if split_gate else 0)),
                         (work, dafter, dbefore, dgate, n, chunks, per_group)))
    plan = calls.Plan(device, 8, buffers, returns, launches)
    if calls.same(given, used):
        _BACKWARD.keep(given, (residual_scale,), plan)
    return plan.run(used)


@dispatch.one_at_a_time
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
