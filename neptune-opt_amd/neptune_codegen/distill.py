"""Distillation from a teacher's top logits: loss and gradient.

There is no reference function for this path; the row state is the logsumexp fold's (max, sum of
exponentials).  Per row of student logits z, with temperature T and the teacher's list (t_k, i_k):

    p = softmax(t / T) over the list's entries with i_k >= 0,   q = softmax(z / T)
    loss = T^2 sum_k p_k (log p_k - log q_{i_k}),   dloss/dz_i = T (q_i - sum of p_k with i_k = i)

Layout contract: logits [..., n] in float32, bfloat16 or float16; top_logits [..., k] in float32 or the
logits' dtype and top_index [..., k] in int32 or int64, with the same leading sizes, 1 <= k <= 1024.  A
negative index marks an absent entry (lists may differ in length); a list without an entry has loss 0
and gradient 0; an index of n or more makes its row's loss and gradient NaN.  Loss and state are fp32,
the gradient has the logits' dtype.  Edge values (infinities, repeated indices) are described in
csrc/kernels/nep_distill.h.
"""
from __future__ import annotations

import math
import threading

from neptune_codegen import calls, hip
from neptune_codegen.emitters import (BASE_OPTIONS, DistillVariant, distill_kernel_name,
                                      emit_distill_source)
from neptune_codegen.template import _validate_row_last

MAX_ENTRIES = 1024
_PROGRAMS: dict = {}
_OPS: dict = {}
_FORWARD, _BACKWARD = calls.Table(), calls.Table()
_lock = threading.Lock()

_FORWARD_ARGS = (hip.PTR,) * 5 + (hip.I64,) * 5 + (hip.I32,) + (hip.F32,) * 3
_BACKWARD_ARGS = (hip.PTR,) * 6 + (hip.I64,) * 6 + (hip.I32,) + (hip.F32,) * 2 + (hip.I64,)


def _program(stage: str, var: DistillVariant) -> hip.Program:
    with _lock:
        prog = _PROGRAMS.get((stage, var))
        if prog is None:
            prog = _PROGRAMS[stage, var] = hip.Program(
                emit_distill_source(stage, var), f"{distill_kernel_name(stage, var)}.hip", BASE_OPTIONS)
        return prog


def _temperature(temperature) -> float:
    # (its square and its reciprocal are fp32 numbers)
    if type(temperature) not in (int, float) or not 1e-18 <= temperature <= 1e18:
        raise ValueError("distillation needs a temperature from 1e-18 to 1e18")
    return float(temperature)


def validate_distill_inputs(logits, top_logits, top_index, *, metadata: bool = False):
    """Leading sizes of a call."""
    import torch

    for t, name in ((logits, "logits"), (top_logits, "top_logits"), (top_index, "top_index")):
        calls.check_tensor(t, f"distillation {name}", metadata=metadata)
    _validate_row_last(logits, metadata=metadata)
    lead = logits.shape[:-1]
    if top_logits.ndim != logits.ndim or top_logits.shape[:-1] != lead:
        raise ValueError(f"distillation top_logits {tuple(top_logits.shape)} must have the leading sizes of "
                         f"the logits {tuple(logits.shape)}")
    if top_index.shape != top_logits.shape:
        raise ValueError(f"distillation top_index {tuple(top_index.shape)} must have the shape of top_logits "
                         f"{tuple(top_logits.shape)}")
    if top_logits.dtype not in (torch.float32, logits.dtype):
        raise TypeError(f"distillation top_logits must be float32 or the logits' dtype, got {top_logits.dtype}")
    if top_index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"distillation top_index must be int32 or int64, got {top_index.dtype}")
    if top_logits.device != logits.device or top_index.device != logits.device:
        raise ValueError("distillation tensors must be on the same device")
    if not 1 <= top_logits.shape[-1] <= MAX_ENTRIES:
        raise NotImplementedError(f"distillation takes lists of 1 to {MAX_ENTRIES} entries")
    if logits.shape[-1] >= 1 << 28:
        raise NotImplementedError("distillation takes rows of less than 2^28 logits")
    return lead


def _check_rows(t, name, shape, logits, *, metadata):
    import torch

    calls.check_tensor(t, f"distillation {name}", metadata=metadata)
    if t.shape != shape or t.dtype != torch.float32 or t.device != logits.device:
        raise ValueError(f"distillation {name} must be float32 {tuple(shape)} on the logits' device, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _variant(z, stride: int, top, index, rows: int, n: int, count: int, stage: str) -> DistillVariant:
    """Lanes per row and 16-byte slots a lane has in flight.

    Forward: a wavefront up to 512 slots (16384 rows of 4096 bf16: 27 us, 37 with 256 lanes) and, where the
    rows fill the chip with wavefronts, up to 1536 (8192 rows of 10007: 32 us, 36); 256 lanes beyond (16384
    rows of 32000: 151 us, 164 with 512, 201 with 1024), 1024 where 512 rows or fewer would leave CUs idle
    (64 rows of 128256: 11 us, 13.4 with 256).  Eight slots in flight where a CU has four workgroups (7168
    rows of 32003: 73.5 us, 77.1 with four), four below (600 rows of 50000: 15.7 us, 17.4).
    Backward, which reads and writes and so wants few rows open at once: a wavefront up to 256 slots (16384
    rows of 1000: 20.4 us, 24.6 with 128), 256 lanes up to 2048 (16384 rows of 4096: 58 us, 67 with a
    wavefront), 1024 beyond (16384 rows of 32000: 368 us, 392 with 256; fp32 4096 rows of 32000: 176, 190).
    A tile of lanes x slots is never wider than the row (16384 rows of 32000 by 1024 lanes take 355 us with
    two slots, 442 with four), and half as wide where a wavefront or 256 lanes that write hold a row, for the
    next tile's loads (4096 columns, forward 27.4 us with four slots, 28.7 with eight; backward 61.7 with one,
    64.1 with two); a row of up to two slots a lane is one tile (16384 rows of 1000: 12.0 us, 13.1)."""
    vec = 16 // z.element_size()
    slots = -(-n // vec)
    aligned = n % vec == 0 and z.data_ptr() % 16 == 0 and stride % vec == 0
    if stage == "forward":
        alone = 1536 if rows >= 4096 else 512
        tpr = 64 if slots <= alone and count <= 256 else 1024 if rows <= 512 and slots > 1024 else 256
        most = 8 if rows >= 1024 else 4
    else:
        parts = _column_parts(rows, slots)
        tpr = 64 if slots <= 256 and count <= 256 else 256 if slots < 2048 or parts > 1 else 1024
        most, slots = 4, -(-slots // parts)
    half = tpr == (64 if stage == "forward" else 256)
    unroll, widest = 1, slots // 2 if half else slots
    while unroll < most and tpr * unroll * 2 <= widest:
        unroll *= 2
    if stage == "forward" and tpr < slots <= 2 * tpr:
        unroll = 2
    entries = 1
    while entries * tpr < count:
        entries *= 2
    name = lambda t: str(t.dtype).replace("torch.", "")  # noqa: E731
    return DistillVariant(name(z), name(top), name(index), not aligned, tpr, unroll, entries)


def _column_parts(rows: int, slots: int) -> int:
    """Parts of a row's columns in the gradient, where rows alone leave CUs idle: eight workgroups of 256
    lanes for each CU, of a slot a lane at least.  bf16 64 rows of 128256 11.9 us, 18.7 whole; one row 5.6, 11.1;
    500 of 50257 23.7, 26.1; fp32 7 of 181248 6.8, 26.0; from 512 rows on nothing is gained."""
    return max(1, min(slots // 256, 2048 // rows)) if rows < 512 and slots > 1024 else 1


def _launch(stage, z, top, index, strides, args, ends):
    """(kernel, grid, arguments) of a stage; `args` are its pointers, `ends` what follows the strides."""
    rows, n, count = z.numel() // z.shape[-1], z.shape[-1], top.shape[-1]
    var = _variant(z, strides[-3], top, index, rows, n, count, stage)
    kernel = _program(stage, var).kernel(distill_kernel_name(stage, var),
                                         _FORWARD_ARGS if stage == "forward" else _BACKWARD_ARGS,
                                         var.wg, calls.device_index(z))
    grid = (-(-rows // var.rows),)
    if stage == "backward":
        vec = 16 // z.element_size()
        per = -(-n // (64 * vec * _column_parts(rows, -(-n // vec)))) * 64 * vec
        grid, ends = grid + (-(-n // per),), ends + (per,)
    return kernel, grid, args + (rows, n) + strides + (count,) + ends


def run_distill(logits, top_logits, top_index, *, temperature: float = 1.0, return_stats: bool = False):
    """Loss [...] of each row in fp32, and with `return_stats` the state [..., 2] (max, sum of
    exponentials) that run_distill_backward takes, on the current stream.  A call whose tensor layouts
    and temperature were seen before reuses that call's kernel and launch shape."""
    import torch

    given, return_stats = (logits, top_logits, top_index), bool(return_stats)
    found = _FORWARD.run(given, (temperature, return_stats))
    if found is not None:
        return found
    metadata = isinstance(logits, torch.Tensor) and calls.is_metadata(logits)
    lead = validate_distill_inputs(*given, metadata=metadata)
    number, temperature = temperature, _temperature(temperature)
    outputs = [(lead, torch.float32)] + ([((*lead, 2), torch.float32)] if return_stats else [])
    if metadata or logits.numel() == 0:
        made = tuple(torch.empty(shape, dtype=dtype, device=logits.device) for shape, dtype in outputs)
        return made if return_stats else made[0]
    (z, sz), (t, st), (i, si) = map(calls.rows_of, given)
    stats = calls.buffer(1) if return_stats else 0
    launch = _launch("forward", z, t, i, (sz, st, si),
                     (calls.tensor(0), calls.tensor(1), calls.tensor(2), calls.buffer(0), stats),
                     (math.log2(math.e) / temperature, 1.0 / temperature, temperature * temperature))
    plan = calls.Plan(calls.device_index(z), 3, outputs, range(len(outputs)), [launch], bare=not return_stats)
    if calls.same(given, (z, t, i)):
        _FORWARD.keep(given, (number, return_stats), plan)
    return plan.run((z, t, i))


def run_distill_backward(grad, logits, top_logits, top_index, stats, *, temperature: float = 1.0):
    """Gradient [..., n] of the logits, in their dtype, for the losses' gradient `grad` [...] in fp32 and
    the state that run_distill returned; fresh and contiguous."""
    import torch

    given = (grad, logits, top_logits, top_index, stats)
    found = _BACKWARD.run(given, (temperature,))
    if found is not None:
        return found
    metadata = isinstance(logits, torch.Tensor) and calls.is_metadata(logits)
    lead = validate_distill_inputs(logits, top_logits, top_index, metadata=metadata)
    _check_rows(grad, "grad", lead, logits, metadata=metadata)
    _check_rows(stats, "stats", (*lead, 2), logits, metadata=metadata)
    number, temperature = temperature, _temperature(temperature)
    if metadata or logits.numel() == 0:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    (z, sz), (t, st), (i, si) = map(calls.rows_of, given[1:4])
    # the rows' gradients have one stride where that can be (a mean's is 0)
    g, sg = calls.rows_of(grad.unsqueeze(-1))
    used = (grad if g.data_ptr() == grad.data_ptr() else g, z, t, i, stats.contiguous())
    launch = _launch("backward", z, t, i, (sg, sz, st, si),
                     (calls.tensor(0), calls.tensor(1), calls.tensor(2), calls.tensor(3), calls.tensor(4),
                      calls.buffer(0)), (math.log2(math.e) / temperature, temperature))
    plan = calls.Plan(calls.device_index(z), 5, [(logits.shape, logits.dtype)], (0,), [launch], bare=True)
    if calls.same(given, used):
        _BACKWARD.keep(given, (number,), plan)
    return plan.run(used)


def as_distill_op(temperature: float = 1.0, lib: str = "neptune"):
    """Differentiable custom op `(Tensor logits, Tensor top_logits, Tensor top_index) -> (Tensor loss,
    Tensor stats)` with the temperature in its name; the gradient is the logits'."""
    import torch

    from neptune_codegen.autotune import parameter_tag

    temperature = _temperature(temperature)
    key = (lib, temperature)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = f"distill{parameter_tag({'t': temperature})}"

    def _forward(logits, top_logits, top_index):
        return run_distill(logits, top_logits, top_index, temperature=temperature, return_stats=True)

    def _forward_fake(logits, top_logits, top_index):
        lead = validate_distill_inputs(logits, top_logits, top_index, metadata=True)
        return (torch.empty(lead, dtype=torch.float32, device=logits.device),
                torch.empty((*lead, 2), dtype=torch.float32, device=logits.device))

    def _backward(grad, logits, top_logits, top_index, stats):
        return run_distill_backward(grad, logits, top_logits, top_index, stats, temperature=temperature)

    def _backward_fake(grad, logits, top_logits, top_index, stats):
        validate_distill_inputs(logits, top_logits, top_index, metadata=True)
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)

    define = torch.library.custom_op
    op = define(f"{lib}::{name}", mutates_args=(),
                schema="(Tensor logits, Tensor top_logits, Tensor top_index) -> (Tensor, Tensor)")(_forward)
    op.register_fake(_forward_fake)
    back = define(f"{lib}::{name}_backward", mutates_args=(),
                  schema="(Tensor grad, Tensor logits, Tensor top_logits, Tensor top_index, Tensor stats) "
                         "-> Tensor")(_backward)
    back.register_fake(_backward_fake)

    def _setup(ctx, inputs, output):
        loss, stats = output
        ctx.save_for_backward(*inputs, stats)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)

    def _grad(ctx, grad, _):
        if grad is None:
            return None, None, None
        return back(grad, *ctx.saved_tensors), None, None

    op.register_autograd(_grad, setup_context=_setup)
    with _lock:
        _OPS[key] = op
    return op
