"""Gradients of the attention fold (attention.py): dQ, dK and dV of O = softmax(scale * Q K^T
[+ causal mask]) V, from the output and logsumexp that the forward pass returned.

There is no reference function for this path (the reference has no attention and no gradients).
The probabilities are recomputed from the logsumexp, P = exp(scale * Q K^T - lse); formulas,
mapping and roundings are in csrc/kernels/nep_attention_bwd.h.  Results are deterministic: no
kernel adds with atomics.

Layout contract: that of run_attention for q, k and v; the output and its gradient have q's shape,
dtype and device, any strides; lse is fp32 [B, H, Sq].  Fresh contiguous gradients of the input
dtype.

A pair hidden by the causal mask contributes nothing whatever it holds: an infinity or NaN in Q, K,
V or dO reaches only the gradients whose formula has it.
"""
from __future__ import annotations

import functools
import math
import threading

from neptune_codegen import calls, hip
from neptune_codegen.attention import K_ROW_STRIDE_MAX, LOG2E, validate_attention_inputs
from neptune_codegen.emitters import (ATTN_BWD_TILE, ATTN_BWD_WAVES, BASE_OPTIONS,
                                      attention_backward_blocks, attention_backward_kernel_name,
                                      emit_attention_backward_source)

_PROGRAMS: dict = {}
_KERNELS: dict = {}
_OPS: dict = {}
_TABLE = calls.Table()
_lock = threading.Lock()

_ROWS_ARGS = (hip.PTR,) * 10 + (hip.I32,) * 4 + (hip.I64,) * 15 + (hip.F32,) * 2 + (hip.I32,)
_OPERAND_ARGS = (hip.I32,) * 4 + (hip.I64,) * 12 + (hip.F32,) * 2 + (hip.I32,)
_KVQ_ARGS = (hip.PTR,) * 12 + _OPERAND_ARGS + (hip.I32,) * 2
_THREADS = 64 * ATTN_BWD_WAVES
_JOIN_ARGS = (hip.PTR,) * 3 + (hip.I64,) + (hip.I32,) * 5


def _program(stage, head_dim, causal, dtype, blocks=1, parts=False) -> hip.Program:
    causal = bool(causal) and stage != "rows"        # one unit for both masks
    key = (stage, head_dim, causal, str(dtype).replace("torch.", ""), blocks, parts)
    with _lock:
        prog = _PROGRAMS.get(key)
        if prog is None:
            name = attention_backward_kernel_name(stage, head_dim, causal, dtype, blocks, parts)
            prog = _PROGRAMS[key] = hip.Program(
                emit_attention_backward_source(stage, head_dim, causal, dtype, blocks, parts),
                f"{name}.hip", BASE_OPTIONS)
        return prog


def unit_kinds(head_dim):
    """(stage, blocks per wave, parts) of the units a call at this head dim may launch."""
    yield "rows", 1, False
    for blocks in range(1, attention_backward_blocks(head_dim) + 1):
        yield "kvq", blocks, False
        yield "kvq", blocks, True


def _kernel(stage, device, head_dim, causal, dtype, blocks=1, parts=False) -> hip.Kernel:
    key = (stage, device, head_dim, causal, dtype, blocks, parts)
    found = _KERNELS.get(key)
    if found is None:
        args, threads = {"rows": (_ROWS_ARGS, 256), "kvq": (_KVQ_ARGS, _THREADS),
                         "kv_join": (_JOIN_ARGS, 256), "q_join": (_JOIN_ARGS, 256)}[stage]
        prog = _program("rows" if stage.endswith("join") else stage, head_dim, causal, dtype, blocks, parts)
        found = _KERNELS[key] = prog.kernel(
            attention_backward_kernel_name(stage, head_dim, causal, dtype, blocks, parts), args, threads, device)
    return found


def validate_attention_backward_inputs(grad, q, k, v, out, lse, grad_lse=None, *, metadata: bool = False):
    import torch

    for t, name in ((grad, "grad"), (q, "q"), (k, "k"), (v, "v"), (out, "out"), (lse, "lse")):
        calls.check_tensor(t, f"attention backward {name}", metadata=metadata)
    shape = validate_attention_inputs(q, k, v, metadata=metadata)
    for t, name in ((grad, "grad"), (out, "out")):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"attention backward {name} must have q's shape, dtype and device, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")
    for t, name in ((lse, "lse"), (grad_lse, "grad_lse")):
        if t is None:
            continue
        calls.check_tensor(t, f"attention backward {name}", metadata=metadata)
        if t.shape != q.shape[:3] or t.dtype != torch.float32 or t.device != q.device:
            raise ValueError(f"attention backward {name} must be float32 {tuple(q.shape[:3])} on q's "
                             f"device, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return shape


def _scale(scale, head_dim: int = 64) -> float:
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    # (the kernels hold lse / scale in fp32)
    if not 2.0 ** -100 <= scale <= calls.MOST_FLOAT:
        raise ValueError("attention scale must be finite and positive, from 2^-100 to 2^125")
    return scale


def _operand(t):
    """(t, or its contiguous copy where a kernel cannot read its rows; batch, head, row strides).
    Rows that overlap (an expanded sequence) are copied too: a tile's rows past the end must read as
    zero."""
    sb, sh, ss, sd = t.stride()
    if t.shape[2] == 1:
        ss = t.shape[3]                              # one row has any stride
    if not (sd == 1 and sb % 8 == 0 and sh % 8 == 0 and ss % 8 == 0 and t.shape[3] <= ss < K_ROW_STRIDE_MAX
            and t.data_ptr() % 16 == 0):
        t = t.contiguous()
        sb, sh, ss, _ = t.stride()
    return t, (sb, sh, ss)


# What `_plan` prices a launch with, in us on MI355X (fits of timings over 34 shapes; of the plans within 1.5 times its
# price the chosen one is within 4% of the fastest in 33 of them, and 10% in causal 1x8x2000x256): a workgroup's
# pass over a 64-row tile with few workgroups on the chip, and a CU's with the chip full (the clock and
# the caches are shared; head dim 64 has two or three workgroups on a CU); and a workgroup's start and end, without
# the mask and with it (its waves then wait for each other on the diagonal).
TILE_US = {("kv", 64, 1): (1.0, 0.9, 4.0, 4.0), ("q", 64, 1): (1.0, 0.82, 3.0, 3.0),
           ("kv", 128, 1): (1.6, 1.7, 7.0, 8.0), ("q", 128, 1): (1.45, 1.45, 7.0, 8.0),
           ("kv", 128, 2): (2.9, 3.07, 11.0, 22.0), ("q", 128, 2): (2.4, 2.45, 11.5, 19.0),
           ("kv", 256, 1): (3.3, 3.57, 12.0, 12.0), ("q", 256, 1): (2.4, 2.62, 8.0, 8.0)}
# A split's further launch and its fp32 sums, written and read (through the caches).
JOIN_US, SUM_BYTES_PER_US, MAX_SUM_BYTES = 4.0, 7e6, 256 << 20
CUS = 256
PARTS = (1, 2, 3, 4, 6, 8, 12, 16, 24, 32)


def _stage_work(stage, units, own, other, head_dim, causal, blocks, per):
    """(items, tiles, longest item's tiles, bytes of split sums) of a stage with blocks of `own` rows
    walking the tiles of the `other` rows in parts of `per`."""
    step = ATTN_BWD_WAVES * blocks // 2              # tiles of a block's own rows
    rows = step * ATTN_BWD_TILE
    count, tiles = -(-own // rows), -(-other // ATTN_BWD_TILE)
    width = head_dim * (2 if stage == "kv" else 1)
    items = total = longest = sums = 0
    for i in range(count):
        n = tiles if not causal else max(0, tiles - step * i) if stage == "kv" else min(tiles, step * (i + 1))
        m = count if not causal else 1
        parts = max(1, -(-n // per))
        items, total, longest = items + m * parts, total + m * n, max(longest, min(n, per))
        sums += m * parts * rows * width * 8 if parts > 1 else 0
        if not causal:
            break
    return units * items, units * total, longest, units * sums


def _launch_cost(works, head_dim, causal, blocks):
    """us of the launch of both stages, {stage: _stage_work(...)} in their order, and of the joins of what it
    splits."""
    items = sum(w[0] for w in works.values())
    busy = longest = joins = last = 0.0
    for stage, (n, tiles, most, sums) in works.items():
        few, full, *ends = TILE_US[stage, head_dim, blocks]
        # head dim 64: a CU's workgroups take turns
        tile = 1.7 * full if head_dim == 64 and items > CUS else few
        last = most * tile + ends[causal]
        late, longest = last > longest, max(longest, last)
        busy += (tiles * full + n * ends[causal]) / CUS
        joins += JOIN_US + sums / SUM_BYTES_PER_US if sums else 0.0
    if items <= CUS:
        return longest + joins
    # the heaviest of a stage start first; what ends last is short, unless the second stage's are longer
    return max(longest, busy + longest / (2 if late else 4 if causal else 8)) + joins


@functools.lru_cache(maxsize=4096)
def _plan_tiles(units, q_tiles, k_tiles, head_dim, causal):
    sq, sk, best = q_tiles * ATTN_BWD_TILE, k_tiles * ATTN_BWD_TILE, None
    for blocks in range(1, attention_backward_blocks(head_dim) + 1):
        found = {}
        for stage, own, other in (("kv", sk, sq), ("q", sq, sk)):
            width, tiles = head_dim * (2 if stage == "kv" else 1), other // ATTN_BWD_TILE
            found[stage] = [(p, _stage_work(stage, units, own, other, head_dim, causal, blocks, -(-tiles // p)))
                            for p in PARTS
                            if p == 1 or p <= tiles // 2 and 4 * p * units * own * width <= MAX_SUM_BYTES]
        cheapest = min((_launch_cost({"kv": kv, "q": q}, head_dim, causal, blocks), blocks, i, j)
                       for i, kv in found["kv"] for j, q in found["q"])
        best = cheapest if best is None else min(best, cheapest)
    return best[1:]


def _plan(units, sq, sk, head_dim, causal):
    """(blocks per wave, kv parts, q parts) of a call, the cheapest by TILE_US; searched once for the same
    tile counts.  Two blocks a wave (head dim 128) read each tile half as often and pass twice the rows
    in 1.7 to 1.8 times the time, with a longer start and end: bf16 causal 4x32x4096x128 1858 us by two,
    2055 by one; full 2x16x4096x128 770 and 876, 8x32x1024x128 476 and 566; but causal 8x32x1024x128 395 and
    383, 2x8x300x128 39 and 22."""
    return _plan_tiles(units, -(-sq // ATTN_BWD_TILE), -(-sk // ATTN_BWD_TILE), head_dim, causal)


def _call_plan(q, k, strides, grad_lse, scale, causal, plan=None) -> calls.Plan:
    """Launches of a call; its tensors are (grad, q, k, v, out, lse, grad_lse)."""
    import torch

    B, H, Sq, D = q.shape
    Sk, units, device = k.shape[2], B * H, calls.device_index(q)
    blocks, kv_parts, q_parts = plan or _plan(units, Sq, Sk, D, causal)
    nq, nk = -(-Sq // ATTN_BWD_TILE), -(-Sk // ATTN_BWD_TILE)
    kv_per, q_per = -(-nq // kv_parts), -(-nk // q_parts)
    kv_parts, q_parts = -(-nq // kv_per), -(-nk // q_per)
    rows = 32 * ATTN_BWD_WAVES * blocks              # of a workgroup
    kind = (device, D, causal, q.dtype)
    # scratch: start values and deltas of every padded query row; fp16's bounds; the parts' fp32 sums
    stats = 4 * units * nq * ATTN_BWD_TILE
    bounds = -(-4 * units * (2 * nq + nk) // 256) * 256
    kv_sums = 8 * kv_parts * units * Sk * D if kv_parts > 1 else 0
    sums = kv_sums + (4 * q_parts * units * Sq * D if q_parts > 1 else 0)
    buffers = [(q.shape, q.dtype), (k.shape, q.dtype), (k.shape, q.dtype),
               ((2 * stats + bounds + sums,), torch.uint8)]
    grad, tq, tk, tv, out, lse, glse = map(calls.tensor, range(7))
    dq, dk, dv = map(calls.buffer, range(3))
    start, ndelta, limit, part = (calls.buffer(3, o) for o in (0, stats, 2 * stats, 2 * stats + bounds))
    qs, ks, vs, gs, os = strides
    sizes, steps = (units, H, Sq, Sk), qs + ks + vs + gs + (scale, scale * LOG2E)
    few = nq if Sk <= ATTN_BWD_TILE else int(causal)     # tiles of rows that see at most a tile of keys
    groups = units * (nq + (nk if q.dtype == torch.float16 else 0) + few)
    kv_groups, q_groups = units * kv_parts * -(-Sk // rows), units * q_parts * -(-Sq // rows)
    qpart = calls.buffer(3, 2 * stats + bounds + kv_sums)
    launches = [
        (_kernel("rows", *kind), (groups,),
         (tq, tk, out, grad, tv, lse, 0 if grad_lse is None else glse, start, ndelta, limit, H, Sq, Sk, units)
         + qs + ks + os + gs + vs + (scale, scale * LOG2E, int(causal))),
        (_kernel("kvq", *kind, blocks, kv_parts > 1 or q_parts > 1), (kv_groups + q_groups,),
         (tq, tk, tv, grad, start, ndelta, limit, dk, dv, dq, part, qpart) + sizes + steps
         + (kv_per, q_per, kv_groups))]
    if kv_parts > 1:
        launches.append((_kernel("kv_join", *kind), (-(-units * 2 * Sk * D // 1024),),
                         (part, dk, dv, units * Sk, Sk, Sq, rows, kv_per, int(causal))))
    if q_parts > 1:
        launches.append((_kernel("q_join", *kind), (-(-units * Sq * D // 1024),),
                         (qpart, dq, 0, units * Sq, Sq, Sk, rows, q_per, int(causal))))
    return calls.Plan(device, 7, buffers, (0, 1, 2), launches)


def run_attention_backward(grad, q, k, v, out, lse, *, grad_lse=None, scale: float | None = None,
                           causal: bool = True):
    """(dq, dk, dv) of run_attention(q, k, v, scale=scale, causal=causal, return_lse=True) for the
    gradient `grad` of its output (and `grad_lse` of its logsumexp), on the current stream.  `out`
    and `lse` are what that call returned.  See the module docstring for the contract.  A call whose
    tensor layouts and options were seen before reuses that call's kernels and launch shapes."""
    causal = bool(causal)
    found = _TABLE.run((grad, q, k, v, out, lse, grad_lse), (scale, causal))
    if found is not None:
        return found
    return _run(grad, q, k, v, out, lse, grad_lse, scale, causal)


def _run(grad, q, k, v, out, lse, grad_lse, scale, causal, plan=None):
    import torch

    metadata = isinstance(q, torch.Tensor) and calls.is_metadata(q)
    validate_attention_backward_inputs(grad, q, k, v, out, lse, grad_lse, metadata=metadata)
    given, number = (grad, q, k, v, out, lse, grad_lse), scale
    scale = _scale(scale, q.shape[3])
    if metadata or q.numel() == 0:
        # without a query nothing reaches the keys
        return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
                torch.zeros(k.shape, dtype=k.dtype, device=k.device),
                torch.zeros(v.shape, dtype=v.dtype, device=v.device))
    (grad, gs), (q, qs), (k, ks), (v, vs), (out, os) = map(_operand, given[:5])
    lse = lse.contiguous()
    grad_lse = grad_lse.contiguous() if grad_lse is not None else None
    used = (grad, q, k, v, out, lse, grad_lse)
    call = _call_plan(q, k, (qs, ks, vs, gs, os), grad_lse, scale, causal, plan)
    if plan is None and calls.same(given, used):
        _TABLE.keep(given, (number, causal), call)
    return call.run(used)


def as_attention_grad_op(scale: float | None = None, causal: bool = True, lib: str = "neptune"):
    """Differentiable custom op `(Tensor q, Tensor k, Tensor v) -> (Tensor out, Tensor lse)` with
    scale and mask in its name: run_attention with its logsumexp, and run_attention_backward for
    both outputs' gradients."""
    import torch

    from neptune_codegen.attention import run_attention
    from neptune_codegen.autotune import parameter_tag

    params = {"scale": _scale(scale)} if scale is not None else {}
    causal = bool(causal)
    key = (lib, tuple(sorted(params.items())), causal)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = f"attention_grad_fold{parameter_tag(params)}_{'causal' if causal else 'full'}"

    def _forward(q, k, v):
        return run_attention(q, k, v, scale=scale, causal=causal, return_lse=True)

    def _forward_fake(q, k, v):
        validate_attention_inputs(q, k, v, metadata=True)
        return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
                torch.empty(q.shape[:3], dtype=torch.float32, device=q.device))

    def _backward(grad, grad_lse, q, k, v, out, lse):
        return run_attention_backward(grad, q, k, v, out, lse, grad_lse=grad_lse, scale=scale, causal=causal)

    def _backward_fake(grad, grad_lse, q, k, v, out, lse):
        validate_attention_backward_inputs(grad, q, k, v, out, lse, grad_lse, metadata=True)
        return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))

    define = torch.library.custom_op
    op = define(f"{lib}::{name}", mutates_args=(),
                schema="(Tensor q, Tensor k, Tensor v) -> (Tensor, Tensor)")(_forward)
    op.register_fake(_forward_fake)
    back = define(f"{lib}::{name}_backward", mutates_args=(),
                  schema="(Tensor grad, Tensor? grad_lse, Tensor q, Tensor k, Tensor v, Tensor out, "
                         "Tensor lse) -> (Tensor, Tensor, Tensor)")(_backward)
    back.register_fake(_backward_fake)

    def _setup(ctx, inputs, output):
        ctx.save_for_backward(*inputs, *output)
        ctx.set_materialize_grads(False)

    def _grad(ctx, grad, grad_lse):
        q, k, v, out, lse = ctx.saved_tensors
        if grad is None and grad_lse is None:
            return None, None, None
        if grad is None:
            grad = torch.zeros_like(out)
        return back(grad, grad_lse, q, k, v, out, lse)

    op.register_autograd(_grad, setup_context=_setup)
    with _lock:
        _OPS[key] = op
    return op
