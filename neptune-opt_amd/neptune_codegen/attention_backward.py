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

import math
import threading

from neptune_codegen import calls, hip
from neptune_codegen.attention import K_ROW_STRIDE_MAX, LOG2E, validate_attention_inputs
from neptune_codegen.emitters import (ATTN_BWD_TILE, ATTN_BWD_WAVES, BASE_OPTIONS,
                                      attention_backward_blocks, attention_backward_kernel_names,
                                      emit_attention_backward_source)

_PROGRAMS: dict = {}
_KERNELS: dict = {}
_OPS: dict = {}
_SEEN = calls.Seen()
_lock = threading.Lock()

_ROWS_ARGS = (hip.PTR,) * 8 + (hip.I32,) * 4 + (hip.I64,) * 9 + (hip.F32,)
_OPERAND_ARGS = (hip.I32,) * 4 + (hip.I64,) * 12 + (hip.F32,) * 2 + (hip.I32,) * 2
_KV_ARGS = (hip.PTR,) * 10 + _OPERAND_ARGS
_Q_ARGS = (hip.PTR,) * 9 + _OPERAND_ARGS
_THREADS = 64 * ATTN_BWD_WAVES
_JOIN_ARGS = (hip.PTR,) * 3 + (hip.I64, hip.I32)


def _program(head_dim, causal, dtype, kv_blocks=1, q_blocks=1, kv_parts=False, q_parts=False) -> hip.Program:
    key = (head_dim, causal, str(dtype).replace("torch.", ""), kv_blocks, q_blocks, kv_parts, q_parts)
    with _lock:
        prog = _PROGRAMS.get(key)
        if prog is None:
            source = emit_attention_backward_source(head_dim, causal, dtype, kv_blocks, q_blocks,
                                                    kv_parts, q_parts)
            name = attention_backward_kernel_names(head_dim, causal, dtype, kv_blocks, q_blocks,
                                                   kv_parts, q_parts)["kv"]
            prog = _PROGRAMS[key] = hip.Program(source, f"{name}_{q_blocks}{'p' if q_parts else ''}.hip",
                                                BASE_OPTIONS)
        return prog


def _kernels(device, head_dim, causal, dtype, kv_blocks, q_blocks, kv_parts, q_parts) -> tuple:
    """(rows, kv, q, kv join or None, q join or None), fetched once per device."""
    key = (device, head_dim, causal, dtype, kv_blocks, q_blocks, kv_parts, q_parts)
    found = _KERNELS.get(key)
    if found is None:
        prog = _program(head_dim, causal, dtype, kv_blocks, q_blocks, kv_parts, q_parts)
        names = attention_backward_kernel_names(head_dim, causal, dtype, kv_blocks, q_blocks, kv_parts,
                                                q_parts)
        found = (prog.kernel(names["rows"], _ROWS_ARGS, 256, device),
                 prog.kernel(names["kv"], _KV_ARGS, _THREADS, device),
                 prog.kernel(names["q"], _Q_ARGS, _THREADS, device),
                 prog.kernel(names["kv_join"], _JOIN_ARGS, 256, device) if kv_parts else None,
                 prog.kernel(names["q_join"], _JOIN_ARGS, 256, device) if q_parts else None)
        _KERNELS[key] = found
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


def _operand(t):
    """(t, or its contiguous copy where a kernel cannot read its rows; batch, head, row strides).
    Rows that overlap (an expanded sequence) are copied too: a tile's rows past the end must read as
    zero."""
    sb, sh, ss, sd = t.stride()
    if not (sd == 1 and sb % 8 == 0 and sh % 8 == 0 and ss % 8 == 0 and ss < K_ROW_STRIDE_MAX
            and (ss >= t.shape[3] or t.shape[2] == 1) and t.data_ptr() % 16 == 0):
        t = t.contiguous()
        sb, sh, ss, _ = t.stride()
    return t, (sb, sh, ss)


class _Call:
    """The launches of one call layout: kernels, grids and the arguments that are not pointers."""

    __slots__ = ("device", "q_shape", "k_shape", "nbytes", "offsets", "sums", "rows", "kv", "q",
                 "kv_join", "q_join")

    def run(self, grad, q, k, v, out, lse, grad_lse, dq, dk, dv):
        import torch

        work = torch.empty(self.nbytes, dtype=torch.uint8, device=q.device)
        base = work.data_ptr()
        start, ndelta, bounds, sums = (base + o for o in self.offsets)
        pq, pk, pv, pg = q.data_ptr(), k.data_ptr(), v.data_ptr(), grad.data_ptr()
        with calls.on_device(self.device):
            stream = hip.current_stream(self.device)
            kernel, grid, rest = self.rows
            kernel.launch(grid, (out.data_ptr(), pg, pv, lse.data_ptr(),
                                 0 if grad_lse is None else grad_lse.data_ptr(), start, ndelta, bounds)
                          + rest, stream)
            kernel, grid, rest = self.kv
            kernel.launch(grid, (pq, pk, pv, pg, start, ndelta, bounds, dk.data_ptr(), dv.data_ptr(), sums)
                          + rest, stream)
            if self.kv_join is not None:
                kernel, grid, rest = self.kv_join
                kernel.launch(grid, (sums, dk.data_ptr(), dv.data_ptr()) + rest, stream)
            kernel, grid, rest = self.q
            kernel.launch(grid, (pq, pk, pv, pg, start, ndelta, bounds, dq.data_ptr(), sums) + rest, stream)
            if self.q_join is not None:
                kernel, grid, rest = self.q_join
                kernel.launch(grid, (sums, dq.data_ptr(), 0) + rest, stream)


def _plan(units, sq, sk, head_dim, causal):
    """(kv blocks, kv parts, q blocks, q parts) of a call."""
    b = attention_backward_blocks(head_dim)
    return b, 1, b, 1


def _prepare(q, k, strides, scale, causal, plan=None) -> _Call:
    import torch

    B, H, Sq, D = q.shape
    Sk, units, device = k.shape[2], B * H, calls.device_index(q)
    kv_blocks, kv_parts, q_blocks, q_parts = plan or _plan(units, Sq, Sk, D, causal)
    nq, nk = -(-Sq // ATTN_BWD_TILE), -(-Sk // ATTN_BWD_TILE)
    kv_per, q_per = -(-nq // kv_parts), -(-nk // q_parts)
    kv_parts, q_parts = -(-nq // kv_per), -(-nk // q_per)
    rows, kv, q_kernel, kv_join, q_join = _kernels(device, D, causal, q.dtype, kv_blocks, q_blocks,
                                                   kv_parts > 1, q_parts > 1)
    call = _Call()
    call.device = device
    # start values and deltas of every padded query row; fp16's bounds; the parts' fp32 sums
    stats = 4 * units * nq * ATTN_BWD_TILE
    bounds = -(-4 * units * (2 * nq + nk) // 256) * 256
    sums = max(8 * kv_parts * units * Sk * D if kv_parts > 1 else 0,
               4 * q_parts * units * Sq * D if q_parts > 1 else 0)
    call.offsets = (0, stats, 2 * stats, 2 * stats + bounds)
    call.nbytes = 2 * stats + bounds + sums
    qs, ks, vs, gs, os = strides
    groups = units * (nq + (nk if q.dtype == torch.float16 else 0))
    kv_groups = units * kv_parts * -(-Sk // (32 * ATTN_BWD_WAVES * kv_blocks))
    q_groups = units * q_parts * -(-Sq // (32 * ATTN_BWD_WAVES * q_blocks))
    join = tuple(-(-units * n * D // 1024) for n in (2 * Sk, Sq))
    for n, threads in ((groups, 256), (kv_groups, _THREADS), (q_groups, _THREADS),
                       (max(join), 256)):
        calls.check_grid(n, threads, "attention backward")
    call.rows = (rows, (groups,), (H, Sq, Sk, units) + os + gs + vs + (scale,))
    tail = (units, H, Sq, Sk) + qs + ks + vs + gs + (scale, scale * LOG2E)
    call.kv = (kv, (kv_groups,), tail + (kv_parts, kv_per))
    call.q = (q_kernel, (q_groups,), tail + (q_parts, q_per))
    call.kv_join = (kv_join, (join[0],), (units * Sk, kv_parts)) if kv_parts > 1 else None
    call.q_join = (q_join, (join[1],), (units * Sq, q_parts)) if q_parts > 1 else None
    return call


def run_attention_backward(grad, q, k, v, out, lse, *, grad_lse=None, scale: float | None = None,
                           causal: bool = True):
    """(dq, dk, dv) of run_attention(q, k, v, scale=scale, causal=causal, return_lse=True) for the
    gradient `grad` of its output (and `grad_lse` of its logsumexp), on the current stream.  `out`
    and `lse` are what that call returned.  See the module docstring for the contract.  A call whose
    tensor layouts and options were seen before reuses that call's kernels and launch shapes."""
    key = call = None
    if scale is None or type(scale) in (int, float):
        key = calls.tensors_key(grad, q, k, v, out, lse, grad_lse)
    if key is not None:
        key += (type(scale), scale, bool(causal))
        call = _SEEN.get(key)
    return _run(grad, q, k, v, out, lse, grad_lse, scale, causal, key, call)


def _run(grad, q, k, v, out, lse, grad_lse, scale, causal, key=None, call=None, plan=None):
    import torch

    if call is None:
        metadata = isinstance(q, torch.Tensor) and calls.is_metadata(q)
        validate_attention_backward_inputs(grad, q, k, v, out, lse, grad_lse, metadata=metadata)
        scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
        if not math.isfinite(scale) or scale <= 0:
            raise ValueError("attention scale must be finite and positive")
        if metadata or q.numel() == 0:
            # without a query nothing reaches the keys
            return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
                    torch.zeros(k.shape, dtype=k.dtype, device=k.device),
                    torch.zeros(v.shape, dtype=v.dtype, device=v.device))
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if call is None:
        given = (q, k, v, grad, out, lse, grad_lse)
        (q, qs), (k, ks), (v, vs), (grad, gs), (out, os) = map(_operand, given[:5])
        lse = lse.contiguous()
        grad_lse = grad_lse.contiguous() if grad_lse is not None else None
        call = _prepare(q, k, (qs, ks, vs, gs, os), scale, bool(causal), plan)
        if key is not None and all(a is b for a, b in zip(given, (q, k, v, grad, out, lse, grad_lse))):
            _SEEN.keep(key, call)
    call.run(grad, q, k, v, out, lse, grad_lse, dq, dk, dv)
    return dq, dk, dv


def as_attention_grad_op(scale: float | None = None, causal: bool = True, lib: str = "neptune"):
    """Differentiable custom op `(Tensor q, Tensor k, Tensor v) -> (Tensor out, Tensor lse)` with
    scale and mask in its name: run_attention with its logsumexp, and run_attention_backward for
    both outputs' gradients."""
    import torch

    from neptune_codegen.attention import run_attention
    from neptune_codegen.autotune import parameter_tag

    params = {"scale": float(scale)} if scale is not None else {}
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
