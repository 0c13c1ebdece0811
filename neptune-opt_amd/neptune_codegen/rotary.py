"""Rotary positions of attention's queries and keys, and their gradients.

There is no reference function for this path.  In attention's layout [batch, heads, seq, dim], pair i
of the first `part` elements of each head is turned by 2 pi * position * turns[i]; the other elements
are copied.  Pairs are (i, i + part/2), or with `interleaved` (2i, 2i + 1).  `turns` is a float64 tensor
[part/2] on the device (turns per position), which `rotary_frequencies` makes, also scaled for contexts
longer than those of training; `magnitude` multiplies the turned elements.  Angles are 64-bit products
reduced to a quarter turn, so far positions keep their precision (csrc/kernels/nep_rotary.h).

Layout contract: q and k of one dtype (float32, bfloat16, float16), batch, seq and dim, with their own
numbers of heads; k may be None; any strides (a copy where the last dimension's is not one).  positions is
int32 or int64, [seq] or [batch, seq].  Outputs are fresh and contiguous.
"""
from __future__ import annotations

import math
import threading

from neptune_codegen import calls, dispatch, hip
from neptune_codegen.emitters import BASE_OPTIONS, emit_rotary_source, rotary_kernel_name

_PROGRAMS: dict = {}
_OPS: dict = {}
_TABLE = calls.Table()
_lock = threading.Lock()
_ARGS = (hip.PTR,) * 6 + (hip.I32,) * 9 + (hip.I64,) * 8 + (hip.F32,) * 2


def rotary_frequencies(part: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int | None = None, slow: float = 1.0, fast: float = 32.0, device="cuda"):
    """(turns, magnitude) for `part` rotated elements: pair i turns base^(-2i/part) radians per position.

    scaling for contexts `factor` times as long as training's:
      "linear"  every rate divided by the factor
      "ntk"     the base raised to base * factor^(part / (part - 2)): the slowest pair slows by the factor,
                the fastest keeps its rate
      "parts"   pairs that turn more than `fast` times within `original_length` positions keep their rate,
                those below `slow` turns are slowed by the factor, with a linear ramp between;
                magnitude 0.1 ln(factor) + 1
    """
    import torch

    if type(part) is not int or part < 2 or part % 2:
        raise ValueError("rotary part must be a positive even number of elements")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("rotary base must be finite and positive")
    if scaling not in ("none", "linear", "ntk", "parts"):
        raise ValueError(f"unknown rotary scaling {scaling!r}; expected 'none', 'linear', 'ntk' or 'parts'")
    if not (math.isfinite(factor) and factor >= 1.0) or (scaling == "none" and factor != 1.0):
        raise ValueError("rotary factor must be finite, at least 1, and 1 without scaling")
    magnitude = 1.0
    if scaling == "ntk":
        if part == 2:
            raise ValueError("rotary scaling 'ntk' needs more than one pair")
        base = base * factor ** (part / (part - 2))
    rates = [base ** (-2.0 * i / part) for i in range(part // 2)]
    if scaling == "linear":
        rates = [r / factor for r in rates]
    elif scaling == "parts":
        if original_length is None or original_length <= 0 or not 0 <= slow < fast:
            raise ValueError("rotary scaling 'parts' needs original_length and 0 <= slow < fast")
        kept = [min(1.0, max(0.0, (original_length * r / (2 * math.pi) - slow) / (fast - slow))) for r in rates]
        rates = [r * (g + (1.0 - g) / factor) for r, g in zip(rates, kept)]
        magnitude = 0.1 * math.log(factor) + 1.0
    turns = torch.tensor([r / (2 * math.pi) for r in rates], dtype=torch.float64, device=device)
    return turns, magnitude


def _program(dtype, index, layout, any_rows) -> hip.Program:
    key = (str(dtype).replace("torch.", ""), index, layout, any_rows)
    with _lock:
        prog = _PROGRAMS.get(key)
        if prog is None:
            prog = _PROGRAMS[key] = hip.Program(emit_rotary_source(*key), f"{rotary_kernel_name(*key)}.hip",
                                                BASE_OPTIONS)
        return prog


def validate_rotary_inputs(q, k, positions, turns, *, metadata: bool = False) -> None:
    import torch

    for t, name in ((q, "q"), (k, "k"), (positions, "positions"), (turns, "turns")):
        if t is not None or name != "k":
            calls.check_tensor(t, f"rotary {name}", metadata=metadata)
            if t.device != q.device:
                raise ValueError("rotary tensors must be on the same device")
    for t, name in ((q, "q"), (k, "k")):
        if t is None:
            continue
        if t.ndim != 4:
            raise ValueError(f"rotary {name} must be [batch, heads, seq, dim]")
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"rotary takes float32, bfloat16 and float16, got {t.dtype} for {name}")
    if k is not None and (k.dtype != q.dtype or (k.shape[0], *k.shape[2:]) != (q.shape[0], *q.shape[2:])):
        raise ValueError(f"rotary q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must share dtype, "
                         "batch, seq and dim")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"rotary positions must be int32 or int64, got {positions.dtype}")
    if positions.shape not in ((q.shape[2],), (q.shape[0], q.shape[2])):
        raise ValueError(f"rotary positions {tuple(positions.shape)} must be [seq] or [batch, seq] of q "
                         f"{tuple(q.shape)}")
    if turns.dtype != torch.float64 or turns.ndim != 1:
        raise TypeError("rotary turns must be a float64 vector (rotary_frequencies)")
    if not 1 <= turns.shape[0] <= q.shape[3] // 2:
        raise ValueError(f"rotary turns of {turns.shape[0]} pairs do not fit heads of {q.shape[3]} elements")


def _heads_per_lane(tokens, slots, heads):
    """Heads per lane: as many as leave 2^18 lanes (four wavefronts for each SIMD of 256 CUs), up to 16.
    More heads share a lane's angles; few tokens need the lanes.  bf16, 4 x 4096 tokens of 32 + 32 heads
    of 128: 96.7 us by 16, 100.9 by 8, 109 by 4; 64 tokens of 32 + 8 heads: 5.4 us by 4, 6.2 by 8."""
    per = 16
    while per > 1 and tokens * slots * -(-heads // per) < 1 << 18:
        per //= 2
    return per


def _run(q, k, positions, turns, magnitude, interleaved, sign):
    import torch

    given, interleaved = (q, k, positions, turns), bool(interleaved)
    found = _TABLE.run(given, (magnitude, interleaved, sign))
    if found is not None:
        return found
    metadata = isinstance(q, torch.Tensor) and calls.is_metadata(q)
    validate_rotary_inputs(*given, metadata=metadata)
    if type(magnitude) not in (int, float) or not abs(magnitude) <= calls.MOST_FLOAT:
        raise ValueError("rotary magnitude must be a number that is finite in fp32")
    if metadata or not (q.numel() or (k is not None and k.numel())):
        return tuple(None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    used = tuple(t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous() for t in (q, k))
    used += (positions, turns.contiguous())
    (batch, heads_q, seq, dim), heads_k = q.shape, k.shape[1] if k is not None else 0
    part, vec = 2 * turns.shape[0], 16 // q.element_size()
    run = part if interleaved else part // 2
    any_rows = bool(dim % vec or run % vec or (dim - part) % vec
                    or any(t is not None and (t.data_ptr() % 16 or any(s % vec for s in t.stride()[:3]))
                           for t in used[:2]))
    turned, rest = -(-run // vec), -(-(dim - part) // vec)
    layout, slots = "pairs" if interleaved else "halves", turned + rest
    # one slot a lane and an exchange within a pair, or both slots: bf16 8 x 2048 tokens of 16 + 16 heads of 100
    # 43 and 80 us, of 96 42 and 61; 4 x 4096 of 32 + 32 heads of 128 95 and 105, 32 + 8 heads 64 of 128 59
    # and 66; (16 + 8 heads, 128 of 256, 75 and 71).  The lanes of a half, and of a token, are a power of two,
    # so that its pairs are in one wavefront.
    lane_run = 2 * (1 << (turned - 1).bit_length())
    lanes = 1 << (lane_run + rest - 1).bit_length()
    if not interleaved and run >= vec and lanes <= 64:
        layout, slots, turned = "exchanged", lanes, lane_run
    heads, tokens = heads_q + heads_k, batch * seq
    if tokens >= 1 << 31:
        raise NotImplementedError("rotary takes less than 2^31 tokens")
    per = _heads_per_lane(tokens, slots, heads)
    device, index = calls.device_index(q), "int32" if positions.dtype == torch.int32 else "int64"
    kernel = _program(q.dtype, index, layout, any_rows).kernel(
        rotary_kernel_name(q.dtype, index, layout, any_rows), _ARGS, 256, device)
    strides = used[0].stride()[:3] + (used[1].stride()[:3] if k is not None else (0, 0, 0))
    strides += (positions.stride(0) if positions.ndim == 2 else 0, positions.stride(-1))
    out = [calls.buffer(0), 0 if k is None else calls.buffer(1)]
    launch = (kernel, (-(-tokens * slots // 256), -(-heads // per)),
              (*map(calls.tensor, range(4)), *out, tokens, seq, dim, part, slots, turned, heads_q, heads_k, per)
              + strides + (sign, float(magnitude)))
    plan = calls.Plan(device, 4, [(t.shape, t.dtype) for t in (q, k) if t is not None],
                      (0, None if k is None else 1), [launch])
    if calls.same(given, used):
        _TABLE.keep(given, (magnitude, interleaved, sign), plan)
    return plan.run(used)


def run_rotary(q, k, positions, turns, *, magnitude: float = 1.0, interleaved: bool = False):
    """(q, k) at their rotary positions, on the current stream (None for a k of None); see the module
    docstring for the contract.  A call whose tensor layouts and numbers were seen before reuses that call's
    kernel and launch shape."""
    return _run(q, k, positions, turns, magnitude, interleaved, 1.0)


def run_rotary_backward(grad_q, grad_k, positions, turns, *, magnitude: float = 1.0, interleaved: bool = False):
    """(dq, dk) of run_rotary for its outputs' gradients: the transposed rotation, by the negative angles."""
    return _run(grad_q, grad_k, positions, turns, magnitude, interleaved, -1.0)


@dispatch.one_at_a_time
def as_rotary_op(magnitude: float = 1.0, interleaved: bool = False, lib: str = "neptune"):
    """Differentiable custom op `(Tensor q, Tensor k, Tensor positions, Tensor turns) -> (Tensor, Tensor)`
    with the magnitude and the layout in its name (a k of no heads stands for none)."""
    import torch

    from neptune_codegen.autotune import parameter_tag

    if type(magnitude) not in (int, float) or not abs(magnitude) <= calls.MOST_FLOAT:
        raise ValueError("rotary magnitude must be a number that is finite in fp32")
    magnitude, interleaved = float(magnitude), bool(interleaved)
    key = (lib, magnitude, interleaved)
    with _lock:
        if key in _OPS:
            return _OPS[key]
    name = f"rotary{parameter_tag({'m': magnitude})}_{'pairs' if interleaved else 'halves'}"

    def body(run):
        def _impl(q, k, positions, turns):
            return run(q, k, positions, turns, magnitude=magnitude, interleaved=interleaved)
        return _impl

    def _fake(q, k, positions, turns):
        validate_rotary_inputs(q, k, positions, turns, metadata=True)
        return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))

    schema = "(Tensor q, Tensor k, Tensor positions, Tensor turns) -> (Tensor, Tensor)"
    define = torch.library.custom_op
    op = define(f"{lib}::{name}", mutates_args=(), schema=schema)(body(run_rotary))
    back = define(f"{lib}::{name}_backward", mutates_args=(), schema=schema)(body(run_rotary_backward))
    op.register_fake(_fake)
    back.register_fake(_fake)

    def _setup(ctx, inputs, output):
        ctx.save_for_backward(*inputs[2:])

    def _grad(ctx, grad_q, grad_k):
        return (*back(grad_q, grad_k, *ctx.saved_tensors), None, None)

    op.register_autograd(_grad, setup_context=_setup)
    with _lock:
        _OPS[key] = op
    return op
