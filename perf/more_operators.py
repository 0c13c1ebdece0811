"""Performance cases of the operators at the two ends of a training step and between its blocks: the
embedding lookup and its gradient, the residual norm with an 8-bit output, and the norm and clipping of
all gradients.

`listed()` names twelve of them, from calls of a few kilobytes to passes of 1.6 GB; `draw()` makes more of
the same ranges.  `run` computes a case in elementary torch operations in 32 bits, or, where `own` is set,
with the framework's kernels; `exact` has the same results in 64 bits.
"""
from __future__ import annotations

import math
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "neptune-opt_amd"))

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
          "int32": torch.int32, "int64": torch.int64,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2, "int32": 4, "int64": 8}
# largest value, bits behind the point and exponent of the smallest normal number
FORMATS = {"e4m3": (448.0, 3, -6), "e5m2": (57344.0, 2, -14)}
EPS = 1e-6
LEAST_SCALE = 2.0 ** -126
MOST_BYTES = 1.0e9           # of a drawn case


def listed() -> list[dict]:
    return [
        # one generated token for each of 64 sequences, a large vocabulary
        {"name": "embedding_token", "kind": "embedding", "dtype": "bf16", "index": "int64", "batch": 64,
         "seq": 1, "vocab": 128256, "ncols": 4096, "scaled": False, "backward": False},
        # a training batch of 16384 tokens, embeddings scaled by the root of their width
        {"name": "embedding_batch", "kind": "embedding", "dtype": "bf16", "index": "int64", "batch": 8,
         "seq": 2048, "vocab": 32000, "ncols": 4096, "scaled": True, "backward": False},
        # gradient of two short prompts in a small model
        {"name": "embedding_backward_small", "kind": "embedding", "dtype": "fp32", "index": "int64",
         "batch": 2, "seq": 77, "vocab": 1000, "ncols": 768, "scaled": False, "backward": True},
        # a training batch's gradient over a large vocabulary (1.05 GB, most of it rows without a token)
        {"name": "embedding_backward_vocab", "kind": "embedding", "dtype": "bf16", "index": "int64",
         "batch": 8, "seq": 2048, "vocab": 128256, "ncols": 4096, "scaled": False, "backward": True},
        # more tokens than vocabulary, odd sizes
        {"name": "embedding_backward_odd", "kind": "embedding", "dtype": "fp16", "index": "int32",
         "batch": 31, "seq": 1777, "vocab": 32003, "ncols": 1001, "scaled": True, "backward": True},
        # one generated token for each of 8 sequences, between two blocks, for an 8-bit product
        {"name": "norm8_token", "kind": "norm8", "dtype": "bf16", "format": "e4m3", "batch": 8, "seq": 1,
         "ncols": 1024, "group": 0, "power_of_two": False, "after": False, "gate": "none",
         "residual_scale": 1.0, "stats": False},
        # a training batch of 16384 tokens, one scale per token, statistics for the gradient
        {"name": "norm8_batch", "kind": "norm8", "dtype": "bf16", "format": "e4m3", "batch": 8, "seq": 2048,
         "ncols": 4096, "group": 0, "power_of_two": False, "after": True, "gate": "sequence",
         "residual_scale": 0.5, "stats": True},
        # blocks of 32 with powers of two for scales, an odd width
        {"name": "norm8_blocks_odd", "kind": "norm8", "dtype": "fp16", "format": "e5m2", "batch": 3,
         "seq": 1777, "ncols": 2999, "group": 32, "power_of_two": True, "after": True, "gate": "none",
         "residual_scale": 1.0, "stats": False},
        # the gradients of a model with 290 parameters (0.9 GB), norms' parameters in 32 bits
        {"name": "gradient_norm_model", "kind": "gradients", "dtype": "bf16", "layers": 32, "width": 1024,
         "hidden": 2816, "vocab": 32000, "clip": "no"},
        # a small model's whole gradient in 32 bits, below the bound: nothing is to be scaled
        {"name": "clip_small", "kind": "gradients", "dtype": "fp32", "layers": 2, "width": 64,
         "hidden": 172, "vocab": 501, "clip": "below"},
        # 16-bit gradients scaled into an optimizer's 32-bit buffers
        {"name": "clip_model", "kind": "gradients", "dtype": "bf16", "layers": 4, "width": 2048,
         "hidden": 5632, "vocab": 32000, "clip": "into fp32"},
        # fp16 gradients of odd sizes scaled into buffers of their own type
        {"name": "clip_odd", "kind": "gradients", "dtype": "fp16", "layers": 6, "width": 777,
         "hidden": 2001, "vocab": 10007, "clip": "into"},
    ]


# ---------------------------------------------------------------- drawn cases
def _log_int(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo: int, hi: int, unit: int) -> int:
    """Half the widths are multiples of `unit`, half are any number."""
    w = _log_int(rng, lo, hi)
    return max(unit, w // unit * unit) if rng.random() < 0.5 else w


def draw(rng) -> dict:
    kind = rng.choice(["embedding", "embedding", "embedding", "norm8", "norm8", "gradients", "gradients"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = SIZE[dtype]
    if kind == "embedding":
        ncols, backward = _width(rng, 16, 16384, 64), rng.random() < 0.6
        vocab = _width(rng, 64, max(64.0, min(200000.0, MOST_BYTES / (size * ncols))), 64)
        batch = _log_int(rng, 1, 64)
        most = max(1.0, min(65536.0, (MOST_BYTES - size * ncols * vocab * backward) / (2.0 * size * ncols)) / batch)
        return {"kind": kind, "dtype": dtype, "index": rng.choice(["int32", "int64"]), "batch": batch,
                "seq": 1 if rng.random() < 0.15 else _log_int(rng, 1, most), "vocab": vocab, "ncols": ncols,
                "scaled": rng.random() < 0.5, "backward": backward}
    if kind == "norm8":
        ncols, batch = _width(rng, 16, 16384, 64), _log_int(rng, 1, 32)
        seq = _log_int(rng, 1, max(1.0, min(8192.0, MOST_BYTES / (6.0 * size * batch * ncols))))
        return {"kind": kind, "dtype": dtype, "format": rng.choice(["e4m3", "e4m3", "e5m2"]), "batch": batch,
                "seq": seq, "ncols": ncols, "group": rng.choice([0, 0, 32, 64, 128]),
                "power_of_two": rng.random() < 0.4, "after": rng.random() < 0.5,
                "gate": rng.choice(["none", "none", "full", "sequence"]),
                "residual_scale": rng.choice([1.0, 0.5, 0.125]), "stats": rng.random() < 0.5}
    clip = rng.choice(["no", "below", "into", "into fp32"])
    width = _width(rng, 32, 2560, 64)
    hidden, vocab = _width(rng, width, 4 * width, 64), _width(rng, 64, 32000, 64)
    layers = _log_int(rng, 1, 32 if clip == "no" else 6)
    case = {"kind": kind, "dtype": dtype, "layers": layers, "width": width, "hidden": hidden, "vocab": vocab,
            "clip": clip}
    while case["layers"] > 1 and work(case)["bytes"] > MOST_BYTES:
        case["layers"] -= 1
    return case


# ---------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dtype)


def _tokens(gen, case):
    """Tokens whose frequency falls with their rank, ranks spread over the vocabulary; sequences end in
    absent tokens (-1)."""
    b, s, v = case["batch"], case["seq"], case["vocab"]
    rank = (torch.rand((b, s), generator=gen, device="cuda").double() * math.log(v)).exp().long().clamp_(1, v) - 1
    step = next(k for k in range(int(v * 0.618) | 1, 2 * v + 3) if math.gcd(k, v) == 1)
    tokens = rank * step % v
    length = torch.randint(s - s // 4, s + 1, (b, 1), generator=gen, device="cuda")
    tokens.masked_fill_(torch.arange(s, device="cuda") >= length, -1)
    return tokens.to(DTYPES[case["index"]])


def _shapes(case):
    """Sizes of a decoder's parameters: embedding, per layer four square matrices, three of the block behind
    them and two norms, a last norm."""
    w, h = case["width"], case["hidden"]
    layer = [(w, w)] * 4 + [(h, w), (h, w), (w, h), (w,), (w,)]
    return [(case["vocab"], w)] + layer * case["layers"] + [(w,)]


def _gradient_dtype(case, shape):
    return torch.float32 if len(shape) == 1 else DTYPES[case["dtype"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case}
    if kind == "embedding":
        b, s, n = case["batch"], case["seq"], case["ncols"]
        state["scale"] = math.sqrt(n) if case["scaled"] else 1.0
        state["tokens"] = _tokens(gen, case)
        if case["backward"]:
            state["grad"] = _randn(gen, (b, s, n), dtype, 0.1)
        else:
            state["table"] = _randn(gen, (case["vocab"], n), dtype, 0.02)
        return state
    if kind == "norm8":
        shape, n = (case["batch"], case["seq"], case["ncols"]), case["ncols"]
        state["x"], state["y"] = _randn(gen, shape, dtype, 2.0), _randn(gen, shape, dtype)
        gate = {"full": shape, "sequence": (shape[0], 1, n)}.get(case["gate"])
        state["gate"] = None if gate is None else _randn(gen, gate, dtype, 0.5)
        state["after"] = (1.0 + _randn(gen, (n,), torch.float32, 0.1)).to(dtype) if case["after"] else None
        state["before"] = (1.0 + _randn(gen, (n,), torch.float32, 0.1)).to(dtype)
        return state
    shapes = _shapes(case)
    # gradients of parameters of one model differ in size
    state["grads"] = [_randn(gen, shape, _gradient_dtype(case, shape), 0.002 * (1 + i % 7))
                      for i, shape in enumerate(shapes)]
    state["max_norm"] = 1e6 if case["clip"] == "below" else 0.25
    state["out"] = None
    if case["clip"].startswith("into"):
        state["out"] = [torch.empty_like(g, dtype=torch.float32 if case["clip"] == "into fp32" else None)
                        for g in state["grads"]]
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _run_own(state, case, kind)
    if kind == "embedding":
        return _embedding_backward(state) if case["backward"] else _embedding(state)
    if kind == "norm8":
        return _norm8(state)
    return _gradients(state)


def _run_own(state, case, kind):
    import neptune_codegen as CG

    if kind == "embedding":
        if case["backward"]:
            return CG.run_embedding_backward(state["grad"], state["tokens"], case["vocab"], scale=state["scale"])
        return CG.run_embedding(state["tokens"], state["table"], scale=state["scale"])
    if kind == "norm8":
        return CG.run_residual_norm_quantized(
            state["x"], state["y"], state["after"], state["before"], gate=state["gate"],
            residual_scale=case["residual_scale"], eps=EPS, dtype=DTYPES[case["format"]],
            group=case["group"] or None, power_of_two=case["power_of_two"], return_stats=case["stats"])
    if case["clip"] == "no":
        return CG.run_gradient_norm(state["grads"])
    norm = CG.run_clip_gradients(state["grads"], state["max_norm"], out=state["out"])
    return norm, state["grads"] if state["out"] is None else state["out"]


def _embedding(state):
    tokens, table = state["tokens"].long(), state["table"]
    rows = table[tokens.clamp(min=0)].float() * state["scale"]
    return rows.masked_fill_((tokens < 0).unsqueeze(-1), 0.0).to(table.dtype)


def _embedding_backward(state):
    grad, tokens = state["grad"], state["tokens"].long().flatten()
    n, vocab = grad.shape[-1], state["case"]["vocab"]
    rows = grad.reshape(-1, n).float() * (tokens >= 0).unsqueeze(-1)
    table = torch.zeros((vocab, n), device=grad.device).index_add_(0, tokens.clamp(min=0), rows)
    return table.mul_(state["scale"]).to(grad.dtype)


def _blocks(h, group):
    """h [..., n] as [..., blocks, group], the last block filled with zeros."""
    n = h.shape[-1]
    group = group or n
    return torch.nn.functional.pad(h, (0, -n % group)).unflatten(-1, (-1, group))


def _norm8(state):
    case, dtype = state["case"], state["x"].dtype
    x, y = state["x"].float(), state["y"].float()
    rate_y = torch.ones_like(x[..., :1])
    if state["after"] is not None:
        rate_y = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        y = y * rate_y * state["after"].float()
    if state["gate"] is not None:
        y = y * state["gate"].float()
    residual = x + case["residual_scale"] * y
    rate_r = torch.rsqrt(residual.square().mean(-1, keepdim=True) + EPS)
    h = _blocks(residual * rate_r * state["before"].float(), case["group"])
    scales = h.abs().amax(-1) / FORMATS[case["format"]][0]
    if case["power_of_two"]:
        # the least power of two that is no less
        m, e = torch.frexp(scales)
        scales = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e))
    scales = scales.clamp(min=LEAST_SCALE)
    values = (h / scales.unsqueeze(-1)).flatten(-2)[..., :case["ncols"]].to(DTYPES[case["format"]])
    stats = (torch.cat((rate_y, rate_r), -1),) if case["stats"] else ()
    return (residual.to(dtype), values, scales, *stats)


def _gradients(state):
    grads, clip = state["grads"], state["case"]["clip"]
    # squares of 32-bit values reach past 32 bits
    total = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    if clip == "no":
        return total
    factor = torch.where(total > state["max_norm"], state["max_norm"] / total, 1.0)
    if state["out"] is None:
        [g.copy_(g.float() * factor) for g in grads]
        return total, grads
    [o.copy_(g.float() * factor) for o, g in zip(state["out"], grads)]
    return total, state["out"]


# ---------------------------------------------------------------- the definitions in 64 bits
def _rounded(v, fmt):
    """v rounded to the 8-bit format, half to even."""
    _, bits, least = FORMATS[fmt]
    exponent = (torch.frexp(v).exponent - 1).clamp(min=least)
    step = torch.ldexp(torch.ones_like(v), exponent - bits)
    return torch.round(v / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "embedding":
        tokens = state["tokens"].long()
        if not case["backward"]:
            out = torch.zeros((*tokens.shape, case["ncols"]), dtype=torch.float64, device="cuda")
            here = tokens >= 0
            out[here] = state["table"].double().index_select(0, tokens[here]) * state["scale"]
            return out
        here = tokens >= 0
        out = torch.zeros((case["vocab"], case["ncols"]), dtype=torch.float64, device="cuda")
        return out.index_put_((tokens[here],), state["grad"][here].double() * state["scale"], accumulate=True)
    if case["kind"] == "norm8":
        mean_square = lambda t: (t * t).sum(-1, keepdim=True) / case["ncols"] + EPS  # noqa: E731
        step = state["y"].double()
        rates = [torch.ones_like(step[..., :1])]
        if case["after"]:
            rates = [1.0 / mean_square(step).sqrt()]
            step = step * rates[0] * state["after"].double()
        if state["gate"] is not None:
            step = step * state["gate"].double()
        residual = state["x"].double() + step * case["residual_scale"]
        rates.append(1.0 / mean_square(residual).sqrt())
        h = residual * rates[1] * state["before"].double()
        n, group = case["ncols"], case["group"] or case["ncols"]
        values, scales = [], []
        for first in range(0, n, group):
            block = h[..., first:first + group]
            scale = block.abs().amax(-1, keepdim=True) / FORMATS[case["format"]][0]
            if case["power_of_two"]:
                scale = 2.0 ** scale.log2().ceil()
            scale = scale.clamp(min=LEAST_SCALE)
            values.append(_rounded(block / scale, case["format"]))
            scales.append(scale)
        stats = (torch.cat(rates, -1),) if case["stats"] else ()
        return (residual, torch.cat(values, -1), torch.cat(scales, -1), *stats)
    total = math.sqrt(math.fsum(torch.dot(g.double().flatten(), g.double().flatten()).item() for g in state["grads"]))
    norm = torch.tensor(total, dtype=torch.float64, device="cuda")
    if case["clip"] == "no":
        return norm
    factor = state["max_norm"] / total if total > state["max_norm"] else 1.0
    return norm, [g.double() * factor for g in state["grads"]]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case) -> dict:
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "embedding":
        tokens, n = case["batch"] * case["seq"], case["ncols"]
        # a token's row, read and written, or added to its row of the table's gradient
        rows = (tokens + case["vocab"]) if case["backward"] else 2 * tokens
        return {"bytes": size * n * rows + SIZE[case["index"]] * tokens, "flops": tokens * n}
    if kind == "norm8":
        rows, n = case["batch"] * case["seq"], case["ncols"]
        gate = {"none": 0, "full": rows, "sequence": case["batch"]}[case["gate"]]
        groups = -(-n // (case["group"] or n))
        # x, y and residual; the 8-bit values and their scales; gammas and gate; rates
        return {"bytes": rows * (n * (3 * size + 1) + 4 * groups) + size * n * (1 + case["after"] + gate)
                + (8 * rows if case["stats"] else 0), "flops": 12 * rows * n}
    count = [(math.prod(s), 4 if len(s) == 1 else size) for s in _shapes(case)]
    out = {"into": lambda b: b, "into fp32": lambda b: 4}.get(case["clip"], lambda b: 0)
    return {"bytes": sum(c * (b + out(b)) for c, b in count),
            "flops": sum(c for c, _ in count) * (3 if case["clip"].startswith("into") else 2)}
