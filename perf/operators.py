"""Performance cases of the training operators: attention's gradients, rotary positions, the
residual norm and the distillation loss, each in the directions that a training step runs.

`listed()` names twelve of them, from calls of a few kilobytes to a 1.4 TFLOP attention gradient
and passes of 1 GB; `draw()` makes more of the same ranges.  `run` computes a case in elementary
torch operations in 32 bits, or, where `own` is set, with the framework's kernels.
"""
from __future__ import annotations

import math
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "neptune-opt_amd"))

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6
FAR = 1 << 20            # positions are below this
# a drawn case stays below these (the largest listed cases are just above them)
MOST_BYTES = 1.0e9
MOST_FLOPS = 1.3e12


def listed() -> list[dict]:
    return [
        # attention of two short ragged prompts in a small model: launches and latency
        {"name": "attention_backward_small", "kind": "attention", "dtype": "bf16", "batch": 2,
         "heads": 4, "sq": 77, "sk": 77, "dim": 64, "causal": True, "layout": "bshd"},
        # a decoder layer's training step over long sequences, projection layout [B, S, H, D]
        {"name": "attention_backward_decoder", "kind": "attention", "dtype": "bf16", "batch": 4,
         "heads": 32, "sq": 4096, "sk": 4096, "dim": 128, "causal": True, "layout": "bshd"},
        # an encoder layer over inputs of an odd length
        {"name": "attention_backward_encoder", "kind": "attention", "dtype": "fp16", "batch": 8,
         "heads": 12, "sq": 777, "sk": 777, "dim": 64, "causal": False, "layout": "bshd"},
        # the queries and shared keys of one generated token for each of 64 sequences, far out
        {"name": "rotary_token", "kind": "rotary", "dtype": "bf16", "batch": 64, "seq": 1,
         "heads_q": 32, "heads_k": 8, "dim": 128, "part": 128, "interleaved": False,
         "backward": False, "scaling": "parts", "factor": 8.0, "layout": "bshd"},
        # a decoder layer's training step: queries and keys from the projection layout
        {"name": "rotary_decoder", "kind": "rotary", "dtype": "bf16", "batch": 4, "seq": 4096,
         "heads_q": 32, "heads_k": 32, "dim": 128, "part": 128, "interleaved": False,
         "backward": False, "scaling": "none", "factor": 1.0, "layout": "bshd"},
        # gradients of neighbouring pairs in half of each head, an odd length
        {"name": "rotary_backward_odd", "kind": "rotary", "dtype": "fp32", "batch": 3, "seq": 1777,
         "heads_q": 12, "heads_k": 4, "dim": 80, "part": 40, "interleaved": True,
         "backward": True, "scaling": "linear", "factor": 4.0, "layout": "bhsd"},
        # one generated token for each of 8 sequences, between two blocks
        {"name": "norm_small", "kind": "norm", "dtype": "bf16", "batch": 8, "seq": 1,
         "ncols": 1024, "after": False, "gate": "none", "residual_scale": 1.0,
         "backward": False, "stats": False},
        # a training batch of 16384 tokens, the block gated by its sequence's condition
        {"name": "norm_gated", "kind": "norm", "dtype": "bf16", "batch": 8, "seq": 2048,
         "ncols": 4096, "after": True, "gate": "sequence", "residual_scale": 0.5,
         "backward": False, "stats": True},
        # its gradients, the condition's and both gammas' among them
        {"name": "norm_gated_backward", "kind": "norm", "dtype": "bf16", "batch": 8, "seq": 2048,
         "ncols": 4096, "after": True, "gate": "sequence", "residual_scale": 0.5,
         "backward": True, "stats": True},
        # a validation batch against a teacher's 8 best of 1000 classes
        {"name": "distill_small", "kind": "distill", "dtype": "fp32", "rows": 16, "vocab": 1000,
         "top": 8, "temperature": 2.0, "backward": False},
        # a language model's training batch against the teacher's 64 best tokens (1.05 GB)
        {"name": "distill_vocab", "kind": "distill", "dtype": "bf16", "rows": 16384,
         "vocab": 32000, "top": 64, "temperature": 1.0, "backward": False},
        # its gradient over a vocabulary with a few added tokens (odd width)
        {"name": "distill_backward_odd", "kind": "distill", "dtype": "bf16", "rows": 7168,
         "vocab": 32003, "top": 64, "temperature": 1.5, "backward": True},
    ]


# ---------------------------------------------------------------- drawn cases
def _log_int(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo: int, hi: int, unit: int) -> int:
    """Half the widths are multiples of `unit`, half are any number."""
    w = _log_int(rng, lo, hi)
    return max(unit, w // unit * unit) if rng.random() < 0.5 else w


def draw(rng) -> dict:
    kind = rng.choice(["attention", "attention", "rotary", "norm", "norm", "distill", "distill"])
    if kind == "attention":
        dim, causal = rng.choice([64, 128, 128, 256]), rng.random() < 0.5
        batch, heads = _log_int(rng, 1, 16), rng.choice([1, 4, 8, 12, 16, 32, 40])
        # a single query sees one key under the causal mask, and its scores have no gradient
        sq = _width(rng, 16 if causal or rng.random() < 0.7 else 1, 8192, 64)
        sk = sq if causal or rng.random() < 0.5 else _width(rng, 16, 8192, 64)
        while 10.0 * batch * heads * sq * sk * dim * (0.5 if causal else 1.0) > MOST_FLOPS:
            sq, sk = (sq + 1) // 2, (sk + 1) // 2
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch, "heads": heads,
                "sq": sq, "sk": sk, "dim": dim, "causal": causal,
                "layout": rng.choice(["bhsd", "bshd"])}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = SIZE[dtype]
    if kind == "rotary":
        dim = rng.choice([64, 128, 128, 256, 2 * _log_int(rng, 8, 128)])
        part = dim if rng.random() < 0.6 else max(2, dim // 4 * 2)
        heads_q = rng.choice([1, 8, 12, 16, 32, 40])
        heads_k = rng.choice([heads_q, 8, 1])
        batch = _log_int(rng, 1, 64)
        seq = 1 if rng.random() < 0.2 else _log_int(rng, 2, 32768)
        while 2.0 * size * batch * seq * (heads_q + heads_k) * dim > 0.5 * MOST_BYTES:
            seq = (seq + 1) // 2
        scaling = rng.choice(["none", "linear", "parts"])
        return {"kind": kind, "dtype": dtype, "batch": batch, "seq": seq, "heads_q": heads_q,
                "heads_k": heads_k, "dim": dim, "part": part, "interleaved": rng.random() < 0.5,
                "backward": rng.random() < 0.5, "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                "layout": rng.choice(["bhsd", "bshd"])}
    if kind == "norm":
        ncols, batch = _width(rng, 16, 16384, 64), _log_int(rng, 1, 32)
        seq = _log_int(rng, 1, max(1.0, min(8192.0, MOST_BYTES / (7.0 * size * batch * ncols))))
        return {"kind": kind, "dtype": dtype, "batch": batch, "seq": seq, "ncols": ncols,
                "after": rng.random() < 0.6, "residual_scale": rng.choice([1.0, 0.5, 0.125]),
                "gate": rng.choice(["none", "full", "sequence", "channel"]),
                "backward": rng.random() < 0.5, "stats": rng.random() < 0.7}
    vocab, backward = _width(rng, 64, 200000, 64), rng.random() < 0.5
    rows = _log_int(rng, 1, max(1.0, min(16384.0, MOST_BYTES / ((2 if backward else 1) * size * vocab))))
    return {"kind": kind, "dtype": dtype, "rows": rows, "vocab": vocab,
            "top": _log_int(rng, 1, min(256, vocab // 2)),
            "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]), "backward": backward}


# ---------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dtype)


def _heads(gen, case, heads, seq, dtype, scale=1.0):
    """[B, H, S, D], contiguous or a view of the projection layout [B, S, H, D]."""
    b, d = case["batch"], case["dim"]
    if case["layout"] == "bshd":
        return _randn(gen, (b, seq, heads, d), dtype, scale).transpose(1, 2)
    return _randn(gen, (b, heads, seq, d), dtype, scale)


def _softmax_rows(case, q, k):
    """Scaled scores of every pair in fp32, hidden ones -inf, and their logsumexp."""
    s = torch.matmul(q.float() * (1.0 / math.sqrt(case["dim"])), k.float().transpose(2, 3).contiguous())
    if case["causal"]:
        s.masked_fill_(torch.ones(s.shape[2:], dtype=torch.bool, device=s.device).triu_(1), -math.inf)
    top = s.amax(-1, keepdim=True)
    return s, top + (s - top).exp_().sum(-1, keepdim=True).log()


def _turns(case):
    """Turns per position of each pair (64 bits) and the factor of the rotated values."""
    part, factor, base = case["part"], case["factor"], 10000.0
    rate = base ** (-torch.arange(0, part, 2, dtype=torch.float64, device="cuda") / part)
    if case["scaling"] == "linear":
        rate = rate / factor
    if case["scaling"] == "parts":
        # pairs that turn more than 32 times within the 4096 positions of pretraining keep their
        # rate, those below one turn are slowed by the whole factor
        kept = ((4096 * rate / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        rate = rate * (kept + (1.0 - kept) / factor)
    return rate / (2 * math.pi), 0.1 * math.log(factor) + 1.0 if case["scaling"] == "parts" else 1.0


def _gate_shape(case):
    b, s, n = case["batch"], case["seq"], case["ncols"]
    return {"full": (b, s, n), "sequence": (b, 1, n), "channel": (n,)}[case["gate"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case}
    if kind == "attention":
        q = _heads(gen, case, case["heads"], case["sq"], dtype)
        k, v = (_heads(gen, case, case["heads"], case["sk"], dtype) for _ in range(2))
        grad = _heads(gen, case, case["heads"], case["sq"], dtype, 0.1)
        # what the forward pass left: the output and its rows' logsumexp
        s, lse = _softmax_rows(case, q, k)
        out = torch.matmul(s.sub_(lse).exp_(), v.float()).to(dtype)
        return {**state, "q": q, "k": k, "v": v, "grad": grad, "out": out, "lse": lse.squeeze(-1)}
    if kind == "rotary":
        b, seq = case["batch"], case["seq"]
        state["q"] = _heads(gen, case, case["heads_q"], seq, dtype)
        state["k"] = _heads(gen, case, case["heads_k"], seq, dtype)
        first = torch.randint(FAR - seq, (b, 1), generator=gen, device="cuda")
        state["positions"] = first + torch.arange(seq, device="cuda")
        state["turns"], state["magnitude"] = _turns(case)
        return state
    if kind == "norm":
        shape, n = (case["batch"], case["seq"], case["ncols"]), case["ncols"]
        state["x"], state["y"] = _randn(gen, shape, dtype, 2.0), _randn(gen, shape, dtype)
        state["gate"] = None if case["gate"] == "none" else _randn(gen, _gate_shape(case), dtype, 0.5)
        state["after"] = (1.0 + _randn(gen, (n,), torch.float32, 0.1)).to(dtype) if case["after"] else None
        state["before"] = (1.0 + _randn(gen, (n,), torch.float32, 0.1)).to(dtype)
        if case["backward"]:
            state["grad_residual"] = _randn(gen, shape, dtype, 0.1)
            state["grad_normed"] = _randn(gen, shape, dtype, 0.1)
            state["stats"] = _norm_forward(state)[2]
        return state
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    state["logits"] = _randn(gen, (rows, vocab), dtype, 3.0)
    # the teacher's best tokens, best first; ends of lists and some rows (prompts) are empty
    state["index"] = torch.rand((rows, vocab), generator=gen, device="cuda").topk(top, -1).indices \
        if rows * vocab < 1 << 22 else _distinct(gen, rows, vocab, top)
    state["top_logits"] = _randn(gen, (rows, top), torch.float32, 3.0).sort(-1, descending=True).values
    length = torch.randint(1, 2 * top + 1, (rows, 1), generator=gen, device="cuda").clamp_(max=top)
    length[torch.rand((rows, 1), generator=gen, device="cuda") < 0.1] = 0
    length[0] = top
    state["index"].masked_fill_(torch.arange(top, device="cuda") >= length, -1)
    if case["backward"]:
        # of a mean over the tokens; fp16 gradients with the usual scaling of the loss
        scale = 65536.0 if dtype == torch.float16 else 1.0
        state["grad"] = torch.rand((rows,), generator=gen, device="cuda") * (scale / rows)
        state["stats"] = _distill_forward(state)[1]
    return state


def _distinct(gen, rows, vocab, top):
    """Distinct columns for each row: one random column out of each of `top` equal ranges."""
    first = torch.arange(top, device="cuda") * vocab // top
    width = (torch.arange(1, top + 1, device="cuda") * vocab // top) - first
    return first + (torch.rand((rows, top), generator=gen, device="cuda") * width).long().clamp_(max=vocab // top - 1)


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _run_own(state, kind)
    if kind == "attention":
        return _attention_backward(state)
    if kind == "rotary":
        return _rotary(state, state["q"]), _rotary(state, state["k"])
    if kind == "norm":
        if case["backward"]:
            return _norm_backward(state)
        return _norm_forward(state)[:3 if case["stats"] else 2]
    return _distill_backward(state) if case["backward"] else _distill_forward(state)


def _run_own(state, kind):
    import neptune_codegen as CG

    case = state["case"]
    if kind == "attention":
        return CG.run_attention_backward(state["grad"], state["q"], state["k"], state["v"],
                                         state["out"], state["lse"], causal=case["causal"])
    if kind == "rotary":
        rotate = CG.run_rotary_backward if case["backward"] else CG.run_rotary
        return rotate(state["q"], state["k"], state["positions"], state["turns"],
                      magnitude=state["magnitude"], interleaved=case["interleaved"])
    if kind == "norm":
        if not case["backward"]:
            return CG.run_residual_norm(state["x"], state["y"], state["after"], state["before"],
                                        gate=state["gate"], residual_scale=case["residual_scale"],
                                        eps=EPS, return_stats=case["stats"])
        grads = CG.run_residual_norm_backward(
            state["grad_residual"], state["grad_normed"], state["x"], state["y"], state["after"],
            state["before"], state["stats"], gate=state["gate"], residual_scale=case["residual_scale"])
        return tuple(g for g in grads if g is not None)
    if case["backward"]:
        return CG.run_distill_backward(state["grad"], state["logits"], state["top_logits"],
                                       state["index"], state["stats"], temperature=case["temperature"])
    return CG.run_distill(state["logits"], state["top_logits"], state["index"],
                          temperature=case["temperature"], return_stats=True)


def _attention_backward(state):
    case, dtype = state["case"], state["q"].dtype
    q, k, v, grad = (state[n].float() for n in ("q", "k", "v", "grad"))
    p, lse = _softmax_rows(case, q, k)
    p.sub_(lse).exp_()
    dv = torch.matmul(p.transpose(2, 3), grad)
    ds = torch.matmul(grad, v.transpose(2, 3))
    ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(1.0 / math.sqrt(case["dim"]))
    return (torch.matmul(ds, k).to(dtype), torch.matmul(ds.transpose(2, 3), q).to(dtype), dv.to(dtype))


def _rotary(state, x):
    case = state["case"]
    part = case["part"]
    angle = 2 * math.pi * torch.frac(state["positions"].double().unsqueeze(-1) * state["turns"])
    if case["backward"]:
        angle = -angle
    cos = (angle.cos() * state["magnitude"]).float().unsqueeze(1)
    sin = (angle.sin() * state["magnitude"]).float().unsqueeze(1)
    rotated, rest = x[..., :part].float(), x[..., part:]
    if case["interleaved"]:
        a, b = rotated[..., 0::2], rotated[..., 1::2]
        rotated = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = rotated[..., :part // 2], rotated[..., part // 2:]
        rotated = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((rotated.to(x.dtype), rest), -1)


def _norm_forward(state):
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
    normed = residual * rate_r * state["before"].float()
    return residual.to(dtype), normed.to(dtype), torch.cat((rate_y, rate_r), -1)


def _norm_backward(state):
    case, dtype = state["case"], state["x"].dtype
    x, y, before = state["x"].float(), state["y"].float(), state["before"].float()
    grad_residual, grad_normed = state["grad_residual"].float(), state["grad_normed"].float()
    rate_y, rate_r = state["stats"][..., :1], state["stats"][..., 1:]
    n = case["ncols"]
    unit = y * rate_y                                   # the block's output over its norm
    scaled = unit * state["after"].float() if case["after"] else unit
    gate = case["residual_scale"] * (state["gate"].float() if state["gate"] is not None
                                     else torch.ones_like(before))
    hat = (x + gate * scaled) * rate_r                  # the residual over its norm
    dhat = grad_normed * before
    dx = grad_residual + rate_r * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))
    dbefore = (grad_normed * hat).view(-1, n).sum(0)
    dscaled = dx * gate
    grads = [dx.to(dtype)]
    if case["after"]:
        dunit = dscaled * state["after"].float()
        grads.append((rate_y * (dunit - unit * (dunit * unit).mean(-1, keepdim=True))).to(dtype))
        grads.append((dscaled * unit).view(-1, n).sum(0).to(dtype))
    else:
        grads.append(dscaled.to(dtype))
    grads.append(dbefore.to(dtype))
    if state["gate"] is not None:
        dgate = case["residual_scale"] * dx * scaled
        grads.append(dgate.sum_to_size(state["gate"].shape).to(dtype))
    return tuple(grads)


def _teacher(state):
    """The teacher's probabilities over its list, 0 at empty entries and over empty lists."""
    absent = state["index"] < 0
    t = (state["top_logits"] / state["case"]["temperature"]).masked_fill(absent, -math.inf)
    p = (t - t.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0)


def _distill_forward(state):
    temperature = state["case"]["temperature"]
    z = state["logits"].float()
    top = z.amax(-1, keepdim=True)
    total = ((z - top) / temperature).exp_().sum(-1, keepdim=True)
    p = _teacher(state)
    log_q = (z.gather(-1, state["index"].clamp(min=0)) - top) / temperature - total.log()
    kept = p > 0
    term = torch.where(kept, p * (torch.where(kept, p, 1.0).log() - log_q), 0.0)
    return temperature ** 2 * term.sum(-1), torch.cat((top, total), -1)


def _distill_backward(state):
    temperature = state["case"]["temperature"]
    p = _teacher(state)
    top, total = state["stats"][:, :1], state["stats"][:, 1:]
    dz = ((state["logits"].float() - top) / temperature).exp_().mul_(p.sum(-1, keepdim=True) / total)
    dz.scatter_add_(-1, state["index"].clamp(min=0), -p)
    return dz.mul_(temperature * state["grad"].unsqueeze(-1)).to(state["logits"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case) -> dict:
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "attention":
        b, h, sq, sk, d = (case[n] for n in ("batch", "heads", "sq", "sk", "dim"))
        # causal: query i sees the keys j <= i
        seen = sum(min(i + 1, sk) for i in range(sq)) if case["causal"] else sq * sk
        # q, grad, out, dq and lse; k, v, dk and dv; five products over the visible pairs
        return {"bytes": b * h * (d * size * (4 * sq + 4 * sk) + 4 * sq), "flops": 10 * b * h * seen * d}
    if kind == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads_q"] + case["heads_k"])
        return {"bytes": 2 * size * n * case["dim"] + 8 * tokens + 4 * case["part"],
                "flops": 3 * n * case["part"]}
    if kind == "norm":
        rows, n = case["batch"] * case["seq"], case["ncols"]
        whole = {"none": 0, "full": rows, "sequence": case["batch"], "channel": 1}[case["gate"]]
        gammas = 2 if case["after"] else 1
        if case["backward"]:       # x, y, both gradients, stats; dx, dy; gammas and gate with theirs
            return {"bytes": size * n * (6 * rows + 2 * whole + 2 * gammas) + 8 * rows, "flops": 30 * rows * n}
        return {"bytes": size * n * (4 * rows + whole + gammas) + (8 * rows if case["stats"] else 0),
                "flops": 9 * rows * n}
    rows, n = case["rows"], case["rows"] * case["vocab"]
    lists = 12 * rows * case["top"] + 12 * rows      # the teacher's; loss (or its gradient), stats
    return {"bytes": (2 if case["backward"] else 1) * size * n + lists, "flops": 4 * n}


# ---------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """From the forward definition in float64, gradients by automatic differentiation."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "attention":
        return _exact_attention(case, state)
    if kind == "rotary":
        return tuple(_exact_rotary(case, state, state[n]) for n in ("q", "k"))
    if kind == "norm":
        return _exact_norm(case, state)
    step = max(1, (1 << 27) // case["vocab"])
    blocks = [_exact_distill(case, state, slice(i, i + step)) for i in range(0, case["rows"], step)]
    if case["backward"]:
        return torch.cat(blocks)
    return tuple(torch.cat(parts) for parts in zip(*blocks))


def _exact_attention(case, state):
    grads = [torch.empty(state[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")]
    seen = torch.ones(case["sq"], case["sk"], dtype=torch.bool, device="cuda")
    if case["causal"]:
        seen = seen.tril_()
    for i in range(case["batch"]):
        for j in range(case["heads"]):
            q, k, v = (state[n][i, j].double().requires_grad_() for n in ("q", "k", "v"))
            s = (q @ k.t()) / math.sqrt(case["dim"])
            out = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v
            for g, d in zip(grads, torch.autograd.grad(out, (q, k, v), state["grad"][i, j].double())):
                g[i, j] = d
    return tuple(grads)


def _exact_rotary(case, state, x):
    part = case["part"]
    turn = state["positions"].double()[:, None, :, None] * state["turns"]
    turn = turn - turn.round()
    unit = torch.polar(torch.full_like(turn, state["magnitude"]), 2 * math.pi * turn)
    if case["backward"]:
        unit = unit.conj()
    x = x.double()
    if case["interleaved"]:
        pairs = x[..., :part].unflatten(-1, (part // 2, 2))
    else:
        pairs = x[..., :part].unflatten(-1, (2, part // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., part:]), -1)


def _exact_norm(case, state):
    leaves = {n: state[n].double() for n in ("x", "y", "after", "before", "gate") if state[n] is not None}
    if case["backward"]:
        leaves = {n: t.requires_grad_() for n, t in leaves.items()}
    block, rates = leaves["y"], [torch.ones_like(leaves["x"][..., :1])]
    if "after" in leaves:
        rates = [(block.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()]
        block = block * rates[0] * leaves["after"]
    residual = leaves["x"] + case["residual_scale"] * (block * leaves["gate"] if "gate" in leaves else block)
    rates.append((residual.pow(2).mean(-1, keepdim=True) + EPS).rsqrt())
    normed = residual * rates[1] * leaves["before"]
    if case["backward"]:
        return torch.autograd.grad((residual, normed), tuple(leaves.values()),
                                   (state["grad_residual"].double(), state["grad_normed"].double()))
    return (residual, normed, torch.cat(rates, -1)) if case["stats"] else (residual, normed)


def _exact_distill(case, state, rows):
    temperature, index = case["temperature"], state["index"][rows]
    z = state["logits"][rows].double()
    if case["backward"]:
        z.requires_grad_()
    t = state["top_logits"][rows].double() / temperature
    log_p = torch.log_softmax(t.masked_fill(index < 0, -1e300), -1)
    live = (index >= 0)
    log_q = torch.log_softmax(z / temperature, -1).gather(-1, index.clamp(min=0))
    loss = temperature ** 2 * (log_p.exp() * (log_p - log_q)).masked_fill(~live, 0.0).sum(-1)
    if case["backward"]:
        return torch.autograd.grad(loss, z, state["grad"][rows].double())[0]
    top = z.amax(-1, keepdim=True)
    return loss, torch.cat((top, ((z - top) / temperature).exp().sum(-1, keepdim=True)), -1)
