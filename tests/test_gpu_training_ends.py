"""A training step from tokens to clipped gradients: embedding, residual norm with an 8-bit output, an 8-bit
product tied to the embedding, distillation, and back, with the table's two gradients added in one tensor and all
gradients clipped into fp32 buffers.

The oracle is the step in float64 on the CPU, from the operators' bfloat16 inputs and with the 8-bit values that they
chose (the rounding's gradient is straight through).  What separates the two are roundings to bfloat16 (2^-8 of a value
at most): embedding, logits (forward), the logits' gradient, the norm's input gradient, dx (backward), and for each
operand's 2-norm one more: 6, relative to a gradient's 2-norm 6 / 256; 8 / 256 is allowed for the fp32 sums.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu
TOL = 8 / 256
EPS = 1e-6


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def make(batch, seq, n, vocab, top, seed):
    g = torch.Generator().manual_seed(seed)
    tokens = ((torch.rand(batch, seq, generator=g) * math.log(vocab)).exp().long() - 1).clamp(0, vocab - 1)
    tokens[-1, seq - seq // 3:] = -1                 # a padded batch
    index = torch.randint(0, vocab, (batch, seq, top), generator=g)
    index[-1, seq - seq // 3:] = -1
    return {"tokens": tokens, "table": torch.randn(vocab, n, generator=g).bfloat16(),
            "y": torch.randn(batch, seq, n, generator=g).bfloat16(),
            "after": (1 + 0.2 * torch.randn(n, generator=g)).bfloat16(),
            "before": (1 + 0.2 * torch.randn(n, generator=g)).bfloat16(),
            "top": torch.randn(batch, seq, top, generator=g), "index": index,
            "grad": torch.rand(batch, seq, generator=g) / (batch * seq)}


def step(p, group, max_norm):
    """(loss, 8-bit values, scales, gradients' norm, clipped gradients of table, gammas and y) by the direct calls."""
    vocab, n = p["table"].shape
    scale = n ** -0.5
    x = CG.run_embedding(p["tokens"], p["table"], scale=math.sqrt(n))
    _, q, s, stats = CG.run_residual_norm_quantized(x, p["y"], p["after"], p["before"], residual_scale=0.5, eps=EPS,
                                                    group=group, power_of_two=group is not None, return_stats=True)
    used = (q.float().unflatten(-1, (s.shape[-1], -1)) * s.unsqueeze(-1)).flatten(-2)
    logits = (used.view(-1, n) @ p["table"].float().t().contiguous() * scale).bfloat16().view(*x.shape[:-1], vocab)
    loss, state = CG.run_distill(logits, p["top"], p["index"], return_stats=True)
    dz = CG.run_distill_backward(p["grad"], logits, p["top"], p["index"], state)
    flat = dz.view(-1, vocab).float()
    dh = (flat @ p["table"].float() * scale).bfloat16().view_as(x)
    dtable = flat.t().contiguous() @ used.view(-1, n) * scale             # fp32, the product's share
    dx, dy, dafter, dbefore, _ = CG.run_residual_norm_backward(None, dh, x, p["y"], p["after"], p["before"], stats,
                                                               residual_scale=0.5)
    CG.run_embedding_backward(dx, p["tokens"], vocab, scale=math.sqrt(n), into=dtable)
    grads = [dtable, dafter, dbefore, dy]
    out = [torch.empty_like(t, dtype=torch.float32) for t in grads]
    norm = CG.run_clip_gradients(grads, max_norm, out=out)
    return loss, q, s, norm, *out


def oracle(p, q, s, max_norm):
    leaf = {k: p[k].double().requires_grad_() for k in ("table", "after", "before", "y")}
    vocab, n = p["table"].shape
    known = (p["tokens"] >= 0).unsqueeze(-1)
    x = torch.where(known, leaf["table"][p["tokens"].clamp(min=0)] * math.sqrt(n), 0.0)
    rate = lambda t: (t.square().mean(-1, keepdim=True) + EPS).rsqrt()  # noqa: E731
    r = x + 0.5 * leaf["y"] * rate(leaf["y"]) * leaf["after"]
    h = r * rate(r) * leaf["before"]
    used = (q.float().double().unflatten(-1, (s.shape[-1], -1)) * s.double().unsqueeze(-1)).flatten(-2)
    h = h + (used - h).detach()
    z = h @ leaf["table"].t() * n ** -0.5
    here = p["index"] >= 0
    t = torch.where(here.any(-1, keepdim=True), p["top"].double().masked_fill(~here, -math.inf), 0.0)
    prob = torch.where(here, t.softmax(-1), 0.0)
    log_q = z.log_softmax(-1).gather(-1, p["index"].clamp(min=0))
    loss = (torch.xlogy(prob, prob) - prob * log_q).sum(-1)
    grads = torch.autograd.grad((loss * p["grad"]).sum(), [leaf[k] for k in ("table", "after", "before", "y")])
    norm = math.sqrt(sum(t.square().sum().item() for t in grads))
    return loss.detach(), norm, [t * min(1.0, max_norm / norm) for t in grads]


@pytest.mark.parametrize("batch,seq,n,vocab,group,max_norm", [
    (2, 33, 128, 501, 32, 1e-3), (3, 130, 256, 2000, None, 1e6), (1, 700, 64, 997, 64, 0.01), (4, 1, 512, 130, 128, 1e-3)])
def test_a_steps_gradients_match_the_formulas(batch, seq, n, vocab, group, max_norm):
    dev = _dev()
    print(f"step {batch}x{seq} {n} of {vocab}", flush=True)
    p = make(batch, seq, n, vocab, 6, seed=seq)
    loss, q, s, norm, *got = step({k: v.to(dev) for k, v in p.items()}, group, max_norm)
    want_loss, want_norm, want = oracle(p, q.cpu(), s.cpu(), max_norm)
    assert (loss.cpu().double() - want_loss).norm() <= TOL * want_loss.norm()
    assert abs(norm.item() - want_norm) <= TOL * want_norm
    assert math.sqrt(sum(t.double().square().sum().item() for t in got)) <= max_norm * (1 + 1e-6) or norm <= max_norm
    for name, a, b in zip(("table", "after", "before", "y"), got, want):
        err = ((a.cpu().double() - b).norm() / b.norm()).item()
        assert err <= 2 * TOL if norm > max_norm else err <= TOL, (name, err)   # (its own and its norm's error)


def test_captured_steps_replay_in_turn_and_at_once():
    dev = _dev()
    sets = [{k: v.to(dev) for k, v in make(2, 150, 128, 1000, 6, seed=s).items()} for s in range(3)]
    run = lambda p: step(p, 32, 1e-3)  # noqa: E731
    same = lambda a, b: torch.equal(a.float(), b.float())  # noqa: E731
    want = [[t.clone() for t in run(p)] for p in sets]
    assert all(same(a, b) for a, b in zip(run(sets[0]), want[0]))
    torch.cuda.synchronize()
    static = [{k: v.clone() for k, v in sets[0].items()} for _ in range(2)]
    graphs, outs = [], []
    for p in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(p))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        print(f"replay {turn}", flush=True)
        picks = [turn % 3, (turn + 1) % 3]
        for p, pick in zip(static, picks):
            for k, v in p.items():
                v.copy_(sets[pick][k])
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager = run(sets[2])                         # the program's own work between replays
        for out, pick in zip(outs, picks):
            assert all(same(a, b) for a, b in zip(out, want[pick]))
        assert all(same(a, b) for a, b in zip(eager, want[2]))
    got = [[], []]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same(a, b) for out in got[i] for a, b in zip(out, want[i]))


class EightBitProduct(torch.autograd.Function):
    """norm(x + y) in 8 bits times w: a differentiable product as a model writes it, straight through the rounding."""

    @staticmethod
    def forward(ctx, x, y, gamma, w):
        _, q, s, stats = CG.run_residual_norm_quantized(x, y, None, gamma, group=32, power_of_two=True, return_stats=True)
        used = (q.float().unflatten(-1, (s.shape[-1], -1)) * s.unsqueeze(-1)).flatten(-2)
        ctx.save_for_backward(x, y, gamma, w, used, stats)
        return (used.flatten(0, -2) @ w.float()).to(x.dtype).view(*x.shape[:-1], -1)

    @staticmethod
    def backward(ctx, grad):
        x, y, gamma, w, used, stats = ctx.saved_tensors
        g = grad.flatten(0, -2).float()
        dh = (g @ w.float().t().contiguous()).to(x.dtype).view_as(x)
        dx, dy, _, dgamma, _ = CG.run_residual_norm_backward(None, dh, x, y, None, gamma, stats)
        return dx, dy, dgamma, (used.flatten(0, -2).t().contiguous() @ g).to(w.dtype)


def test_a_model_trains_through_autograd():
    # twelve steps of plain descent run, with finite gradients of every parameter, clipped as asked for
    dev = _dev()
    g = torch.Generator().manual_seed(3)
    p = {k: v.to(dev) for k, v in make(2, 40, 64, 300, 4, seed=1).items()}
    table = torch.randn(300, 64, generator=g).bfloat16().to(dev).requires_grad_()
    gamma = torch.ones(64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    w = (0.1 * torch.randn(64, 300, generator=g)).bfloat16().to(dev).requires_grad_()
    embed, distill, params = CG.as_embedding_op(8.0), CG.as_distill_op(), [table, gamma, w]
    print("training through autograd", flush=True)
    for _ in range(12):
        x = embed(p["tokens"], table)
        loss = distill(EightBitProduct.apply(x, p["y"], gamma, w), p["top"], p["index"])[0].mean()
        grads = torch.autograd.grad(loss, params)
        before = CG.run_gradient_norm(grads)
        norm = CG.run_clip_gradients(grads, 0.1)
        assert torch.equal(norm, before) and torch.isfinite(norm) and norm > 0
        assert CG.run_gradient_norm(grads) <= 0.1 * (1 + 2.0 ** -7) or norm <= 0.1
        with torch.no_grad():
            for t, d in zip(params, grads):
                t.sub_(d)
    assert torch.isfinite(loss)
