"""A training step through the operators of a decoder layer trained from a teacher: residual norms, rotary
positions, attention and distillation, forward and backward, together.

The oracle is the same step in float64 on the CPU, with torch's autograd.  Its inputs are the operators' own
bfloat16 values, so what separates the two are roundings to bfloat16 (2^-8 of a value at most).  On the
longest way from the loss back to a parameter lie the layer's values (norm, projection, rotation, scores'
weights, attention, projection, norm, logits: 8) and their gradients (8): relative to a gradient's 2-norm,
16 / 256.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu

TOL = 16 / 256


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def parameters(batch, seq, heads, dim, vocab, top, seed):
    g = torch.Generator().manual_seed(seed)
    e = heads * dim
    r = lambda *s, by=1.0: (by * torch.randn(*s, generator=g)).bfloat16()  # noqa: E731
    p = {"x": r(batch, seq, e), "y": r(batch, seq, e), "gate": r(batch, 1, e),
         "after": r(e, by=0.3) + 1, "before": r(e, by=0.3) + 1, "after2": r(e, by=0.3) + 1, "before2": r(e, by=0.3) + 1,
         "wq": r(e, e, by=e ** -0.5), "wk": r(e, e, by=e ** -0.5), "wv": r(e, e, by=e ** -0.5),
         "wo": r(e, e, by=e ** -0.5), "head": r(e, vocab, by=e ** -0.5)}
    fixed = {"top": torch.randn(batch * seq, top, generator=g),
             "index": torch.stack([torch.randperm(vocab, generator=g)[:top] for _ in range(batch * seq)]),
             "positions": torch.randint(0, 4096, (batch, seq), generator=g)}
    fixed["index"][::5, 1:] = -1                     # some rows name one token
    fixed["index"][2] = -1                           # and one none
    return p, fixed


def layer(p, fixed, turns, heads, interleaved, ops):
    """Loss of every row; `ops` are the operators or their plain forms."""
    batch, seq, e = p["x"].shape
    split = lambda t: t.view(batch, seq, heads, e // heads).transpose(1, 2)  # noqa: E731
    r, h = ops["norm"](p["x"], p["y"], p["after"], p["before"], p["gate"])
    h = h.reshape(-1, e)
    q, k, v = (split(h @ p[w]) for w in ("wq", "wk", "wv"))
    q, k = ops["rotary"](q, k, fixed["positions"], turns, interleaved)
    o = ops["attention"](q, k, v).transpose(1, 2).reshape(-1, e) @ p["wo"]
    _, h = ops["norm"](r, o.view(batch, seq, e), p["after2"], p["before2"], None)
    return ops["distill"](h.reshape(-1, e) @ p["head"], fixed["top"], fixed["index"])


def plain_norm(x, y, after, before, gate):
    rate = lambda t: (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    step = y * rate(y) * after
    r = x + 0.5 * (step if gate is None else step * gate)
    return r, r * rate(r) * before


def plain_rotary(q, k, positions, turns, interleaved):
    angle = 2 * math.pi * positions[:, None, :, None].double() * turns

    def turn(t):
        a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else t.chunk(2, -1)
        a, b = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
        return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)

    return turn(q), turn(k)


def plain_attention(q, k, v):
    s = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
    hidden = torch.ones(s.shape[-2:], dtype=torch.bool).triu(1)
    return s.masked_fill(hidden, -math.inf).softmax(-1) @ v


def plain_distill(z, top, index):
    here = index >= 0
    q = (z / 2).log_softmax(-1).gather(-1, index.clamp(min=0))
    t = top.double().div(2).masked_fill(~here, -math.inf)
    t = torch.where(here.any(-1, keepdim=True), t, 0.0)   # (a row without an entry: 0, not NaN)
    p = torch.where(here, t.softmax(-1), 0.0)
    return 4 * (torch.xlogy(p, p) - p * q).sum(-1)


PLAIN = {"norm": plain_norm, "rotary": plain_rotary, "attention": plain_attention, "distill": plain_distill}


def operators():
    norm, attention, distill = CG.as_residual_norm_op(0.5), CG.as_attention_grad_op(), CG.as_distill_op(2.0)
    halves, pairs = CG.as_rotary_op(), CG.as_rotary_op(interleaved=True)
    return {"norm": lambda *a: norm(*a)[:2], "attention": lambda *a: attention(*a)[0],
            "rotary": lambda q, k, positions, turns, i: (pairs if i else halves)(q, k, positions, turns),
            "distill": lambda *a: distill(*a)[0]}


@pytest.mark.parametrize("batch,seq,heads,dim,vocab,interleaved", [
    (2, 33, 3, 64, 501, False), (1, 130, 2, 128, 1000, True), (3, 1, 2, 64, 130, False)])
def test_a_layers_gradients_match_the_formulas(batch, seq, heads, dim, vocab, interleaved):
    dev = _dev()
    print(f"training step {batch}x{seq} heads {heads} dim {dim}", flush=True)
    p, fixed = parameters(batch, seq, heads, dim, vocab, 8, seed=seq)
    turns, _ = CG.rotary_frequencies(dim, device="cpu")
    weights = torch.rand(batch * seq, generator=torch.Generator().manual_seed(1))

    mine = {n: t.to(dev).requires_grad_() for n, t in p.items()}
    here = {n: t.to(dev) for n, t in fixed.items()}
    loss = layer(mine, here, turns.to(dev), heads, interleaved, operators())
    got = torch.autograd.grad((loss * weights.to(dev)).sum(), list(mine.values()))

    plain = {n: t.double().requires_grad_() for n, t in p.items()}
    want_loss = layer(plain, fixed, turns, heads, interleaved, PLAIN)
    want = torch.autograd.grad((want_loss * weights).sum(), list(plain.values()))
    assert (loss.cpu().double() - want_loss).norm() <= TOL * want_loss.norm()
    assert loss[2] == 0
    for n, a, b in zip(p, got, want):
        if seq == 1 and n in ("wq", "wk"):
            # one key: its weight is 1 whatever the scores; what is left is the rounding of dP - delta
            assert a.float().norm() <= TOL * got[list(p).index("wv")].float().norm()
            continue
        err = (a.cpu().double() - b).norm() / b.norm()
        assert err <= TOL, f"{n}: {err}"


def chain(p, turns):
    """A step by the direct entry points alone, in place of the projections the layer's own rows."""
    x, y, gate, after, before, positions, top, index, grad = p
    batch, seq, e = x.shape
    split = lambda t: t.view(batch, seq, e // 64, 64).transpose(1, 2)  # noqa: E731
    join = lambda t: t.transpose(1, 2).reshape(batch, seq, e)  # noqa: E731
    r, h, stats = CG.run_residual_norm(x, y, after, before, gate=gate, return_stats=True)
    q, k = CG.run_rotary(split(h), split(r), positions, turns)
    v = split(h)
    o, lse = CG.run_attention(q, k, v, return_lse=True)
    r2, z, stats2 = CG.run_residual_norm(r, join(o), None, before, return_stats=True)
    loss, state = CG.run_distill(z, top, index, return_stats=True)
    dz = CG.run_distill_backward(grad, z, top, index, state)
    dr, do, _, dbefore2, _ = CG.run_residual_norm_backward(None, dz, r, join(o), None, before, stats2)
    dq, dk, dv = CG.run_attention_backward(split(do), q, k, v, o, lse)
    dq, dk = CG.run_rotary_backward(dq, dk, positions, turns)
    dx, dy, dafter, dbefore, dgate = CG.run_residual_norm_backward(
        dr.add_(join(dk)), join(dq).add_(join(dv)), x, y, after, before, stats, gate=gate)
    return loss, dx, dy, dafter, dbefore, dbefore2, dgate


def chain_inputs(dev, seed, batch=2, seq=150, heads=3):
    e = heads * 64
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    return [t.to(dev) for t in (r(batch, seq, e), r(batch, seq, e), r(batch, 1, e), r(e), r(e),
                                torch.randint(0, 1 << 20, (batch, seq), generator=g),
                                torch.randn(batch, seq, 16, generator=g),
                                torch.randint(-1, e, (batch, seq, 16), generator=g),
                                torch.randn(batch, seq, generator=g))]


def test_two_captured_steps_replay_in_turn_and_at_once():
    dev = _dev()
    turns, _ = CG.rotary_frequencies(64, device=dev)
    inputs = [chain_inputs(dev, s) for s in (1, 2)]
    others = [chain_inputs(dev, s) for s in (3, 4)]
    want = [[t.clone() for t in chain(p, turns)] for p in inputs]
    want_others = [[t.clone() for t in chain(p, turns)] for p in others]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for p in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(chain(p, turns))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    first = [[t.clone() for t in p] for p in inputs]
    for turn in range(4):
        print(f"replay {turn}", flush=True)
        data, expect = (first, want) if turn % 2 == 0 else (others, want_others)
        for p, d in zip(inputs, data):
            for t, s in zip(p, d):
                t.copy_(s)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):          # both at once
                graph.replay()
        torch.cuda.synchronize()
        eager = chain(others[0], turns)              # the program's own work between replays
        for out, e in zip(outs, expect):
            assert all(torch.equal(a, b) for a, b in zip(out, e))
        assert all(torch.equal(a, b) for a, b in zip(eager, want_others[0]))


def test_steps_on_two_streams_at_once():
    dev = _dev()
    turns, _ = CG.rotary_frequencies(64, device=dev)
    inputs = [chain_inputs(dev, s) for s in (5, 6)]
    want = [[t.clone() for t in chain(p, turns)] for p in inputs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(chain(inputs[i], turns))
    torch.cuda.synchronize()
    for runs, expect in zip(got, want):
        for out in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, expect))


def test_a_padded_batch_leaves_the_rows_behind_alone():
    # sequences of 150 and 90 rows: what stands in the padding does not reach the rows before it
    dev = _dev()
    turns, _ = CG.rotary_frequencies(64, device=dev)
    p = chain_inputs(dev, 7)
    p[7][1, 90:] = -1                                # no teacher there
    p[8][1, 90:] = 0.0
    want = [t.clone() for t in chain(p, turns)]
    for t in (p[0], p[1]):
        t[1, 90:] *= 1000.0
    got = chain(p, turns)
    for a, b in zip(got[:3], want):                  # loss, dx, dy
        assert torch.equal(a[0], b[0]) and torch.equal(a[1, :90], b[1, :90])
        assert not a[1, 90:].float().abs().any()


def test_operators_keep_the_registration_contracts():
    # schema, fake outputs, autograd registration and traced gradients (torch.library.opcheck)
    dev = _dev()
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev).requires_grad_()  # noqa: E731
    turns, _ = CG.rotary_frequencies(64, device=dev)
    heads = [r(2, 3, 40, 64) for _ in range(3)]
    x, y, gamma, gate = r(2, 9, 96), r(2, 9, 96), r(96), r(2, 1, 96)
    calls = [(CG.as_attention_grad_op(), heads), (CG.as_rotary_op(), (*heads[:2], torch.arange(40, device=dev), turns)),
             (CG.as_residual_norm_op(), (x, y, gamma, gamma.detach().clone().requires_grad_(), gate)),
             (CG.as_residual_norm_op(), (x, y, None, gamma, None)),
             (CG.as_distill_op(), (r(6, 50), torch.randn(6, 4, generator=g).to(dev),
                                   torch.randint(0, 50, (6, 4), generator=g).to(dev)))]
    for op, args in calls:
        print(f"contracts of {op}", flush=True)
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_autograd_registration", "test_faketensor",
                                                    "test_aot_dispatch_static"))


def test_a_traced_layer_gives_the_same_bits():
    dev = _dev()
    p, fixed = parameters(2, 33, 3, 64, 130, 8, seed=3)
    turns, _ = CG.rotary_frequencies(64, device=dev)
    here = {n: t.to(dev) for n, t in fixed.items()}
    ops = operators()
    print("traced layer", flush=True)
    results = []
    for wrap in (lambda f: f, lambda f: torch.compile(f, backend="aot_eager", fullgraph=True)):
        mine = {n: t.to(dev).requires_grad_() for n, t in p.items()}
        loss = wrap(lambda q: layer(q, here, turns, 3, False, ops))(mine)
        results.append([loss.detach(), *torch.autograd.grad(loss.sum(), list(mine.values()))])
    assert all(torch.equal(a, b) for a, b in zip(*results))
