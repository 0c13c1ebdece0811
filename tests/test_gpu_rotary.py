"""Rotary positions against complex products in 64 bits.

Tolerance: cosine and sine are within 2^-22 (their argument within 2^-24, three roundings), the products
and the sum add 2^-23, all relative to |a| + |b| of the pair times the magnitude; then half a step of the
output's type.  Copied elements are equal bit by bit.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


def turned(x, positions, turns, magnitude, interleaved, sign):
    """(result, |a| + |b| of each element's pair) in float64 on the CPU."""
    x, positions, turns = x.double().cpu(), positions.cpu(), turns.cpu()
    part = 2 * len(turns)
    if positions.ndim == 1:
        positions = positions.unsqueeze(0)
    turn = positions.double()[:, None, :, None] * turns
    unit = torch.polar(torch.full_like(turn, magnitude), sign * 2 * math.pi * (turn - turn.round()))
    pairs = x[..., :part].unflatten(-1, (part // 2, 2) if interleaved else (2, part // 2))
    if not interleaved:
        pairs = pairs.transpose(-1, -2)
    out = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    size = pairs.abs().sum(-1, keepdim=True).expand_as(pairs)
    if not interleaved:
        out, size = out.transpose(-1, -2), size.transpose(-1, -2)
    rest = x[..., part:]
    return torch.cat((out.flatten(-2), rest), -1), torch.cat((size.flatten(-2), torch.zeros_like(rest)), -1)


def heads(b, h, s, d, dtype, dev, layout, seed):
    g = torch.Generator().manual_seed(seed)
    if layout == "bshd":
        return torch.randn(b, s, h, d, generator=g).to(dtype).to(dev).transpose(1, 2)
    return torch.randn(b, h, s, d, generator=g).to(dtype).to(dev)


def near(got, x, positions, turns, magnitude, interleaved, sign):
    want, size = turned(x, positions, turns, magnitude, interleaved, sign)
    part = 2 * len(turns)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert torch.equal(got[..., part:], x[..., part:])
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 1e-30
    ratio = ((got.double().cpu() - want).abs() / (2.0 ** -21 * magnitude * size + u * want.abs() + tiny)).max().item()
    assert ratio <= 1.0, ratio


CASES = [  # batch, heads of q and k, seq, dim, part, layout
    (1, 1, 1, 1, 64, 64, "bhsd"), (2, 32, 8, 1, 128, 128, "bshd"), (3, 4, 2, 33, 64, 32, "bshd"),
    (1, 2, 2, 100, 80, 40, "bhsd"), (2, 3, 1, 17, 50, 24, "bshd"), (1, 5, 0, 9, 6, 2, "bhsd"),
    (2, 8, 8, 300, 256, 256, "bhsd"), (1, 9, 4, 65, 24, 22, "bshd"), (1, 3, 3, 7, 7, 6, "bhsd")]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,hk,s,d,part,layout", CASES)
def test_rotation_and_its_transpose(b, hq, hk, s, d, part, layout, dtype, interleaved):
    dev = _dev()
    print(f"rotary {b}x{s} {hq}+{hk} heads d={d}/{part} {layout} {dtype} interleaved={interleaved}", flush=True)
    q, k = heads(b, hq, s, d, dtype, dev, layout, 0), heads(b, hk, s, d, dtype, dev, layout, 1)
    turns, magnitude = CG.rotary_frequencies(part, scaling="parts", factor=4.0, original_length=2048, device=dev)
    far = torch.arange(s, device=dev) + torch.tensor([1 << 20, 12345, 7], device=dev)[:b, None]
    for positions in (far, far[0].to(torch.int32)):
        for run, sign in ((CG.run_rotary, 1), (CG.run_rotary_backward, -1)):
            for _ in range(2):                       # the second is the seen call
                qo, ko = run(q, k if hk else None, positions, turns, magnitude=magnitude, interleaved=interleaved)
                near(qo, q, positions, turns, magnitude, interleaved, sign)
                if hk:
                    near(ko, k, positions, turns, magnitude, interleaved, sign)
                else:
                    assert ko is None


def test_far_and_negative_positions():
    dev = _dev()
    x = heads(1, 1, 6, 64, torch.float32, dev, "bhsd", 2)
    positions = torch.tensor([0, -1, (1 << 31) - 1, 1 << 40, -(1 << 33) - 7, 3], device=dev)
    turns, _ = CG.rotary_frequencies(64, device=dev)
    print("rotary far positions", flush=True)
    qo, _ = CG.run_rotary(x, None, positions, turns)
    # (a 64-bit product of 2^40 turns is itself within 2^-14 of a turn in both)
    for i in (0, 1, 2, 5):
        near(qo[:, :, i:i + 1].contiguous(), x[:, :, i:i + 1], positions[i:i + 1], turns, 1.0, False, 1)
    norm = lambda t: t[..., :32].square() + t[..., 32:].square()  # noqa: E731
    assert ((norm(qo) - norm(x)).abs() <= 2.0 ** -19 * norm(x)).all()
    assert torch.equal(qo[0, 0, 0], x[0, 0, 0])


def test_strides_alignment_and_copies():
    dev = _dev()
    turns, _ = CG.rotary_frequencies(32, device=dev)
    positions = torch.arange(20, device=dev)
    wide = heads(2, 3, 20, 83, torch.bfloat16, dev, "bhsd", 3)
    print("rotary strides", flush=True)
    for q in (wide[..., :64], wide[..., 8:72], wide[..., 3:67], wide[..., :64].transpose(2, 3).contiguous().transpose(2, 3),
              wide[:, :1, :, :64].expand(2, 3, 20, 64)):
        qo, ko = CG.run_rotary(q, q, positions, turns)
        assert torch.equal(qo, ko) and torch.equal(qo, CG.run_rotary(q.contiguous(), None, positions, turns)[0])
        near(qo, q, positions, turns, 1.0, False, 1)
    strided = torch.arange(40, device=dev)[::2]
    assert torch.equal(CG.run_rotary(wide[..., :64], None, strided, turns)[0],
                       CG.run_rotary(wide[..., :64], None, strided.contiguous(), turns)[0])


def test_registered_operator_and_captured_replays():
    dev = _dev()
    turns, _ = CG.rotary_frequencies(64, device=dev)
    q, k = heads(2, 4, 30, 64, torch.bfloat16, dev, "bshd", 4), heads(2, 2, 30, 64, torch.bfloat16, dev, "bshd", 5)
    positions = torch.arange(30, device=dev).expand(2, 30).contiguous()
    op = CG.as_rotary_op(interleaved=True)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k)]
    print("rotary through autograd", flush=True)
    out = op(*leaves, positions, turns)
    grads = [torch.randn(t.shape, generator=torch.Generator().manual_seed(6)).to(t.dtype).to(dev) for t in out]
    got = torch.autograd.grad(out, leaves, grads)
    want = CG.run_rotary_backward(*grads, positions, turns, interleaved=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = CG.run_rotary(q, k, positions, turns)
    for i in range(4):
        positions.add_(1000)
        graph.replay()
        want = CG.run_rotary(q, k, positions, turns)
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1]), i
    empty = torch.empty(2, 0, 30, 64, dtype=torch.bfloat16, device=dev)
    assert op(q, empty, positions, turns)[1].shape == empty.shape
    none = torch.empty(0, 4, 30, 64, dtype=torch.bfloat16, device=dev)
    assert CG.run_rotary(none, None, positions[0], turns)[0].shape == none.shape
