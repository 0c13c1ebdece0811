"""The residual norm and its gradients against the formulas in 64 bits, by automatic differentiation
of the forward definition.

Tolerances.  A row's sum of squares runs through at most 64 additions one after another and the rate
adds an ulp, so rates are within 2^-18; an element then is a product of a few factors: 2^-17 of its own
terms' sizes, plus half a step of the output's type.  Gradients of a row subtract means of products of
such elements: 2^-16 of the row's largest terms.  Column sums over rows add 2^-16 of the sum of the
terms' sizes.
"""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import residual_norm as RN

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


def make(lead, n, dtype, after=True, gate=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": 2 * rand(*lead, n), "y": rand(*lead, n), "after": 1 + 0.2 * rand(n) if after else None,
         "before": 1 + 0.2 * rand(n), "gate": None if gate is None else 0.5 * rand(*gate, n),
         "dr": rand(*lead, n), "dh": rand(*lead, n)}
    return {k: None if v is None else v.to(dtype) for k, v in t.items()}


def formulas(t, scale):
    """Outputs, rates and gradients in float64."""
    leaf = {k: v.double().requires_grad_() for k, v in t.items() if v is not None and k not in ("dr", "dh")}
    rate_y = torch.ones_like(leaf["x"][..., :1])
    c = leaf["y"]
    if "after" in leaf:
        rate_y = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
        c = c * rate_y * leaf["after"]
    block = scale * c * leaf["gate"] if "gate" in leaf else scale * c
    r = leaf["x"] + block
    rate_r = (r.square().mean(-1, keepdim=True) + EPS).rsqrt()
    h = r * rate_r * leaf["before"]
    grads = torch.autograd.grad((r, h), tuple(leaf.values()), (t["dr"].double(), t["dh"].double()))
    return r.detach(), h.detach(), torch.cat((rate_y, rate_r), -1).detach(), dict(zip(leaf, grads)), block.detach()


def call(t, scale, dev, **kw):
    d = {k: None if v is None else v.to(dev) for k, v in t.items()}
    out = CG.run_residual_norm(d["x"], d["y"], d["after"], d["before"], gate=d["gate"], residual_scale=scale,
                               eps=EPS, return_stats=True)
    back = lambda: CG.run_residual_norm_backward(  # noqa: E731
        d["dr"], d["dh"], d["x"], d["y"], d["after"], d["before"], out[2], gate=d["gate"], residual_scale=scale)
    return d, out, back


def check(t, scale, dev):
    d, (r, h, stats), back = call(t, scale, dev)
    again = CG.run_residual_norm(d["x"], d["y"], d["after"], d["before"], gate=d["gate"], residual_scale=scale,
                                 eps=EPS)
    assert torch.equal(r, again[0]) and torch.equal(h, again[1])
    grads = dict(zip(("x", "y", "after", "before", "gate"), back()))
    for a, b in zip(grads.values(), back()):
        assert (a is None and b is None) or torch.equal(a, b)
    want_r, want_h, want_s, want, block = formulas(t, scale)
    u, dtype = torch.finfo(t["x"].dtype).eps / 2, t["x"].dtype
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30

    def near(name, got, ref, off):
        assert got.shape == ref.shape and got.is_contiguous()
        ratio = ((got.double().cpu() - ref).abs() / (off + u * ref.abs() + tiny)).max().item()
        assert ratio <= 1.0, (name, ratio)

    size_r = t["x"].double().abs() + block.abs()
    near("residual", r, want_r, 2.0 ** -17 * size_r)
    near("normed", h, want_h, 2.0 ** -16 * size_r * want_s[..., 1:] * t["before"].double().abs())
    assert ((stats.double().cpu() - want_s) / want_s).abs().max() <= 2.0 ** -17
    # terms of dx: dr and rate_r a; of dy: s g dx and its row
    a = (t["dh"].double() * t["before"].double()).abs()
    k = size_r * want_s[..., 1:]
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    size_x = t["dr"].double().abs() + want_s[..., 1:] * (a + k * mean(a * k))
    near("dx", grads["x"], want["x"], 2.0 ** -16 * size_x)
    w = torch.full_like(size_x, abs(scale)) if t["gate"] is None else abs(scale) * t["gate"].double().abs()
    unit = (t["y"].double() * want_s[..., :1]).abs()
    dc = w * size_x
    if t["after"] is not None:
        b = dc * t["after"].double().abs()
        near("dy", grads["y"], want["y"], 2.0 ** -15 * want_s[..., :1] * (b + unit * mean(b * unit)))
        near("dafter", grads["after"], want["after"], 2.0 ** -15 * (dc * unit).flatten(0, -2).sum(0))
        c = unit * t["after"].double().abs()
    else:
        near("dy", grads["y"], want["y"], 2.0 ** -15 * dc)
        assert grads["after"] is None
        c = unit
    near("dbefore", grads["before"], want["before"], 2.0 ** -15 * (t["dh"].double().abs() * k).flatten(0, -2).sum(0))
    if t["gate"] is None:
        assert grads["gate"] is None
    else:
        near("dgate", grads["gate"], want["gate"], 2.0 ** -15 * (abs(scale) * size_x * c).sum_to_size(want["gate"].shape))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,n,after,gate", [
    ((1,), 1, True, None), ((3,), 5, True, (3,)), ((2, 7), 64, True, (2, 1)), ((9,), 1000, False, None),
    ((4, 33), 1024, True, (4, 1)), ((700,), 96, True, ()), ((2, 3, 5), 333, True, (2, 3, 1)),
    ((1, 130), 4096, True, (1, 1)), ((40,), 2999, False, (40,)), ((5,), 8192, True, (5,)), ((2, 3), 16384, True, (2, 1)),
    ((3,), 10007, True, ()), ((600, 2), 128, True, (600, 1)), ((1000,), 16, False, ())])
def test_outputs_and_gradients_match_the_formulas(lead, n, after, gate, dtype):
    dev = _dev()
    print(f"residual norm {lead} x {n} after={after} gate={gate} {dtype}", flush=True)
    check(make(lead, n, dtype, after, gate), 0.5, dev)


def test_strided_operands_and_copies():
    dev = _dev()
    t = make((6, 10), 520, torch.bfloat16, True, (6, 1), seed=1)
    d, out, back = call(t, 1.5, dev)
    want = (*out, *back())
    print("residual norm strides", flush=True)
    wide = torch.zeros(6, 10, 1100, dtype=torch.bfloat16, device=dev)
    for offset in (0, 8, 3):                      # aligned, aligned, element by element
        wide[..., offset:offset + 520] = d["x"]
        x = wide[..., offset:offset + 520]
        y = d["y"].transpose(0, 1).contiguous().transpose(0, 1)          # rows of two strides: copied
        out = CG.run_residual_norm(x, y, d["after"], d["before"], gate=d["gate"], residual_scale=1.5, eps=EPS,
                                   return_stats=True)
        grads = CG.run_residual_norm_backward(d["dr"], d["dh"], x, y, d["after"], d["before"], out[2],
                                              gate=d["gate"], residual_scale=1.5)
        for a, b in zip((*out, *grads), want):
            assert torch.equal(a, b), offset
    zeros = torch.zeros_like(d["dr"])
    a = CG.run_residual_norm_backward(None, d["dh"], d["x"], d["y"], d["after"], d["before"], out[2],
                                      gate=d["gate"], residual_scale=1.5)
    b = CG.run_residual_norm_backward(zeros, d["dh"], d["x"], d["y"], d["after"], d["before"], out[2],
                                      gate=d["gate"], residual_scale=1.5)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_rows_of_zeros_and_non_finite_rows_stay_apart():
    dev = _dev()
    t = make((12,), 600, torch.float32, True, None, seed=2)
    t["x"][3], t["y"][3] = 0.0, 0.0
    t["x"][5, 7], t["y"][6, 9], t["dh"][7, 0] = float("nan"), float("inf"), float("nan")
    print("residual norm edge rows", flush=True)
    _, (r, h, _), back = call(t, 1.0, dev)
    dx, dy, dafter, dbefore, _ = back()
    want_r, want_h, _, want, _ = formulas(t, 1.0)
    fine = [0, 1, 2, 3, 4, 8, 9, 10, 11]
    for a, b in ((r, want_r), (h, want_h), (dx, want["x"]), (dy, want["y"])):
        assert torch.isfinite(a[fine]).all()
        # rows of size 1; the zero row's rate is 1000
        assert (a[fine].double().cpu() - b[fine]).abs().max() <= 2.0 ** -14 * max(1.0, b[fine].abs().max().item())
    assert not r[3].any() and not h[3].any()
    assert dx[7].isnan().any() and h[6].isnan().any() and dbefore.isnan().any()


def test_gradient_matches_differences():
    dev = _dev()
    t = make((3,), 24, torch.float32, True, (3,), seed=3)
    _, _, back = call(t, 0.7, dev)
    grads = dict(zip(("x", "y", "after", "before", "gate"), back()))
    print("residual norm differences", flush=True)
    step = 1e-4
    for name in grads:
        for at in (0, grads[name].numel() - 1):
            values = []
            for sign in (1, -1):
                s = {k: v.double().clone() for k, v in t.items()}
                s[name].view(-1)[at] += sign * step
                r, h, *_ = formulas(s, 0.7)
                values.append(((r * s["dr"]).sum() + (h * s["dh"]).sum()).item())
            slope = (values[0] - values[1]) / (2 * step)
            # the differences' own error is step^2 times a third derivative of order 1
            assert abs(grads[name].view(-1)[at].item() - slope) <= 1e-5 * max(1.0, abs(slope)), (name, at)


def test_registered_operator_and_captured_replays():
    dev = _dev()
    t = make((4, 50), 256, torch.bfloat16, True, (4, 1), seed=4)
    d, out, back = call(t, 0.5, dev)
    want = back()
    op = CG.as_residual_norm_op(0.5, EPS)
    leaves = [d[k].clone().requires_grad_() for k in ("x", "y", "after", "before", "gate")]
    print("residual norm through autograd", flush=True)
    r, h, _ = op(*leaves)
    got = torch.autograd.grad((r, h), leaves, (d["dr"], d["dh"]), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    only = torch.autograd.grad(h, leaves[0], d["dh"])[0]
    assert torch.equal(only, CG.run_residual_norm_backward(None, d["dh"], *(d[k] for k in ("x", "y", "after", "before")),
                                                           out[2], gate=d["gate"], residual_scale=0.5)[0])
    plain = CG.as_residual_norm_op(0.5, EPS)(leaves[0], leaves[1], None, leaves[3], None)
    assert plain[0].shape == d["x"].shape
    torch.autograd.grad(plain[1], leaves[:2] + leaves[3:4], d["dh"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = CG.run_residual_norm(d["x"], d["y"], d["after"], d["before"], gate=d["gate"], residual_scale=0.5,
                                   eps=EPS, return_stats=True)
        got = CG.run_residual_norm_backward(d["dr"], d["dh"], d["x"], d["y"], d["after"], d["before"], out[2],
                                            gate=d["gate"], residual_scale=0.5)
    for i in range(4):
        d["y"].copy_(torch.randn(t["y"].shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        graph.replay()
        fresh = CG.run_residual_norm(d["x"], d["y"], d["after"], d["before"], gate=d["gate"], residual_scale=0.5,
                                     eps=EPS, return_stats=True)
        ref = CG.run_residual_norm_backward(d["dr"], d["dh"], d["x"], d["y"], d["after"], d["before"], fresh[2],
                                            gate=d["gate"], residual_scale=0.5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*out, *got), (*fresh, *ref))), i


def test_no_rows():
    dev = _dev()
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    g = torch.ones(64, dtype=torch.bfloat16, device=dev)
    r, h, s = CG.run_residual_norm(x, x, g, g, gate=g, return_stats=True)
    assert r.shape == h.shape == (0, 64) and s.shape == (0, 2)
    grads = CG.run_residual_norm_backward(x, x, x, x, g, g, s, gate=g)
    assert grads[0].shape == (0, 64) and not grads[2].any() and not grads[3].any() and not grads[4].any()
    assert RN._chunks(5, 1, 5, "none", 8) == (1, 1)
