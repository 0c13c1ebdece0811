"""Gradients of the attention fold against the formulas in 64 bits, element by element.

Tolerance of each element, from the roundings the kernels make (u = half a step of the type, bf16
2^-8, fp16 2^-11): P and dS are rounded to the type for their products, O is (so delta is off by up
to u sum |dO O|), and the result is.  The fp32 rest (scores, exponential, sums of up to some
thousand terms) gets 2^-13 of the sums of absolute values.
"""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import attention_backward as AB

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


def formulas(grad, q, k, v, scale, causal, grad_lse=None, u=0.0, rest=0.0):
    """((dq, dk, dv), their tolerances) in float64 on the CPU."""
    g, q, k, v = (t.double().cpu() for t in (grad, q, k, v))
    s = scale * (q @ k.transpose(2, 3))
    hidden = torch.zeros(s.shape[2:], dtype=torch.bool)
    if causal:
        hidden = torch.ones_like(hidden).triu_(1)
    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    out = p @ v
    dp = g @ v.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    if grad_lse is not None:
        delta = delta - grad_lse.double().cpu().unsqueeze(-1)
    ds = p * (dp - delta)
    grads = (scale * (ds @ k), scale * (ds.transpose(2, 3) @ q), p.transpose(2, 3) @ g)
    size = (g.abs() * out.abs()).sum(-1, keepdim=True)
    if grad_lse is not None:
        size = size + grad_lse.double().cpu().abs().unsqueeze(-1)
    # P's relative error: the exponent's (a score's sum and lse, both in 32 bits) and the rounding
    # to the type; P <= 1 and the exponential are within `rest`
    ds_off = u * ds.abs() + p * (u * size + rest * (g.abs() @ v.abs().transpose(2, 3) + size))
    off = (scale * (ds_off @ k.abs()), scale * (ds_off.transpose(2, 3) @ q.abs()),
           (u + rest) * (p.transpose(2, 3) @ g.abs()))
    return grads, tuple((1 + u) * o + u * d.abs() + 2.0 ** -24 for o, d in zip(off, grads))


def check(got, grad, q, k, v, scale, causal, grad_lse=None):
    u = torch.finfo(q.dtype).eps / 2
    want, off = formulas(grad, q, k, v, scale, causal, grad_lse, u, 2.0 ** -13)
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, off):
        assert a.dtype == q.dtype and a.is_contiguous() and a.shape == b.shape
        ratio = ((a.double().cpu() - b).abs() / t).max().item() if a.numel() else 0.0
        assert ratio <= 1.0, (name, ratio)


def inputs(shape, sk, dtype, dev, layout="bhsd", seed=0, grad_scale=1.0):
    B, H, Sq, D = shape
    g = torch.Generator().manual_seed(seed)

    def one(s, scale=1.0):
        if layout == "bshd":
            return (scale * torch.randn(B, s, H, D, generator=g)).to(dtype).to(dev).transpose(1, 2)
        return (scale * torch.randn(B, H, s, D, generator=g)).to(dtype).to(dev)

    return one(Sq), one(sk), one(sk), one(Sq, grad_scale)


CASES = [  # (B, H, Sq, D), Sk, causal, layout
    ((1, 1, 1, 64), 1, False, "bhsd"), ((1, 2, 1, 128), 1, True, "bhsd"),
    ((1, 1, 32, 64), 32, False, "bhsd"), ((1, 1, 64, 128), 64, True, "bhsd"),
    ((2, 3, 77, 64), 77, True, "bshd"), ((1, 2, 130, 128), 130, True, "bshd"),
    ((1, 2, 257, 128), 300, False, "bhsd"), ((1, 2, 300, 64), 257, True, "bhsd"),
    ((2, 1, 65, 256), 65, True, "bshd"), ((1, 2, 140, 256), 201, False, "bhsd"),
    ((1, 1, 1, 128), 513, False, "bhsd"), ((1, 1, 513, 64), 1, False, "bhsd"),
    ((1, 1, 100, 128), 400, True, "bhsd"), ((1, 1, 400, 256), 100, True, "bhsd"),
    ((1, 2, 1000, 128), 1000, True, "bshd"), ((1, 2, 700, 64), 900, False, "bshd"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,sk,causal,layout", CASES)
def test_gradients_match_the_formulas(shape, sk, causal, layout, dtype):
    dev = _dev()
    print(f"attention backward {shape} sk={sk} causal={causal} {layout} {dtype}", flush=True)
    q, k, v, grad = inputs(shape, sk, dtype, dev, layout)
    out, lse = CG.run_attention(q, k, v, causal=causal, return_lse=True)
    got = CG.run_attention_backward(grad, q, k, v, out, lse, causal=causal)
    check(got, grad, q, k, v, 1.0 / math.sqrt(shape[3]), causal)
    again = CG.run_attention_backward(grad, q, k, v, out, lse, causal=causal)    # the seen call
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("plan", [(1, 3, 3), (2, 2, 4), (1, 1, 2), (2, 5, 1)])
@pytest.mark.parametrize("shape,sk,causal", [((1, 2, 700, 128), 700, True), ((2, 1, 300, 128), 650, False),
                                             ((1, 1, 650, 64), 300, True), ((1, 2, 200, 128), 500, True)])
def test_split_ranges_and_two_blocks_match_the_formulas(shape, sk, causal, plan):
    dev = _dev()
    print(f"attention backward plan {plan} {shape} sk={sk} causal={causal}", flush=True)
    q, k, v, grad = inputs(shape, sk, torch.bfloat16, dev, "bshd", seed=1)
    out, lse = CG.run_attention(q, k, v, causal=causal, return_lse=True)
    if shape[3] != 128:
        plan = (1, *plan[1:])
    got = AB._run(grad, q, k, v, out, lse, None, None, causal, plan=plan)
    check(got, grad, q, k, v, 1.0 / math.sqrt(shape[3]), causal)


@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_split_ranges_at_head_dim_256(dtype, parts):
    dev = _dev()
    q, k, v, grad = inputs((1, 2, 420, 256), 420, dtype, dev, seed=2)
    print(f"attention backward d=256 {dtype} parts={parts}", flush=True)
    out, lse = CG.run_attention(q, k, v, causal=True, return_lse=True)
    got = AB._run(grad, q, k, v, out, lse, None, None, True, plan=(1, parts, parts))
    check(got, grad, q, k, v, 1.0 / 16, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_gradient_of_the_logsumexp_and_another_scale(dtype, causal):
    dev = _dev()
    print(f"attention backward grad_lse {dtype} causal={causal}", flush=True)
    q, k, v, grad = inputs((2, 2, 150, 64), 150, dtype, dev, seed=3)
    grad_lse = torch.randn(2, 2, 150, generator=torch.Generator().manual_seed(4)).to(dev)
    out, lse = CG.run_attention(q, k, v, scale=0.3, causal=causal, return_lse=True)
    got = CG.run_attention_backward(grad, q, k, v, out, lse, grad_lse=grad_lse, scale=0.3, causal=causal)
    check(got, grad, q, k, v, 0.3, causal, grad_lse)


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 10])
def test_fp16_gradients_keep_their_precision_at_any_size(size):
    """dS in fp16 is scaled per head: gradients of 2^-12 are not lost to subnormals and those of 2^10
    do not overflow (their own rounding to fp16 is in the tolerance, an absolute 2^-24)."""
    dev = _dev()
    print(f"attention backward fp16 gradients of size {size}", flush=True)
    q, k, v, grad = inputs((1, 2, 600, 128), 600, torch.float16, dev, seed=5, grad_scale=size)
    out, lse = CG.run_attention(q, k, v, causal=True, return_lse=True)
    got = CG.run_attention_backward(grad, q, k, v, out, lse, causal=True)
    check(got, grad, q, k, v, 1.0 / math.sqrt(128), True)


def test_strides_and_copies_give_the_same_bits():
    """Strided, expanded and unaligned operands (the last two copied) against contiguous ones."""
    dev = _dev()
    q, k, v, grad = inputs((2, 3, 130, 64), 130, torch.bfloat16, dev, "bshd", seed=6)
    k = k[:, :1].expand(2, 3, 130, 64)                              # one key head for all
    base = torch.zeros(2 * 3 * 130 * 64 + 1, dtype=torch.bfloat16, device=dev)
    base[1:] = v.contiguous().view(-1)
    unaligned = base[1:].view(2, 3, 130, 64)
    print("attention backward strides", flush=True)
    out, lse = CG.run_attention(q, k, v, causal=True, return_lse=True)
    want = CG.run_attention_backward(grad.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(),
                                     out, lse, causal=True)
    for g in (grad, grad.contiguous()):
        got = CG.run_attention_backward(g, q, k, unaligned, out.transpose(1, 2).contiguous().transpose(1, 2),
                                        lse.transpose(1, 2).contiguous().transpose(1, 2), causal=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    row = grad[:, :, :1].expand(2, 3, 130, 64)                      # rows that overlap
    got = CG.run_attention_backward(row, q, k, v, out, lse, causal=True)
    want = CG.run_attention_backward(row.contiguous(), q, k, v, out, lse, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def masked_formulas(grad, q, k, v, out, lse, scale):
    """The causal gradients pair by pair from the forward pass's out and lse (a row with an infinite
    score has a logsumexp of NaN there): a hidden pair adds nothing, whatever it holds."""
    g, q, k, v, out = (t[0, 0].double().cpu() for t in (grad, q, k, v, out))
    n = q.shape[0]
    seen = torch.ones(n, n, dtype=torch.bool).tril_()
    s = (scale * (q[:, None] * k[None]).sum(-1)).masked_fill(~seen, -math.inf)
    p = torch.where(seen, (s - lse[0, 0].double().cpu().unsqueeze(-1)).exp(), 0.0)
    dp = torch.where(seen, (g[:, None] * v[None]).sum(-1), 0.0)
    ds = torch.where(seen, p * (dp - (g * out).sum(-1, keepdim=True)), 0.0)
    pick = lambda w, x: torch.where(seen[:, :, None], w[:, :, None] * x, 0.0)  # noqa: E731
    return (scale * pick(ds, k[None]).sum(1), scale * pick(ds, q[:, None]).sum(0), pick(p, g[:, None]).sum(0))


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (128, torch.float16),
                                       (256, torch.bfloat16)])
@pytest.mark.parametrize("where,row,value", [("q", 70, math.inf), ("grad", 70, math.nan), ("k", 70, -math.inf),
                                             ("v", 70, math.nan), ("grad", 149, math.inf), ("k", 149, math.nan),
                                             ("q", 31, math.nan), ("v", 64, math.inf)])
def test_hidden_infinities_and_nans_reach_nothing(where, row, value, dim, dtype):
    dev = _dev()
    print(f"attention backward {value} in {where}[{row}] d={dim} {dtype}", flush=True)
    t = dict(zip("qkvg", inputs((1, 1, 150, dim), 150, dtype, dev, seed=7)))
    t["grad"] = t.pop("g")
    t[where][0, 0, row, 3] = value
    q, k, v, grad = t["q"], t["k"], t["v"], t["grad"]
    scale = 1.0 / math.sqrt(dim)
    out, lse = CG.run_attention(q, k, v, causal=True, return_lse=True)
    got = CG.run_attention_backward(grad, q, k, v, out, lse, causal=True)
    want = masked_formulas(grad, q, k, v, out, lse, scale)
    u = torch.finfo(dtype).eps / 2
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        a = a[0, 0].double().cpu()
        fine = torch.isfinite(b)
        assert torch.equal(torch.isfinite(a), fine), (name, int((torch.isfinite(a) != fine).sum()))
        # the size of a row's terms bounds what their roundings add up to: sums of 150 terms at most
        off = (a - b)[fine].abs().max().item() if fine.any() else 0.0
        size = b[fine].abs().max().item() if fine.any() else 1.0
        assert off <= 16 * u * max(1.0, size), (name, off, size)
    for a, b in zip(got, CG.run_attention_backward(grad, q, k, v, out, lse, causal=True)):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_registered_operator_has_the_formulas_gradients():
    dev = _dev()
    op = CG.as_attention_grad_op(causal=True)
    q, k, v, grad = inputs((1, 2, 140, 64), 140, torch.bfloat16, dev, "bshd", seed=8)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    print("attention backward through autograd", flush=True)
    out, lse = op(*leaves)
    assert torch.equal(out, CG.run_attention(q, k, v, causal=True))
    grad_lse = torch.randn(lse.shape, generator=torch.Generator().manual_seed(9)).to(dev)
    got = torch.autograd.grad((out, lse), leaves, (grad, grad_lse), retain_graph=True)
    check(got, grad, q, k, v, 1.0 / 8, True, grad_lse)
    check(torch.autograd.grad(out, leaves, grad, retain_graph=True), grad, q, k, v, 1.0 / 8, True)
    only = torch.autograd.grad(lse, leaves, grad_lse)
    check(only, torch.zeros_like(grad), q, k, v, 1.0 / 8, True, grad_lse)


def test_captured_gradients_replay():
    dev = _dev()
    q, k, v, grad = inputs((1, 4, 300, 128), 300, torch.float16, dev, seed=10)
    out, lse = CG.run_attention(q, k, v, causal=True, return_lse=True)
    CG.run_attention_backward(grad, q, k, v, out, lse)
    print("attention backward captured", flush=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = CG.run_attention_backward(grad, q, k, v, out, lse)
    for i in range(4):
        grad.copy_(torch.randn(grad.shape, generator=torch.Generator().manual_seed(20 + i)).to(dev))
        graph.replay()
        want = CG.run_attention_backward(grad, q, k, v, out, lse)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_no_queries_give_zero_key_gradients():
    dev = _dev()
    q = torch.empty(1, 2, 0, 64, dtype=torch.bfloat16, device=dev)
    k = torch.randn(1, 2, 5, 64, device=dev).bfloat16()
    dq, dk, dv = CG.run_attention_backward(q, q, k, k, q, torch.empty(1, 2, 0, device=dev), causal=False)
    assert dq.shape == q.shape and not dk.any() and not dv.any()
