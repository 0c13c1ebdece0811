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
