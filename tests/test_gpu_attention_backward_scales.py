"""Attention's gradients where the output's gradients of a head's rows differ in size by powers of two (a batch
with weights per token, a scaled loss).

Tolerances: those of test_gpu_attention_backward.py, and in fp16 the half step of a subnormal dS.  A query's dS
words are dS 2^(15 - e) with its bound |dO_i| max|v| + |delta_i| in [2^(e-1), 2^e), so 2^-25 of them is 2^-39
of the bound at most; a key's share the largest bound 2 |dO| max|v| + |dlse| of the queries from its tile of 64
rows on (of all without the mask).  (Bounds are 2^-10 above the norms, which the factor 1.01 covers.)
"""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import attention_backward as AB
from test_gpu_attention_backward import _dev, formulas, inputs

pytestmark = pytest.mark.gpu


def subnormal(q, k, v, grad, grad_lse, scale, causal):
    """(dq, dk) that half steps of subnormal words make at most."""
    q, k, v, g = (t.double().cpu() for t in (q, k, v, grad))
    most = v.norm(dim=-1).amax(-1)[..., None]
    norm, lse = g.norm(dim=-1) * most, 0.0 if grad_lse is None else grad_lse.double().cpu().abs()
    seen = torch.ones(q.shape[2], k.shape[2], dtype=torch.float64)
    if causal:
        seen = seen.tril()
    own = 1.01 * (2 * norm + lse)                    # (|delta_i| <= |dO_i| max|v| + |dlse_i|)
    dq = 2.0 ** -39 * own[..., None] * (seen @ k.abs())
    after = torch.arange(q.shape[2])[None, :] >= torch.arange(k.shape[2])[:, None] // 64 * 64
    after = after if causal else torch.ones_like(after)
    theirs = torch.where(after, own[..., None, :], 0.0).amax(-1)
    dk = 2.0 ** -39 * theirs[..., None] * (seen.T @ q.abs())
    return scale * dq, scale * dk


def check(got, grad, q, k, v, scale, causal, grad_lse=None):
    u = torch.finfo(q.dtype).eps / 2
    want, off = formulas(grad, q, k, v, scale, causal, grad_lse, u, 2.0 ** -13)
    more = (*subnormal(q, k, v, grad, grad_lse, scale, causal), 0.0) if q.dtype == torch.float16 else (0.0,) * 3
    for name, a, b, t, m in zip(("dq", "dk", "dv"), got, want, off, more):
        ratio = ((a.double().cpu() - b).abs() / (t + m)).max().item()
        assert ratio <= 1.0, (name, ratio)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape,plan", [((1, 2, 400, 64), None), ((2, 1, 333, 128), None), ((1, 1, 500, 128), (2, 1, 1)),
                                        ((1, 2, 300, 128), (1, 2, 3)), ((1, 1, 260, 256), None), ((1, 3, 40, 64), None)])
@pytest.mark.parametrize("rows", ["mixed", "first", "last"])
def test_rows_of_different_sizes(rows, shape, plan, causal, dtype):
    dev = _dev()
    print(f"attention backward scales {rows} {shape} plan={plan} causal={causal} {dtype}", flush=True)
    q, k, v, grad = inputs(shape, shape[2], dtype, dev, seed=21)
    seq = shape[2]
    large = {"mixed": torch.rand(seq, generator=torch.Generator().manual_seed(22)) < 0.1,
             "first": torch.arange(seq) < min(64, seq // 2), "last": torch.arange(seq) >= seq - 5}[rows]
    grad = grad * torch.where(large, 2.0 ** 10, 2.0 ** -10).to(dev)[:, None].to(dtype)
    out, lse = CG.run_attention(q, k, v, causal=causal, return_lse=True)
    got = AB._run(grad, q, k, v, out, lse, None, None, causal, plan=plan)
    check(got, grad, q, k, v, 1.0 / math.sqrt(shape[3]), causal)


@pytest.mark.parametrize("causal", [True, False])
def test_one_large_gradient_of_the_logsumexp(causal):
    dev = _dev()
    print(f"attention backward large grad_lse causal={causal}", flush=True)
    q, k, v, grad = inputs((1, 2, 200, 64), 200, torch.float16, dev, seed=23, grad_scale=2.0 ** -9)
    grad_lse = torch.full((1, 2, 200), 2.0 ** -9, device=dev)
    grad_lse[:, :, 3] = 2.0 ** 12
    out, lse = CG.run_attention(q, k, v, causal=causal, return_lse=True)
    got = CG.run_attention_backward(grad, q, k, v, out, lse, grad_lse=grad_lse, causal=causal)
    check(got, grad, q, k, v, 1.0 / 8, causal, grad_lse)


def test_rows_without_a_gradient():
    dev = _dev()
    print("attention backward rows without a gradient", flush=True)
    q, k, v, grad = inputs((1, 2, 150, 128), 150, torch.float16, dev, seed=24)
    grad[:, :, 10:100] = 0
    out, lse = CG.run_attention(q, k, v, return_lse=True)
    got = CG.run_attention_backward(grad, q, k, v, out, lse)
    assert not got[0][:, :, 10:100].any()
    check(got, grad, q, k, v, 128 ** -0.5, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_that_every_query_passes_over(dim, causal):
    """One key takes all but e^-19 of each row, and the gradient is large: the other keys' dV are well above the
    type's smallest numbers, from P around 2^-27.  P's words hold 2^14 P, so a subnormal one is off by up to 2^-39."""
    dev = _dev()
    print(f"attention backward of passed-over keys {dim} causal={causal}", flush=True)
    q, k, v, grad = inputs((1, 2, 16, dim), 16 if causal else 64, torch.float16, dev, seed=25, grad_scale=2.0 ** 12)
    q, k = (1 + q / 16).half(), (k / 64).half()
    k[:, :, 0] = 19 / dim ** 0.5
    out, lse = CG.run_attention(q, k, v, causal=causal, return_lse=True)
    _, _, dv = CG.run_attention_backward(grad, q, k, v, out, lse, causal=causal)
    u = 2.0 ** -11
    (_, _, want), (_, _, off) = formulas(grad, q, k, v, dim ** -0.5, causal, None, u, 2.0 ** -13)
    off = off + 2.0 ** -39 * grad.double().cpu().abs().sum(2, keepdim=True)
    assert 2.0 ** -16 < want[:, :, 1:].abs().median() < 2.0 ** -9
    assert ((dv.double().cpu() - want).abs() / off).max() <= 1.0
