"""The registered attention operator with gradients refuses at its construction what its backward would."""
import pytest
import torch

import neptune_codegen as CG


@pytest.mark.parametrize("scale", [0, 0.0, -0.125, 1e-31, 2.0 ** -101, 2.0 ** 126, float("inf"), float("nan")])
def test_scales_that_the_backward_refuses(scale):
    with pytest.raises(ValueError, match="scale"):
        CG.as_attention_grad_op(scale)


@pytest.mark.parametrize("scale", [2.0 ** -100, 1, 0.125, 2.0 ** 125])
def test_scales_that_both_passes_take(scale):
    q = torch.empty((1, 2, 8, 64), dtype=torch.bfloat16, device="meta", requires_grad=True)
    out, lse = CG.as_attention_grad_op(scale)(q, q, q)
    (dq,) = torch.autograd.grad((out, lse), q, (out, lse))
    assert dq.shape == q.shape
