"""Numbers of the training operators that fp32 cannot hold are refused, whether the call has data or not."""
import numpy as np
import pytest
import torch

import neptune_codegen as CG


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("temperature", [1e-19, 1e19, -1.0, float("nan"), float("inf"), 10 ** 400, np.float64(2.0)])
def test_temperatures(temperature):
    for rows in (4, 0):
        lists = meta(rows, 3, dtype=torch.float32), meta(rows, 3, dtype=torch.int64)
        with pytest.raises(ValueError, match="temperature"):
            CG.run_distill(meta(rows, 9), *lists, temperature=temperature)
        with pytest.raises(ValueError, match="temperature"):
            CG.run_distill_backward(meta(rows, dtype=torch.float32), meta(rows, 9), *lists,
                                    meta(rows, 2, dtype=torch.float32), temperature=temperature)
    with pytest.raises(ValueError, match="temperature"):
        CG.as_distill_op(temperature)


def test_temperatures_at_the_ends():
    lists = meta(4, 3, dtype=torch.float32), meta(4, 3, dtype=torch.int64)
    for temperature in (1e-18, 1, 1e18):
        assert CG.run_distill(meta(4, 9), *lists, temperature=temperature).shape == (4,)


@pytest.mark.parametrize("number", [1e300, -1e39, float("-inf"), float("nan"), 10 ** 400, False])
def test_residual_scales_and_magnitudes(number):
    x, g = meta(2, 64), meta(64)
    with pytest.raises(ValueError, match="residual_scale"):
        CG.run_residual_norm(x, x, None, g, residual_scale=number)
    with pytest.raises(ValueError, match="residual_scale"):
        CG.run_residual_norm_backward(None, x, x, x, None, g, meta(2, 2, dtype=torch.float32), residual_scale=number)
    with pytest.raises(ValueError, match="magnitude"):
        CG.run_rotary(meta(1, 2, 3, 64), None, meta(3, dtype=torch.int64), meta(32, dtype=torch.float64),
                      magnitude=number)


@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-39, -1e-6, 1e39, float("inf")])
def test_epsilons(eps):
    with pytest.raises(ValueError, match="eps"):
        CG.run_residual_norm(meta(2, 64), meta(2, 64), None, meta(64), eps=eps)


@pytest.mark.parametrize("scale", [1e-31, 1e39, -0.1, float("inf")])
def test_attention_scales(scale):
    q, lse = meta(1, 2, 8, 64), meta(1, 2, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="scale"):
        CG.run_attention_backward(q, q, q, q, q, lse, scale=scale)
