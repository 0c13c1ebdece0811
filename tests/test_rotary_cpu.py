"""Rotary positions without a GPU: frequencies, refusals, metadata calls."""
import math

import pytest
import torch

import neptune_codegen as CG


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


Q, K, P, T = meta(2, 4, 9, 64), meta(2, 1, 9, 64), meta(9, dtype=torch.int64), meta(16, dtype=torch.float64)


@pytest.mark.parametrize("args,kw,error", [
    ((meta(2, 4, 9, 64, dtype=torch.float64), None, P, T), {}, TypeError), ((meta(4, 9, 64), None, P, T), {}, ValueError),
    ((Q, meta(2, 1, 8, 64), P, T), {}, ValueError), ((Q, meta(2, 1, 9, 64, dtype=torch.float16), P, T), {}, ValueError),
    ((Q, K, meta(8, dtype=torch.int64), T), {}, ValueError), ((Q, K, meta(1, 9, dtype=torch.int64), T), {}, ValueError),
    ((Q, K, meta(9, dtype=torch.float32), T), {}, TypeError), ((Q, K, P, meta(16, dtype=torch.float32)), {}, TypeError),
    ((Q, K, P, meta(33, dtype=torch.float64)), {}, ValueError), ((Q, K, P, meta(0, dtype=torch.float64)), {}, ValueError),
    ((Q, K, None, T), {}, TypeError), ((Q, K, P, T), {"magnitude": math.nan}, ValueError),
    ((torch.zeros(1, 1, 1, 4), None, torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.float64)), {}, ValueError)])
def test_refusals(args, kw, error):
    for run in (CG.run_rotary, CG.run_rotary_backward):
        with pytest.raises(error):
            run(*args, **kw)


def test_metadata_calls():
    q, k = CG.run_rotary(Q, K, P, T)
    assert q.shape == Q.shape and k.shape == K.shape and q.dtype == Q.dtype
    assert CG.run_rotary_backward(Q, None, meta(2, 9, dtype=torch.int32), T, interleaved=True)[1] is None
    op = CG.as_rotary_op()
    assert op is CG.as_rotary_op(1.0, False) and op(Q, K, P, T)[1].shape == K.shape


def test_frequencies():
    turns, magnitude = CG.rotary_frequencies(8, base=100.0, device="cpu")
    assert magnitude == 1.0 and turns.dtype == torch.float64
    torch.testing.assert_close(2 * math.pi * turns, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75]).double(),
                               rtol=1e-7, atol=0)
    linear, _ = CG.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear * 4, turns)
    ntk, _ = CG.rotary_frequencies(8, base=100.0, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == turns[0] and abs(ntk[-1] * 4 / turns[-1] - 1) < 1e-12
    parts, magnitude = CG.rotary_frequencies(128, scaling="parts", factor=8.0, original_length=4096, device="cpu")
    plain, _ = CG.rotary_frequencies(128, device="cpu")
    kept = parts / plain
    assert abs(magnitude - (0.1 * math.log(8) + 1)) < 1e-15
    assert (kept[4096 * plain > 32] == 1).all() and ((kept * 8 - 1).abs()[4096 * plain < 1] < 1e-12).all()
    assert (kept.diff() <= 0).all()


@pytest.mark.parametrize("kw", [{"part": 7}, {"part": 0}, {"base": 0.0}, {"scaling": "other"}, {"factor": 2.0},
                                {"scaling": "linear", "factor": 0.5}, {"scaling": "parts", "factor": 2.0},
                                {"scaling": "ntk", "factor": 2.0, "part": 2},
                                {"scaling": "parts", "factor": 2.0, "original_length": 100, "slow": 5.0, "fast": 5.0}])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        CG.rotary_frequencies(**{"part": 8, "device": "cpu", **kw})
