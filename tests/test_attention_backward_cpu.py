"""Attention's gradients without a GPU: refusals, metadata calls, launch choice, and every unit's
compilation."""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import attention_backward as AB


def meta(shape=(1, 2, 8, 64), dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def call(**kw):
    t = {"grad": meta(), "q": meta(), "k": meta(), "v": meta(), "out": meta(),
         "lse": meta((1, 2, 8), torch.float32), **kw}
    more = {n: t.pop(n) for n in ("grad_lse", "scale", "causal") if n in t}
    return CG.run_attention_backward(t["grad"], t["q"], t["k"], t["v"], t["out"], t["lse"], **more)


@pytest.mark.parametrize("kw,error", [
    ({"grad": meta((1, 2, 9, 64))}, ValueError), ({"grad": meta(dtype=torch.float16)}, ValueError),
    ({"out": meta((1, 2, 8, 128))}, ValueError), ({"grad": None}, TypeError),
    ({"lse": meta((1, 2, 8))}, ValueError), ({"lse": meta((1, 2, 9), torch.float32)}, ValueError),
    ({"grad_lse": meta((1, 2, 8), torch.float64)}, ValueError), ({"grad_lse": 1.0}, TypeError),
    ({"scale": 0.0}, ValueError), ({"scale": float("nan")}, ValueError), ({"k": meta((1, 2, 8, 128))}, ValueError),
    ({n: meta((1, 2, 8, 32)) for n in ("q", "k", "v", "grad", "out")}, NotImplementedError),
    ({n: meta(dtype=torch.float32) for n in ("q", "k", "v", "grad", "out")}, TypeError)])
def test_refusals(kw, error):
    with pytest.raises(error):
        call(**kw)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        CG.run_attention_backward(q, q, q, q, q, torch.zeros(1, 1, 4))


def test_metadata_calls():
    dq, dk, dv = call(k=meta((1, 2, 5, 64)), v=meta((1, 2, 5, 64)))
    assert dq.shape == (1, 2, 8, 64) and dk.shape == dv.shape == (1, 2, 5, 64)
    assert dq.dtype == dk.dtype == torch.bfloat16 and dq.device.type == "meta"
    op = CG.as_attention_grad_op(causal=False)
    assert op is CG.as_attention_grad_op(causal=False)
    out, lse = op(meta(), meta(), meta())
    assert out.shape == (1, 2, 8, 64) and lse.shape == (1, 2, 8) and lse.dtype == torch.float32


def test_launch_choice_follows_the_measured_shapes():
    # (units, sq, sk, head dim, causal): the cheapest of the sweep or within a few percent of it
    assert AB._plan(128, 4096, 4096, 128, True) == (2, 1, 1)
    assert AB._plan(96, 777, 777, 64, False) == (1, 1, 1)
    assert AB._plan(8, 77, 77, 64, True) == (1, 1, 1)
    assert AB._plan(64, 512, 512, 128, True) == (1, 1, 1)
    assert AB._plan(28, 576, 576, 256, True) == (1, 1, 1)
    assert AB._plan(16, 8000, 77, 64, False)[1] >= 8          # few keys: the queries are split
    assert AB._plan(16, 16, 8000, 128, False)[2] >= 4         # few queries: the keys are split
    for units in (1, 7, 300):
        for sq in (1, 64, 65, 5000):
            for sk in (1, 1000):
                for dim in (64, 128, 256):
                    for causal in (True, False):
                        blocks, kp, qp = AB._plan(units, sq, sk, dim, causal)
                        assert 1 <= kp <= max(1, -(-sq // 64)) and 1 <= qp <= max(1, -(-sk // 64))
                        assert 8 * kp * units * sk * dim <= AB.MAX_SUM_BYTES or kp == 1
                        assert blocks == 1 or blocks == 2 and dim == 128


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_units_compile(head_dim, dtype):
    for stage, blocks, parts in AB.unit_kinds(head_dim):
        for causal in ((True, False) if stage != "rows" else (False,)):
            assert AB._program(stage, head_dim, causal, dtype, blocks, parts).precompile() > 0
