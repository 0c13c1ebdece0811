"""The distillation operators without a GPU: refusals, metadata calls and launch choice."""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import distill as DI


def meta(shape=(4, 100), dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def lists(k=8, rows=4):
    return meta((rows, k), torch.float32), meta((rows, k), torch.int64)


@pytest.mark.parametrize("logits,top,index,kw,error", [
    (meta(dtype=torch.float64), *lists(), {}, TypeError), (meta(), None, lists()[1], {}, TypeError),
    (meta(), lists(rows=3)[0], lists()[1], {}, ValueError), (meta(), lists()[0], lists(9)[1], {}, ValueError),
    (meta(), meta((4, 8), torch.float16), lists()[1], {}, TypeError),
    (meta(), lists()[0], meta((4, 8), torch.int16), {}, TypeError),
    (meta(), *lists(1025), {}, NotImplementedError), (meta(), *lists(0), {}, NotImplementedError),
    (meta(), *lists(), {"temperature": 0.0}, ValueError), (meta(), *lists(), {"temperature": math.inf}, ValueError),
    (meta(), *lists(), {"temperature": True}, ValueError), (meta((4, 2, 100)), *lists(), {}, ValueError)])
def test_refusals(logits, top, index, kw, error):
    with pytest.raises(error):
        CG.run_distill(logits, top, index, **kw)
    with pytest.raises(error):
        CG.run_distill_backward(meta((4,), torch.float32), logits, top, index, meta((4, 2), torch.float32), **kw)


def test_gradient_refusals():
    for grad, stats in ((meta((4,)), meta((4, 2), torch.float32)), (meta((5,), torch.float32), meta((4, 2), torch.float32)),
                        (meta((4,), torch.float32), meta((4,), torch.float32))):
        with pytest.raises(ValueError):
            CG.run_distill_backward(grad, meta(), *lists(), stats)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="device"):
        CG.run_distill(torch.zeros(2, 5), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.long))


def test_metadata_calls():
    loss, stats = CG.run_distill(meta((2, 4, 100)), meta((2, 4, 8), torch.float32), meta((2, 4, 8), torch.int32),
                                 return_stats=True)
    assert loss.shape == (2, 4) and stats.shape == (2, 4, 2) and loss.dtype == torch.float32
    dz = CG.run_distill_backward(meta((4,), torch.float32), meta(), *lists(), meta((4, 2), torch.float32))
    assert dz.shape == (4, 100) and dz.dtype == torch.bfloat16
    op = CG.as_distill_op(2)
    assert op is CG.as_distill_op(2.0)
    assert op(meta(), *lists())[0].shape == (4,)


def test_lists_fit_the_lanes():
    for rows in (1, 300, 20000):
        for n in (1, 5, 1000, 50257, 262144):
            for k in (1, 64, 65, 256, 257, 1024):
                for dtype in (torch.float32, torch.bfloat16):
                    z = meta((rows, n), dtype)
                    t, i = meta((rows, k), torch.float32), meta((rows, k), torch.int64)
                    for stage in ("forward", "backward"):
                        var = DI._variant(z, n, t, i, rows, n, k, stage)
                        assert var.tpr * var.entries >= k and var.tpr in (64, 256, 1024) and var.unroll <= 8
                        assert DI._program(stage, var).source
