"""The residual norm's 8-bit output without a GPU: refusals, metadata calls, launch shapes."""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import residual_norm as RN


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


X, G = meta(2, 3, 70), meta(70)


@pytest.mark.parametrize("args,kw,error", [
    ((X, X, G, G), {"dtype": torch.float16}, TypeError), ((X, X, G, G), {"dtype": torch.uint8}, TypeError),
    ((X, X, G, G), {"dtype": "e4m3"}, TypeError), ((X, X, G, G), {"group": 16}, ValueError),
    ((X, X, G, G), {"group": 32.0}, ValueError), ((X, X, G, G), {"group": 0}, ValueError),
    ((X, X, G, G), {"eps": 0.0}, ValueError), ((X, X, G, G), {"residual_scale": math.nan}, ValueError),
    ((X, meta(2, 70), G, G), {}, ValueError), ((X, X, G, None), {}, TypeError),
    ((X, X, G, G), {"gate": meta(3, 70)}, ValueError), ((meta(2, 16385),) * 2 + (meta(16385),) * 2, {}, NotImplementedError)])
def test_refusals(args, kw, error):
    with pytest.raises(error):
        CG.run_residual_norm_quantized(*args, **kw)


def test_operator_refusals():
    for kw, error in (({"dtype": torch.float32}, TypeError), ({"group": 7}, ValueError), ({"eps": -1.0}, ValueError)):
        with pytest.raises(error):
            CG.as_residual_norm_quantized_op(**kw)


def test_cpu_tensors_are_refused():
    x, g = torch.zeros(2, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="device"):
        CG.run_residual_norm_quantized(x, x, g, g)


def test_metadata_calls():
    r, q, s = CG.run_residual_norm_quantized(X, X, G, G)
    assert r.shape == q.shape == X.shape and r.dtype == X.dtype and q.dtype == torch.float8_e4m3fn
    assert s.shape == (2, 3, 1) and s.dtype == torch.float32
    r, q, s, t = CG.run_residual_norm_quantized(X, X, None, G, gate=meta(2, 1, 70), dtype=torch.int8, group=32,
                                                power_of_two=True, return_stats=True)
    assert q.dtype == torch.int8 and s.shape == (2, 3, 3) and t.shape == (2, 3, 2)
    op = CG.as_residual_norm_quantized_op(0.5, dtype=torch.float8_e5m2, group=64)
    assert op is CG.as_residual_norm_quantized_op(0.5, 1e-6, torch.float8_e5m2, 64, False)
    assert op is not CG.as_residual_norm_quantized_op(0.5, dtype=torch.float8_e5m2, group=64, power_of_two=True)
    assert op(X, X, G, G, None)[2].shape == (2, 3, 2)


def test_blocks_lie_in_slots():
    # (what the kernel asserts when it is compiled), and lanes hold every column
    for n in (1, 7, 8, 31, 40, 200, 721, 1000, 1110, 2048, 2999, 4095, 4096, 7479, 8192, 8773, 10007, 12544, 16384):
        for dtype in (torch.float32, torch.bfloat16):
            for rows in (1, 1023, 1024, 100000):
                vec = 16 // meta(1, dtype=dtype).element_size()
                tags = set()
                for block in (0, *RN.BLOCKS):
                    var = RN._quantized_variant(meta(rows, n, dtype=dtype), n % 8 == 0, rows, n, True, "none", "int8",
                                                block, False)
                    assert var.tpr * var.nv * vec >= n and var.tpr <= var.wg <= 1024 and var.wg % var.tpr == 0
                    assert not block or (min(block // vec, var.tpr) <= 64
                                         and (var.nv == 1 or var.tpr * vec % block == 0))
                    tags.add(var.tag())
                assert len(tags) == 4
