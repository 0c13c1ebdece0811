"""The residual norm without a GPU: refusals, metadata calls, gate shapes and launch choice."""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import residual_norm as RN


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


X, G = meta(2, 3, 64), meta(64)


@pytest.mark.parametrize("args,kw,error", [
    ((meta(2, 3, 64, dtype=torch.float64), X, G, G), {}, TypeError), ((X, meta(2, 64), G, G), {}, ValueError),
    ((X, X, meta(63), G), {}, ValueError), ((X, X, G, None), {}, TypeError), ((X, X, G, meta(2, 64)), {}, ValueError),
    ((X, X, G, meta(64, dtype=torch.float32)), {}, ValueError), ((X, None, G, G), {}, TypeError),
    ((X, X, G, G), {"gate": meta(3, 64)}, ValueError), ((X, X, G, G), {"gate": meta(1, 3, 64)}, ValueError),
    ((X, X, G, G), {"gate": meta(2, 1, 1)}, ValueError), ((X, X, G, G), {"gate": 0.5}, TypeError),
    ((X, X, G, G), {"residual_scale": math.nan}, ValueError), ((X, X, G, G), {"eps": 0.0}, ValueError),
    ((meta(2, 16385),) * 2 + (meta(16385),) * 2, {}, NotImplementedError)])
def test_refusals(args, kw, error):
    with pytest.raises(error):
        CG.run_residual_norm(*args, **kw)


def test_gradient_refusals():
    stats = meta(2, 3, 2, dtype=torch.float32)
    for grads, s, kw in (((X, meta(2, 64)), stats, {}), ((meta(2, 3, 64, dtype=torch.float16), X), stats, {}),
                         ((X, X), meta(2, 3, dtype=torch.float32), {}), ((X, X), stats, {"residual_scale": math.inf})):
        with pytest.raises(ValueError):
            CG.run_residual_norm_backward(*grads, X, X, G, G, s, **kw)
    with pytest.raises(TypeError):
        CG.run_residual_norm_backward(X, None, X, X, G, G, stats)


def test_cpu_tensors_are_refused():
    x, g = torch.zeros(2, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="device"):
        CG.run_residual_norm(x, x, g, g)


def test_metadata_calls():
    r, h, s = CG.run_residual_norm(X, X, None, G, gate=meta(2, 1, 64), return_stats=True)
    assert r.shape == h.shape == X.shape and s.shape == (2, 3, 2) and s.dtype == torch.float32
    dx, dy, da, db, dg = CG.run_residual_norm_backward(None, X, X, X, None, G, s, gate=meta(2, 1, 64))
    assert dx.shape == dy.shape == X.shape and da is None and db.shape == (64,) and dg.shape == (2, 1, 64)
    op = CG.as_residual_norm_op(0.5)
    assert op is CG.as_residual_norm_op(0.5, 1e-6)
    assert op(X, X, G, G, None)[0].shape == X.shape


@pytest.mark.parametrize("shape,gate,want", [((2, 3, 64), (2, 3, 64), (6, 1)), ((2, 3, 64), (2, 1, 64), (2, 3)),
                                             ((2, 3, 64), (1, 1, 64), (1, 6)), ((2, 3, 64), (64,), (1, 6)),
                                             ((2, 1, 64), (2, 1, 64), (2, 1)), ((5, 64), (1, 64), (1, 5))])
def test_gate_groups(shape, gate, want):
    assert RN._gate_groups(meta(*gate), meta(*shape)) == want


def test_workgroups_cover_the_rows_once():
    for rows, groups in ((1, 1), (7, 7), (1000, 1), (1000, 8), (1000, 500), (60000, 30000), (16384, 8), (300, 300),
                         (512, 256), (514, 257)):
        group = rows // groups
        for kind in ("none", "rows", "group"):
            for rpw in (1, 2, 8, 64):
                chunks, per_group = RN._chunks(rows, groups, group, kind, rpw)
                seen = [0] * rows
                gr, gn = (group, groups) if kind == "group" else (rows, 1)
                for c in range(chunks):          # as the kernel walks them
                    g0 = c // per_group if per_group else c
                    for gi in range(g0, g0 + 1 if per_group else gn, chunks):
                        first, end = gi * gr + (c % per_group * rpw if per_group else 0), (gi + 1) * gr
                        assert first < end
                        for base in range(first, end, rpw * max(per_group, 1)):
                            for r in range(base, min(base + rpw, end)):
                                seen[r] += 1
                assert seen == [1] * rows and chunks <= 256


def test_rows_fit_the_lanes():
    for n in (1, 7, 8, 64, 1000, 4096, 8192, 10007, 16384):
        for dtype in (torch.float32, torch.bfloat16):
            for backward in (False, True):
                for rows in (1, 100000):
                    var = RN._variant(meta(rows, n, dtype=dtype), n % 8 == 0, rows, n, True, "group", backward)
                    vec = 16 // meta(1, dtype=dtype).element_size()
                    assert var.tpr * var.nv * vec >= n and var.tpr <= var.wg <= 1024
                    # the column sums' LDS
                    assert not backward or 4 * var.wg * var.nv * vec <= 65536
