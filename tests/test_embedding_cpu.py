"""The embedding without a GPU: refusals, metadata calls, and launches that cover tokens and columns."""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import embedding as EM


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


I, T, G = meta(2, 3, dtype=torch.int64), meta(10, 16), meta(2, 3, 16)


@pytest.mark.parametrize("args,kw,error", [
    ((I, meta(10)), {}, ValueError), ((I, meta(0, 16)), {}, ValueError), ((I, meta(10, 0)), {}, ValueError),
    ((meta(2, 3, dtype=torch.int16), T), {}, TypeError), ((meta(2, 3), T), {}, TypeError),
    ((I, meta(10, 16, dtype=torch.float64)), {}, TypeError), ((I, None), {}, TypeError), (([1], T), {}, TypeError),
    ((I, T), {"scale": math.inf}, ValueError), ((I, T), {"scale": math.nan}, ValueError),
    ((I, T), {"scale": "1"}, ValueError), ((I, T), {"scale": torch.ones(())}, ValueError)])
def test_refusals(args, kw, error):
    with pytest.raises(error):
        CG.run_embedding(*args, **kw)


@pytest.mark.parametrize("args,kw,error", [
    ((meta(2, 16), I, 10), {}, ValueError), ((meta(2, 3, 0), I, 10), {}, ValueError), ((G, I, 0), {}, ValueError),
    ((G, I, True), {}, ValueError), ((G, I, 10.0), {}, ValueError), ((G, I.int().float(), 10), {}, TypeError),
    ((G.double(), I, 10), {}, TypeError), ((G, I, 10), {"scale": -math.inf}, ValueError),
    ((G, I, 1 << 31), {}, NotImplementedError), ((G, I, (1 << 24) + 1), {}, NotImplementedError),
    ((meta(1 << 13, 1 << 13, 2), meta(1 << 13, 1 << 13, dtype=torch.int32), 10), {}, NotImplementedError),
    ((G, I, 10), {"into": meta(10, 15)}, ValueError), ((G, I, 10), {"into": meta(11, 16)}, ValueError),
    ((G, I, 10), {"into": meta(10, 16, dtype=torch.float16)}, TypeError),
    ((G.float(), I, 10), {"into": meta(10, 16)}, TypeError), ((G, I, 10), {"into": meta(16, 10).T}, ValueError),
    ((G, I, 10), {"into": meta(1, 16).expand(10, 16)}, ValueError), ((G, I, 10), {"into": [1]}, TypeError),
    ((G, I, 10), {"into": meta(10, 16).requires_grad_()}, ValueError)])
def test_gradient_refusals(args, kw, error):
    with pytest.raises(error):
        CG.run_embedding_backward(*args, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="device"):
        CG.run_embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 4))
    with pytest.raises(ValueError, match="device"):
        CG.run_embedding_backward(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64), 3)


def test_metadata_calls():
    assert CG.run_embedding(I, T, scale=4).shape == (2, 3, 16)
    assert CG.run_embedding(meta(dtype=torch.int32), T).shape == (16,)
    grad = CG.run_embedding_backward(G, I, 10)
    assert grad.shape == (10, 16) and grad.dtype == torch.bfloat16
    into = meta(10, 16, dtype=torch.float32)
    assert CG.run_embedding_backward(G, I, 10, into=into) is into
    assert CG.run_embedding(I, meta((1 << 24) + 1, 16)).shape == (2, 3, 16)
    with pytest.raises(NotImplementedError):         # which its gradient would refuse
        CG.as_embedding_op(2.0)(I, meta((1 << 24) + 1, 16))
    op = CG.as_embedding_op(2.0)
    assert op is CG.as_embedding_op(2) and op(I, T).shape == (2, 3, 16)


def test_the_workgroups_that_order_tokens_count_every_row():
    for vocab in (1, 2, 7, 255, 256, 257, 32000, 128256, 1 << 18, (1 << 18) + 1, 1 << 27, (1 << 31) - 1):
        shares = 1 << EM._shares(vocab)
        assert -(-vocab // shares) <= EM.MOST_KEYS and (shares <= 256 or -(-vocab // (shares // 2)) > EM.MOST_KEYS)
        # rows of workgroup w, as the kernel counts them
        mine = [(vocab - 1 - w) // shares + 1 if w < vocab else 0 for w in range(min(shares, 4096))]
        if shares <= 4096:
            assert sum(mine) == vocab


def test_tokens_have_one_stride():
    x = torch.arange(24).view(4, 6)
    for t, stride in ((x, 1), (x[:, ::2], None), (x[:, 1], 6), (x.T, None), (x[0, 0], 0), (x[:1, :1].expand(4, 6), 0)):
        flat, step = EM._flat(t)
        assert flat.numel() == t.numel()
        if stride is not None:
            assert flat.data_ptr() == t.data_ptr() and step == stride
        walked = flat.as_strided((t.numel(),), (step,), flat.storage_offset())
        assert torch.equal(walked, t.reshape(-1))
    flat, step = EM._flat(x[:, 1], 5)                # further apart than a gradient reads them: copied
    assert step == 1 and flat.data_ptr() != x[:, 1].data_ptr() and torch.equal(flat.reshape(-1), x[:, 1])
    assert EM._flat(x[:, 1], 6)[1] == 6
