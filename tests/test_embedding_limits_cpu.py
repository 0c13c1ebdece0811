"""What the embedding's gradient refuses, the differentiable operator refuses before it runs, without a GPU."""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import embedding as EM


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def tokens(*shape):
    return meta(*shape, dtype=torch.int64)


@pytest.mark.parametrize("dtype,most", [(torch.float32, 65535 * 256), (torch.bfloat16, 65535 * 512)])
def test_rows_of_more_columns_than_the_join_has(dtype, most):
    op = CG.as_embedding_op(2.0)
    for n, count, taken in ((most, 513, True), (most + 1, 513, False), (most + 1, 512, True), (most + 1, 70000, False)):
        i, table, grad = tokens(count), meta(2, n, dtype=dtype), meta(count, n, dtype=dtype)
        if taken:
            # (the launch that would be refused: one 64-word part of the row in each of the grid's second dimension)
            assert count <= EM.FEW or -(-(-(-n * dtype.itemsize // 16)) // 64) <= 65535
            assert op(i, table).shape == (count, n) and CG.run_embedding_backward(grad, i, 2).shape == (2, n)
            continue
        with pytest.raises(NotImplementedError):
            op(i, table)
        with pytest.raises(NotImplementedError):
            CG.run_embedding_backward(grad, i, 2)
        assert CG.run_embedding(i, table).shape == (count, n)


def test_a_refused_call_does_not_run(monkeypatch):
    ran = []
    monkeypatch.setattr(EM, "run_embedding", lambda *a, **k: ran.append(a) or torch.zeros(1))
    op = CG.as_embedding_op(7.0)
    table = torch.zeros(1, 1).expand(EM.MOST_ROWS + 1, 1)
    with pytest.raises(NotImplementedError):
        op(torch.zeros(2, dtype=torch.int64), table)
    assert not ran
    op(torch.zeros(2, dtype=torch.int64), table[1:])
    op(torch.zeros(2, dtype=torch.int64), torch.zeros(3))        # (refused by the lookup)
    assert len(ran) == 2
