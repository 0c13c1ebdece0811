"""The embedding's gradient is refused where it would be added to the memory that holds the tokens."""
import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu


def test_tokens_in_the_tables_memory_are_refused():
    assert torch.cuda.is_available()
    print("tokens in a table", flush=True)
    into = torch.zeros(10, 16, device="cuda")
    grad, tokens = torch.ones(4, 16, device="cuda"), torch.arange(4, device="cuda")
    inside = into.view(torch.int64)[9, :4]           # (zeros)
    for _ in range(2):                               # (the second time its layout is known)
        with pytest.raises(ValueError, match="overlap"):
            CG.run_embedding_backward(grad, inside, 10, into=into)
        assert not into.any()
        CG.run_embedding_backward(grad, tokens, 10, into=into)
        assert (into[:4] == 1).all() and not into[4:].any()
        into.zero_()
