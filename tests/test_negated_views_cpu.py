"""Views that negate what their memory holds (the imag of a conjugate) are refused by the direct entry points, whose
kernels would read them with the other sign: without a GPU."""
import pytest
import torch

import neptune_codegen as CG

NEG = torch._neg_view
X, G, I = torch.ones(2, 3, 16), torch.ones(16), torch.zeros(2, 3, dtype=torch.int64)
TOP = torch.zeros(2, 3, 2, dtype=torch.int64)


@pytest.mark.parametrize("call", [
    lambda: CG.run_embedding(I, NEG(torch.ones(10, 16))),
    lambda: CG.run_embedding_backward(NEG(X), I, 10),
    lambda: CG.run_residual_norm(NEG(X), X, G, G),
    lambda: CG.run_residual_norm_quantized(NEG(X), X, None, G),
    lambda: CG.run_residual_norm_quantized(torch.complex(X, X).conj().imag, X, G, G),
    lambda: CG.run_residual_norm_backward(X, X, NEG(X), X, G, G, torch.ones(2, 3, 2)),
    lambda: CG.run_distill(NEG(X), torch.ones(2, 3, 2), TOP),
    lambda: CG.run_rotary(NEG(torch.ones(1, 2, 3, 16)), torch.ones(1, 2, 3, 16), torch.zeros(1, 3, dtype=torch.int64),
                          torch.ones(8, dtype=torch.float64))])
def test_negated_views_are_refused(call):
    with pytest.raises(ValueError, match="negates"):
        call()


def test_what_is_added_to_is_no_negated_view_either():
    from neptune_codegen import embedding as EM

    grad = torch.empty(2, 3, 16, device="meta")
    with pytest.raises(ValueError, match="negates"):
        EM.calls.check_tensor(NEG(torch.ones(10, 16)), "embedding into", metadata=False)
    EM.calls.check_tensor(grad, "grad", metadata=True)
