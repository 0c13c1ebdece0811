"""Tensors that only wrap others (a DTensor is one) have no memory for a kernel: refused by name, without a GPU."""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import calls, gradients as GR


class Wrapper(torch.Tensor):
    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.alias.default:
            return Wrapper(*args[0].shape, dtype=args[0].dtype)
        return NotImplemented


I64 = torch.int64
X, G = Wrapper(2, 3, 16), Wrapper(16)


@pytest.mark.parametrize("call", [
    lambda: CG.run_embedding(Wrapper(2, 3, dtype=I64), Wrapper(10, 16)),
    lambda: CG.run_embedding_backward(X, Wrapper(2, 3, dtype=I64), 10),
    lambda: CG.run_embedding_backward(X, Wrapper(2, 3, dtype=I64), 10, into=Wrapper(10, 16)),
    lambda: CG.run_residual_norm_quantized(X, X, G, G),
    lambda: CG.run_residual_norm(X, X, G, G, gate=X),
    lambda: CG.run_distill(X, Wrapper(2, 3, 2), Wrapper(2, 3, 2, dtype=I64)),
    lambda: CG.run_gradient_norm([X]),
    lambda: CG.run_clip_gradients([X, G], 1.0),
    lambda: CG.run_clip_gradients([X], 1.0, norm=Wrapper()),
    lambda: calls.check_tensor(X, "x", metadata=False)])
def test_wrappers_are_refused(call):
    with pytest.raises(TypeError, match="Wrapper without memory of its own"):
        call()


def test_tensors_without_elements_have_no_memory_either():
    calls.check_tensor(Wrapper(0, 3), "x", metadata=False)       # (nothing is read)
    calls.check_tensor(torch.empty(4, device="meta"), "x", metadata=True)


def test_a_norm_is_never_none(monkeypatch):
    class Calls:                                     # which takes no list
        norm = staticmethod(lambda tensors: None)
        clip = staticmethod(lambda *args: None)

    monkeypatch.setattr(GR, "_calls", lambda device=None: Calls)
    monkeypatch.setattr(GR, "_CALLS", None)
    with pytest.raises(TypeError, match="plain tensors"):
        CG.run_gradient_norm([Wrapper(0)])
    with pytest.raises(ValueError, match="plain tensors"):
        CG.run_clip_gradients([Wrapper(0)], 1.0)
