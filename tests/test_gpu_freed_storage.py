"""Tensors whose storage was freed are refused, also where a call's layout is known.

A freed tensor never leaves `refusal`, which catches every error and returns plain values: a report that printed the
tensor's elements would read its memory.
"""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import dispatch

pytestmark = pytest.mark.gpu


def refusal(call, like, view):
    """What `call` says to a freed tensor, and whether the host takes the tensor's elements to be in memory."""
    whole = torch.empty_like(like)
    given = view(whole)                              # (torch makes no view of a freed tensor)
    whole.untyped_storage().resize_(0)
    held = bool(dispatch.extension().in_memory(given))
    said = "held, so not called"
    if not held:                                     # (nothing is launched on it)
        try:
            call(given)
            said = "no error"
        except Exception as error:
            said = f"{type(error).__name__}: {error}"
    return said, held


@pytest.mark.parametrize("name", ["embedding", "tokens", "embedding gradient", "added to", "residual norm", "8-bit norm",
                                  "distillation", "norm", "norm of a view", "norm of many", "clipping", "clipping into"])
def test_freed_tensors_are_refused(name):
    assert torch.cuda.is_available()
    print(f"freed: {name}", flush=True)
    make = lambda *s, **k: torch.ones(*s, device="cuda", **k)  # noqa: E731
    x, y, g, table, grad = make(4, 64), make(4, 64), make(64), make(10, 64), make(4, 64)
    tokens, top, index = torch.arange(4, device="cuda"), make(4, 2), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    many, whole = [make(300, 301), make(5)], lambda t: t
    call, like, view = {
        "embedding": (lambda t: CG.run_embedding(tokens, t), table, whole),
        "tokens": (lambda t: CG.run_embedding(t, table), tokens, whole),
        "embedding gradient": (lambda t: CG.run_embedding_backward(t, tokens, 10), grad, whole),
        "added to": (lambda t: CG.run_embedding_backward(grad, tokens, 10, into=t), table, whole),
        "residual norm": (lambda t: CG.run_residual_norm(x, t, None, g), y, whole),
        "8-bit norm": (lambda t: CG.run_residual_norm_quantized(x, y, None, t), g, whole),
        "distillation": (lambda t: CG.run_distill(t, top, index), x, whole),
        "norm": (lambda t: CG.run_gradient_norm([x, t]), y, whole),
        "norm of a view": (lambda t: CG.run_gradient_norm([x, t]), y, lambda t: t[1:]),
        "norm of many": (lambda t: CG.run_gradient_norm([*many, t]), y, whole),
        "clipping": (lambda t: CG.run_clip_gradients([many[1], t], 1e9), y, whole),
        "clipping into": (lambda t: CG.run_clip_gradients([x], 1e9, out=[t]), y, whole)}[name]
    for _ in range(2):                               # (the second time the layout is known)
        call(view(like))
    said, held = refusal(call, like, view)
    assert not held and said.startswith("TypeError") and "without memory" in said
    call(view(like))
