"""Operators that several threads ask for at once are registered once, without a GPU."""
import threading

import pytest
import torch

import neptune_codegen as CG


def at_once(make, count=6):
    start, got = threading.Barrier(count), []

    def ask():
        start.wait()
        try:
            got.append(make())
        except Exception as error:                   # (what the test reports)
            got.append(error)

    threads = [threading.Thread(target=ask) for _ in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert len(got) == count
    return got


def scale(i):
    return 300.0 + i                                 # (of no other test's operators)


MAKERS = {
    "embedding": lambda i: CG.as_embedding_op(scale(i)),
    "residual norm": lambda i: CG.as_residual_norm_op(scale(i)),
    "8-bit residual norm": lambda i: CG.as_residual_norm_quantized_op(scale(i), dtype=torch.int8, group=32),
    "gradients' norm": lambda i: CG.as_gradient_norm_op(f"once{i}"),
    "clipping": lambda i: CG.as_clip_gradients_op(f"once{i}"),
    "rotary": lambda i: CG.as_rotary_op(scale(i)),
    "distillation": lambda i: CG.as_distill_op(scale(i)),
    "attention": lambda i: CG.as_attention_op(scale(i)),
    "attention's gradients": lambda i: CG.as_attention_grad_op(scale(i)),
    "fold": lambda i: CG.as_triton_op("logsumexp", lib=f"once{i}"),
    "readout": lambda i: CG.as_readout_op("logsumexp", lib=f"once{i}"),
    "state": lambda i: CG.as_state_op("rms_norm", {"eps": 1e-6}, lib=f"once{i}"),
    "segment": lambda i: CG.as_segment_op("segment_sum", lib=f"once{i}"),
}


@pytest.mark.parametrize("name", MAKERS)
def test_threads_get_one_operator(name):
    for i in range(4):
        got = at_once(lambda: MAKERS[name](i))
        assert all(op is got[0] for op in got) and not isinstance(got[0], Exception), got


def test_different_operators_at_once():
    names, i = list(MAKERS), iter(range(10 ** 6))
    got = at_once(lambda: MAKERS[names[(k := next(i)) % len(names)]](100 + k), 2 * len(names))
    assert not [op for op in got if isinstance(op, Exception)]
