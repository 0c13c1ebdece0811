"""Errors of the training operators' kept calls: those of their first calls, and of the framework's other folds.
Each is raised by the host before anything is launched."""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import calls, dispatch, hip

pytestmark = pytest.mark.gpu


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def test_a_refused_launch_is_a_hip_error():
    dev = _dev()
    code = calls._dtype_code(torch.float32)
    nothing = (1, (0, 1, 1), 64, 0, bytes(8), ())    # a grid of no workgroups: the library refuses it unread
    plan = dispatch.extension().CallPlan(1, ((code, (1,)),), [0], True, (nothing,))
    with pytest.raises(hip.HipError, match="empty grid"):
        plan.run((torch.ones(1, device=dev),))


def test_results_that_do_not_fit_are_out_of_memory_errors():
    dev = _dev()
    turns, _ = CG.rotary_frequencies(64, device=dev)
    one = torch.ones((1, 1, 1, 64), dtype=torch.bfloat16, device=dev)
    q = one.expand(64, 1 << 14, 1 << 14, 64)         # 2^41 bytes of results from one row
    positions = torch.zeros(1, dtype=torch.int64, device=dev).expand(1 << 14)
    print("rotary of 2^41 bytes", flush=True)
    for _ in range(2):
        with pytest.raises(torch.OutOfMemoryError):
            CG.run_rotary(q, None, positions, turns)
    got, _ = CG.run_rotary(one, None, positions[:1], turns)
    assert torch.equal(got, one)
