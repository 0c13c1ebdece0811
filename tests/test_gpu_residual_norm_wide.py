"""Gradients of the residual norm of more than 8192 columns in the forms without a norm behind the block, whose
column sums are fewer: formulas and tolerances as in test_gpu_residual_norm.py."""
import pytest
import torch

from test_gpu_residual_norm import _dev, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,n,gate", [
    ((11,), 8200, (11,)), ((3, 5), 12288, (3, 5)), ((300,), 12289, (300,)), ((7,), 16384, (7,)),
    ((270,), 16381, (270,)), ((2, 140), 16384, None), ((9,), 9001, None), ((4, 6), 16384, (4, 1)), ((30,), 12283, ())])
def test_wide_rows_without_a_norm_behind_the_block(lead, n, gate, dtype):
    dev = _dev()
    print(f"residual norm {lead} x {n} gate={gate} {dtype}", flush=True)
    check(make(lead, n, dtype, False, gate), 0.5, dev)
