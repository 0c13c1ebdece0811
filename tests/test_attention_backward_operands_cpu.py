"""Which layouts the attention gradients' kernels read in place, and the row stride that they are given: rows past
a tile's last must lie outside of the last row, for they read as zero."""
import functools

import pytest
import torch

from neptune_codegen import attention_backward as AB

zeros = functools.partial(torch.zeros, dtype=torch.bfloat16)


@pytest.mark.parametrize("make,copied,stride", [
    (lambda: zeros(2, 3, 5, 64), False, 64),
    (lambda: zeros(2, 5, 3, 64).transpose(1, 2), False, 192),
    (lambda: zeros(2, 3, 1, 64).as_strided((2, 3, 1, 64), (192, 64, 0, 1)), False, 64),
    (lambda: zeros(2, 3, 1, 64).as_strided((2, 3, 1, 64), (192, 64, 8, 1)), False, 64),
    (lambda: zeros(2, 3, 1, 64).as_strided((2, 3, 1, 64), (192, 64, 1 << 25, 1)), False, 64),
    (lambda: zeros(2, 3, 1, 64).expand(2, 3, 5, 64), True, 64),
    (lambda: zeros(5 * 8 + 64).as_strided((1, 1, 5, 64), (64, 64, 8, 1)), True, 64),
    (lambda: zeros(2, 3, 5, 72)[..., 4:68], True, 64),
    (lambda: zeros(2, 3, 64, 5).transpose(2, 3), True, 64),
])
def test_row_strides(make, copied, stride):
    t = make()
    used, steps = AB._operand(t)
    assert (used is not t) == copied and steps[2] == stride
    assert torch.equal(used, t)
