"""The type of the residual norm's 8-bit output is a torch type, never its name, without a GPU."""
import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import residual_norm as RN

X, G = torch.empty(2, 70, dtype=torch.bfloat16, device="meta"), torch.empty(70, dtype=torch.bfloat16, device="meta")


@pytest.mark.parametrize("name", ["int8", "torch.int8", "float8_e5m2"])
def test_names_of_types_are_refused(name):
    codes = dict(RN._CODES)
    with pytest.raises(TypeError, match="8-bit outputs"):
        CG.run_residual_norm_quantized(X, X, G, G, dtype=name)
    assert RN._CODES == codes                        # (a name among them would find a call kept for its type)
    with pytest.raises(TypeError, match="8-bit outputs"):
        CG.as_residual_norm_quantized_op(0.75, dtype=name)


def test_a_refused_name_leaves_the_types_operator_whole():
    with pytest.raises(TypeError):
        CG.as_residual_norm_quantized_op(0.625, dtype="int8")
    assert CG.as_residual_norm_quantized_op(0.625, dtype=torch.int8)(X, X, G, G, None)[1].dtype == torch.int8
