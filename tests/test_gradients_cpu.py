"""The gradients' norm and clipping without a GPU: refusals and metadata calls."""
import math

import pytest
import torch

import neptune_codegen as CG
from neptune_codegen import gradients as GR


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("tensors,error", [
    ([], TypeError), (meta(3), TypeError), ([None], TypeError), ([meta(3, dtype=torch.float64)], TypeError),
    ([meta(3, dtype=torch.int32)], TypeError), ([meta(3), torch.zeros(3)], ValueError), ((t for t in [meta(3)]), TypeError)])
def test_lists_are_refused(tensors, error):
    with pytest.raises(error):
        CG.run_gradient_norm(tensors)
    with pytest.raises(error):
        CG.run_clip_gradients(tensors, 1.0)


@pytest.mark.parametrize("kw,error", [
    ({"max_norm": -1.0}, ValueError), ({"max_norm": math.nan}, ValueError), ({"max_norm": math.inf}, ValueError),
    ({"max_norm": torch.ones(())}, ValueError), ({"out": [meta(2, 3)]}, ValueError),
    ({"out": [meta(2, 3), meta(5)]}, ValueError), ({"out": [meta(2, 3), meta(4, dtype=torch.float16)]}, TypeError),
    ({"out": meta(2, 3)}, TypeError), ({"norm": 1.0}, TypeError), ({"norm": meta(1, dtype=torch.float32)}, ValueError),
    ({"norm": meta()}, ValueError)])
def test_clipping_is_refused(kw, error):
    with pytest.raises(error):
        CG.run_clip_gradients([meta(2, 3), meta(4)], **{"max_norm": 1.0, **kw})


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="device"):
        CG.run_gradient_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="device"):
        CG.run_clip_gradients([torch.zeros(3)], 1.0)


def test_metadata_calls():
    ts = [meta(2, 3), meta(4, dtype=torch.float32), meta(0)]
    for norm in (CG.run_gradient_norm(ts), CG.run_clip_gradients(ts, 1.0),
                 CG.run_clip_gradients(ts, 1, out=[meta(2, 3, dtype=torch.float32), ts[1], meta(0)],
                                       norm=meta(dtype=torch.float32))):
        assert norm.shape == () and norm.dtype == torch.float32 and norm.device.type == "meta"
    assert CG.as_gradient_norm_op() is CG.as_gradient_norm_op()
    assert CG.as_gradient_norm_op()(ts).shape == () and CG.as_clip_gradients_op()(ts, 1.0).shape == ()


def test_tensors_without_gaps():
    x = torch.zeros(4, 6, 2)
    for t, dense in ((x, True), (x.transpose(0, 2), True), (x[:, :3], False), (x[1], True), (x[:, 1:2, :1], False),
                     (x.expand(2, 4, 6, 2), False), (x[:1].expand(1, 6, 2), True), (torch.zeros(()), True),
                     (x[:0], True), (x[:1, :, :1], False)):
        assert GR._dense(t) == dense


def test_a_launch_fits_its_arguments():
    # 4096 bytes with the 256 that the compiler may add
    for _, args in GR._KERNELS:
        assert sum(4 if a in (GR.hip.I32, GR.hip.F32) else 8 for a in args) + 16 + 256 <= 4096
    assert GR.TENSORS * 32 <= 3584 and GR.MOST_TENSORS <= 64 * 64        # two ballots find a tensor
