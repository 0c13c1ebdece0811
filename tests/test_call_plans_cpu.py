"""Calls kept by layout (neptune_codegen/calls.py): plans, keys and refusals, without a GPU."""
import pytest
import torch

from neptune_codegen import calls, dispatch


def plan(returns, bare=False, launches=()):
    buffers = [((2, 3), torch.float32), ((0, 4), torch.bfloat16), ((16,), torch.uint8)]
    return calls.Plan(0, 2, buffers, returns, launches, bare)


def test_results_have_the_planned_shapes_and_absent_ones_are_none():
    a = torch.ones(3)
    out = plan((0, None, 1)).run((a, None))
    assert out[0].shape == (2, 3) and out[0].dtype == torch.float32 and out[1] is None
    assert out[2].shape == (0, 4) and out[2].dtype == torch.bfloat16
    assert plan((0,), bare=True).run((None, a)).shape == (2, 3)
    first, second = plan((0,)).run((a, None))[0], plan((0,)).run((a, None))[0]
    assert first.data_ptr() != second.data_ptr()


def test_wrong_calls_are_refused():
    a = torch.ones(3)
    with pytest.raises(RuntimeError, match="expected 2 tensors"):
        plan((0,)).run((a,))
    with pytest.raises(RuntimeError, match="no tensor"):
        plan((0,)).run((None, None))
    with pytest.raises(RuntimeError, match="no such result"):
        plan((3,))
    with pytest.raises(RuntimeError, match="one bare result"):
        plan((0, 1), bare=True)
    native = dispatch.extension().CallPlan
    code = calls._dtype_code(torch.float32)
    for patch in ((4, 0, 0), (0, 1, 0), (0, -2, 0)):  # past the image, no such tensor, no such buffer
        with pytest.raises(RuntimeError, match="bad pointer"):
            native(1, ((code, (1,)),), [0], True, ((1, (1, 1, 1), 64, 0, bytes(8), (patch,)),))
    with pytest.raises(RuntimeError, match="bad launch"):
        native(1, ((code, (1,)),), [0], True, ((0, (1, 1, 1), 64, 0, bytes(8), ()),))


def test_calls_without_a_key_are_not_kept():
    table, a = calls.Table(), torch.ones(3)
    table.keep((a, None), (1.0, False), plan((0,)))              # not on a device
    assert table.run((a, None), (1.0, False)) is None
    assert table.native().size() == 0
    assert not table.native().keep((a.to("meta"),), (1.0,), plan((0,)).native)
    assert not table.native().keep((None,), ("text",), plan((0,)).native)
    assert not table.native().keep((None,), (1 << 80,), plan((0,)).native)


def test_numbers_are_told_apart_by_type_and_value():
    table = calls.Table()
    table.keep((None, None), (1, True), plan((0,)))
    for numbers in ((1.0, True), (1, 1), (True, True), (None, True), (2, True), (1, False)):
        assert table.run((None, None), numbers) is None
    with pytest.raises(RuntimeError, match="no tensor"):         # found, and run
        table.run((None, None), (1, True))


@pytest.mark.parametrize("make,stride,copied", [
    (lambda: torch.ones(4, 6), 6, False),
    (lambda: torch.ones(4, 10)[:, :6], 10, False),
    (lambda: torch.ones(2, 4, 10)[:, :, :6], 10, False),
    (lambda: torch.ones(2, 5, 10)[:, :4, :6], 6, True),          # two row strides
    (lambda: torch.ones(4, 2, 6).transpose(0, 1), 6, True),
    (lambda: torch.ones(6, 4).T, 6, True),
    (lambda: torch.ones(1, 6).expand(4, 6), 0, False),
    (lambda: torch.ones(6), 0, False),
    (lambda: torch.ones(1, 1, 6), 0, False),
    (lambda: torch.ones(4, 3)[:, :1], 3, False),
])
def test_row_strides(make, stride, copied):
    t = make()
    used, step = calls.rows_of(t)
    assert step == stride and (used is not t) == copied
    assert torch.equal(used, t)


def test_grids_past_one_launch_are_refused():
    calls.check_grid(((1 << 24) - 1, 65535), 256, "k")
    for grid in ((1 << 24,), (1, 65536)):
        with pytest.raises(NotImplementedError):
            calls.check_grid(grid, 256, "k")
