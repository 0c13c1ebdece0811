"""What a gradient is added to in place overlaps nothing that the call reads: without a GPU, by the memory of CPU
tensors."""
import pytest
import torch

from neptune_codegen import embedding as EM


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_tokens_in_the_tables_memory_are_found(index):
    into = torch.zeros(10, 16)
    grad, tokens = torch.zeros(4, 16), torch.zeros(4, dtype=index)
    assert EM._apart(into, grad, tokens)
    inside = into.view(index).flatten()
    for t, apart in ((inside[:4], False), (inside[-4:], False), (inside[::3], False), (inside[:0], True)):
        assert EM._apart(into, grad, t) == apart
    assert EM._apart(into[:5], grad, into[5:].view(index).flatten()[:4])
    assert not EM._apart(into, into[2:6], tokens)
    assert EM._apart(into, grad.to("meta"), inside.to("meta")) and EM._apart(into.to("meta"), grad, inside)


def test_overlap_is_that_of_the_first_and_last_elements():
    from neptune_codegen import calls

    x = torch.zeros(64)
    for a, b, want in ((x[:8], x[8:], False), (x[:8], x[7:], True), (x[8:], x[:8], False), (x[7:], x[:8], True),
                       (x[:15:2], x[15:], False), (x[:16:2], x[14:], True), (x.view(8, 8)[:, :2], x[58:], False),
                       (x.view(8, 8)[:, :2], x[57:], True), (x.view(8, 8).T, x[63:], True), (x[:1].expand(9), x[1:], False),
                       (x[5:5], x, False), (x, x[5:5], False), (x, x, True), (x[:9], x.view(torch.int64)[4:], True)):
        assert calls.overlap(a, b) == calls.overlap(b, a) == want
