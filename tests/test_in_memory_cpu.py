"""Whether a tensor's elements are in its storage, which the direct entry points ask of each call, without a GPU."""
import pytest
import torch

from neptune_codegen import dispatch


def freed(t, size=0):
    t.untyped_storage().resize_(size)
    return t


def test_elements_in_their_storage():
    inside, x = dispatch.extension().in_memory, torch.zeros(4, 6)
    for t in (x, x[1:], x.T, x[:, ::2], x[3:, 5:], x[:1].expand(9, 6), torch.zeros(()), x[4:], torch.zeros(0, 3),
              torch.nn.Parameter(x), x.view(torch.int32), torch.zeros(7, dtype=torch.bfloat16)[1:]):
        assert inside(t)


@pytest.mark.parametrize("view", [lambda t: t, lambda t: t[1:], lambda t: t.T, lambda t: t[3:, 5:],
                                  lambda t: t[:1].expand(9, 6), lambda t: t[:, ::5]])
def test_elements_of_a_freed_storage(view):
    inside = dispatch.extension().in_memory
    x = torch.zeros(4, 6)
    t = view(x)
    freed(x)
    assert not inside(t)                             # (a view's address is its offset, not null)
    assert inside(t[:0])


def test_elements_behind_a_shortened_storage():
    inside = dispatch.extension().in_memory
    x = torch.zeros(4, 6)
    first, last, columns = x[:2], x[2:], x[:, :1]
    freed(x, 12 * 4)
    assert inside(first) and not inside(last) and not inside(x) and not inside(columns) and inside(columns[:2])
