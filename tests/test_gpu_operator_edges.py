"""Ends of the training operators' ranges: layouts by lane exchange, the widest launches, offsets past 32 bits,
calls without rows.  Tolerances as in the operators' own tests; where one call is compared with another, both
round the same fp32 value whose sums may be added in another order (2^-20 of a row's sum) to the output type.
"""
import pytest
import torch

import neptune_codegen as CG
from test_gpu_distill import check as check_distill, make as make_distill
from test_gpu_residual_norm import check as check_norm, make as make_norm
from test_gpu_rotary import heads, near

pytestmark = pytest.mark.gpu


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def close(a, b, size=None):
    """Equal up to a rounding of the output type and 2^-20 of `size` (default: the largest value)."""
    a, b = a.double(), b.double()
    size = b.abs().max() if size is None else size
    u = 2.0 ** -8
    assert ((a - b).abs() <= 2 * u * b.abs() + 2.0 ** -20 * size + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("part", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_rotary_halves_a_power_of_two_apart(part, dtype):
    dev = _dev()
    print(f"rotary part {part} {dtype}", flush=True)
    turns, _ = CG.rotary_frequencies(part, device=dev)
    positions = torch.tensor([0, 5, 70000, 123], device=dev)
    for lead in ((1, 3), (2, 33)):                   # few lanes; several heads a lane
        q = heads(*lead, 4, part, dtype, dev, "bshd", part)
        for run, sign in ((CG.run_rotary, 1), (CG.run_rotary_backward, -1)):
            near(run(q, q, positions, turns)[1], q, positions, turns, 1.0, False, sign)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,n,after,gate", [((3, 7), 8193, True, (3, 1)), ((2, 5), 12288, False, None),
                                               ((11,), 10240, True, (11,)), ((2, 3), 12289, True, ()),
                                               ((300,), 9000, True, None)])
def test_norms_of_wide_rows(lead, n, after, gate, dtype):
    dev = _dev()
    print(f"residual norm {lead}x{n} {dtype} after={after} gate={gate}", flush=True)
    check_norm(make_norm(lead, n, dtype, after, gate), 0.5, dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1040, 17000), (1030, 16387), (520, 8200), (1, 140000)])
def test_distillation_of_wide_rows(rows, n, dtype):
    dev = _dev()
    print(f"distill {rows}x{n} {dtype}", flush=True)
    check_distill(*make_distill(rows, n, 5, dtype, 9), 1.5, dev)


def test_distillation_past_32_bits():
    dev = _dev()
    rows, n, k = 70000, 65536, 8                     # 2^32 + 293 * 10^6 logits
    print("distill past 2^32 logits", flush=True)
    z = torch.zeros((rows, n), dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(0)
    z[-5:] = torch.randn((5, n), generator=g, device=dev).bfloat16()
    top = torch.randn((rows, k), generator=g, device=dev)
    index = torch.randint(0, n, (rows, k), generator=g, device=dev)
    index[:-5] = -1
    grad = torch.ones(rows, device=dev)
    loss, stats = CG.run_distill(z, top, index, return_stats=True)
    few = [t[-5:].clone() for t in (z, top, index, grad)]
    want, want_stats = CG.run_distill(*few[:3], return_stats=True)
    close(loss[-5:], want)
    close(stats[-5:], want_stats)
    dz = CG.run_distill_backward(grad, z, top, index, stats)
    close(dz[-5:], CG.run_distill_backward(few[3], *few[:3], want_stats), 2.0 ** -8)
    assert not dz[:-5].any() and not loss[:-5].any()


def test_norms_past_32_bits():
    dev = _dev()
    rows, n = 263000, 16384                          # 2^32 + 14 * 10^6 elements
    print("residual norm past 2^32 elements", flush=True)
    g = torch.Generator(device=dev).manual_seed(1)
    x, y = (torch.zeros((rows, n), dtype=torch.bfloat16, device=dev) for _ in range(2))
    for t in (x, y):
        t[-6:] = torch.randn((6, n), generator=g, device=dev).bfloat16()
    gamma = torch.ones(n, dtype=torch.bfloat16, device=dev)
    few = x[-6:].clone(), y[-6:].clone()
    r, h, stats = CG.run_residual_norm(x, y, gamma, gamma, return_stats=True)
    want = CG.run_residual_norm(*few, gamma, gamma, return_stats=True)
    for a, b in zip((r, h, stats), want):
        close(a[-6:], b)
    assert not r[:-6].any() and not h[:-6].any()
    del r, h
    dx, dy, _, _, _ = CG.run_residual_norm_backward(x, y, x, y, gamma, gamma, stats)
    wx, wy, _, _, _ = CG.run_residual_norm_backward(*few, *few, gamma, gamma, want[2])
    close(dx[-6:], wx)
    close(dy[-6:], wy)


def test_rotary_past_32_bits():
    dev = _dev()
    heads_, seq, dim = 2, 17_000_000, 128            # 2^32 + 57 * 10^6 elements
    print("rotary past 2^32 elements", flush=True)
    turns, _ = CG.rotary_frequencies(dim, device=dev)
    q = torch.zeros((1, heads_, seq, dim), dtype=torch.bfloat16, device=dev)
    q[:, :, -3:] = torch.randn((1, heads_, 3, dim), generator=torch.Generator(device=dev).manual_seed(2),
                               device=dev).bfloat16()
    positions = torch.arange(seq, device=dev)
    out, _ = CG.run_rotary(q, None, positions, turns)
    few, _ = CG.run_rotary(q[:, :, -3:].contiguous(), None, positions[-3:], turns)
    assert torch.equal(out[:, :, -3:], few) and not out[:, :, :-3].any()


def test_attention_gradients_of_rows_past_32_bits():
    dev = _dev()
    seq, wide, dim = 1100, 1 << 21, 64               # the last row 2.3 * 10^9 elements from the first
    print("attention gradients past 2^31 elements", flush=True)
    store = torch.zeros((seq, wide), dtype=torch.bfloat16, device=dev)
    rows = store[:, :dim][None, None]
    q = torch.randn((1, 1, seq, dim), generator=torch.Generator(device=dev).manual_seed(3), device=dev).bfloat16()
    rows.copy_(q)
    out, lse = CG.run_attention(q, q, q, return_lse=True)
    want = CG.run_attention_backward(q, q, q, q, out, lse)
    got = CG.run_attention_backward(rows, rows, rows, rows, out, lse)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_without_rows():
    dev = _dev()
    turns, _ = CG.rotary_frequencies(64, device=dev)
    none = torch.empty((2, 3, 0, 64), dtype=torch.bfloat16, device=dev)
    assert CG.run_rotary(none, none[:, :1], torch.empty(0, dtype=torch.int64, device=dev), turns)[1].shape == (2, 1, 0, 64)
    z = torch.empty((0, 100), dtype=torch.bfloat16, device=dev)
    lists = torch.empty((0, 4), device=dev), torch.empty((0, 4), dtype=torch.int64, device=dev)
    loss, stats = CG.run_distill(z, *lists, return_stats=True)
    assert loss.shape == (0,) and stats.shape == (0, 2)
    assert CG.run_distill_backward(loss, z, *lists, stats).shape == (0, 100)
    no_keys = torch.empty((2, 0, 5, 64), dtype=torch.bfloat16, device=dev)
    five = torch.ones((2, 3, 5, 64), dtype=torch.bfloat16, device=dev)
    q, k = CG.run_rotary(five, no_keys, torch.arange(5, device=dev), turns)
    assert torch.equal(q[:, :, 0], five[:, :, 0]) and k.shape == no_keys.shape
