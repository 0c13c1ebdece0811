"""The distillation loss and its gradient against the formulas in 64 bits.

Tolerances.  Sums of positive fp32 terms run through at most 128 additions one after another, so the
row's sum of exponentials is within 2^-17 of its value; a logarithm, a difference or a product adds a
few 2^-23 of the quantities it is made of.  So the loss is within 2^-17 T^2 sum p (|a| + |logs| + 1), a
being an entry's log p - log q, and q within 2^-17 + 2^-22 |z - max| / T of its value; the gradient's own
rounding adds half a step of its type.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


def formulas(z, t, index, temperature, grad=None):
    """(loss, its tolerance, gradient, its tolerance) in float64 on the CPU; rows without a list and
    rows with an index past the end are the caller's."""
    z, t, index = z.double().cpu(), t.double().cpu(), index.long().cpu()
    n = z.shape[1]
    absent = (index < 0) | (index >= n)
    t = (t / temperature).masked_fill(absent, -math.inf)
    log_st = torch.logsumexp(t, -1, keepdim=True)
    p = (t - log_st).exp().nan_to_num(0.0)
    log_q_all = torch.log_softmax(z / temperature, -1)
    log_q = log_q_all.gather(-1, index.masked_fill(absent, 0))
    a = torch.where(p > 0, t - log_st - log_q, 0.0)
    loss = temperature ** 2 * (p * a).sum(-1)
    top = z.amax(-1, keepdim=True)
    logs = (torch.logsumexp(z / temperature, -1, keepdim=True) - top / temperature).abs() + log_st.abs().nan_to_num(0.0)
    off = 2.0 ** -17 * temperature ** 2 * (p * (a.abs() + logs + 1.0)).sum(-1)
    if grad is None:
        return loss, off, None, None
    g = temperature * grad.double().cpu().unsqueeze(-1)
    q = log_q_all.exp() * p.sum(-1, keepdim=True)
    ptot = torch.zeros_like(q).scatter_add_(-1, index.masked_fill(absent, 0), p.masked_fill(absent, 0.0))
    far = ((z - top) / temperature).abs().nan_to_num(0.0, posinf=0.0)
    dz_off = g.abs() * (q * (2.0 ** -17 + 2.0 ** -22 * far) + 2.0 ** -17 * ptot)
    return loss, off, g * (q - ptot), dz_off


def make(rows, n, k, dtype, seed=0, top_dtype=torch.float32, index_dtype=torch.int64, twice=False):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(rows, n, generator=g)).to(dtype)
    t = (3 * torch.randn(rows, k, generator=g)).to(top_dtype)
    index = torch.stack([torch.randperm(n, generator=g)[:k] if k <= n else torch.randint(n, (k,), generator=g)
                         for _ in range(rows)])
    if twice:
        index = torch.randint(min(n, 5), (rows, k), generator=g)
    length = torch.randint(1, k + 1, (rows, 1), generator=g)
    length[0] = k
    index[torch.arange(k)[None] >= length] = -1
    grad = torch.rand(rows, generator=g)
    return z, t, index.to(index_dtype), grad


def check(z, t, index, grad, temperature, dev, view=lambda x: x):
    zd, td, xd, gd = (x.to(dev) for x in (z, t, index, grad))
    zd = view(zd)
    loss, stats = CG.run_distill(zd, td, xd, temperature=temperature, return_stats=True)
    dz = CG.run_distill_backward(gd, zd, td, xd, stats, temperature=temperature)
    want, off, dwant, doff = formulas(z, t, index, temperature, grad)
    ratio = ((loss.double().cpu() - want).abs() / (off + 1e-30)).max().item()
    assert loss.dtype == torch.float32 and ratio <= 1.0, ("loss", ratio)
    assert torch.equal(CG.run_distill(zd, td, xd, temperature=temperature), loss)
    assert dz.dtype == z.dtype and dz.is_contiguous()
    u = torch.finfo(z.dtype).eps / 2
    tiny = 2.0 ** -25 if z.dtype == torch.float16 else 1e-37
    ratio = ((dz.double().cpu() - dwant).abs() / (doff * (1 + u) + u * dwant.abs() + tiny)).max().item()
    assert ratio <= 1.0, ("gradient", ratio)
    assert torch.equal(CG.run_distill_backward(gd, zd, td, xd, stats, temperature=temperature), dz)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 2, 2), (5, 33, 7), (9, 1000, 8), (4, 10007, 64), (600, 4100, 3),
                                      (2, 50257, 200), (700, 8200, 100), (6, 32000, 64), (1, 65536, 1024)])
def test_loss_and_gradient_match_the_formulas(rows, n, k, dtype):
    dev = _dev()
    print(f"distill {rows}x{n} k={k} {dtype}", flush=True)
    check(*make(rows, n, k, dtype), 1.0 if rows % 2 else 2.5, dev)


@pytest.mark.parametrize("top_dtype,index_dtype", [(torch.bfloat16, torch.int32), (torch.float32, torch.int32),
                                                   (torch.bfloat16, torch.int64)])
def test_types_of_the_lists(top_dtype, index_dtype):
    dev = _dev()
    print(f"distill lists {top_dtype} {index_dtype}", flush=True)
    check(*make(7, 3000, 20, torch.bfloat16, 1, top_dtype, index_dtype), 1.5, dev)


@pytest.mark.parametrize("n,k", [(5, 40), (3000, 64), (9000, 300), (20000, 1000)])
def test_an_index_that_comes_again_adds_its_probabilities(n, k):
    dev = _dev()
    print(f"distill repeated indices n={n} k={k}", flush=True)
    check(*make(6, n, k, torch.float32, 2, twice=True), 1.0, dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows(dtype):
    dev = _dev()
    z, t, index, grad = make(8, 1003, 16, dtype, 3)
    wide = torch.zeros(8, 1100, dtype=dtype)
    wide[:, 5:1008] = z
    print(f"distill strided {dtype}", flush=True)
    check(z, t, index, grad, 1.0, dev, lambda _: wide.to(dev)[:, 5:1008])
    columns = z.t().contiguous()
    check(z, t, index, grad, 1.0, dev, lambda _: columns.to(dev).t())


def test_leading_sizes_and_a_mean_gradient():
    dev = _dev()
    z, t, index, _ = make(12, 500, 9, torch.bfloat16, 4)
    zd, td, xd = z.view(3, 4, 500).to(dev), t.view(3, 4, 9).to(dev), index.view(3, 4, 9).to(dev)
    print("distill leading sizes", flush=True)
    loss, stats = CG.run_distill(zd, td, xd, return_stats=True)
    assert loss.shape == (3, 4) and stats.shape == (3, 4, 2)
    flat = CG.run_distill(z.to(dev), t.to(dev), index.to(dev))
    assert torch.equal(loss.view(-1), flat)
    one = torch.full((), 0.25, device=dev)
    dz = CG.run_distill_backward(one.expand(3, 4), zd, td, xd, stats)
    assert torch.equal(dz, CG.run_distill_backward(torch.full((3, 4), 0.25, device=dev), zd, td, xd, stats))
    single = CG.run_distill(z[0].to(dev), t[0].to(dev), index[0].to(dev))
    assert single.shape == () and torch.equal(single, flat[0])


@pytest.mark.parametrize("n", [300, 20003])
def test_empty_lists_masked_logits_and_bad_indices(n):
    dev = _dev()
    z, t, index, grad = make(8, n, 6, torch.float32, 5)
    index[:] = torch.arange(6) * 7 + 1
    index[0] = -1                                    # no entry
    z[0, 3] = math.nan
    t[1] = -math.inf                                 # entries without probability
    z[2, index[2, 1]] = -math.inf                    # a masked token the teacher gives some
    t[3, 2] = -math.inf                              # an entry without, at a masked token
    z[3, index[3, 2]] = -math.inf
    z[4, n // 2:] = -math.inf                        # a masked part of the vocabulary
    index[5, 4] = n                                  # past the end
    t[6, 1] = math.nan
    z[7, 9] = math.inf
    print(f"distill edge rows n={n}", flush=True)
    zd, td, xd, gd = (x.to(dev) for x in (z, t, index, grad))
    loss, stats = CG.run_distill(zd, td, xd, return_stats=True)
    dz = CG.run_distill_backward(gd, zd, td, xd, stats).cpu()
    loss = loss.cpu()
    assert loss[0] == 0 and not dz[0].any()
    assert loss[1] == 0 and not dz[1].any()
    assert loss[2] == math.inf
    assert loss[5].isnan() and dz[5].isnan().all()
    assert loss[6].isnan() and dz[6].isnan().all()
    assert loss[7].isnan()
    want, off, dwant, doff = formulas(z, t, index, 1.0, grad)
    for r in (3, 4):
        assert abs(loss[r].double() - want[r]) <= off[r]
    for r in (2, 3, 4):
        assert torch.isfinite(dz[r]).all()
        assert ((dz[r].double() - dwant[r]).abs() <= doff[r] + 2.0 ** -24 * dwant[r].abs() + 1e-37).all(), r


def test_gradient_matches_differences():
    """Central differences of the loss's formula in 64 bits around the kernel's gradient."""
    dev = _dev()
    z, t, index, grad = make(2, 40, 5, torch.float32, 6)
    zd, td, xd, gd = (x.to(dev) for x in (z, t, index, grad))
    print("distill differences", flush=True)
    _, stats = CG.run_distill(zd, td, xd, temperature=2.0, return_stats=True)
    dz = CG.run_distill_backward(gd, zd, td, xd, stats, temperature=2.0).double().cpu()
    h = 1e-4
    for r, j in ((0, int(index[0, 0])), (0, 39), (1, int(index[1, 0])), (1, 0)):
        shifted = [z.double().clone() for _ in range(2)]
        shifted[0][r, j] += h
        shifted[1][r, j] -= h
        up, down = (formulas(s, t, index, 2.0)[0][r] for s in shifted)
        # the third derivative of the loss is below T^2 / T^3: h^2 / 6 of it, and 32-bit roundings
        assert abs(dz[r, j] - grad[r].double() * (up - down) / (2 * h)) <= 1e-6


def test_registered_operator_and_captured_replays():
    dev = _dev()
    z, t, index, grad = make(20, 5000, 30, torch.bfloat16, 7)
    zd, td, xd, gd = (x.to(dev) for x in (z, t, index, grad))
    op = CG.as_distill_op(temperature=2.0)
    leaf = zd.clone().requires_grad_()
    print("distill through autograd", flush=True)
    loss, stats = op(leaf, td, xd)
    (dz,) = torch.autograd.grad(loss, leaf, gd)
    assert torch.equal(dz, CG.run_distill_backward(gd, zd, td, xd, stats, temperature=2.0))
    assert torch.equal(loss.detach(), CG.run_distill(zd, td, xd, temperature=2.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, stats = CG.run_distill(zd, td, xd, temperature=2.0, return_stats=True)
        dz = CG.run_distill_backward(gd, zd, td, xd, stats, temperature=2.0)
    for i in range(4):
        zd.copy_((3 * torch.randn(z.shape, generator=torch.Generator().manual_seed(i))).to(z.dtype))
        graph.replay()
        want, ws = CG.run_distill(zd, td, xd, temperature=2.0, return_stats=True)
        wz = CG.run_distill_backward(gd, zd, td, xd, ws, temperature=2.0)
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(dz, wz), i
