"""The residual norm's 8-bit output against its definition in 64 bits.

Tolerances.  The normed value h before its rounding is that of run_residual_norm: within 2^-16 of its terms' sizes
(tests/test_gpu_residual_norm.py).  A scale is the largest of them over the format's largest value: within 2^-16 of
the block's largest size, and an fp32 quotient (2^-23).  A value q is h / scale (a reciprocal, a product and a step from it, 2^-22),
rounded: off by that, and by half a step of the format at h / scale.  With fp32 inputs h is two products from the
residual and the rate, and scales and values are to the bit the quotient, reciprocal, product and step.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu
E4, E5, I8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.int8
MOST = {E4: 448.0, E5: 57344.0, I8: 127.0}
LEAST = 2.0 ** -126
EPS = 1e-6


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def make(lead, n, dtype, after=True, gate=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": 2 * rand(*lead, n), "y": rand(*lead, n), "after": 1 + 0.2 * rand(n) if after else None,
         "before": 1 + 0.2 * rand(n), "gate": None if gate is None else 0.5 * rand(*gate, n)}
    return {k: None if v is None else v.to(dtype) for k, v in t.items()}


def formulas(t, scale):
    """(residual, its terms' sizes, rates, normed, its terms' sizes) in float64."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    c, rates = d["y"], [torch.ones_like(d["y"][..., :1])]
    if d["after"] is not None:
        rates = [(c.square().mean(-1, keepdim=True) + EPS).rsqrt()]
        c = c * rates[0] * d["after"]
    if d["gate"] is not None:
        c = c * d["gate"]
    r = d["x"] + scale * c
    rate = (r.square().mean(-1, keepdim=True) + EPS).rsqrt()
    size = d["x"].abs() + (scale * c).abs()
    return r, size, torch.cat([*rates, rate], -1), r * rate * d["before"], size * rate * d["before"].abs()


def blocks(v, group):
    return torch.nn.functional.pad(v, (0, -v.shape[-1] % (group or v.shape[-1]))).unflatten(-1, (-1, group or v.shape[-1]))


def steps(v, fmt):
    """Step of the format at magnitude v, a little over it."""
    if fmt == I8:
        return torch.ones_like(v)
    bits, least = (3, -6) if fmt == E4 else (2, -14)
    return 2.0 ** ((v * (1 + 2.0 ** -10)).clamp(min=2.0 ** least).log2().floor() - bits)


def check(t, dev, fmt, group, power, scale=0.5):
    d = {k: None if v is None else v.to(dev) for k, v in t.items()}
    args = (d["x"], d["y"], d["after"], d["before"])
    kw = dict(gate=d["gate"], residual_scale=scale, eps=EPS)
    given = dict(dtype=fmt, group=group, power_of_two=power)
    r, q, s, stats = CG.run_residual_norm_quantized(*args, **kw, **given, return_stats=True)
    again = CG.run_residual_norm_quantized(*args, **kw, **given)
    as_bytes = lambda v: v.view(torch.uint8)  # noqa: E731
    assert torch.equal(r, again[0]) and torch.equal(as_bytes(q), as_bytes(again[1])) and torch.equal(s, again[2])
    want_r, size_r, want_stats, h, size = formulas(t, scale)
    # as run_residual_norm's (whose bits they need not have: an fp16 sum may be rounded once, or to fp32 first)
    u = torch.finfo(r.dtype).eps / 2
    tiny = 2.0 ** -25 if r.dtype == torch.float16 else 0.0
    assert ((r.double().cpu() - want_r).abs() <= 2.0 ** -17 * size_r + u * want_r.abs() + tiny).all()
    assert ((stats.double().cpu() - want_stats).abs() <= 2.0 ** -17 * want_stats).all()
    n = t["x"].shape[-1]
    assert q.dtype == fmt and q.shape == r.shape and s.shape == (*r.shape[:-1], -(-n // group) if group else 1)
    assert q.is_contiguous() and s.is_contiguous()
    hb, sb = blocks(h, group), blocks(size, group)
    got = s.double().cpu()
    off = 2.0 ** -16 * sb.amax(-1) / MOST[fmt]
    want = hb.abs().amax(-1) / MOST[fmt]
    if power:
        assert (torch.frexp(got).mantissa == 0.5).all() and (got >= LEAST).all()
        assert (got >= want - off).all() and ((got / 2 < want + off) | (got == LEAST)).all()
    else:
        assert ((got - want.clamp(min=LEAST)).abs() <= off + 2.0 ** -22 * want).all()
    values = blocks(q.float().cpu().double(), group)
    ratio = hb / got.unsqueeze(-1)
    allowed = 2.0 ** -16 * sb / got.unsqueeze(-1) + 2.0 ** -22 * ratio.abs() + 0.5 * steps(ratio.abs(), fmt)
    assert ((values - ratio).abs() <= allowed).all()
    assert values.abs().max() <= MOST[fmt]
    if t["x"].dtype == torch.float32:
        # (the residual is not rounded, and normed two products from it)
        hf = blocks(r * stats[..., 1:] * d["before"], group)
        # quotients in 64 bits, then rounded, are those of fp32 (on the device torch divides by a number as it
        # multiplies by its reciprocal)
        if not power:
            assert torch.equal(s, (hf.abs().amax(-1).double() / MOST[fmt]).float().clamp(min=LEAST))
        inverse, d = (1.0 / s.double()).float().unsqueeze(-1), s.double().unsqueeze(-1)
        v = hf * inverse
        if not power:                                # one step from the product to the quotient
            rest = (hf.double() - v.double() * d).float()
            v = (v.double() + rest.double() * inverse.double()).float()
        v = v.flatten(-2)[..., :n]
        v = v.round().clamp(-127, 127) if fmt == I8 else v
        assert torch.equal(as_bytes(q), as_bytes(v.to(fmt)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,n,after,gate", [
    ((1,), 1, True, None), ((3,), 5, True, (3,)), ((2, 7), 64, True, (2, 1)), ((9,), 1000, False, None),
    ((4, 33), 1024, True, (4, 1)), ((700,), 96, True, ()), ((2, 3, 5), 333, True, (2, 3, 1)), ((5,), 8, False, None),
    ((1, 130), 4096, True, (1, 1)), ((1100,), 4096, False, None), ((40,), 2999, False, (40,)), ((1100,), 2999, True, None),
    ((5,), 8192, True, (5,)), ((2, 3), 16384, True, (2, 1)), ((3,), 10007, True, ()), ((600, 2), 128, True, (600, 1)),
    ((1000,), 16, False, ()), ((17,), 40, True, None), ((1030,), 8773, True, (1030,)), ((1050,), 1110, True, ()),
    ((1025,), 12544, False, None), ((1024,), 721, True, None)])
def test_values_and_scales(lead, n, after, gate, dtype):
    dev = _dev()
    t = make(lead, n, dtype, after, gate, seed=n)
    forms = ((E4, None, False), (E5, 32, True), (I8, 128, False), (E4, 64, True), (E5, None, True),
             (I8, None, True), (E4, 128, False), (E5, 64, False), (I8, 32, False))
    # (two of the nine for each case and type: each is a kernel of its own)
    first = (7 * n + lead[0] + 4 * dtype.itemsize) % 9
    for fmt, group, power in (forms[first], forms[(first + 4) % 9]):
        print(f"8-bit norm {lead} x {n} {dtype} {fmt} {group} {power}", flush=True)
        check(t, dev, fmt, group, power)


def test_powers_of_two_at_their_edges():
    # blocks whose largest magnitude is at, just over and just under the format's largest value times a power
    dev = _dev()
    for fmt in (E4, E5, I8):
        m = MOST[fmt]
        edges = [m * 2.0 ** k * f for k in (-20, -8, 0, 9) for f in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -23, 0.5, 1.9)]
        n = 32 * len(edges)
        before = torch.ones(n)
        before[::32] = torch.tensor(edges)
        before[1::32] = torch.tensor(edges) / 3
        for k in range(2, 32):
            before[k::32] = 0.0
        x = torch.ones(2, n, device=dev)
        print(f"powers of two for {fmt}", flush=True)
        # (the rate of a row of ones is 1 - 5e-7: out it comes, by an eps that fp32 does not see)
        _, h = CG.run_residual_norm(x, torch.zeros_like(x), None, before.to(dev), eps=1e-30)
        assert torch.equal(h[0].cpu(), before)
        _, q, s = CG.run_residual_norm_quantized(x, torch.zeros_like(x), None, before.to(dev), eps=1e-30, dtype=fmt,
                                                 group=32, power_of_two=True)
        for e, got, v in zip(before[::32].double().tolist(), s[0].tolist(), q[0].float().cpu()[::32].tolist()):
            # the least power of two with e / got <= m
            assert math.frexp(got)[0] == 0.5 and e / got <= m < 2 * e / got, (fmt, e, got)
            assert abs(v * got - e) <= 0.5 * steps(torch.tensor(e / got, dtype=torch.float64), fmt).item() * got


def test_zeros_tiny_and_non_finite_blocks():
    dev = _dev()
    t = make((8,), 256, torch.float32, False, None, seed=3)
    t["x"][0], t["y"][0] = 0.0, 0.0
    t["before"][32:64] = 0.0
    t["before"][64:96] = 1e-38
    t["before"][96:128] = 1e-44
    t["x"][2, 5], t["x"][3, 200] = math.nan, math.inf
    d = {k: None if v is None else v.to(dev) for k, v in t.items()}
    for fmt in (E4, E5, I8):
        for power in (False, True):
            print(f"edge blocks {fmt} {power}", flush=True)
            _, q, s = CG.run_residual_norm_quantized(d["x"], d["y"], None, d["before"], dtype=fmt, group=32,
                                                     power_of_two=power)
            q, s = q.float().cpu(), s.cpu()
            assert (s[0] == LEAST).all() and not q[0].any()              # a row of zeros
            fine = [1, 4, 5, 6, 7]
            assert torch.isfinite(s[fine]).all() and (s[fine] >= LEAST).all() and not q[fine, 32:64].any()
            assert (s[fine, 1] == LEAST).all() and (s[fine, 3] == LEAST).all()
            assert s[2].isnan().all()                                    # the rate of a NaN is one
            assert s[3, 6].isnan() and torch.isfinite(s[3, [0, 4, 5, 7]]).all()    # inf times a rate of 0
            _, q, s = CG.run_residual_norm_quantized(d["x"], d["y"], None, d["before"], dtype=fmt, power_of_two=power)
            assert s[2:4].isnan().all() and torch.isfinite(s[[0, 1, 4, 5, 6, 7]]).all()
            big = d["before"].clone()
            big[7] = math.inf
            _, q, s = CG.run_residual_norm_quantized(d["x"], d["y"], None, big, dtype=fmt, group=32, power_of_two=power)
            assert torch.isinf(s[fine, 0]).all() and torch.isfinite(s[fine, 1:]).all()
            # what the block stands for is not finite in any column
            assert not torch.isfinite(q[fine].float()[:, :32] * s[fine, :1]).any()


def test_strides_and_a_scale_for_the_gradient():
    dev = _dev()
    t = make((6, 10), 520, torch.bfloat16, True, (6, 1), seed=1)
    d = {k: v.to(dev) for k, v in t.items()}
    call = lambda x, y: CG.run_residual_norm_quantized(  # noqa: E731
        x, y, d["after"], d["before"], gate=d["gate"], group=64, return_stats=True)
    want = call(d["x"], d["y"])
    wide = torch.zeros(6, 10, 1100, dtype=torch.bfloat16, device=dev)
    for offset in (0, 8, 3):
        print(f"8-bit norm at {offset}", flush=True)
        wide[..., offset:offset + 520] = d["x"]
        got = call(wide[..., offset:offset + 520], d["y"].transpose(0, 1).contiguous().transpose(0, 1))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # the gradient goes straight through the rounding: the norm's own
    grad = torch.randn(6, 10, 520, device=dev).bfloat16()
    plain = CG.run_residual_norm(d["x"], d["y"], d["after"], d["before"], gate=d["gate"], return_stats=True)
    back = [CG.run_residual_norm_backward(None, grad, d["x"], d["y"], d["after"], d["before"], st, gate=d["gate"])
            for st in (want[3], plain[2])]
    assert all(torch.equal(a, b) for a, b in zip(*back))


def test_captured_replays_and_the_registered_operator():
    dev = _dev()
    t = make((4, 50), 256, torch.bfloat16, True, (4, 1), seed=4)
    d = {k: v.to(dev) for k, v in t.items()}
    op = CG.as_residual_norm_quantized_op(0.5, EPS, E4, 32, True)
    args = (d["x"], d["y"], d["after"], d["before"], d["gate"])
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # noqa: E731
    direct = lambda: CG.run_residual_norm_quantized(  # noqa: E731
        *args[:4], gate=args[4], residual_scale=0.5, eps=EPS, dtype=E4, group=32, power_of_two=True, return_stats=True)
    assert all(same(a, b) for a, b in zip(op(*args), direct()))
    print("contracts of the 8-bit norm", flush=True)
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = direct()
    for i in range(4):
        d["y"].copy_(torch.randn(4, 50, 256, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        ref = direct()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(out, ref)), i


def test_a_seen_layout_does_not_lend_its_type():
    dev = _dev()
    x, g = torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    values = [CG.run_residual_norm_quantized(x, x, None, g, **kw)[1] for kw in ({}, {"dtype": E4}, {"dtype": E5}, {"dtype": I8}) * 2]
    assert [v.dtype for v in values] == [E4, E4, E5, I8] * 2
    for kw in ({"dtype": torch.float16}, {"dtype": "float8_e4m3fn"}, {"dtype": 0}):
        with pytest.raises(TypeError):
            CG.run_residual_norm_quantized(x, x, None, g, **kw)
    CG.run_residual_norm_quantized(x, x, None, g, group=32)
    for group in (32.0, True, 33):
        with pytest.raises(ValueError):
            CG.run_residual_norm_quantized(x, x, None, g, group=group)


def test_no_rows():
    dev = _dev()
    x, g = torch.empty(0, 64, dtype=torch.bfloat16, device=dev), torch.ones(64, dtype=torch.bfloat16, device=dev)
    r, q, s = CG.run_residual_norm_quantized(x, x, g, g, group=32)
    assert r.shape == q.shape == (0, 64) and s.shape == (0, 2)
