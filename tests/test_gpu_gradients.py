"""The gradients' norm and clipping against their definition in 64 bits.

Tolerances.  Squares and sums are fp64 (n additions: n 2^-53, nothing beside fp32), so the norm is off by its one
rounding: 2^-24, and 2^-24 (1 + 2^-16) is allowed.  The factor is the fp32 quotient of max_norm and that norm, an
element one fp32 product, rounded to its type: the same bits as torch's.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def model(sizes, dev, seed=0, by=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(by * torch.randn(shape, generator=g)).to(dtype).to(dev) for shape, dtype in sizes]


def norm64(ts):
    return math.sqrt(math.fsum(t.detach().double().cpu().square().sum().item() for t in ts))


def check_norm(got, ts):
    want = norm64(ts)
    assert got.shape == () and got.dtype == F32
    assert abs(got.item() - want) <= 2.0 ** -24 * (1 + 2.0 ** -16) * want + 2.0 ** -150
    return got


LISTS = {
    "one": [((1,), F32)], "scalar": [((), BF16)], "small": [((3, 5), F16), ((7,), F32), ((2, 2, 2), BF16)],
    "empty": [((0,), F32), ((4, 0), BF16)], "some empty": [((0,), F32), ((9,), BF16), ((3, 0), F16), ((1,), F16)],
    "layer": [((96, 96), BF16), ((96,), F32), ((257, 33), BF16), ((31,), F16)],
    "many": [((1 + 37 * i % 101, 3), (F32, BF16, F16)[i % 3]) for i in range(300)],
    "112": [((5,), BF16)] * 112, "113": [((5,), BF16)] * 113, "224": [((9,), F32)] * 224, "4096": [((3,), F16)] * 4096, "4500": [((1 + i % 5,), F32) for i in range(4500)],
    "64 KB": [((16384,), F32)], "over 64 KB": [((16384,), F32), ((1,), F16)], "16 pieces": [((4096 * 3 + 5,), F16), ((4096,), BF16)],
    "piece": [((8192,), F32), ((8193,), F32), ((8191,), F32), ((16384,), BF16), ((24577,), F16)],
    "large": [((4096, 2049), BF16), ((5000, 1111), F32), ((3000001,), F16)],
    "larger": [((20000, 4096), BF16), ((70000001,), BF16), ((4097, 4097), F32)],
}


@pytest.mark.parametrize("name", LISTS)
def test_norm_and_clipping(name):
    dev = _dev()
    print(f"gradients {name}", flush=True)
    ts = model(LISTS[name], dev)
    norm = check_norm(CG.run_gradient_norm(ts), ts)
    assert torch.equal(norm, CG.run_gradient_norm(tuple(ts)))
    for bound in (0.25, 1e9, 0.0):
        factor = torch.where(norm > bound, torch.tensor(bound, device=dev) / norm, 1.0)
        want = [(t.float() * factor).to(t.dtype) for t in ts]
        wider = [t.float() * factor for t in ts]
        for given in (None, norm):
            own = [t.clone() for t in ts]
            assert torch.equal(CG.run_clip_gradients(own, bound, norm=given), norm)
            assert all(torch.equal(a, b) for a, b in zip(own, want))
            out = [torch.full_like(t, 7) for t in ts]
            assert torch.equal(CG.run_clip_gradients(ts, bound, norm=given, out=out), norm)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            out = [torch.full_like(t, 7, dtype=F32) for t in ts]
            CG.run_clip_gradients(ts, bound, norm=given, out=out)
            assert all(torch.equal(a, b) for a, b in zip(out, wider))
    if norm > 0:
        clipped = [t.clone() for t in ts]
        CG.run_clip_gradients(clipped, 0.5 * norm.item())
        # elements are rounded to their types after the scaling
        assert abs(norm64(clipped) / norm64(ts) - 0.5) <= 0.5 * 2.0 ** -8


def test_any_alignment_order_and_mixed_outputs():
    dev = _dev()
    base = torch.randn(5000, device=dev)
    half = torch.randn(5001, device=dev).bfloat16()
    for at in range(1, 9):
        print(f"gradients at {at}", flush=True)
        ts = [base[at:at + 1000], half[at:at + 2003], half[4001 - at:4001 - at + 7], base[3000 + at:3001 + at]]
        norm = check_norm(CG.run_gradient_norm(ts), ts)
        factor = torch.tensor(0.1, device=dev) / norm
        whole, whole_half = base.clone(), half.clone()
        own = [whole[at:at + 1000], whole_half[at:at + 2003], whole_half[4001 - at:4001 - at + 7],
               whole[3000 + at:3001 + at]]
        CG.run_clip_gradients(own, 0.1)
        assert all(torch.equal(a, (b.float() * factor).to(b.dtype)) for a, b in zip(own, ts))
        # what lies between is left alone
        for t, ranges, before in ((whole, ((0, at), (at + 1000, 3000 + at), (3001 + at, 5000)), base),
                                  (whole_half, ((0, at), (at + 2003, 4001 - at), (4008 - at, 5001)), half)):
            for a, b in ranges:
                assert torch.equal(t[a:b], before[a:b])
    cube = torch.randn(3, 4, 5, 6, device=dev).half()
    ts = [cube.permute(2, 0, 3, 1), torch.randn(2, 3, 4, 4, device=dev).to(memory_format=torch.channels_last)]
    norm = check_norm(CG.run_gradient_norm(ts), ts)
    out = [torch.empty_like(t) for t in ts]          # (of the same order)
    mixed = [out[0], ts[1].clone(memory_format=torch.preserve_format)]
    CG.run_clip_gradients([ts[0], mixed[1]], 1.0, out=mixed)               # one of them in place
    factor = 1.0 / norm
    assert all(torch.equal(a, (b.float() * factor).to(b.dtype)) for a, b in zip(mixed, ts))
    # with gaps, expanded or named twice: the norm reads what the tensors hold
    ts = [cube[:, :, 1:3], cube[:1, :1, :1, :1].expand(2, 3, 4, 5), cube[0], cube[0], cube[:1].transpose(1, 3)]
    check_norm(CG.run_gradient_norm(ts), ts)
    ts = [torch._neg_view(base), torch.complex(base, base).conj().imag]     # negated when they are read
    check_norm(CG.run_gradient_norm(ts), ts)
    with pytest.raises(ValueError):
        CG.run_clip_gradients(ts[:1], 1.0)


def test_the_ends_of_the_range():
    dev = _dev()
    for values in ([3e38, -2e38, 1e-30], [1e-44, 2e-44, -1.4e-45], [1e-22] * 5, [0.0, -0.0]):
        ts = [torch.tensor(values, device=dev), torch.tensor(values, device=dev).bfloat16()]
        if max(values) > 1e38:
            ts[0] /= 2
            ts = ts[:1]
        print(f"gradients of {values[0]}", flush=True)
        check_norm(CG.run_gradient_norm(ts), ts)
    big = [torch.full((100,), 3e38, device=dev)]      # a norm that fp32 does not hold
    before = big[0].clone()
    assert CG.run_clip_gradients(big, 1.0) == math.inf and torch.equal(big[0], before)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_gradients_without_a_finite_norm_stay_as_they_are(bad):
    dev = _dev()
    ts = model(LISTS["layer"], dev)
    ts[2][5, 7] = bad
    before = [t.clone() for t in ts]
    norm = CG.run_clip_gradients(ts, 0.5)
    assert norm.isnan() if math.isnan(bad) else norm == math.inf
    same = lambda a, b: torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))  # noqa: E731
    assert all(same(a, b) for a, b in zip(ts, before))
    out = [torch.zeros_like(t) for t in ts]
    CG.run_clip_gradients(ts, 0.5, out=out)
    assert all(same(a, b) for a, b in zip(out, before))


def test_refused_calls_on_the_device():
    dev = _dev()
    x, y = torch.ones(64, device=dev), torch.ones(64, device=dev)
    before = x.clone()
    for ts, kw in (([x, x], {}), ([x[:40], x[30:]], {}), ([x, y], {"out": [y, x]}), ([x], {"out": [y], "norm": y[0]}),
                   ([x[::2]], {}), ([x.view(8, 8)[:, :4]], {}), ([x[:1].expand(5)], {}), ([x.view(8, 8)], {"out": [y.view(8, 8).T]}),
                   ([x.clone().requires_grad_()], {}), ([y], {"out": [x.clone().requires_grad_()]}),
                   ([x, y], {"norm": x[3]}), ([x[:32].bfloat16(), x], {"out": [x[:32], y]})):
        with pytest.raises(ValueError):
            CG.run_clip_gradients(ts, 0.5, **kw)
    with pytest.raises(ValueError):
        CG.run_clip_gradients([x, torch.ones(3)], 0.5)
    with pytest.raises(ValueError):
        CG.run_gradient_norm([x, torch.ones(3)])
    assert torch.equal(x, before)
    from neptune_codegen import hip

    with hip.recording(), pytest.raises(NotImplementedError):
        CG.run_gradient_norm([x])
    # one tensor read twice, and a norm read while another list is written
    out = [torch.empty_like(x), torch.empty_like(x)]
    CG.run_clip_gradients([x, x], 1.0, out=out)
    assert torch.equal(out[0], out[1])


def test_written_tensors_are_known_to_autograd():
    dev = _dev()
    x, y = torch.ones(9, device=dev), torch.ones(9, device=dev)
    CG.run_clip_gradients([x], 1.0)
    assert x._version == 1
    version = y._version
    CG.run_clip_gradients([x], 0.5, out=[y])
    assert y._version == version + 1 and x._version == 1
    with torch.inference_mode():
        z = torch.ones(9, device=dev)
        CG.run_clip_gradients([z], 1.0)
    p = torch.nn.Parameter(torch.ones(4, device=dev))
    (p * 2).sum().backward()
    assert CG.run_clip_gradients([p.grad], 1.0) == 4.0 and (p.grad == 0.5).all()
    check_norm(CG.run_gradient_norm([p]), [p])


def test_captured_replays_and_streams():
    dev = _dev()
    sizes = LISTS["many"] + LISTS["large"]
    sets = [model(sizes, dev, seed=s) for s in range(3)]

    def step(ts):
        out = [torch.empty_like(t, dtype=F32) for t in ts]
        norm = CG.run_clip_gradients(ts, 0.5, out=out)
        return [CG.run_gradient_norm(out), norm, *out]

    want = [[t.clone() for t in step(s)] for s in sets]
    static = [[t.clone() for t in sets[0]] for _ in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        print(f"replay {turn}", flush=True)
        picks = [turn % 3, (turn + 1) % 3]
        for s, p in zip(static, picks):
            for a, b in zip(s, sets[p]):
                a.copy_(b)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager = step(sets[2])
        for out, p in zip(outs, picks):
            assert all(torch.equal(a, b) for a, b in zip(out, want[p]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[2]))
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for run in got[i] for a, b in zip(run, want[i]))


def test_registered_operators_keep_their_contracts():
    dev = _dev()
    ts = model(LISTS["layer"], dev)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    print("contracts of the gradients' operators", flush=True)
    torch.library.opcheck(CG.as_gradient_norm_op(), (ts,), test_utils=tests)
    torch.library.opcheck(CG.as_clip_gradients_op(), (ts, 0.5), test_utils=tests)
    own = [t.clone() for t in ts]
    norm = CG.as_clip_gradients_op()(own, 0.5)
    assert torch.equal(norm, CG.run_clip_gradients(ts, 0.5))
    assert all(torch.equal(a, b) for a, b in zip(own, ts))


def test_more_than_32_bits_of_bytes():
    dev = _dev()
    print("a gradient of 2^31 + 9 elements", flush=True)
    t = torch.zeros((1 << 31) + 9, dtype=BF16, device=dev)
    t[0], t[1 << 30], t[-1], t[-9] = 3.0, 4.0, 12.0, 84.0
    assert CG.run_clip_gradients([t[:5], t[5:]], 17.0) == math.sqrt(9 + 16 + 144 + 7056)
    assert [t[i].item() for i in (0, 1 << 30, -1, -9)] == [
        (torch.tensor(v) * (torch.tensor(17.0) / math.sqrt(7225))).bfloat16().item() for v in (3.0, 4.0, 12.0, 84.0)]
