"""The embedding and its gradient against the definition in 64 bits.

Tolerances.  The lookup is one fp32 product, rounded: its bits are those of torch's product.  A gradient's
row of c terms is c - 1 fp32 additions in some order, a product by the scale and (added into a tensor) one more
addition: off by at most (c + 2) 2^-24 times the sum of the terms' sizes, and half a step of the result.
"""
import math

import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def make_tokens(kind, count, vocab, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        t = torch.full((count,), vocab // 2)
    elif kind == "distinct":
        t = torch.arange(count).flip(0) % vocab
    elif kind == "none":
        t = torch.full((count,), -1)
    elif kind == "few":
        t = torch.randint(0, min(3, vocab), (count,), generator=g) * max(1, (vocab - 1) // 2)
        t = t.clamp(max=vocab - 1)
    else:
        t = ((torch.rand(count, generator=g, dtype=torch.float64) * math.log(vocab + 1)).exp().long() - 1).clamp(0, vocab - 1)
        t[torch.rand(count, generator=g) < 0.1] = -1
        if kind == "past":
            t[torch.rand(count, generator=g) < 0.1] = vocab
            t[torch.rand(count, generator=g) < 0.1] = vocab + 5
            t[torch.rand(count, generator=g) < 0.1] = torch.iinfo(dtype).max
            t[torch.rand(count, generator=g) < 0.1] = torch.iinfo(dtype).min
    return t.to(dtype)


def want_lookup(tokens, table, scale):
    known = (tokens >= 0) & (tokens < table.shape[0])
    rows = (table.float()[torch.where(known, tokens, 0).long()] * scale)
    rows[tokens < 0] = 0.0
    rows[tokens >= table.shape[0]] = math.nan
    return rows.to(table.dtype)


def want_gradient(grad, tokens, vocab, scale, into=None):
    """(sum, what it may be off by) in float64 on the CPU."""
    n = grad.shape[-1]
    here = (tokens >= 0) & (tokens < vocab)
    at, rows = tokens[here].long(), grad[here].double().reshape(-1, n) * scale
    total = torch.zeros(vocab, n, dtype=torch.float64).index_add_(0, at, rows)
    size = torch.zeros(vocab, n, dtype=torch.float64).index_add_(0, at, rows.abs())
    count = torch.bincount(at, minlength=vocab).unsqueeze(-1)
    dtype = grad.dtype
    if into is not None:
        dtype = into.dtype
        total, size = total + into.double(), size + into.double().abs()
    off = (count + 2) * 2.0 ** -24 * size
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return total, off * (1 + u) + u * total.abs() + tiny


def check_gradient(grad, tokens, vocab, scale, dev, into=None):
    d, i = grad.to(dev), tokens.to(dev)
    args = dict(scale=scale)
    got = CG.run_embedding_backward(d, i, vocab, **args, into=None if into is None else into.to(dev).clone())
    again = CG.run_embedding_backward(d, i, vocab, **args, into=None if into is None else into.to(dev).clone())
    assert torch.equal(got, again)                   # one order
    want, off = want_gradient(grad, tokens, vocab, scale, into)
    assert got.shape == want.shape and got.dtype == (grad.dtype if into is None else into.dtype)
    ratio = ((got.double().cpu() - want).abs() / off).max().item()
    assert ratio <= 1.0, ratio
    named = torch.zeros(vocab, dtype=torch.bool)
    named[tokens[(tokens >= 0) & (tokens < vocab)].long()] = True
    rest = torch.zeros_like(got[0]).cpu() if into is None else into[~named]
    assert (got.cpu()[~named] == rest).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocab,n", [(1, 1, 1), (1, 50, 16), (5, 3, 7), (77, 1000, 768), (64, 500, 4096),
                                           (300, 20, 1001), (1000, 7, 3), (33, 100, 16384), (2, 9, 20011)])
def test_lookup(count, vocab, n, dtype):
    dev = _dev()
    g = torch.Generator().manual_seed(count + n)
    table = torch.randn(vocab, n, generator=g).to(dtype)
    for index, kind, scale in ((torch.int64, "past", 1.0), (torch.int32, "past", 0.3), (torch.int64, "zipf", -64)):
        print(f"lookup {count} of {vocab} x {n} {dtype} {index} {kind}", flush=True)
        tokens = make_tokens(kind, count, vocab, seed=n, dtype=index)
        got = CG.run_embedding(tokens.to(dev), table.to(dev), scale=scale).cpu()
        want = want_lookup(tokens, table, scale)
        assert got.dtype == dtype and got.shape == want.shape
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocab,n,kind", [
    (1, 1, 1, "one"), (1, 9, 8, "distinct"), (2, 9, 64, "one"), (15, 40, 7, "zipf"), (16, 40, 8, "one"),
    (17, 40, 9, "one"), (64, 1000, 768, "distinct"), (100, 3, 3, "zipf"), (500, 1000, 129, "few"),
    (1023, 511, 96, "past"), (1024, 512, 32, "one"), (1025, 513, 40, "one"), (1025, 2000, 33, "past"),
    (4096, 100000, 24, "zipf"), (4097, 300000, 17, "zipf"), (4097, 5, 130, "few"), (9000, 9000, 16, "distinct"),
    (12288, 70, 64, "past"), (12289, 31, 5, "one"), (777, 50, 2048, "few"), (64, 10, 16384, "few"), (50, 20, 20011, "zipf"),
    (300, 10, 64, "none"), (512, 90, 40, "zipf"), (511, 5000, 96, "past"), (513, 90, 40, "zipf"), (40000, 50000, 8, "one"), (300000, 131072, 3, "few"), (300000, 2000, 2, "zipf"), (256, 300, 48, "zipf"), (255, 7, 1000, "past"), (256, 3000, 9, "one"), (257, 40, 520, "few"),
    (200, 5000, 2048, "zipf"), (30, 70000, 24, "distinct"), (100, 2000, 513, "none"), (3, 1000, 5000, "past"), (20000, 32003, 101, "zipf"), (70000, 100, 8, "zipf")])
def test_gradient(count, vocab, n, kind, dtype):
    dev = _dev()
    print(f"gradient {count} of {vocab} x {n} {kind} {dtype}", flush=True)
    g = torch.Generator().manual_seed(count)
    index = torch.int32 if count % 2 else torch.int64
    tokens = make_tokens(kind, count, vocab, seed=vocab, dtype=index)
    grad = torch.randn(count, n, generator=g).to(dtype)
    check_gradient(grad, tokens, vocab, 1.0, dev)
    for into in {dtype, torch.float32}:
        check_gradient(grad, tokens, vocab, 2.5, dev, torch.randn(vocab, n, generator=g).to(into))


def test_strides_and_alignments():
    dev = _dev()
    g = torch.Generator().manual_seed(1)
    vocab, n, b, s = 97, 72, 5, 30
    table, grad = torch.randn(vocab, n, generator=g).half(), torch.randn(b, s, n, generator=g).half()
    tokens = make_tokens("past", b * s, vocab, 3).view(b, s)
    want, want_grad = want_lookup(tokens, table, 1.0), CG.run_embedding_backward(grad.to(dev), tokens.to(dev), vocab)
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(9.0), b.cpu().nan_to_num(9.0))  # noqa: E731
    wide, wide_grad = torch.zeros(vocab, n + 50).half().to(dev), torch.zeros(b, s, n + 50).half().to(dev)
    for offset in (0, 8, 1, 3):
        print(f"embedding offset {offset}", flush=True)
        wide[:, offset:offset + n], wide_grad[..., offset:offset + n] = table.to(dev), grad.to(dev)
        i = tokens.to(dev).repeat_interleave(2, dim=1)[:, ::2]             # two elements apart
        assert same(CG.run_embedding(i, wide[:, offset:offset + n]), want)
        assert torch.equal(CG.run_embedding_backward(wide_grad[..., offset:offset + n], i, vocab), want_grad)
        into = torch.ones(vocab, n + 50, device=dev)
        part = into[:, offset:offset + n]
        CG.run_embedding_backward(grad.to(dev), i, vocab, into=part)
        ref = CG.run_embedding_backward(grad.to(dev), i, vocab, into=torch.ones(vocab, n, device=dev))
        assert torch.equal(part, ref)
        assert (into[:, :offset] == 1).all() and (into[:, offset + n:] == 1).all()
    for apart in (16, 17):                           # read in place, and copied
        i = tokens.to(dev).flatten().repeat_interleave(apart)[::apart]
        for _ in range(2):
            assert torch.equal(CG.run_embedding_backward(grad.to(dev).flatten(0, 1), i, vocab), want_grad)
        many = make_tokens("past", 5000, vocab, 3).to(dev)
        rows = torch.randn(5000, 16, device=dev)
        assert torch.equal(CG.run_embedding_backward(rows, many.repeat_interleave(apart)[::apart], vocab),
                           CG.run_embedding_backward(rows, many, vocab))
    # other orders: a table by columns, tokens by columns, a gradient of one row for all tokens
    assert same(CG.run_embedding(tokens.to(dev).T.contiguous().T, table.to(dev).T.contiguous().T), want)
    row = grad[:1, :1].to(dev).expand(b, s, n)
    assert torch.equal(CG.run_embedding_backward(row, tokens.to(dev), vocab),
                       CG.run_embedding_backward(row.contiguous(), tokens.to(dev), vocab))
    assert torch.equal(CG.run_embedding_backward(grad.to(dev).transpose(0, 1).contiguous().transpose(0, 1),
                                                 tokens.to(dev), vocab), want_grad)


def test_no_tokens_and_one():
    dev = _dev()
    table = torch.randn(5, 12, device=dev)
    none = torch.zeros(0, 3, dtype=torch.int64, device=dev)
    assert CG.run_embedding(none, table).shape == (0, 3, 12)
    grad = CG.run_embedding_backward(torch.zeros(0, 3, 12, device=dev), none, 5)
    assert grad.shape == (5, 12) and not grad.any()
    assert CG.run_embedding_backward(torch.zeros(0, 3, 12, device=dev), none, 5, into=table) is table
    one = torch.tensor(3, device=dev)
    assert torch.equal(CG.run_embedding(one, table), table[3])
    assert torch.equal(CG.run_embedding_backward(table[0], one, 5)[3], table[0])


def test_non_finite_rows_stay_apart():
    dev = _dev()
    g = torch.Generator().manual_seed(2)
    tokens = make_tokens("zipf", 600, 40, 5)
    grad = torch.randn(600, 96, generator=g).bfloat16()
    clean = CG.run_embedding_backward(grad.to(dev), tokens.to(dev), 40)
    bad = grad.clone()
    at = int((tokens == 7).nonzero()[0])
    bad[at, 5], bad[tokens < 0] = math.inf, math.nan
    got = CG.run_embedding_backward(bad.to(dev), tokens.to(dev), 40)
    assert got[7, 5] == math.inf
    got[7, 5] = clean[7, 5]
    assert torch.equal(got, clean)
    into = torch.full((40, 96), math.nan, device=dev)
    CG.run_embedding_backward(grad.to(dev), torch.full((600,), 3, device=dev), 40, into=into)
    assert into.isnan().all()


def test_gradient_matches_differences():
    dev = _dev()
    g = torch.Generator().manual_seed(4)
    table = torch.randn(6, 10, generator=g).to(dev).requires_grad_()
    tokens = torch.tensor([[0, 3, 3], [5, -1, 0]], device=dev)
    weights = torch.randn(2, 3, 10, generator=g).to(dev)
    op = CG.as_embedding_op(1.5)
    grad = torch.autograd.grad((op(tokens, table) * weights).sum(), table)[0]
    for v, j in ((0, 0), (3, 9), (5, 4), (1, 1)):
        values = []
        for sign in (1, -1):
            t = table.detach().double().cpu()
            t[v, j] += sign * 1e-3
            rows = torch.where(tokens.cpu().unsqueeze(-1) >= 0, 1.5 * t[tokens.cpu().clamp(min=0)], 0.0)
            values.append((rows * weights.cpu().double()).sum().item())
        # (linear: the differences are off by 64-bit roundings alone)
        assert abs(grad[v, j].item() - (values[0] - values[1]) / 2e-3) <= 1e-5


def test_refused_calls_on_the_device():
    dev = _dev()
    grad, tokens = torch.zeros(4, 8, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="device"):
        CG.run_embedding(tokens.cpu(), grad)
    with pytest.raises(ValueError, match="overlap"):
        CG.run_embedding_backward(grad, tokens, 4, into=grad)
    with pytest.raises(ValueError, match="grad"):
        CG.run_embedding_backward(grad, tokens, 4, into=torch.zeros(4, 8, device=dev, requires_grad=True))
    into = torch.zeros(4, 8, device=dev)
    CG.run_embedding_backward(grad, tokens, 4, into=into)
    with pytest.raises(ValueError, match="grad"):    # of a layout seen before
        CG.run_embedding_backward(grad, tokens, 4, into=into.clone().requires_grad_())


def test_written_tensors_are_known_to_autograd():
    dev = _dev()
    grad, tokens = torch.ones(4, 8, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    for _ in range(2):
        into = torch.zeros(4, 8, device=dev)
        before = into._version
        CG.run_embedding_backward(grad, tokens, 4, into=into)
        assert into._version == before + 1 and (into[0] == 4).all()


def test_captured_replays_and_streams():
    dev = _dev()
    vocab, n, count = 5000, 256, 6000
    g = torch.Generator().manual_seed(8)
    sets = [(make_tokens("zipf", count, vocab, s).to(dev), torch.randn(count, n, generator=g).bfloat16().to(dev),
             torch.randn(vocab, n, generator=g).bfloat16().to(dev)) for s in range(3)]

    def step(tokens, grad, table):
        into = table.float()
        return (CG.run_embedding(tokens, table, scale=16.0), CG.run_embedding_backward(grad, tokens, vocab),
                CG.run_embedding_backward(grad, tokens, vocab, into=into))

    want = [[t.clone() for t in step(*s)] for s in sets]
    torch.cuda.synchronize()
    static = [[t.clone() for t in sets[0]] for _ in range(2)]
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
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
        eager = step(*sets[2])
        for out, p in zip(outs, picks):
            assert all(torch.equal(a, b) for a, b in zip(out, want[p]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[2]))


def test_registered_operator_keeps_its_contracts():
    dev = _dev()
    table = torch.randn(40, 24, device=dev).requires_grad_()
    tokens = make_tokens("zipf", 12, 40, 1).view(3, 4).to(dev)
    print("contracts of the embedding", flush=True)
    torch.library.opcheck(CG.as_embedding_op(3.0), (tokens, table),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor",
                                      "test_aot_dispatch_static"))


@pytest.mark.parametrize("rows,n", [(1 << 20, 2056), (70000, 32768)])
def test_tables_past_32_bits_of_offsets(rows, n):
    dev = _dev()
    print(f"table {rows} x {n}", flush=True)
    table = torch.zeros(rows, n, dtype=torch.bfloat16, device=dev)       # more than 2^31 elements
    tokens = torch.tensor([0, rows - 1, rows // 2, rows - 1, 5], device=dev)
    table[tokens] = torch.randn(5, n, device=dev).bfloat16()
    out = CG.run_embedding(tokens, table)
    assert torch.equal(out, table[tokens])
    grad = CG.run_embedding_backward(out, tokens, rows)
    assert torch.equal(grad[rows - 1], (out[1].float() * 2).bfloat16()) and torch.equal(grad[5], out[4])
    named = grad.view(rows, -1).any(-1).nonzero().flatten()
    assert named.tolist() == sorted({0, rows - 1, rows // 2, 5})
