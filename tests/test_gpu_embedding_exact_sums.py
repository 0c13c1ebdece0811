"""The embedding's gradient where its sums are exact: every entry counts once, from its own position.

The gradients are whole numbers from -8 to 8, drawn for each position and column, and no row has 2^21 tokens or more,
so that a sum over any of a row's entries is below 2^24 and fp32 holds it, in whatever order the entries are added: the
result is the sum in 64-bit integers, to the bit.  An entry that is lost, doubled or read from another position
changes it, also among many thousands (where a rounding's allowance would hide hundreds).
"""
import pytest
import torch

import neptune_codegen as CG

pytestmark = pytest.mark.gpu
MOST_OF_A_ROW = 1 << 21


def _dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def make(kind, count, vocab, n, seed):
    """(tokens, gradient) on the CPU, both whole numbers."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda high: torch.randint(0, high, (count,), generator=g)  # noqa: E731
    if kind == "one":
        t = torch.full((count,), vocab // 2)
    elif kind == "few":
        t = rand(3) * ((vocab - 1) // 2)
    elif kind == "share":                            # one workgroup's rows (every 256th)
        t = rand(-(-vocab // 256)) * 256
    elif kind == "falling":
        t = (vocab ** torch.rand(count, generator=g, dtype=torch.float64)).long() - 1
    elif kind == "runs":                             # each row's tokens are neighbours
        t = torch.arange(count) * vocab // count
    else:
        t = rand(vocab)
    t = t.clamp(0, vocab - 1)
    if kind != "one":
        t[torch.rand(count, generator=g) < 0.05] = -1
        t[torch.rand(count, generator=g) < 0.05] = vocab
    return t, torch.randint(-8, 9, (count, n), generator=g)


def sums(tokens, grad, vocab):
    here = (tokens >= 0) & (tokens < vocab)
    at = tokens[here].long()
    assert torch.bincount(at, minlength=1).max() < MOST_OF_A_ROW
    # (64-bit floats hold these sums; bincount adds them quickly)
    return torch.stack([torch.bincount(at, weights=grad[here, c].double(), minlength=vocab)
                        for c in range(grad.shape[1])], 1).float()


def check(tokens, grad, vocab, dev, dtypes):
    want = sums(tokens.cpu(), grad, vocab)
    for dtype in dtypes:
        into = None if dtype == torch.float32 else torch.zeros(vocab, grad.shape[1], device=dev)
        got = CG.run_embedding_backward(grad.to(dtype).to(dev), tokens.to(dev), vocab, into=into)
        wrong = (got.cpu() != want).any(-1).nonzero().flatten()
        assert wrong.numel() == 0, (dtype, wrong[:8].tolist())


@pytest.mark.parametrize("kind,count,vocab,n", [
    ("one", 40000, 50000, 8), ("few", 300000, 131072, 3), ("falling", 300000, 2000, 2), ("share", 300000, 131072, 4),
    ("share", 40000, 1025, 8), ("runs", 200000, 1000, 3), ("any", 300000, 700, 5), ("one", 1200000, 3, 2),
    ("falling", 55087, 32003, 33), ("one", 512, 9, 40), ("falling", 511, 300, 7), ("one", 513, 9, 40),
    ("few", 1024, 70, 16), ("one", 1025, 1, 3), ("one", 16 * 1024 + 1, 300, 2), ("one", 16 * 1024 * 17, 300, 1)])
def test_every_entry_counts_once(kind, count, vocab, n):
    dev = _dev()
    print(f"exact sums: {count} of {vocab} x {n}, {kind}", flush=True)
    tokens, grad = make(kind, count, vocab, n, seed=count + n)
    check(tokens.int() if count % 2 else tokens, grad, vocab, dev, (torch.float32, torch.bfloat16, torch.float16))


def test_tokens_far_apart():
    dev = _dev()
    count, vocab, n = 5000003, 70001, 2
    print(f"exact sums: {count} tokens, sixteen elements apart", flush=True)
    tokens, grad = make("falling", count, vocab, n, seed=5)
    apart = torch.full((count * 16,), 7, dtype=torch.int64, device=dev)[::16]
    apart.copy_(tokens.to(dev))
    assert apart.stride() == (16,)
    check(apart, grad, vocab, dev, (torch.float32,))


def test_the_most_tokens():
    dev = _dev()
    count, vocab, n = (1 << 26) - 1, 2003, 1
    print(f"exact sums: {count} tokens", flush=True)
    tokens, grad = make("any", count, vocab, n, seed=6)
    check(tokens.int(), grad, vocab, dev, (torch.float32,))
    print("the same in 64 bits", flush=True)
    check(tokens, grad, vocab, dev, (torch.bfloat16,))
