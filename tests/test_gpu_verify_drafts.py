"""Verification of drafted tokens: the tokens are whole numbers and equal the reference's, whose sums are
64-bit too (in another order: a number within 1e-13 of a border could differ; none of these does)."""

import pytest
import torch

from oracle import generate as og
from testt_amd import head

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, B, F = torch.float16, torch.bfloat16, torch.float32


def make(batch, k, vocab, dtype, seed=0, kept=1.0, noise=0.7):
    gen = torch.Generator().manual_seed(seed)
    z = 2.0 * torch.randn(batch, k + 1, vocab, generator=gen)
    zd = z[:, :k] + noise * torch.randn(batch, k, vocab, generator=gen)
    if kept < 1:
        for t in (z, zd):
            t.masked_fill_(torch.rand(t.shape, generator=gen) > kept, float("-inf"))
            t[..., 0] = 0.0
    p, q = z.softmax(-1).to(dtype), zd.softmax(-1).to(dtype)
    drafts = torch.multinomial(q.float().reshape(-1, vocab), 1, generator=gen).view(batch, k) if k else \
        torch.zeros(batch, 0, dtype=torch.int64)
    return p, q, drafts, torch.rand(batch, k + 1, generator=gen)


def check(p, drafts, u, q=None, lengths=None):
    dev = [None if t is None else t.to(DEV) for t in (p, drafts, u, q, lengths)]
    got = head.verify_drafts(*dev)
    want = og.verify_drafts(p, drafts, u, q, lengths)
    assert got.tokens.dtype == torch.int64 and got.accepted.dtype == torch.int32
    assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])
    return got


@pytest.mark.parametrize("dtype", [H, B, F])
@pytest.mark.parametrize("batch,k,vocab,kept", [
    (1, 1, 1, 1.0), (3, 2, 7, 1.0), (40, 4, 100, 1.0), (9, 5, 4096, 0.1), (8, 3, 4097, 1.0), (5, 8, 32003, 0.02),
    (2, 4, 151936, 1.0), (3, 70, 33, 1.0), (1, 130, 9, 1.0), (4, 0, 999, 1.0)])
def test_against_the_reference(batch, k, vocab, kept, dtype):
    p, q, drafts, u = make(batch, k, vocab, dtype, batch + k, kept)
    check(p, drafts, u, q)
    check(p, drafts, u)
    lengths = torch.arange(batch, dtype=torch.int32) % (k + 2) - (1 if k > 2 else 0)
    check(p, drafts, u, q, lengths)
    check(p, drafts, u, None, lengths)


def test_accepted_prefixes_of_every_length():
    """Equal distributions accept everything; a row that gives the drafted token nothing ends it there."""
    p, _, drafts, u = make(70, 66, 50, F, 3)
    q = p[:, :66].clone()
    for b in range(66):
        p[b, b].scatter_(0, drafts[b, b:b + 1], 0.0)
    got = check(p, drafts, u, q)
    assert got.accepted.tolist() == [*range(66), 66, 66, 66, 66]


def test_borders():
    """Exact fractions: u q = p is refused; a prefix sum that equals the number is passed over, so are
    weights of zero."""
    p = torch.tensor([[[0.25, 0.0, 0.25, 0.5, 0.0]] * 2])
    q = torch.tensor([[[0.5, 0.5, 0.0, 0.0, 0.0]]])
    for u0, uk, n in ((0.5, 0.0, 0), (0.5 - 2 ** -25, 0.0, 1), (0.75, 0.25, 0), (0.75, 0.5, 0), (0.0, 0.25, 1),
                      (0.0, 0.5, 1), (0.0, 0.75, 1), (0.75, 1 - 2 ** -24, 0), (0.0, 1 - 2 ** -24, 1),
                      (0.0, 1.0, 1), (0.75, 7.0, 0)):
        got = check(p, torch.tensor([[0]]), torch.tensor([[u0, uk]]), q)
        assert int(got.accepted) == n
    # the draft's distribution covers the target's: nothing is left, so the target's own row is drawn from
    for uk in (0.0, 0.3, 0.9):
        check(p, torch.tensor([[1]]), torch.tensor([[0.9, uk]]), torch.tensor([[[0.5, 0.5, 0.5, 0.5, 0.5]]]))


def test_unusable_probabilities():
    inf, nan = float("inf"), float("nan")
    p = torch.tensor([[[nan, -1.0, 0.5, inf, 0.25]] * 2])
    for x in range(-1, 6):
        for uk in (0.0, 0.5, 0.7, 0.99):
            d = torch.tensor([[x]])
            check(p, d, torch.tensor([[0.1, uk]]), torch.tensor([[[0.1, nan, 0.2, 0.1, inf]]]))
            check(p, d, torch.tensor([[0.1, uk]]))
    zero = torch.zeros(2, 2, 3000)
    got = check(zero, torch.zeros(2, 1, dtype=torch.int64), torch.rand(2, 2))
    assert bool((got.tokens == -1).all())
    # one column alone, first, last and within
    for at in (0, 1, 2999):
        z = zero.clone()
        z[..., at] = 1e-30
        got = check(z, torch.zeros(2, 1, dtype=torch.int64), torch.tensor([[0.9, 0.0], [0.9, 0.99]]))
    numbers = torch.tensor([[0.1, nan]])
    check(p, torch.tensor([[2]]), numbers)
    check(p, torch.tensor([[2]]), torch.tensor([[nan, 0.2]]))


def test_long_rows():
    """More columns than 256 parts of 4096: parts are searched in steps."""
    vocab = (1 << 20) + 4099 * 3
    gen = torch.Generator().manual_seed(4)
    p = torch.rand(1, 2, vocab, generator=gen)
    for uk in (0.0, 0.11, 0.5, 0.97, 1 - 2 ** -24):
        check(p, torch.tensor([[vocab - 1]]), torch.tensor([[0.99999, uk]]))
        check(p, torch.tensor([[5]]), torch.tensor([[0.0, uk]]), p[:, :1] * 0.5)


def test_the_distribution_is_the_targets():
    """40000 drafts of a skewed draft over 6 tokens: each token's count within 6 standard deviations."""
    n = 8192
    gen = torch.Generator().manual_seed(5)
    p = torch.tensor([0.3, 0.05, 0.2, 0.0, 0.4, 0.05])
    q = torch.tensor([0.05, 0.5, 0.1, 0.2, 0.1, 0.05])
    drafts = torch.multinomial(q, n, replacement=True, generator=gen).view(n, 1)
    got = head.verify_drafts(p.expand(n, 2, 6).contiguous().to(DEV), drafts.to(DEV),
                             torch.rand(n, 2, generator=gen).to(DEV), q.expand(n, 1, 6).contiguous().to(DEV))
    count = torch.bincount(got.tokens[:, 0].cpu(), minlength=6).double()
    assert bool(((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all())


def test_views_and_replays():
    p, q, drafts, u = (t.to(DEV) for t in make(6, 3, 700, F, 6))
    a = head.verify_drafts(p, drafts, u, q)
    wide = torch.zeros(6, 4, 704, device=DEV)
    wide[..., :700] = p
    b = head.verify_drafts(wide[..., :700], drafts.t().contiguous().t(), u, q)
    assert torch.equal(a.tokens, b.tokens)
    lengths = torch.full((6,), 3, dtype=torch.int32, device=DEV)
    head.verify_drafts(p, drafts, u, q, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = head.verify_drafts(p, drafts, u, q, lengths)
    for i in range(4):
        u.copy_(torch.rand(6, 4, generator=torch.Generator().manual_seed(i)))
        lengths.copy_(torch.arange(6, dtype=torch.int32) % 4)
        graph.replay()
        torch.cuda.synchronize()
        now = head.verify_drafts(p, drafts, u, q, lengths)
        assert torch.equal(out.tokens, now.tokens) and torch.equal(out.accepted, now.accepted)


def test_refusals():
    p, q, drafts, u = (t.to(DEV) for t in make(2, 3, 50, F, 7))
    lengths = torch.ones(2, dtype=torch.int32, device=DEV)
    for error, args in [
            (TypeError, (p.double(), drafts, u, q.double())), (ValueError, (p[0], drafts, u)),
            (TypeError, (p, drafts.int(), u)), (ValueError, (p, drafts[:, :2], u)), (TypeError, (p, drafts, u.half())),
            (ValueError, (p, drafts, u[:, :3])), (TypeError, (p, drafts, u, q.half())),
            (ValueError, (p, drafts, u, q[..., :40])), (ValueError, (p, drafts.cpu(), u)),
            (TypeError, (p, drafts, u, q, lengths.long())), (ValueError, (p, drafts, u, q, lengths[:1])),
            (TypeError, (p, None, u)), (ValueError, (p[..., :0], drafts, u))]:
        with pytest.raises(error):
            head.verify_drafts(*args)
    with pytest.raises(RuntimeError, match="no backward for target_probs"):
        head.verify_drafts(p.clone().requires_grad_(True), drafts, u)
    none = head.verify_drafts(p[:0], drafts[:0], u[:0])
    assert none.tokens.shape == (0, 4) and none.accepted.shape == (0,)
