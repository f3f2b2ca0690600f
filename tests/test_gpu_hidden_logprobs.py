"""head.fused_token_logprobs: the numbers are token_logprobs's on the same fp16 head product, bit for bit,
and the hidden rows' gradient is the 64-bit logits' gradient times the weight up to fp16's roundings.

With G the logits' gradient, g the row's largest upstream gradient and T the temperature, the kernel's
fp16 logits' gradient is held at a power of two s that brings g / T to 32 or more, so an entry is off by at
most |G| 2^-11 + 2^-25 / s (the second part below fp16's normal range), 1 / s <= g / (32 T).  Roundings of
different columns are independent, uniform within those bounds: a hidden entry's error from them has the
standard deviation sqrt(sum W^2 (|G| 2^-11 + 2^-25 / s)^2 / 3), of which 8 are taken.  Added to it are the
roundings of the result (to fp16 at the scale s, and once more), the kernel's own relative error of G and
an fp32 sum of V terms, both of the sum of absolute products."""

import pytest
import torch

from oracle.logprobs import token_logprobs as reference
from testt_amd import head
from tests.test_gpu_token_logprobs import U, bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"


def data(rows, vocab, width, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    hidden = (spread * torch.randn(rows, width, generator=g)).half().to(DEV)
    weight = (0.3 * torch.randn(vocab, width, generator=g)).half().to(DEV)
    return hidden, weight, torch.randint(0, vocab, (rows,), generator=g).to(DEV), g


def chunk_logits(hidden, weight):
    return [head._head_logits(h, weight) for h in hidden.split(head.CHUNK_ROWS)]


def check_grad(got, hidden, weight, tok, ups, top_k, temperature):
    """ups: upstream gradients of logprob, entropy and top_logprobs, or None."""
    z = torch.cat(chunk_logits(hidden, weight)).cpu().double().requires_grad_(True)
    w = weight.cpu().double()
    want = reference(z, tok.cpu(), top_k, temperature)
    some = [(o, u.cpu().double()) for o, u in zip(want, ups) if u is not None]
    G, = torch.autograd.grad([o for o, _ in some], z, [u for _, u in some])
    sizes = [u.abs().reshape(len(u), -1) for _, u in some]
    largest = torch.cat(sizes, -1).amax(-1, keepdim=True)
    rel, _, x, p = bounds(z.detach(), temperature)
    total = torch.cat(sizes, -1).sum(-1, keepdim=True)
    logp = torch.where(p > 0, p.clamp(min=1e-300).log().abs(), 0)
    own = (p * total * (logp + want[1].detach()[:, None] + 2) / temperature + G.abs()) * 4 * (
        rel[:, None] + 8 * U * (1 + x.abs().clamp(max=200)))
    s = largest / (32 * temperature)                 # (at least 1 / the scale)
    off = G.abs() * 2.0 ** -11 + 2.0 ** -25 * s
    dh = G @ w
    tol = 8 * ((off ** 2 / 3) @ w ** 2).sqrt() + own @ w.abs() + \
        len(w) * U * (G.abs() @ w.abs()) + 2.0 ** -10 * 1.01 * dh.abs() + 2.0 ** -25 * (1 + s)
    bad = ~((got.cpu().double() - dh).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.any(-1).nonzero().flatten()[:8].tolist(),
                           float(((got.cpu().double() - dh).abs() / tol).max()))


@pytest.mark.parametrize("rows", [3, 2500])
def test_values_and_gradients(rows):
    """Each output's gradient by itself and all together, over chunks; ignored and unknown tokens."""
    print(f"hidden rows {rows}", flush=True)
    hidden, weight, tok, g = data(rows, 1016, 64, rows)
    tok[0] = -100
    if rows > 3:
        tok[2047:2050] = torch.tensor([-100, 1016, -7], device=DEV)
    k, t = 4, 0.9
    leaf = hidden.clone().requires_grad_(True)
    got = head.fused_token_logprobs(leaf, weight, tok, k, t)
    parts = [head.token_logprobs(z, tk, k, t) for z, tk in
             zip(chunk_logits(hidden, weight), tok.split(head.CHUNK_ROWS))]
    for a, b in zip(got, (torch.cat(o) for o in zip(*parts))):
        assert a.shape == b.shape and ((a == b) | (a.isnan() & b.isnan())).all()
    all_ups = [torch.randn(o.shape, generator=g).to(DEV) for o in got[:3]]
    known = torch.where((tok >= 0) & (tok < 1016), 1.0, 0.0)
    all_ups[0] = all_ups[0] * known                  # (an unknown token's NaN has no gradient)
    safe = torch.where(known.bool(), tok, -100)
    for keep in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        ups = [u if on else None for u, on in zip(all_ups, keep)]
        outs = [o for o, on in zip(got, keep) if on]
        grad, = torch.autograd.grad(outs, leaf, [u for u in ups if u is not None],
                                    retain_graph=True)
        check_grad(grad, hidden, weight, safe, ups, k, t)


@pytest.mark.parametrize("spread", [0.02, 1.0])      # near-uniform rows and peaked ones
@pytest.mark.parametrize("vocab", [1016, 151936])
def test_rows_with_small_gradients(vocab, spread):
    """Rows that have a small gradient beside others with a large one keep fp16's precision: an entropy
    bonus alone, or alternatives, at 1/1000 to 1/100000 of the largest row's advantage."""
    print(f"small gradients {vocab} spread {spread}", flush=True)
    hidden, weight, tok, _ = data(8, vocab, 64, vocab, spread)
    g_lp = torch.tensor([1e4, 0, 0, 0, 1e4, 0, 1.0, 0], device=DEV)
    g_ent = torch.tensor([0, 10.0, 1.0, 0.1, 0.1, 0, 0, 0], device=DEV)
    g_top = torch.zeros(8, 2, device=DEV)
    g_top[5, 1] = 0.5
    leaf = hidden.clone().requires_grad_(True)
    got = head.fused_token_logprobs(leaf, weight, tok, 2, 1.0)
    grad, = torch.autograd.grad(got[:3], leaf, [g_lp, g_ent, g_top])
    check_grad(grad, hidden, weight, tok, [g_lp, g_ent, g_top], 2, 1.0)
    assert grad[7].eq(0).all()


def test_a_row_without_finite_gradient_stays_alone():
    """An infinite or NaN upstream gradient makes its own row's gradient NaN or infinite, no other's."""
    hidden, weight, tok, _ = data(6, 1016, 64, 1)
    up = torch.tensor([1.0, float("inf"), 0.25, float("nan"), 0.0, 3.0], device=DEV)
    leaf = hidden.clone().requires_grad_(True)
    grad, = torch.autograd.grad(head.fused_token_logprobs(leaf, weight, tok).logprob, leaf, up)
    assert not grad[1].isfinite().any() and not grad[3].isfinite().any()
    rest = [0, 2, 4, 5]
    check_grad(grad[rest], hidden[rest], weight, tok[rest], [up[rest], None, None], 0, 1.0)


def test_no_rows():
    hidden = torch.zeros(0, 64, dtype=torch.float16, device=DEV).requires_grad_(True)
    weight = torch.zeros(1016, 64, dtype=torch.float16, device=DEV)
    out = head.fused_token_logprobs(hidden, weight, torch.zeros(0, dtype=torch.int64, device=DEV), 3)
    grad, = torch.autograd.grad([out.logprob.sum() + out.top_logprobs.sum()], hidden)
    assert grad.shape == (0, 64) and out.top_ids.shape == (0, 3)


@pytest.mark.parametrize("vocab,width", [(1017, 64), (1016, 36), (7, 8)])
def test_sizes_that_the_split_product_does_not_take(vocab, width):
    hidden, weight, tok, g = data(5, vocab, width, vocab)
    leaf = hidden.clone().requires_grad_(True)
    got = head.fused_token_logprobs(leaf, weight, tok, 3, 0.8)
    ups = [torch.randn(o.shape, generator=g).to(DEV) for o in got[:3]]
    grad, = torch.autograd.grad(got[:3], leaf, ups)
    check_grad(grad, hidden, weight, tok, ups, 3, 0.8)


def test_graph_replay():
    """Forward and backward captured and replayed on other rows, with eager work between."""
    hidden, weight, tok, g = data(300, 5000, 64, 9)
    ups = [torch.randn(300, generator=g).to(DEV) * 10.0 ** -(torch.arange(300, device=DEV) % 6)
           for _ in range(2)]

    def step(h):
        leaf = h.detach().requires_grad_(True)
        out = head.fused_token_logprobs(leaf, weight, tok, 4)
        grad, = torch.autograd.grad([out.logprob, out.entropy], leaf, ups)
        return [o.detach() for o in out] + [grad]

    static = hidden.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i in range(4):
        new = (hidden.float() * (1 - 0.2 * i)).half()
        static.copy_(new)
        graph.replay()
        want = step(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
