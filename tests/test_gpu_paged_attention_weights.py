"""The weights of the paged attention hold more bits than the cache's type: they meet the values as two numbers of
it, a rounded one and what is left of it.

Scores are exact here (one element of each query is not zero, keys hold sixteenths, scale 1), so a weight is off by
its exponent's roundings alone: scores up to 4, times log2(e), less the reference: 3 * 6 * 2^-24 in the exponent
and 2^-22 of the exponential, top and bottom, under 2^-18 together.  A weight's two numbers: 2^-16 of it in
bf16, 2^-22 in fp16 and 2^-25 absolute beside a largest weight of at least 1; sums over n keys n 2^-24; the output's
rounding eps / 2 of it, and 2^-25 for an fp16 one below 2^-14."""

import pytest
import torch

from oracle import generate as og
from testt_amd import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, B = torch.float16, torch.bfloat16
I32 = torch.int32


def exact_scores(lengths, news, page, nh, nkv, d, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need), generator=gen).tolist()
    table = [[order.pop() if i < n else -1 for i in range(max(need))] for n in need]
    k = torch.zeros(sum(need), nkv, page, d)
    k[..., 5] = torch.randint(-64, 65, k.shape[:3], generator=gen) / 16
    v = torch.randn(k.shape, generator=gen)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    q = torch.zeros(cu[-1], nh, d)
    q[..., 5] = torch.randint(0, 2, q.shape[:2], generator=gen) * 2 - 1
    return q.view(cu[-1], -1).to(dtype), k.to(dtype), v.to(dtype), table, cu


def run(q, k, v, table, lengths, cu, scale=1.0):
    dev = lambda x: torch.tensor(x, dtype=I32, device=DEV)        # noqa: E731
    return attention.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), dev(table), dev(lengths), dev(cu), scale)


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("lengths,news,page,nh,nkv,d", [
    ([96, 33], [1, 1], 16, 4, 2, 64), ([200], [1], 24, 6, 1, 96), ([130, 260], [1, 1], 32, 12, 2, 128),
    ([100], [1], 16, 2, 1, 256), ([1500, 7], [1, 1], 64, 4, 4, 128), ([90, 300], [9, 7], 16, 8, 2, 128),
    ([140], [12], 16, 4, 2, 64), ([160], [40], 32, 2, 1, 96), ([120], [20], 16, 2, 1, 256)])
def test_weights_hold_more_bits_than_the_cache(lengths, news, page, nh, nkv, d, dtype):
    q, k, v, table, cu = exact_scores(lengths, news, page, nh, nkv, d, dtype, d + len(lengths))
    got = run(q, k, v, table, lengths, cu).cpu().double()
    want, weight = og.paged_attention(q, k, v, table, lengths, cu, 1.0)
    n, eps = max(lengths), torch.finfo(dtype).eps
    tol = (2.0 ** -18 + (2.0 ** -16 if dtype == B else 2.0 ** -22) + n * 2.0 ** -24) * weight + eps / 2 * want.abs()
    if dtype == H:
        tol = tol + n * 2.0 ** -25 * float(v.double().abs().max()) + 2.0 ** -25
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("news", [1, 3])
@pytest.mark.parametrize("score", [-10.0, -14.0, -17.625])
@pytest.mark.parametrize("top", [0, 8190])
def test_many_small_weights_beside_a_large_one(top, score, news, dtype):
    """One key's weight is 1 and its value 0; thousands weigh e^score and have values of 1.  600 sequences of the
    same pages, so that a workgroup takes many chunks of one.  The exponent is at most 26: its roundings change a
    weight by 2^-17; 600 additions of a lane, 2^-14; an fp16 weight's absolute error is 2^-38 of the largest."""
    n, d, page, batch, nh = 8192, 16, 256, 600, 16
    k, v = torch.zeros(2, n // page, 1, page, d)
    k[..., 0], v[..., 1] = score, 1.0
    k[top // page, 0, top % page] = 0
    v[top // page, 0, top % page] = 0
    q = torch.zeros(batch * news, nh, d)
    q[..., 0] = 1
    got = run(q.view(batch * news, -1).to(dtype), k.to(dtype), v.to(dtype), [list(range(n // page))] * batch,
              [n] * batch, list(range(0, batch * news + 1, news)))
    got = got.cpu().double().view(batch, news, nh, d)
    p = torch.tensor(score, dtype=torch.float64).exp()
    for i in range(news):
        m = n - news + i                     # keys beside the large one, if the token sees it
        want = m * p / (1 + m * p) if top <= m else torch.ones((), dtype=torch.float64)
        tol = (2.0 ** -14 + 2.0 ** -17 + 2.0 ** -16 + torch.finfo(dtype).eps / 2) * want + n * 2.0 ** -38
        assert bool(((got[:, i, :, 1] - want).abs() <= tol).all()), float((got[:, i, :, 1] / want - 1).abs().max())
    assert not bool(got[..., 2:].any())


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("news", [1, 20])
@pytest.mark.parametrize("q_at", [2.0 ** e for e in (-2, 4, 8, 11, 12, 13, 14)] + [2.0 ** 15])
@pytest.mark.parametrize("order", ["rising", "falling", "flat", "below zero"])
def test_scores_of_any_size(order, q_at, news, dtype):
    """Scores from hundreds to 2 * 10^9, steps of 512 q_at apart, so that the largest ones a token sees have all the
    weight (its neighbours' is below 2^-180); equal ones share it.  Their values are one of 1 and 2: exact."""
    n, d, page = 300, 32, 16
    k, v = torch.zeros(2, 19, 1, page, d)
    t = torch.arange(n)
    step = {"rising": t // 3, "falling": (n - 1 - t) // 3, "flat": torch.full((n,), 50), "below zero": t // 3 - 101}[order]
    k[t // page, 0, t % page, 3] = 512.0 * step
    v[t // page, 0, t % page, 7] = 1.0 + t % 3 // 2
    q = torch.zeros(news, 2, d)
    q[..., 3] = q_at
    got = run(q.view(news, -1).to(dtype), k.to(dtype), v.to(dtype), [list(range(19))], [n], [0, news])
    for i in range(news):
        seen = n - news + i + 1
        best = (step[:seen] == step[:seen].max()).nonzero()[:, 0]
        want = float((1.0 + best % 3 // 2).double().mean())
        far = (got.cpu().view(news, 2, d)[i, :, 7].double() - want).abs().max()
        assert float(far) <= want * (torch.finfo(dtype).eps / 2 + 2.0 ** -15), (i, float(far))
