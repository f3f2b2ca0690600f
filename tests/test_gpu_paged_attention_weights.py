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
