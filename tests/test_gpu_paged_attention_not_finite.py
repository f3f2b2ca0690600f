"""Keys and values that are no numbers, in the paged attention: they reach the tokens that see them, a value's in its
own column, and no others.  A value leaves the other results' bits as they are without it; a key may raise the
reference value of rows beside its own, so that their weights are rounded elsewhere: 2^-16 of each weight, both
times, and the output's rounding eps / 2, both times."""

import pytest
import torch

from test_gpu_paged_attention import make, seqs
from testt_amd import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, B = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def run(q, k, v, table, lengths, cu):
    return attention.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), *seqs(table, lengths, cu)).cpu()


SHAPES = [(4, 2, 64, 3), (12, 2, 128, 5), (8, 1, 80, 4), (4, 4, 128, 24), (2, 1, 256, 20), (8, 8, 96, 9)]


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("nh,nkv,d,news", SHAPES)
def test_a_later_tokens_value(nh, nkv, d, news, what, dtype):
    """The value of the last but one new token, one column of one key head: this token and the last one have it."""
    lengths = [40, 131, 1000]
    q, k, v, table, cu = make(lengths, [news] * 3, 16, nh, nkv, d, dtype, 1)
    want = run(q, k, v, table, lengths, cu)
    at, col, h = 129, d - 3, nkv - 1
    v[table[1][at // 16], h, at % 16, col] = what
    got = run(q, k, v, table, lengths, cu)
    hit = torch.zeros(3, news, nh, d, dtype=torch.bool)
    hit[1, -2:, h * (nh // nkv):, col] = True
    hit = hit.view(got.shape)
    assert bool((got[hit].isnan() if what != what else got[hit] == what).all())
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("what", [NAN, INF, -INF])
@pytest.mark.parametrize("nh,nkv,d,news", SHAPES)
def test_a_later_tokens_key(nh, nkv, d, news, what, dtype):
    """The key of the last new token: the others are what they were."""
    lengths = [40, 131, 1000]
    q, k, v, table, cu = make(lengths, [news] * 3, 16, nh, nkv, d, dtype, 2)
    want = run(q, k, v, table, lengths, cu).view(3, news, -1)
    k[table[1][130 // 16], :, 130 % 16] = what
    got = run(q, k, v, table, lengths, cu).view(3, news, -1)
    got[1, -1] = want[1, -1] = 0
    tol = torch.finfo(dtype).eps * want.double().abs() + 4 * 2.0 ** -16 * float(v.double().nan_to_num(0).abs().max())
    assert bool(((got.double() - want.double()).abs() <= tol).all())
    assert torch.equal(got[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("length", [1, 20, 300, 5000])
def test_infinite_values_that_are_seen(length, dtype):
    """One token a sequence: an infinity stays one, of both signs a NaN, each in its column."""
    q, k, v, table, _ = make([length, length], [1, 1], 32, 6, 2, 64, dtype, 3)
    want = run(q, k, v, table, [length, length], None).view(2, 2, 3, 64)
    row = lambda t: v[table[0][t // 32], 1, t % 32]       # noqa: E731
    row(0)[7], row(length - 1)[9], row(length // 2)[11] = INF, -INF, NAN
    row(0)[13], row(length - 1)[13] = INF, -INF
    got = run(q, k, v, table, [length, length], None).view(2, 2, 3, 64)
    mine = got[0, 1]
    assert bool((mine[:, 7] == INF).all()) and bool((mine[:, 9] == -INF).all()) and bool(mine[:, 11].isnan().all())
    assert length == 1 or bool(mine[:, 13].isnan().all())
    for c in (7, 9, 11, 13):
        got[0, 1, :, c] = want[0, 1, :, c] = 0
    assert torch.equal(got, want)
