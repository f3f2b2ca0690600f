"""Rows of sequences whose bounds leave the rows, in the paged attention: zeros, as rows of no sequence, and the
others' as ever."""

import pytest
import torch

from test_gpu_paged_attention import check, make, seqs
from testt_amd import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def over_nan(q, *args):
    """The attention, its output over memory that held NaN."""
    stale = [torch.full(q.shape, float("nan"), dtype=q.dtype, device=DEV) for _ in range(4)]
    torch.cuda.synchronize()
    del stale
    return attention.paged_attention(q, *args)


@pytest.mark.parametrize("cu,valid", [([0, 2, 4, 99], [0, 1]), ([-3, 2, 4, 6], [1, 2]), ([-3, 2, 4, 99], [1]),
                                      ([-9, -5, 0, 6], [2]), ([0, 6, 6, 7], [0, 1]), ([7, 8, 9, 9], []),
                                      ([1, 3, 5, 1 << 30], [0, 1]), ([-(1 << 31), 1, 1, 5], [1, 2]),
                                      ([5, 4, 3, 2], []), ([6, 0, 0, 0], [])])
@pytest.mark.parametrize("lengths", [[20, 9, 300], [3000, 2500, 2000]])
def test_rows_of_impossible_bounds_are_zeros(cu, valid, lengths):
    q, k, v, table, _ = make(lengths, [2, 2, 2], 16, 4, 2, 64, torch.float16, 9)
    got = over_nan(q.to(DEV), k.to(DEV), v.to(DEV), *seqs(table, lengths, cu))
    none = torch.ones(6, dtype=torch.bool)
    for b in valid:
        rows = slice(cu[b], cu[b + 1])
        none[rows] = False
        if cu[b] < cu[b + 1]:
            check(got[rows], q[rows], k, v, [table[b]], [lengths[b]], [0, cu[b + 1] - cu[b]], torch.float16)
    assert not bool(got[none.to(DEV)].any())


@pytest.mark.parametrize("over", [1, 40, 1 << 24])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (32, 1, 128)])
def test_the_last_of_many_sequences_passes_the_rows(nh, nkv, d, over):
    lengths = [(i * 37) % 400 for i in range(90)]
    q, k, v, table, cu = make(lengths, [3] * 90, 32, nh, nkv, d, torch.float16, 3)
    got = over_nan(q.to(DEV), k.to(DEV), v.to(DEV), *seqs(table, lengths, cu[:-1] + [cu[-1] + over]))
    check(got[:267], q[:267], k, v, table[:-1], lengths[:-1], cu[:-1], torch.float16)
    assert not bool(got[267:].any())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("beyond", [1, 2, 4, 9, (1 << 31) - 1 - 64])
@pytest.mark.parametrize("news", [1, 5, 24])
def test_tokens_stand_where_the_append_puts_them_beyond_the_table(news, beyond, dtype):
    """Lengths that pass the block table: token i stands at length - news + i all the same, and sees the keys up to
    there that the table holds."""
    cap = 64
    q, k, v, table, _ = make([cap, 30], [news, news], 16, 4, 2, 64, dtype, 5)
    args = q.to(DEV), k.to(DEV), v.to(DEV)
    lengths = [cap + beyond, 30]
    got = attention.paged_attention(*args, *seqs(table, lengths, [0, news, 2 * news]))
    # each token by itself, at its place
    rows = torch.cat([q[i:i + 1] for i in range(2 * news)])
    alone = [min(max(n - news + i + 1, 0), cap) for n in lengths for i in range(news)]
    check(got, rows, k, v, [table[b] for b in (0, 1) for _ in range(news)], alone, None, dtype)
    check(got, q, k, v, table, lengths, [0, news, 2 * news], dtype)
