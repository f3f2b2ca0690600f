"""The rotation, its gradient and the append at the sizes where a wavefront takes two or three groups of heads: groups
in threes, even and odd in number, the last one full or not; fp32 heads over 256.  Tolerances as in
test_gpu_rotary.py and test_gpu_rope_append.py."""

import pytest
import torch

from oracle import generate as og
from test_gpu_rope_append import close, dev, dev_seqs
from test_gpu_rotary import check
from testt_amd import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, B, F = torch.float16, torch.bfloat16, torch.float32


def tokens_of(groups):
    """So many that a wavefront's items are over 4096."""
    return -(-4096 // groups) + 3


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,heads,groups,d,r", [
    # pairs of runs that are whole lines: eight heads of 128, four of 256 a group
    (H, 20, 3, 128, 128), (B, 13, 2, 128, 128), (H, 40, 5, 128, 128), (B, 24, 3, 256, 128), (H, 30, 8, 256, 256),
    # runs in memory order: eight heads of 64, five of 96, six of 80
    (H, 12, 2, 64, 64), (B, 19, 3, 64, 32), (B, 11, 3, 96, 24), (H, 7, 2, 80, 80),
    # fp32: four heads of 64 in order, two of 512 and one of 1024 in pairs of runs
    (F, 9, 3, 64, 64), (F, 5, 3, 512, 512), (F, 7, 4, 512, 256), (F, 9, 5, 512, 512), (F, 3, 2, 272, 16),
    (F, 2, 2, 1024, 1024), (H, 3, 2, 528, 528)])
def test_rotary_and_gradient(dtype, heads, groups, d, r, interleaved):
    tokens = tokens_of(groups)
    gen = torch.Generator().manual_seed(heads + d)
    cos, sin = (t.float().to(DEV) for t in og.rotary_tables(90, r))
    x = torch.randn(tokens, heads, d, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    dy = torch.randn(tokens, heads, d, generator=gen).to(dtype).to(DEV)
    pos = torch.randint(-2, 92, (tokens,), generator=gen).to(DEV)
    y = rope.rotary(x, cos, sin, pos, interleaved)
    check(y, x.detach(), cos, sin, pos, interleaved, dtype)
    dx, = torch.autograd.grad(y, x, dy)
    check(dx, dy, cos, -sin, pos, interleaved, dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,lora", [(H, H), (B, F), (H, F), (B, None)])
@pytest.mark.parametrize("nh,nkv,d,r,groups", [
    (12, 4, 128, 128, 3), (9, 2, 128, 64, 2), (32, 4, 128, 128, 5), (80, 30, 16, 16, 3), (70, 10, 16, 4, 2),
    (7, 4, 256, 256, 4), (5, 1, 240, 240, 2)])
def test_append(nh, nkv, d, r, groups, dtype, lora, interleaved):
    tokens, page = tokens_of(groups), 16
    news = [tokens // 2, 0, tokens // 3]
    news.append(tokens - sum(news) - 2)              # (two rows of no sequence)
    lengths = [news[0] + 5, 4, news[2] - 7, news[3]]
    gen = torch.Generator().manual_seed(nh + d)
    cu = [0, *torch.tensor(news).cumsum(0).tolist()]
    qkv = torch.randn(tokens, (nh + 2 * nkv) * d, generator=gen).to(dtype)
    lq = lv = None
    if lora is not None:
        lq = (0.1 * torch.randn(tokens, nh * d, generator=gen)).to(lora)
        lv = (0.1 * torch.randn(tokens, nkv * d, generator=gen)).to(lora)
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + 1, generator=gen).tolist()
    table = [[order.pop() if i < n else -1 for i in range(max(need))] for n in need]
    table[0][3], table[2][1] = -1, 1 << 20           # (tokens without a page)
    cos, sin = (t.float() for t in og.rotary_tables(news[0], r))      # (the last five are beyond the tables)
    pages = torch.full((2, sum(need) + 1, nkv, page, d), 7.0).to(dtype)
    k, v = pages.to(DEV)
    q = rope.rope_append(*dev(qkv, lq, lv, cos, sin), k, v, *dev_seqs(table, lengths, cu), interleaved)
    want = og.rope_append(qkv, lq, lv, cos, sin, *pages, table, lengths, cu, interleaved)
    size = 3 * float(qkv.float().abs().max()) + 3
    for got, ref in zip((q, k, v), want):
        close(got, ref, dtype, size)
    assert bool((q == 0).all(1).any())
