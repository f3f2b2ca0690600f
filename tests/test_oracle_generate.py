"""The 64-bit references of the generating program's operators, against what defines them: turns that
depend on distances alone, a cache that is a plain sequence cut up, tokens distributed as the target."""

import math

import pytest
import torch

from oracle import generate as g


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotated_products_depend_on_the_distance(interleaved):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 1, 12, generator=gen, dtype=torch.float64)
    cos, sin = g.rotary_tables(64, 8, 1e4)
    def product(a, b):
        y = g.rotary(x, cos, sin, torch.tensor([a, b]), interleaved)
        return float((y[0] * y[1]).sum())
    assert abs(product(3, 10) - product(40, 47)) < 1e-12
    assert abs(product(3, 10) - product(3, 11)) > 1e-6


def test_rotary_gradient_by_differences():
    gen = torch.Generator().manual_seed(2)
    cos, sin = g.rotary_tables(9, 6, 100.0)
    x = torch.randn(4, 2, 8, generator=gen, dtype=torch.float64).requires_grad_(True)
    for interleaved in (False, True):
        assert torch.autograd.gradcheck(
            lambda t: g.rotary(t, cos, sin, torch.tensor([0, 8, 3, 9]), interleaved), (x,))


def test_scaled_frequencies():
    """linear: positions divided; dynamic: the lowest frequency divided by the growth; yarn: the first pairs as
    they were, the last ones divided by the factor."""
    dim, theta = 64, 1e4
    plain, _ = g.frequencies(dim, theta)
    a, _ = g.rotary_tables(40, dim, theta, {"rope_type": "linear", "factor": 4.0})
    b, _ = g.rotary_tables(10, dim, theta)
    assert torch.allclose(a[::4], b)
    dyn, _ = g.frequencies(dim, theta, {"rope_type": "dynamic", "factor": 2.0,
                                        "original_max_position_embeddings": 128}, 512)
    assert dyn[0] == 1.0 and abs(plain[-1] / dyn[-1] - (2.0 * 4 - 1)) < 1e-9
    same, _ = g.frequencies(dim, theta, {"rope_type": "dynamic", "factor": 2.0,
                                         "original_max_position_embeddings": 512}, 512)
    assert same == plain
    yarn, gain = g.frequencies(dim, theta, {"rope_type": "yarn", "factor": 8.0,
                                            "original_max_position_embeddings": 4096}, 512)
    assert yarn[:4] == plain[:4] and abs(yarn[-1] * 8 / plain[-1] - 1) < 1e-12
    assert gain == 0.1 * math.log(8.0) + 1


def test_the_paged_cache_is_a_sequence_cut_up():
    gen = torch.Generator().manual_seed(3)
    d, nh, n_kv, page, n = 16, 4, 2, 3, 8
    qkv = torch.randn(n, (nh + 2 * n_kv) * d, generator=gen, dtype=torch.float64)
    cos, sin = g.rotary_tables(32, d)
    pages = torch.full((5, n_kv, page, d), float("nan"), dtype=torch.float64)
    table = [[4, 0, 2]]
    q, k, v = g.rope_append(qkv, None, None, cos, sin, pages, pages.clone(), table, [n], [0, n])
    out, _ = g.paged_attention(q, k, v, table, [n], [0, n])
    x = qkv.view(n, -1, d)
    rot = g.rotary(x[:, :nh + n_kv], cos, sin, torch.arange(n))
    qh, kh, vh = rot[:, :nh], rot[:, nh:], x[:, nh + n_kv:]
    z = torch.einsum("ihd,jhd->hij", qh, kh.repeat_interleave(2, 1)) / d ** 0.5
    z = z.masked_fill(torch.ones(n, n).triu(1).bool(), float("-inf"))
    want = torch.einsum("hij,jhd->ihd", z.softmax(-1), vh.repeat_interleave(2, 1)).reshape(n, -1)
    assert torch.allclose(out, want, atol=1e-12)
    # the last token alone, as a decoding step sees it
    last, _ = g.paged_attention(q[-1:], k, v, table, [n])
    assert torch.allclose(last, want[-1:], atol=1e-12)


def test_verified_tokens_have_the_targets_distribution():
    """Over a grid of both numbers, weighted by the draft's probabilities, the first token's distribution is
    the target's, to the grid's spacing."""
    p = torch.tensor([[[0.5, 0.2, 0.3], [0.1, 0.1, 0.8]]], dtype=torch.float64)
    q = torch.tensor([[[0.1, 0.6, 0.3]]], dtype=torch.float64)
    n = 60
    grid = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    got = torch.zeros(3, dtype=torch.float64)
    for x in range(3):
        for a in grid:
            for b in grid:
                tokens, _ = g.verify_drafts(p, torch.tensor([[x]]), torch.tensor([[a, b]]), q)
                got[int(tokens[0, 0])] += q[0, 0, x] / n ** 2
    assert float((got - p[0, 0]).abs().max()) < 2 / n


def test_chosen_drafts_keep_the_targets_distribution():
    p = torch.tensor([[[0.5, 0.2, 0.3], [0.1, 0.1, 0.8]]], dtype=torch.float64)
    n = 60
    grid = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    for x in range(3):
        got = torch.zeros(3, dtype=torch.float64)
        for a in grid:
            for b in grid:
                tokens, _ = g.verify_drafts(p, torch.tensor([[x]]), torch.tensor([[a, b]]))
                got[int(tokens[0, 0])] += 1 / n ** 2
        assert float((got - p[0, 0]).abs().max()) < 2 / n
