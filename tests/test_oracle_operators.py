"""The 64-bit references of token_logprobs, qk_norm_rope and dropout: against the generator's published
outputs and against finite differences."""

import pytest
import torch

from oracle.dropout import keep_mask, philox4x32
from oracle.logprobs import token_logprobs
from oracle.qk_norm import qk_norm_rope

# Known-answer vectors of Philox4x32-10 published with the paper's reference implementation.
KAT = [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
]


@pytest.mark.parametrize("counter,key,words", KAT)
def test_philox_known_answers(counter, key, words):
    assert tuple(philox4x32(counter, key)) == words


def test_keep_share():
    """Of n draws about (1 - p) n are kept: within 6 standard deviations."""
    n, p = 64 * 200, 0.3
    kept = int(keep_mask(range(64), 200, p, 1234567890123, 5).sum())
    assert abs(kept - (1 - p) * n) < 6 * (n * p * (1 - p)) ** 0.5


@pytest.mark.parametrize("temperature", [1.0, 0.5])
def test_logprobs_gradient_by_differences(temperature):
    g = torch.Generator().manual_seed(3)
    z = torch.randn(3, 11, generator=g, dtype=torch.float64)
    z[1, 4:9] = float("-inf")
    tok = torch.tensor([4, 2, -100])
    free = torch.isfinite(z)

    def f(values):
        out = token_logprobs(z.masked_scatter(free, values), tok, 3, temperature)
        return out[0], out[1], out[2]

    assert torch.autograd.gradcheck(f, (z[free].clone().requires_grad_(True),))


def test_qk_norm_gradient_by_differences():
    g = torch.Generator().manual_seed(4)
    m, nh, nkv, d, seq = 4, 2, 1, 16, 5
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)
    cos, sin = rnd(seq, d).detach(), rnd(seq, d).detach()
    pos = torch.tensor([0, 3, 7, 99])
    f = lambda qkv, lq, lv, wq, wk: qk_norm_rope(qkv, lq, lv, wq, wk, cos, sin, pos, 2, seq, nh,
                                                 nkv, d, 1e-3)
    assert torch.autograd.gradcheck(f, (rnd(m, (nh + 2 * nkv) * d), rnd(m, nh * d),
                                        rnd(m, nkv * d), rnd(d), rnd(d)))
