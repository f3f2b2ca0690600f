"""head.token_logprobs where the logits are large beside the temperature: masks of -1e9 and beyond, rows
far from zero, temperatures down to 1e-20; values, alternatives and gradients against 64 bits.

The tolerances are test_gpu_token_logprobs's (none of them grows with the row's distance from zero: all is
taken relative to its maximum).  The temperature is an fp32 number, and the upstream gradients are
proportional to it, so that the logits' gradients stay in the type's range.  One term is added to them: the
hardware's base-2 exponential gives 0 for a result below fp32's normal range, so a probability is off by
2^-126 at most and a gradient by that times the probability's factor in it."""

import math

import pytest
import torch

from oracle.logprobs import token_logprobs as reference
from testt_amd import head
from tests.test_gpu_token_logprobs import DEV, U, bounds, check, logits_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def compare(z, tok, top_k, temperature, copies):
    """`copies` of the rows z against the reference on z."""
    temperature = float(torch.tensor(temperature))
    rows, vocab = z.shape
    leaf = z.repeat(copies, 1).to(DEV).requires_grad_(True)
    got = head.token_logprobs(leaf, tok.repeat(copies).to(DEV), top_k, temperature)
    g = torch.Generator().manual_seed(7)
    ups = [temperature * torch.randn(*s, generator=g) for s in ((rows,), (rows,), (rows, top_k))]
    grad, = torch.autograd.grad(got[:3], leaf, [
        u.repeat(copies, *(1,) * (u.dim() - 1)).to(DEV) for u in ups])
    zd = z.double().requires_grad_(True)
    want = reference(zd, tok, top_k, temperature)
    ref, = torch.autograd.grad(want[:3], zd, [u.double() for u in ups])
    rel, e, x, p = bounds(zd.detach(), temperature)
    x = x.abs()
    tok_x = x.gather(-1, tok[:, None])[:, 0]
    top_x = x.gather(-1, want[3])
    factor = ((ups[0].abs() + ups[2].abs().sum(-1))[:, None] + ups[1].abs()[:, None] *
              (x.clamp(max=200) + 2 * want[1].detach()[:, None] + 2)) / temperature
    size = p * factor
    rel_p = rel[:, None] + 8 * U * (1 + x.clamp(max=200))
    eps = torch.finfo(z.dtype).eps
    for c in range(0, copies, max(1, copies // 3)):
        part = slice(c * rows, (c + 1) * rows)
        check(got.logprob[part], want[0], rel + 4 * U * (tok_x + 1), "logprob")
        check(got.entropy[part], want[1], (rel + 4 * U) * (2 + 2 * e), "entropy")
        check(got.top_logprobs[part], want[2], rel[:, None] + 4 * U * (top_x + 1), "top")
        assert torch.equal(got.top_ids[part].cpu(), want[3])
        check(grad[part], ref, eps / 2 * ref.abs() + (size + ref.abs()) * 4 * rel_p +
              2.0 ** -126 * factor + torch.finfo(z.dtype).smallest_normal * eps, "dlogits")


@pytest.mark.parametrize("temperature", [1e-30, 9.9e29])
@pytest.mark.parametrize("dtype", TYPES)
def test_ends_of_the_temperature_range(temperature, dtype):
    z, tok = logits_of(5, 3001, dtype, 8)
    tok = torch.where(tok < 0, 5, tok)
    z[2] = 1.25
    compare(z, tok, 4, temperature, 1)


# rows cut into parts, and enough of them to stay whole
@pytest.mark.parametrize("copies", [1, 150])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-3, 1e-6, 1e-9, 1e-12, 1e-20])
def test_small_temperatures(temperature, dtype, copies):
    print(f"temperature {temperature} {dtype} x {copies}", flush=True)
    z, tok = logits_of(8, 20011, dtype, 3)
    tok = torch.where(tok < 0, 5, tok)
    z[1] = (8 + 3 * temperature * torch.randn(20011, generator=torch.Generator().manual_seed(1))).to(dtype)
    z[2] = 4.5                                       # every column equal
    z[3] = -z[3].abs()
    compare(z, tok, 5, temperature, copies)


@pytest.mark.parametrize("copies", [1, 150])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.6, 0.05, 1e-5])
def test_rows_far_from_zero(temperature, dtype, copies):
    """Masks of -1e9 to -1e20 (fp16: its lowest value's like) on whole rows and on all but a few columns;
    rows around +-2^20 T / log2(e) and 2^24 times as much, where the largest value of a lane, a part and
    the row rise from one side of such a border to the other."""
    print(f"far rows T {temperature} {dtype} x {copies}", flush=True)
    vocab = 20011
    g = torch.Generator().manual_seed(11)
    far = [-6e4, -65504.0, -3e4] if dtype is torch.float16 else [-1e9, -1e10, -1e20]
    rows = [torch.full((vocab,), v) for v in far]
    some = torch.full((vocab,), far[1])
    some[5:4000:7] = torch.randn(571, generator=g)
    rows += [some, -rows[1], torch.where(torch.arange(vocab) % 3 == 0, far[0], far[1])]
    most = torch.finfo(dtype).max
    near = 3 * torch.randn(vocab, generator=g)
    rise = torch.linspace(-14, 14, vocab)
    for border in (2.0 ** 20, 2.0 ** 24, 2.0 ** 44):
        at = border * temperature / math.log2(math.e)
        if at * 1.01 > most:
            continue
        # (formed in fp64, so that the columns differ by the temperature's multiples where the type can)
        rows += [(s * at + temperature * d.double()) for s in (1, -1) for d in (rise, near)]
    z = torch.stack([r.double().clamp(-most, most).to(dtype) for r in rows])
    tok = torch.randint(0, vocab, (len(rows),), generator=g)
    compare(z, tok, 8, temperature, copies)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_row_of_a_large_vocabulary(dtype):
    """A row with nothing but the mask's -1e9: a uniform distribution."""
    z = torch.full((2, 151936), -1e9).to(dtype)
    z[1, ::2] = -2e9
    compare(z, torch.tensor([3, 151934]), 3, 0.6, 1)
