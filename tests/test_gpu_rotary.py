"""Rotary tables and the rotation against 64 bits.

Tolerances: a table entry is rounded once from an error of 1e-9 (angles in 64 bits, series cut below
3e-14): 2^-24 of itself and 2e-9.  A rotated element is two products and a sum, each rounded to fp32
(3 * 2^-24 of |a c| + |b s|, doubled), then rounded to its type: half of its eps, and half of fp16's smallest
step 2^-24."""

import pytest
import torch

from oracle import generate as og
from testt_amd import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, B, F = torch.float16, torch.bfloat16, torch.float32


def yarn(**kw):
    return {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 256, **kw}


@pytest.mark.parametrize("seq,dim,theta,scaling", [
    (1, 2, 1e4, None), (7, 20, 1e4, None), (512, 128, 1e6, None), (300, 256, 5e5, None),
    (100, 64, 1e4, {"rope_type": "linear", "factor": 2.5}),
    (100, 64, 1e4, {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 100}),
    (101, 80, 1e4, {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 50}),
    (64, 2, 1e4, {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 50}),
    (1025, 128, 1e6, yarn()), (64, 96, 1e4, yarn(beta_fast=16.0, beta_slow=2.0)),
    (64, 32, 1e4, yarn(attention_factor=0.75)), (64, 64, 1e4, yarn(original_max_position_embeddings=4)),
    (9, 64, 1e4, {"rope_type": "default"}), (0, 64, 1e4, None)])
def test_tables(seq, dim, theta, scaling):
    got = rope.rotary_tables(seq, dim, theta, scaling, device=DEV)
    want = og.rotary_tables(seq, dim, theta, scaling)
    for a, b in zip(got, want):
        assert a.dtype == F and tuple(a.shape) == (seq, dim // 2)
        assert bool(((a.cpu().double() - b).abs() <= 2.0 ** -24 * b.abs() + 2e-9).all())


def test_tables_of_far_positions():
    """Position 2^20 and more: angles of a million radians."""
    seq = (1 << 20) + 5
    got = rope.rotary_tables(seq, 64, 1e4, device=DEV)
    want = og.rotary_tables(seq, 64, 1e4, start=seq - 9)
    for a, b in zip(got, want):
        assert bool(((a[-9:].cpu().double() - b).abs() <= 2.0 ** -24 * b.abs() + 2e-9).all())


def test_tables_of_given_frequencies():
    freq = torch.tensor([1.0, -0.25, 1e-7, 3.0], dtype=torch.float64)
    ang = torch.arange(50, dtype=torch.float64)[:, None] * freq
    for given in (freq, freq.tolist()):
        cos, sin = rope.rotary_tables(50, 8, inv_freq=given, device=DEV)
        assert bool(((cos.cpu().double() - ang.cos()).abs() <= 2.0 ** -24 + 2e-9).all())
        assert bool(((sin.cpu().double() - ang.sin()).abs() <= 2.0 ** -24 + 2e-9).all())


def test_tables_mscale():
    scaling = yarn(mscale=1.0, mscale_all_dim=0.5)
    cos, _ = rope.rotary_tables(4, 16, 1e4, scaling, device=DEV)
    import math
    gain = (0.1 * math.log(4.0) + 1) / (0.05 * math.log(4.0) + 1)
    assert abs(float(cos[0, 0]) - gain) < 1e-6


def check(got, x, cos, sin, pos, interleaved, dtype):
    want = og.rotary(x.double().cpu(), cos.cpu(), sin.cpu(), pos.cpu(), interleaved)
    ones = og.rotary(x.double().cpu().abs(), cos.cpu().abs(), -sin.cpu().abs(), pos.cpu(), interleaved)
    # (|a c| + |b s| of one element of each pair, |b c| - |a s| of the other: bounded by the pair's norms)
    far = ones.abs() + x.double().cpu().abs().amax(-1, keepdim=True) * 2
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 6 * 2.0 ** -24 * far + 2.0 ** -25
    if dtype == F:
        tol = 6 * 2.0 ** -24 * far
    assert bool(((got.detach().cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [H, B, F])
@pytest.mark.parametrize("tokens,heads,d,r", [
    (1, 1, 64, 64), (8, 12, 128, 128), (5, 3, 80, 20), (5, 3, 80, 80), (3, 7, 96, 24), (4, 2, 128, 64),
    (9, 5, 256, 256), (2, 40, 128, 32), (3, 2, 7, 4), (2, 3, 2, 2), (3, 1, 200, 150), (700, 14, 128, 128),
    (2, 3, 1040, 16)])
def test_rotary_and_gradient(tokens, heads, d, r, dtype, interleaved):
    gen = torch.Generator().manual_seed(tokens * 31 + d + r)
    cos, sin = (t.to(DEV) for t in og.rotary_tables(40, r))
    cos, sin = cos.float(), sin.float()
    x = torch.randn(tokens, heads, d, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    dy = torch.randn(tokens, heads, d, generator=gen).to(dtype).to(DEV)
    pos = torch.randint(0, 40, (tokens,), generator=gen).to(DEV)
    if tokens > 2:
        pos[1], pos[2] = -1, 40
    y = rope.rotary(x, cos, sin, pos, interleaved)
    assert y.dtype == dtype and y.is_contiguous()
    check(y, x.detach(), cos, sin, pos, interleaved, dtype)
    dx, = torch.autograd.grad(y, x, dy)
    check(dx, dy, cos, -sin, pos, interleaved, dtype)


def test_gradient_by_differences():
    """fp32: the rotation is linear, so f(x + e) - f(x - e) is exact up to its roundings."""
    gen = torch.Generator().manual_seed(5)
    cos, sin = rope.rotary_tables(16, 12, device=DEV)
    x = torch.randn(3, 2, 16, generator=gen).to(DEV).requires_grad_(True)
    w = torch.randn(3, 2, 16, generator=gen).to(DEV)
    e = torch.randn(3, 2, 16, generator=gen).to(DEV)
    pos = torch.tensor([3, 15, 0], device=DEV)
    g, = torch.autograd.grad((rope.rotary(x, cos, sin, pos, True) * w).sum(), x)
    with torch.no_grad():
        diff = ((rope.rotary(x + e, cos, sin, pos, True) - rope.rotary(x - e, cos, sin, pos, True)).double()
                * w.double()).sum() / 2
    # 96 terms of a few units, each rounded a few times
    assert abs(float((g.double() * e.double()).sum() - diff)) < 96 * 16 * 2.0 ** -22


@pytest.mark.parametrize("interleaved", [False, True])
def test_strides(interleaved):
    """Query columns of q|k|v rows, heads before tokens, tables whose columns stand twice, broadcast and
    transposed gradients, int32 positions."""
    gen = torch.Generator().manual_seed(6)
    rows = torch.randn(6, 5 * 64, generator=gen).to(H).to(DEV)
    cos, sin = (torch.cat([t, t], 1).float().to(DEV) for t in og.rotary_tables(30, 64))
    pos = torch.tensor([0, 1, 2, 7, 29, 3], device=DEV)
    q = rows[:, :3 * 64].view(6, 3, 64)
    a = rope.rotary(q, cos[:, :32], sin[:, :32], pos.int(), interleaved)
    b = rope.rotary(q.contiguous(), cos[:, :32].contiguous(), sin[:, :32].contiguous(), pos, interleaved)
    assert torch.equal(a, b)
    t = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rope.rotary(t, cos[:, :32], sin[:, :32], pos, interleaved), b)
    odd = torch.empty(6 * 3 * 64 + 1, dtype=H, device=DEV)[1:].view(6, 3, 64).copy_(q)
    assert torch.equal(rope.rotary(odd, cos[:, :32], sin[:, :32], pos, interleaved), b)
    last = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rope.rotary(last, cos[:, :32], sin[:, :32], pos, interleaved), b)
    x = q.contiguous().requires_grad_(True)
    y = rope.rotary(x, cos[:, :32], sin[:, :32], pos, interleaved)
    dx, = torch.autograd.grad(y, x, torch.ones(1, 1, 64, dtype=H, device=DEV).expand(6, 3, 64), retain_graph=True)
    dx2, = torch.autograd.grad(y, x, torch.ones(6, 3, 64, dtype=H, device=DEV), retain_graph=True)
    assert torch.equal(dx, dx2)
    g = torch.randn(6, 64, 3, generator=gen).to(H).to(DEV).transpose(1, 2)
    dx, = torch.autograd.grad(y, x, g, retain_graph=True)
    dx2, = torch.autograd.grad(y, x, g.contiguous())
    assert torch.equal(dx, dx2)


def test_bits_of_the_training_rotation():
    """A whole head by halves: the bits of rope_pack_tokens."""
    from testt_amd import workloads
    qkv, _, _, pos = workloads.rope_inputs((9, 4), 16, seed=3, device=DEV)
    cos, sin = workloads.rope_tables(16, device=DEV)
    rows, _, _, _ = rope.rope_pack_tokens(qkv, None, None, cos, sin, pos, 2, 16, 12, 2, 128)
    got = rope.rotary(qkv[:, :14 * 128].view(-1, 14, 128), cos[:, :64], sin[:, :64], pos % 16)
    assert torch.equal(got.view(-1, 14 * 128), rows[:, :14 * 128])


def test_nothing_and_no_tables():
    cos = torch.zeros(0, 8, device=DEV)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    x = torch.ones(2, 3, 16, device=DEV)
    assert not bool(rope.rotary(x, cos, cos, pos).any())
    assert rope.rotary(x[:0], cos, cos, pos[:0]).shape == (0, 3, 16)


def test_refusals():
    cos, sin = rope.rotary_tables(8, 16, device=DEV)
    x, pos = torch.zeros(2, 3, 16, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    bad = [(ValueError, (x[0], cos, sin, pos)), (TypeError, (x.double(), cos, sin, pos)),
           (ValueError, (x[:, :, :8], cos, sin, pos)), (TypeError, (x, cos.half(), sin, pos)),
           (ValueError, (x, cos, sin[:4], pos)), (ValueError, (x, cos.cpu(), sin, pos)),
           (ValueError, (x, cos, sin, pos[:1])), (ValueError, (x, cos, sin, pos.float())),
           (ValueError, (x, cos[0], sin, pos)), (TypeError, (None, cos, sin, pos))]
    for error, args in bad:
        with pytest.raises(error):
            rope.rotary(*args)
    with pytest.raises(RuntimeError, match="no backward for cos"):
        rope.rotary(x, cos.clone().requires_grad_(True), sin, pos)


def test_differentiated_twice():
    """The gradient is a rotation of the upstream gradient, so a gradient of it turns back."""
    gen = torch.Generator().manual_seed(9)
    cos, sin = rope.rotary_tables(8, 16, device=DEV)
    pos = torch.tensor([3, 7], device=DEV)
    x, w, c = (torch.randn(2, 3, 16, generator=gen).to(DEV).requires_grad_(True) for _ in range(3))
    g, = torch.autograd.grad((rope.rotary(x, cos, sin, pos, True) * w).sum(), x, create_graph=True)
    dw, = torch.autograd.grad((g * c.detach()).sum(), w, create_graph=True)
    assert torch.equal(dw, rope.rotary(c, cos, sin, pos, True))
