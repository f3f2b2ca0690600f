"""rope.qk_norm_rope and attention.norm_rope_attention against 64 bits.

Tolerances.  With u = 2^-24 a head's mean of squares is a sum of D <= 256 products over 16 lanes (16
terms a lane, 4 steps across): relative error below 32 u; the root, the division, the two products and
the rotation add 8 more roundings, so an output is within 48 u of the sum of its two terms' sizes, and
rounded once to the rows' type (eps / 2).  The gradient has the same steps and one more such mean.  A
weight's gradient sums rows * heads terms, each within 64 u, in chains of at most 4 + rows * heads / 64
additions here."""

import pytest
import torch

from oracle.qk_norm import qk_norm_rope as reference
from testt_amd import attention, rope, workloads

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24

CASES = [  # lengths, seq, nh, nkv, d, dtype, lora dtype, eps
    ((512, 152, 128, 96), 512, 12, 2, 128, torch.float16, torch.float16, 1e-6),
    ((512, 152, 128, 96), 512, 12, 2, 128, torch.float16, torch.float32, 1e-6),
    ((1,) * 8, 1, 12, 2, 128, torch.float16, None, 1e-6),       # one token per sequence
    ((700,), 4096, 32, 8, 128, torch.bfloat16, None, 1e-5),
    ((33, 0, 5), 64, 3, 1, 64, torch.float16, torch.float16, 1e-6),
    ((40,), 40, 5, 0, 96, torch.bfloat16, torch.bfloat16, 1e-6),   # idle lanes, no key heads
    ((17, 2), 20, 6, 3, 80, torch.float16, None, 1e-6),
    ((9,), 9, 2, 1, 256, torch.bfloat16, torch.float32, 1e-6),
    ((31,), 31, 7, 2, 16, torch.float16, None, 1e-6),
    ((21,), 21, 2, 2, 32, torch.bfloat16, None, 1e-6),
    ((3000, 2500), 3000, 4, 2, 240, torch.float16, None, 1e-6),
    ((), 8, 4, 2, 128, torch.float16, None, 1e-6),                 # no tokens
]


def inputs(lengths, seq, nh, nkv, d, dtype, ldt, seed=0):
    g = torch.Generator().manual_seed(seed + d + nh)
    pos = workloads.ragged_positions(lengths, seq) if lengths else torch.zeros(0, dtype=torch.int64)
    m = pos.numel()
    rnd = lambda *s: torch.randn(*s, generator=g)
    cos, sin = workloads.rope_tables(seq, d)
    return dict(qkv=rnd(m, (nh + 2 * nkv) * d).to(dtype),
                lq=rnd(m, nh * d).mul(0.1).to(ldt) if ldt else None,
                lv=rnd(m, nkv * d).mul(0.1).to(ldt) if ldt else None,
                wq=1 + 0.2 * rnd(d), wk=1 + 0.2 * rnd(d), cos=cos, sin=sin, pos=pos,
                dout=rnd(m, (nh + 2 * nkv) * d).mul(0.01).to(dtype))


NAMES = ("qkv", "lq", "lv", "wq", "wk")


def run(x, batch, seq, nh, nkv, d, eps):
    t = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    for n in NAMES:
        if t[n] is not None:
            t[n].requires_grad_(True)
    out = rope.qk_norm_rope(t["qkv"], t["lq"], t["lv"], t["wq"], t["wk"], t["cos"], t["sin"],
                            t["pos"], batch, seq, nh, nkv, d, eps)
    out.backward(t["dout"])
    return out.detach().cpu(), {n: t[n].grad.cpu() for n in NAMES if t[n] is not None}


def oracle(x, batch, seq, nh, nkv, d, eps):
    t = {k: None if v is None else (v if k == "pos" else v.double()) for k, v in x.items()}
    for n in NAMES:
        if t[n] is not None:
            t[n].requires_grad_(True)
    out = reference(t["qkv"], t["lq"], t["lv"], t["wq"], t["wk"], t["cos"], t["sin"], t["pos"],
                    batch, seq, nh, nkv, d, eps)
    out.backward(t["dout"])
    return out.detach(), {n: t[n].grad for n in NAMES if t[n] is not None}


def within(got, want, scale, dtype, what):
    half = torch.finfo(dtype).eps / 2
    tol = half * want.abs() + scale * (1 + half) + torch.finfo(dtype).smallest_normal * 2 * half
    bad = (got.double() - want).abs() > tol
    assert got.shape == want.shape and not bad.any(), (what, int(bad.sum()),
                                                       float((got.double() - want).abs().max()))


@pytest.mark.parametrize("lengths,seq,nh,nkv,d,dtype,ldt,eps", CASES)
def test_forward_and_gradients(lengths, seq, nh, nkv, d, dtype, ldt, eps):
    print(f"qk_norm_rope {lengths} seq {seq} heads {nh}/{nkv} x {d} {dtype} lora {ldt}", flush=True)
    batch = max(len(lengths), 1)
    x = inputs(lengths, seq, nh, nkv, d, dtype, ldt)
    out, grads = run(x, batch, seq, nh, nkv, d, eps)
    want, wgrads = oracle(x, batch, seq, nh, nkv, d, eps)
    m = x["pos"].numel()
    assert out.dtype == dtype
    if m == 0:
        assert out.shape == want.shape and grads["wq"].eq(0).all() and grads["wk"].eq(0).all()
        return
    # sizes of the terms: both halves of a rotated pair, then the head's norm times |w|
    def pair(t):
        t = t.abs().view(m, nh + 2 * nkv, d)
        return (t + t.roll(d // 2, -1)).reshape(m, -1)

    within(out, want, 48 * U * 2 * pair(want), dtype, "out")
    g = wgrads["qkv"].abs().view(m, nh + 2 * nkv, d)
    # a gradient is r (gw - n mean(gw n)): its terms are at most r (|gw| + |n| |gw|_2)
    r = x["qkv"].double().view(m, -1, d).add(
        0 if x["lq"] is None else torch.cat([x["lq"].double().view(m, nh, d),
                                             torch.zeros(m, 2 * nkv, d)], 1).double())
    rinv = 1 / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    gw = pair(x["dout"].double()).view(m, -1, d) * 2.0
    size = rinv * (gw + (r * rinv).abs() * gw.square().mean(-1, keepdim=True).sqrt()) + g
    within(grads["qkv"], wgrads["qkv"], (96 * U * size).reshape(m, -1), dtype, "dqkv")
    if ldt is not None:
        assert torch.equal(grads["lq"].to(dtype), grads["qkv"][:, :nh * d])
        assert torch.equal(grads["lv"].to(dtype), grads["qkv"][:, (nh + nkv) * d:])
    for n, heads in (("wq", slice(0, nh)), ("wk", slice(nh, nh + nkv))):
        terms = (gw * (r * rinv).abs())[:, heads].sum((0, 1))
        chain = 64 + m * (nh + 2 * nkv) / 64
        assert ((grads[n].double() - wgrads[n]).abs() <= U * chain * terms + 1e-12).all(), n


def test_positions_outside_the_tables():
    """Rows of zeros, no gradient, nothing added to the weights' gradients."""
    x = inputs((20, 12), 32, 12, 2, 128, torch.float16, torch.float16, 3)
    x["pos"][3], x["pos"][17], x["pos"][30] = -1, 64, 1 << 40
    out, grads = run(x, 2, 32, 12, 2, 128, 1e-6)
    want, wgrads = oracle(x, 2, 32, 12, 2, 128, 1e-6)
    for r in (3, 17, 30):
        assert out[r].eq(0).all() and grads["qkv"][r].eq(0).all()
    within(out, want, 1e-4, torch.float16, "out")
    assert ((grads["wq"] - wgrads["wq"]).abs() < 1e-3).all()


def test_zero_rows_and_large_values():
    """A head of zeros gives zeros (not NaN); fp16's largest values do not overflow the mean."""
    x = inputs((6,), 8, 2, 1, 128, torch.float16, None, 4)
    x["qkv"][2] = 0
    x["qkv"][3] = 65504.0
    out, grads = run(x, 1, 8, 2, 1, 128, 1e-6)
    want, wgrads = oracle(x, 1, 8, 2, 1, 128, 1e-6)
    assert out[2, :384].eq(0).all() and torch.isfinite(grads["qkv"]).all()
    within(out[3], want[3], 48 * U * 4 * want[3].abs().max(), torch.float16, "large")


def test_weights_of_other_types_and_frozen_weights():
    x = inputs((12,), 16, 4, 2, 128, torch.float16, None, 5)
    t = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    w16 = t["wq"].half().requires_grad_(True)
    out = rope.qk_norm_rope(t["qkv"], None, None, w16, t["wk"], t["cos"], t["sin"],
                            t["pos"].to(torch.int32), 1, 16, 4, 2, 128)
    out.backward(t["dout"])
    assert w16.grad.dtype == torch.float16 and t["wk"].grad is None
    again = rope.qk_norm_rope(t["qkv"], None, None, w16.float(), t["wk"], t["cos"], t["sin"],
                              t["pos"], 1, 16, 4, 2, 128)
    assert torch.equal(out, again)


def test_refusals():
    x = {k: None if v is None else v.to(DEV) for k, v in
         inputs((8,), 8, 4, 2, 128, torch.float16, None, 6).items()}
    args = dict(qkv=x["qkv"], lora_q=None, lora_v=None, q_weight=x["wq"], k_weight=x["wk"],
                cos=x["cos"], sin=x["sin"], pos_idx=x["pos"], batch=1, seq=8, n_heads=4, n_kv=2,
                head_dim=128)
    for change, error in ((dict(head_dim=100), ValueError), (dict(n_heads=3), ValueError),
                          (dict(qkv=x["qkv"].float()), TypeError),
                          (dict(q_weight=x["wq"][:64]), ValueError),
                          (dict(pos_idx=x["pos"][:7]), ValueError), (dict(seq=9), ValueError),
                          (dict(lora_q=x["qkv"]), ValueError), (dict(eps=-1.0), ValueError),
                          (dict(qkv=x["qkv"].t()), ValueError)):
        with pytest.raises(error):
            rope.qk_norm_rope(**{**args, **change})


def test_attention_over_normalised_rows():
    """norm_rope_attention is the varlen attention of qk_norm_rope's rows, and its gradient reaches
    qkv, the deltas and the weights: against float32 attention on the same fp16 rows (2e-3 absolute,
    as the attention's own tests), and one weight's gradient against a difference."""
    lengths, seq, nh, nkv, d = (40, 17), 64, 4, 2, 128
    x = {k: None if v is None else v.to(DEV) for k, v in
         inputs(lengths, seq, nh, nkv, d, torch.float16, torch.float16, 7).items()}
    cu = attention.cu_seqlens_of(x["pos"], 2, seq)
    leaves = [x[n].requires_grad_(True) for n in NAMES]
    call = lambda wq: attention.norm_rope_attention(x["qkv"], x["lq"], x["lv"], wq, x["wk"],
                                                    x["cos"], x["sin"], x["pos"], cu, 2, seq, nh,
                                                    nkv)
    out = call(x["wq"])
    rows = rope.qk_norm_rope(x["qkv"], x["lq"], x["lv"], x["wq"], x["wk"], x["cos"], x["sin"],
                             x["pos"], 2, seq, nh, nkv, d).detach().float()
    start = 0
    for n in lengths:
        part = rows[start:start + n].view(n, nh + 2 * nkv, d).transpose(0, 1)
        q, k, v = part[:nh], part[nh:nh + nkv], part[nh + nkv:]
        k, v = k.repeat_interleave(nh // nkv, 0), v.repeat_interleave(nh // nkv, 0)
        sc = (q @ k.transpose(1, 2).contiguous()) / d ** 0.5
        sc = sc.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), float("-inf"))
        ref = (torch.softmax(sc, -1) @ v).transpose(0, 1).reshape(n, nh * d)
        assert (out[start:start + n].float() - ref).abs().max() < 2e-3
        start += n
    up = torch.randn(out.shape, device=DEV)
    grads = torch.autograd.grad(out, leaves, up.half())
    assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in grads)
    # directional difference along wq's gradient; fp16 rows bound how small the step may be
    dirn = grads[3] / grads[3].norm()
    with torch.no_grad():
        h = 0.25
        f = lambda w: float((call(w).double() * up.half().double()).sum())
        slope = (f(x["wq"] + h * dirn) - f(x["wq"] - h * dirn)) / (2 * h)
    assert abs(slope - float(grads[3].norm())) < 0.05 * float(grads[3].norm())


@pytest.mark.parametrize("rows,nh,nkv", [(1, 4, 2), (9, 4, 0), (9, 4, 2)])
def test_gradients_of_leaves_share_no_memory(rows, nh, nkv):
    """Two backwards add up in every leaf's .grad by themselves."""
    d = 64
    leaves = [torch.randn(rows, (nh + 2 * nkv) * d, device=DEV).half().requires_grad_(True),
              torch.randn(rows, nh * d, device=DEV).half().requires_grad_(True),
              torch.randn(rows, nkv * d, device=DEV).half().requires_grad_(True) if nkv else None]
    w = torch.ones(d, device=DEV)
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(16, d))
    pos = torch.arange(rows, device=DEV)
    given = [t for t in leaves if t is not None]
    up = torch.randn(rows, (nh + 2 * nkv) * d, device=DEV).half()
    once = None
    for _ in range(2):
        rope.qk_norm_rope(*leaves, w, w, cos, sin, pos, 1, 16, nh, nkv, d).backward(up)
        if once is None:
            once = [t.grad.clone() for t in given]
    assert len({t.grad.untyped_storage().data_ptr() for t in given}) == len(given)
    for t, g in zip(given, once):
        assert torch.equal(t.grad, (g.float() * 2).half())
