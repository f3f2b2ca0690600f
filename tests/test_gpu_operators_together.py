"""The operators as a training program runs them: embedding -> decoder layers with per-head q/k norms
and counter-based LoRA dropout -> final norm -> log probabilities of the sampled tokens -> a
policy-gradient loss, and back to the table, the norms and the LoRA parameters, against an fp32 eager
model with the same weights (dequantized by the oracle) and the same masks (drawn by the oracle).

The layer's products run in fp16, as in tests/test_gpu_layer_step.py, whose relative-norm tolerance
(2e-2 a layer) is taken: 3e-2 for what passes through two layers and the head."""

import numpy as np
import pytest
import torch

from oracle.dropout import keep_mask
from oracle.logprobs import token_logprobs
from oracle.nf4 import dequant_state
from oracle.qk_norm import qk_norm_rope
from testt_amd import embedding, head, layer, model, workloads
from testt_amd.dropout import CounterDropout
from testt_amd.rmsnorm import add_rmsnorm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
H, INTER, NH, NKV, VOCAB, SEQ = 256, 512, 2, 1, 1000, 48
P, CALL = 0.2, 3


def rel_err(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def build(head_dim, seed, drops):
    w = layer.synthetic_layer(DEV, hidden=H, inter=INTER, n_heads=NH, n_kv=NKV, head_dim=head_dim,
                              seed=seed)
    g = torch.Generator().manual_seed(seed)
    w.q_norm, w.k_norm = ((1 + 0.2 * torch.randn(head_dim, generator=g)).to(DEV).requires_grad_(True)
                          for _ in range(2))
    w.qk_eps = 1e-5
    w.lora_dropout = drops
    return w


def leaves(w):
    return [*w.lora_q, *w.lora_v, w.q_norm, w.k_norm]


def reference(s, delta, w, pos, batch, seq, cos, sin, masks):
    """One layer in fp32; masks: the (q, v) keep masks of the LoRA dropouts or None."""
    nh, nkv, hd = w.n_heads, w.n_kv, w.head_dim
    wd = {n: torch.from_numpy(dequant_state(getattr(w, n)).astype(np.float32)).to(DEV)
          for n in ("q", "k", "v", "o", "gate", "up", "down")}

    def norm(x, weight):
        return weight * (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + w.eps))

    s = s if delta is None else s + delta
    y = norm(s, w.input_norm)
    qkv = y @ torch.cat([wd["q"], wd["k"], wd["v"]]).t() + w.qkv_bias.float()
    rows = [y if m is None else torch.where(m, y / (1 - P), 0) for m in masks]
    lq = (rows[0] @ w.lora_q[0].t()) @ w.lora_q[1].t() * w.scaling
    lv = (rows[1] @ w.lora_v[0].t()) @ w.lora_v[1].t() * w.scaling
    r = qk_norm_rope(qkv, lq, lv, w.q_norm, w.k_norm, cos, sin, pos, batch, seq, nh, nkv, hd,
                     w.qk_eps).view(-1, nh + 2 * nkv, hd)
    out = []
    for b in range(batch):
        part = r[(pos // seq) == b].transpose(0, 1)
        n = part.shape[1]
        k, v = (part[i:i + nkv].repeat_interleave(nh // nkv, 0) for i in (nh, nh + nkv))
        sc = (part[:nh] @ k.transpose(1, 2).contiguous()) / hd ** 0.5
        sc = sc.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), float("-inf"))
        out.append((torch.softmax(sc, -1) @ v).transpose(0, 1).reshape(n, nh * hd))
    s = s + torch.cat(out) @ wd["o"].t()
    y2 = norm(s, w.post_norm)
    return s, (torch.nn.functional.silu(y2 @ wd["gate"].t()) * (y2 @ wd["up"].t())) @ wd["down"].t()


def batch_of(lengths):
    amask = torch.zeros(len(lengths), SEQ, dtype=torch.int64, device=DEV)
    for b, n in enumerate(lengths):
        amask[b, :n] = 1
    return amask, amask.reshape(-1).nonzero().squeeze(1)


def masks_of(pos, drops):
    return [torch.from_numpy(keep_mask(pos.tolist(), H, P, d.seed, d.call)).to(DEV) for d in drops]


@pytest.mark.parametrize("head_dim", [128, 64])     # 64: the padded path on torch's attention
@pytest.mark.parametrize("dropout", [False, True])
def test_layer_with_norms_and_counter_dropout(head_dim, dropout):
    print(f"layer head_dim {head_dim} dropout {dropout}", flush=True)
    amask, pos = batch_of((48, 17))
    drops = tuple(CounterDropout(P, 100 + i) for i in range(2)) if dropout else None
    w = build(head_dim, 5, drops)
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(SEQ, head_dim))
    g = torch.Generator().manual_seed(8)
    rnd = lambda scale: scale * torch.randn(pos.numel(), H, generator=g).to(DEV)
    s0, d0, gs, gd = rnd(1.0), rnd(0.5), rnd(1e-2), rnd(1e-2)
    masks = [None, None]
    if dropout:
        for d in drops:
            d.call = CALL
        masks = masks_of(pos, drops)
    a, b = s0.clone().requires_grad_(True), d0.half().requires_grad_(True)
    s, d = layer.decoder_layer(a, b, w, pos, 2, SEQ, cos, sin, layer.key_valid_of(amask))
    got = torch.autograd.grad([s, d], [a, b, *leaves(w)], [gs, gd.half()])
    ra, rb = s0.clone().requires_grad_(True), d0.half().float().requires_grad_(True)
    rs, rd = reference(ra, rb, w, pos, 2, SEQ, cos, sin, masks)
    want = torch.autograd.grad([rs, rd], [ra, rb, *leaves(w)], [gs, gd.half().float()])
    assert rel_err(s, rs) < 2e-2 and rel_err(d, rd) < 2e-2
    for i, (x, y) in enumerate(zip(got, want)):
        assert rel_err(x, y) < 2e-2, (i, rel_err(x, y))
    if dropout:
        assert all(d.call == CALL + 1 for d in drops)


def run(table, final_norm, layers, ids, tokens, adv, pos, batch, cos, sin):
    """(loss, the log probabilities) of one policy-gradient step through the package."""
    s = embedding.embedding(ids, table, out_dtype=torch.float32)
    delta = None
    for w in layers:
        s, delta = layer.decoder_layer(s, delta, w, pos, batch, SEQ, cos, sin, None)
    _, y, _ = add_rmsnorm(s, delta, final_norm, 1e-6)
    out = head.fused_token_logprobs(y, table.detach(), tokens, top_k=4, temperature=0.8)
    return -(out.logprob * adv).sum() - 0.01 * out.entropy.mean(), out


def test_policy_gradient_step():
    amask, pos = batch_of((48, 31, 1))
    g = torch.Generator().manual_seed(21)
    m = pos.numel()
    drops = [tuple(CounterDropout(P, 10 * i + j) for j in range(2)) for i in range(2)]
    layers = [build(128, 30 + i, drops[i]) for i in range(2)]
    table = (0.05 * torch.randn(VOCAB, H, generator=g)).half().to(DEV).requires_grad_(True)
    final_norm = (1 + 0.1 * torch.randn(H, generator=g)).to(DEV)
    ids = torch.randint(0, VOCAB, (m,), generator=g).to(DEV)
    ids[5:20] = 7                                     # a token of many places
    tokens = torch.randint(0, VOCAB, (m,), generator=g).to(DEV)
    tokens[:9] = -100
    adv = torch.randn(m, generator=g).to(DEV) / m
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(SEQ, 128))
    masks = [masks_of(pos, d) for d in drops]
    loss, out = run(table, final_norm, layers, ids, tokens, adv, pos, 3, cos, sin)
    params = [table] + [p for w in layers for p in leaves(w)]
    got = torch.autograd.grad(loss, params)

    t32 = table.detach().float().requires_grad_(True)
    s, delta = t32[ids], None
    for w, mk in zip(layers, masks):
        s, delta = reference(s, delta, w, pos, 3, SEQ, cos, sin, mk)
    s = s + delta
    y = final_norm * (s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + 1e-6))
    lp, ent, _, _ = token_logprobs(y @ t32.detach().t(), tokens, 4, 0.8)
    ref = -(lp * adv).sum() - 0.01 * ent.mean()
    want = torch.autograd.grad(ref, [t32] + [p for w in layers for p in leaves(w)])
    assert rel_err(out.logprob, lp) < 3e-2 and rel_err(out.entropy, ent) < 3e-2
    for i, (a, b) in enumerate(zip(got, want)):
        assert rel_err(a, b) < 3e-2, (i, rel_err(a, b))
    # the same calls again: the same bits, forward and backward
    for d in drops:
        for x in d:
            x.call = 0
    again, _ = run(table, final_norm, layers, ids, tokens, adv, pos, 3, cos, sin)
    assert torch.equal(again, loss)
    for a, b in zip(torch.autograd.grad(again, params), got):
        assert torch.equal(a, b)


def test_model_with_counter_dropout():
    """CounterDropout as a model's LoRA dropout, through fused_forward: the step repeats bit for bit
    when the call number does, and the draws change otherwise."""
    hf = workloads.qwen2_qlora(DEV, n_layers=2, vocab=VOCAB, hidden=H, inter=INTER, n_heads=NH,
                               n_kv=NKV, dropout=0.3)
    drops = []
    for lyr in hf.model.layers:
        for proj in (lyr.self_attn.q_proj, lyr.self_attn.v_proj):
            d = CounterDropout(0.3, 50 + len(drops))
            proj.lora_dropout["default"] = d
            drops.append(d)
    hf.train()
    ids = torch.randint(0, VOCAB, (2, SEQ), device=DEV)
    amask, _ = batch_of((SEQ, 20))
    labels = torch.where(amask.bool(), ids, -100)

    def step():
        with torch.autocast("cuda", dtype=torch.float16):
            assert model.can_run(hf, ids, amask, labels, {})
            loss = model.fused_forward(hf, ids, amask, labels, None).loss
        return loss.detach(), torch.autograd.grad(loss, workloads.lora_parameters(hf))

    a, ga = step()
    b, _ = step()
    assert all(d.call == 2 for d in drops) and not torch.equal(a, b)
    for d in drops:
        d.call = 0
    c, gc = step()
    assert torch.equal(a, c) and all(torch.equal(x, y) for x, y in zip(ga, gc))


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    """No operator has a forward-mode derivative: a dual tensor raises, also without gradients."""
    import torch.autograd.forward_ad as ad
    from testt_amd import dropout, embedding, head, rope
    z = torch.randn(4, 200, device=DEV)
    tok = torch.arange(4, device=DEV)
    qkv, w = torch.randn(4, 3 * 64, device=DEV).half(), torch.ones(64, device=DEV)
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(16, 64))
    with torch.set_grad_enabled(grad), ad.dual_level():
        dual = lambda t: ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: head.token_logprobs(dual(z), tok, 2),
                     lambda: dropout.dropout(dual(z), 0.5, 1),
                     lambda: dropout.dropout(z, 0.5, 1, residual=dual(z)),
                     lambda: embedding.embedding(tok, dual(z)),
                     lambda: rope.qk_norm_rope(qkv, None, None, dual(w), w, cos, sin, tok, 1, 16, 1, 1,
                                               64)):
            with pytest.raises(RuntimeError, match="jvp"):
                call()


def test_second_derivatives_are_refused():
    """A gradient taken with create_graph and differentiated again raises, also where the upstream
    gradient is a constant (a gradient penalty would otherwise lose its second-order part in silence)."""
    from testt_amd import dropout, embedding, head, rope
    leaf = lambda *s: torch.randn(*s, device=DEV).requires_grad_(True)
    tok = torch.arange(4, device=DEV)
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(16, 64))
    w = torch.ones(64, device=DEV)
    for x, call in (
            (leaf(4, 200), lambda x: head.token_logprobs(x, tok, 2).entropy),
            (leaf(4, 200), lambda x: dropout.dropout(x, 0.5, 1)),
            (leaf(4, 200), lambda x: embedding.embedding(tok, x)),
            (torch.randn(4, 192, device=DEV).half().requires_grad_(True),
             lambda x: rope.qk_norm_rope(x, None, None, w, w, cos, sin, tok, 1, 16, 1, 1, 64))):
        g, = torch.autograd.grad(call(x).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            (call(x).float().sum() + g.float().pow(2).sum()).backward()
