"""model.fused_forward on a model whose attention normalises queries and keys per head: loss and gradients
against the fp32 chain of test_gpu_operators_together (its tolerance: fp16 products, 3e-2 of the norm)."""

import pytest
import torch

from testt_amd import model, workloads
from tests.test_gpu_operators_together import (DEV, H, INTER, NH, NKV, SEQ, VOCAB, batch_of, reference,
                                               rel_err)

pytestmark = pytest.mark.gpu


def build(dtype, trained):
    hf = workloads.qwen2_qlora(DEV, n_layers=2, vocab=VOCAB, hidden=H, inter=INTER, n_heads=NH, n_kv=NKV)
    norm = type(hf.model.norm)
    g = torch.Generator().manual_seed(4)
    for lyr in hf.model.layers:
        for name in ("q_norm", "k_norm"):
            n = norm(128, eps=1e-5).to(DEV)
            n.weight = torch.nn.Parameter((1 + 0.2 * torch.randn(128, generator=g)).to(DEV, dtype),
                                          requires_grad=trained)
            setattr(lyr.self_attn, name, n)
    return hf.train()


@pytest.mark.parametrize("dtype,trained", [(torch.float32, True), (torch.float32, False),
                                           (torch.float16, False), (torch.float16, True)])
def test_step_with_head_norms(dtype, trained):
    print(f"model norms {dtype} trained {trained}", flush=True)
    hf = build(dtype, trained)
    amask, pos = batch_of((SEQ, 20))
    ids = torch.randint(0, VOCAB, (2, SEQ), generator=torch.Generator().manual_seed(2)).to(DEV)
    labels = torch.where(amask.bool(), ids, -100)
    params = workloads.lora_parameters(hf)
    norms = [n.weight for lyr in hf.model.layers for n in (lyr.self_attn.q_norm, lyr.self_attn.k_norm)]
    with torch.autocast("cuda", dtype=torch.float16):
        assert model.can_run(hf, ids, amask, labels, {})
        loss = model.fused_forward(hf, ids, amask, labels, None).loss
    got = torch.autograd.grad(loss, params + (norms if trained else []))

    plan = model.model_plan(hf)
    cos, sin = model.rotary_tables(hf.model.rotary_emb.inv_freq, SEQ)
    s, delta = hf.model.embed_tokens.weight.float()[ids.reshape(-1)[pos]], None
    wide = [w.float() if dtype is not torch.float32 else w for w in norms]
    if trained and dtype is not torch.float32:
        wide = [w.detach().requires_grad_(True) for w in wide]
    for i, lp in enumerate(plan.layers):
        w = plan.layer_weights(lp)
        w.q_norm, w.k_norm = wide[2 * i:2 * i + 2]
        s, delta = reference(s, delta, w, pos, 2, SEQ, cos, sin, [None, None])
    s = s + delta
    y = hf.model.norm.weight.float() * (
        s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + hf.model.norm.variance_epsilon))
    ref = torch.nn.functional.cross_entropy(y @ hf.model.embed_tokens.weight.float().t(),
                                            model.shifted_targets(labels, pos), ignore_index=-100)
    want = torch.autograd.grad(ref, params + (wide if trained else []))
    assert rel_err(loss, ref) < 3e-2
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == (params + norms)[i].dtype and rel_err(a, b) < 3e-2, (i, rel_err(a, b))
