"""Frozen and trained norms of queries and keys in the model plan's layer weights (CPU)."""

import torch

from testt_amd import model
from tests.test_model_norms_host import head_norm, tiny


def test_plan_widens_frozen_head_norms():
    """Frozen norms come as the kernel reads them (fp32, as the layer's own norms); trained ones as the
    parameters that take the gradient."""
    hf = tiny()
    for lyr in hf.model.layers:
        for name in ("q_norm", "k_norm"):
            n = head_norm(128)
            n.weight = torch.nn.Parameter((1 + torch.rand(128)).half(), requires_grad=name == "k_norm")
            setattr(lyr.self_attn, name, n)
    plan = model.model_plan(hf)
    lw = plan.layer_weights(plan.layers[1])
    attn = hf.model.layers[1].self_attn
    assert lw.q_norm.dtype == torch.float32 and torch.equal(lw.q_norm, attn.q_norm.weight.float())
    assert lw.k_norm is attn.k_norm.weight
