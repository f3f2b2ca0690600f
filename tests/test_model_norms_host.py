"""The model plan of attentions that normalise queries and keys per head (CPU)."""

import pytest
import torch

from testt_amd import model, workloads


def tiny():
    return workloads.qwen2_qlora("cpu", n_layers=2, vocab=1000, hidden=256, inter=512, n_heads=2,
                                 n_kv=1)


def head_norm(n, eps=1e-5):
    norm = torch.nn.Module()
    norm.weight, norm.variance_epsilon = torch.nn.Parameter(torch.ones(n)), eps
    return norm


def test_plan_takes_the_norms():
    hf = tiny()
    for lyr in hf.model.layers:
        lyr.self_attn.q_norm, lyr.self_attn.k_norm = head_norm(128), head_norm(128)
    plan = model.model_plan(hf)
    lw = plan.layer_weights(plan.layers[0])
    attn = hf.model.layers[0].self_attn
    assert lw.q_norm is attn.q_norm.weight and lw.k_norm is attn.k_norm.weight
    assert lw.qk_eps == 1e-5
    without = model.model_plan(tiny())
    assert without.layer_weights(without.layers[0]).q_norm is None


@pytest.mark.parametrize("q,k", [((128, 1e-5), None), ((128, 1e-5), (128, 1e-6)),
                                 ((256, 1e-5), (256, 1e-5))])
def test_plan_refuses_other_norms(q, k, capsys):
    """A norm on only one of them, two different eps, a norm over all heads at once."""
    hf = tiny()
    attn = hf.model.layers[1].self_attn
    attn.q_norm = head_norm(*q)
    if k is not None:
        attn.k_norm = head_norm(*k)
    assert model.model_plan(hf) is None
    assert "norm" in capsys.readouterr().out
