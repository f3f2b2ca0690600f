"""A model's rope_scaling: the frequencies of the 64-bit reference and of rope.rotary_tables against transformers' own,
which are fp32 (a few roundings of 2^-24), on the CPU."""

import logging

import pytest
import torch

from oracle import generate as og
from testt_amd import rope

transformers = pytest.importorskip("transformers")
rope_utils = pytest.importorskip("transformers.modeling_rope_utils")


def theirs(dim, theta, scaling):
    """(frequencies, gain) of transformers."""
    log = logging.getLogger("transformers.modeling_rope_utils")
    level = log.level
    log.setLevel(logging.ERROR)
    try:
        config = transformers.Qwen2Config(hidden_size=2 * dim, num_attention_heads=2, head_dim=dim,
                                          max_position_embeddings=32768,
                                          rope_parameters={**scaling, "rope_theta": theta})
        freq, gain = rope_utils.ROPE_INIT_FUNCTIONS[scaling["rope_type"]](config, "cpu")
    finally:
        log.setLevel(level)
    return freq.double(), gain


def yarn(**kw):
    return {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, **kw}


CASES = [(64, 1e4, yarn()), (128, 1e6, yarn(factor=32.0)), (64, 1e4, yarn(truncate=True)),
         (64, 1e4, yarn(beta_fast=16.0, beta_slow=2.0, attention_factor=0.75)),
         (64, 1e4, {"rope_type": "linear", "factor": 2.5}),
         (64, 150000.0, yarn(factor=32.0, truncate=False)), (128, 1e6, yarn(truncate=False)),
         (96, 5e5, yarn(beta_fast=20.0, beta_slow=1.5, truncate=False))]


@pytest.mark.parametrize("dim,theta,scaling", CASES)
def test_the_reference_has_transformers_frequencies(dim, theta, scaling):
    want, gain = theirs(dim, theta, scaling)
    got, mine = og.frequencies(dim, theta, scaling)
    assert float((torch.tensor(got, dtype=torch.float64) / want - 1).abs().max()) < 16 * 2.0 ** -24
    assert abs(mine - gain) < 1e-12


@pytest.mark.parametrize("dim,theta,scaling", CASES[-3:])
def test_frequencies_between_pairs(dim, theta, scaling):
    want, _ = theirs(dim, theta, scaling)
    got = rope._yarn_between(dim, theta, scaling["factor"], scaling["original_max_position_embeddings"],
                             scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0))
    assert float((torch.tensor(got, dtype=torch.float64) / want - 1).abs().max()) < 16 * 2.0 ** -24


def test_truncate_is_a_truth_value():
    with pytest.raises(TypeError, match="truncate"):
        rope.rotary_tables(8, 16, scaling=yarn(truncate="no"))


def test_two_bases_are_refused():
    for scaling in ({"rope_type": "default", "rope_theta": 1e6}, yarn(rope_theta=1e6)):
        with pytest.raises(ValueError, match="rope_theta"):
            rope.rotary_tables(8, 16, 1e4, scaling)
    with pytest.raises(ValueError, match="theta"):
        rope.rotary_tables(8, 16, scaling=yarn(rope_theta=0.5))
    with pytest.raises(ValueError, match="theta"):
        rope.rotary_tables(8, 16, 0.0)


@pytest.mark.parametrize("scaling,match", [
    (yarn(short_factor=[1.0]), "short_factor"), (yarn(low_freq_factor=1.0), "low_freq_factor"),
    ({"rope_type": "linear", "factor": 2.0, "beta_fast": 32.0}, "beta_fast"),
    ({"rope_type": "linear", "factor": 2.0, "attention_factor": 0.5}, "attention_factor"),
    ({"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 64, "alpha": 2.0}, "alpha"),
    ({"rope_type": "default", "factor": 2.0}, "factor"), ({"rope_type": "default", "truncate": True}, "truncate"),
    (yarn(partial_rotary_factor=0.5), "partial_rotary_factor"),
    ({"rope_type": "default", "partial_rotary_factor": 0.25}, "partial_rotary_factor")])
def test_keys_that_would_be_passed_over_are_refused(scaling, match):
    with pytest.raises(ValueError, match=match):
        rope.rotary_tables(8, 16, scaling=scaling)


def test_scalings_of_configurations_are_read():
    """What transformers' configurations hold comes as far as the device."""
    for scaling in ({"rope_type": "default"}, {"rope_type": "linear", "factor": 2.0}, yarn(truncate=False), yarn()):
        config = transformers.Qwen2Config(rope_parameters={**scaling, "rope_theta": 1e6})
        with pytest.raises(ValueError, match="no CPU path"):
            rope.rotary_tables(8, 16, scaling=config.rope_scaling, device="cpu")
        rope._check_scaling({**config.rope_scaling, "partial_rotary_factor": 1.0, "beta_fast": None, "type": None})
    rope._check_scaling({"rope_type": "linear", "factor": 2.0, "original_max_position_embeddings": 64})
