"""Tables from a model's rope_scaling on the GPU, against 64 bits; tolerances as in test_gpu_rotary.py."""

from fractions import Fraction

import pytest
import torch

from oracle import generate as og
from testt_amd import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"


def same(got, want):
    for a, b in zip(got, want):
        assert bool(((a.cpu().double() - b).abs() <= 2.0 ** -24 * b.abs() + 2e-9).all())


@pytest.mark.parametrize("seq,dim,theta,kw", [
    (4097, 64, 150000.0, dict(factor=32.0)), (300, 128, 1e6, {}), (65, 96, 5e5, dict(beta_fast=20.0, beta_slow=1.5)),
    (33, 64, 1e4, dict(attention_factor=0.75))])
def test_yarn_between_pairs(seq, dim, theta, kw):
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "truncate": False, **kw}
    same(rope.rotary_tables(seq, dim, theta, scaling, device=DEV), og.rotary_tables(seq, dim, theta, scaling))
    scaling["truncate"] = True
    whole = rope.rotary_tables(seq, dim, theta, scaling, device=DEV)
    del scaling["truncate"]
    assert all(torch.equal(a, b) for a, b in zip(whole, rope.rotary_tables(seq, dim, theta, scaling, device=DEV)))


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default", "rope_theta": 1e6}, {"rope_type": "linear", "factor": 2.0, "rope_theta": 5e5},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "rope_theta": 150000.0}])
def test_the_base_stands_in_the_scaling(scaling):
    """transformers keeps rope_theta beside the scaling."""
    theta = scaling["rope_theta"]
    want = og.rotary_tables(300, 64, theta, scaling)
    same(rope.rotary_tables(300, 64, scaling=scaling, device=DEV), want)
    same(rope.rotary_tables(300, 64, theta, scaling, device=DEV), want)
    same(rope.rotary_tables(300, 64, device=DEV), og.rotary_tables(300, 64, 1e4))
    bare = {k: v for k, v in scaling.items() if k != "rope_theta"}
    same(rope.rotary_tables(300, 64, scaling=bare, device=DEV), og.rotary_tables(300, 64, 1e4, bare))


# pi, to 50 digits
PI = Fraction("3.14159265358979323846264338327950288419716939937510")


@pytest.mark.parametrize("seq,freq", [
    ((1 << 21) + 5, [1e6, -999999.9, 123456.78901234567, 1.0]), ((1 << 24) + 1, [1e6]), (1 << 20, [1e6] * 4),
    (700, [987654.321, 1e6, 0.3]), ((1 << 24) + 3, [0.1, 1.0, 700.7, 3e4])])
def test_far_angles_of_given_frequencies(seq, freq):
    """Angles of up to 10^13 rad, reduced by whole numbers here: a double's product with a position is not the
    angle (2^21 * 10^6 rad in 64 bits is off by 1e-4)."""
    cos, sin = rope.rotary_tables(seq, 2 * len(freq), inv_freq=freq, device=DEV)
    rows = sorted({0, 1, 17, 127, seq // 3, seq // 2, *range(seq - 40, seq)})
    at = [[float(Fraction(f) * t % (2 * PI)) for f in freq] for t in rows]
    ang = torch.tensor(at, dtype=torch.float64)
    same((cos[rows], sin[rows]), (ang.cos(), ang.sin()))
