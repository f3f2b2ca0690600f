"""Arguments of the operators around the layer that are no plain tensors or numbers."""

import pytest
import torch

from testt_amd import dropout, embedding, head, rope, workloads

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Sub(torch.Tensor):
    """A subclass that keeps torch's own protocol: operators on it give it back."""


def calls():
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g).to(DEV)
    tok = torch.arange(6, device=DEV)
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(8, 64))
    w = 1 + 0.1 * rnd(64)
    return [
        (rnd(6, 500), lambda x: head.token_logprobs(x, tok, 3, 0.7)),
        (rnd(6, 64), lambda x: dropout.dropout(x, 0.4, 3, residual=x)),
        (rnd(9, 32).half(), lambda x: embedding.embedding(tok, x, 2.0, torch.float32, 1)),
        (rnd(6, 192).half(), lambda x: rope.qk_norm_rope(x, None, None, w, w, cos, sin, tok, 1, 8, 1, 1,
                                                         64)),
    ]


def first(out):
    return out[0] if isinstance(out, tuple) else out


@pytest.mark.parametrize("i", range(4))
def test_subclasses_come_back(i):
    """Values and gradients of a subclass are the plain tensor's, in the subclass's type."""
    x, call = calls()[i]
    plain = x.clone().requires_grad_(True)
    want = call(plain)
    sub = x.clone().as_subclass(Sub).requires_grad_(True)
    got = call(sub)
    assert type(got) is Sub or (type(got) is head.TokenLogprobs and all(type(o) is Sub for o in got))
    for a, b in zip(got if isinstance(got, tuple) else [got], want if isinstance(want, tuple) else [want]):
        assert torch.equal(a.as_subclass(torch.Tensor), b)
    first(want).float().sum().backward()
    first(got).float().sum().backward()
    assert torch.equal(sub.grad.as_subclass(torch.Tensor), plain.grad)
    assert type(call(torch.nn.Parameter(x))) is type(want)


def test_numbers_that_want_a_gradient_are_refused():
    """No gradient is given for a temperature, scale, probability or eps: a tensor that asks for one
    raises instead of staying without in silence; other tensors of one number are taken."""
    num = lambda v, grad: torch.tensor(v, device=DEV, requires_grad=grad)
    (z, _), (x, _), (t, _), (q, _) = calls()
    tok = torch.arange(6, device=DEV)
    cos, sin = (c.to(DEV) for c in workloads.rope_tables(8, 64))
    w = torch.ones(64, device=DEV)
    weight = torch.randn(500, 64, device=DEV).half()
    norm = lambda e: rope.qk_norm_rope(q, None, None, w, w, cos, sin, tok, 1, 8, 1, 1, 64, e)
    for name, value, call in (
            ("temperature", 0.5, lambda v: head.token_logprobs(z, tok, 0, v)),
            ("temperature", 0.5, lambda v: head.fused_token_logprobs(x.half(), weight, tok, 0, v)),
            ("p", 0.5, lambda v: dropout.dropout(x, v, 1)),
            ("scale", 0.5, lambda v: embedding.embedding(tok, t, v)),
            ("scale", 0.5, lambda v: embedding.embedding(tok, t, v, padding_idx=0)),
            ("eps", 0.5, norm)):
        with pytest.raises(TypeError, match=name):
            call(num(value, True))
        assert torch.equal(first(call(num(value, False))), first(call(value)))
        with torch.no_grad():
            assert torch.equal(first(call(num(value, True))), first(call(value)))
