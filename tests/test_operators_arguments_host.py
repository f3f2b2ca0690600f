"""Arguments of the operators around the layer that are no plain tensors, or are left out (CPU)."""

import pytest
import torch

from testt_amd import dropout, embedding, head, rope


class Seen(torch.Tensor):
    """A subclass with a protocol of its own."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        return func, args, kwargs


class Wrapper(torch.Tensor):
    """A tensor that holds no memory."""

    @staticmethod
    def __new__(cls, shape, dtype):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda:0")

    __torch_function__ = torch._C._disabled_torch_function_impl

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} was called on a wrapper")


def seen(*shape):
    return torch.zeros(*shape).as_subclass(Seen)


TOK = torch.zeros(4, dtype=torch.int64)
W = torch.ones(16)


@pytest.mark.parametrize("call,func", [
    (lambda: head.token_logprobs(seen(4, 8), TOK, 2, 0.5), head.token_logprobs),
    (lambda: head.token_logprobs(torch.zeros(4, 8), seen(4)), head.token_logprobs),
    (lambda: dropout.dropout(seen(4, 8), 0.5, 1), dropout.dropout),
    (lambda: dropout.dropout(torch.zeros(4, 8), 0.5, seen(1)), dropout.dropout),
    (lambda: dropout.dropout(torch.zeros(4, 8), 0.5, 1, rows=seen(4)), dropout.dropout),
    (lambda: dropout.dropout(torch.zeros(4, 8), 0.5, 1, residual=seen(4, 8)), dropout.dropout),
    (lambda: embedding.embedding(TOK, seen(4, 8), padding_idx=1), embedding.embedding),
    (lambda: embedding.embedding(seen(4), torch.zeros(4, 8)), embedding.embedding),
    (lambda: rope.qk_norm_rope(seen(4, 48), None, None, W, W, W, W, TOK, 1, 4, 1, 1, 16),
     rope.qk_norm_rope),
    (lambda: rope.qk_norm_rope(torch.zeros(4, 48), None, None, W, seen(16), W, W, TOK, 1, 4, 1, 1, 16),
     rope.qk_norm_rope),
    (lambda: rope.qk_norm_rope(torch.zeros(4, 48), None, seen(4, 16), W, W, W, W, TOK, 1, 4, 1, 1, 16),
     rope.qk_norm_rope),
])
def test_a_subclass_is_asked(call, func):
    assert call()[0] is func


def test_wrappers_without_memory_are_refused():
    z, h = Wrapper((4, 8), torch.float32), Wrapper((4, 48), torch.float16)
    tok = Wrapper((4,), torch.int64)
    for call in (lambda: head.token_logprobs(z, tok), lambda: dropout.dropout(z, 0.5, 1),
                 lambda: dropout.dropout(z, 0.5, 1, rows=tok), lambda: embedding.embedding(tok, z),
                 lambda: rope.qk_norm_rope(h, None, None, Wrapper((16,), torch.float32),
                                           Wrapper((16,), torch.float32), Wrapper((4, 16), torch.float32),
                                           Wrapper((4, 16), torch.float32), tok, 1, 4, 1, 1, 16)):
        with pytest.raises(TypeError, match="memory"):
            call()
    assert not embedding.supported(z)


def test_counter_dropout_needs_a_seed():
    """Modules left at one default seed would all draw the same mask."""
    with pytest.raises(TypeError, match="seed"):
        dropout.CounterDropout(0.1)
    with pytest.raises(TypeError, match="seed"):
        dropout.CounterDropout()
    assert dropout.CounterDropout(0.1, 0).seed == 0
