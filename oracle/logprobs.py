"""Log probabilities of given tokens, entropy and top alternatives in 64 bits, from the definition."""

import torch


def token_logprobs(logits, tokens, top_k=0, temperature=1.0):
    """(logprob, entropy, top_logprobs, top_ids) over the last dimension, differentiable in float64
    `logits`; token -100 gives 0, another token outside the vocabulary NaN."""
    vocab = logits.shape[-1]
    lp = torch.log_softmax(logits / temperature, -1)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * torch.where(p > 0, lp, 0), 0).sum(-1)
    # (a NaN in the row has to reach the entropy, as the where above would drop it)
    entropy = torch.where(torch.isnan(lp).any(-1), float("nan"), entropy)
    ok = (tokens >= 0) & (tokens < vocab)
    at = torch.where(ok, tokens, 0)[..., None]
    logprob = torch.where(ok, lp.gather(-1, at)[..., 0], float("nan"))
    logprob = torch.where(tokens == -100, 0.0, logprob)
    order = torch.where(torch.isnan(logits), float("-inf"), logits.detach())
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :top_k]
    return logprob, entropy, lp.gather(-1, ids), ids
