"""Per-head RMS norm of queries and keys followed by the rotation, in 64 bits."""

import torch


def qk_norm_rope(qkv, lora_q, lora_v, wq, wk, cos, sin, pos, batch, seq, nh, nkv, d, eps):
    """float64 rows [M, (nh + 2 nkv) d], differentiable in qkv, the deltas and the weights; a token
    whose position lies outside [0, batch * seq) gives zeros."""
    m = qkv.shape[0]
    x = qkv.view(m, nh + 2 * nkv, d)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if lora_q is not None:
        q = q + lora_q.view(m, nh, d)
    if lora_v is not None:
        v = v + lora_v.view(m, nkv, d)
    known = (pos >= 0) & (pos < batch * seq)
    t = torch.where(known, pos, 0) % max(seq, 1)
    c, s = cos[t][:, None], sin[t][:, None]

    def rotated(h, w):
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w
        a, b = y[..., :d // 2], y[..., d // 2:]
        return y * c + torch.cat([-b, a], -1) * s

    out = torch.cat([rotated(q, wq), rotated(k, wk), v], 1).flatten(1)
    return torch.where(known[:, None], out, 0.0)
