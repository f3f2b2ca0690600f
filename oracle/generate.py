"""The operators of a generating program in 64 bits, from their definitions: tables of rotary positions, the
rotation, the paged cache and its attention, the verification of drafted tokens.  Loops over tokens and
sequences, on the CPU."""

import math

import torch


def frequencies(dim, theta, scaling=None, seq=0):
    """(radians a position of each pair, gain)."""
    kind = "default" if scaling is None else scaling["rope_type"]
    gain = 1.0
    if kind == "dynamic":
        n0 = scaling["original_max_position_embeddings"]
        if seq > n0 and dim > 2:
            theta = theta * (scaling["factor"] * seq / n0 - scaling["factor"] + 1) ** (dim / (dim - 2))
    freq = [theta ** (-2 * i / dim) for i in range(dim // 2)]
    if kind == "linear":
        freq = [f / scaling["factor"] for f in freq]
    if kind == "yarn":
        n0 = scaling["original_max_position_embeddings"]
        # pair i turns n0 theta^(-2 i / dim) / (2 pi) times within n0
        at = [dim / 2 * math.log(n0 / (2 * math.pi * turns)) / math.log(theta)
              for turns in (scaling.get("beta_fast", 32), scaling.get("beta_slow", 1))]
        if scaling.get("truncate", True):
            at = [math.floor(at[0]), math.ceil(at[1])]
        low, high = max(at[0], 0), min(at[1], dim - 1)
        r = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(dim // 2)]
        freq = [f * (1 - x) + f / scaling["factor"] * x for f, x in zip(freq, r)]
        gain = scaling.get("attention_factor", 0.1 * math.log(scaling["factor"]) + 1)
    return freq, gain


def rotary_tables(seq, dim, theta=1e4, scaling=None, start=0):
    freq, gain = frequencies(dim, theta, scaling, seq)
    ang = torch.arange(start, seq, dtype=torch.float64)[:, None] * torch.tensor(freq, dtype=torch.float64)
    return gain * ang.cos(), gain * ang.sin()


def rotary(x, cos, sin, pos, interleaved=False):
    """x [M, heads, D] (64 bits, differentiable); a position outside the tables gives zeros."""
    half = cos.shape[1]
    known = (pos >= 0) & (pos < cos.shape[0])
    at = torch.where(known, pos, 0)
    if cos.shape[0] == 0:
        return x * 0
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.where(known[:, None, None], torch.cat([turned, x[..., 2 * half:]], -1), 0.0)


def places(rows, cu, lengths, table, page, n_pages, n_pos=None):
    """For each row (sequence, position, page, slot), or None where it has no place."""
    out = [None] * rows
    bounds = [(b, b + 1) for b in range(len(lengths))] if cu is None else list(zip(cu[:-1], cu[1:]))
    for b, (lo, hi) in enumerate(bounds):
        for r in range(lo, hi):
            t = lengths[b] - (hi - r)
            if t < 0 or (n_pos is not None and t >= n_pos) or t // page >= len(table[b]):
                continue
            if 0 <= table[b][t // page] < n_pages:
                out[r] = (b, t, table[b][t // page], t % page)
    return out


def rope_append(qkv, lora_q, lora_v, cos, sin, k, v, table, lengths, cu=None, interleaved=False):
    """(q rows, k pages, v pages) in 64 bits, after the append."""
    n_pages, n_kv, page, d = k.shape
    m, heads = qkv.shape[0], qkv.shape[1] // d
    nh = heads - 2 * n_kv
    x = qkv.double().view(m, heads, d).clone()
    if lora_q is not None:
        x[:, :nh] += lora_q.double().view(m, nh, d)
    if lora_v is not None:
        x[:, nh + n_kv:] += lora_v.double().view(m, n_kv, d)
    at = places(m, cu, lengths, table, page, n_pages, None if cos is None else cos.shape[0])
    pos = torch.tensor([-1 if p is None else p[1] for p in at], dtype=torch.int64)
    if cos is not None:
        x[:, :nh + n_kv] = rotary(x[:, :nh + n_kv], cos, sin, pos, interleaved)
    k, v = k.double().clone(), v.double().clone()
    for r, p in enumerate(at):
        if p is None:
            x[r] = 0
        else:
            k[p[2], :, p[3]] = x[r, nh:nh + n_kv]
            v[p[2], :, p[3]] = x[r, nh + n_kv:]
    return x[:, :nh].reshape(m, -1), k, v


def paged_attention(q, k, v, table, lengths, cu=None, scale=None):
    """(out [M, NH D], weight): softmax(scale q.k) v over the keys that each row sees, and the same sum
    of |v|, the scale of its rounding errors."""
    n_pages, n_kv, page, d = k.shape
    m, nh = q.shape[0], q.shape[1] // d
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(m, nh, d, dtype=torch.float64)
    weight = torch.zeros_like(out)
    bounds = [(b, b + 1) for b in range(len(lengths))] if cu is None else list(zip(cu[:-1], cu[1:]))
    for b, (lo, hi) in enumerate(bounds):
        length, held = lengths[b], max(min(lengths[b], len(table[b]) * page), 0)
        keys = [(table[b][t // page], t % page) if 0 <= table[b][t // page] < n_pages else None
                for t in range(held)]
        seen = [t for t in range(held) if keys[t] is not None]
        if not seen:
            continue
        p, s = (torch.tensor([keys[t][i] for t in seen]) for i in (0, 1))
        kb, vb = k[p, :, s].double(), v[p, :, s].double()        # [keys, n_kv, d]
        for r in range(lo, hi):
            n = sum(t <= length - (hi - r) for t in seen)
            if n == 0:
                continue
            for h in range(nh):
                g = h // (nh // n_kv)
                w = torch.softmax(scale * (kb[:n, g] @ q[r, h * d:(h + 1) * d].double()), 0)
                out[r, h], weight[r, h] = w @ vb[:n, g], w @ vb[:n, g].abs()
    return out.view(m, -1), weight.view(m, -1)


def verify_drafts(target, drafts, uniforms, draft_probs=None, lengths=None):
    """(tokens [B, K + 1], accepted [B])."""
    batch, k, vocab = target.shape[0], target.shape[1] - 1, target.shape[2]
    mass = lambda t: torch.where((t > 0) & torch.isfinite(t), t, 0.0).double()  # noqa: E731
    tokens = torch.full((batch, k + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(batch, dtype=torch.int32)
    for b in range(batch):
        n, length, refused = 0, k if lengths is None else min(max(int(lengths[b]), 0), k), False
        while n < length and not refused:
            x = int(drafts[b, n])
            known = 0 <= x < vocab
            px = float(mass(target[b, n, x])) if known else 0.0
            qx = 1.0 if draft_probs is None else float(mass(draft_probs[b, n, x])) if known else 0.0
            if known and float(uniforms[b, n]) * qx < px:
                tokens[b, n] = x
                n += 1
            else:
                refused = True
        p = mass(target[b, n])
        w = p
        if refused and draft_probs is not None:
            w = (p - mass(draft_probs[b, n])).clamp(min=0)
        elif refused:
            w = p.clone()
            if 0 <= int(drafts[b, n]) < vocab:
                w[int(drafts[b, n])] = 0
        if not bool((w > 0).any()):
            w = p
        upto = torch.cumsum(w, 0)
        if bool((w > 0).any()):
            past = (upto > float(uniforms[b, k]) * upto[-1]) & (w > 0)
            at = past if bool(past.any()) else w > 0
            tokens[b, n] = int(at.nonzero()[0 if bool(past.any()) else -1])
        accepted[b] = n
    return tokens, accepted
