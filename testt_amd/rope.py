"""Q/K/V assembly for attention on gfx950: LoRA add + rotary embedding + scatter to the padded
layout.  Drop-in for solution/rope.py.

The fused q/k/v GEMM output (fp16, unpadded tokens) is read once per token by
testt_amd/csrc/rope_pack.hip, which adds the LoRA outputs in fp32, rotates q and k in fp32 and
writes fp16 q/k/v directly into [batch, heads, seq, head_dim] at the token's padded position,
the layout SDPA takes; padded positions with no token are zeroed by the same launch.  Backward
is the transposed rotation, gathering per token and writing the fp16 gradient of the q/k/v GEMM
output; the LoRA branches get views of the same buffer.
"""

import torch
from torch.overrides import handle_torch_function, has_torch_function

from . import _ext
from ._common import next_pow2
from ._index import as_index, inverse_map


def _consts(n_heads, n_kv, head_dim):
    """The reference's compile-time constants (solution/rope.py:131-133), kept for callers."""
    return dict(NH=n_heads, NKV=n_kv, HALF=head_dim // 2, NH_P=next_pow2(n_heads),
                NKV_P=next_pow2(n_kv))


def _table(t, seq, head_dim, name, device):
    t = t.detach()
    if t.dtype != torch.float32:
        t = t.float()
    t = _ext.require(t.contiguous(), name, ndim=2, device=device)
    if t.shape[0] < seq or t.shape[1] != head_dim:
        raise ValueError(f"{name} must be [>= {seq}, {head_dim}], got {tuple(t.shape)}")
    return t


def _lora_pair(lora_q, lora_v):
    """Both LoRA deltas in one element type (fp16 or fp32) and its ABI code."""
    ts = [t for t in (lora_q, lora_v) if t is not None]
    if not ts:
        return lora_q, lora_v, _ext.DTYPE_F16
    if all(t.dtype == torch.float16 for t in ts):
        dtype, code = torch.float16, _ext.DTYPE_F16
    else:
        dtype, code = torch.float32, _ext.DTYPE_F32
    conv = [None if t is None else t.detach().to(dtype).contiguous() for t in (lora_q, lora_v)]
    return conv[0], conv[1], code


class RopePack(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, lora_q, lora_v, cos, sin, pos_idx, batch, seq, n_heads, n_kv, head_dim):
        if pos_idx.dtype is torch.int64 and pos_idx.is_cuda and pos_idx.dim() == 1:
            rows, slots = pos_idx.numel(), batch * seq
            inv = inverse_map(pos_idx.contiguous(), slots) if rows != slots else None
            done = _ext.host().rope_fwd(qkv, lora_q, lora_v, cos, sin, pos_idx, inv, batch, seq,
                                        n_heads, n_kv, head_dim)
            if done is not None:
                ctx.save_for_backward(cos, sin, pos_idx)
                ctx.dims = (rows, batch, seq, n_heads, n_kv, head_dim)
                return done
        _ext.require(qkv, "qkv", dtype=torch.float16, ndim=2)
        rows = qkv.shape[0]
        dev = qkv.device
        width = (n_heads + 2 * n_kv) * head_dim
        if qkv.shape[1] != width:
            raise ValueError(f"qkv width {qkv.shape[1]} != (n_heads + 2*n_kv) * head_dim = {width}")
        if head_dim % 2:
            raise ValueError("head_dim must be even")
        pos = as_index(pos_idx)
        if pos.numel() != rows:
            raise ValueError(f"pos_idx has {pos.numel()} entries for {rows} rows")
        lq, lv, code = _lora_pair(lora_q, lora_v)
        if lq is not None and tuple(lq.shape) != (rows, n_heads * head_dim):
            raise ValueError(f"lora_q shape {tuple(lq.shape)} != {(rows, n_heads * head_dim)}")
        if lv is not None and tuple(lv.shape) != (rows, n_kv * head_dim):
            raise ValueError(f"lora_v shape {tuple(lv.shape)} != {(rows, n_kv * head_dim)}")
        cos32 = _table(cos, seq, head_dim, "cos", dev)
        sin32 = _table(sin, seq, head_dim, "sin", dev)
        q = torch.empty((batch, n_heads, seq, head_dim), dtype=torch.float16, device=dev)
        k = torch.empty((batch, n_kv, seq, head_dim), dtype=torch.float16, device=dev)
        v = torch.empty((batch, n_kv, seq, head_dim), dtype=torch.float16, device=dev)
        slots = batch * seq
        # Positions without a token are zeroed by the kernel; with as many (distinct) tokens as
        # positions there are none.
        inv = inverse_map(pos, slots) if rows != slots else None
        if rows or inv is not None:
            _ext.call("soupk_rope_pack_fwd", _ext.ptr(qkv), _ext.ptr(lq), _ext.ptr(lv), code,
                      _ext.ptr(cos32), _ext.ptr(sin32), _ext.ptr(pos), _ext.ptr(inv), _ext.ptr(q),
                      _ext.ptr(k), _ext.ptr(v), rows, batch, seq, n_heads, n_kv, head_dim,
                      _ext.stream_of(qkv))
        ctx.save_for_backward(cos32, sin32, pos)
        ctx.dims = (rows, batch, seq, n_heads, n_kv, head_dim)
        return q, k, v

    @staticmethod
    def backward(ctx, grad_q, grad_k, grad_v):
        cos, sin, pos_idx = ctx.saved_tensors
        rows, batch, seq, n_heads, n_kv, head_dim = ctx.dims
        need_qkv, need_lq, need_lv = ctx.needs_input_grad[:3]
        if not (need_qkv or need_lq or need_lv):
            return (None,) * 11
        width = (n_heads + 2 * n_kv) * head_dim
        dqkv = _ext.host().rope_bwd(grad_q, grad_k, grad_v, cos, sin, pos_idx, batch, seq,
                                    n_heads, n_kv, head_dim)
        launched = dqkv is not None
        if not launched:
            dqkv = torch.empty((rows, width), dtype=torch.float16, device=pos_idx.device)
            grads = [g.to(torch.float16).contiguous() if g is not None else None
                     for g in (grad_q, grad_k, grad_v)]
        if rows and not launched:
            _ext.call("soupk_rope_pack_bwd", _ext.ptr(grads[0]), _ext.ptr(grads[1]),
                      _ext.ptr(grads[2]), _ext.ptr(cos), _ext.ptr(sin), _ext.ptr(pos_idx),
                      _ext.ptr(dqkv), rows, batch, seq, n_heads, n_kv, head_dim,
                      _ext.stream_of(dqkv))
        q_cols = n_heads * head_dim
        v_start = (n_heads + n_kv) * head_dim
        return ((dqkv if need_qkv else None),
                (dqkv[:, :q_cols] if need_lq else None),
                (dqkv[:, v_start:] if need_lv else None),
                None, None, None, None, None, None, None, None)


def rope_pack(qkv, lora_q, lora_v, cos, sin, pos_idx, batch, seq, n_heads, n_kv, head_dim):
    return RopePack.apply(qkv.contiguous(),
                          lora_q.contiguous() if lora_q is not None else None,
                          lora_v.contiguous() if lora_v is not None else None,
                          cos.contiguous(), sin.contiguous(), pos_idx, batch, seq,
                          n_heads, n_kv, head_dim)


def rope_pack_tokens(qkv, lora_q, lora_v, cos, sin, pos_idx, batch, seq, n_heads, n_kv,
                     head_dim):
    """The RoPE pack forward without the scatter: fp16 [rows, (n_heads + 2*n_kv) * head_dim] in
    qkv's own token-major layout -- q + lora_q rotated, k rotated, v + lora_v -- with the same
    arithmetic as RopePack (bit-identical values), for the varlen attention, which reads the
    real tokens where they are (no padded layout, no zero rows).  head_dim 128.  A token whose
    position lies outside [0, batch*seq) gets a row of zeros.  Not differentiable by itself:
    attention.RopeAttention carries its backward (fused into the attention backward)."""
    if head_dim == 128:
        out = _ext.host().rope_tokens(qkv, lora_q, lora_v, cos, sin, pos_idx, batch, seq, n_heads,
                                      n_kv)
        if out is not None:
            return out, cos, sin, pos_idx
    _ext.require(qkv, "qkv", dtype=torch.float16, ndim=2)
    rows = qkv.shape[0]
    dev = qkv.device
    width = (n_heads + 2 * n_kv) * head_dim
    if qkv.shape[1] != width:
        raise ValueError(f"qkv width {qkv.shape[1]} != (n_heads + 2*n_kv) * head_dim = {width}")
    if head_dim != 128:
        raise ValueError("rope_pack_tokens handles head_dim 128 (use RopePack otherwise)")
    pos = as_index(pos_idx)
    if pos.numel() != rows:
        raise ValueError(f"pos_idx has {pos.numel()} entries for {rows} rows")
    lq, lv, code = _lora_pair(lora_q, lora_v)
    if lq is not None and tuple(lq.shape) != (rows, n_heads * head_dim):
        raise ValueError(f"lora_q shape {tuple(lq.shape)} != {(rows, n_heads * head_dim)}")
    if lv is not None and tuple(lv.shape) != (rows, n_kv * head_dim):
        raise ValueError(f"lora_v shape {tuple(lv.shape)} != {(rows, n_kv * head_dim)}")
    cos32 = _table(cos, seq, head_dim, "cos", dev)
    sin32 = _table(sin, seq, head_dim, "sin", dev)
    out = torch.empty((rows, width), dtype=torch.float16, device=dev)
    if rows:
        _ext.call("soupk_rope_pack_tokens", _ext.ptr(qkv), _ext.ptr(lq),
                  _ext.ptr(lv), code, _ext.ptr(cos32), _ext.ptr(sin32), _ext.ptr(pos),
                  _ext.ptr(out), rows, batch, seq, n_heads, n_kv, head_dim, _ext.stream_of(out))
    return out, cos32, sin32, pos


def qk_norm_rope(qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos_idx, batch, seq, n_heads,
                 n_kv, head_dim, eps=1e-6):
    """rope_pack_tokens for models that normalise queries and keys per head: the q|k|v rows
    [M, (n_heads + 2*n_kv) * head_dim] with every query and key head (after its LoRA delta)
    RMS-normalised over head_dim, multiplied by q_weight or k_weight [head_dim] and rotated, the
    value heads with their delta; in the rows' type (fp16 or bf16), fp32 inside with one rounding.
    Differentiable in qkv, the deltas and the weights.

    lora_q [M, n_heads*head_dim] / lora_v [M, n_kv*head_dim]: None, the rows' type or fp32.  cos,
    sin, pos_idx, batch, seq as rope_pack_tokens; head_dim a multiple of 16 up to 256.  A token
    whose position lies outside [0, batch*seq) gets a row of zeros (and passes no gradient)."""
    tensors = (qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos_idx)
    if has_torch_function(tensors):
        return handle_torch_function(qk_norm_rope, tensors, *tensors, batch, seq, n_heads, n_kv, head_dim,
                                     eps)
    done = _ext.host().qk_norm_rope(qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos_idx, batch,
                                    seq, n_heads, n_kv, head_dim, eps)
    if done is not None:
        return done
    _ext.refuse_dispatching(*tensors)
    _ext.require(qkv, "qkv", ndim=2)
    _ext.dtype_code(qkv, "qkv", (torch.float16, torch.bfloat16))
    rows, dev = qkv.shape[0], qkv.device
    if n_heads <= 0 or n_kv < 0 or head_dim <= 0 or head_dim % 16 or head_dim > 256:
        raise ValueError(f"qk_norm_rope takes head dims that are multiples of 16 up to 256 and at "
                         f"least one query head, got {n_heads}, {n_kv} heads of {head_dim}")
    width = (n_heads + 2 * n_kv) * head_dim
    if qkv.shape[1] != width:
        raise ValueError(f"qkv width {qkv.shape[1]} != (n_heads + 2*n_kv) * head_dim = {width}")
    deltas = []
    for t, name, heads in ((lora_q, "lora_q", n_heads), (lora_v, "lora_v", n_kv)):
        if t is not None:
            if not isinstance(t, torch.Tensor) or t.device != dev:
                raise ValueError(f"{name} must be a tensor on {dev}")
            if t.dtype not in (qkv.dtype, torch.float32):
                raise TypeError(f"{name} must be {qkv.dtype} or torch.float32, got {t.dtype}")
            if tuple(t.shape) != (rows, heads * head_dim):
                raise ValueError(f"{name} shape {tuple(t.shape)} != {(rows, heads * head_dim)}")
            t = t.contiguous()
        deltas.append(t)
    if any(t is not None and t.dtype == torch.float32 for t in deltas):
        deltas = [None if t is None else t.float() for t in deltas]     # (one type for both)
    weights = []
    for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if not isinstance(t, torch.Tensor) or t.device != dev or tuple(t.shape) != (head_dim,) or \
                not t.dtype.is_floating_point:
            raise ValueError(f"{name} must be a floating-point tensor of {head_dim} on {dev}")
        weights.append(t.float().contiguous())
    if not isinstance(pos_idx, torch.Tensor) or pos_idx.device != dev or pos_idx.dim() != 1 or \
            pos_idx.numel() != rows or pos_idx.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"pos_idx must be {rows} integer positions on {dev}")
    if batch < 0 or seq < 0 or batch * seq >= 1 << 31:
        raise ValueError(f"batch ({batch}) and seq ({seq}) must span fewer than 2^31 positions")
    eps = _ext.number(eps, "eps")
    if not 0.0 <= eps <= 3e38:
        raise ValueError(f"eps must be a non-negative number, got {eps}")
    return _ext.checked(_ext.host().qk_norm_rope(
        qkv, *deltas, *weights, _table(cos, seq, head_dim, "cos", dev),
        _table(sin, seq, head_dim, "sin", dev), as_index(pos_idx), batch, seq, n_heads, n_kv,
        head_dim, eps))
