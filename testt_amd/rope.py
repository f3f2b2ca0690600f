"""Q/K/V assembly for attention on gfx950: LoRA add + rotary embedding + scatter to the padded
layout.  Drop-in for solution/rope.py.

The fused q/k/v GEMM output (fp16, unpadded tokens) is read once per token by
testt_amd/csrc/rope_pack.hip, which adds the LoRA outputs in fp32, rotates q and k in fp32 and
writes fp16 q/k/v directly into [batch, heads, seq, head_dim] at the token's padded position,
the layout SDPA takes; padded positions with no token are zeroed by the same launch.  Backward
is the transposed rotation, gathering per token and writing the fp16 gradient of the q/k/v GEMM
output; the LoRA branches get views of the same buffer.

For generation: tables scaled for long contexts (rotary_tables), the rotation by itself, of part of a
head and in either layout (rotary), and the same step as above into a paged key-value cache
(rope_append), in testt_amd/csrc/rotary.hip.
"""

import math
from collections.abc import Mapping

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


# --------------------------------------------------------------------------------------------
# Rotary positions in either layout, of part of a head, scaled for long contexts; new tokens into
# a paged cache (csrc/rotary.hip)

_SCALINGS = {"default": 0, "linear": 1, "dynamic": 2, "yarn": 3}     # SOUPK_ROPE_*
_NO_GRAD = ("{} has no backward for {}: call it under torch.no_grad(), or detach what wants a "
            "gradient")


def refuse_grad(operator, *named):
    """Raises for a tensor that would want a gradient of an operator that gives none."""
    for t, name in named:
        if isinstance(t, torch.Tensor) and \
                (torch.is_grad_enabled() and t.requires_grad
                 or torch.autograd.forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(_NO_GRAD.format(operator, name))


def _positive(scaling, key, default=None):
    value = scaling.get(key)
    if value is None:
        value = default
    if value is None:
        raise ValueError(f"rope scaling {scaling.get('rope_type')!r} needs {key!r}")
    return _ext.number(value, key)


# What a scaling of each kind may say: the kind, the base, and a model's trained length where it has no part in
# the frequencies.
_EVERY_SCALING = ("rope_type", "type", "rope_theta", "original_max_position_embeddings")
_SCALING_KEYS = {"default": (), "linear": ("factor",), "dynamic": ("factor",),
                 "yarn": ("factor", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim",
                          "truncate")}


def _check_scaling(scaling):
    """The kind of a rope scaling; raises for a key that would be passed over."""
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in _SCALINGS:
        raise ValueError(f"rope scaling must be one of {', '.join(_SCALINGS)}, got {kind!r} (other "
                         "schemes: pass their frequencies as inv_freq)")
    if scaling.get("partial_rotary_factor") not in (None, 1):
        raise ValueError("partial_rotary_factor is not read: multiply the head dim by it for rotary_dim, and leave "
                         "it out of scaling")
    for key, value in scaling.items():
        if value is not None and key not in (*_EVERY_SCALING, *_SCALING_KEYS[kind], "partial_rotary_factor"):
            raise ValueError(f"rope scaling {kind!r} does not read {key!r}: leave it out, or pass frequencies "
                             "as inv_freq")
    return kind


def rotary_tables(seq, rotary_dim, theta=None, scaling=None, inv_freq=None, device="cuda"):
    """(cos, sin) fp32 [seq, rotary_dim / 2] of positions 0 .. seq - 1, for rotary() and
    rope_append(): pair i turns by theta^(-2 i / rotary_dim) a position (theta: scaling's rope_theta, or
    10000, unless given).  The angles are formed in 64 bits, so far positions keep their places (in
    fp32 an angle at position 2^20 is 0.03 rad off).

    scaling: None or a dict in the form of transformers' `rope_scaling`, for contexts longer than the
    trained one -- rope_type "default", "linear" (factor), "dynamic" (factor,
    original_max_position_embeddings, which transformers leaves to the configuration's
    max_position_embeddings; takes effect where seq exceeds it) or "yarn" (those two and, optionally,
    beta_fast, beta_slow, attention_factor, mscale, mscale_all_dim, truncate).  A key that its kind does
    not read raises.  inv_freq: rotary_dim / 2 frequencies on the host (numbers, or a CPU tensor) in
    place of theta and scaling.  rotary_dim: even, at most 256.  The layer's own tables [seq, head_dim]
    hold every column twice: their first half (cos[:, :head_dim // 2]) is this form."""
    if scaling is None and inv_freq is None and isinstance(device, str) and device == "cuda":
        done = _ext.host().rotary_tables(seq, rotary_dim, 1e4 if theta is None else theta, 0, 1.0, 1.0, 32.0, 1.0,
                                         1.0, None, -1)
        if done is not None:
            return done
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"rotary tables are made on a HIP device (got {device}); the soupk kernels "
                         "have no CPU path")
    for v, name in ((seq, "seq"), (rotary_dim, "rotary_dim")):
        if isinstance(v, bool) or not isinstance(v, int):
            raise TypeError(f"{name} must be an int, got {type(v).__name__}")
    if not 0 <= seq < 1 << 31:
        raise ValueError(f"seq must lie in [0, 2^31), got {seq}")
    if not 2 <= rotary_dim <= 256 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and lie in [2, 256], got {rotary_dim}")
    if scaling is not None and not isinstance(scaling, Mapping):
        raise TypeError(f"scaling must be None or a dict, got {type(scaling).__name__}")
    told = None if scaling is None else scaling.get("rope_theta")
    if theta is None:
        theta = 1e4 if told is None else told
    elif told is not None and _ext.number(theta, "theta") != _ext.number(told, "rope_theta"):
        raise ValueError(f"theta {theta} is not scaling's rope_theta {told}: pass one of them")
    theta = _ext.number(theta, "theta")
    if not 1.0 < theta <= 1e30:
        raise ValueError(f"theta must lie in (1, 1e30], got {theta}")
    kind, factor, original, fast, slow, gain = "default", 1.0, 1.0, 32.0, 1.0, 1.0
    if inv_freq is not None:
        if scaling is not None:
            raise ValueError("inv_freq takes the place of theta and scaling: pass one of them")
        if isinstance(inv_freq, torch.Tensor):
            if inv_freq.device.type != "cpu":
                raise ValueError(f"inv_freq must be on the host, got {inv_freq.device}")
            inv_freq = inv_freq.detach().double().tolist()
        inv_freq = tuple(float(f) for f in inv_freq)
        if len(inv_freq) != rotary_dim // 2 or not all(abs(f) <= 1e6 for f in inv_freq):
            raise ValueError(f"inv_freq must hold {rotary_dim // 2} frequencies of at most 1e6 rad")
    elif scaling is not None:
        kind = _check_scaling(scaling)
        if kind != "default":
            factor = _positive(scaling, "factor")
            if not 1.0 <= factor <= 1e6:
                raise ValueError(f"factor must lie in [1, 1e6], got {factor}")
        if kind in ("dynamic", "yarn"):
            original = _positive(scaling, "original_max_position_embeddings")
            if not 1.0 <= original <= 1 << 31:
                raise ValueError(f"original_max_position_embeddings must lie in [1, 2^31], got {original}")
        if kind == "yarn":
            fast, slow = _positive(scaling, "beta_fast", 32.0), _positive(scaling, "beta_slow", 1.0)
            if not 0.0 < slow <= fast <= 1e6:
                raise ValueError(f"0 < beta_slow <= beta_fast <= 1e6 is needed, got {slow}, {fast}")
            gain = _yarn_gain(scaling, factor)
            truncate = scaling.get("truncate")
            if not isinstance(truncate, (bool, type(None))):
                raise TypeError(f"truncate must be True or False, got {truncate!r}")
            if truncate is False:
                inv_freq = _yarn_between(rotary_dim, theta, factor, original, fast, slow)
    index = device.index if device.index is not None else torch.cuda.current_device()
    return _ext.checked(_ext.host().rotary_tables(seq, rotary_dim, theta, _SCALINGS[kind], factor,
                                                  original, fast, slow, gain, inv_freq, index))


def _yarn_between(dim, theta, factor, original, fast, slow):
    """YaRN's frequencies where the ramp begins and ends between pairs (csrc/rotary.hip widens it to whole ones)."""
    low, high = (dim * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(theta))
                 for turns in (fast, slow))
    low, high = max(low, 0.0), min(high, dim - 1.0)
    freq = []
    for i in range(dim // 2):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        f = theta ** (-2.0 * i / dim)
        freq.append(f / factor * ramp + f * (1.0 - ramp))
    return tuple(freq)


def _yarn_gain(scaling, factor):
    """What the cosines and sines are multiplied by: attention_factor, or 0.1 m ln(factor) + 1 of
    mscale over that of mscale_all_dim, or of m = 1."""
    def of(m):
        return 0.1 * m * math.log(factor) + 1.0

    gain = scaling.get("attention_factor")
    if gain is None:
        m, every = scaling.get("mscale"), scaling.get("mscale_all_dim")
        gain = of(float(m)) / of(float(every)) if m and every else of(1.0)
    gain = _ext.number(gain, "attention_factor")
    if not abs(gain) <= 1e30:
        raise ValueError(f"attention_factor must be a number of at most 1e30, got {gain}")
    return gain


def _half_table(t, name, head_dim, device):
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be torch.float32, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] < 1 or 2 * t.shape[1] > head_dim:
        raise ValueError(f"{name} must be [positions, R / 2] with R at most the head dim {head_dim}, "
                         f"got {tuple(t.shape)}")


def _half_tables(cos, sin, head_dim, device):
    _half_table(cos, "cos", head_dim, device)
    _half_table(sin, "sin", head_dim, device)
    if cos.shape != sin.shape:
        raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} differ")
    if cos.stride() != sin.stride() or (cos.stride(1) != 1 and cos.shape[1] > 1):
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin


def rotary(x, cos, sin, pos, interleaved=False):
    """x [M, heads, D] with the leading R = 2 * cos.shape[1] elements of every head turned by the angles
    of position pos[m], the others as they are; in x's type (fp16, bf16 or fp32), fp32 inside,
    differentiable in x.

    Pairs are (i, i + R/2) (transformers' rotate_half) or, interleaved, (2 i, 2 i + 1).  x: any token
    and head strides, a head's elements adjacent (query columns of q|k|v rows, viewed as heads).
    cos, sin: fp32 [positions, R/2] (rotary_tables(), or the first half of the layer's tables), any
    row stride.  pos: int64 or int32 [M]; a token whose position lies outside the tables gets zeros
    (and passes no gradient)."""
    tensors = (x, cos, sin, pos)
    if has_torch_function(tensors):
        return handle_torch_function(rotary, tensors, *tensors, interleaved)
    done = _ext.host().rotary(x, cos, sin, pos, interleaved)
    if done is not None:
        return done
    _ext.refuse_dispatching(*tensors)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"x must be a HIP device tensor (got device {x.device}); the soupk kernels "
                         "have no CPU path")
    _ext.dtype_code(x, "x")
    if x.dim() != 3 or not 1 <= x.shape[1] <= 1 << 16 or not 2 <= x.shape[2] <= 1 << 16:
        raise ValueError(f"x must be [tokens, heads, head_dim], got {tuple(x.shape)}")
    cos, sin = _half_tables(cos, sin, x.shape[2], x.device)
    refuse_grad("rotary", (cos, "cos"), (sin, "sin"))
    if not isinstance(pos, torch.Tensor) or pos.device != x.device or pos.dim() != 1 or \
            pos.numel() != x.shape[0] or pos.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"pos must be {x.shape[0]} integer positions on {x.device}")
    if x.stride(2) != 1:
        x = x.contiguous()
    return _ext.checked(_ext.host().rotary(x, cos, sin, as_index(pos), bool(interleaved)))


def check_pages(k_pages, v_pages, block_table, lengths, cu_seqlens, rows):
    """(n_kv, page_size, head_dim) of a paged cache and its sequences' int32 tensors, or an error."""
    _ext.refuse_dispatching(k_pages, v_pages, block_table, lengths, cu_seqlens)
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a HIP device tensor (got device {t.device}); the soupk "
                             "kernels have no CPU path")
        _ext.dtype_code(t, name, (torch.float16, torch.bfloat16))
        if t.dim() != 4 or 0 in t.shape:
            raise ValueError(f"{name} must be [pages, n_kv, page_size, head_dim], got {tuple(t.shape)}")
        _, n_kv, page, d = t.shape
        if t.stride()[1:] != (page * d, d, 1) or (t.shape[0] > 1 and t.stride(0) < n_kv * page * d):
            raise ValueError(f"{name} must hold each page's elements adjacent, got strides {t.stride()}")
        if t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) % 8):
            raise ValueError(f"{name}'s pages must be aligned to 16 bytes")
    if v_pages.dtype != k_pages.dtype:
        raise TypeError(f"v_pages must be {k_pages.dtype} as k_pages, got {v_pages.dtype}")
    if v_pages.shape != k_pages.shape or \
            v_pages.device != k_pages.device or \
            (k_pages.shape[0] > 1 and v_pages.stride(0) != k_pages.stride(0)):
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must agree in "
                         "shape, strides and device")
    if d % 16 or d > 256:
        raise ValueError(f"head_dim must be a multiple of 16 up to 256, got {d}")
    if n_kv > 1 << 16 or page >= 1 << 31 or k_pages.shape[0] >= 1 << 31:
        raise ValueError(f"too many pages, key heads or slots: {tuple(k_pages.shape)}")
    dev = k_pages.device
    _ext.require(lengths, "lengths", dtype=torch.int32, ndim=1, device=dev)
    _ext.require(block_table, "block_table", dtype=torch.int32, ndim=2, device=dev)
    batch = lengths.numel()
    if block_table.shape[0] != batch:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {batch} lengths")
    if block_table.shape[1] * page > 1 << 30:
        raise ValueError(f"block_table spans {block_table.shape[1]} pages of {page}, over 2^30 positions")
    if cu_seqlens is not None:
        _ext.require(cu_seqlens, "cu_seqlens", dtype=torch.int32, ndim=1, device=dev)
        if cu_seqlens.numel() != batch + 1:
            raise ValueError(f"cu_seqlens must hold {batch + 1} bounds, got {cu_seqlens.numel()}")
    elif rows != batch:
        raise ValueError(f"{rows} rows for {batch} sequences: without cu_seqlens each has one new token")
    return n_kv, page, d


def rope_append(qkv, lora_q, lora_v, cos, sin, k_pages, v_pages, block_table, lengths,
                cu_seqlens=None, interleaved=False):
    """The new tokens' step between the q|k|v projection and the attention of a decoding layer:
    returns the queries [M, n_heads * D], rotated with their LoRA delta, and writes the rotated keys
    and the values with theirs into a paged cache (attention.paged_attention reads it).

    qkv: fp16 or bf16 [M, (n_heads + 2 * n_kv) * D] in the token-major layout of rope_pack_tokens
    (whose bits the queries, keys and values have); lora_q, lora_v: None, the rows' type or fp32.
    cos, sin: as rotary(), or None where the rows are rotated already (qk_norm_rope's).
    k_pages, v_pages: [pages, n_kv, page_size, D] of qkv's type, written in place.  block_table:
    int32 [batch, pages of a sequence]; lengths: int32 [batch], each sequence's tokens with the new
    ones; cu_seqlens: int32 [batch + 1], where each one's new tokens start in qkv (None: one each).
    Token i of a sequence's n new ones stands at t = length - n + i: its angle, and slot
    t % page_size of page block_table[b, t // page_size].  A token without a place -- no sequence, t
    outside [0, positions) or the block table, a page outside [0, pages) -- gets a row of zeros and is
    written nowhere, so a captured graph's padding costs nothing: give it length 0.

    No gradient is given.  Two sequences may share pages that neither writes."""
    tensors = (qkv, lora_q, lora_v, cos, sin, k_pages, v_pages, block_table, lengths, cu_seqlens)
    if has_torch_function(tensors):
        return handle_torch_function(rope_append, tensors, *tensors, interleaved)
    done = _ext.host().rope_append(*tensors, interleaved)
    if done is not None:
        return done
    _ext.refuse_dispatching(*tensors)
    refuse_grad("rope_append", (qkv, "qkv"), (lora_q, "lora_q"), (lora_v, "lora_v"), (cos, "cos"),
                (sin, "sin"), (k_pages, "k_pages"), (v_pages, "v_pages"))
    _ext.require(qkv, "qkv", ndim=2)
    rows, dev = qkv.shape[0], qkv.device
    n_kv, _, d = check_pages(k_pages, v_pages, block_table, lengths, cu_seqlens, rows)
    if qkv.dtype != k_pages.dtype or k_pages.device != dev:
        raise TypeError(f"qkv ({qkv.dtype} on {dev}) must have the pages' type and device "
                        f"({k_pages.dtype} on {k_pages.device})")
    n_heads = qkv.shape[1] // d - 2 * n_kv
    if qkv.shape[1] % d or not 1 <= n_heads <= 1 << 16:
        raise ValueError(f"qkv width {qkv.shape[1]} is no (n_heads + 2 * {n_kv}) * {d}")
    deltas = []
    for t, name, heads in ((lora_q, "lora_q", n_heads), (lora_v, "lora_v", n_kv)):
        if t is not None:
            if not isinstance(t, torch.Tensor) or t.device != dev:
                raise ValueError(f"{name} must be a tensor on {dev}")
            if t.dtype not in (qkv.dtype, torch.float32):
                raise TypeError(f"{name} must be {qkv.dtype} or torch.float32, got {t.dtype}")
            if tuple(t.shape) != (rows, heads * d):
                raise ValueError(f"{name} shape {tuple(t.shape)} != {(rows, heads * d)}")
            t = t.contiguous()
        deltas.append(t)
    if any(t is not None and t.dtype == torch.float32 for t in deltas):
        deltas = [None if t is None else t.float() for t in deltas]     # (one type for both)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin are given together, or neither")
    if cos is not None:
        cos, sin = _half_tables(cos, sin, d, dev)
    return _ext.checked(_ext.host().rope_append(qkv, *deltas, cos, sin, k_pages, v_pages, block_table,
                                                lengths, cu_seqlens, bool(interleaved)))
