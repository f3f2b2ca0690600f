"""Dropout whose mask is drawn from a counter and never stored (testt_amd/csrc/dropout.hip).

    dropout(x, p, seed, call=0, rows=None, residual=None)   differentiable in x and residual
    CounterDropout(p, seed)                                 the same as a torch.nn.Dropout module

Element (r, c) of x, viewed as rows of its last dimension, is dropped when word c % 4 of
Philox4x32-10 (Salmon et al. 2011) at the counter (c / 4, R, call) under the key `seed` is below
p * 2^32; R is rows[r], or r itself.  The draw depends on nothing else -- not on the batch's shape,
nor on what was drawn before -- so the backward redraws it instead of reading a mask, tokens kept
without their padding draw what they would draw in the padded layout (rows = the padded positions),
and a step can be repeated.  torch's own dropout draws from the generator's state and keeps a byte
per element (the reference's path, solution/model.py:195-206)."""

import torch
from torch.overrides import handle_torch_function, has_torch_function

from . import _ext


def _check_p(p):
    p = _ext.number(p, "p")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    return p


def _check_word(v, name):
    if isinstance(v, bool) or not isinstance(v, int):
        raise TypeError(f"{name} must be an int, got {type(v).__name__}")
    if not 0 <= v < 1 << 64:
        raise ValueError(f"{name} must lie in [0, 2^64), got {v}")


def _check_seed(seed, device):
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a seed tensor must be one int64 on {device}, got {seed.dtype} "
                             f"{tuple(seed.shape)} on {seed.device}")
    else:
        _check_word(seed, "seed")


def dropout(x, p, seed, call=0, rows=None, residual=None):
    """residual + x with each element dropped with probability p and the others divided by 1 - p
    (without `residual`: that product alone), in residual's or x's type.

    x: fp16, bf16 or fp32, any shape, its last dimension the columns; p in [0, 1] (in steps of
    2^-32); seed: an int in [0, 2^64), or an int64 device tensor of one element that a captured
    graph reads on each replay; call: an int in [0, 2^64) that tells draws of one seed apart (a
    step's or layer's number); rows: int64, the row number in [0, 2^32) that each row draws as;
    residual: x's shape, x's type or fp32.  The sum is rounded once.  p = 1 gives the residual (or
    zeros) exactly, whatever x holds."""
    if has_torch_function((x, seed, rows, residual)):
        return handle_torch_function(dropout, (x, seed, rows, residual), x, p, seed, call, rows, residual)
    done = _ext.host().dropout(x, p, seed, call, rows, residual)
    if done is not None:
        return done
    _ext.refuse_dispatching(x, seed, rows, residual)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"x must be a HIP device tensor (got device {x.device}); the soupk kernels "
                         "have no CPU path")
    _ext.dtype_code(x, "x")
    p = _check_p(p)
    _check_seed(seed, x.device)
    _check_word(call, "call")
    if x.dim() and x.shape[-1] > 1 << 32:
        raise ValueError(f"x has {x.shape[-1]} columns, at most 2^32 are drawn for")
    if rows is not None:
        _ext.require(rows, "rows", dtype=torch.int64, device=x.device)
        n_rows = x.shape[:-1].numel() if x.dim() else 1
        if rows.numel() != n_rows:
            raise ValueError(f"rows holds {rows.numel()} numbers for {n_rows} rows")
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != x.shape or \
                residual.device != x.device:
            raise ValueError(f"residual must be a tensor of x's shape {tuple(x.shape)} on "
                             f"{x.device}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"residual must be {x.dtype} or torch.float32, got {residual.dtype}")
        residual = residual.contiguous()
    return _ext.checked(_ext.host().dropout(x.contiguous(), p, seed, call, rows, residual))


class CounterDropout(torch.nn.Dropout):
    """dropout() as a module: in training mode each forward draws under `seed` with the next call
    number (`self.call`, which may be set, e.g. to repeat a step); in eval mode, or with p = 0, x
    itself.  As the LoRA dropout of a layer or model of this package (it is a torch.nn.Dropout) it
    runs on the real tokens' rows alone and draws at their padded positions.

    The seed has no default: modules of one seed draw the same mask at the same positions, so those that
    are to draw independently (of two projections, of the layers, of data-parallel ranks) get seeds of
    their own.
    A forward that is run again inside a backward (activation checkpointing) raises: it would draw with
    another call number than the first run did; such a program calls dropout() with the step's number."""

    def __init__(self, p=0.5, seed=None):
        super().__init__(_check_p(p))
        if seed is None:
            raise TypeError("CounterDropout needs a seed of its own: modules of one seed draw the same mask")
        if not isinstance(seed, torch.Tensor):
            _check_word(seed, "seed")
        self.seed = seed
        self.call = 0

    def rows(self, x, rows):
        """forward(x) for rows that stand at the positions `rows`."""
        if not self.training or self.p == 0.0:
            return x
        if torch._C._current_graph_task_id() != -1:     # (this thread is inside a backward)
            raise RuntimeError("CounterDropout was called inside a backward pass (a checkpointed "
                               "forward?), where its call number is not the first run's; use "
                               "dropout.dropout() with a call number of the program's own")
        out = dropout(x, self.p, self.seed, self.call, rows)
        self.call += 1
        return out

    def forward(self, x):
        return self.rows(x, None)

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}, call={self.call}"
