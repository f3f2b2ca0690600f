"""Embedding lookup with a scale, and its gradient by sorted tokens
(testt_amd/csrc/embedding.hip).

    embedding(ids, table, scale=1.0, out_dtype=None, padding_idx=None)

The lookup writes the scaled rows in the output's type in one launch (the fp32 residual stream of
an fp16 table: what the model path takes).  The table's gradient is dense, in the table's type: the
tokens are sorted by id, stably, and every row's gradient is summed over its tokens in their order
in fp32 and rounded once -- the same bits every time, unlike sums by atomics."""

import torch
from torch.overrides import handle_torch_function, has_torch_function

from . import _ext


def embedding(ids, table, scale=1.0, out_dtype=None, padding_idx=None):
    """table[ids] * scale, [*ids.shape, H], in out_dtype (the table's type, the default, or fp32);
    fp32 inside, rounded once.  Differentiable in `table`.

    ids: int64 or int32 of any shape; an id outside [0, V) gives a row of zeros and no gradient.
    table: contiguous fp16, bf16 or fp32 [V, H].  padding_idx: a row that gets no gradient (its
    values are looked up like any other's), as torch's."""
    if has_torch_function((ids, table)):
        return handle_torch_function(embedding, (ids, table), ids, table, scale, out_dtype, padding_idx)
    if padding_idx is None and (out_dtype is None or out_dtype is torch.float32):
        done = _ext.host().embedding(ids, table, scale, out_dtype is torch.float32, -1)
        if done is not None:
            return done
    _ext.refuse_dispatching(ids, table)
    _ext.require(table, "table", ndim=2)
    _ext.dtype_code(table, "table")
    if not isinstance(ids, torch.Tensor):
        raise TypeError(f"ids must be a tensor, got {type(ids).__name__}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be torch.int64 or torch.int32, got {ids.dtype}")
    if ids.device != table.device:
        raise ValueError(f"ids are on {ids.device}, expected {table.device}")
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in (table.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {table.dtype} or torch.float32, got {out_dtype}")
    if padding_idx is not None:
        if not -table.shape[0] <= padding_idx < table.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} lies outside the table of "
                             f"{table.shape[0]} rows")
        padding_idx = int(padding_idx) % table.shape[0]
    return _ext.checked(_ext.host().embedding(
        ids.to(torch.int64).contiguous(), table, _ext.number(scale, "scale"), out_dtype is torch.float32,
        -1 if padding_idx is None else padding_idx))


def supported(table):
    """A table that embedding() takes and no subclass has a say in."""
    return (type(table) in (torch.Tensor, torch.nn.Parameter) and table.is_cuda and table.dim() == 2 and table.dtype in _ext.DTYPES
            and table.is_contiguous())
