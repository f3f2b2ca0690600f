"""Refusals of the generating program's operators, on the CPU: Python arguments before a launch, and the C
entry points' own checks."""

import ctypes

import pytest
import torch

from testt_amd import _ext, attention, head, rope

H, I32 = torch.float16, torch.int32


def _cache(d=16):
    return torch.zeros(3, 1, 4, d, dtype=H), torch.zeros(2, 2, dtype=I32), torch.ones(2, dtype=I32)


def test_cpu_tensors_are_refused():
    pages, table, lengths = _cache()
    cos = torch.zeros(8, 8)
    with pytest.raises(ValueError, match="no CPU path"):
        rope.rotary_tables(8, 16, device="cpu")
    with pytest.raises(ValueError, match="no CPU path"):
        rope.rotary(torch.zeros(2, 1, 16), cos, cos, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="no CPU path"):
        rope.rope_append(torch.zeros(2, 48, dtype=H), None, None, cos, cos, pages, pages, table, lengths)
    with pytest.raises(ValueError, match="no CPU path"):
        attention.paged_attention(torch.zeros(2, 16, dtype=H), pages, pages, table, lengths)
    with pytest.raises(ValueError, match="no CPU path"):
        head.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))


@pytest.mark.parametrize("kw,error,match", [
    (dict(seq=-1), ValueError, "seq"), (dict(seq=True), TypeError, "seq"),
    (dict(seq=2.0), TypeError, "seq"), (dict(rotary_dim=7), ValueError, "even"),
    (dict(rotary_dim=258), ValueError, "even"), (dict(rotary_dim=0), ValueError, "even"),
    (dict(theta=1.0), ValueError, "theta"), (dict(theta=float("nan")), ValueError, "theta"),
    (dict(scaling={"rope_type": "other"}), ValueError, "inv_freq"),
    (dict(scaling="linear"), TypeError, "dict"),
    (dict(scaling={"rope_type": "linear"}), ValueError, "factor"),
    (dict(scaling={"rope_type": "linear", "factor": 0.5}), ValueError, "factor"),
    (dict(scaling={"rope_type": "yarn", "factor": 2.0}), ValueError, "original"),
    (dict(scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 64,
                   "beta_fast": 1.0, "beta_slow": 2.0}), ValueError, "beta"),
    (dict(scaling={"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 64,
                   "attention_factor": float("inf")}), ValueError, "attention_factor"),
    (dict(inv_freq=[1.0] * 7), ValueError, "inv_freq"),
    (dict(inv_freq=[1.0] * 7 + [float("nan")]), ValueError, "inv_freq"),
    (dict(inv_freq=[1.0] * 8, scaling={"rope_type": "default"}), ValueError, "one of them"),
])
def test_tables_arguments(kw, error, match):
    args = dict(seq=8, rotary_dim=16)
    args.update(kw)
    with pytest.raises(error, match=match):
        rope.rotary_tables(**args)


class Seen(torch.Tensor):
    """A subclass with a protocol of its own."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        return func, args, kwargs


def seen(*shape):
    return torch.zeros(*shape).as_subclass(Seen)


def test_a_subclass_is_asked():
    pages, table, lengths = _cache()
    cos, pos = torch.zeros(8, 8), torch.zeros(2, dtype=torch.int64)
    for call, func in (
            (lambda: rope.rotary(seen(2, 1, 16), cos, cos, pos), rope.rotary),
            (lambda: rope.rotary(torch.zeros(2, 1, 16), cos, cos, seen(2)), rope.rotary),
            (lambda: rope.rope_append(torch.zeros(2, 48), None, None, cos, cos, seen(3, 1, 4, 16), pages, table,
                                      lengths), rope.rope_append),
            (lambda: attention.paged_attention(seen(2, 16), pages, pages, table, lengths),
             attention.paged_attention),
            (lambda: head.verify_drafts(seen(1, 2, 8), pos, cos), head.verify_drafts)):
        assert call()[0] is func


A = 4096       # an aligned address that is never read: every call below is refused before a launch
TABLES = (A, A, 8, 16, None, 1e4, 0, 1.0, 1.0, 32.0, 1.0, 1.0, None)
ROTARY = (A, 0, 16, 16, A, A, 8, 8, A, A, 2, 1, 16, 16, 0, 0, None)
APPEND = (A, None, None, 0, A, A, 8, 8, 16, 0, None, A, A, 2, 4, A, A, A, 8, 64, 4, 0, 2, 1, 1, 16, None)
PAGED = (A, 16, A, A, 8, 64, 4, A, 4, A, None, 2, A, 0, 2, 1, 1, 16, 0.25, A, 1 << 30, None)
VERIFY = (A, A, 1, A, A, None, A, A, 2, 3, 100, A, 1 << 20, None)


def but(args, **at):
    args = list(args)
    for k, v in at.items():
        args[int(k[1:])] = v
    return tuple(args)


BAD = [("soupk_rotary_tables", but(TABLES, _2=-1)), ("soupk_rotary_tables", but(TABLES, _3=15)),
       ("soupk_rotary_tables", but(TABLES, _3=258)), ("soupk_rotary_tables", but(TABLES, _5=1.0)),
       ("soupk_rotary_tables", but(TABLES, _6=4)), ("soupk_rotary_tables", but(TABLES, _6=1, _7=0.0)),
       ("soupk_rotary_tables", but(TABLES, _6=2, _8=0.0)),
       ("soupk_rotary_tables", but(TABLES, _6=3, _8=64.0, _10=64.0)),
       ("soupk_rotary_tables", but(TABLES, _11=float("nan"))), ("soupk_rotary_tables", but(TABLES, _0=A + 4)),
       ("soupk_rotary_tables", but(TABLES, _1=None)),
       # the rotation: type, sizes, strides, missing or odd addresses
       ("soupk_rotary", but(ROTARY, _1=3)), ("soupk_rotary", but(ROTARY, _10=-1)),
       ("soupk_rotary", but(ROTARY, _11=0)), ("soupk_rotary", but(ROTARY, _13=18)),
       ("soupk_rotary", but(ROTARY, _13=15)), ("soupk_rotary", but(ROTARY, _13=0)),
       ("soupk_rotary", but(ROTARY, _2=-16)), ("soupk_rotary", but(ROTARY, _0=A + 1)),
       ("soupk_rotary", but(ROTARY, _4=None)), ("soupk_rotary", but(ROTARY, _8=A + 4)),
       ("soupk_rotary", but(ROTARY, _9=None)),
       # the append
       ("soupk_rope_append", but(APPEND, _21=1)), ("soupk_rope_append", but(APPEND, _25=24)),
       ("soupk_rope_append", but(APPEND, _25=272)), ("soupk_rope_append", but(APPEND, _24=0)),
       ("soupk_rope_append", but(APPEND, _23=0)), ("soupk_rope_append", but(APPEND, _20=0)),
       ("soupk_rope_append", but(APPEND, _14=1 << 30)), ("soupk_rope_append", but(APPEND, _19=63)),
       ("soupk_rope_append", but(APPEND, _8=18)), ("soupk_rope_append", but(APPEND, _1=A, _3=2)),
       ("soupk_rope_append", but(APPEND, _11=None)), ("soupk_rope_append", but(APPEND, _12=None)),
       ("soupk_rope_append", but(APPEND, _16=None)), ("soupk_rope_append", but(APPEND, _15=None)),
       # the attention
       ("soupk_paged_attention", but(PAGED, _13=1)), ("soupk_paged_attention", but(PAGED, _17=24)),
       ("soupk_paged_attention", but(PAGED, _15=3, _16=2)), ("soupk_paged_attention", but(PAGED, _14=3)),
       ("soupk_paged_attention", but(PAGED, _4=0)), ("soupk_paged_attention", but(PAGED, _5=63)),
       ("soupk_paged_attention", but(PAGED, _5=68)), ("soupk_paged_attention", but(PAGED, _2=A + 8)),
       ("soupk_paged_attention", but(PAGED, _6=0)), ("soupk_paged_attention", but(PAGED, _8=1 << 30)),
       ("soupk_paged_attention", but(PAGED, _9=None)), ("soupk_paged_attention", but(PAGED, _7=None)),
       ("soupk_paged_attention", but(PAGED, _18=float("nan"))), ("soupk_paged_attention", but(PAGED, _20=64)),
       ("soupk_paged_attention", but(PAGED, _19=A + 8)), ("soupk_paged_attention", but(PAGED, _10=A, _11=0)),
       ("soupk_paged_attention", but(PAGED, _14=(1 << 23) + 1, _11=(1 << 23) + 1)),
       # the verification
       ("soupk_verify_drafts", but(VERIFY, _2=3)), ("soupk_verify_drafts", but(VERIFY, _8=-1)),
       ("soupk_verify_drafts", but(VERIFY, _9=-1)), ("soupk_verify_drafts", but(VERIFY, _10=0)),
       ("soupk_verify_drafts", but(VERIFY, _12=16)), ("soupk_verify_drafts", but(VERIFY, _0=None)),
       ("soupk_verify_drafts", but(VERIFY, _3=None)), ("soupk_verify_drafts", but(VERIFY, _4=None)),
       ("soupk_verify_drafts", but(VERIFY, _1=A + 1)), ("soupk_verify_drafts", but(VERIFY, _11=A + 4)),
       ("soupk_verify_drafts_workspace", (1 << 40, 100, A)), ("soupk_verify_drafts_workspace", (1, 100, None)),
       ("soupk_paged_attention_workspace", (1, 1, 2, 1, 16, 4, 4, None))]


@pytest.mark.parametrize("name,args", BAD)
def test_invalid_arguments_rejected_before_launch(name, args):
    with pytest.raises(_ext.SoupkError, match="status 1"):
        _ext.call(name, *args)


@pytest.mark.parametrize("name,args", [
    ("soupk_rotary_tables", but(TABLES, _0=None, _1=None, _2=0)), ("soupk_rotary", but(ROTARY, _0=None, _10=0)),
    ("soupk_rope_append", but(APPEND, _0=None, _22=0)),
    ("soupk_paged_attention", but(PAGED, _0=None, _10=A, _14=0)),
    ("soupk_verify_drafts", but(VERIFY, _0=None, _8=0))])
def test_empty_work_is_a_no_op(name, args):
    _ext.call(name, *args)


def test_workspaces():
    need = ctypes.c_int64()
    _ext.call("soupk_verify_drafts_workspace", 2, 151936, ctypes.addressof(need))
    assert need.value == 2 * 16 * -(-151936 // 1024)
    _ext.call("soupk_verify_drafts_workspace", 1, 1 << 24, ctypes.addressof(need))
    assert need.value <= 16 * 256
    _ext.call("soupk_paged_attention_workspace", 1, 1, 12, 2, 128, 8, 16, ctypes.addressof(need))
    assert 16 < need.value < 1 << 26
