"""New tokens into a paged cache, against 64 bits and bit for bit against the training path's rotation.

Tolerance: a sum with the delta, two products and a sum, each rounded to fp32, then one rounding to the type."""

import pytest
import torch

from oracle import generate as og
from testt_amd import rope, workloads

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, B, F = torch.float16, torch.bfloat16, torch.float32
I32 = torch.int32


def make(lengths, news, page, n_heads, n_kv, d, dtype, seed=0, spare=2, width=None, lora=None):
    """A cache of NaN pages in random order, qkv rows, deltas of type `lora`."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    width = max(need + [1]) if width is None else width
    order = torch.randperm(sum(need) + spare, generator=gen).tolist()
    table = [[order.pop() if i < n else -1 for i in range(width)] for n in need]
    n_pages = sum(need) + spare
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    m = cu[-1]
    qkv = torch.randn(m, (n_heads + 2 * n_kv) * d, generator=gen).to(dtype)
    lq = lv = None
    if lora is not None:
        lq = (0.1 * torch.randn(m, n_heads * d, generator=gen)).to(lora)
        lv = (0.1 * torch.randn(m, n_kv * d, generator=gen)).to(lora)
    pages = torch.full((2, n_pages, n_kv, page, d), float("nan")).to(dtype)
    return qkv, lq, lv, pages, table, cu


def dev_seqs(table, lengths, cu):
    return (torch.tensor(table, dtype=I32, device=DEV).reshape(len(lengths), len(table[0]) if table else 1),
            torch.tensor(lengths, dtype=I32, device=DEV),
            None if cu is None else torch.tensor(cu, dtype=I32, device=DEV))


def dev(*ts):
    return tuple(None if t is None else t.to(DEV) for t in ts)


def close(got, want, dtype, size):
    """size: a bound of the intermediate values' magnitude."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 8 * 2.0 ** -24 * size + 2.0 ** -25
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert bool(((got - want).abs() <= tol)[~want.isnan()].all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lengths,news,page,nh,nkv,d,r,dtype,lora", [
    ([5, 1, 17, 32], [1, 1, 1, 1], 16, 12, 2, 128, 128, H, H),
    ([5, 1, 17, 32], [1, 1, 1, 1], 16, 12, 2, 128, 128, H, F),
    ([7, 0, 40, 3], [3, 0, 40, 1], 5, 4, 4, 64, 32, B, None),
    ([9, 9], [2, 5], 1, 3, 1, 80, 20, B, B),
    ([300, 2], [300, 2], 24, 8, 8, 96, 96, H, None),
    ([130], [130], 64, 2, 1, 256, 256, B, F),
    ([21, 4], [4, 4], 8, 1, 1, 16, 2, H, H),
    ([700, 650, 800], [700, 650, 800], 128, 6, 3, 48, 48, B, None)])
def test_append(lengths, news, page, nh, nkv, d, r, dtype, lora, interleaved):
    qkv, lq, lv, pages, table, cu = make(lengths, news, page, nh, nkv, d, dtype, 3, lora=lora)
    cos, sin = (t.float() for t in og.rotary_tables(max(lengths), r))
    k, v = pages.to(DEV)
    version = k._version, v._version
    q = rope.rope_append(*dev(qkv, lq, lv, cos, sin), k, v, *dev_seqs(table, lengths, cu), interleaved)
    assert k._version > version[0] and v._version > version[1]
    want = og.rope_append(qkv, lq, lv, cos, sin, *pages, table, lengths, cu, interleaved)
    size = 3 * float(qkv.float().abs().max()) + 3
    for got, ref in zip((q, k, v), want):
        close(got, ref, dtype, size)
    if all(n == 1 for n in news):       # without bounds: one token each, the same bits
        k2, v2 = pages.to(DEV)
        q2 = rope.rope_append(*dev(qkv, lq, lv, cos, sin), k2, v2, *dev_seqs(table, lengths, None),
                              interleaved=interleaved)
        assert torch.equal(q, q2) and torch.equal(k.nan_to_num(9), k2.nan_to_num(9))
        assert torch.equal(v.nan_to_num(9), v2.nan_to_num(9))


def test_bits_of_the_training_path():
    """fp16, head dim 128: the bits of rope_pack_tokens, deltas included."""
    lengths, seq = (20, 9), 32
    qkv, lq, lv, pos = workloads.rope_inputs(lengths, seq, seed=4, device=DEV)
    cos, sin = workloads.rope_tables(seq, device=DEV)
    rows, _, _, _ = rope.rope_pack_tokens(qkv, lq, lv, cos, sin, pos, 2, seq, 12, 2, 128)
    k, v = torch.zeros(2, 5, 2, 8, 128, dtype=H, device=DEV)
    table = [[3, 0, 2], [4, 1, -1]]
    q = rope.rope_append(qkv, lq, lv, cos[:, :64], sin[:, :64], k, v, *dev_seqs(table, lengths, [0, 20, 29]))
    assert torch.equal(q, rows[:, :1536])
    for b, (lo, n) in enumerate(((0, 20), (20, 9))):
        for t in range(n):
            at = table[b][t // 8], slice(None), t % 8
            assert torch.equal(k[at].reshape(-1), rows[lo + t, 1536:1792])
            assert torch.equal(v[at].reshape(-1), rows[lo + t, 1792:])


def test_without_tables_rows_are_copied():
    qkv, lq, lv, pages, table, cu = make([6, 3], [4, 3], 4, 2, 1, 80, H, 5, lora=H)
    k, v = pages.to(DEV)
    q = rope.rope_append(*dev(qkv, None, None), None, None, k, v, *dev_seqs(table, [6, 3], cu))
    want = og.rope_append(qkv, None, None, None, None, *pages, table, [6, 3], cu)
    for got, ref in zip((q, k, v), want):
        close(got, ref, H, 0.0)


def test_tokens_without_a_place():
    """Before the sequence's start, beyond the tables, the block table or the pages, in no sequence: zeros, and
    nothing is written."""
    page, d = 4, 16
    lengths, news = [2, 9, 13, 8, 0, 5], [4, 1, 1, 2, 0, 2]
    table = [[0, -1, -1], [1, 2, 3], [4, 5, 6], [7, 99, 0], [8, 8, 8], [9, -1, 9]]
    cu = [0, 4, 5, 6, 8, 8, 10]
    gen = torch.Generator().manual_seed(6)
    qkv = torch.randn(13, 3 * d, generator=gen).to(H)        # three rows of no sequence
    cos, sin = (t.float() for t in og.rotary_tables(9, d))
    pages = torch.full((2, 10, 1, page, d), 7.0).to(H)
    k, v = pages.to(DEV)
    q = rope.rope_append(*dev(qkv, None, None, cos, sin), k, v, *dev_seqs(table, lengths, cu))
    want = og.rope_append(qkv, None, None, cos, sin, *pages, table, lengths, cu)
    for got, ref in zip((q, k, v), want):
        close(got, ref, H, 12.0)
    # 2 - 4 + 0, + 1 < 0; 12 beyond the tables; page 99; page -1; no sequence
    assert not bool(q[[0, 1, 5, 6, 7, 9, 10, 11, 12]].any()) and bool(q[[2, 3, 4, 8]].any(1).all())


@pytest.mark.parametrize("cu", [[0, 5, 3, 6], [-3, 2, 4, 6], [0, 2, 4, 99], [4, 4, 4, 4]])
def test_impossible_bounds_stay_inside(cu):
    """Bounds that do not ascend, or leave the rows: only memory of the cache's pages may be written."""
    gen = torch.Generator().manual_seed(7)
    qkv = torch.randn(6, 3 * 16, generator=gen).to(H).to(DEV)
    cos, sin = rope.rotary_tables(16, 16, device=DEV)
    k, v = torch.zeros(2, 4, 1, 4, 16, dtype=H, device=DEV)
    guard = torch.zeros(4, 1, 4, 16, dtype=H, device=DEV)
    q = rope.rope_append(qkv, None, None, cos, sin, k, v, *dev_seqs([[0], [1], [2]], [4, 4, 4], cu))
    assert q.shape == (6, 16) and not bool(guard.any()) and not bool(k[3].any())


def test_pages_of_one_buffer():
    """Keys and values of a page side by side: pages a stride apart; sizes past 2^31 elements."""
    page, n_kv, d = 16, 2, 128
    per = 2 * n_kv * page * d
    n = (1 << 31) // per + 3
    both = torch.empty(n, 2, n_kv, page, d, dtype=H, device=DEV)
    k, v = both[:, 0], both[:, 1]
    both[-2:] = 0
    both[:1] = 0
    gen = torch.Generator().manual_seed(8)
    qkv = torch.randn(2, 16 * d, generator=gen).to(H).to(DEV)
    cos, sin = rope.rotary_tables(64, d, device=DEV)
    rope.rope_append(qkv, None, None, cos, sin, k, v, *dev_seqs([[0, n - 1], [n - 2, -1]], [17, 16], None))
    want = qkv.view(2, 16, d)
    turned = rope.rotary(want[:, 12:14], cos, sin, torch.tensor([16, 15], device=DEV))
    assert torch.equal(both[n - 1, 0, :, 0], turned[0]) and torch.equal(both[n - 1, 1, :, 0], want[0, 14:])
    assert torch.equal(both[n - 2, 0, :, 15], turned[1]) and torch.equal(both[n - 2, 1, :, 15], want[1, 14:])
    assert not bool(both[0].any()) and not bool(both[n - 2, :, :, :15].any())


def test_many_sequences():
    """More than 64 and more than 64 * 64 bounds are searched in rounds."""
    for batch in (63, 64, 65, 200, 4200):
        news = [(i * 7) % 3 for i in range(batch)]
        lengths = [n + (i % 5) for i, n in enumerate(news)]
        qkv, _, _, pages, table, cu = make(lengths, news, 4, 1, 1, 16, H, batch)
        k, v = pages.to(DEV)
        q = rope.rope_append(*dev(qkv, None, None), None, None, k, v, *dev_seqs(table, lengths, cu))
        want = og.rope_append(qkv, None, None, None, None, *pages, table, lengths, cu)
        for got, ref in zip((q, k, v), want):
            close(got, ref, H, 0.0)


def test_refusals():
    k, v = torch.zeros(2, 4, 2, 4, 32, dtype=H, device=DEV)
    table, lengths, _ = dev_seqs([[0], [1]], [1, 1], None)
    qkv = torch.zeros(2, 7 * 32, dtype=H, device=DEV)
    cos, sin = rope.rotary_tables(4, 32, device=DEV)
    ok = dict(qkv=qkv, lora_q=None, lora_v=None, cos=cos, sin=sin, k_pages=k, v_pages=v, block_table=table,
              lengths=lengths)
    rope.rope_append(**ok)
    lora = torch.zeros(2, 96, dtype=H, device=DEV)
    for error, kw in [
            (TypeError, dict(qkv=qkv.bfloat16())), (ValueError, dict(qkv=qkv[:, :40].contiguous())),
            (ValueError, dict(qkv=qkv[:, :128].contiguous())), (ValueError, dict(qkv=qkv.t())),
            (ValueError, dict(qkv=qkv[:1])), (TypeError, dict(k_pages=k.float(), v_pages=v.float())),
            (ValueError, dict(k_pages=k[:, :1])), (ValueError, dict(k_pages=k[:2])),
            (ValueError, dict(k_pages=k.transpose(1, 2), v_pages=v.transpose(1, 2))),
            (ValueError, dict(k_pages=k[:1].expand(4, 2, 4, 32), v_pages=v[:1].expand(4, 2, 4, 32))),
            (ValueError, dict(k_pages=k[..., :24].contiguous(), v_pages=v[..., :24].contiguous())),
            (ValueError, dict(k_pages=k[:0], v_pages=v[:0])), (TypeError, dict(block_table=table.long())),
            (TypeError, dict(lengths=lengths.long())), (ValueError, dict(lengths=lengths.cpu())),
            (ValueError, dict(block_table=table[:1])), (ValueError, dict(cu_seqlens=lengths)),
            (ValueError, dict(cos=None)), (TypeError, dict(cos=cos.half(), sin=sin.half())),
            (ValueError, dict(cos=torch.zeros(4, 17, device=DEV), sin=torch.zeros(4, 17, device=DEV))),
            (ValueError, dict(lora_q=lora[:, :32])), (TypeError, dict(lora_q=lora.bfloat16())),
            (ValueError, dict(lora_v=lora))]:
        with pytest.raises(error):
            rope.rope_append(**{**ok, **kw})
    for name in ("qkv", "cos", "k_pages"):
        with pytest.raises(RuntimeError, match=f"no backward for {name}"):
            rope.rope_append(**{**ok, name: ok[name].clone().requires_grad_(True)})
    with torch.no_grad():
        rope.rope_append(**{**ok, "qkv": qkv.clone().requires_grad_(True)})
    with torch.inference_mode():
        rope.rope_append(**{**ok, "k_pages": k.clone(), "v_pages": v.clone()})
