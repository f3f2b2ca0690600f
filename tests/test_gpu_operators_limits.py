"""The operators around the layer where 32-bit offsets end, from two threads and streams at once, and in
two captured graphs: the results of the same rows alone."""

import threading

import pytest
import torch

from testt_amd import dropout, embedding, head, rope, workloads

pytestmark = pytest.mark.gpu
DEV = "cuda"
H = torch.float16


def fill(*shape):
    """A large tensor of varied values without the time of a full draw: a drawn block, repeated."""
    n = 1
    for s in shape:
        n *= s
    block = torch.randn(1 << 22, device=DEV).to(H)
    return block.repeat(-(-n // block.numel()))[:n].view(shape)


def test_logits_past_two_to_the_31_elements():
    rows, vocab = 14200, 151936
    assert rows * vocab > 1 << 31
    z = fill(rows, vocab).requires_grad_(True)
    tok = torch.randint(0, vocab, (rows,), device=DEV)
    out = head.token_logprobs(z, tok, 3)
    up = torch.randn(rows, device=DEV)
    g, = torch.autograd.grad(out.logprob, z, up)
    for part in (slice(0, 40), slice(rows - 40, rows)):
        zp = z.detach()[part].clone().requires_grad_(True)
        alone = head.token_logprobs(zp, tok[part], 3)
        assert torch.equal(alone.top_ids, out.top_ids[part])
        # (few rows are cut into parts, whose sums join in another order: 64 fp32 steps of values ~ 12)
        assert (alone.logprob - out.logprob[part]).abs().max() < 64 * 2.0 ** -24 * 16
        ga, = torch.autograd.grad(alone.logprob, zp, up[part])
        # both rounded to fp16 once, from probabilities a few fp32 steps apart
        assert ((ga.float() - g[part].float()).abs() <= 2.0 ** -10 * ga.float().abs() + 2.0 ** -24).all()


def test_embedding_past_two_to_the_31_elements():
    vocab, width = 1_400_100, 1536
    assert vocab * width > 1 << 31
    table = fill(vocab, width).requires_grad_(True)
    ids = torch.tensor([0, vocab - 1, vocab - 1, 1_398_102, 5, vocab], device=DEV)
    y = embedding.embedding(ids, table)
    assert torch.equal(y[:5], table.detach()[ids[:5]]) and y[5].eq(0).all()
    dout = torch.randn_like(y)
    g, = torch.autograd.grad(y, table, dout)
    want = torch.zeros(4, width, device=DEV)
    want[0], want[1], want[2] = dout[0].float(), dout[1].float() + dout[2].float(), dout[3].float()
    want[3] = dout[4].float()
    assert torch.equal(g[torch.tensor([0, vocab - 1, 1_398_102, 5], device=DEV)], want.half())
    named = torch.zeros(vocab, dtype=torch.bool, device=DEV)
    named[ids[:5]] = True
    for i in range(0, vocab, 100_000):                 # every other row is zero
        rows = g[i:i + 100_000]
        assert not rows[~named[i:i + 100_000]].any()


def test_dropout_and_norm_past_two_to_the_31_elements():
    rows, cols = 5, 430_000_007
    assert rows * cols > 1 << 31
    x = fill(rows, cols)
    y = dropout.dropout(x, 0.3, 9, 2)
    last = dropout.dropout(x[4:, :].clone(), 0.3, 9, 2, rows=torch.tensor([4], device=DEV))
    assert torch.equal(y[4:], last)
    del x, y, last
    nh, nkv, d, m = 32, 8, 128, 350_000
    assert m * (nh + 2 * nkv) * d > 1 << 31
    qkv = fill(m, (nh + 2 * nkv) * d)
    pos = torch.arange(m, device=DEV) % 4096
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(4096, d))
    w = torch.ones(d, device=DEV).requires_grad_(True)
    qkv.requires_grad_(True)
    args = (w, w, cos, sin)
    out = rope.qk_norm_rope(qkv, None, None, *args, pos, 1, 4096, nh, nkv, d)
    g, = torch.autograd.grad(out, qkv, out.detach())
    tail = qkv.detach()[-100:].clone().requires_grad_(True)
    alone = rope.qk_norm_rope(tail, None, None, *args, pos[-100:].contiguous(), 1, 4096, nh, nkv, d)
    ga, = torch.autograd.grad(alone, tail, alone.detach())
    assert torch.equal(out.detach()[-100:], alone.detach()) and torch.equal(g[-100:], ga)


def test_more_rows_than_a_launch_takes():
    """A grid spans fewer than 2^32 threads: more rows than that gives workgroups for are launched in turn."""
    rows, vocab = (1 << 24) + 77, 5
    z = fill(rows, vocab).requires_grad_(True)
    tok = torch.arange(rows, device=DEV) % vocab
    out = head.token_logprobs(z, tok, 2)
    g, = torch.autograd.grad(out.logprob, z, torch.ones(rows, device=DEV))
    for at in (0, (1 << 23) - 50, (1 << 24) - 50, rows - 100):
        part = slice(at, at + 100)
        zp = z.detach()[part].clone().requires_grad_(True)
        alone = head.token_logprobs(zp, tok[part], 2)
        ga, = torch.autograd.grad(alone.logprob, zp, torch.ones(100, device=DEV))
        assert all(torch.equal(a, o[part]) for a, o in zip(alone, out))
        assert torch.equal(ga, g[part])
    del z, tok, out, g
    m, d = (1 << 26) + 77, 16
    qkv = fill(m, d).requires_grad_(True)
    pos = torch.arange(m, device=DEV) % 64
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(64, d))
    w = torch.ones(d, device=DEV)
    y = rope.qk_norm_rope(qkv, None, None, w, w, cos, sin, pos, 1, 64, 1, 0, d)
    g, = torch.autograd.grad(y, qkv, y.detach())
    for at in (0, (1 << 25) - 50, (1 << 26) - 50, m - 100):
        part = slice(at, at + 100)
        qp = qkv.detach()[part].clone().requires_grad_(True)
        alone = rope.qk_norm_rope(qp, None, None, w, w, cos, sin, pos[part].clone(), 1, 64, 1, 0, d)
        ga, = torch.autograd.grad(alone, qp, alone.detach())
        assert torch.equal(y.detach()[part], alone.detach()) and torch.equal(ga, g[part])


def steps(seed):
    """One forward and backward of each operator on its own data: a function that runs them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    z, tok = rnd(60, 20011).half(), torch.randint(0, 20011, (60,), generator=g, device=DEV)
    table, ids = rnd(4000, 264).half(), torch.randint(0, 300, (700,), generator=g, device=DEV)
    x = rnd(300, 1536).half()
    qkv, pos = rnd(200, 8 * 128).half(), torch.arange(200, device=DEV)
    cos, sin = (t.to(DEV) for t in workloads.rope_tables(256, 128))
    w = 1 + 0.1 * rnd(128)
    ups = [rnd(60), rnd(700, 264).half(), rnd(300, 1536).half(), rnd(200, 8 * 128).half()]

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (z, table, x, qkv, w)]
        outs = [head.token_logprobs(leaves[0], tok, 6), embedding.embedding(ids, leaves[1]),
                dropout.dropout(leaves[2], 0.2, seed, 1),
                rope.qk_norm_rope(leaves[3], None, None, leaves[4], leaves[4], cos, sin, pos, 1, 256,
                                  4, 2, 128)]
        lp = outs[0]
        grads = torch.autograd.grad([lp.logprob, *outs[1:]], leaves, ups)
        return [lp.logprob.detach(), lp.entropy.detach(), lp.top_ids,
                *(o.detach() for o in outs[1:]), *grads]

    return run


def test_two_threads_on_two_streams():
    runs = [steps(1), steps(2)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = runs[i]()
            stream.synchronize()
        except Exception as exc:  # noqa: BLE001 - reported by the test's thread
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not errors and all(g is not None for g in got)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_captured_graphs_in_turn():
    runs = [steps(3), steps(4)]
    want = [r() for r in runs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for r in runs:
            r()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()              # one pool: their workspaces share memory
    for r in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(r())
        graphs.append(graph)
    kept = [None, None]
    for i in (0, 1, 0, 1, 1, 0):
        graphs[i].replay()
        kept[i] = [t.clone() for t in outs[i]]
        steps(5)()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(kept[i], want[i]))
