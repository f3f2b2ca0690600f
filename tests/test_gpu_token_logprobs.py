"""head.token_logprobs against 64 bits: values, alternatives (exactly) and gradients.

Tolerances.  With u = 2^-24 and x = (z - max z) / T, an exponential's relative error is below
4 u (1 + |x|) (the difference, the product and the base-2 exponential each round once; |x| < 104
where it is not zero), a lane adds at most V / 1024 + 16 chunk sums and the workgroup 16 more, so the
sum S is within u (V / 1024 + 64 + 4 E) relative, E = sum p |x|, and so are ln S absolutely and the
probabilities relatively (with their own |x| in place of E); the token's own x adds 4 u |x|.  The
gradient is p (...) with those factors, rounded once to the logits' type (eps / 2)."""

import pytest
import torch

from oracle.logprobs import token_logprobs as reference
from testt_amd import head

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24

CASES = [  # rows, vocab, dtype, top_k, temperature
    (1, 151936, torch.float16, 20, 1.0),      # cut into parts
    (5, 151936, torch.bfloat16, 8, 0.7),
    (300, 151936, torch.float16, 5, 1.0),     # one workgroup a row or few parts
    (1500, 5000, torch.float16, 32, 1.0),
    (7, 32003, torch.float32, 32, 2.0),       # odd rows: unaligned, a tail
    (9, 32003, torch.float16, 1, 1.0),
    (1100, 2049, torch.bfloat16, 3, 1.0),
    (3, 1, torch.float16, 1, 1.0),            # one column
    (4, 7, torch.float16, 7, 1.0),            # less than a chunk, all of it ranked
    (4, 9, torch.float32, 9, 1.0),
    (2, 255, torch.float32, 0, 1.0),
    (1, 1031, torch.float16, 32, 1.3),
    (0, 64, torch.float16, 2, 1.0),
]


def logits_of(rows, vocab, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = 2.5 * torch.randn(rows, vocab, generator=g)
    tok = torch.randint(0, vocab, (rows,), generator=g)
    if rows:
        z[torch.arange(rows), tok] += 6 * torch.rand(rows, generator=g)
        tok[::4] = -100 if rows > 1 else tok[::4]
    return z.to(dtype), tok


def bounds(z, temperature):
    """(relative error of S and absolute of ln S, sum p |x|) of float64 rows."""
    x = (z - z.amax(-1, keepdim=True)) / temperature
    p = torch.softmax(z / temperature, -1)
    e = torch.where(p > 0, p * x.abs(), 0).sum(-1)
    return U * (z.shape[-1] / 1024 + 64 + 4 * e), e, x, p


def check(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.detach()
    assert got.shape == want.shape, what
    # (fp32's lowest value over a temperature below 1 is beyond fp32: it rounds to -inf)
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * float("inf"), want)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    assert not bad.any(), (f"{what}: {int(bad.sum())} off, worst "
                           f"{float((got - want).abs()[bad].max())} for "
                           f"{float(torch.as_tensor(tol).expand(want.shape)[bad].min())}")


def compare(z, tok, top_k, temperature, grads=True, seed=1):
    """The kernels on `z` against the reference on the same values."""
    dt = z.dtype
    leaf = z.detach().clone().to(DEV).requires_grad_(True)
    got = head.token_logprobs(leaf, tok.to(DEV), top_k, temperature)
    zd = z.double().requires_grad_(True)
    want = reference(zd, tok, top_k, temperature)
    rel, e, x, p = bounds(zd.detach(), temperature)
    tok_x = x.gather(-1, tok.clamp(0, z.shape[-1] - 1)[..., None])[..., 0].abs()
    tok_x = torch.nan_to_num(tok_x, posinf=0.0)
    check(got.logprob, want[0], rel + 4 * U * (tok_x + 1), "logprob")
    check(got.entropy, want[1], (rel + 4 * U) * (2 + 2 * e), "entropy")
    top_x = torch.nan_to_num(x.gather(-1, want[3]).abs(), posinf=0.0)
    check(got.top_logprobs, want[2], rel[..., None] + 4 * U * (top_x + 1), "top")
    assert torch.equal(got.top_ids.cpu(), want[3])
    if not grads or z.numel() == 0:
        return got, leaf
    g = torch.Generator().manual_seed(seed)
    ups = [torch.randn(w.shape, generator=g) for w in want[:3]]
    outs = [o for o, u in zip(got[:3], ups) if u.numel()]
    torch.autograd.backward(outs, [u.to(DEV) for u in ups if u.numel()])
    ref, = torch.autograd.grad(want[:3], zd, [u.double() for u in ups])
    weight = ups[0].abs().double() + ups[2].abs().double().sum(-1)
    logp = torch.where(p > 0, p.clamp(min=1e-300).log().abs(), 0)
    size = p * (weight[..., None] + ups[1].abs().double()[..., None] * (logp + want[1].detach()[
        ..., None] + 2)) / temperature
    rel_p = rel[..., None] + 8 * U * (1 + x.abs().clamp(max=200))
    tol = torch.finfo(dt).eps / 2 * ref.abs() + (size + ref.abs()) * 4 * rel_p + \
        torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    check(leaf.grad, ref, tol, "dlogits")
    return got, leaf


@pytest.mark.parametrize("rows,vocab,dtype,top_k,temperature", CASES)
def test_values_and_gradient(rows, vocab, dtype, top_k, temperature):
    print(f"logprobs {rows} x {vocab} {dtype} top {top_k} T {temperature}", flush=True)
    z, tok = logits_of(rows, vocab, dtype, rows + vocab)
    compare(z, tok, top_k, temperature)


@pytest.mark.parametrize("rows,vocab", [(6, 20000), (1200, 4100)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_masked_rows(rows, vocab, dtype):
    """-inf and lowest-value masks that leave many, few, one or no columns; equal logits; a row that
    rises all the way (the candidate list overflows); +inf."""
    print(f"masked {rows} x {vocab} {dtype}", flush=True)
    z, tok = logits_of(rows, vocab, dtype, 5)
    low = torch.finfo(dtype).min
    z[0, 7:] = float("-inf")
    z[0, 5], tok[0] = 1.0, 3
    z[1] = low
    z[1, 11000 % vocab], tok[1] = 2.0, 11000 % vocab
    z[2] = low                                       # nothing but the lowest value: uniform
    z[3] = 1.5                                       # every column equal
    z[4] = torch.linspace(-9, 9, vocab).to(dtype)
    z[5] = float("-inf")
    z[5, vocab - 1], tok[5] = -3.0, vocab - 1
    compare(z, tok, 8, 1.0)
    compare(z, tok, 32, 0.5, seed=2)


@pytest.mark.parametrize("vocab", [7000, 8192, 40000, 40007])
@pytest.mark.parametrize("dtype,top_k", [(torch.float16, 32), (torch.float32, 32),
                                         (torch.float32, 3), (torch.bfloat16, 8)])
def test_rising_rows(vocab, dtype, top_k):
    """Rows that rise from left to right, whole (enough of them not to be cut into parts): the lists of
    candidates overflow and the row is searched.  Others among them fall, or rise in a few wide steps
    of equal columns."""
    print(f"rising {vocab} {dtype} top {top_k}", flush=True)
    rows = 1030
    z, tok = logits_of(8, vocab, dtype, vocab)
    ramp = torch.linspace(-8, 8, vocab)
    z[0], z[1] = ramp.to(dtype), ramp.flip(0).to(dtype)
    z[2] = (ramp * 0.5).floor().to(dtype)
    z[3] = (ramp * 4).floor().to(dtype)
    z[4, : vocab // 2] = float("-inf")
    z[4, vocab // 2:] = ramp[vocab // 2:].to(dtype)
    z[5] = float("-inf")
    z[5, vocab // 3: vocab // 3 + 20] = 1.0
    many = z.repeat(rows // 8 + 1, 1)[:rows]
    got = head.token_logprobs(many.to(DEV), tok.repeat(rows // 8 + 1)[:rows].to(DEV), top_k)
    want = reference(z.double(), tok, top_k)
    ids = want[3].repeat(rows // 8 + 1, 1)[:rows]
    assert torch.equal(got.top_ids.cpu(), ids)
    lp = want[2].repeat(rows // 8 + 1, 1)[:rows]
    rel, _, x, _ = bounds(z.double(), 1.0)
    tol = (rel[:, None] + 4 * U * (x.gather(-1, want[3]).abs().nan_to_num(posinf=0.0) + 1)).repeat(
        rows // 8 + 1, 1)[:rows]
    check(got.top_logprobs, lp, tol, "top")


@pytest.mark.parametrize("dtype,top_k", [(torch.float32, 32), (torch.float32, 2),
                                         (torch.float16, 32), (torch.bfloat16, 8)])
@pytest.mark.parametrize("vocab", [40007, 151936])
def test_rows_that_rise_with_noise(vocab, dtype, top_k):
    """Rows whose candidates overflow the lists in each of their ways: noise on a rise; a rise of which
    long runs are equal; and the large columns in a few threads' places (K - 1 of them, so that the
    bound of the threads' largest lies below them all), rising and random."""
    print(f"noisy rise {vocab} {dtype} top {top_k}", flush=True)
    rows = 1030 if vocab < 100000 else 600
    z, tok = logits_of(6, vocab, dtype, vocab + 1)
    ramp = torch.linspace(-8, 8, vocab)
    noise = torch.randn(6, vocab, generator=torch.Generator().manual_seed(vocab))
    cols = 16 // z.element_size()
    place = (torch.arange(vocab) // cols) % 256
    comb = torch.where(place < top_k - 1, 20.0, 0.0)
    z[0] = (ramp + noise[0]).to(dtype)
    z[1] = (ramp * 8).floor().to(dtype)
    z[2] = (comb + ramp).to(dtype)
    z[3] = (comb + noise[3]).to(dtype)
    z[4] = comb.to(dtype)
    reps = rows // 6 + 1
    got = head.token_logprobs(z.repeat(reps, 1)[:rows].to(DEV), tok.repeat(reps)[:rows].to(DEV), top_k)
    want = reference(z.double(), tok, top_k)
    assert torch.equal(got.top_ids.cpu(), want[3].repeat(reps, 1)[:rows])
    rel, _, x, _ = bounds(z.double(), 1.0)
    tol = rel[:, None] + 4 * U * (x.gather(-1, want[3]).abs().nan_to_num(posinf=0.0) + 1)
    check(got.top_logprobs, want[2].repeat(reps, 1)[:rows], tol.repeat(reps, 1)[:rows], "top")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [33, 130, 257, 600, 1031])
def test_few_columns(vocab, dtype):
    """Rows of fewer chunks than the bound has groups: most columns reach it, and the list is thinned.
    Random, rising, equal and nearly all masked rows."""
    print(f"few columns {vocab} {dtype}", flush=True)
    z, tok = logits_of(7, vocab, dtype, vocab)
    z[1] = torch.linspace(-3, 3, vocab).to(dtype)
    z[2] = 1.0
    z[3] = (torch.arange(vocab) % 3).to(dtype)
    z[4] = float("-inf")
    z[4, 5:8] = 2.0
    tok[4] = 6
    compare(z, tok, 32, 1.0, grads=False)
    compare(z[:1], tok[:1], 20, 1.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_equal_columns_in_every_part(dtype):
    """One long row, cut into parts that all offer the same values: the join's list is thinned."""
    z = torch.zeros(2, 151936, dtype=dtype)
    z[1] = (torch.arange(151936) % 5 == 3).to(dtype)
    compare(z, torch.tensor([7, 151935]), 32, 1.0, grads=False)


def test_rows_without_a_distribution():
    """A row of -inf alone, one with NaN, one with +inf: NaN numbers, ordered ids; other rows
    unharmed, and a row without upstream gradient keeps a zero gradient."""
    z, tok = logits_of(6, 9000, torch.float32, 9)
    z[1] = float("-inf")
    z[2, 77] = float("nan")
    z[3, 8000] = float("inf")
    tok[:] = torch.tensor([1, 2, 3, 4, -100, 6])
    leaf = z.clone().to(DEV).requires_grad_(True)
    got = head.token_logprobs(leaf, tok.to(DEV), 4)
    want = reference(z.double(), tok, 4)
    for r in (1, 2, 3):
        assert got.logprob[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all()
    assert torch.equal(got.top_ids.cpu(), want[3])
    assert got.top_ids[1].tolist() == [0, 1, 2, 3] and int(got.top_ids[3, 0]) == 8000
    for r in (0, 4, 5):
        assert abs(float(got.entropy[r].detach()) - float(want[1][r])) < 1e-5
    up = torch.zeros(6, device=DEV)
    up[[0, 4]] = 1.0
    got.logprob.backward(up)
    assert leaf.grad[[1, 2, 3, 4, 5]].eq(0).all() and leaf.grad[0].abs().sum() > 0


def test_tokens_outside_the_vocabulary():
    z, _ = logits_of(4, 500, torch.float16, 2)
    tok = torch.tensor([-100, 500, -1, 3], device=DEV)
    leaf = z.to(DEV).requires_grad_(True)
    got = head.token_logprobs(leaf, tok)
    assert float(got.logprob[0].detach()) == 0 and got.logprob[1:3].isnan().all()
    got.logprob.sum().backward()
    assert leaf.grad[:3].eq(0).all() and leaf.grad[3].abs().sum() > 0


def test_strided_batches():
    """[batch, seq, V] shifted by a position, a transposed batch, columns of a wider row, one row for
    all: the same values as the packed copy."""
    z, _ = logits_of(12, 1001, torch.float16, 4)
    base = z.view(3, 4, 1001).to(DEV)
    tok = torch.randint(0, 900, (3, 3), device=DEV)
    for view in (base[:, 1:], base[:, :3], base.transpose(0, 1)[:3], base[:, 1:, 50:951],
                 base[:1, 1:].expand(3, 3, 1001)):
        packed = view.contiguous()
        a = head.token_logprobs(view, tok, 5)
        b = head.token_logprobs(packed, tok, 5)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    # the gradient of a view lands in its rows of the whole tensor
    leaf = base[:, 1:].clone().requires_grad_(True)
    ga, = torch.autograd.grad(head.token_logprobs(leaf, tok).logprob.sum(), leaf)
    src = base.clone().requires_grad_(True)
    gb, = torch.autograd.grad(head.token_logprobs(src[:, 1:], tok).logprob.sum(), src)
    assert torch.equal(gb[:, 1:], ga) and gb[:, 0].eq(0).all()


def test_gradient_by_differences():
    z, tok = logits_of(3, 40, torch.float32, 8)
    tok = torch.tensor([4, 39, 0])
    up = torch.tensor([0.7, -1.1, 0.4], device=DEV)
    f = lambda v: (lambda o: (o.logprob * up).sum() + 0.5 * (o.entropy * up).sum() +
                   0.3 * o.top_logprobs.sum())(head.token_logprobs(v, tok.to(DEV), 3, 0.8))
    leaf = z.to(DEV).requires_grad_(True)
    grad, = torch.autograd.grad(f(leaf), leaf)
    step = 2.0 ** -6
    worst = 0.0
    for r, col in ((0, 4), (0, 17), (1, 39), (1, 3), (2, 0), (2, 20)):
        d = torch.zeros_like(z)
        d[r, col] = step
        slope = (f((z + d).to(DEV)) - f((z - d).to(DEV))) / (2 * step)
        worst = max(worst, abs(float(slope) - float(grad[r, col])))
    # rounding of f (about 20, eps 2^-24 each of ~10 terms) over the step, and h^2 / 6 times the
    # third derivative (below 4 / T^3)
    assert worst < 200 * U / step + step ** 2 * 8


def test_absent_gradients_and_no_grad():
    z, tok = logits_of(5, 3000, torch.float16, 6)
    leaf = z.to(DEV).requires_grad_(True)
    out = head.token_logprobs(leaf, tok.to(DEV), 4)
    g_ent, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)
    g_lp, = torch.autograd.grad(out.logprob.sum(), leaf, retain_graph=True)
    both, = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), leaf, retain_graph=True)
    # each was rounded to fp16 once
    tol = 2.0 ** -11 * (g_ent.abs() + g_lp.abs() + both.abs()).float() + 2.0 ** -24
    assert ((g_ent.float() + g_lp.float() - both.float()).abs() <= tol).all()
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(out.logprob.sum(), leaf, create_graph=True)
        torch.autograd.grad(g.sum(), leaf)
    with torch.no_grad():
        again = head.token_logprobs(leaf, tok.to(DEV), 4)
    assert all(torch.equal(a, b) for a, b in zip(again, out)) and not again.logprob.requires_grad


@pytest.mark.parametrize("rows", [3, 2500])
def test_hidden_form(rows):
    """fused_token_logprobs is token_logprobs of the fp16 head product, chunk by chunk; its gradient is
    dlogits @ weight (logits' gradient in fp16 beside the fp32 one: eps / 2 of each entry, over sqrt of
    the sum's size at most the sum of absolute products)."""
    print(f"hidden rows {rows}", flush=True)
    g = torch.Generator().manual_seed(rows)
    hidden = torch.randn(rows, 64, generator=g).half().to(DEV)
    weight = (0.3 * torch.randn(1016, 64, generator=g)).half().to(DEV)
    tok = torch.randint(0, 1016, (rows,), generator=g).to(DEV)
    tok[0] = -100
    leaf = hidden.clone().requires_grad_(True)
    got = head.fused_token_logprobs(leaf, weight, tok, 4, 0.9)
    logits = torch.cat([torch.nn.functional.linear(h, weight) for h in hidden.split(2048)])
    want = head.token_logprobs(logits.requires_grad_(True), tok, 4, 0.9)
    # the library's product may sum in another order at another row count: one fp16 step of a logit
    step = logits.abs().max() * 2.0 ** -10
    for a, b in zip(got[:3], want[:3]):
        assert (a - b).abs().max() <= 4 * step / 0.9 * 8
    up = torch.randn(rows, device=DEV) / rows
    (got.logprob * up).sum().backward()
    z = logits.detach().double().requires_grad_(True)
    ref = reference(z.cpu(), tok.cpu(), 4, 0.9)
    d, = torch.autograd.grad(ref[0], z, up.double().cpu())
    dh = d.to(DEV) @ weight.double()
    mass = d.abs().to(DEV) @ weight.double().abs()
    # p moves by a logit's fp16 step over T (both products), the gradient of the logits rounds to fp16,
    # and so does the result (with an fp16 subnormal step)
    tol = mass * (2 * float(step) / 0.9 * 2 + 2.0 ** -10) + 2.0 ** -10 * dh.abs() + 2.0 ** -24
    assert ((leaf.grad.double() - dh).abs() <= tol).all()
    assert leaf.grad[0].eq(0).all()


def test_graph_replay():
    """Forward and backward captured and replayed on changed logits, with eager work between."""
    z, tok = logits_of(40, 20000, torch.float16, 3)
    z, tok = z.to(DEV), tok.to(DEV)
    up = torch.randn(40, device=DEV)

    def step(v):
        leaf = v.detach().requires_grad_(True)
        out = head.token_logprobs(leaf, tok, 6)
        g, = torch.autograd.grad(out.logprob, leaf, up)
        return (*out, g)

    static = z.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i in range(4):
        new = (z.float() * (1 + 0.1 * i)).half()
        static.copy_(new)
        graph.replay()
        want = step(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_other_stream():
    z, tok = logits_of(64, 30000, torch.float16, 12)
    z, tok = z.to(DEV), tok.to(DEV)
    want = head.token_logprobs(z, tok, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = head.token_logprobs(z, tok, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
