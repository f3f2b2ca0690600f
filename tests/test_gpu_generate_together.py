"""The generating operators as a program uses them: prompts and drafted tokens through a small attention model
with a paged cache, its outputs against the training path's attention over the whole sequences, its
tokens against the reference's verification; beside other calls on other streams, threads and in graphs."""

import threading

import pytest
import torch

from oracle import generate as og
from testt_amd import attention, head, rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, I32 = torch.float16, torch.int32
NH, NKV, D, HID, V, PAGE = 4, 2, 128, 64, 97, 16


class Tiny:
    """One layer: embedding, q|k|v with LoRA deltas, attention, head."""

    def __init__(self, seed, theta=1e4, noise=0.0):
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=gen)     # noqa: E731
        self.emb, self.wqkv = rnd(V, HID), rnd(HID, (NH + 2 * NKV) * D) / HID ** 0.5
        self.wq, self.wv = 0.1 * rnd(HID, NH * D) / 8, 0.1 * rnd(HID, NKV * D) / 8
        self.wo, self.wh = rnd(NH * D, HID) / (NH * D) ** 0.5, 3 * rnd(HID, V) / HID ** 0.5
        if noise:
            self.wh = self.wh + noise * torch.randn(HID, V, generator=torch.Generator().manual_seed(99))
        for name, t in list(vars(self).items()):
            setattr(self, name, t.to(DEV))
        self.cos, self.sin = rope.rotary_tables(128, D, theta, {"rope_type": "yarn", "factor": 2.0,
                                                                 "original_max_position_embeddings": 64},
                                                device=DEV)

    def rows(self, ids):
        x = self.emb[ids]
        return x, (x @ self.wqkv).to(H), (x @ self.wq).to(H), (x @ self.wv).to(H)

    def logits(self, x, attn):
        return (x + attn.float() @ self.wo) @ self.wh

    def full(self, ids, lengths):
        """The training path over whole sequences, ids sorted by sequence."""
        x, qkv, lq, lv = self.rows(ids)
        pos = torch.cat([b * 128 + torch.arange(n) for b, n in enumerate(lengths)]).to(DEV)
        cos, sin = (torch.cat([t, t], 1) for t in (self.cos, self.sin))
        cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0)], dtype=I32, device=DEV)
        attn = attention.rope_attention(qkv, lq, lv, cos, sin, pos, cu, len(lengths), 128, NH, NKV)
        return attn, self.logits(x, attn)

    def step(self, ids, cache, lengths, cu):
        x, qkv, lq, lv = self.rows(ids)
        q = rope.rope_append(qkv, lq, lv, self.cos, self.sin, cache[0], cache[1], cache[2], lengths, cu)
        attn = attention.paged_attention(q, cache[0], cache[1], cache[2], lengths, cu)
        return attn, self.logits(x, attn)


def new_cache(batch, seed):
    gen = torch.Generator().manual_seed(seed)
    n = batch * 8 + 1
    pages = torch.full((2, n, NKV, PAGE, D), float("nan"), dtype=H, device=DEV)
    table = torch.randperm(n, generator=gen)[:batch * 8].view(batch, 8).to(I32).to(DEV)
    return pages[0], pages[1], table


def ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def bounds(news):
    return ints([0, *torch.tensor(news).cumsum(0)])


# fp16 attention of up to 128 keys, values of about unit size: scores agree to the rounding of the same fp16
# rows, probabilities and outputs are rounded to fp16 in both, 4 roundings of 2^-11 of values up to 4
TOL = 4 * 4 * 2.0 ** -11


def test_prompts_then_single_tokens():
    m = Tiny(1)
    gen = torch.Generator().manual_seed(2)
    seqs = [torch.randint(0, V, (n,), generator=gen) for n in (30, 7, 52)]
    prompts = [17, 1, 48]
    cache = new_cache(3, 3)
    with torch.no_grad():
        want, _ = m.full(torch.cat(seqs).to(DEV), [len(s) for s in seqs])
        want = want.split([len(s) for s in seqs])
        got, _ = m.step(torch.cat([s[:n] for s, n in zip(seqs, prompts)]).to(DEV), cache, ints(prompts),
                        bounds(prompts))
        for a, b, n in zip(got.split(prompts), want, prompts):
            assert float((a.float() - b[:n].float()).abs().max()) < TOL
        # then a token at a time; a finished sequence goes on as a row of length 0
        for i in range(13):
            at = [n + i for n in prompts]
            live = [t < len(s) for t, s in zip(at, seqs)]
            ids = torch.stack([s[min(t, len(s) - 1)] for t, s in zip(at, seqs)]).to(DEV)
            got, _ = m.step(ids, cache, ints([t + 1 if on else 0 for t, on in zip(at, live)]), None)
            for b in range(3):
                if live[b]:
                    assert float((got[b].float() - want[b][at[b]].float()).abs().max()) < TOL
                else:
                    assert not bool(got[b].any())


def test_drafted_tokens():
    """Drafts of a second model, verified three at a time: the kept tokens are the reference's, and the cache
    goes on from them as if they alone had been appended."""
    target, draft = Tiny(1), Tiny(1, noise=0.3)
    gen = torch.Generator().manual_seed(4)
    rand = lambda *s: torch.rand(*s, generator=gen)          # noqa: E731
    batch, K = 3, 3
    seqs = [torch.randint(0, V, (n,), generator=gen).tolist() for n in (9, 20, 2)]
    caches = new_cache(batch, 5), new_cache(batch, 6)
    refused = kept = 0
    with torch.no_grad():
        for m, cache in zip((target, draft), caches):        # all but the last token of each prompt
            news = [len(s) - 1 for s in seqs]
            ids = torch.tensor([t for s in seqs for t in s[:-1]], device=DEV)
            m.step(ids, cache, ints(news), bounds(news))
        pending = [[s[-1]] for s in seqs]                    # tokens that the draft's cache lacks
        for _ in range(8):
            drafts, q = [], []
            for i in range(K):
                news = [len(p) if i == 0 else 1 for p in pending]
                ids = [t for p in pending for t in p] if i == 0 else drafts[-1]
                lens = [len(s) + i for s in seqs]
                _, z = draft.step(torch.tensor(ids, device=DEV), caches[1], ints(lens), bounds(news))
                last = torch.tensor(news).cumsum(0) - 1
                q.append(z[last.to(DEV)].softmax(-1))
                drafts.append(torch.multinomial(q[-1].cpu(), 1, generator=gen)[:, 0].tolist())
            q = torch.stack(q, 1)
            x = torch.tensor(drafts).t().contiguous()
            news = [K + 1] * batch
            ids = torch.cat([torch.tensor([s[-1] for s in seqs])[:, None], x], 1).reshape(-1)
            attn, z = target.step(ids.to(DEV), caches[0], ints([len(s) + K for s in seqs]), bounds(news))
            want, _ = target.full(torch.tensor([t for s, d in zip(seqs, x.tolist()) for t in s + d],
                                               device=DEV), [len(s) + K for s in seqs])
            at = 0
            for b, s in enumerate(seqs):
                at += len(s) + K
                far = (attn[4 * b:4 * b + 4].float() - want[at - 4:at].float()).abs().max()
                assert float(far) < TOL
            p = z.softmax(-1).view(batch, K + 1, V)
            u = rand(batch, K + 1)
            got = head.verify_drafts(p, x.to(DEV), u.to(DEV), q)
            ref = og.verify_drafts(p.cpu(), x, u, q.cpu())
            assert torch.equal(got.tokens.cpu(), ref[0]) and torch.equal(got.accepted.cpu(), ref[1])
            pending = []
            for b in range(batch):
                n = int(got.accepted[b])
                new = got.tokens[b, :n + 1].tolist()
                pending.append(new[-2:] if n == K else new[-1:])
                seqs[b] += new
                kept += n
                refused += n < K
    assert kept > 0 and refused > 0


def test_two_streams_and_threads():
    """Calls at once, each with its own cache, equal to themselves alone."""
    m = Tiny(7)
    gen = torch.Generator().manual_seed(8)
    ids = [torch.randint(0, V, (60,), generator=gen).to(DEV) for _ in range(2)]
    probs = torch.rand(4, 3, 20000, generator=gen).to(DEV)
    x, u = torch.randint(0, 20000, (4, 2), generator=gen).to(DEV), torch.rand(4, 3, generator=gen).to(DEV)

    def run(i, out):
        with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            for _ in range(20):
                cache = new_cache(2, i)
                attn, _ = m.step(ids[i], cache, ints([40, 20]), bounds([40, 20]))
                verdict = head.verify_drafts(probs, x, u)
            torch.cuda.current_stream().synchronize()
            out[i] = attn, verdict.tokens

    torch.cuda.synchronize()
    alone, both = {}, {}
    for i in range(2):
        run(i, alone)
    threads = [threading.Thread(target=run, args=(i, both)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert torch.equal(alone[i][0], both[i][0]) and torch.equal(alone[i][1], both[i][1])


def test_a_decoding_step_in_two_graphs():
    """Two captured steps over one cache, replayed in turn with the lengths moved on, against eager steps."""
    m = Tiny(9)
    gen = torch.Generator().manual_seed(10)
    cache, mirror = new_cache(2, 11), new_cache(2, 11)
    ids, lengths = torch.randint(0, V, (2,), generator=gen).to(DEV), ints([1, 1])
    with torch.no_grad():
        for c in (cache, mirror):
            m.step(ids, c, lengths, None)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = m.step(ids, cache, lengths, None)
            graphs.append((g, out))
        for i in range(40):
            ids.copy_(torch.randint(0, V, (2,), generator=gen))
            lengths.copy_(torch.tensor([i + 1, max(i - 7, 0)]))
            g, out = graphs[i % 2]
            g.replay()
            torch.cuda.synchronize()
            want = m.step(ids, mirror, lengths, None)
            assert torch.equal(out[0], want[0])
            same = torch.equal(cache[0].nan_to_num(9), mirror[0].nan_to_num(9))
            assert same, f"step {i}"
