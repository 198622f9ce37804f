"""Prompts with continuations that are stepped, taken back and ended in a SharedCache, against lists of keys and values and attention in 64 bits, and the run of the three
operators together: tables, attention, log probabilities.

Tolerances as in the attention's own tests: 1e-4 for float32; for bfloat16 2^-8 of the weighted mean of |v| and of the output beside it."""
import random

import numpy as np
import pytest
import torch

from kappai_b200 import SharedCache
from kappai_b200.cache import CacheError, OutOfPages, OutOfSlots
from kappai_b200.ops.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


class Plain:
    def __init__(self, H, G, hd):
        self.H, self.G, self.hd, self.kv = H, G, hd, {}

    def split(self, qkv):
        x = qkv.double().cpu().numpy()
        H, G, hd = self.H, self.G, self.hd
        return x[:, :H * hd].reshape(-1, G, H // G, hd), x[:, H * hd:(H + G) * hd].reshape(-1, G, hd), x[:, (H + G) * hd:].reshape(-1, G, hd)

    def run(self, seq, qkv, scale=None):
        q, k, v = self.split(qkv)
        old = self.kv.get(seq, (k[:0], v[:0]))
        K, V = np.concatenate([old[0], k]), np.concatenate([old[1], v])
        self.kv[seq] = K, V
        out, off = np.zeros(q.shape), np.zeros(q.shape)
        for r in range(len(q)):
            n = len(old[0]) + r + 1
            for g in range(self.G):
                s = q[r, g] @ K[:n, g].T * (scale or self.hd ** -0.5)
                e = np.exp(s - s.max(1, keepdims=True))
                e /= e.sum(1, keepdims=True)
                out[r, g] = e @ V[:n, g]
                off[r, g] = e @ np.abs(V[:n, g]) + np.abs(out[r, g])
        return out.reshape(len(q), -1), off.reshape(len(q), -1)


def near(got, want, off, dtype):
    tol = 1e-4 + (2.0 ** -8 * off if dtype == torch.bfloat16 else 0)
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("dtype,hd,page,H,G", [(torch.bfloat16, 64, 16, 8, 2), (torch.bfloat16, 128, 64, 4, 1), (torch.float32, 64, 16, 6, 2), (torch.float32, 96, 7, 4, 4)])
def test_forks_steps_and_ends(dtype, hd, page, H, G):
    rng = random.Random(hd + page)
    gen = torch.Generator("cuda").manual_seed(page)
    make = lambda n: torch.randn((n, (H + 2 * G) * hd), generator=gen, device="cuda").to(dtype)  # noqa: E731
    c, plain = SharedCache(H, G, hd, n_pages=4000 // page + 40, max_seqs=24, max_len=700, page_size=page, dtype=dtype), Plain(H, G, hd)

    def fork(P, n):
        x = make(P)
        out, seqs = c.fork(x, n)
        near(out, *plain.run("p", x), dtype)
        for s in seqs:
            plain.kv[s] = plain.kv["p"]
        del plain.kv["p"]
        c.check()
        return seqs

    def step(seqs=None, rows=None):
        ids = c.live() if seqs is None else seqs
        n = [1] * len(ids) if rows is None else rows
        x = make(sum(n))
        out, at = c.step(x, seqs, rows), 0
        for s, r in zip(ids, n):
            near(out[at:at + r], *plain.run(s, x[at:at + r]), dtype)
            at += r
        assert [c.length(s) for s in ids] == [len(plain.kv[s][0]) for s in ids]
        c.check()

    a = fork(300, 7)
    for _ in range(3):
        step()
    b = fork(page * 3, 5)                                # ends with a page
    step()
    step([a[0], a[3], b[2]], [3, 1, 20])
    back = [a[0], b[2]]
    c.take_back(back, [2, 20])
    plain.kv[a[0]] = tuple(t[:-2] for t in plain.kv[a[0]])
    plain.kv[b[2]] = tuple(t[:-20] for t in plain.kv[b[2]])
    c.check()
    step()
    free = c.pages_free
    c.end([a[1], a[6]])
    c.check()
    assert c.pages_free > free
    d = fork(5, 2)                                       # shorter than a page, in slots of its own
    step(None, [rng.randint(1, 4) for _ in c.live()])
    c.end(a[:1] + a[2:6])                                # the first prompt's last continuations: it goes too
    c.check()
    step()
    e = fork(1, 3)
    step()
    with pytest.raises(CacheError):
        c.step(make(1), [a[5]])                          # (numbers are given again; this one has not been)
    with pytest.raises(CacheError):
        c.take_back([e[0]], [2])
    with pytest.raises(OutOfSlots):
        c.fork(make(1), 23)
    c.end(sorted(b + d + e))
    c.check()
    assert c.pages_free == c.n_pages and c.live() == []


def test_pages_run_out_without_a_trace():
    c = SharedCache(4, 2, 64, n_pages=6, max_seqs=8, max_len=64, page_size=16)
    make = lambda n: torch.randn((n, 8 * 64), device="cuda").bfloat16()  # noqa: E731
    out, seqs = c.fork(make(40), 3)                      # 3 pages, a copy of the last for each
    with pytest.raises(OutOfPages):
        c.step(make(30), seqs, [10, 10, 10])
    c.check()
    c.step(make(24), seqs, [8, 8, 8])
    with pytest.raises(OutOfPages):
        c.step(make(3))
    with pytest.raises(CacheError):
        c.step(make(17), seqs[:1], [17])                 # longer than max_len
    c.check()
    assert [c.length(s) for s in seqs] == [48] * 3


def test_prompt_of_many_continuations_with_a_long_tail():
    """More rows of copied tails than a call takes."""
    c = SharedCache(1, 1, 32, n_pages=1100, max_seqs=1100, max_len=130, page_size=100)
    x = torch.randn((99, 3 * 32), device="cuda").bfloat16()
    _, seqs = c.fork(x, 1000)
    c.check()
    y = torch.randn((1000, 3 * 32), device="cuda").bfloat16()
    out, plain = c.step(y), Plain(1, 1, 32)
    plain.run("p", x)
    for i in (0, 1, 499, 999):
        plain.kv[i] = plain.kv["p"]
        near(out[i:i + 1], *plain.run(i, y[i:i + 1]), torch.bfloat16)


def test_a_decoder_that_samples_many_answers_and_scores_them():
    """A toy decoder of one attention layer: a prompt is forked, its continuations decode greedily from different first tokens and are scored; each comes out
    as it does by itself, computed in 64 bits from its whole text."""
    V, H, G, hd, P, n, new = 500, 8, 2, 64, 150, 9, 12
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    emb, w_qkv, w_out = r(V, 128), r(128, (H + 2 * G) * hd) * 128 ** -0.5, r(H * hd, V) * (H * hd) ** -0.5 * 8
    text = torch.randint(0, V, (P,), generator=gen, device="cuda")
    c = SharedCache(H, G, hd, n_pages=64, max_seqs=16, max_len=256, page_size=16, dtype=torch.float32)
    _, seqs = c.fork((emb[text] @ w_qkv).contiguous(), n)
    toks = torch.arange(n, device="cuda", dtype=torch.int32) * 7
    story, scores = [toks], []
    for _ in range(new):
        logits = c.step((emb[story[-1].long()] @ w_qkv).contiguous()) @ w_out
        toks = logits.argmax(1).to(torch.int32)
        got = token_logprobs(logits, toks, 3)
        assert (got.rank == 0).all() and torch.equal(got.top_ids[:, 0], toks)
        scores.append(got.logprob)
        story.append(toks)
    story, scores = torch.stack(story, 1).cpu(), torch.stack(scores, 1).double().cpu().numpy()
    E, Wq, Wo = (t.double().cpu().numpy() for t in (emb, w_qkv, w_out))
    for i in range(n):
        whole = np.concatenate([text.cpu().numpy(), story[i, :-1].numpy()])
        plain = Plain(H, G, hd)
        out, _ = plain.run(0, torch.from_numpy(E[whole] @ Wq))
        x = out[P:] @ Wo
        lp = x - x.max(1, keepdims=True)
        lp -= np.log(np.exp(lp).sum(1, keepdims=True))
        # scores are sums of 512 products of values up to 1e-4 off each, times weights of 0.35: 1e-4 * 8; greedy tokens may differ where two logits are that near
        for t in range(new):
            assert lp[t].max() - lp[t, story[i, t + 1]] <= 2e-3
            assert abs(lp[t, story[i, t + 1]] - scores[i, t]) <= 2e-3
