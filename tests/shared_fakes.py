"""Stand-ins on the CPU, as their documentation has them, for the device calls that a SharedCache makes, and lists of keys and values that its programs
are compared with.  What a call's host bounds leave out comes as NaN."""
import random

import numpy as np
import torch

from kappai_b200 import SharedCache
from kappai_b200.cache import OutOfPages, OutOfSlots


def page_tables(block_table, length, delta, free_pages, n_free, page_size, cu_rows, seg_pos, row_seg, positions, slot_map, status, own_from):
    ps, at, back = page_size, int(n_free), []
    blocks = lambda n: -(-n // ps)  # noqa: E731
    old, after = length.tolist(), []
    for i, (n, d, own) in enumerate(zip(old, delta.tolist(), own_from.tolist())):
        own = min(own, blocks(n))
        a = 0 if n + d <= 0 else (max(n + d, min(n, own * ps)) if d < 0 else n + d)
        after.append(a)
        for b in range(max(blocks(a), own), blocks(n)):
            back.append(int(block_table[i, b]))
        if d < 0:
            block_table[i, blocks(a) if a == 0 else max(blocks(a), own):] = -1
    for page in reversed(back):
        free_pages[at] = page
        at += 1
    row = 0
    for i, (n, d, a) in enumerate(zip(old, delta.tolist(), after)):
        for b in range(blocks(n), blocks(a)):
            assert at > 0, "the caller announced too few pages"
            at -= 1
            block_table[i, b] = free_pages[at]
        cu_rows[i], seg_pos[i] = row, n if d > 0 else a
        for pos in range(n, n + max(d, 0)):
            row_seg[row], positions[row], slot_map[row] = i, pos, int(block_table[i, pos // ps]) * ps + pos % ps
            row += 1
        length[i] = a
    cu_rows[len(old)], n_free[0], status[0] = row, at, 0


def qk_norm_rope_kv(qkv, q_w, k_w, eps, cos, sin, rotary, interleaved, positions, slots, q, pages, page_size, H, G, hd):
    q.copy_(qkv[:, :H * hd])
    kv = qkv[:, H * hd:].reshape(-1, 2, G, hd)
    pages[slots.long() // page_size, :, :, slots.long() % page_size] = kv


def attention_shared(q, cache, block_table, cu_rows, seg_pos, group_seqs, prefix_len, out, scale, page_size, H, G, hd, max_rows, max_group_rows, max_prefix, max_own):
    cu, pos, first, prefix, ps = cu_rows.tolist(), seg_pos.tolist(), group_seqs.tolist(), prefix_len.tolist(), page_size
    assert len(cu) == len(pos) + 1 and len(first) == len(prefix) + 1 and block_table.shape[0] >= len(pos) and out.shape == q.shape
    assert first == sorted(first) and 0 <= first[0] and first[-1] <= len(pos) and max_rows >= 1 and max_group_rows >= 1
    out.fill_(float("nan"))
    for i in range(len(pos)):
        group = next((g for g in range(len(prefix)) if first[g] <= i < first[g + 1]), None)
        P = min(prefix[group], max_prefix) if group is not None else 0
        for r in range(cu[i], cu[i + 1]):
            n = pos[i] + r - cu[i] + 1
            if r - cu[i] >= max_rows or (P and r - cu[first[group]] >= max_group_rows):
                continue
            assert pos[i] >= P, "a row before its prefix' end"
            key = np.arange(n)
            pages = np.where(key < P, block_table[first[group] if P else i].numpy()[key // ps], block_table[i].numpy()[key // ps])
            kv = cache[torch.from_numpy(pages).long(), :, :, torch.from_numpy(key % ps)].double()          # [n, 2, G, hd]
            s = torch.einsum("grd,ngd->grn", q[r].double().reshape(G, H // G, hd), kv[:, 0]) * scale
            out[r] = torch.einsum("grn,ngd->grd", torch.softmax(s, -1), kv[:, 1]).flatten().to(out.dtype)
    return out


def install(monkeypatch):
    """The stand-ins in their places."""
    from kappai_b200.ops import kernels, shared, tables

    monkeypatch.setattr(tables, "page_tables", page_tables)
    monkeypatch.setattr(kernels, "qk_norm_rope_kv", qk_norm_rope_kv)
    monkeypatch.setattr(shared, "attention_shared", attention_shared)


class Program:
    """A SharedCache beside lists of keys and values: every call's rows are compared with attention over those, in 64 bits."""

    def __init__(self, H, G, hd, near, seed=0, device="cpu", **kw):
        self.H, self.G, self.hd, self.near, self.kv, self.prompt_of, self.n_prompts = H, G, hd, near, {}, {}, 0
        self.gen = torch.Generator(device).manual_seed(seed)
        self.c = SharedCache(H, G, hd, device=device if device == "cpu" else "cuda:0", **kw)

    def make(self, n):
        return torch.randn((n, (self.H + 2 * self.G) * self.hd), generator=self.gen, device=self.gen.device).to(self.c.pages.dtype)

    def attend(self, old, x, rows=None):
        """What the rows of x behind the keys ``old`` are to give (of ``rows`` only), with the weighted mean of |v| beside it, and the keys with theirs."""
        x = x.double().cpu()
        H, G, hd = self.H, self.G, self.hd
        q, kv = x[:, :H * hd].reshape(-1, G, H // G, hd), x[:, H * hd:].reshape(-1, 2, G, hd)
        whole = kv if old is None else torch.cat([old, kv])
        out, off = [], []
        for r in range(len(x)) if rows is None else rows:
            n = len(whole) - len(x) + r + 1
            p = torch.softmax(torch.einsum("grd,ngd->grn", q[r], whole[:n, 0]) * hd ** -0.5, -1)
            out.append(torch.einsum("grn,ngd->grd", p, whole[:n, 1]).flatten())
            off.append(torch.einsum("grn,ngd->grd", p, whole[:n, 1].abs()).flatten() + out[-1].abs())
        return torch.stack(out), torch.stack(off), whole

    def check(self):
        self.c.check()
        assert self.c.live() == sorted(self.kv) and [self.c.length(s) for s in self.c.live()] == [len(self.kv[s]) for s in self.c.live()]

    def fork(self, P, n):
        x = self.make(P)
        out, seqs = self.c.fork(x, n)
        want, off, whole = self.attend(None, x)
        self.near(out, want, off)
        assert not set(seqs) & set(self.kv)
        for s in seqs:
            self.kv[s], self.prompt_of[s] = whole, (self.n_prompts, P)
        self.n_prompts += 1
        self.check()
        return seqs

    def step(self, seqs=None, rows=None):
        ids = self.c.live() if seqs is None else seqs
        rows = rows or [1] * len(ids)
        x, at = self.make(sum(rows)), 0
        out = self.c.step(x, seqs, rows)
        for s, r in zip(ids, rows):
            want, off, self.kv[s] = self.attend(self.kv[s], x[at:at + r])
            self.near(out[at:at + r], want, off)
            at += r
        self.check()

    def take_back(self, seqs, tokens):
        self.c.take_back(seqs, tokens)
        for s, t in zip(seqs, tokens):
            self.kv[s] = self.kv[s][:len(self.kv[s]) - t]
        self.check()

    def end(self, seqs):
        self.c.end(seqs)
        for s in seqs:
            del self.kv[s], self.prompt_of[s]
        self.check()

    def random(self, seed, calls, longest, most):
        """Forks of up to ``longest`` tokens into up to ``most`` continuations, steps of some, drafts taken back, some ended, until the calls are made."""
        rng = random.Random(seed)
        some = lambda: sorted(rng.sample(self.c.live(), rng.randint(1, len(self.c.live()))))  # noqa: E731
        refused = 0
        for _ in range(calls):
            what = rng.choice(["fork", "fork", "step", "step", "step", "take_back", "end", "end"]) if self.kv else "fork"
            before = self.c.pages_free
            try:
                if what == "fork":
                    self.fork(rng.randint(1, longest), rng.randint(1, most))
                elif what == "step":
                    seqs = some()
                    self.step(*(rng.choice([(None, None), (seqs, [rng.choice([1, 1, rng.randint(1, 5)]) for _ in seqs])])))
                elif what == "take_back":
                    seqs = some()
                    self.take_back(seqs, [rng.randint(0, min(7, len(self.kv[s]) - self.prompt_of[s][1])) for s in seqs])
                else:
                    self.end(some())
            except (OutOfPages, OutOfSlots):
                refused += 1
                assert self.c.pages_free == before
                self.check()
                if self.kv:
                    self.end(some())
        self.end(self.c.live())
        assert self.c.pages_free == self.c.n_pages
        return refused
