"""One attention layer's keys and values for prompts with many continuations each: the prompt's pages are held once.

A :class:`SharedCache` runs the layer's attention for programs of one's own: ``fork`` runs a prompt and makes continuations of it, ``step`` gives
continuations their next rows, ``take_back`` drops their last ones (drafts that were refused), ``end`` ends them.  The block tables, lengths and the stack of
free pages lie on the device, where :func:`~kappai_b200.ops.tables.page_tables` moves them; the host counts along and knows no page's number.  A
prompt's keys are read once for all of its continuations' rows (:func:`~kappai_b200.ops.shared.attention_shared`).

Keys are stored as they are given: with a rotary encoding, rotated before they come here.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .kv4 import _on_its_device
from .manager import CacheError, OutOfPages, OutOfSlots


class SharedCache:
    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, n_pages: int, max_seqs: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda:0"):
        """``n_pages`` pages of ``page_size`` keys; at most ``max_seqs`` sequences at a time, each prompt and each continuation one of them, of at most
        ``max_len`` tokens, the prompt's among them."""
        from ..ops.kernels import MAX_STEP_ROWS
        from ..ops.shared import SHARED_HEAD_DIMS, SHARED_MAX_KEYS
        from ..ops.tables import MAX_TABLE_SEQS

        if num_kv_heads < 1 or num_heads < 1 or num_heads % num_kv_heads or head_dim not in SHARED_HEAD_DIMS:
            raise CacheError(f"{num_heads} query heads over {num_kv_heads} kv heads of {head_dim} values; head sizes are {SHARED_HEAD_DIMS}")
        if min(n_pages, max_seqs, max_len, page_size) < 1 or max_seqs > MAX_TABLE_SEQS:
            raise CacheError(f"n_pages={n_pages}, max_seqs={max_seqs} (at most {MAX_TABLE_SEQS}), max_len={max_len} and page_size={page_size} must be positive")
        width = -(-max_len // page_size)
        if n_pages * page_size >= 1 << 31 or width * page_size > SHARED_MAX_KEYS or max_seqs * width >= (1 << 31) - 1:
            raise CacheError(f"{n_pages} pages of {page_size} keys for {max_seqs} sequences of {max_len}: slots and keys are 32-bit numbers")
        if dtype not in (torch.float32, torch.bfloat16):
            raise CacheError(f"dtype {dtype}: expected float32 or bfloat16")
        self.H, self.G, self.hd, self.page_size, self.max_len, self.n_pages = int(num_heads), int(num_kv_heads), int(head_dim), int(page_size), int(max_len), int(n_pages)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._most = MAX_STEP_ROWS
        i32 = dict(dtype=torch.int32, device=self.device)
        self.pages = torch.zeros((n_pages, 2, self.G, self.page_size, self.hd), dtype=dtype, device=self.device)
        self.block_table = torch.full((max_seqs, width), -1, **i32)
        self.lengths, self.own_from = torch.zeros(max_seqs, **i32), torch.zeros(max_seqs, **i32)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, **i32)              # (the lowest number is taken first)
        self.n_free, self.status = torch.full((1,), n_pages, **i32), torch.zeros(1, **i32)
        self._cu, self._pos = torch.zeros(max_seqs + 1, **i32), torch.zeros(max_seqs, **i32)
        # the host's count
        self._length, self._own, self._prompt = [0] * max_seqs, [0] * max_seqs, [-1] * max_seqs       # (a sequence's prompt; its own number: it is one)
        self._groups: Dict[int, List[int]] = {}                     # prompt -> its live continuations
        self._free = self.n_pages

    # -- questions
    def length(self, seq: int) -> int:
        """Keys of a continuation, its prompt's among them."""
        self._check([seq], "length")
        return self._length[seq]

    def live(self) -> List[int]:
        """The continuations that there are, in the order in which a step takes their rows."""
        return sorted(s for c in self._groups.values() for s in c)

    @property
    def pages_free(self) -> int:
        return self._free

    def _check(self, seqs: Sequence[int], what: str) -> None:
        if list(seqs) != sorted(set(seqs)):
            raise CacheError(f"{what}: every continuation once, in ascending order")
        for s in seqs:
            if not (0 <= s < len(self._prompt)) or self._prompt[s] < 0 or self._prompt[s] == s:
                raise CacheError(f"{what}: no continuation {s!r}")

    def _blocks(self, n: int) -> int:
        return -(-n // self.page_size)

    # -- changes
    def _move(self, change: Dict[int, int], n_rows: int, beside: Sequence[int] = ()):
        """The lengths' step on the device, and the same on the host: (positions, slots) of its rows, and the numbers ``beside``, which go to the
        device in the same copy."""
        from ..ops.tables import page_tables

        n_seq = len(self._length)
        numbers = np.zeros(n_seq + len(beside), dtype=np.int32)
        for s, d in change.items():
            numbers[s] = d
        numbers[n_seq:] = beside
        numbers = self._upload(numbers)
        delta_d = numbers[:n_seq]
        row_seg, positions, slots = torch.empty((3, n_rows), dtype=torch.int32, device=self.device).unbind(0)
        page_tables(self.block_table, self.lengths, delta_d, self.free_pages, self.n_free, self.page_size, self._cu, self._pos, row_seg, positions, slots,
                    self.status, own_from=self.own_from)
        for s, d in change.items():
            before, self._length[s] = self._blocks(self._length[s]), self._length[s] + d
            self._free -= max(self._blocks(self._length[s]), self._own[s]) - max(before, self._own[s])
        return positions, slots, numbers[n_seq:]

    def _forget(self, over: Sequence[int]) -> None:
        """These sequences are no more, whatever they had got."""
        index = self._upload(np.asarray(over)).long()
        self._move({s: -self._length[s] for s in over if self._length[s]}, 0)
        self.own_from.index_fill_(0, index, 0)
        for s in over:
            self._own[s], self._prompt[s] = 0, -1

    def _upload(self, a) -> torch.Tensor:
        t = torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32))
        return t.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else t

    def _room(self, pages: int) -> None:
        if pages > self._free:
            raise OutOfPages(f"need {pages} pages, {self._free} free")

    def _attend(self, qkv, out, positions, slots, scale, lo: int, hi: int, **bounds) -> torch.Tensor:
        """The rows' attention into ``out``; ``lo`` to ``hi`` - 1 are the sequences that may have any, and groups count from ``lo``."""
        from ..ops.kernels import qk_norm_rope_kv
        from ..ops.shared import attention_shared

        H, G, hd = self.H, self.G, self.hd
        q = self._out(qkv)
        qk_norm_rope_kv(qkv, None, None, 0.0, None, None, 0, False, positions, slots, q, self.pages, self.page_size, H, G, hd)
        return attention_shared(q, self.pages, self.block_table[lo:hi], self._cu[lo:hi + 1], self._pos[lo:hi], out=out, scale=scale,
                                page_size=self.page_size, H=H, G=G, hd=hd, **bounds)

    def _scale(self, scale: Optional[float], what: str) -> float:
        if scale is None:
            return self.hd ** -0.5
        if not 0.0 < scale < float("inf"):
            raise CacheError(f"{what}: the scale is a positive number, got {scale}")
        return scale

    def _rows(self, qkv: torch.Tensor, n: int, what: str) -> None:
        w = (self.H + 2 * self.G) * self.hd
        if not isinstance(qkv, torch.Tensor) or qkv.device != self.device or qkv.dtype != self.pages.dtype or tuple(qkv.shape) != (n, w) or qkv.stride(1) != 1:
            raise CacheError(f"{what}: rows [{n}, {w}] of queries, keys and values in {self.pages.dtype} on {self.device} were announced, got "
                             f"{tuple(qkv.shape) if isinstance(qkv, torch.Tensor) else qkv!r}")

    def _out(self, qkv: torch.Tensor) -> torch.Tensor:
        return torch.empty((qkv.shape[0], self.H * self.hd), dtype=qkv.dtype, device=qkv.device)

    # -- the operators
    @_on_its_device
    def fork(self, qkv: torch.Tensor, n: int, scale: Optional[float] = None) -> Tuple[torch.Tensor, List[int]]:
        """A prompt's rows [tokens, (num_heads + 2 num_kv_heads) * head_dim] (queries, keys, values; as many as there are), and ``n`` continuations of it: the rows'
        causal attention [tokens, num_heads * head_dim], and the continuations' numbers.  ``scale``: head_dim ** -0.5 unless given.  Nothing is taken
        by a call that fails, for instance where the pages do not suffice (:class:`~.manager.OutOfPages`) or fewer than ``n + 1`` sequences are free
        (:class:`~.manager.OutOfSlots`)."""
        P = qkv.shape[0] if isinstance(qkv, torch.Tensor) and qkv.dim() == 2 else 0
        if P < 1 or n < 1 or P > self.max_len:
            raise CacheError(f"fork: a prompt of {P} tokens (at most {self.max_len}) with {n} continuations")
        self._rows(qkv, P, "fork")
        scale = self._scale(scale, "fork")
        whole, tail = divmod(P, self.page_size)
        self._room(self._blocks(P) + (n if tail else 0))
        free = [s for s, p in enumerate(self._prompt) if p < 0]
        if len(free) <= n:
            raise OutOfSlots(f"need {n + 1} sequences, {len(free)} are free")
        # (in a row where there are so many: a step reads a prompt once for each stretch of its continuations)
        first = next((i for i in range(len(free) - n) if free[i + n] - free[i] == n), 0)
        at, seqs = free[first], free[first + 1:first + 1 + n]
        try:
            none, out = self._upload(np.zeros(1)), self._out(qkv)
            for a in range(0, P, self._most):                       # (as many rows as a call takes)
                b = min(P, a + self._most)
                positions, slots, _ = self._move({at: b - a}, b - a)
                self._attend(qkv[a:b], out[a:b], positions, slots, scale, at, at + 1, group_seqs=none, prefix_len=none[:0], max_rows=b - a,
                             max_group_rows=b - a, max_prefix=0, max_own=b)
            # the continuations' tables begin with the prompt's whole pages; a page that it ends in each has for itself
            rows = self._upload(np.asarray(seqs)).long()
            self.block_table[rows, :whole] = self.block_table[at, :whole]
            self.own_from.index_fill_(0, rows, whole)
            self.lengths.index_fill_(0, rows, whole * self.page_size)
            for s in seqs:
                self._length[s], self._own[s] = whole * self.page_size, whole
            if tail:
                for a in range(0, tail, self._most):
                    rows_each = min(tail - a, self._most)
                    for i in range(0, n, self._most // rows_each):
                        part = seqs[i:i + self._most // rows_each]
                        self._move({s: rows_each for s in part}, len(part) * rows_each)
                self.pages[self.block_table[rows, whole].long(), :, :, :tail] = self.pages[self.block_table[at, whole].long(), :, :, :tail]
        except BaseException:
            self._forget([at] + seqs)
            raise
        for s in [at] + seqs:
            self._prompt[s] = at
        self._groups[at] = seqs
        return out, list(seqs)

    @_on_its_device
    def step(self, qkv: torch.Tensor, seqs: Optional[Sequence[int]] = None, rows: Optional[Sequence[int]] = None, scale: Optional[float] = None) -> torch.Tensor:
        """The next ``rows[i]`` (None: one each) tokens of ``seqs[i]`` (None: all that are live; ascending): their keys and values join the cache, and what is
        returned is each row's causal attention over its prompt and its own continuation, [rows, num_heads * head_dim].  All get their pages or
        none does, and a call that fails leaves everything as it was."""
        seqs = self.live() if seqs is None else list(seqs)
        self._check(seqs, "step")
        rows = [1] * len(seqs) if rows is None else [int(r) for r in rows]
        if len(rows) != len(seqs) or min(rows, default=1) < 1:
            raise CacheError("step: a positive number of rows for every continuation")
        self._rows(qkv, sum(rows), "step")
        if sum(rows) > self._most:
            raise CacheError(f"step: {sum(rows)} rows, a call takes {self._most}")
        scale = self._scale(scale, "step")
        if not seqs:
            return qkv[:, :self.H * self.hd].clone()
        after = [self._length[s] + r for s, r in zip(seqs, rows)]
        if max(after) > self.max_len:
            raise CacheError(f"step: a continuation of {max(after)} tokens, max_len={self.max_len}")
        self._room(sum(self._blocks(a) - max(self._blocks(self._length[s]), self._own[s]) for a, s in zip(after, seqs)))
        # Groups: stretches of these continuations that are of one prompt.  (A prompt that was forked into the places which ended continuations left stands
        # among another's; what lies between a stretch's members, and up to the next stretch, has no rows.)
        prompts = [self._prompt[s] for s in seqs]
        starts, group_rows = [], []
        for i, r in enumerate(rows):
            if not i or prompts[i] != prompts[i - 1]:
                starts.append(i)
                group_rows.append(0)
            group_rows[-1] += r
        prefix, lo, hi = [self._length[prompts[i]] for i in starts], seqs[0], seqs[-1] + 1
        positions, slots, groups = self._move(dict(zip(seqs, rows)), sum(rows), [seqs[i] - lo for i in starts] + [hi - lo] + prefix)
        try:
            return self._attend(qkv, self._out(qkv), positions, slots, scale, lo, hi, group_seqs=groups[:len(starts) + 1], prefix_len=groups[len(starts) + 1:],
                                max_rows=max(rows), max_group_rows=max(group_rows), max_prefix=max(prefix),
                                max_own=max(a - self._length[p] for a, p in zip(after, prompts)))
        except BaseException:
            self._move({s: -r for s, r in zip(seqs, rows)}, 0)
            raise

    @_on_its_device
    def take_back(self, seqs: Sequence[int], tokens: Sequence[int]) -> None:
        """The last ``tokens[i]`` tokens of ``seqs[i]`` (ascending) are dropped, none of its prompt's; pages that hold nothing then come back."""
        self._check(seqs, "take_back")
        if len(tokens) != len(seqs):
            raise CacheError("take_back: a number of tokens for every continuation")
        for s, t in zip(seqs, tokens):
            if t < 0 or t > self._length[s] - self._length[self._prompt[s]]:
                raise CacheError(f"take_back: {t} tokens of continuation {s}, which has {self._length[s] - self._length[self._prompt[s]]} behind its prompt")
        change = {s: -int(t) for s, t in zip(seqs, tokens) if t}
        if change:
            self._move(change, 0)

    @_on_its_device
    def end(self, seqs: Sequence[int]) -> None:
        """These continuations (ascending) are no more; with a prompt's last one its own pages come back too."""
        self._check(seqs, "end")
        gone = set(seqs)
        prompts = [p for p, c in self._groups.items() if gone.issuperset(c)]
        over = sorted(gone) + prompts
        if not over:
            return
        kept = {p: [s for s in c if s not in gone] for p, c in self._groups.items() if p not in prompts}
        self._forget(over)
        self._groups = kept

    def check(self) -> None:
        """The device's count is the host's, and no page is lost or held twice (synchronises; for tests and doubts)."""
        if int(self.status) or self.lengths.tolist() != self._length or int(self.n_free) != self._free:
            raise CacheError(f"the device counts otherwise: status {int(self.status)}, {int(self.n_free)} pages free, {self._free} expected")
        held = self.free_pages[:self._free].tolist()
        for table, n, own in zip(self.block_table.tolist(), self._length, self._own):
            held += table[own:self._blocks(n)]
        if sorted(held) != list(range(self.n_pages)):
            raise CacheError("pages lost, or held twice")
