"""One attention layer's keys and values in 4 bits, for several sequences, with eviction by the weight that keys got.

A :class:`Kv4Cache` owns the pages (``csrc/kv4.cuh`` has their bytes), who holds which (a :class:`~.manager.PagePool`), and, where
``mass`` is asked for, how much softmax weight every cached key has got so far.  Sequences grow by ``append``, are read by
``attend`` and shrink by ``evict``; all rows of a call run together, whatever their sequences' lengths.

Keys are stored as they are given: with a rotary encoding they are rotated before they come here, so a key that moves to another
place by an eviction keeps the position it was written with.  The causal order is that of the cache: a row reads the keys that were there
before it.
"""
from __future__ import annotations

from functools import wraps
from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .manager import CacheError, PagePool


def _on_its_device(method):
    """The cache's device is the current one while a method of it runs: launches go to that device's current stream."""
    @wraps(method)
    def run(self, *args, **kw):
        if self.device.type != "cuda":
            return method(self, *args, **kw)
        with torch.cuda.device(self.device):
            return method(self, *args, **kw)

    return run


class Kv4Cache:
    def __init__(self, num_kv_heads: int, head_dim: int, n_pages: int, page_size: int = 64, mass: bool = False, device="cuda:0"):
        """``n_pages`` pages of ``page_size`` keys (a power of two, at least 16) for all sequences together.  An eviction holds the old pages and
        the new ones for as long as the keys take to move."""
        from ..ops.kv4 import kv4_page_bytes

        if num_kv_heads < 1:
            raise CacheError(f"num_kv_heads={num_kv_heads} must be positive")
        self.G, self.hd, self.page_size = int(num_kv_heads), int(head_dim), int(page_size)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        record = kv4_page_bytes(self.page_size, self.hd)
        if n_pages * self.page_size >= 1 << 31:
            raise CacheError(f"{n_pages} pages of {self.page_size} keys: slots are 32-bit numbers, below 2^31")
        self.pool = PagePool(n_pages, self.page_size)
        self.pages = torch.zeros((n_pages, self.G, record), dtype=torch.uint8, device=self.device)
        self.mass: Optional[torch.Tensor] = None
        if mass:
            self.mass = torch.zeros((n_pages, self.G, self.page_size), dtype=torch.float32, device=self.device)
        self._length: Dict[Hashable, int] = {}

    # -- sequences
    def add(self, seq: Hashable) -> None:
        self.pool.open(seq)
        self._length[seq] = 0

    def free(self, seq: Hashable) -> None:
        """The sequence has ended: its pages are given back."""
        self.pool.close(seq)
        del self._length[seq]

    def length(self, seq: Hashable) -> int:
        """Keys that the sequence has in the cache."""
        return self._length[seq]

    def bytes_per_token(self) -> int:
        """Bytes of a token's keys and values in all kv heads (without what ``mass`` takes)."""
        return self.pages.shape[1] * self.pages.shape[2] // self.page_size

    # -- tables of a call, brought to the device by one copy
    def _upload(self, arrays: Sequence[np.ndarray]) -> List[torch.Tensor]:
        flat = torch.from_numpy(np.concatenate([np.ascontiguousarray(a, dtype=np.int32).reshape(-1) for a in arrays]))
        if self.device.type == "cuda":
            flat = flat.pin_memory().to(self.device, non_blocking=True)
        out, at = [], 0
        for a in arrays:
            out.append(flat[at:at + a.size].view(a.shape))
            at += a.size
        return out

    def _table(self, seqs: Sequence[Hashable]) -> np.ndarray:
        tables = [self.pool.table(s) for s in seqs]
        t = np.zeros((len(seqs), max(1, max(map(len, tables), default=1))), dtype=np.int32)
        for i, pages in enumerate(tables):
            t[i, :len(pages)] = pages
        return t

    def _slots(self, seq: Hashable, a: int, b: int) -> np.ndarray:
        """Slots of keys a .. b - 1 of a sequence."""
        key = np.arange(a, b)
        return np.asarray(self.pool.table(seq), dtype=np.int64)[key // self.page_size] * self.page_size + key % self.page_size

    def _check(self, seqs: Sequence[Hashable], rows: Sequence[int], what: str) -> None:
        if len(seqs) != len(rows) or len(set(seqs)) != len(seqs):
            raise CacheError(f"{what}: every sequence once, with a number of rows each")
        for s, n in zip(seqs, rows):
            if s not in self._length:
                raise CacheError(f"{what}: no sequence {s!r}")
            if n < 1:
                raise CacheError(f"{what}: {n} rows of sequence {s!r}")

    # -- the three operators
    @_on_its_device
    def append(self, k: torch.Tensor, v: torch.Tensor, seqs: Sequence[Hashable], rows: Sequence[int]) -> None:
        """The next ``rows[i]`` keys and values of ``seqs[i]``: k and v are [sum of rows, num_kv_heads * head_dim], float32 or bfloat16,
        possibly columns of a wider product.  All sequences get their pages or none does (:class:`~.manager.OutOfPages`)."""
        from ..ops.kv4 import kv4_write

        self._check(seqs, rows, "append")
        need = sum(self.pool.pages_needed(s, self._length[s] + n) for s, n in zip(seqs, rows))
        if need > self.pool.n_free:
            from .manager import OutOfPages

            raise OutOfPages(f"need {need} pages, {self.pool.n_free} free")
        if k.shape[0] != sum(rows):
            raise CacheError(f"append: {k.shape[0]} rows of keys, {sum(rows)} were announced")
        if not seqs:
            return
        held = [len(self.pool.table(s)) for s in seqs]
        try:
            for s, n in zip(seqs, rows):
                self.pool.extend(s, self._length[s] + n)
            fresh = [page for s, h in zip(seqs, held) for page in self.pool.table(s)[h:]]
            slots = np.concatenate([self._slots(s, self._length[s], self._length[s] + n) for s, n in zip(seqs, rows)])
            slots_d, fresh_d = self._upload([slots, np.asarray(fresh, dtype=np.int32)])
            if self.mass is not None and fresh:
                self.mass.index_fill_(0, fresh_d.long(), 0.0)                    # (a page may have been another sequence's)
            kv4_write(k, v, self.pages, slots_d, self.page_size, self.G, self.hd)
        except BaseException:
            for s, h in reversed(list(zip(seqs, held))):
                self.pool.cut(s, h)
            raise
        for s, n in zip(seqs, rows):
            self._length[s] += n

    @_on_its_device
    def attend(self, q: torch.Tensor, seqs: Sequence[Hashable], rows: Sequence[int], num_heads: int, scale: float,
               window: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the last ``rows[i]`` tokens of ``seqs[i]`` (their keys and values have been appended): q is [sum of rows,
        num_heads * head_dim], the heads that share a kv head beside one another.  Where the cache keeps ``mass``, the weight that
        every key gets, summed over the rows and over the heads of its kv head, is added to it.  ``window`` counts places of the cache: after an
        eviction these are the keys that stayed, which differ from head to head, and no longer positions of the text."""
        from ..ops.kv4 import kv4_attention

        self._check(seqs, rows, "attend")
        past = [self._length[s] - n for s, n in zip(seqs, rows)]
        if min(past, default=0) < 0:
            raise CacheError("attend: more rows than keys; append them first")
        if q.dim() != 2 or q.shape[0] != sum(rows):
            raise CacheError(f"attend: {sum(rows)} rows of queries were announced, got a tensor of shape {tuple(q.shape)}")
        out = torch.empty((q.shape[0], q.shape[1]), dtype=q.dtype, device=q.device) if out is None else out
        if not seqs:
            return out
        cu, pos, table = self._upload([np.concatenate([[0], np.cumsum(rows)]), np.asarray(past), self._table(seqs)])
        return kv4_attention(q, self.pages, table, cu, pos, out, scale, window, self.page_size, num_heads, self.G, self.hd, max(rows),
                             max(p + n for p, n in zip(past, rows)), min_rows=min(rows), mass=self.mass)

    @_on_its_device
    def evict(self, seqs: Sequence[Hashable], keep: int, recent: int = 0, first: int = 0) -> torch.Tensor:
        """Of each sequence every kv head keeps ``keep`` keys: the ``first`` first, the ``recent`` last and those with the most mass of the
        others; a sequence that has no more keeps all.  Returns the indices that the kept keys had, int32 [sequences, kv heads, keep],
        -1 behind the last.  Needs free pages for the keys that stay."""
        from ..ops.kv4 import kv4_evict
        from .manager import OutOfPages

        if self.mass is None:
            raise CacheError("evict: this cache keeps no mass (mass=True)")
        self._check(seqs, [1] * len(seqs), "evict")
        kept = torch.full((len(seqs), self.G, keep), -1, dtype=torch.int32, device=self.device)
        todo = [s for s in seqs if self._length[s] > 0]
        stay = [min(self._length[s], keep) for s in todo]
        if sum(map(self.pool.pages_for, stay)) > self.pool.n_free:
            raise OutOfPages(f"need {sum(map(self.pool.pages_for, stay))} pages for the keys that stay, {self.pool.n_free} free")
        if not todo:
            return kept
        old = self._table(todo)
        moved = [("moved", s) for s in todo]
        for m, n in zip(moved, stay):
            self.pool.open(m)
            self.pool.extend(m, n)
        lengths = np.asarray([self._length[s] for s in todo])
        new = self._table(moved)
        old_d, new_d, len_d = self._upload([old, new, lengths])
        part = kept if len(todo) == len(seqs) else torch.full((len(todo), self.G, keep), -1, dtype=torch.int32, device=self.device)
        try:
            # places behind the last key of a page hold nothing yet
            fresh = torch.from_numpy(np.unique(np.concatenate([self.pool.table(m) for m in moved]))).to(self.device)
            self.mass.index_fill_(0, fresh, 0.0)
            kv4_evict(self.pages, self.mass, old_d, len_d, self.pages, self.mass, new_d, part, int(lengths.max()), keep, recent, first, self.page_size,
                      self.G, self.hd)
        except Exception:
            for m in moved:
                self.pool.close(m)
            raise
        for s, m, n in zip(todo, moved, stay):
            self.pool.take_over(s, m)
            self._length[s] = n
        if part is not kept:
            kept[torch.tensor([i for i, s in enumerate(seqs) if self._length[s] > 0], device=self.device)] = part
        return kept

    @_on_its_device
    def read(self, seq: Hashable, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The sequence's keys and values as the cache holds them, [length, num_kv_heads * head_dim]."""
        from ..ops.kv4 import kv4_read

        if seq not in self._length:
            raise CacheError(f"read: no sequence {seq!r}")
        slots, = self._upload([self._slots(seq, 0, self._length[seq])])
        return kv4_read(self.pages, slots, self.page_size, self.G, self.hd, dtype)

    @_on_its_device
    def mass_of(self, seq: Hashable) -> torch.Tensor:
        """The weight that the sequence's keys have got, [kv heads, length] (float32)."""
        if self.mass is None:
            raise CacheError("mass_of: this cache keeps no mass (mass=True)")
        if seq not in self._length:
            raise CacheError(f"mass_of: no sequence {seq!r}")
        table = torch.from_numpy(np.asarray(self.pool.table(seq), dtype=np.int64)).to(self.device)
        return self.mass[table].transpose(0, 1).reshape(self.G, -1)[:, :self._length[seq]]
