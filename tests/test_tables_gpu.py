"""Tables made on the GPU against a plain walk over the sequences in Python: whole numbers, compared for equality."""
import random

import numpy as np
import pytest
import torch

from kappai_b200.ops.kernels import KernelError
from kappai_b200.ops.tables import page_tables

pytestmark = pytest.mark.gpu


class Plain:
    """Lists of pages, one sequence after the other."""

    def __init__(self, lengths, ps, width, n_pages, seed=0, shared=None):
        rng = random.Random(seed)
        pages = list(range(n_pages))
        rng.shuffle(pages)
        self.ps, self.width, self.n_pages = ps, width, n_pages
        self.length, self.own = list(lengths), list(shared or [0] * len(lengths))
        self.table = [[pages.pop() for _ in range(-(-n // ps))] for n in lengths]
        self.free = pages

    def device(self, cap):
        S = len(self.length)
        t = np.full((S, self.width), -1, dtype=np.int32)
        for i, row in enumerate(self.table):
            t[i, :len(row)] = row
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        new = lambda n: torch.full((n,), -77, dtype=torch.int32, device="cuda")  # noqa: E731
        return {"block_table": i32(t), "length": i32(self.length), "free_pages": i32(self.free + [-9] * (self.n_pages - len(self.free))),
                "n_free": i32([len(self.free)]), "cu_rows": new(S + 1), "seg_pos": new(S), "row_seg": new(cap), "positions": new(cap), "slot_map": new(cap),
                "status": new(1), "own_from": i32(self.own)}

    def step(self, delta, cap):
        """The step's status and tables; the pages and lengths move if it can be made."""
        ps = self.ps
        after, status = [], 0
        for n, d, own, row in zip(self.length, delta, self.own, self.table):
            a = 0 if n + d <= 0 else (min(n, max(n + d, min(own, len(row)) * ps)) if d < 0 else n + d)
            after.append(a)
            if -(-a // ps) > self.width:
                status |= 2
        fits = [(-(-a // ps), len(row)) if -(-a // ps) <= self.width else (len(row), len(row)) for a, row in zip(after, self.table)]
        back = sum(max(0, o - max(n, min(own, o))) for (n, o), own in zip(fits, self.own) if n < o)
        if sum(max(0, n - o) for n, o in fits) > len(self.free) + back:
            status |= 1
        if sum(max(d, 0) for d, (n, o), a in zip(delta, fits, after) if -(-a // ps) <= self.width) > cap:
            status |= 4
        cu, pos, rows = [0], [], []
        if status:
            return status, [0] * (len(delta) + 1), list(self.length), []
        came = []
        for i, a in enumerate(after):
            blocks = -(-a // ps)
            if blocks < len(self.table[i]):
                own = min(self.own[i], len(self.table[i]))
                came += self.table[i][max(blocks, own):]
                self.table[i] = self.table[i][:0 if a == 0 and self.length[i] + delta[i] <= 0 else max(blocks, own)]
        self.free += came[::-1]
        for i, a in enumerate(after):
            while len(self.table[i]) < -(-a // ps):
                self.table[i].append(self.free.pop())
            d = max(delta[i], 0)
            for p in range(self.length[i], self.length[i] + d):
                rows.append((i, p, self.table[i][p // ps] * ps + p % ps))
            pos.append(self.length[i] if d else a)
            cu.append(cu[-1] + d)
            self.length[i] = a
        return 0, cu, pos, rows


def run(dev, delta, ps):
    d = torch.tensor(delta, dtype=torch.int32, device="cuda")
    page_tables(dev["block_table"], dev["length"], d, dev["free_pages"], dev["n_free"], ps, dev["cu_rows"], dev["seg_pos"], dev["row_seg"], dev["positions"],
                dev["slot_map"], dev["status"], own_from=dev["own_from"])


def check(plain, dev, delta, cap, ps):
    status, cu, pos, rows = plain.step(delta, cap)
    run(dev, delta, ps)
    host = {k: v.tolist() for k, v in dev.items()}
    assert host["status"] == [status]
    assert host["cu_rows"] == cu and host["seg_pos"] == pos
    pad = cap - len(rows)
    assert host["row_seg"] == [r[0] for r in rows] + [0] * pad
    assert host["positions"] == [r[1] for r in rows] + [-1] * pad
    assert host["slot_map"] == [r[2] for r in rows] + [-1] * pad
    assert host["length"] == plain.length and host["n_free"] == [len(plain.free)]
    assert host["free_pages"][:len(plain.free)] == plain.free
    assert host["block_table"] == [row + [-1] * (plain.width - len(row)) for row in plain.table]
    return status


@pytest.mark.parametrize("S,ps,longest,cap", [(1, 64, 200, 64), (7, 1, 30, 50), (64, 16, 500, 64), (65, 3, 100, 2000), (1500, 16, 300, 5000), (33, 100, 1000, 65535),
                                              (8192, 64, 150, 9000)])
def test_steps_of_many_kinds(S, ps, longest, cap):
    """Sequences grow, are cut back and end, some with shared first blocks, for several steps; then every step is taken back."""
    rng = random.Random(S + ps)
    lengths = [rng.choice([0, 1, ps, rng.randint(0, longest)]) for _ in range(S)]
    own = [rng.choice([0, 0, n // ps, n // ps // 2, 3]) for n in lengths]
    width = -(-longest // ps) + 6
    plain = Plain(lengths, ps, width, S * width, seed=S, shared=own)
    dev = plain.device(cap)
    for step in range(4):
        room = max(1, min(3 * ps, cap // S))
        delta = [rng.choice([1, 1, 0, rng.randint(1, room), -1, -rng.randint(1, 3 * ps), -n]) for n in plain.length]
        while sum(max(d, 0) for d in delta) > cap:
            delta = [d if d <= 0 else d // 2 for d in delta]
        check(plain, dev, delta, cap, ps)


def test_a_step_taken_back_leaves_the_stack_as_it_was():
    plain = Plain([5, 0, 64, 63, 200, 17], 16, 40, 200, seed=3)
    dev = plain.device(400)
    before = {k: v.clone() for k, v in dev.items()}
    for delta in ([1, 1, 1, 1, 1, 1], [40, 70, -3, 1, -200, -17], [-5, 3, -64, 0, 20, 99]):
        check(plain, dev, delta, 400, 16)
        check(plain, dev, [-d for d in delta], 400, 16)
        for k in ("block_table", "length", "n_free"):
            assert torch.equal(dev[k], before[k])
        n = int(dev["n_free"])
        assert torch.equal(dev["free_pages"][:n], before["free_pages"][:n])


@pytest.mark.parametrize("delta,cap,want", [([50, 1], 100, 1), ([70, 1], 100, 3), ([1, 8], 8, 4), ([2 ** 31 - 1, 2 ** 31 - 1], 100, 2), ([200, 200], 30, 2), ([1, 30], 100, 1), ([1, 29], 100, 0)])
def test_a_step_that_cannot_be_made_changes_nothing(delta, cap, want):
    plain = Plain([16, 3], 16, 5, 4, seed=1)
    dev = plain.device(cap)
    before = {k: dev[k].clone() for k in ("block_table", "length", "n_free", "free_pages")}
    if want == 3:
        plain.width, dev = 4, {**dev, "block_table": dev["block_table"][:, :4].contiguous()}
        before["block_table"] = dev["block_table"].clone()
        want = 2
    assert check(plain, dev, delta, cap, 16) == want
    if want:
        for k, v in before.items():
            assert torch.equal(dev[k], v)


@pytest.mark.parametrize("what,value", [("length", -1), ("length", 200), ("own_from", -2), ("n_free", -1), ("n_free", 21)])
def test_numbers_that_make_no_sense(what, value):
    plain = Plain([16, 3], 16, 5, 20, seed=1)
    dev = plain.device(30)
    dev[what][0] = value
    before = {k: v.clone() for k, v in dev.items()}
    run(dev, [1, 1], 16)
    assert int(dev["status"]) & 8 and dev["cu_rows"].tolist() == [0, 0, 0] and dev["slot_map"].tolist() == [-1] * 30
    for k in ("block_table", "length", "n_free", "free_pages"):
        assert torch.equal(dev[k], before[k])


def test_no_sequences_and_no_rows():
    plain = Plain([], 16, 4, 8)
    dev = plain.device(5)
    check(plain, dev, [], 5, 16)
    plain = Plain([30, 20], 16, 4, 8)
    dev = plain.device(0)
    check(plain, dev, [-3, -20], 0, 16)


def test_captured_decode_steps():
    """A captured step of one more token a sequence, replayed: lengths and pages live on the device."""
    plain = Plain([15, 1, 0, 47], 16, 10, 40, seed=5)
    dev = plain.device(6)
    d = torch.ones(4, dtype=torch.int32, device="cuda")
    keep = {k: v.clone() for k, v in dev.items()}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        page_tables(dev["block_table"], dev["length"], d, dev["free_pages"], dev["n_free"], 16, dev["cu_rows"], dev["seg_pos"], dev["row_seg"], dev["positions"],
                    dev["slot_map"], dev["status"], own_from=dev["own_from"])
    for k, v in keep.items():
        dev[k].copy_(v)
    for _ in range(40):
        _, cu, pos, rows = plain.step([1] * 4, 6)
        g.replay()
        assert dev["slot_map"].tolist() == [r[2] for r in rows] + [-1] * 2 and dev["positions"].tolist() == [r[1] for r in rows] + [-1] * 2
    assert dev["length"].tolist() == plain.length and dev["n_free"].tolist() == [len(plain.free)]


def test_refusals():
    dev = Plain([16, 3], 16, 5, 20).device(30)
    delta = torch.ones(2, dtype=torch.int32, device="cuda")
    order = ("block_table", "length", "delta", "free_pages", "n_free", "page_size", "cu_rows", "seg_pos", "row_seg", "positions", "slot_map", "status", "own_from")

    def call(**kw):
        a = {**dev, "delta": delta, "page_size": 16, **kw}
        page_tables(*[a[k] for k in order[:-1]], own_from=a["own_from"])

    call()
    for kw in ({"delta": delta.long()}, {"delta": delta[:1]}, {"page_size": 0}, {"cu_rows": dev["cu_rows"][:2]}, {"seg_pos": dev["seg_pos"][:1]},
               {"positions": dev["positions"][:3]}, {"row_seg": dev["row_seg"][::2]}, {"status": dev["slot_map"]}, {"n_free": dev["slot_map"]},
               {"own_from": delta[:1]}, {"block_table": dev["block_table"][:1]}, {"block_table": dev["block_table"].t()}, {"length": dev["length"].cpu()},
               {"page_size": 2 ** 28}, {"slot_map": torch.empty(65536, dtype=torch.int32, device="cuda"), "row_seg": torch.empty(65536, dtype=torch.int32, device="cuda"),
                                        "positions": torch.empty(65536, dtype=torch.int32, device="cuda")}):
        with pytest.raises(KernelError):
            call(**kw)
