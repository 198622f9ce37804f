"""Programs over a SharedCache whose device calls are stand-ins on the CPU that do what their documentation says: which keys a continuation reads, and what a call
leaves behind."""
import pytest
import torch

import shared_fakes
from kappai_b200.cache import CacheError, OutOfSlots
from shared_fakes import Program


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    shared_fakes.install(monkeypatch)


def near(got, want, off):
    # the stand-in's sums are of 64 bits and rounded once, to float32 (2^-24 of a value)
    assert (((got.double() - want).abs()) <= 1e-10 + 2.0 ** -24 * want.abs()).all()


def program(seed=0, **kw):
    a = dict(n_pages=200, max_seqs=16, max_len=400, page_size=8, dtype=torch.float32)
    a.update(kw)
    return Program(4, 2, 32, near, seed, **a)


def test_a_fork_into_the_gap_that_ended_continuations_left():
    """A second prompt among the first one's continuations: those behind it still read their own prompt."""
    p = program()
    a = p.fork(160, 8)
    p.step()
    p.end(a[1:5])
    b = p.fork(32, 2)
    assert a[0] < b[0] < a[5]
    p.step()
    p.step([a[0], b[1], a[5], a[7]], [1, 3, 2, 1])
    p.end(b[:1])
    p.step()
    p.end(a[:1])
    p.step()


@pytest.mark.parametrize("seed", range(6))
def test_random_programs(seed):
    p = program(seed, page_size=(8, 5, 16)[seed % 3], max_seqs=(12, 24)[seed % 2])
    p.random(seed, 60, 90, 5)


def test_a_call_takes_no_more_sequences_than_may_have_rows(monkeypatch):
    """Spare places of the cache are not in the attention's way, and its work is cut for those that are."""
    from kappai_b200.ops import shared

    took = []

    def attention_shared(q, cache, block_table, cu_rows, seg_pos, *args, **kw):
        took.append(seg_pos.numel())
        return shared_fakes.attention_shared(q, cache, block_table, cu_rows, seg_pos, *args, **kw)

    monkeypatch.setattr(shared, "attention_shared", attention_shared)
    p = program(max_seqs=257)
    a = p.fork(40, 8)
    b = p.fork(9, 20)
    p.step()
    p.step(a)
    p.step([a[2], a[5]], [2, 1])
    p.step(b[-1:])
    assert took == [1, 1, b[-1] - a[0] + 1, 8, a[5] - a[2] + 1, 1]


class Refused(Exception):
    pass


@pytest.mark.parametrize("P", [24, 29])                  # whole pages, and a page that each continuation has a copy of
@pytest.mark.parametrize("what,call", [("page_tables", 1), ("page_tables", 2), ("qk_norm_rope_kv", 1), ("attention_shared", 1), ("copy", 1)])
def test_a_call_that_fails_leaves_everything_as_it_was(what, call, P, monkeypatch):
    """Whatever of a fork's or a step's calls refuses: pages, lengths and places are those of before, and what comes next is right."""
    from kappai_b200.ops import kernels, shared, tables

    p = program()
    a, c, armed = p.fork(21, 3), p.c, [0]
    p.step()

    def refusing(run):
        def counted(*args, **kw):
            armed[0] -= 1
            if armed[0] == 0:
                raise Refused
            return run(*args, **kw)
        return counted

    def state():
        return c.pages_free, list(c._length), list(c._own), list(c._prompt), c.live(), sorted(c.free_pages[:c._free].tolist())

    kept = state()
    if what == "copy":                                   # (the keys' own writing is the first one to the pages)
        plain, copy = torch.Tensor.__setitem__, refusing(torch.Tensor.__setitem__)
        monkeypatch.setattr(torch.Tensor, "__setitem__", lambda self, *args: (copy if self is c.pages else plain)(self, *args))
        call = 2
    else:
        monkeypatch.setattr({"qk_norm_rope_kv": kernels, "attention_shared": shared, "page_tables": tables}[what], what, refusing(getattr(shared_fakes, what)))
    if P % c.page_size or call == 1:
        armed[0] = call
        with pytest.raises(Refused):
            c.fork(p.make(P), 4)
        assert state() == kept
        p.check()
    if call == 1:
        armed[0] = 1
        with pytest.raises(Refused):
            c.step(p.make(9), a, [5, 3, 1])
        assert state() == kept
        p.check()
    armed[0] = 0
    p.fork(P, 4)
    p.step()
    p.end(a)
    p.step()


@pytest.mark.parametrize("page_size", [8, 150])
def test_a_prompt_of_more_rows_than_a_call_takes(page_size):
    """... runs in portions, as do the copies of the page that it ends in."""
    p = program(page_size=page_size)
    p.c._most = 40
    p.fork(133, 5)
    p.fork(40, 2)
    p.fork(41, 3)
    p.step()
    p.step(None, [3] * 10)
    with pytest.raises(CacheError):
        p.c.step(p.make(50), None, [5] * 10)
    p.check()


def test_a_fork_into_scattered_places():
    """Places that are free suffice, in a row or not."""
    p = program(max_seqs=9)
    a, b, c = p.fork(20, 2), p.fork(16, 1), p.fork(9, 3)
    p.step()
    p.end(a)
    p.end(c[1:])
    d = p.fork(30, 4)                                    # a prompt and four, where three and two are free
    p.step()
    p.step(sorted([d[0], b[0], c[0], d[3]]), [2, 1, 3, 1])
    with pytest.raises(OutOfSlots):
        p.c.fork(p.make(3), 1)
    p.end(d[1:])
    p.fork(5, 2)
    p.step()
