"""Attention behind a shared prefix against the definition in numpy in 64 bits.

Tolerances.  float32: a score is a sum of at most 256 products of numbers of a few units, off by a few dozen float32 roundings of values up to about 100,
1e-5 absolute; a weight is then off by 1e-5 of itself and so is an output of weights that sum to 1, against values of about 4: 1e-4.  bfloat16, in which a
rounding is off by at most half a step, 2^-8 of the value: the weights p are rounded as they enter the product with V and the output o once more, so an output
is off by at most 2^-8 (sum p |v| + |o|), which the plain implementation adds up for each one, and the 1e-4 of the float32 part."""
import numpy as np
import pytest
import torch

from kappai_b200.ops import kernels as K
from kappai_b200.ops.kernels import KernelError
from kappai_b200.ops.shared import SHARED_HEAD_DIMS, attention_shared, shared_cut

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


class Batch:
    """Groups of (prefix length, [(own keys, rows) of each sequence]) in shuffled pages; what no sequence holds is NaN."""

    def __init__(self, groups, H, G, hd, ps, dtype="bf16", seed=0, copies=True, wider=0):
        rng = np.random.default_rng(seed)
        self.H, self.G, self.hd, self.ps, self.dtype = H, G, hd, ps, dtype
        self.groups = groups
        seqs = [(g, p, own, rows) for g, (p, ss) in enumerate(groups) for own, rows in ss]
        need = sum(-(-p // ps) for p, _ in groups) + sum(-(-(p + own) // ps) - p // ps for _, p, own, _ in seqs) + 3
        order = list(rng.permutation(need))
        cache = np.full((need, 2, G, ps, hd), np.nan, dtype=np.float32)
        width = max([1] + [-(-(p + own) // ps) for _, p, own, _ in seqs]) + wider
        self.table = np.zeros((len(seqs), width), dtype=np.int32)
        self.k, self.v, i = [], [], 0
        big = 1.0 + 3.0 * (rng.random((2, 1, G, hd)) < 0.1)
        make = lambda n: (rng.standard_normal((2, n, G, hd)) * big).astype(np.float32)  # noqa: E731
        if dtype == "bf16":
            raw = make
            make = lambda n: torch.from_numpy(raw(n)).bfloat16().float().numpy()  # noqa: E731
        for p, ss in groups:
            pre, whole = make(p), [order.pop() for _ in range(p // ps)]
            for j, pg in enumerate(whole):
                cache[pg] = pre[:, j * ps:(j + 1) * ps].transpose(0, 2, 1, 3)
            tail = None
            for own, rows in ss:
                mine = make(own)
                kv = np.concatenate([pre, mine], 1)
                pages = list(whole)
                for b in range(p // ps, -(-(p + own) // ps)):
                    pg = order.pop()
                    part = kv[:, b * ps:(b + 1) * ps].transpose(0, 2, 1, 3)
                    cache[pg, :, :, :part.shape[2]] = part
                    pages.append(pg)
                self.table[i, :len(pages)] = pages
                self.k.append(kv[0]), self.v.append(kv[1])
                i += 1
        self.seqs = seqs
        self.cu = np.concatenate([[0], np.cumsum([s[3] for s in seqs])]).astype(np.int32)
        self.pos = np.array([p + own - rows for _, p, own, rows in seqs], dtype=np.int32)
        n = int(self.cu[-1])
        self.q = torch.from_numpy(rng.standard_normal((n, H * hd)).astype(np.float32)).to(DT[dtype]).cuda()
        self.cache = torch.from_numpy(cache).to(DT[dtype]).cuda()
        self.scale = hd ** -0.5

    def args(self, out=None, q=None, **kw):
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        first = np.concatenate([[0], np.cumsum([len(ss) for _, ss in self.groups])])
        q = self.q if q is None else q
        a = dict(q=q, cache=self.cache, block_table=i32(self.table), cu_rows=i32(self.cu), seg_pos=i32(self.pos), group_seqs=i32(first),
                 prefix_len=i32([p for p, _ in self.groups]), out=torch.full_like(self.q, 7.0) if out is None else out, scale=self.scale, page_size=self.ps, H=self.H, G=self.G,
                 hd=self.hd, max_rows=max(s[3] for s in self.seqs), max_group_rows=max(sum(r for _, r in ss) for _, ss in self.groups),
                 max_prefix=max(p for p, _ in self.groups), max_own=max(s[2] for s in self.seqs))
        a.update(kw)
        return a

    def plain(self):
        q = self.q.double().cpu().numpy().reshape(-1, self.G, self.H // self.G, self.hd)
        out, off = np.zeros(q.shape), np.zeros(q.shape)
        with np.errstate(all="ignore"):
            for i in range(len(self.seqs)):
                for r in range(self.cu[i], self.cu[i + 1]):
                    n = self.pos[i] + r - self.cu[i] + 1
                    if n <= 0:
                        continue
                    k, v = self.k[i][:n].astype(np.float64), self.v[i][:n].astype(np.float64)
                    for g in range(self.G):
                        s = q[r, g] @ k[:, g].T * self.scale
                        e = np.exp(s - s.max(1, keepdims=True))
                        e /= e.sum(1, keepdims=True)
                        out[r, g] = e @ v[:, g]
                        off[r, g] = e @ np.abs(v[:, g]) + np.abs(out[r, g])
        return out.reshape(self.q.shape), 1e-4 + (2.0 ** -8 * off.reshape(self.q.shape) if self.dtype == "bf16" else 0.0 * off.reshape(self.q.shape))

    def check(self, got=None):
        a = self.args()
        got = attention_shared(**a) if got is None else got
        torch.cuda.synchronize()
        assert not any(K.read_status().values())
        (want, off), have = self.plain(), got.double().cpu().numpy()
        np.testing.assert_array_equal(np.isfinite(have), np.isfinite(want))
        ok = np.isfinite(want)
        assert (np.abs(have - want)[ok] <= off[ok]).all()
        return got


def spread(lo, hi, n, rows=(1,)):
    return [(lo + (hi - lo) * i // max(1, n - 1), rows[i % len(rows)]) for i in range(n)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", SHARED_HEAD_DIMS)
def test_head_sizes(hd, dtype):
    Batch([(200, spread(1, 90, 3)), (67, spread(3, 150, 4, (1, 3)))], 8, 2, hd, 16, dtype, seed=hd).check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (6, 2), (5, 1), (12, 1), (32, 8), (20, 1), (70, 1), (140, 1)])
def test_head_layouts(H, G, dtype):
    Batch([(130, spread(1, 70, 5, (1, 2)))], H, G, 64, 32, dtype, seed=H).check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("ps", [1, 7, 16, 64, 100, 128, 256])
def test_page_sizes_and_prefixes_that_end_anywhere(ps, dtype):
    Batch([(p, spread(1, 60, 3)) for p in (1, ps, ps + 1, 2 * ps - 1, 300)], 8, 4, 64, ps, dtype, seed=ps).check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("groups", [
    [(0, [(1, 1)])],                                             # one key and nothing shared
    [(0, spread(5, 700, 6))],                                    # nothing shared
    [(1, [(1, 1)])],
    [(5000, [(1, 1)])],                                          # a group of one
    [(3000, spread(1, 1, 40))],
    [(64, spread(1, 3000, 3))],                                  # own keys shared out over a cluster
    [(700, spread(40, 300, 3, (37, 1, 20)))],                    # portions behind the prefix
    [(0, [(3, 3)]), (129, spread(2, 9, 2, (2,))), (2048, [(700, 1)]), (1, spread(1, 5, 7))],
    [(333, [(20, 0), (30, 2), (10, 0)]), (100, [(4, 0)])],       # sequences without a row, a group without one
])
def test_shapes_of_batches(groups, dtype):
    Batch(groups, 8, 2, 64, 16, dtype, seed=len(groups)).check()


def test_many_columns_of_a_group():
    Batch([(1111, spread(1, 40, 90))], 16, 2, 64, 64, "bf16").check()
    Batch([(500, spread(1, 30, 70)), (900, spread(1, 30, 10))], 8, 1, 128, 64, "bf16").check()
    Batch([(500, spread(1, 30, 70)), (900, spread(1, 30, 10))], 8, 1, 64, 64, "f32").check()


@pytest.mark.parametrize("seqs,rows", [(1, 5), (5, 1), (13, 1), (31, 1), (33, 1), (50, 2), (200, 1)])
@pytest.mark.parametrize("hd,ps", [(64, 64), (64, 16), (128, 32), (128, 256)])
def test_many_tiles_of_keys_a_cta(seqs, rows, hd, ps, monkeypatch):
    """As if the GPU had few SMs: a CTA takes a long way through the keys, with all, few or a single one of its warps' columns there."""
    from kappai_b200.ops import shared

    monkeypatch.setattr(shared, "_SMS", 2)
    shared.shared_cut.cache_clear()
    try:
        Batch([(4000, spread(rows, 30, seqs, (rows,)))], 8, 2, hd, ps, "bf16", seed=seqs).check()
        Batch([(2570, spread(rows, 300, seqs, (rows,)))], 6, 2, hd, ps, "bf16", seed=seqs).check()
    finally:
        shared.shared_cut.cache_clear()


@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "bf16"), (64, "f32")])
def test_rows_without_a_key(hd, dtype):
    """Rows at positions before 0 read nothing: zeros, not NaN."""
    b = Batch([(0, [(3, 3), (5, 1)])], 8, 2, hd, 16, dtype)
    b.pos[0] = -2
    got = b.check()
    assert (got[:2] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "bf16"), (256, "bf16"), (96, "f32")])
def test_what_a_row_does_not_read_has_no_part_in_it(hd, dtype, bad):
    """Keys and values of later rows that are not finite reach the rows that read them and no others (pages hold NaN behind the last key throughout)."""
    b = Batch([(90, [(30, 4), (21, 5), (1, 1)])], 8, 2, hd, 16, dtype, seed=3)
    for i, at in ((0, 90 + 28), (1, 90 + 20)):
        for what, kv in ((1, b.v), (0, b.k)):
            if what == 0 and i == 0:
                continue
            kv[i][at, 1, 5] = bad
            b.cache[int(b.table[i, at // 16]), what, 1, at % 16, 5] = bad
    b.check()


@pytest.mark.parametrize("hd", [64, 128])
def test_values_that_are_not_finite_in_the_prefix_reach_every_row(hd):
    b = Batch([(300, spread(1, 40, 60)), (50, spread(1, 9, 3))], 8, 2, hd, 64, "bf16", seed=3)
    for i in range(60):
        b.v[i][17, 1, 5] = np.nan
    b.cache[int(b.table[0, 0]), 1, 1, 17, 5] = float("nan")
    b.check()


@pytest.mark.parametrize("dtype", list(DT))
def test_large_scores(dtype):
    b = Batch([(400, spread(1, 90, 40))], 8, 2, 64, 64, dtype, seed=5)
    b.q *= 40
    (want, off), got = b.plain(), attention_shared(**b.args()).double().cpu().numpy()
    # scores of up to a few thousand are off by 2^-22 of themselves or so, 1e-3, and weights by as much
    assert (np.abs(got - want) <= off + 4e-3 * max(np.abs(v).max() for v in b.v)).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_strided_rows(dtype):
    b = Batch([(333, spread(1, 90, 20))], 8, 2, 64, 16, dtype, seed=5)
    n, w = b.q.shape
    for lead, width in ((0, w + 8), (8, 3 * w), (3, w + 5)):
        wide, place = torch.zeros((n, lead + width), dtype=b.q.dtype, device="cuda"), torch.full((n + 2, lead + width), 3.0, dtype=b.q.dtype, device="cuda")
        wide[:, lead:lead + w] = b.q
        got = attention_shared(**b.args(q=wide[:, lead:lead + w], out=place[:n, lead:lead + w]))
        b.check(got)                                                 # (rows at other addresses may take another form, which rounds otherwise)
        assert (place[n:] == 3).all() and (place[:, :lead] == 3).all() and (place[:, lead + w:] == 3).all()


def test_rows_behind_the_last_sequence_are_left():
    b = Batch([(100, spread(1, 9, 3))], 8, 2, 64, 16)
    q = torch.cat([b.q, torch.full((4, b.q.shape[1]), float("nan"), dtype=b.q.dtype, device="cuda")])
    out = torch.full_like(q, 5.0)
    attention_shared(**b.args(q=q, out=out))
    b.check(out[:3])
    assert (out[3:] == 5).all()


def test_sequences_in_no_group():
    b = Batch([(0, spread(9, 80, 5))], 8, 2, 64, 16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    b.check(attention_shared(**b.args(group_seqs=torch.zeros(1, dtype=torch.int32, device="cuda"), prefix_len=none, max_prefix=0)))
    some = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    b.check(attention_shared(**b.args(group_seqs=some, prefix_len=torch.zeros(1, dtype=torch.int32, device="cuda"))))


def test_against_the_attention_of_single_rows():
    """The same batch through attention_split, which reads the prefix once a row."""
    b = Batch([(1500, spread(1, 100, 16))], 32, 8, 64, 64, "bf16", seed=2)
    a = b.args()
    got = attention_shared(**a)
    n, chunks = b.q.shape[0], -(-1600 // 256)
    row_seg, at = torch.arange(n, dtype=torch.int32, device="cuda"), a["seg_pos"]
    ref, scratch = torch.empty_like(b.q), torch.empty(K.attention_split_scratch(n, 32, 64, chunks), device="cuda")
    K.attention_split(b.q, torch.nan_to_num(b.cache), a["block_table"], row_seg, at, ref, scratch, chunks, b.scale, None, 64, 32, 8, 64)
    assert (np.abs((got.double() - ref.double()).cpu().numpy()) <= 2 * b.plain()[1]).all()      # (both are that near to the definition)


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_the_same_call_gives_the_same_bits_on_another_stream_and_captured(dtype, hd):
    b = Batch([(700, spread(1, 300, 40)), (300, spread(1, 30, 12))], 16, 4, hd, 64, dtype, seed=6)
    want = attention_shared(**b.args())
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for stream in (s, t):
        with torch.cuda.stream(stream):
            got = attention_shared(**b.args())
        stream.synchronize()
        assert torch.equal(want, got)
    a = b.args()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attention_shared(**a)
    for _ in range(3):
        a["out"].zero_()
        g.replay()
        assert torch.equal(want, a["out"])


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("bf16", 128), ("bf16", 96), ("f32", 64)])
def test_bounds_may_be_wider_than_what_is_there(dtype, hd):
    """A captured call has bounds for steps to come."""
    b = Batch([(700, spread(1, 300, 20)), (30, spread(1, 30, 3, (1, 2)))], 16, 4, hd, 16, dtype, seed=6, wider=400)
    for kw in ({"max_prefix": 6000}, {"max_own": 5000}, {"max_rows": 9}, {"max_group_rows": 100}, {"max_prefix": 5000, "max_own": 3000, "max_rows": 4, "max_group_rows": 64}):
        b.check(attention_shared(**b.args(**kw)))


@pytest.mark.parametrize("groups,hd", [(31, 64), (33, 64), (40, 128), (70, 128)])
def test_many_groups(groups, hd):
    Batch([((37 * i) % 200, spread(1, 9, 3 + i % 7, (1, 2))) for i in range(groups)], 8, 1, hd, 16, "bf16", seed=groups).check()


def test_two_calls_at_once():
    """Calls on two streams, of different sizes, beside one another: each has scratch of its own."""
    a, b = Batch([(3000, spread(1, 200, 40))], 16, 4, 64, 64, "bf16", seed=1), Batch([(900, spread(1, 90, 9))], 16, 4, 128, 64, "bf16", seed=2)
    want = [attention_shared(**x.args()) for x in (a, b)]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    args = [[x.args() for _ in range(8)] for x in (a, b)]
    torch.cuda.synchronize()
    for i in range(8):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(attention_shared(**args[j][i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


@pytest.mark.parametrize("dtype,ps", [("bf16", 64), ("bf16", 60), ("f32", 64)])
def test_pages_beyond_32_bit_offsets(dtype, ps):
    """The last pages of a cache of more than 2^31 values: by TMA, copy by copy, and in float32."""
    b = Batch([(200, spread(1, 70, 9))], 8, 2, 128, ps, dtype, seed=4)
    used = b.cache.shape[0]
    n_pages = (1 << 31) // (2 * 2 * ps * 128) + used + 5
    far = torch.empty((n_pages, 2, 2, ps, 128), dtype=b.cache.dtype, device="cuda")
    far[n_pages - used:] = b.cache
    b.cache, b.table = far, np.where(b.table >= 0, b.table + n_pages - used, 0).astype(np.int32)
    b.check()
    del far, b
    torch.cuda.empty_cache()


@pytest.mark.parametrize("hd", SHARED_HEAD_DIMS)
@pytest.mark.parametrize("ps", [8, 24, 64, 128])
def test_heads_and_pages(hd, ps):
    """Tiles by boxes of 32 and of 64 values, and copy by copy; few columns, more and many; own keys that end in their first tile of keys, or cross into a second."""
    Batch([(100, spread(1, 60, 5))], 8, 2, hd, ps, "bf16", seed=hd + ps).check()
    Batch([(333, spread(1, 3, 2, (1, 2))), (64, spread(30, 64, 9))], 6, 2, hd, ps, "bf16", seed=hd + ps).check()
    Batch([(190, spread(5, 140, 3, (5, 1, 3)))], 16, 2, hd, ps, "bf16", seed=hd + ps).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_joins_of_many_parts(hd):
    """Few sequences with many columns behind a long prefix: a cluster shares the join."""
    Batch([(5000, spread(4, 20, 2, (4, 3)))], 16, 2, hd, 64, "bf16", seed=hd).check()


def test_refusals():
    b = Batch([(40, spread(1, 9, 3))], 8, 2, 64, 16)
    ok = b.args()
    attention_shared(**ok)
    for kw in ({"H": 7}, {"H": 16}, {"G": 4}, {"hd": 48}, {"page_size": 8}, {"page_size": 0}, {"max_rows": 0}, {"max_group_rows": 0}, {"max_prefix": -1},
               {"max_own": -1}, {"max_prefix": 10 ** 6}, {"q": ok["q"].float()}, {"q": ok["q"].half()}, {"out": ok["out"].float()}, {"out": ok["out"][:2]},
               {"q": ok["q"].cpu()}, {"cu_rows": ok["cu_rows"][:3]}, {"cu_rows": ok["cu_rows"].long()}, {"group_seqs": ok["prefix_len"]},
               {"block_table": ok["block_table"][:2]}, {"block_table": ok["block_table"][0]}, {"cache": ok["cache"][:, :1]}, {"cache": ok["cache"][:0]},
               {"q": ok["q"].t().contiguous().t()}, {"scale": 0.0}, {"scale": -0.1}, {"scale": float("nan")}):
        with pytest.raises(KernelError):
            attention_shared(**{**ok, **kw})


@pytest.mark.parametrize("tc", [False, True])
def test_how_the_work_is_cut(tc):
    for args in ((1, 8, 1, 8, 2048, 150, 8, 4), (5, 80, 4, 40, 12000, 300, 4, 4), (1, 1, 1, 1, 0, 1, 1, 1), (1, 256, 1, 256, 100000, 10, 8, 12), (2, 9, 3, 20, 1, 0, 1, 128)):
        c = shared_cut(*args, tc)
        per = args[3] if not c.tile else ({0: 128 // args[7] * 2, 1: 128 // args[7], 2: 64 // args[7]}[c.mode] if c.tile == 128 else c.tile / args[7])      # rows a tile
        assert per * c.tiles >= args[3] and c.own_tile * c.own_tiles >= args[2] * args[7] and 1 <= c.ctas <= 8
        assert c.chunks <= 64 and c.chunks * c.chunk >= args[4] and c.chunk % (128 if c.tile == 128 else 64) == 0
