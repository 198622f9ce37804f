"""The 4-bit cache's kernels at the edges of what they promise, against the definition in 64 bits.

The plain implementation and its tolerances are those of test_kv4_gpu.py; where a test has one of its own it says how that was derived.
"""
import numpy as np
import pytest
import torch

from kappai_b200 import Kv4Cache
from kappai_b200.ops import kv4
from kappai_b200.ops.kernels import KernelError, read_status
from test_kv4_gpu import DEV, Paged, plain_attention, plain_values

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def attend(P, q, rows, H, scale=None, window=None, mass=None, table=None, pos=None, min_rows=None, out=None):
    """kv4_attention of the last `rows[i]` keys' rows of every sequence."""
    cu = np.concatenate([[0], np.cumsum(rows)])
    pos = [n - r for n, r in zip(P.lengths, rows)] if pos is None else pos
    out = torch.full_like(q, float("nan")) if out is None else out
    return kv4.kv4_attention(q, P.pages, P.table_d if table is None else table, i32(cu.tolist()), i32(pos), out, P.hd ** -0.5 if scale is None else scale, window,
                             P.page, H, P.G, P.hd, max(rows), max(1, max(p + r for p, r in zip(pos, rows))), min_rows=min(rows) if min_rows is None else min_rows,
                             mass=mass)


def queries(n, width, dtype, seed=1):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((n, width)).astype(np.float32)).to(dtype)


def near(have, want, most, dtype):
    """test_kv4_gpu.py's bounds: 1e-4 for float32 rows, the output's rounding and two of fp16 for bfloat16 ones."""
    if dtype == torch.float32:
        np.testing.assert_allclose(have, want, rtol=0, atol=1e-4)
    else:
        assert (np.abs(have - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * most).all(), np.abs(have - want).max()


# dtype, head size and rows behind 700 keys that take each form: split, its chunks joined, tiled, tcgen05
FORMS = [(torch.bfloat16, 64, 1), (torch.bfloat16, 128, 3), (torch.float32, 96, 2), (torch.float32, 64, 60), (torch.bfloat16, 96, 60), (torch.bfloat16, 64, 60),
         (torch.bfloat16, 128, 60), (torch.bfloat16, 128, 300)]


@pytest.mark.parametrize("dtype,hd,rows,lengths", [(torch.bfloat16, 64, [1, 1], [9000, 300]), (torch.float32, 64, [60], [700]), (torch.bfloat16, 64, [60], [700]),
                                                   (torch.bfloat16, 128, [1, 60], [9000, 700])])
def test_scratch_is_held_until_the_launch_has_returned(dtype, hd, rows, lengths, monkeypatch):
    """What the allocator gives somebody else while a launcher runs is not what the launcher was handed.  (Nothing is launched here.)"""
    H, G = 4, 2
    P = Paged(lengths, G, hd, 16, 3, dtype)
    q, mass = queries(sum(rows), H * hd, dtype).to(DEV), P.mass()
    handed, calls, empty = {}, [], torch.empty

    def noted(*a, **kw):
        t = empty(*a, **kw)
        handed[t.data_ptr()] = t.numel() * t.element_size()
        return t

    def launcher(what, fn, *args, **kw):
        assert set(handed) & {a for a in args if isinstance(a, int)}
        theirs = [empty(n, dtype=torch.uint8, device=DEV) for n in handed.values() for _ in range(2)]
        calls.append(what)
        assert not any(t.data_ptr() in handed for t in theirs), f"{what} was handed memory that is free"

    out = torch.empty_like(q)
    monkeypatch.setattr(kv4, "_run", launcher)
    monkeypatch.setattr(torch, "empty", noted)
    attend(P, q, rows, H, mass=mass, out=out)
    assert calls and handed


def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    """The launch goes to the current device's stream.  (A stand-in says that device 1 is current; nothing is launched.)"""
    P = Paged([40], 2, 64, 16, 0)
    new, kept, mass = Paged([8], 2, 64, 16, 1), torch.empty((1, 2, 8), dtype=torch.int32, device=DEV), P.mass()
    q, k, s = torch.zeros((1, 256), device=DEV), torch.zeros((2, 128), device=DEV), i32([0, 1])
    calls = [lambda: kv4.kv4_write(k, k, P.pages, s, 16, 2, 64), lambda: kv4.kv4_read(P.pages, s, 16, 2, 64), lambda: attend(P, q, [1], 4),
             lambda: kv4.kv4_evict(P.pages, mass, P.table_d, i32([40]), new.pages, new.mass(), new.table_d, kept, 40, 8, 2, 1, 16, 2, 64)]
    for call in calls:
        call()
    launched = []
    monkeypatch.setattr(kv4, "_device", lambda: 1, raising=False)
    monkeypatch.setattr(kv4, "_run", lambda *a, **kw: launched.append(a))
    for call in calls:
        with pytest.raises(KernelError, match="current device"):
            call()
    assert not launched


def test_a_cache_works_on_its_own_device(monkeypatch):
    """Every operator of a cache runs with the cache's device as the current one, whichever was before."""
    c = Kv4Cache(2, 64, 16, page_size=16, mass=True, device=DEV)
    assert c.device.index == torch.cuda.current_device()
    entered = []
    real = torch.cuda.device

    class Noted(real):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    monkeypatch.setattr(torch.cuda, "device", Noted)
    x = torch.randn((40, 128), device=DEV)
    c.add("a")
    for call in (lambda: c.append(x, x, ["a"], [40]), lambda: c.attend(torch.randn((2, 256), device=DEV), ["a"], [2], 4, 0.125), lambda: c.evict(["a"], 20),
                 lambda: c.read("a"), lambda: c.mass_of("a")):
        before = len(entered)
        call()
        assert entered[before:] and set(entered) == {c.device.index}


@pytest.mark.parametrize("dtype,hd,rows", FORMS)
@pytest.mark.parametrize("n", [700, 3000])
def test_weights_of_keys_that_sequences_share(dtype, hd, rows, n):
    """Several samples of one prompt: block tables that name the same pages.  Every sequence's weights reach the keys' mass.  (Each of the sequences' sums is off by
    1e-5 of itself, their addition by less: the bounds of test_kv4_gpu.py hold for the whole.)"""
    H, G, S = 4, 2, 8 if rows < 100 else 3
    P = Paged([n], G, hd, 16, 3, dtype)
    q, mass = queries(S * rows, H * hd, dtype), P.mass(5)
    m0 = mass.clone()
    table = P.table_d.expand(S, -1).contiguous()
    attend(P, q.to(DEV), [rows] * S, H, mass=mass, table=table, pos=[n - rows] * S)
    want = sum(plain_attention(x.double().numpy().reshape(rows, H, hd), P.k[0], P.v[0], n - rows, hd ** -0.5, None, H)[1] for x in q.split(rows))
    np.testing.assert_allclose(P.mass_of(mass, 0), P.mass_of(m0, 0) + want, rtol=1e-5, atol=1e-6)
    assert not any(read_status().values())


@pytest.mark.parametrize("dtype,hd,rows", FORMS)
@pytest.mark.parametrize("value", [0.0, 1e6, 1e10, -1e30, 3e38])
@pytest.mark.parametrize("n", [1, 20000])
def test_values_that_are_all_the_same(dtype, hd, rows, value, n):
    """Groups without a range: scale 0, all of the value in the minimum.  The output is that value: float32 sums of up to 20,000 weights, at most 2,500 of them added
    one after another (a thread's share of a tile's keys), are off by 2500 x 2^-24 of themselves, the sum of weights above and below the line: 3e-4."""
    rows = min(rows, n)
    H, G = 4, 2
    P = Paged([n], G, hd, 16, 3, dtype)
    k = torch.randn((n, G * hd), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    v = torch.full((n, G * hd), value, dtype=dtype, device=DEV)
    kv4.kv4_write(k, v, P.pages, P.slots(0, n), 16, G, hd)
    out = attend(P, queries(rows, H * hd, dtype).to(DEV), [rows], H).double().cpu().numpy()
    want = float(torch.tensor(value).bfloat16())
    np.testing.assert_allclose(out, want, rtol=3e-4 if dtype == torch.float32 else 2.0 ** -8 + 3e-4, atol=0)


@pytest.mark.parametrize("dtype,hd,rows", FORMS)
@pytest.mark.parametrize("scale", [1.0, 1e10, 1e-12])
def test_values_without_a_range_before_others(dtype, hd, rows, scale):
    """The first half of the keys have values without a range, the others have one.  (Bounds as for values of many sizes in test_kv4_gpu.py.)"""
    H, G, n = 4, 2, 1400
    P = Paged([n], G, hd, 16, 3, dtype, scale=scale)
    v = torch.from_numpy((P.v[0] * 1.0).astype(np.float32)).to(dtype)
    v[:n // 2] = (torch.arange(n // 2)[:, None, None] % 7 - 3.0) * scale
    kv4.kv4_write(torch.from_numpy(P.k[0].astype(np.float32)).reshape(n, -1).to(dtype).to(DEV), v.reshape(n, -1).to(DEV), P.pages, P.slots(0, n), 16, G, hd)
    kq, vq = (x.double().cpu().numpy().reshape(n, G, hd) for x in kv4.kv4_read(P.pages, P.slots(0, n), 16, G, hd, torch.float32))
    q = queries(rows, H * hd, dtype)
    s = hd ** -0.5 / scale
    out = attend(P, q.to(DEV), [rows], H, scale=s).double().cpu().numpy().reshape(rows, H, hd)
    want, _ = plain_attention(q.double().numpy().reshape(rows, H, hd), kq, vq, n - rows, s, None, H)
    top = np.abs(vq).max()
    assert (np.abs(out - want) <= (1e-3 if dtype == torch.float32 else 2.0 ** -7) * top).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 96])
def test_groups_whose_range_is_above_float32s(dtype, hd):
    """Finite values whose difference is not finite in float32.  A power of two changes neither codes nor the rounding of scale and minimum, so what is
    to be read are the values of the rows divided by 16, times 16."""
    n, G, page = 12, 2, 16
    rng = np.random.default_rng(2)
    x = rng.uniform(-3.2e38, 3.2e38, (n, G * hd)).astype(np.float32)
    x[0] = np.where(np.arange(G * hd) % 2, 3.2e38, -3.2e38)
    x[1] = np.linspace(-3e38, 3e38, G * hd)
    x[2, :hd] = rng.standard_normal(hd)                                       # (a head of ordinary values beside one that is not)
    x[3] = np.where(np.arange(G * hd) % 5, 1e-30, np.where(np.arange(G * hd) % 2, 2e38, -2e38))
    x = torch.from_numpy(x).to(dtype)
    pages = torch.zeros((1, G, kv4.kv4_page_bytes(page, hd)), dtype=torch.uint8, device=DEV)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    kv4.kv4_write(x.to(DEV), x.to(DEV), pages, slots, page, G, hd)
    want = (plain_values((x.float().numpy() / np.float32(16.0)).reshape(n, G, hd), hd) * 16.0).reshape(n, G * hd)
    assert np.isfinite(want).all() and np.abs(want).max() < 3.4e38
    for have in kv4.kv4_read(pages, slots, page, G, hd, torch.float32):
        have = have.cpu().numpy()
        # (the division by 16 leaves of 1e-30 what it was; the read rounds s c + z once, to float32)
        assert np.array_equal(have, want.astype(np.float32))


@pytest.mark.parametrize("dtype,hd,rows", FORMS + [(torch.bfloat16, 256, 1), (torch.float32, 256, 30), (torch.bfloat16, 32, 30)])
@pytest.mark.parametrize("factor", [2.0 ** 30, 2.0 ** 45, 2.0 ** -45])
def test_a_query_does_not_change_its_neighbours(dtype, hd, rows, factor):
    """Queries of one head, and of one row, that are much larger or smaller than the others beside which they are computed."""
    H, G, n = 4, 2, 700
    P = Paged([n], G, hd, 16, 3, dtype)
    q = queries(rows, H * hd, dtype).view(rows, H, hd)
    other = torch.zeros((rows, H), dtype=torch.bool)
    other[:, 1] = other[rows // 2] = True
    other[:, 3] = False
    x = torch.where(other[..., None], q * factor, q).to(dtype)
    out = attend(P, x.reshape(rows, -1).to(DEV), [rows], H).double().cpu().numpy().reshape(rows, H, hd)
    want, _ = plain_attention(x.double().numpy(), P.k[0], P.v[0], n - rows, hd ** -0.5, None, H)
    ordinary = ~other.numpy() if factor > 1 else np.ones((rows, H), dtype=bool)      # (scores of 1e10 themselves are off by thousands)
    near(out[ordinary], want[ordinary], np.abs(P.v[0]).max(), dtype)


@pytest.mark.parametrize("dtype,hd,rows", FORMS)
@pytest.mark.parametrize("window", [701, 2 ** 29, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 40])
def test_a_window_that_no_row_exceeds_is_none(dtype, hd, rows, window):
    H, G, n = 4, 2, 700
    P = Paged([n], G, hd, 16, 3, dtype)
    q = queries(rows, H * hd, dtype).to(DEV)
    m0, m1 = P.mass(), P.mass()
    a = attend(P, q, [rows], H, mass=m0)
    b = attend(P, q, [rows], H, mass=m1, window=window)
    assert torch.equal(a, b) and torch.equal(m0, m1) and abs(float(m1.sum()) - rows * H) < 1e-3 * rows * H


def test_block_tables_of_more_keys_than_indices_hold():
    """Keys are counted in 32 bits, with room for what is added to them."""
    page, hd = 32768, 32
    pages = torch.zeros((2, 1, kv4.kv4_page_bytes(page, hd)), dtype=torch.uint8, device=DEV)
    wide, mass = torch.zeros((1, 32769), dtype=torch.int32, device=DEV), torch.zeros((2, 1, page), device=DEV)
    q = torch.zeros((1, hd), device=DEV)
    with pytest.raises(KernelError, match="keys"):
        kv4.kv4_attention(q, pages, wide, i32([0, 1]), i32([5]), torch.empty_like(q), 0.1, None, page, 1, 1, hd, 1, 6)
    with pytest.raises(KernelError, match="keys"):
        kv4.kv4_evict(pages, mass, wide, i32([40]), pages, mass, i32([[1]]), torch.empty((1, 1, 8), dtype=torch.int32, device=DEV), 40, 8, 2, 1, page, 1, hd)
    kv4.kv4_attention(q, pages, wide[:, :32768].contiguous(), i32([0, 1]), i32([5]), torch.empty_like(q), 0.1, None, page, 1, 1, hd, 1, 6)


def test_numbers_of_rows_and_heads_that_make_no_sense_are_refused():
    """None of these is launched: without rows or heads nothing would be written, or a division by zero raised."""
    P = Paged([40], 2, 64, 16, 0)
    q = torch.zeros((1, 256), device=DEV)
    ok = dict(q=q, pages=P.pages, block_table=P.table_d, cu_rows=i32([0, 1]), seg_pos=i32([39]), out=torch.zeros_like(q), scale=0.1, window=None, page_size=16, H=4,
              G=2, hd=64, max_rows=1, max_context=40)
    for bad in (dict(max_rows=0), dict(max_rows=-3), dict(min_rows=2), dict(H=0, q=q[:, :0], out=q[:, :0]), dict(H=-2)):
        with pytest.raises(KernelError):
            kv4.kv4_attention(**{**ok, **bad})


def test_a_prompt_beside_decoded_rows_asks_for_no_more_scratch_than_it_needs(monkeypatch):
    """31 sequences decode behind up to 131,072 keys while another's prompt runs: scores for a row a sequence are half a gigabyte, for the eight rows that
    the split form could take of each they would be four.  (Nothing is launched.)"""
    H, G, hd, page, n = 32, 8, 64, 128, 131072
    pages = torch.zeros((2, G, kv4.kv4_page_bytes(page, hd)), dtype=torch.uint8, device=DEV)
    mass = torch.zeros((2, G, page), device=DEV)
    table = torch.zeros((32, n // page), dtype=torch.int32, device=DEV)
    rows = [1] * 31 + [200]
    q = torch.zeros((sum(rows), H * hd), dtype=torch.bfloat16, device=DEV)
    calls = []
    monkeypatch.setattr(kv4, "_run", lambda what, *a, **kw: calls.append(what))
    out = torch.empty_like(q)
    cu, pos = i32(np.concatenate([[0], np.cumsum(rows)]).tolist()), i32([n - r for r in rows])
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    kv4.kv4_attention(q, pages, table, cu, pos, out, 0.125, None, page, H, G, hd, max(rows), n, min_rows=1, mass=mass)
    assert calls == ["kv4_attention", "kv4_attention_tc"]
    assert torch.cuda.max_memory_allocated() - before <= 1.2 * 2 ** 30


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 96), (torch.float32, 64)])
@pytest.mark.parametrize("with_mass", [False, True])
@pytest.mark.parametrize("limit", [0, 300000, 2 ** 30])
def test_a_mixed_call_with_little_scratch(dtype, hd, with_mass, limit, monkeypatch):
    """The fewer rows the split form may take, the more go to the others: the results are the same."""
    monkeypatch.setattr(kv4, "KV4_SCRATCH", limit, raising=False)
    H, G, lengths, rows = 8, 2, [900, 400, 33, 150, 8, 300], [1, 2, 3, 150, 8, 5]
    P = Paged(lengths, G, hd, 16, 3, dtype)
    q, mass = queries(sum(rows), H * hd, dtype), P.mass(5) if with_mass else None
    m0 = mass.clone() if with_mass else None
    out = attend(P, q.to(DEV), rows, H, mass=mass).double().cpu().numpy()
    at = 0
    for i, r in enumerate(rows):
        want, got = plain_attention(q[at:at + r].double().numpy().reshape(r, H, hd), P.k[i], P.v[i], lengths[i] - r, hd ** -0.5, None, H)
        near(out[at:at + r].reshape(r, H, hd), want, np.abs(P.v[i]).max(), dtype)
        if with_mass:
            np.testing.assert_allclose(P.mass_of(mass, i), P.mass_of(m0, i) + got, rtol=1e-5, atol=1e-6)
        at += r
    assert not any(read_status().values())


@pytest.mark.parametrize("dtype,hd,rows", FORMS + [(torch.bfloat16, 256, 30), (torch.bfloat16, 64, 9), (torch.float32, 128, 8)])
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_finite_reach_the_rows_that_read_them_only(dtype, hd, rows, window, bad):
    """A value that a row's mask hides from it, a later token's or one behind the window, has no part in the row, whatever it is."""
    H, G, n = 4, 2, 700
    P = Paged([n], G, hd, 16, 3, dtype)
    x = torch.from_numpy(P.v[0].astype(np.float32)).to(dtype)
    first = n - rows
    x[first + rows // 2, 1, 5] = bad                                          # a row in the middle, one value of kv head 1
    x[n - 1, 0, hd - 1] = bad                                                 # the last
    x[max(0, first - 20), 0, 0] = bad                                         # a key that the window hides from the later rows
    k = torch.from_numpy(P.k[0].astype(np.float32)).to(dtype)
    kv4.kv4_write(k.reshape(n, -1).to(DEV), x.reshape(n, -1).to(DEV), P.pages, P.slots(0, n), 16, G, hd)
    kq, vq = (t.double().cpu().numpy().reshape(n, G, hd) for t in kv4.kv4_read(P.pages, P.slots(0, n), 16, G, hd, torch.float32))
    q = queries(rows, H * hd, dtype)
    out = attend(P, q.to(DEV), [rows], H, window=window).double().cpu().numpy().reshape(rows, H, hd)
    with np.errstate(invalid="ignore"):
        want, _ = plain_attention(q.double().numpy().reshape(rows, H, hd), kq, vq, first, hd ** -0.5, window, H)
    assert np.array_equal(np.isfinite(out), np.isfinite(want))
    fine = np.isfinite(want)
    near(out[fine], want[fine], np.abs(vq[np.isfinite(vq)]).max(), dtype)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("with_mass", [False, True])
def test_lengths_that_differ_much(dtype, hd, with_mass):
    """One long sequence among many short ones, and one without a key: chunks that most sequences have nothing in."""
    H, G = 8, 2
    lengths = [30, 1, 12000, 0, 257] + list(range(2, 60))
    rows = [1] * len(lengths)
    P = Paged(lengths, G, hd, 16, 3, dtype)
    q, mass = queries(len(rows), H * hd, dtype), P.mass(5) if with_mass else None
    m0 = mass.clone() if with_mass else None
    out = attend(P, q.to(DEV), rows, H, mass=mass).double().cpu().numpy()
    for i, n in enumerate(lengths):
        want, got = plain_attention(q[i:i + 1].double().numpy().reshape(1, H, hd), P.k[i], P.v[i], n - 1, hd ** -0.5, None, H)
        near(out[i:i + 1].reshape(1, H, hd), want, np.abs(P.v[i]).max() if n else 0.0, dtype)
        if with_mass:
            np.testing.assert_allclose(P.mass_of(mass, i), P.mass_of(m0, i) + got, rtol=1e-5, atol=1e-6)
    assert not any(read_status().values())


@pytest.mark.parametrize("dtype,hd,rows", FORMS + [(torch.bfloat16, 64, 2), (torch.float32, 64, 2), (torch.bfloat16, 64, 9)])
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("n", [100, 1500, 9000])
def test_weights_that_are_no_numbers_reach_the_keys_that_are_read_only(dtype, hd, rows, window, n):
    """A row with a NaN in its query has weights that are NaN: its keys' masses are, those of keys that it does not read are not."""
    H, G = 4, 2
    rows = min(rows, n)
    P = Paged([n], G, hd, 16, 3, dtype)
    q, mass = queries(rows, H * hd, dtype), P.mass(5)
    m0 = mass.clone()
    x = q.clone()
    x[rows // 3, hd + 3] = float("nan")                                       # head 1, of kv head 0
    attend(P, x.to(DEV), [rows], H, window=window, mass=mass)
    hi = n - rows + rows // 3
    read = np.arange(n) <= hi if window is None else (np.arange(n) <= hi) & (np.arange(n) > hi - window)
    have = P.mass_of(mass, 0)
    assert np.isnan(have[0, read]).all() and not np.isnan(have[0, ~read]).any() and not np.isnan(have[1]).any()
    _, want = plain_attention(q.double().numpy().reshape(rows, H, hd), P.k[0], P.v[0], n - rows, hd ** -0.5, window, H)
    ok = ~np.isnan(have)
    np.testing.assert_allclose(have[ok], (P.mass_of(m0, 0) + want)[ok], rtol=1e-5, atol=1e-6)
