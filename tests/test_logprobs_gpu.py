"""Log probabilities of given tokens, entropy, rank and alternatives against numpy in 64 bits.

Tolerances.  A log probability is (x - max) - log S.  The sum S of positive terms is off by at most one rounding a term of a thread's share of the row
(V / 256 terms, with a vector's and the joins' some 40 more, each 2^-24 of the sum) and as much again for the exponentials (two units in the last place and the rounding
of their argument: its size times 2^-24, weighed with e^-size, below 2^-24 on the whole): (V / 256 + 40) 2^-23 relative in S, so absolute in log S; the differences round
to 2^-24 of themselves each.  The entropy is log S - W / S with |W / S| at most log V: the same error once for log S and twice for the quotient times log V.
Ids and ranks are compared for equality."""
import numpy as np
import pytest
import torch

from kappai_b200.ops.kernels import KernelError
from kappai_b200.ops.logprobs import MAX_TOP_LOGPROBS, token_logprobs

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def plain(x, ids, top):
    """numpy, float64: log probability, entropy, rank, top ids, their log probabilities."""
    n, V = x.shape
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        lp = (x - m) - np.log(e.sum(1, keepdims=True))          # (m + log S would lose log S where m is large)
        lp[np.isneginf(m[:, 0])] = -np.inf
        p = np.exp(lp)
        ent = -np.where(p > 0, p * lp, 0.0).sum(1)
    order = np.stack([np.lexsort((np.arange(V), -row))[:top] for row in x]) if top else np.zeros((n, 0), dtype=np.int64)
    given = np.where((ids >= 0) & (ids < V), ids, 0)
    there = (ids >= 0) & (ids < V)
    mine = x[np.arange(n), given]
    rank = np.where(there, (x > mine[:, None]).sum(1), -1)
    return np.where(there, lp[np.arange(n), given], 0.0), ent, rank, order, np.take_along_axis(lp, order, 1), x - m


def check(logits, ids, top):
    got = token_logprobs(logits, ids, top)
    x = logits.double().cpu().numpy()
    V = x.shape[1]
    i = np.full(x.shape[0], -1) if ids is None else ids.cpu().numpy()
    lp, ent, rank, tid, tlp, d = plain(x, i, top)
    s = (V / 256 + 40) * 2.0 ** -23
    close = lambda a, b, tol: np.all((a == b) | (np.abs(a - b) <= tol))  # noqa: E731
    a = got.logprob.cpu().double().numpy()
    with np.errstate(invalid="ignore"):
        assert close(a, lp, s + 2.0 ** -22 * np.nan_to_num(np.abs(lp), posinf=0))
        assert close(got.entropy.cpu().double().numpy(), ent, s * (1 + 2 * np.log(V)) + 2.0 ** -23 * np.log(V))
        np.testing.assert_array_equal(got.rank.cpu().numpy(), rank)
        np.testing.assert_array_equal(got.top_ids.cpu().numpy(), tid)
        assert close(got.top_logprobs.cpu().double().numpy(), tlp, s + 2.0 ** -22 * np.nan_to_num(np.abs(tlp), posinf=0))
    return got


def rows(n, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, V), generator=g, device="cuda") * scale
    ids = torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32)
    return x.to(DT[dtype]), ids


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,V,top", [(1, 65536, 5), (3, 1, 1), (5, 7, 7), (4, 33, 32), (17, 1000, 0), (9, 4099, 32), (700, 515, 8), (2, 100003, 20), (64, 16384, 20),
                                     (160, 9001, 3)])
def test_sizes(n, V, top, dtype):
    check(*rows(n, V, dtype, seed=V + n), top)


@pytest.mark.parametrize("dtype", list(DT))
def test_columns_of_wider_rows_at_any_address(dtype):
    x, ids = rows(6, 5003, dtype)
    for a, b in [(1, 5000), (3, 4999), (7, 5003), (8, 5002)]:
        check(x[:, a:b], ids % (b - a), 9)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [300, 70000])
def test_equal_logits_go_by_index(dtype, V):
    x, ids = rows(5, V, dtype)
    x[0] = 1.5                                   # all equal
    x[1] = torch.round(x[1])                     # many equal
    x[2, ::2], x[2, 1::2] = 0.0, -0.0            # both zeros are equal
    x[3] = x[3].abs().neg()                      # only negative ones
    x[4, :] = -1e30
    check(x, ids, 32)


@pytest.mark.parametrize("dtype", list(DT))
def test_masked_logits(dtype):
    x, ids = rows(8, 9000, dtype)
    x[0, 5:] = float("-inf")                     # fewer tokens than alternatives
    x[1] = float("-inf")                         # no token at all
    x[2, ::2] = float("-inf")
    x[3] = torch.finfo(DT[dtype]).min            # the lowest value everywhere: all alike
    x[4, 1:] = torch.finfo(DT[dtype]).min
    x[5, :4000] = torch.finfo(DT[dtype]).min
    x[6] = float("-inf")
    x[6, 8999] = -2.0
    ids[2], ids[4], ids[6] = 2, 7, 8999
    got = check(x, ids, 20)
    assert got.logprob[1] == float("-inf") and got.entropy[1] == 0 and got.top_ids[1].tolist() == list(range(20))
    assert got.logprob[6] == 0 and got.entropy[6] == 0


@pytest.mark.parametrize("V", [200, 30000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_are_not_finite(V, bad):
    x, ids = rows(4, V, "f32")
    x[1, V // 2], x[2, V - 1] = bad, bad
    got, want = token_logprobs(x, ids, 4), token_logprobs(x[[0, 3]], ids[[0, 3]], 4)
    for r in (1, 2):
        assert torch.isnan(got.logprob[r]) and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprobs[r]).all()
        assert got.top_ids[r].tolist() == [-1] * 4
    np.testing.assert_array_equal(got.top_ids[[0, 3]].cpu(), want.top_ids.cpu())
    np.testing.assert_array_equal(got.logprob[[0, 3]].cpu(), want.logprob.cpu())


@pytest.mark.parametrize("V", [2048, 65536])
def test_logits_that_crowd_in_a_few_threads_shares(V):
    """Every 1024th piece of four is large: the candidates outnumber the room for them in the small share of each thread."""
    x, ids = rows(600, V, "f32")
    at = torch.arange(V, device="cuda")
    near = (at % 1024) < 128
    x[:] = torch.where(near, x + 50.0, x)
    x[1, :] = torch.where((at % 1024) < 4, 90.0 + at / V, torch.zeros_like(x[1]))
    check(x[:40], ids[:40], 32)
    check(x, ids, 32)


def test_tokens_that_are_none():
    x, ids = rows(5, 700, "f32")
    ids[:] = torch.tensor([-1, 700, -7, 699, 0], dtype=torch.int32)
    got = check(x, ids, 2)
    assert got.logprob[:3].tolist() == [0, 0, 0] and got.rank[:3].tolist() == [-1] * 3
    check(x, None, 2)


def test_no_rows():
    got = token_logprobs(torch.empty((0, 100), device="cuda"), None, 3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)


def test_the_same_call_gives_the_same_bits_alone_or_among_others():
    """Rows do not depend on one another as long as they are cut the same way; the same call does so bit by bit."""
    x, ids = rows(64, 30011, "f32")
    a, b = token_logprobs(x, ids, 7), token_logprobs(x, ids, 7)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_another_stream_and_a_captured_call():
    x, ids = rows(20, 20000, "f32")
    want = token_logprobs(x, ids, 5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = token_logprobs(x, ids, 5)
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = token_logprobs(x, ids, 5)
    x2, ids2 = rows(20, 20000, "f32", seed=9)
    want = token_logprobs(x2, ids2, 5)
    x.copy_(x2), ids.copy_(ids2)
    g.replay()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets():
    n, V = 20000, 110001
    x = torch.empty((n, V), dtype=torch.bfloat16, device="cuda")
    part, ids = rows(50, V, "bf16")
    for r in range(0, n, 50):
        x[r:r + 50] = part
    got, want = token_logprobs(x, ids.repeat(n // 50), 3), token_logprobs(part, ids, 3)
    check(part, ids, 3)
    # other cuts of a row, other orders of its sums: near, and the same ids
    assert torch.equal(got.top_ids, want.top_ids.repeat(n // 50, 1)) and torch.equal(got.rank, want.rank.repeat(n // 50))
    assert (got.logprob - want.logprob.repeat(n // 50)).abs().max() <= 2 * (V / 256 + 40) * 2.0 ** -23 + 2.0 ** -21 * want.logprob.abs().max()
    del x
    torch.cuda.empty_cache()


def test_two_calls_at_once():
    a, b = rows(300, 30011, "f32"), rows(5, 65536, "bf16", seed=3)
    want = [token_logprobs(*a, 9), token_logprobs(*b, 20)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for j, (s, args) in enumerate(zip(streams, ((*a, 9), (*b, 20)))):
            with torch.cuda.stream(s):
                got[j].append(token_logprobs(*args))
    torch.cuda.synchronize()
    for w, calls in zip(want, got):
        assert all(torch.equal(s, t) for c in calls for s, t in zip(w, c))


def test_refusals():
    x, ids = rows(4, 100, "f32")
    for bad in (lambda: token_logprobs(x.half(), ids), lambda: token_logprobs(x, ids.long()), lambda: token_logprobs(x, ids[:3]), lambda: token_logprobs(x, ids, 33),
                lambda: token_logprobs(x, ids, -1), lambda: token_logprobs(x[:, :8], ids, 9), lambda: token_logprobs(x.t(), None), lambda: token_logprobs(x[0], None),
                lambda: token_logprobs(x.cpu(), ids), lambda: token_logprobs(x, ids.cpu()), lambda: token_logprobs(x[:, :0], ids)):
        with pytest.raises(KernelError):
            bad()
    assert MAX_TOP_LOGPROBS == 32
