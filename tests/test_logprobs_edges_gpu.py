"""Log probabilities of rows at the edges: rows of which nothing is a number, masked rows of large logits, logits on both sides of where differences are taken.

Tolerances: those of test_logprobs_gpu.py, whose derivation holds for logits of any size: the exponentials' arguments are rounded once, to 2^-24 of themselves."""
import pytest
import torch

from kappai_b200.ops.logprobs import logprob_parts, token_logprobs
from test_logprobs_gpu import DT, check, rows

pytestmark = pytest.mark.gpu


@pytest.fixture
def filled_memory():
    """New tensors hold NaN, or the largest whole number, until they are written."""
    torch.use_deterministic_algorithms(True)
    yield
    torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,V,top,parts", [(6, 2000, 5, 1), (6, 5000, 5, 2), (7, 65536, 5, 4), (7, 65536, 32, 4), (8, 65536, 0, 8), (400, 9000, 3, 1), (130, 9000, 7, 2)])
def test_rows_without_numbers(n, V, top, parts, dtype, filled_memory):
    assert logprob_parts(n, V, top) == parts
    x, ids = rows(n, V, dtype, seed=n)
    good = x.clone()
    nan = torch.full_like(x[0], float("nan"))
    x[0] = nan
    x[1] = -nan                                          # (the sign bit set)
    x[2], x[2, 7], x[2, V - 3] = nan, 1.0, -2.0          # fewer numbers than alternatives
    x[3], x[3, ::2] = -nan, -float("inf")
    x[4, 11:] = float("nan")
    got, want = token_logprobs(x, ids, top), token_logprobs(good, ids, top)
    for r in range(5):
        assert torch.isnan(got.logprob[r]) and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprobs[r]).all()
        assert got.top_ids[r].tolist() == [-1] * top
    for a, b in zip(got, want):
        assert torch.equal(a[5:], b[5:])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", [6, 400])
@pytest.mark.parametrize("most", [30.0, 200.0, 1000.0, 9e5, -9e5])
def test_masked_rows_of_large_logits(most, n, dtype):
    """Scattered logits that are masked beside others of any size: the sums of both are of the same numbers."""
    x, ids = rows(n, 9001, dtype, seed=3, scale=1.0)
    step = max(1.0, abs(most) * torch.finfo(DT[dtype]).eps)
    x = (most - (x.float().abs() * step)).to(DT[dtype])
    mask = torch.rand(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(int(abs(most)))) < 0.02
    x[mask] = -float("inf")
    x[n // 2:][mask[n // 2:]] = torch.finfo(DT[dtype]).min
    check(x, ids, 5)
    check(x[:, 1:], ids.clamp(max=8999), 5)              # (single values before and behind the pieces)


@pytest.mark.parametrize("n", [6, 400])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_on_both_sides_of_a_million(sign, n):
    """Up to a million a thread's sums are by a fused product, beyond it by differences, and a row has threads of both kinds."""
    x, ids = rows(n, 9001, "f32", seed=4)
    x = torch.round(x * 16) / 16 + sign * 1e6
    x[1, ::3] = -float("inf")
    check(x, ids, 5)
