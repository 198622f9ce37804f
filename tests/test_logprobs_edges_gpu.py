"""Log probabilities of rows at the edges: rows of which nothing is a number."""
import pytest
import torch

from kappai_b200.ops.logprobs import logprob_parts, token_logprobs
from test_logprobs_gpu import DT, rows

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
