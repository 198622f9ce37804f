"""What a SharedCache refuses before anything runs: no device is needed."""
import pytest
import torch

from kappai_b200 import SharedCache
from kappai_b200.cache import CacheError, OutOfPages, OutOfSlots


def cache(**kw):
    a = dict(num_heads=4, num_kv_heads=2, head_dim=64, n_pages=8, max_seqs=6, max_len=100, page_size=16, dtype=torch.float32, device="cpu")
    a.update(kw)
    return SharedCache(**a)


def rows(n, width=(4 + 4) * 64):
    return torch.zeros(n, width)


@pytest.mark.parametrize("kw", [{"num_heads": 3}, {"num_kv_heads": 0}, {"head_dim": 48}, {"n_pages": 0}, {"max_seqs": 0}, {"max_seqs": 8193}, {"max_len": 0},
                                {"page_size": 0}, {"dtype": torch.float16}, {"n_pages": 2, "page_size": 2 ** 30, "device": "meta"}, {"max_len": 2 ** 31, "device": "meta"}])
def test_sizes(kw):
    with pytest.raises(CacheError):
        cache(**kw)


def test_calls():
    c = cache()
    for bad in (lambda: c.fork(rows(0), 1), lambda: c.fork(rows(5), 0), lambda: c.fork(rows(101), 1), lambda: c.fork(rows(5, 100), 1), lambda: c.fork(rows(5).bfloat16(), 1),
                lambda: c.fork(rows(5), 1, scale=0.0), lambda: c.fork(rows(512)[:, :8].t(), 1), lambda: c.step(rows(1)), lambda: c.step(rows(1), [1]), lambda: c.length(0),
                lambda: c.take_back([0], [1]), lambda: c.end([3]), lambda: c.fork(None, 1)):
        with pytest.raises(CacheError):
            bad()
    with pytest.raises(OutOfPages):
        c.fork(rows(100), 3)                             # 7 pages and a copy of the last for each
    with pytest.raises(OutOfSlots):
        c.fork(rows(16), 6)
    assert c.live() == [] and c.pages_free == 8
    c.end([])
    assert c.step(rows(0)).shape == (0, 256)
