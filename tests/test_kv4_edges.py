"""The 4-bit cache's bookkeeping where a call is wrong, or nothing is there: no device is needed for any of it."""
import pytest
import torch

from kappai_b200 import Kv4Cache
from kappai_b200.cache import CacheError
from kappai_b200.ops import kv4
from kappai_b200.ops.kernels import KernelError


def held(n, n_pages=8, mass=False):
    """A cache whose sequence "a" has n keys, nothing of them written."""
    c = Kv4Cache(2, 64, n_pages, page_size=16, mass=mass, device="cpu")
    c.add("a")
    c.pool.extend("a", n)
    c._length["a"] = n
    return c


@pytest.mark.parametrize("shape", [(3, 256), (5, 256), (0, 256), (4, 4, 64), (1024,)])
def test_attend_takes_as_many_queries_as_rows(shape):
    """Fewer would be read, and their outputs written, behind the tensors' ends; more would leave rows of the output as they were."""
    with pytest.raises(CacheError, match="rows of queries"):
        held(20).attend(torch.zeros(shape), ["a"], [4], 4, 0.125)


def test_slots_are_32_bit_numbers():
    """A slot above 2^31 would turn negative, which is the name of no slot: what is written there would be lost."""
    with pytest.raises(CacheError, match="2\\^31"):
        Kv4Cache(1, 32, n_pages=2 ** 11, page_size=2 ** 20, device="meta")
    Kv4Cache(1, 32, n_pages=2 ** 11 - 1, page_size=2 ** 20, device="meta")


@pytest.mark.parametrize("k,v", [(torch.zeros(20, 128), torch.zeros(20, 128)), (torch.zeros(20, 128), torch.zeros(19, 128)), (torch.zeros(20, 64), torch.zeros(20, 64))])
def test_an_append_that_fails_takes_no_pages(k, v):
    c = held(10)
    free, table = c.pool.n_free, list(c.pool.table("a"))
    with pytest.raises(KernelError):
        c.append(k, v, ["a"], [20])
    assert c.length("a") == 10 and c.pool.n_free == free and c.pool.table("a") == table
    c.pool.check()


def test_a_page_pool_takes_pages_back():
    from kappai_b200.cache import PagePool

    pool = PagePool(6, 16)
    pool.open("a")
    pool.extend("a", 50)
    stamp, table = pool.version("a"), list(pool.table("a"))
    pool.cut("a", 4)
    assert pool.table("a") == table and pool.version("a") == stamp
    pool.cut("a", 1)
    pool.check()
    assert pool.table("a") == table[:1] and pool.n_free == 5 and pool.version("a") != stamp
    pool.extend("a", 50)
    assert pool.table("a") == table                 # (in the order in which they were handed out)
    pool.check()


def test_calls_for_no_sequence():
    c, none = held(10, mass=True), torch.zeros(0, 128)
    c.append(none, none, [], [])
    assert c.attend(torch.zeros(0, 256), [], [], 4, 0.125).shape == (0, 256) and c.evict([], 4).shape == (0, 2, 4)
    with pytest.raises(CacheError):
        c.append(torch.zeros(1, 128), torch.zeros(1, 128), [], [])
    assert c.length("a") == 10
