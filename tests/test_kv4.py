"""The 4-bit cache without a device: page arithmetic, the split form's chunks, who holds which page, refusals."""
import pytest
import torch

from kappai_b200.cache import CacheError, PagePool
from kappai_b200.ops import kv4
from kappai_b200.ops.kernels import KernelError


@pytest.mark.parametrize("page,hd,want", [(16, 32, 16 * (32 + 8)), (64, 64, 64 * (64 + 8)), (16, 96, 16 * (96 + 24)), (128, 128, 128 * (128 + 16)),
                                          (32, 192, 32 * (192 + 24)), (64, 256, 64 * (256 + 32))])
def test_page_bytes(page, hd, want):
    assert kv4.kv4_page_bytes(page, hd) == want


@pytest.mark.parametrize("page,hd", [(8, 64), (0, 64), (24, 64), (48, 64), (64, 16), (64, 48), (64, 160), (64, 0), (64, 512)])
def test_page_sizes_and_head_sizes_that_are_refused(page, hd):
    with pytest.raises(KernelError):
        kv4.kv4_page_bytes(page, hd)


@pytest.mark.parametrize("hd", kv4.KV4_HEAD_DIMS)
@pytest.mark.parametrize("n_seg,rows,context,window,H,G", [(1, 1, 1, 0, 1, 1), (1, 1, 700, 0, 32, 8), (64, 1, 2101, 0, 32, 8), (2, 1, 131072, 0, 16, 8),
                                                           (5, 8, 5003, 1024, 12, 4), (300, 2, 90000, 16, 8, 8), (1, 3, 10 ** 6, 0, 64, 1)])
def test_chunks_cover_the_keys_that_are_read(hd, n_seg, rows, context, window, H, G):
    tile = 256 if hd <= 64 else (128 if hd <= 128 else 64)
    n, chunk = kv4.kv4_chunks(n_seg, rows, context, window, H, G, hd)
    assert chunk % tile == 0 and n >= 1
    # a segment's chunks begin at the tile of its first row's first key
    for past in {0, max(0, context - rows)}:
        first = max(0, past - window + 1) if window else 0
        base = first // tile * tile if window else 0
        assert base + n * chunk >= past + min(rows, context - past)
    assert n * chunk < (context if not window else min(context, window + rows + tile)) + chunk


def test_functions_want_cuda_tensors():
    z = torch.zeros
    pages, i32 = z((2, 1, kv4.kv4_page_bytes(16, 32)), dtype=torch.uint8), z(1, dtype=torch.int32)
    with pytest.raises(KernelError, match="CUDA"):
        kv4.kv4_write(z((1, 32)), z((1, 32)), pages, i32, 16, 1, 32)
    with pytest.raises(KernelError, match="CUDA"):
        kv4.kv4_read(pages, i32, 16, 1, 32)
    with pytest.raises(KernelError, match="CUDA"):
        kv4.kv4_attention(z((1, 32)), pages, z((1, 2), dtype=torch.int32), z(2, dtype=torch.int32), i32, z((1, 32)), 1.0, None, 16, 1, 1, 32, 1, 1)
    mass = z((2, 1, 16))
    with pytest.raises(KernelError, match="CUDA"):
        kv4.kv4_evict(pages, mass, z((1, 2), dtype=torch.int32), i32, pages, mass, z((1, 2), dtype=torch.int32), z((1, 1, 4), dtype=torch.int32), 8, 4, 1, 0,
                      16, 1, 32)


def test_a_page_pool_hands_one_table_over():
    pool = PagePool(6, 16)
    pool.open("a")
    pool.extend("a", 50)                       # four pages
    pool.open("b")
    pool.extend("b", 20)                       # two pages: none is left
    stamp, table = pool.version("a"), pool.table("b")
    pool.take_over("a", "b")
    pool.check()
    assert pool.table("a") == table and pool.n_free == 4 and pool.version("a") != stamp
    with pytest.raises(CacheError):
        pool.close("b")
    pool.close("a")
    pool.check()
    assert pool.n_free == 6
