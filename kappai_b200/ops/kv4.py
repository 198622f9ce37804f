"""Python faces of the kernels over a cache held in 4 bits (``csrc/kv4.cuh`` has its bytes and its arithmetic).

Pages are one uint8 tensor ``[n_pages, G, page_bytes]``: of every kv head one record with the codes of ``page_size`` keys,
those of their values, the keys' ranges and the values' ranges.  Key ``j`` of a sequence lies in page ``block_table[j //
page_size]`` at place ``j % page_size``, as in the 16-bit cache.  Each function checks its tensors (the current device's, dtype, layout),
launches on the current CUDA stream and raises :class:`~kappai_b200.ops.kernels.KernelError` on any error.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .build import load_library
from .kernels import STREAM, KernelError, _need, _raw_device, _rows_2d, _run, dtype_code

KV4_HEAD_DIMS = (32, 64, 96, 128, 192, 256)
# Segments of few columns (rows times the query heads of a kv head) take the split form, where eight columns share a block of keys.  Measured against
# the tcgen05 form, 32 heads over 8 of 64 values, 64 columns: 8 x 4000 keys 51 us against 67, 1 x 32000 52 against 122; 96 columns: 73 against
# 67, 88 against 122.  With mass, whose scores it keeps in memory: 32 columns, 8 x 4000 keys 66 against 106, 1 x 500 29 against 20; 64 columns
# 136 against 106.
KV4_SHORT_COLS, KV4_SHORT_COLS_MASS, KV4_SHORT_ROWS_MASS = 64, 32, 16
KV4_MAX_KEYS = 1 << 30     # that a block table has room for: the kernels count keys, and add windows and tiles to them, in 32 bits
# Bytes of scratch up to which the split form takes all the rows that it could.  It is indexed by the most rows that a segment may have, so that beside a
# prompt 31 decoded rows behind 131,072 keys with mass would ask for 4.3 GB; above the limit segments of several rows go to the other forms.
KV4_SCRATCH = 1 << 30
USE_TC_KV4 = True          # longer ones of bfloat16 rows with heads of 64 or 128 run on the tcgen05 tensor cores
_CTAS = 148 * 4            # CTAs of the split form that an even spread over the SMs wants

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
# Argument types of the launchers: a step makes a call a layer, and plain integers that ctypes converts itself cost a third of
# what an object an argument does.
_LAUNCHERS = {
    "kp_kv4_write": ("kv4", [_P, _L, _P, _L, _P, _L, _P] + [_I] * 5 + [_P]),
    "kp_kv4_read": ("kv4", [_P, _L, _P, _P, _P] + [_I] * 5 + [_P]),
    "kp_kv4_attention": ("kv4", [_P, _L, _P, _L, _P, _I, _P, _P, _I, _P, _L, _F] + [_I] * 12 + [_P, _P, _P, _I, _P, _P, _P, _I, _P]),
    "kp_kv4_attention_tc": ("kv4_tc", [_P, _L, _P, _P, _I, _P, _P, _I, _P, _L, _F] + [_I] * 9 + [_P, _P, _P]),
    "kp_kv4_evict": ("kv4_evict", [_P, _P, _P, _I, _P, _P, _P, _P, _I, _P] + [_I] * 8 + [_P]),
}
_fns = {}


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        lib, types = _LAUNCHERS[name]
        fn = getattr(load_library(lib), name)
        fn.argtypes = types
        _fns[name] = fn
    return fn


def kv4_group(hd: int) -> int:
    """Values of a head that share a scale and a minimum."""
    return 64 if hd % 64 == 0 else 32


@lru_cache(maxsize=None)
def kv4_page_bytes(page_size: int, hd: int) -> int:
    """Bytes of a page of one kv head: ``page_size`` keys and values of 4 bits, and 4 bytes a group of either."""
    if hd not in KV4_HEAD_DIMS or page_size < 16 or page_size & (page_size - 1):
        raise KernelError(f"a 4-bit cache has heads of {KV4_HEAD_DIMS} values and pages of a power of two of keys, at least 16, "
                          f"got head size {hd}, page size {page_size}")
    return page_size * (hd + 8 * (hd // kv4_group(hd)))


_device = _raw_device or torch.cuda.current_device      # number of the current device


def _here(t: torch.Tensor) -> int:
    """The current device's number, asked for once a call; a number that no tensor has where ``t`` is on no device."""
    return _device() if isinstance(t, torch.Tensor) and t.is_cuda else -2


def _unlike(t: torch.Tensor, name: str, dtype: torch.dtype, contiguous: bool = True) -> None:
    _need(t, name, dtype, contiguous)
    raise KernelError(f"{name}: is on {t.device}; all tensors of a call are on the current device, to whose stream its launches go")


def _have(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int) -> int:
    """The address of a contiguous tensor of that type on device ``dev``, the current one."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        _unlike(t, name, dtype)
    return t.data_ptr()


def _have_rows(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, width: int, dev: int) -> Tuple[int, int]:
    """Address and row stride of a tensor [n, width] with contiguous rows on device ``dev``, the current one."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != dev:
        _unlike(t, name, dtype, contiguous=False)
    if t.shape != (n, width):
        raise KernelError(f"{name}: expected [{n}, {width}], got {tuple(t.shape)}")
    return t.data_ptr(), _rows_2d(t, name)


def _have_pages(t: torch.Tensor, name: str, page_size: int, G: int, hd: int, dev: int) -> int:
    at = _have(t, name, torch.uint8, dev)
    shape = t.shape
    if len(shape) != 3 or shape[1] != G or shape[2] != kv4_page_bytes(page_size, hd):
        raise KernelError(f"{name}: expected [n_pages, {G}, {kv4_page_bytes(page_size, hd)}], got {tuple(t.shape)}")
    return at


def _have_mass(t: torch.Tensor, name: str, pages: torch.Tensor, page_size: int, G: int, dev: int) -> int:
    at = _have(t, name, torch.float32, dev)
    if t.shape != (pages.shape[0], G, page_size):
        raise KernelError(f"{name}: expected [{pages.shape[0]}, {G}, {page_size}], got {tuple(t.shape)}")
    return at


def kv4_write(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, slot_map: torch.Tensor, page_size: int, G: int, hd: int) -> None:
    """Rows of keys and values [n, G hd] (float32 or bfloat16; columns of wider rows will do) to the slots ``slot_map`` names
    (int32: page * page_size + place; -1: nowhere).  A group is cut into 16 equal steps from its smallest value on, ``s =
    bfloat16((max - min) / 15)``, ``z = bfloat16(min)``, ``c = round((x - z) / s)`` (halves to even, within 0..15; 0 where s is
    0).  A group with a value that is not finite reads as NaN.  No slot is named twice (which row it then holds, or parts of which, is not fixed)."""
    dev = _here(pages)
    slots = _have(slot_map, "slot_map", torch.int32, dev)
    at, n, code = _have_pages(pages, "pages", page_size, G, hd, dev), slot_map.numel(), dtype_code(k.dtype)
    pk, ldk = _have_rows(k, "k", k.dtype, n, G * hd, dev)
    pv, ldv = _have_rows(v, "v", k.dtype, n, G * hd, dev)
    _run("kv4_write", _fn("kp_kv4_write"), pk, ldk, pv, ldv, at, pages.shape[0], slots, n, page_size, G, hd, code, STREAM)


def kv4_read(pages: torch.Tensor, slot_map: torch.Tensor, page_size: int, G: int, hd: int,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values in the slots, as rows [n, G hd] of ``dtype`` (a slot of -1 reads as zeros)."""
    dev = _here(pages)
    slots = _have(slot_map, "slot_map", torch.int32, dev)
    at, n, code = _have_pages(pages, "pages", page_size, G, hd, dev), slot_map.numel(), dtype_code(dtype)
    k, v = torch.empty((2, n, G * hd), dtype=dtype, device=pages.device).unbind(0)
    _run("kv4_read", _fn("kp_kv4_read"), at, pages.shape[0], slots, k.data_ptr(), v.data_ptr(), n, page_size, G, hd, code, STREAM)
    return k, v


@lru_cache(maxsize=4096)
def kv4_chunks(n_seg: int, max_rows: int, max_context: int, window: int, H: int, G: int, hd: int, usual_rows: Optional[int] = None) -> Tuple[int, int]:
    """(number of chunks, keys a chunk) of the split form: as many CTAs as fill the SMs, none with less than a tile of keys.  Up to 16
    such chunks are made 8: those are one cluster, which joins them itself and spares a launch.  ``usual_rows`` (None: the most): the rows
    that most segments have (beside portions of prompts that is the fewest: decoded tokens')."""
    tile = 256 if hd <= 64 else (128 if hd <= 128 else 64)
    span = min(max_context, window + max_rows + tile - 1) if window else max_context      # from the first tile that a row reads
    want = max(1, _CTAS // max(1, n_seg * G * -(-(usual_rows or max_rows) * (H // G) // 8)))
    n = -(-span // tile)
    if min(n, want) <= 16:
        want = min(want, 8)
    chunk = -(-n // want) * tile
    return -(-span // chunk), chunk


def kv4_short_rows(R: int, mass: bool) -> int:
    """The most rows of a segment that the split form takes, with R query heads a kv head (one row it always takes)."""
    return max(1, min(KV4_SHORT_COLS_MASS // R, KV4_SHORT_ROWS_MASS) if mass else KV4_SHORT_COLS // R)


def kv4_tc_ok(q: torch.Tensor, out: torch.Tensor, hd: int, scale: float) -> bool:
    """Does the tcgen05 form take these rows (bfloat16, heads of 64 or 128, rows on 16-byte boundaries)?"""
    return (USE_TC_KV4 and q.dtype == torch.bfloat16 and hd in (64, 128) and scale > 0 and q.stride(0) % 8 == 0 and out.stride(0) % 8 == 0
            and q.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 0)


def kv4_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, cu_rows: torch.Tensor, seg_pos: torch.Tensor,
                  out: torch.Tensor, scale: float, window: Optional[int], page_size: int, H: int, G: int, hd: int, max_rows: int,
                  max_context: int, min_rows: int = 1, mass: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the rows q [n, H hd] over their sequences' 4-bit pages (this step's keys and values already in them).

    Rows ``cu_rows[i] .. cu_rows[i + 1] - 1`` belong to sequence ``i``; the first of them stands at key ``seg_pos[i]`` and reads
    the keys up to that one, of which ``window`` (None: all) the last; a row that reads none gives zeros, and what a row does not read has
    no part in it, finite or not.  ``out`` is other memory than ``q``; ``cu_rows`` ends with at most the rows of ``q``.  ``max_rows`` and
    ``min_rows`` bound the rows of a sequence, ``max_context`` the last key that any row reads, counted from 1 (host integers).  ``mass`` (float32
    [n_pages, G, page_size]): the softmax weight of every key, summed over the rows and the query heads of its kv head, is added
    to the key's entry, in a fixed order: the same call gives the same bits.  Sequences whose tables name the same pages each add their
    weights; only the order in which these sums arrive is then not fixed."""
    if G < 1 or H < 1 or H % G:
        raise KernelError(f"kv4_attention: {H} query heads over {G} kv heads")
    if max_rows < 1 or max_rows < min_rows:
        raise KernelError(f"kv4_attention: a sequence has between min_rows={min_rows} and max_rows={max_rows} rows")
    dev = _here(pages)
    n, n_seg, code = q.shape[0], seg_pos.numel(), dtype_code(q.dtype)
    pq, ldq = _have_rows(q, "q", q.dtype, n, H * hd, dev)
    po, ldo = _have_rows(out, "out", q.dtype, n, H * hd, dev)
    at = _have_pages(pages, "pages", page_size, G, hd, dev)
    table, cu, pos = _have(block_table, "block_table", torch.int32, dev), _have(cu_rows, "cu_rows", torch.int32, dev), _have(seg_pos, "seg_pos", torch.int32, dev)
    shape = block_table.shape
    if cu_rows.numel() != n_seg + 1 or len(shape) != 2 or shape[0] < n_seg:
        raise KernelError("kv4_attention: cu_rows has one entry more than seg_pos, block_table a row for each of them")
    if window is not None and window < 1:
        raise KernelError("kv4_attention: the window is a positive number of keys")
    width = shape[1]
    if max_context < 1 or max_context > width * page_size or width * page_size > KV4_MAX_KEYS:
        raise KernelError(f"kv4_attention: max_context={max_context} does not lie within the block table's {width} pages, or these have more than {KV4_MAX_KEYS} keys")
    pm = None if mass is None else _have_mass(mass, "mass", pages, page_size, G, dev)
    if not n or not n_seg:
        return out
    R = H // G
    most = kv4_short_rows(R, pm is not None)
    short = min(max_rows, most) if min_rows <= most else 0
    tiled = max_rows > most
    if window is None or window >= max_context:
        window = 0
    if short:
        n_chunks, chunk = kv4_chunks(n_seg, short, max_context, window, H, G, hd, min_rows if tiled else None)
        if short > 1 and short > min_rows:
            row_bytes = 4 * n_seg * H * n_chunks * ((hd + 2 if n_chunks > 1 else 0) + (chunk if pm else 0))
            if short * row_bytes > KV4_SCRATCH:
                short, tiled = max(min_rows, 1, KV4_SCRATCH // row_bytes), True
                n_chunks, chunk = kv4_chunks(n_seg, short, max_context, window, H, G, hd, min_rows)
    else:
        n_chunks, chunk = kv4_chunks(1, 1, 1, 0, 1, 1, hd)     # (nothing is cut)
    tc = tiled and kv4_tc_ok(q, out, hd, scale)
    if short or (tiled and not tc):
        # one allocation for what the launches hand one another: results of chunks, their (shift, sum), scores, logarithms of sums.  It has a
        # name until this function returns: another thread would be given memory that is free before the launch that uses it is queued.
        fused = n_chunks <= 8 and (pm is None or short * R <= 8)
        places, many = n_seg * short * H, n_chunks > 1 and not fused
        sizes = (places * n_chunks * hd if many else 0, places * n_chunks * 2 if many else 0,
                 places * n_chunks * chunk if pm else 0, places if pm and not fused else 0, n * H if pm and tiled and not tc else 0)
        total = sum(sizes)
        scratch = torch.empty(total, dtype=torch.float32, device=q.device) if total else None
        p0 = scratch.data_ptr() if total else 0
        p1 = p0 + 4 * sizes[0]
        p2 = p1 + 4 * sizes[1]
        p3 = p2 + 4 * sizes[2]
        _run("kv4_attention", _fn("kp_kv4_attention"), pq, ldq, at, pages.shape[0], table, width, cu, pos, n_seg, po, ldo, scale, window, page_size, H, G,
             hd, n, short, max_rows if tiled and not tc else 0, n_chunks, chunk, fused, max_context, p0, p1, p2, n_chunks * chunk, p3, p3 + 4 * sizes[3], pm, code, STREAM)
    if tc:
        images = torch.empty(_tc_scratch(n, n_seg, H, G, hd), dtype=torch.uint8, device=q.device) if pm else None
        _run("kv4_attention_tc", _fn("kp_kv4_attention_tc"), pq, ldq, at, table, width, cu, pos, n_seg, po, ldo, scale, window, page_size, H, G, hd, n,
             short + 1, max_rows, max_context, pm, images.data_ptr() if pm else None, STREAM)
    return out


def _tc_scratch(n: int, n_seg: int, H: int, G: int, hd: int) -> int:
    fn = load_library("kv4_tc").kp_kv4_tc_scratch
    fn.restype = ctypes.c_longlong
    return fn(n, n_seg, H, G, hd)


def kv4_evict(pages: torch.Tensor, mass: torch.Tensor, block_table: torch.Tensor, n_keys: torch.Tensor, new_pages: torch.Tensor,
              new_mass: torch.Tensor, new_table: torch.Tensor, kept: torch.Tensor, max_keys: int, keep: int, recent: int, first: int,
              page_size: int, G: int, hd: int) -> torch.Tensor:
    """Of every sequence's ``n_keys[i]`` keys (int32; at most ``max_keys``) each kv head keeps ``keep``: the ``first`` first, the
    ``recent`` last and of the others those with the most ``mass`` (equal: the lowest index); all, where there are not more.
    They move with their mass to places 0, 1, ... of ``new_table``'s pages, in their order.  The new pages are none of the
    sequences' old ones.  ``kept`` (int32 [n, G, keep]) gets the old indices, -1 behind the last."""
    dev = _here(pages)
    at, new_at = _have_pages(pages, "pages", page_size, G, hd, dev), _have_pages(new_pages, "new_pages", page_size, G, hd, dev)
    pm, new_pm = _have_mass(mass, "mass", pages, page_size, G, dev), _have_mass(new_mass, "new_mass", new_pages, page_size, G, dev)
    table, new_t = _have(block_table, "block_table", torch.int32, dev), _have(new_table, "new_table", torch.int32, dev)
    keys, pk, n = _have(n_keys, "n_keys", torch.int32, dev), _have(kept, "kept", torch.int32, dev), n_keys.numel()
    if keep < 1 or min(recent, first) < 0 or first + recent > keep:
        raise KernelError(f"kv4_evict: keep={keep} is positive and not less than first={first} and recent={recent} together")
    if block_table.dim() != 2 or new_table.dim() != 2 or min(block_table.shape[0], new_table.shape[0]) < n or tuple(kept.shape) != (n, G, keep):
        raise KernelError("kv4_evict: block tables with a row a sequence and kept of [sequences, kv heads, keep]")
    if max_keys < 1 or max_keys > block_table.shape[1] * page_size or min(keep, max_keys) > new_table.shape[1] * page_size:
        raise KernelError("kv4_evict: the block tables hold max_keys keys, and the ones that stay")
    if max(block_table.shape[1], new_table.shape[1]) * page_size > KV4_MAX_KEYS:
        raise KernelError(f"kv4_evict: block tables of at most {KV4_MAX_KEYS} keys")
    _run("kv4_evict", _fn("kp_kv4_evict"), at, pm, table, block_table.shape[1], keys, new_at, new_pm, new_t, new_table.shape[1], pk, n, max_keys, keep,
         recent, first, page_size, G, hd, STREAM)
    return kept
