"""Python faces of the kernels over a cache held in 4 bits (``csrc/kv4.cuh`` has its bytes and its arithmetic).

Pages are one uint8 tensor ``[n_pages, G, page_bytes]``: of every kv head one record with the codes of ``page_size`` keys,
those of their values, the keys' ranges and the values' ranges.  Key ``j`` of a sequence lies in page ``block_table[j //
page_size]`` at place ``j % page_size``, as in the 16-bit cache.  Each function checks its tensors (device, dtype, layout),
launches on the current CUDA stream and raises :class:`~kappai_b200.ops.kernels.KernelError` on any error.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .build import load_library
from .kernels import STREAM, KernelError, _need, _ptr, _rows_2d, _run, dtype_code

KV4_HEAD_DIMS = (32, 64, 96, 128, 192, 256)
KV4_SHORT_ROWS = 8         # segments of at most this many rows share their keys out over many CTAs
USE_TC_KV4 = True          # longer ones of bfloat16 rows with heads of 64 or 128 run on the tcgen05 tensor cores
_CTAS = 148 * 4            # CTAs of the split form that an even spread over the SMs wants


def kv4_group(hd: int) -> int:
    """Values of a head that share a scale and a minimum."""
    return 64 if hd % 64 == 0 else 32


def kv4_page_bytes(page_size: int, hd: int) -> int:
    """Bytes of a page of one kv head: ``page_size`` keys and values of 4 bits, and 4 bytes a group of either."""
    if hd not in KV4_HEAD_DIMS or page_size < 16 or page_size & (page_size - 1):
        raise KernelError(f"a 4-bit cache has heads of {KV4_HEAD_DIMS} values and pages of a power of two of keys, at least 16, "
                          f"got head size {hd}, page size {page_size}")
    return page_size * (hd + 8 * (hd // kv4_group(hd)))


def _pages(t: torch.Tensor, name: str, page_size: int, G: int, hd: int) -> None:
    _need(t, name, torch.uint8)
    if t.dim() != 3 or tuple(t.shape[1:]) != (G, kv4_page_bytes(page_size, hd)):
        raise KernelError(f"{name}: expected [n_pages, {G}, {kv4_page_bytes(page_size, hd)}], got {tuple(t.shape)}")


def _mass(t: torch.Tensor, name: str, pages: torch.Tensor, page_size: int, G: int) -> None:
    _need(t, name, torch.float32)
    if tuple(t.shape) != (pages.shape[0], G, page_size):
        raise KernelError(f"{name}: expected [{pages.shape[0]}, {G}, {page_size}], got {tuple(t.shape)}")


def kv4_write(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, slot_map: torch.Tensor, page_size: int, G: int, hd: int) -> None:
    """Rows of keys and values [n, G hd] (float32 or bfloat16; columns of wider rows will do) to the slots ``slot_map`` names
    (int32: page * page_size + place; -1: nowhere).  A group is cut into 16 equal steps from its smallest value on, ``s =
    bfloat16((max - min) / 15)``, ``z = bfloat16(min)``, ``c = round((x - z) / s)`` (halves to even, within 0..15; 0 where s is
    0).  A group with a value that is not finite reads as NaN."""
    _need(k, "k", contiguous=False); _need(v, "v", k.dtype, contiguous=False); _need(slot_map, "slot_map", torch.int32)
    _pages(pages, "pages", page_size, G, hd)
    n = slot_map.numel()
    if tuple(k.shape) != (n, G * hd) or tuple(v.shape) != (n, G * hd):
        raise KernelError(f"kv4_write: expected k and v of [{n}, {G * hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    _run("kv4_write", load_library("kv4").kp_kv4_write, _ptr(k), ctypes.c_longlong(_rows_2d(k, "k")), _ptr(v), ctypes.c_longlong(_rows_2d(v, "v")),
         _ptr(pages), ctypes.c_longlong(pages.shape[0]), _ptr(slot_map), n, page_size, G, hd, dtype_code(k.dtype), STREAM)


def kv4_read(pages: torch.Tensor, slot_map: torch.Tensor, page_size: int, G: int, hd: int,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values in the slots, as rows [n, G hd] of ``dtype`` (a slot of -1 reads as zeros)."""
    _need(slot_map, "slot_map", torch.int32)
    _pages(pages, "pages", page_size, G, hd)
    code, n = dtype_code(dtype), slot_map.numel()
    k = torch.empty((n, G * hd), dtype=dtype, device=pages.device)
    v = torch.empty_like(k)
    _run("kv4_read", load_library("kv4").kp_kv4_read, _ptr(pages), ctypes.c_longlong(pages.shape[0]), _ptr(slot_map), _ptr(k), _ptr(v), n, page_size,
         G, hd, code, STREAM)
    return k, v


def kv4_chunks(n_seg: int, max_rows: int, max_context: int, window: Optional[int], H: int, G: int, hd: int) -> Tuple[int, int]:
    """(number of chunks, keys a chunk) of the split form: as many CTAs as fill the SMs, none with less than a tile a warp."""
    least = 256 if hd <= 64 else (128 if hd <= 128 else 64)
    span = max_context if not window else min(max_context, window + max_rows)
    want = max(1, _CTAS // max(1, n_seg * G * -(-max_rows * (H // G) // 8)))
    chunk = max(least, -(-span // want))
    chunk = -(-chunk // least) * least
    return -(-max_context // chunk), chunk


def kv4_tc_ok(q: torch.Tensor, out: torch.Tensor, hd: int, scale: float) -> bool:
    """Does the tcgen05 form take these rows (bfloat16, heads of 64 or 128, rows on 16-byte boundaries)?"""
    return (USE_TC_KV4 and q.dtype == torch.bfloat16 and hd in (64, 128) and scale > 0 and q.stride(0) % 8 == 0 and out.stride(0) % 8 == 0
            and q.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 0)


def kv4_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, cu_rows: torch.Tensor, seg_pos: torch.Tensor,
                  out: torch.Tensor, scale: float, window: Optional[int], page_size: int, H: int, G: int, hd: int, max_rows: int,
                  max_context: int, min_rows: int = 1, mass: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the rows q [n, H hd] over their sequences' 4-bit pages (this step's keys and values already in them).

    Rows ``cu_rows[i] .. cu_rows[i + 1] - 1`` belong to sequence ``i``; the first of them stands at key ``seg_pos[i]`` and reads
    the keys up to that one, of which ``window`` (None: all) the last; a row that reads none gives zeros.  ``max_rows`` and
    ``min_rows`` bound the rows of a sequence, ``max_context`` the keys that any row reads (host integers).  ``mass`` (float32
    [n_pages, G, page_size]): the softmax weight of every key, summed over the rows and the query heads of its kv head, is added
    to the key's entry (in a fixed order: the same call gives the same bits)."""
    _need(q, "q", contiguous=False); _need(out, "out", q.dtype, contiguous=False)
    _need(block_table, "block_table", torch.int32); _need(cu_rows, "cu_rows", torch.int32); _need(seg_pos, "seg_pos", torch.int32)
    _pages(pages, "pages", page_size, G, hd)
    n, n_seg = q.shape[0], seg_pos.numel()
    if G < 1 or H % G or tuple(q.shape) != (n, H * hd) or tuple(out.shape) != (n, H * hd):
        raise KernelError("kv4_attention: shape mismatch")
    if cu_rows.numel() != n_seg + 1 or block_table.dim() != 2 or block_table.shape[0] < n_seg:
        raise KernelError("kv4_attention: cu_rows has one entry more than seg_pos, block_table a row for each of them")
    if window is not None and window < 1:
        raise KernelError("kv4_attention: the window is a positive number of keys")
    if max_context < 1 or max_context > block_table.shape[1] * page_size:
        raise KernelError(f"kv4_attention: max_context={max_context} does not lie within the block table's {block_table.shape[1]} pages")
    if mass is not None:
        _mass(mass, "mass", pages, page_size, G)
    short = min(max_rows, KV4_SHORT_ROWS) if min_rows <= KV4_SHORT_ROWS else 0
    n_chunks, chunk = kv4_chunks(n_seg, max(short, 1), max_context, window, H, G, hd)
    part_o = part_ml = scores = lse_split = lse = None
    floats = lambda count: torch.empty(count, dtype=torch.float32, device=q.device)  # noqa: E731
    places = n_seg * short * H
    tiled = max_rows > KV4_SHORT_ROWS
    tc = tiled and kv4_tc_ok(q, out, hd, scale)
    if short and n_chunks > 1:
        part_o, part_ml = floats(places * n_chunks * hd), floats(places * n_chunks * 2)
    if mass is not None:
        if short:
            scores, lse_split = floats(places * n_chunks * chunk), floats(places)
        if tiled and not tc:
            lse = floats(n * H)
    ldq, ldo = ctypes.c_longlong(_rows_2d(q, "q")), ctypes.c_longlong(_rows_2d(out, "out"))
    if short or (tiled and not tc):
        _run("kv4_attention", load_library("kv4").kp_kv4_attention, _ptr(q), ldq, _ptr(pages), ctypes.c_longlong(pages.shape[0]), _ptr(block_table), block_table.shape[1], _ptr(cu_rows),
             _ptr(seg_pos), n_seg, _ptr(out), ldo, ctypes.c_float(scale), int(window or 0), page_size, H, G, hd, n, short, int(tiled and not tc),
             n_chunks, chunk, max_context, _ptr(part_o), _ptr(part_ml), _ptr(scores), n_chunks * chunk, _ptr(lse_split), _ptr(lse), _ptr(mass),
             dtype_code(q.dtype), STREAM)
    if tc:
        lib, scratch = load_library("kv4_tc"), None
        if mass is not None:
            lib.kp_kv4_tc_scratch.restype = ctypes.c_longlong
            scratch = torch.empty(lib.kp_kv4_tc_scratch(n, n_seg, H, G, hd), dtype=torch.uint8, device=q.device)
        _run("kv4_attention_tc", lib.kp_kv4_attention_tc, _ptr(q), ldq, _ptr(pages), _ptr(block_table), block_table.shape[1], _ptr(cu_rows),
             _ptr(seg_pos), n_seg, _ptr(out), ldo, ctypes.c_float(scale), int(window or 0), page_size, H, G, hd, n, short + 1, max_context,
             _ptr(mass), _ptr(scratch), STREAM)
    return out


def kv4_evict(pages: torch.Tensor, mass: torch.Tensor, block_table: torch.Tensor, n_keys: torch.Tensor, new_pages: torch.Tensor,
              new_mass: torch.Tensor, new_table: torch.Tensor, kept: torch.Tensor, max_keys: int, keep: int, recent: int, first: int,
              page_size: int, G: int, hd: int) -> torch.Tensor:
    """Of every sequence's ``n_keys[i]`` keys (int32; at most ``max_keys``) each kv head keeps ``keep``: the ``first`` first, the
    ``recent`` last and of the others those with the most ``mass`` (equal: the lowest index); all, where there are not more.
    They move with their mass to places 0, 1, ... of ``new_table``'s pages, in their order.  The new pages are none of the
    sequences' old ones.  ``kept`` (int32 [n, G, keep]) gets the old indices, -1 behind the last."""
    _pages(pages, "pages", page_size, G, hd); _pages(new_pages, "new_pages", page_size, G, hd)
    _mass(mass, "mass", pages, page_size, G); _mass(new_mass, "new_mass", new_pages, page_size, G)
    for t, nm in ((block_table, "block_table"), (new_table, "new_table"), (n_keys, "n_keys"), (kept, "kept")):
        _need(t, nm, torch.int32)
    n = n_keys.numel()
    if keep < 1 or min(recent, first) < 0 or first + recent > keep:
        raise KernelError(f"kv4_evict: keep={keep} is positive and not less than first={first} and recent={recent} together")
    if block_table.dim() != 2 or new_table.dim() != 2 or min(block_table.shape[0], new_table.shape[0]) < n or tuple(kept.shape) != (n, G, keep):
        raise KernelError("kv4_evict: block tables with a row a sequence and kept of [sequences, kv heads, keep]")
    if max_keys < 1 or max_keys > block_table.shape[1] * page_size or min(keep, max_keys) > new_table.shape[1] * page_size:
        raise KernelError("kv4_evict: the block tables hold max_keys keys, and the ones that stay")
    _run("kv4_evict", load_library("kv4_evict").kp_kv4_evict, _ptr(pages), _ptr(mass), _ptr(block_table), block_table.shape[1], _ptr(n_keys),
         _ptr(new_pages), _ptr(new_mass), _ptr(new_table), new_table.shape[1], _ptr(kept), n, max_keys, keep, recent, first, page_size, G, hd, STREAM)
    return kept
