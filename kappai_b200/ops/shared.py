"""Python face of attention behind a shared prefix (``csrc/shared.cuh`` has its formulas and how the work is cut)."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple

import torch

from .build import load_library
from .kernels import F32, STREAM, KernelError, _run, dtype_code
from .kv4 import _have, _have_rows, _here, _unlike

SHARED_HEAD_DIMS = (32, 64, 96, 128, 192, 256)
SHARED_MAX_KEYS = 1 << 30      # that a block table has room for: the kernels count keys in 32 bits
_SMS = 148
_MAX_CHUNKS, _MAX_CLUSTER = 64, 8
_AXIS = 65535                  # a grid's second and third axis
_SCRATCH = 1 << 28             # values of scratch above which a prefix is cut into fewer chunks
TC_MIN_COLS = 16               # columns of a group above which the tcgen05 form takes its prefix

USE_TC_SHARED = True           # the prefix's part of bfloat16 rows with heads of 64 or 128 runs on the tcgen05 tensor cores

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
_attention_shared, _prefix_tc = {}, None


def _tc_address() -> int:
    """The address of the prefix's tcgen05 form, which the launcher of both calls."""
    global _prefix_tc
    if _prefix_tc is None:
        _prefix_tc = ctypes.cast(load_library("shared_tc").kp_attention_shared_prefix_tc, ctypes.c_void_p).value
    return _prefix_tc


def _launcher(f32: bool):
    fn = _attention_shared.get(f32)
    if fn is None:
        fn = load_library("shared_f32").kp_attention_shared_f32 if f32 else load_library("shared").kp_attention_shared
        fn.argtypes = [_P, _L, _P, _L, _P, _I, _P, _P, _P, _P, _I, _I, _I, _P, _L, _P, _P, _I, _I, _F] + [_I] * 11 + [_P, _I, _I, _P]
        _attention_shared[f32] = fn
    return fn


class SharedCut(NamedTuple):
    """How the work of a call is cut."""

    tile: int          # columns of a tile of the prefix (0: there is none; 128: the tcgen05 form)
    mode: int          # of that: 0, 256 columns a CTA; 1, 128, whose tiles of keys two sets of warps take in turn; 2, 64, with half a tile of keys a warp
    budget: int        # of that: CTAs that the prefixes of all groups are shared out over (0: chunks are of one length)
    tiles: int         # of columns, a group
    chunks: int        # of a prefix, at most (0: there is none)
    chunk: int         # keys a chunk (with a budget: at least)
    own_tile: int      # columns of a tile of a sequence's own keys
    own_tiles: int     # of those, a sequence
    ctas: int          # that share a tile's own keys


@lru_cache(maxsize=4096)
def shared_cut(n_groups: int, n_seq: int, max_rows: int, max_group_rows: int, max_prefix: int, max_own: int, G: int, R: int, tc: bool, f32: bool = False,
               most: int = _MAX_CHUNKS, hd: int = 64) -> SharedCut:
    """Keys are shared out until the SMs have work, none with less than a few tiles of keys, a prefix over at most ``most`` CTAs a tile of columns.  Tiles are
    no wider than the columns need."""
    def columns(n):
        return 8 if n <= 8 else (16 if n <= 16 else (32 if n <= 32 and f32 else 64))

    def own(chunks):
        # (a cluster shares the join of its columns' parts as well as the keys; 64 columns take twice as long for a tile of keys as 8, and with wide heads want
        # an SM for themselves beside the prefix's)
        cols = max_rows * R
        tile = columns(cols)
        tiles, least = -(-cols // tile), 96 if f32 else (128 if tile == 64 else 384)
        return tile, tiles, max(1, min(_SMS // (2 * n_seq * tiles * G) if tile == 64 and hd > 128 else -(-2 * _SMS // (n_seq * tiles * G)), _MAX_CLUSTER, max(-(-max_own // least), -(-chunks * min(cols, tile) // 256))))

    if not max_prefix:
        return SharedCut(0, 0, 0, 1, 0, 64, *own(0))
    cols = max_group_rows * R
    if tc and cols > TC_MIN_COLS:
        mode = 2 if max_group_rows <= 64 // R else (1 if max_group_rows <= 128 // R else 0)
        tiles = 1 if mode else -(-max_group_rows // (128 // R * 2))
        keys, items = -(-max_prefix // 128), n_groups * tiles * G
        if 1 < n_groups <= 32 and items <= _SMS:
            # (a prefix that is all there is has the shortest chunks)
            least = max(-(-keys * tiles * G // _SMS), -(-keys // most))
            return SharedCut(128, mode, _SMS, tiles, -(-keys // least), least * 128, *own(-(-keys // least)))
        chunk = -(-keys // min(max(1, _SMS // items), -(-keys // (2 if mode else 1)), most)) * 128
        return SharedCut(128, mode, 0, tiles, -(-max_prefix // chunk), chunk, *own(-(-max_prefix // chunk)))
    tile = columns(cols)
    while f32 and tile > 16 and n_groups * -(-cols // tile) * G * -(-max_prefix // 128) < _SMS:
        tile //= 2             # (few CTAs have narrower tiles: 20 rows of 6 heads of 256 behind 274 keys, 64 columns a tile 95 us, 16 62)
    tiles = -(-cols // tile)
    chunks = max(1, min(-(-(3 if f32 else 2) * _SMS // (n_groups * tiles * G)), most, -(-max_prefix // (128 if f32 else 256))))
    chunk = -(-max_prefix // (chunks * 64)) * 64
    return SharedCut(tile, 0, 0, tiles, -(-max_prefix // chunk), chunk, *own(-(-max_prefix // chunk)))


def shared_tc_ok(ldq: int, q: int, n_pages: int, page_size: int, G: int, R: int, hd: int) -> bool:
    """Can the tcgen05 form take the prefix of a call with bfloat16 rows (heads of 64 or 128, rows ``ldq`` values apart, one behind the other, on 16-byte boundaries from address ``q``
    on, pages of which a tile of 128 keys is made)?"""
    return (USE_TC_SHARED and (hd == 64 or hd == 128) and R <= 128 and ldq % 8 == 0 and ldq >= G * R * hd and q % 16 == 0
            and page_size % 8 == 0 and (page_size % 128 == 0 or 128 % page_size == 0) and n_pages * 2 * G * page_size < 2 ** 31 - 1)


def attention_shared(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, cu_rows: torch.Tensor, seg_pos: torch.Tensor, group_seqs: torch.Tensor,
                     prefix_len: torch.Tensor, out: torch.Tensor, scale: float, page_size: int, H: int, G: int, hd: int, max_rows: int, max_group_rows: int,
                     max_prefix: int, max_own: int) -> torch.Tensor:
    """Causal attention of the rows q [n, H hd] over their sequences' pages, where groups of sequences share their first keys: those are read once
    for all rows of a group.

    ``cache`` [pages, 2, G, page_size, hd] has keys and values (this step's in them already).  Rows ``cu_rows[i] .. cu_rows[i + 1] - 1`` belong to
    sequence ``i``, the first of them stands at key ``seg_pos[i]`` and reads the keys up to that one; ``block_table[i]`` has all of the sequence's pages,
    the shared ones in front.  Sequences ``group_seqs[g] .. group_seqs[g + 1] - 1`` are group ``g``: the first ``prefix_len[g]`` keys are the same for all of
    them (read from the pages of the group's first sequence; a page that the prefix ends in may be each sequence's own copy), and no row stands before
    their end (``seg_pos[i] >= prefix_len[g]``).  A sequence in no group shares nothing.  All int32 on the device.

    Host bounds: ``max_rows`` rows of a sequence, ``max_group_rows`` rows of a group, ``max_prefix`` shared keys, ``max_own`` keys of a sequence
    behind them.  ``out`` is other memory than ``q``; rows behind ``cu_rows[-1]`` are left as they were, and a row that reads no key gives zeros.  Keys and values
    that a row does not read may be anything; where it reads an infinite value the output is infinite or NaN.  float32 or bfloat16,
    accumulated in float32; the sums' order is fixed, so the same call gives the same bits."""
    if G < 1 or H < 1 or H % G:
        raise KernelError(f"attention_shared: {H} query heads over {G} kv heads")
    if hd not in SHARED_HEAD_DIMS or page_size < 1:
        raise KernelError(f"attention_shared: heads of {SHARED_HEAD_DIMS} values and pages of at least one key, got {hd} and {page_size}")
    if max_rows < 1 or max_group_rows < 1 or max_prefix < 0 or max_own < 0:
        raise KernelError(f"attention_shared: max_rows={max_rows} and max_group_rows={max_group_rows} are positive, max_prefix={max_prefix} and max_own={max_own} not negative")
    if not 0.0 < scale < float("inf"):
        raise KernelError(f"attention_shared: the scale is a positive number, got {scale}")
    dev, dtype, i32 = _here(cache), q.dtype, torch.int32
    f32 = dtype_code(dtype) == F32
    at = _have(cache, "cache", dtype, dev)
    for i, t in enumerate((block_table, cu_rows, seg_pos, group_seqs, prefix_len)):
        if not isinstance(t, torch.Tensor) or t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            _unlike(t, ("block_table", "cu_rows", "seg_pos", "group_seqs", "prefix_len")[i], i32)
    n, n_seq, n_groups = q.shape[0], seg_pos.numel(), prefix_len.numel()
    pq, ldq = _have_rows(q, "q", dtype, n, H * hd, dev)
    po, ldo = _have_rows(out, "out", dtype, n, H * hd, dev)
    shape, pages = block_table.shape, cache.shape
    if len(pages) != 5 or pages[1:] != (2, G, page_size, hd) or at % 16:
        raise KernelError(f"attention_shared: cache of [pages, 2, {G}, {page_size}, {hd}] on a 16-byte boundary, got {tuple(pages)}")
    if cu_rows.numel() != n_seq + 1 or group_seqs.numel() != n_groups + 1 or len(shape) != 2 or shape[0] < n_seq:
        raise KernelError("attention_shared: cu_rows has one entry more than seg_pos, group_seqs one more than prefix_len, block_table a row for each sequence")
    if not n or not n_seq:
        return out
    width = shape[1]
    if not pages[0] or width < 1 or width * page_size > SHARED_MAX_KEYS or max_prefix > width * page_size:
        raise KernelError(f"attention_shared: max_prefix={max_prefix} does not lie within the block table's {width} pages, these have more than {SHARED_MAX_KEYS} keys, "
                          "or there is no page")
    R = H // G
    if not n_groups:
        max_prefix = 0
    cut = shared_cut(max(1, n_groups), n_seq, min(max_rows, n), min(max_group_rows, n), max_prefix, max_own, G, R,
                     not f32 and shared_tc_ok(ldq, pq, pages[0], page_size, G, R, hd), f32, max(1, min(_MAX_CHUNKS, _SCRATCH // (n * H * (hd + 2)))), hd)
    tile, mode, budget, tiles, chunks, chunk, own_tile, own_tiles, ctas = cut
    if -(-max(n_groups * tiles, n_seq * own_tiles) // _AXIS) * G > _AXIS or max(n_groups * tiles, n_seq * own_tiles) >= 2 ** 31 - 2 ** 16:
        raise KernelError(f"attention_shared: {n_seq} sequences in {n_groups} groups are more than a launch takes")
    tc = tile == 128
    p0 = p1 = scratch = None
    if chunks:
        scratch = torch.empty(n * H * chunks * (hd + 2), dtype=torch.float32, device=q.device)       # (has a name until the launches are queued)
        p0 = scratch.data_ptr()
        p1 = p0 + 4 * n * H * chunks * hd
    _run("attention_shared", _launcher(f32), pq, ldq, at, pages[0], block_table.data_ptr(), width, cu_rows.data_ptr(), seg_pos.data_ptr(), group_seqs.data_ptr(),
         prefix_len.data_ptr(), n, n_seq, n_groups, po, ldo, p0, p1, chunks, chunk, scale, page_size, H, G, hd, max_prefix, 64 if tc else (tile or 8), tiles, own_tile,
         own_tiles, ctas, max_own, _tc_address() if tc else None, mode, budget, STREAM)
    return out
