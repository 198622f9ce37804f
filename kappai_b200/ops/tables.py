"""Python face of the kernel that makes a step's tables on the GPU (``csrc/tables.cu``)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .build import load_library
from .kernels import MAX_STEP_ROWS, STREAM, KernelError, _run
from .kv4 import _here, _unlike

MAX_TABLE_SEQS = 8192      # sequences of a call: their sums lie in shared memory

# bits of a call's status word
TABLES_NO_PAGES, TABLES_TOO_NARROW, TABLES_NO_ROOM, TABLES_NO_SENSE = 1, 2, 4, 8

_P, _I = ctypes.c_void_p, ctypes.c_int
_NAMES = ("block_table", "length", "delta", "free_pages", "n_free", "cu_rows", "seg_pos", "row_seg", "positions", "slot_map", "status", "own_from")
_page_tables = None


def _launcher():
    global _page_tables
    if _page_tables is None:
        fn = load_library("tables").kp_page_tables
        fn.argtypes = [_P, _I, _P, _P, _P, _P, _I, _P, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P]
        _page_tables = fn
    return _page_tables


def page_tables(block_table: torch.Tensor, length: torch.Tensor, delta: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor, page_size: int,
                cu_rows: torch.Tensor, seg_pos: torch.Tensor, row_seg: torch.Tensor, positions: torch.Tensor, slot_map: torch.Tensor,
                status: torch.Tensor, own_from: Optional[torch.Tensor] = None) -> None:
    """One step of the sequences' lengths and pages, with the tables that its rows need; everything is int32 on the device, and nothing of it passes
    through the host, so a call can be captured and replayed.

    ``length[i]`` tokens of sequence ``i`` lie in the pages ``block_table[i, :ceil(length / page_size)]``, and it changes by ``delta[i]``: a positive
    one gives it that many rows, for which it gets pages where its last one is full; a negative one takes its last tokens back, with the
    pages that are then empty; one that leaves no token ends it.  The first ``own_from[i]`` blocks (None: none) are other sequences' too: their
    pages are never given back, and a sequence is cut back no further than to their end unless it ends.  Free pages are the first ``n_free[0]``
    numbers of ``free_pages`` (with room for all pages), taken from the end; pages come back there such that a step and the one that takes it
    back (the negated ``delta``) leave the stack as it was.  Entries of pages that were given back, or forgotten, become -1.

    The step's rows, sequence by sequence: ``cu_rows`` [n + 1] gets each sequence's first row, ``seg_pos`` [n] the position of that row (the new length
    where there is none), and ``row_seg``, ``positions``, ``slot_map`` (of one length, the most rows that a step may have) each row's sequence, position
    and slot (page * page_size + place); behind the last row these hold 0, -1 and -1.

    ``status`` [1] gets 0, or the sum of what kept the step from being made: 1 too few free pages, 2 a block table too narrow, 4 more rows than
    room for them, 8 lengths or counts that make no sense.  A sequence that adds 2 or 8 asks for no rows and pages: 1 and 4 are about the others.
    Then nothing changes, and the step has no rows."""
    dev, i32 = _here(block_table), torch.int32
    given = (block_table, length, delta, free_pages, n_free, cu_rows, seg_pos, row_seg, positions, slot_map, status) if own_from is None else (
        block_table, length, delta, free_pages, n_free, cu_rows, seg_pos, row_seg, positions, slot_map, status, own_from)
    for i, t in enumerate(given):
        if not isinstance(t, torch.Tensor) or t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            _unlike(t, _NAMES[i], i32)
    S, cap, P = length.numel(), slot_map.numel(), free_pages.numel()
    if block_table.dim() != 2 or block_table.shape[0] != S or delta.numel() != S or seg_pos.numel() != S or cu_rows.numel() != S + 1 or (
            own_from is not None and own_from.numel() != S):
        raise KernelError("page_tables: a row of the block table, a change, a position and an own_from for every length; cu_rows has one entry more")
    if row_seg.numel() != cap or positions.numel() != cap or n_free.numel() != 1 or status.numel() != 1:
        raise KernelError("page_tables: row_seg, positions and slot_map are of one length, n_free and status have one entry")
    if S > MAX_TABLE_SEQS or cap > MAX_STEP_ROWS:
        raise KernelError(f"page_tables: at most {MAX_TABLE_SEQS} sequences and {MAX_STEP_ROWS} rows, got {S} and {cap}")
    width = block_table.shape[1]
    if page_size < 1 or S * width >= 2 ** 31 - 1 or max(P, width) * page_size >= 2 ** 31:
        raise KernelError("page_tables: slots and positions are 32-bit numbers, below 2^31")
    _run("page_tables", _launcher(), block_table.data_ptr(), width, length.data_ptr(), delta.data_ptr(), None if own_from is None else own_from.data_ptr(),
         free_pages.data_ptr(), P, n_free.data_ptr(), page_size, S, cap, cu_rows.data_ptr(), seg_pos.data_ptr(), row_seg.data_ptr(), positions.data_ptr(),
         slot_map.data_ptr(), status.data_ptr(), STREAM)
