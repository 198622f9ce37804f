"""Python face of the log probabilities' kernel (``csrc/logprobs.cu``)."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from .build import load_library
from .kernels import STREAM, KernelError, _rows_2d, _run, dtype_code
from .kv4 import _have, _here, _unlike

MAX_TOP_LOGPROBS = 32      # alternatives of a row
_CTAS = 148 * 2            # CTAs up to which rows are shared out over clusters
_LEAST = 2048              # logits below which a CTA has too little to do

_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_token_logprobs = None


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` says of each row, on the device."""

    logprob: torch.Tensor          # float32 [n]: the given token's log probability (0 where none is given)
    entropy: torch.Tensor          # float32 [n]: of the row's distribution, in nats
    rank: torch.Tensor             # int32 [n]: how many tokens have a larger logit than the given one (-1 where none is given)
    top_ids: torch.Tensor          # int32 [n, top]: the tokens with the largest logits, equal ones by index
    top_logprobs: torch.Tensor     # float32 [n, top]: their log probabilities


def _launcher():
    global _token_logprobs
    if _token_logprobs is None:
        fn = load_library("logprobs").kp_token_logprobs
        fn.argtypes = [_P, _L, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _I, _P]
        _token_logprobs = fn
    return _token_logprobs


@lru_cache(maxsize=4096)
def logprob_parts(n: int, V: int, top: int) -> int:
    """CTAs that share a row: as many as two an SM, none with less than a few thousand logits.  Measured, 64 rows of 65536 float32 logits with twenty
    alternatives: 1, 2, 4 and 8 CTAs a row 14.3, 11.9, 11.6 and 22.1 us; 120 rows 14.8, 14.0, 22.4 and 33.7; one row 13.3, 10.5, 8.5 and 8.9, without alternatives
    10.3, 7.0, 5.1 and 4.6."""
    parts = 1
    while parts < 4 and n * parts * 2 <= _CTAS and V // (parts * 2) >= _LEAST:
        parts *= 2
    return 8 if parts == 4 and not top and n * 16 <= _CTAS and V // 8 >= _LEAST else parts


def token_logprobs(logits: torch.Tensor, ids: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """Log probabilities under the softmax of each row of ``logits`` [n, vocab] (float32 or bfloat16; rows may lie any distance apart):
    of the token ``ids[r]`` (int32; -1, or a number that is no token: none), and of the ``top`` (at most 32) tokens with the largest logits; the row's
    entropy; and the given token's rank.

    Logits of -inf have no probability; a row of nothing else has log probabilities of -inf and no entropy.  A row with a NaN or +inf gives NaN, and
    -1 for its alternatives."""
    dev = _here(logits)
    if dev < 0 or logits.get_device() != dev:
        _unlike(logits, "logits", logits.dtype if isinstance(logits, torch.Tensor) else torch.float32, contiguous=False)
    code, ld, (n, V) = dtype_code(logits.dtype), _rows_2d(logits, "logits"), logits.shape
    if V < 1 or top < 0 or top > MAX_TOP_LOGPROBS or top > V:
        raise KernelError(f"token_logprobs: top={top} of {V} tokens; at most {MAX_TOP_LOGPROBS}, and no more than there are")
    pid = None
    if ids is not None:
        pid = _have(ids, "ids", torch.int32, dev)
        if ids.numel() != n:
            raise KernelError(f"token_logprobs: one token a row, got {ids.numel()} for {n} rows")
    if n > (2 ** 31 - 1) // 8:
        raise KernelError(f"token_logprobs: {n} rows are more than a launch takes")
    # (tensors of their own: views of one cost more than they save)
    where, shape, steps = logits.device, (n, top), (top, 1)
    logprob = torch.empty(n, dtype=torch.float32, device=where)
    entropy = torch.empty_like(logprob)
    rank = torch.empty(n, dtype=torch.int32, device=where)
    top_ids = torch.empty_strided(shape, steps, dtype=torch.int32, device=where)
    top_logprobs = torch.empty_strided(shape, steps, dtype=torch.float32, device=where)
    if n:
        _run("token_logprobs", _launcher(), logits.data_ptr(), ld, pid, n, V, top, logprob_parts(n, V, top), logprob.data_ptr(), entropy.data_ptr(), rank.data_ptr(),
             top_ids.data_ptr(), top_logprobs.data_ptr(), code, STREAM)
    return TokenLogprobs(logprob, entropy, rank, top_ids, top_logprobs)
