"""What the model thought of a token: host side of :func:`kappai_b200.ops.logprobs.token_logprobs`."""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Tuple

import torch


@dataclass
class TokenLogprob:
    """A token under the model's own distribution at its place: no penalty, temperature or filter of the sampler has a part in it."""

    token: int
    logprob: float
    rank: int                                       # tokens with a larger logit
    entropy: float                                  # of the distribution, in nats
    top: List[Tuple[int, float]] = field(default_factory=list)      # the tokens with the largest logits and their log probabilities


def packed(got) -> torch.Tensor:
    """A :class:`~kappai_b200.ops.logprobs.TokenLogprobs` as one float32 tensor [n, 3 + 2 top], whole numbers as their bits: for one copy."""
    bits = lambda t: t.view(torch.float32)  # noqa: E731
    return torch.cat((got.logprob[:, None], got.entropy[:, None], bits(got.rank)[:, None], got.top_logprobs, bits(got.top_ids)), 1)


def unpacked(host: torch.Tensor, row: int, token: int, top: int) -> TokenLogprob:
    """Row ``row`` of what :func:`packed` made, on the host, with its first ``top`` alternatives."""
    f, i = host[row], host[row].view(torch.int32)
    most = (host.shape[1] - 3) // 2
    return TokenLogprob(token, float(f[0]), int(i[2]), float(f[1]),
                        list(zip(i[3 + most:3 + most + top].tolist(), f[3:3 + top].tolist())))
