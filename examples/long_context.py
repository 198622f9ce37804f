"""One attention layer over a long text with a bounded cache: keys and values in 4 bits, most of them evicted by their weight.

    python examples/long_context.py [--tokens 8192] [--budget 2048] [--new 64]

A prompt is run in portions through :class:`kappai_b200.Kv4Cache`; whenever the cache has more keys than the budget, each kv head
keeps the first ones, the recent ones and those that got the most attention.  Then tokens are decoded one at a time.  The rows'
outputs are compared with exact attention over all keys (and so are those of a 4-bit cache that keeps every key), and what the cache takes
with what 16-bit keys and values would.
Keys and queries are made so that some keys matter to every later query, as the keys of a trained model do.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from kappai_b200 import Kv4Cache  # noqa: E402


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--budget", type=int, default=2048)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--portion", type=int, default=1024)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--dim", type=int, default=64)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    H, G, hd, dev = a.heads, a.kv_heads, a.dim, "cuda"
    n, scale, page = a.tokens + a.new, hd ** -0.5, 64
    gen = torch.Generator(device=dev).manual_seed(a.seed)
    topic = torch.randn((G, hd), generator=gen, device=dev)
    k = torch.randn((n, G, hd), generator=gen, device=dev)
    k += topic * (2.0 * (torch.rand((n, G, 1), generator=gen, device=dev) < 0.05))
    q = torch.randn((n, G, H // G, hd), generator=gen, device=dev) + 0.5 * topic[:, None]
    v = torch.randn((n, G, hd), generator=gen, device=dev)
    q, k, v = (x.reshape(n, -1).bfloat16() for x in (q, k, v))

    cache = Kv4Cache(G, hd, n_pages=2 * (-(-(a.budget + a.portion) // page)) + 2, page_size=page, mass=True, device=dev)
    cache.add("text")
    outs, evicted = [], 0
    at = 0
    while at < n:
        rows = min(a.portion, a.tokens - at) if at < a.tokens else 1
        cache.append(k[at:at + rows], v[at:at + rows], ["text"], [rows])
        outs.append(cache.attend(q[at:at + rows], ["text"], [rows], H, scale))
        at += rows
        if cache.length("text") > a.budget:
            evicted += cache.length("text") - a.budget
            cache.evict(["text"], a.budget, recent=a.budget // 4, first=4)
    out = torch.cat(outs).float().view(n, H, hd)

    # the decoded rows over every key: from 4 bits, and exactly
    whole = Kv4Cache(G, hd, n_pages=-(-n // page), page_size=page, device=dev)
    whole.add("text")
    whole.append(k, v, ["text"], [n])
    all_keys = whole.attend(q[a.tokens:], ["text"], [a.new], H, scale).float().view(a.new, H, hd)
    kk, vv = (x.float().view(n, G, hd).repeat_interleave(H // G, 1) for x in (k, v))
    s = torch.einsum("rhd,khd->hrk", q[a.tokens:].float().view(a.new, H, hd), kk) * scale
    s.masked_fill_(torch.arange(n, device=dev) > torch.arange(a.tokens, n, device=dev)[:, None], float("-inf"))
    want = torch.einsum("hrk,khd->rhd", torch.softmax(s, -1), vv)
    got = out[a.tokens:]
    error, error_4bit = (float((x - want).norm() / want.norm()) for x in (got, all_keys))
    weight = torch.softmax(s, -1)
    held, full = cache.length("text") * cache.bytes_per_token(), n * G * hd * 4
    print(f"{a.tokens} tokens of prompt, {a.new} decoded; {evicted} keys evicted, {cache.length('text')} kept "
          f"({held / 1e6:.2f} MB, {full / 1e6:.2f} MB with all keys in 16 bits)")
    print(f"decoded rows: relative difference from exact attention over all {n} keys {error:.3f}, of which all keys in 4 bits {error_4bit:.3f} "
          f"(the {a.budget} largest weights of a row hold {float(weight.topk(min(a.budget, n), -1).values.sum(-1).mean()):.3f} of it)")
    return {"error": error, "error_4bit": error_4bit, "kept": cache.length("text"), "evicted": evicted, "held": held, "full": full}


if __name__ == "__main__":
    main()
