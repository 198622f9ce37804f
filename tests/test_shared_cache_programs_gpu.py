"""Random programs over a SharedCache on the device, against lists of keys and values and attention in 64 bits.

Tolerances as in the attention's own tests: 1e-4 for float32; for bfloat16 2^-8 of the weighted mean of |v| and of the output beside it."""
import pytest
import torch

from kappai_b200.ops import kernels as K
from shared_fakes import Program

pytestmark = pytest.mark.gpu


def program(H, G, hd, seed=0, **kw):
    a = dict(n_pages=300, max_seqs=16, max_len=700, page_size=16, dtype=torch.bfloat16)
    a.update(kw)

    def near(got, want, off):
        assert ((got.double().cpu() - want).abs() <= 1e-4 + (2.0 ** -8 * off if got.dtype == torch.bfloat16 else 0.0 * off)).all()

    return Program(H, G, hd, near, seed, device="cuda", **a)


@pytest.mark.parametrize("dtype,H,G,hd", [(torch.bfloat16, 8, 2, 64), (torch.bfloat16, 16, 1, 128), (torch.float32, 4, 2, 64)])
def test_a_fork_into_the_gap_that_ended_continuations_left(dtype, H, G, hd):
    p = program(H, G, hd, dtype=dtype)
    a = p.fork(160, 8)
    p.step()
    p.end(a[1:5])
    b = p.fork(32, 2)
    assert a[0] < b[0] < a[5]
    p.step()
    p.step([a[0], b[1], a[5], a[7]], [1, 3, 2, 1])
    p.end(b[:1])
    p.step()
    p.end(a[:1])
    p.step()


@pytest.mark.parametrize("seed,dtype,H,G,hd,page", [(0, torch.bfloat16, 8, 2, 64, 16), (1, torch.bfloat16, 16, 1, 128, 64), (2, torch.float32, 4, 2, 64, 7),
                                                    (3, torch.bfloat16, 6, 2, 96, 24), (4, torch.bfloat16, 32, 2, 64, 32)])
def test_random_programs(seed, dtype, H, G, hd, page):
    p = program(H, G, hd, seed, dtype=dtype, page_size=page, max_seqs=14)
    p.random(seed, 70, 300, 6)
    torch.cuda.synchronize()
    assert not any(K.read_status().values())


@pytest.mark.parametrize("P,n,H,G,hd", [(4096, 256, 32, 8, 128), (8000, 256, 32, 8, 64), (3001, 8000, 16, 2, 64)])
def test_long_prompts_in_caches_of_many_places(P, n, H, G, hd):
    """The prompt's rows, and a step of all of its continuations, whatever the cache has room for besides."""
    p = program(H, G, hd, page_size=64, max_len=P + 64, n_pages=P // 64 + 2 * n + 10, max_seqs=min(8192, 2 * n))
    x, some = p.make(P), [0, 1, 63, 64, 1000, P - 2, P - 1]
    out, seqs = p.c.fork(x, n)
    want, off, whole = p.attend(None, x, some)
    p.near(out[some], want, off)
    y = p.make(n)
    out = p.c.step(y)
    for i in (0, 1, n // 2, n - 1):
        want, off, _ = p.attend(whole, y[i:i + 1])
        p.near(out[i:i + 1], want, off)
    p.c.end(seqs[:n // 2])
    p.kv = {s: torch.cat([whole, y[i:i + 1, H * hd:].double().cpu().reshape(1, 2, G, hd)]) for i, s in enumerate(seqs) if i in (n // 2, n - 1)}
    p.prompt_of = dict.fromkeys(p.kv)
    z = p.make(3)
    out = p.c.step(z, [seqs[n // 2], seqs[n - 1]], [1, 2])
    for s, a, b in ((seqs[n // 2], 0, 1), (seqs[n - 1], 1, 3)):
        want, off, _ = p.attend(p.kv[s], z[a:b])
        p.near(out[a:b], want, off)
    p.c.check()


def test_a_prompt_of_more_rows_than_a_call_takes():
    """A very long text and questions about it: the text runs in portions."""
    P, n, H, G, hd = 120001, 24, 16, 8, 64
    p = program(H, G, hd, page_size=64, max_len=P + 1000, n_pages=P // 64 + 2 * n + 10, max_seqs=n + 1)
    x, some = p.make(P), [0, 65534, 65535, 65536, P - 1]
    out, seqs = p.c.fork(x, n)
    want, off, whole = p.attend(None, x, some)
    p.near(out[some], want, off)
    y = p.make(n)
    out = p.c.step(y)
    for i in (0, 11, n - 1):
        want, off, _ = p.attend(whole, y[i:i + 1])
        p.near(out[i:i + 1], want, off)
    p.c.check()
