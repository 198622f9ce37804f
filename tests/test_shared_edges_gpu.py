"""Attention behind a shared prefix at its edges: more places for sequences, groups and tiles of columns than a grid's second and third axis count.  Tolerances are those of
test_shared_gpu.py."""
import pytest
import torch

from kappai_b200.ops.shared import attention_shared, shared_cut
from test_shared_gpu import DT, Batch, spread

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DT))
def test_many_places_for_sequences_and_one_with_many_rows(dtype):
    assert shared_cut(1, 300, 700, 700, 0, 700, 1, 32, False, dtype == "f32").own_tiles * 300 > 65535
    Batch([(0, [(1, 0)] * 150 + [(700, 700)] + [(1, 0)] * 149)], 32, 1, 64, 64, dtype).check()


@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (96, "bf16"), (64, "f32")])
def test_many_groups_of_which_one_has_many_rows(hd, dtype):
    assert shared_cut(1000, 1501, 300, 300, 70, 300, 1, 32, True).own_tiles * 1501 > 65535 and shared_cut(1000, 1501, 300, 300, 70, 300, 1, 32, False).tiles * 1000 > 65535
    groups = [(17, [(2, 1)])] * 499 + [(70, [(300, 300)])] + [(5, spread(1, 9, 2))] * 500
    Batch(groups, 32, 1, hd, 16, dtype).check()


@pytest.mark.parametrize("hd,G", [(64, 2), (128, 1)])
def test_prefixes_of_which_one_is_much_longer(hd, G):
    """The chunks' length is found among hundreds."""
    Batch([(17, spread(1, 5, 5))] * 15 + [(50001, spread(1, 9, 5))] + [(300, spread(1, 5, 5))] * 12, 4 * G, G, hd, 64, "bf16", seed=hd).check()


@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "bf16"), (96, "bf16"), (64, "f32")])
def test_calls_one_behind_another_in_which_few_places_have_rows(hd, dtype):
    """Calls that follow one another use the same scratch: each ends before the next one's kernels write there, whichever of its places have rows, or none."""
    last = Batch([(3000, [(9, 0)] * 60 + [(40, 3)])], 8, 2, hd, 64, dtype, seed=1)
    first = Batch([(2500, [(30, 3)] + [(9, 0)] * 60)], 8, 2, hd, 64, dtype, seed=2)
    none = Batch([(2500, [(9, 1)] * 40)], 8, 2, hd, 64, dtype, seed=3)
    want, out = [b.check() for b in (last, first)], []
    a = none.args()
    a["cu_rows"].zero_()
    for i in range(30):
        for j, b in enumerate((last, first)):
            out.append((j, b.args()))
    torch.cuda.synchronize()
    for j, args in out:
        attention_shared(**args)
        attention_shared(**a)
    torch.cuda.synchronize()
    assert all(torch.equal(args["out"], want[j]) for j, args in out) and (a["out"] == 7).all()


@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "bf16"), (64, "f32")])
@pytest.mark.parametrize("step", [0, 8])
def test_rows_that_lie_in_one_another(step, hd, dtype):
    """One row for all, and rows that begin within the one before."""
    b = Batch([(333, spread(1, 90, 20))], 8, 2, hd, 16, dtype, seed=5)
    n, w = b.q.shape
    flat = torch.randn(w + n * step, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(b.q.dtype)
    q = flat.as_strided((n, w), (step, 1))
    b.q = q.contiguous()
    b.check(attention_shared(**b.args(q=q)))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("seqs", [3, 12, 30, 60])
@pytest.mark.parametrize("hd", [64, 128, 96])
def test_values_of_the_prefix_that_are_not_finite(hd, seqs, bad):
    """They reach every row, in their place and no other, and nothing there is finite (NaN perhaps where the definition gives an infinite one)."""
    b = Batch([(300, spread(1, 40, seqs)), (50, spread(1, 9, 3))], 8, 2, hd, 64, "bf16", seed=3)
    for i in range(seqs):
        b.v[i][17, 1, 5] = bad
    b.cache[int(b.table[0, 0]), 1, 1, 17, 5] = bad
    b.check()
