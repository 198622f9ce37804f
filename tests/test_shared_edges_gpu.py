"""Attention behind a shared prefix at its edges: more places for sequences, groups and tiles of columns than a grid's second and third axis count.  Tolerances are those of
test_shared_gpu.py."""
import pytest

from kappai_b200.ops.shared import shared_cut
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
