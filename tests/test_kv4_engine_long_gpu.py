"""The engine with its attention's keys and values in 4 bits where a context has several chunks, sequences' lengths differ much, keys leave a window
(and their pages the sequence), and a layer reads the cache of another.

Tolerances.  Both sides quantise numbers that differ by a few float32 roundings.  Of a quarter of a million values a few lie that near to a half between
two codes, or their group's scale or minimum to one between two bfloat16 numbers, and fall to either side.  A code is a fifteenth of a group's range in
one of 64 values of one key: 3 % of that key, and no more of what any row reads.  So the bound of 32-bit runs is 5 % of the logits' spread; with bfloat16 it is
the 15 % of test_kv4_engine_gpu.py.  A key too many or too few, or one of another sequence, moves these models' logits by far more.
"""
import json

import numpy as np
import pytest

import plain_tupalorn
from kappai_b200 import ModelRunner
from kappai_b200.models import tupalorn
from kappai_b200.ops.kernels import read_status
from kappai_b200.weights import write_random_model
from kappai_b200.weights.safetensors_io import save_safetensors
from test_kv4_engine_gpu import Plain4, steps
from test_kv4_gpu import plain_values
from tiny_configs import TINY_D
from tupalorn_configs import _attention, _layer, _mamba2, _model, make_weights

pytestmark = pytest.mark.gpu

WINDOWS = _model(211, 128, [
    _layer(_attention(4, 2, 64, 64, 40), 128, 1.0),
    _layer(_mamba2(4, 16, 16, 2, 3, 4), None),
    _layer(_attention(4, 2, 64, 64, 100, kv_from=0), 128, 1.0),
    _layer(_attention(2, 1, 32, 32, None), 96, 1.0),
], softcap=12.0, max_positions=400)


def compare(runner, seqs, cuts, plain, dtype):
    got = steps(runner, seqs, cuts)
    for have, s in zip(got, seqs):
        want = plain(s)
        assert np.abs(have - want).max() <= (0.05 if dtype == "float32" else 0.15) * float(np.std(want))
    assert not any(read_status().values())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [False, True])
def test_contexts_of_several_chunks(tmp_path, dtype, graphs):
    write_random_model(TINY_D, str(tmp_path), 3)
    rng = np.random.default_rng(1)
    seqs = [rng.integers(0, TINY_D["vocab_size"], n).tolist() for n in (640, 12, 615, 3)]
    runner = ModelRunner(str(tmp_path), dtype=dtype, max_tokens=2048, max_requests=4, page_size=16, cuda_graphs=graphs, kv_bits=4)
    plain = Plain4(str(tmp_path), storage=None if dtype == "float32" else "bfloat16")
    compare(runner, seqs, [2, 3, 5, 500, 602, 606] + list(range(607, 641)), plain.logits, dtype)


@pytest.mark.parametrize("graphs", [False, True])
def test_windows_and_a_borrowed_cache(tmp_path, graphs, monkeypatch):
    """(In 32 bits: with bfloat16 the codes that fall to the other side move this model's logits, whose gains are large, by a quarter of their spread here and
    there, and there is no plain form of it with that storage.)"""
    (tmp_path / "config.json").write_text(json.dumps(WINDOWS))
    save_safetensors(str(tmp_path / "model.safetensors"), make_weights(WINDOWS, 8))
    own = plain_tupalorn.attention_keys_values

    def quantised(h, w, m, eps):
        return tuple(plain_values(x.astype(np.float32), x.shape[-1]) for x in own(h, w, m, eps))

    monkeypatch.setattr(plain_tupalorn, "attention_keys_values", quantised)
    # (this design asks for softmax weights in 32 bits, which goes with a cache in 16: here it does not)
    monkeypatch.setattr(tupalorn, "SOFTMAX_WEIGHTS", "operand")
    rng = np.random.default_rng(2)
    seqs = [rng.integers(0, WINDOWS["vocab"], n).tolist() for n in (260, 25, 230)]
    runner = ModelRunner(str(tmp_path), dtype="float32", max_tokens=1024, max_requests=3, page_size=16, max_step_tokens=256, cuda_graphs=graphs, kv_bits=4)
    compare(runner, seqs, [20, 23, 24, 25, 90, 150, 200] + list(range(201, 261)), plain_tupalorn.PlainTupalorn(str(tmp_path)).forward, "float32")
