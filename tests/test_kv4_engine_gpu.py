"""The engine with its attention's keys and values in 4 bits, against the plain model with its keys and values quantised.

Tolerances.  float32: as everywhere (tests/tolerances.py), since both quantise the same numbers; a number that lies within a float32 rounding of a half
between two codes could fall to either side, a chance of about 1e-5 for a whole run of these sizes.  bfloat16: activations that differ by
2^-9 of themselves fall to another code in one or two cases of a hundred, which adds to the rounding of 16-bit storage (5 % of the logits'
spread) about half as much again as the quantisation itself leaves: 15 % of the spread in all.
"""
import numpy as np
import pytest
import torch

from kappai_b200 import Engine, EngineArgs, ModelRunner, SamplingParams, StepEntry
from kappai_b200.config.schema import ConfigError
from kappai_b200.engine.runner import EngineError
from kappai_b200.ops.kernels import read_status
from kappai_b200.weights import write_random_model
from plain_lfm2 import PlainLfm2, attention, linear, rmsnorm, rope_neox, rope_tables, round_bf16
from test_kv4_gpu import plain_values
from tiny_configs import TINY_A, TINY_D
from tolerances import FP32_ATOL

pytestmark = pytest.mark.gpu

HEADS_32 = dict(TINY_D, hidden_size=96, num_attention_heads=6, num_key_value_heads=2, head_dim=32, block_ff_dim=160)
HEADS_128 = dict(TINY_D, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
CONFIGS = {"d64": (TINY_D, 3), "d32": (HEADS_32, 4), "d128": (HEADS_128, 5)}


class Plain4(PlainLfm2):
    """Keys behind the rotation and values are replaced by what 4 bits leave of them."""

    def attention_mixer(self, h, i):
        w, p = self.w, f"model.layers.{i}.self_attn."
        T = h.shape[0]
        q, k, v = (self.st(linear(h, w[p + n + "_proj.weight"])).reshape(T, heads, self.hd) for n, heads in (("q", self.H), ("k", self.G), ("v", self.G)))
        q, k = rmsnorm(q, w[p + "q_layernorm.weight"], self.eps), rmsnorm(k, w[p + "k_layernorm.weight"], self.eps)
        cos, sin = rope_tables(T, self.hd, self.theta)
        q, k = self.st(rope_neox(q, cos, sin)), self.st(rope_neox(k, cos, sin))
        o = self.st(attention(q, plain_values(k, self.hd), plain_values(v, self.hd), self.hd ** -0.5))
        return linear(o.reshape(T, self.H * self.hd), w[p + "out_proj.weight"])


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for name, (cfg, seed) in CONFIGS.items():
        d = str(tmp_path_factory.mktemp("kv4_" + name))
        write_random_model(cfg, d, seed)
        out[name] = d
    return out


def steps(runner, seqs, cuts):
    """The sequences' logits at every place, their tokens run in portions that end at ``cuts``, all sequences side by side."""
    got = [[] for _ in seqs]
    at = 0
    for cut in cuts:
        entries = [StepEntry(i, s[at:cut], list(range(len(s[at:cut])))) for i, s in enumerate(seqs) if s[at:cut]]
        logits = runner.step(entries).float().cpu().numpy()
        r = 0
        for e in entries:
            got[e.req].append(logits[r:r + len(e.tokens)])
            r += len(e.tokens)
        at = cut
    for i in range(len(seqs)):
        runner.end(i)
    return [np.concatenate(g) for g in got]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(CONFIGS))
@pytest.mark.parametrize("graphs", [False, True])
def test_logits(folders, name, dtype, graphs):
    rng = np.random.default_rng(1)
    seqs = [rng.integers(0, CONFIGS[name][0]["vocab_size"], n).tolist() for n in (90, 37, 61)]
    runner = ModelRunner(folders[name], dtype=dtype, max_tokens=512, max_requests=3, page_size=16, cuda_graphs=graphs, kv_bits=4)
    # a prompt in portions, a few tokens at once, then one at a time
    got = steps(runner, seqs, [30, 33, 34] + list(range(35, 91)))
    whole = steps(runner, seqs, [90])
    plain = Plain4(folders[name], storage=None if dtype == "float32" else "bfloat16")
    for have, other, s in zip(got, whole, seqs):
        want = plain.logits(s)
        tol = FP32_ATOL if dtype == "float32" else 0.15 * float(np.std(want))
        assert np.abs(have - want).max() <= tol and np.abs(other - want).max() <= tol
    assert not any(read_status().values())


def test_generation_and_what_the_cache_takes(folders):
    prompts = [[5, 9, 200, 17], list(range(40))]
    outs = {}
    for bits in (16, 4):
        eng = Engine(EngineArgs(model=folders["d64"], dtype="float32", max_batch=2, max_step_tokens=16, page_size=16, kv_tokens=256, kv_bits=bits))
        outs[bits] = (eng.generate(prompts, SamplingParams(temperature=0.0, n_predict=12)), eng.runner.storage.total_bytes(),
                      [eng.runner.storage.bytes_per_token(g) for g in eng.runner.storage.groups])
        assert eng.runner.cache_plan.cache_bytes == eng.runner.storage.total_bytes()
        eng.shutdown()
    assert [len(o) for o in outs[4][0]] == [12, 12]
    # 64 values and their range: 32 + 4 bytes in place of 256, for keys and for values, in two layers of one kv head
    assert outs[4][2] == [2 * 2 * 36] and outs[16][2] == [2 * 2 * 256]


def test_what_is_refused(folders, tmp_path):
    with pytest.raises(EngineError, match="kv_bits"):
        ModelRunner(folders["d64"], max_tokens=64, kv_bits=8)
    with pytest.raises(EngineError, match="power of two"):
        ModelRunner(folders["d64"], max_tokens=64, page_size=24, kv_bits=4)
    write_random_model(TINY_A, str(tmp_path / "a"), 0)                # heads of 16
    with pytest.raises(ConfigError, match="4 bits"):
        ModelRunner(str(tmp_path / "a"), max_tokens=64, page_size=16, kv_bits=4)
    conv_only = dict(TINY_D, layer_types=["conv"] * 3)
    write_random_model(conv_only, str(tmp_path / "c"), 0)
    with pytest.raises(EngineError, match="no mixer"):
        ModelRunner(str(tmp_path / "c"), max_tokens=64, page_size=16, kv_bits=4)


def test_command_line(folders, capsys):
    from kappai_b200.cli import main

    assert main(["-m", folders["d64"], "-p", "5,17,3", "-n", "6", "-t", "0", "--kv-bits", "4", "--dtype", "float32", "-c", "64", "--max-batch", "1", "--stream", "0"]) == 0
    assert len(capsys.readouterr().out.split()) == 6
