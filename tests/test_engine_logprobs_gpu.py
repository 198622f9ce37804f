"""Log probabilities through the engine: of sampled tokens, of prompts, on the command line.

Tolerances are those of the engine's logits (tolerances.py): a log probability is a logit less a logarithm of a sum of their exponentials, so it is off by at most twice what
the logits are."""
import os
import subprocess
import sys

import numpy as np
import pytest

from tolerances import tol_for

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def engine(model_dir, dtype="float32", **kw):
    from kappai_b200 import Engine, EngineArgs
    args = dict(model=model_dir, dtype=dtype, max_batch=4, max_step_tokens=32, page_size=16, kv_tokens=2048)
    args.update(kw)
    return Engine(EngineArgs(**args))


def log_softmax(x):
    x = np.asarray(x, dtype=np.float64)
    x = x - x.max(-1, keepdims=True)
    return x - np.log(np.exp(x).sum(-1, keepdims=True))


def check(said, logits, token, dtype, top):
    lp = log_softmax(logits)
    tol = 2 * tol_for(dtype, logits)
    assert said.token == token and abs(said.logprob - lp[token]) <= tol
    p = np.exp(lp)
    assert abs(said.entropy + (p * lp).sum()) <= tol * (2 + np.log(len(lp)))
    assert (lp > lp[token] + tol).sum() <= said.rank <= (lp > lp[token] - tol).sum()
    assert len(said.top) == top and len({t for t, _ in said.top}) == top
    for t, v in said.top:
        assert abs(v - lp[t]) <= tol
    assert [v for _, v in said.top] == sorted((v for _, v in said.top), reverse=True)
    if top:
        assert lp.max() - said.top[0][1] <= tol


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B"])
def test_scores_of_prompts(name, dtype, model_dirs, plain_models):
    plain = plain_models[name]
    V = plain.cfg["vocab_size"]
    rng = np.random.default_rng(50)
    prompts = [rng.integers(0, V, n).tolist() for n in (1, 40, 2, 7, 90, 33, 1, 5)]
    eng = engine(model_dirs[name], dtype)
    got = eng.score(prompts, top=3)
    assert [len(g) for g in got] == [len(p) - 1 for p in prompts]
    for p, g in zip(prompts, got):
        logits = plain.logits(p)
        for j, said in enumerate(g):
            check(said, logits[j], p[j + 1], dtype, 3)
    eng.runner.cache.check()
    assert eng.runner.cache.slots.n_free == 4
    if dtype == "float32":                        # cut into other portions: the same bits (the engine's 32-bit path)
        eng.SCORE_ROWS = 13
        assert eng.score(prompts, top=3) == got
        assert [[s.logprob for s in g] for g in eng.score(prompts)] == [[s.logprob for s in g] for g in got]


@pytest.mark.parametrize("look_ahead", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sampled_tokens_come_with_theirs(dtype, look_ahead, model_dirs, plain_models):
    """Requests that want alternatives, none, or nothing, together; some sample with a penalty, which has no part in what is said."""
    from kappai_b200 import SamplingParams
    plain = plain_models["B"]
    rng = np.random.default_rng(51)
    prompts = [rng.integers(0, plain.cfg["vocab_size"], n).tolist() for n in (9, 30, 3, 17)]
    params = [SamplingParams(temperature=0.0, n_predict=12, logprobs=5), SamplingParams(temperature=0.9, seed=3, n_predict=9), SamplingParams(temperature=0.9, seed=4, n_predict=14, logprobs=0),
              SamplingParams(temperature=0.7, seed=5, n_predict=10, logprobs=32, repeat_penalty=1.3)]
    eng = engine(model_dirs["B"], dtype, look_ahead=look_ahead)
    ids = [eng.add_request(p, sp) for p, sp in zip(prompts, params)]
    while eng.has_work():
        eng.step()
    same = engine(model_dirs["B"], dtype, look_ahead=look_ahead)
    from dataclasses import replace
    assert [eng.requests[i].output for i in ids] == same.generate(prompts, [replace(sp, logprobs=None) for sp in params])      # asking changes no token
    for i, p, sp in zip(ids, prompts, params):
        r = eng.requests[i]
        assert len(r.logprobs) == (0 if sp.logprobs is None else len(r.output))
        logits = plain.logits(p + r.output)
        for j, said in enumerate(r.logprobs):
            check(said, logits[len(p) + j - 1], r.output[j], dtype, sp.logprobs)


def test_preempted_requests_say_each_token_once(model_dirs):
    from kappai_b200 import SamplingParams
    rng = np.random.default_rng(52)
    prompts = [rng.integers(0, 256, n).tolist() for n in (30, 40, 20, 50)]
    sp = SamplingParams(temperature=0.0, n_predict=40, logprobs=2)
    want = engine(model_dirs["B"], "float32")
    a = [want.add_request(p, sp) for p in prompts]
    while want.has_work():
        want.step()
    tight = engine(model_dirs["B"], "float32", kv_tokens=16 * 14)
    b = [tight.add_request(p, sp) for p in prompts]
    while tight.has_work():
        tight.step()
    assert tight.scheduler.n_preemptions > 0
    assert [tight.requests[i].logprobs for i in b] == [want.requests[i].logprobs for i in a]


def test_refusals(model_dirs):
    from kappai_b200 import SamplingParams
    from kappai_b200.engine.runner import EngineError
    eng = engine(model_dirs["A"])
    for bad in (-1, 33):
        with pytest.raises(ValueError):
            eng.add_request([1], SamplingParams(logprobs=bad))
        with pytest.raises(ValueError):
            eng.score([[1, 2]], top=bad)
    for p in ([], [10 ** 9], [-1], [0] * (eng.runner.max_model_len + 1)):
        with pytest.raises(ValueError):
            eng.score([p])
    small = engine(model_dirs["B"], kv_tokens=32)
    with pytest.raises(EngineError):
        small.score([[1] * 60])
    assert small.runner.cache.slots.n_free == 4 and all(p.n_free == p.n_pages for p in small.runner.cache.pools.values())
    assert len(small.score([[1, 2, 3]])[0]) == 2
    eng.add_request([1, 2], SamplingParams(temperature=0.0, n_predict=3))
    with pytest.raises(EngineError, match="under way"):
        eng.score([[1, 2]])
    while eng.has_work():
        eng.step()
    assert eng.score([]) == [] and eng.score([[1]]) == [[]]


def test_command_line(model_dirs):
    def run(*flags):
        return subprocess.run([sys.executable, "-m", "kappai_b200.cli", "-m", model_dirs["B"], "--fp32", "-p", "5 17 3", *flags], cwd=ROOT, capture_output=True, text=True, timeout=300)

    a = run("-t", "0", "-n", "4", "--logprobs", "2")
    assert a.returncode == 0, a.stderr
    tokens = [int(t) for t in a.stdout.split()]
    said = [line for line in a.stderr.splitlines() if line.startswith("[logprobs] request 0 token ")]
    assert [int(line.split()[4]) for line in said] == tokens and all(" rank 0 " in line and line.count("]=") == 2 for line in said)
    b = run("--score")
    assert b.returncode == 0, b.stderr
    want = engine(model_dirs["B"]).score([[5, 17, 3]])[0]
    assert b.stdout.split() == [f"{s.logprob:.6f}" for s in want]
