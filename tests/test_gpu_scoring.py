"""Scores, forks and beams together on the device: the log probabilities' kernels and the copies of pages as the engine uses them."""
import json
import os
import subprocess
import sys

import pytest
import torch

import helpers
import plain_gemma2
import scoring_cases as sc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# Of a log probability, the difference of two numbers as exact as logits are: the engine's tests allow a logit of these models 2e-4 (32-bit) and
# 2e-2 (bfloat16) of the largest, which the cap holds below 30.  Both bounds here are below twice that.
TOL = {"float32": 2e-4, "bfloat16": 0.5}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    out = {}
    for name, cfg in (("A", helpers.TINY_A), ("E", helpers.TINY_E)):
        folder = helpers.write_model(str(tmp_path_factory.mktemp("scoring") / name), cfg, seed=4, dtype=torch.bfloat16, draw="loud")
        out[name] = (folder, cfg, helpers.read_tensors(folder))
    return out


def _engine(folder, dtype, **how):
    from kungfu_b200 import Engine
    return Engine(folder, dtype=dtype, device=DEV, **{**dict(ctx=512, batch=64, parallel=8, page_size=16), **how})


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(sc.ARCHITECTURES))
@pytest.mark.parametrize("prompt_len", [1, 4, 23])
def test_forks_of_every_architecture(tmp_path, name, prompt_len, dtype):
    cfg, write = sc.ARCHITECTURES[name]
    run = sc.runner(write(str(tmp_path / "m")), dtype=dtype, device=DEV)
    sc.check_forks(run, cfg.get("vocab_size", cfg.get("vocab")), prompt_len)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,lengths", [("A", [2, 17, 40, 63, 1]), ("E", [300, 70, 513, 2, 129])])
@pytest.mark.parametrize("top", [0, 5])
def test_scores_of_prompts(models, name, lengths, top, dtype):
    folder, cfg, tensors = models[name]
    eng = _engine(folder, dtype, ctx=1024, batch=200, page_size=64 if name == "E" else 8)
    prompts = [helpers.random_tokens(n, cfg["vocab_size"], 7 + n) for n in lengths]
    got = eng.score(prompts, top=top)
    for p, scores in zip(prompts, got):
        assert len(scores) == len(p) - 1
        want = sc.plain_scores(cfg, tensors, p) if len(p) > 1 else []
        for s, t, (lp, ent, _rank, row) in zip(scores, p[1:], want):
            assert s.token == t and abs(s.logprob - lp) < TOL[dtype] and abs(s.entropy - ent) < 10 * TOL[dtype]
            if top:
                assert s.rank is not None and len(s.top) == top
                assert all(abs(v - float(row[i])) < TOL[dtype] for i, v in s.top)
                if s.rank < top:                              # the token is among its alternatives, where its rank says
                    assert s.top[s.rank] == (t, s.logprob)
    assert eng.runner.cache.n_live == 0
    # the fused head and the stored logits say the same: on the 32-bit path they are one and the same kernel
    other = eng.score(prompts, top=0 if top else 5)
    gap = max(abs(a.logprob - b.logprob) for g, o in zip(got, other) for a, b in zip(g, o))
    assert gap < 1e-4, gap


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False])
def test_scores_of_produced_tokens(models, dtype, graphs):
    """Greedy and drawn tokens of several requests in padded, replayed steps; prompts and decode rows in one step."""
    from kungfu_b200.sampling import Sampling
    folder, cfg, tensors = models["E"]
    eng = _engine(folder, dtype, cuda_graphs=graphs, page_size=64)
    prompts = [helpers.random_tokens(n, cfg["vocab_size"], 30 + n) for n in (5, 170, 33, 90, 12)]
    rules = [Sampling(temperature=t) for t in (0.0, 0.9, 0.0, 1.2, 0.0)]
    wants = (3, 0, 64, None, 1)
    ids = []
    for p, r, k in zip(prompts, rules, wants):
        ids.append(eng.add_request(p, r, max_tokens=14, ignore_eos=True, logprobs=k))
        eng.step()
        eng.step()
    while not eng.idle:
        eng.step()
    for i, p, k in zip(ids, prompts, wants):
        r = eng.requests[i]
        assert len(r.output) == 14 and len(r.scores) == (0 if k is None else 14)
        want = sc.plain_scores(cfg, tensors, p + r.output)[len(p) - 1:]
        for s, t, (lp, _ent, _rank, _row) in zip(r.scores, r.output, want):
            assert s.token == t and abs(s.logprob - lp) < TOL[dtype] and len(s.top) == k
            if r.sampling.temperature == 0.0:
                assert s.rank == 0 and (k == 0 or s.top[0] == (t, s.logprob))
    # the same tokens as without scores
    plain = _engine(folder, dtype, cuda_graphs=graphs, page_size=64)
    again = []
    for p, r in zip(prompts, rules):
        again.append(plain.add_request(p, r, max_tokens=14, ignore_eos=True))
        plain.step()
        plain.step()
    while not plain.idle:
        plain.step()
    assert [plain.requests[i].output for i in again] == [eng.requests[i].output for i in ids]


@pytest.mark.parametrize("graphs", [True, False])
def test_a_forked_request_goes_on_by_itself(models, graphs):
    from kungfu_b200.sampling import Sampling
    folder, cfg, tensors = models["A"]
    prompt = helpers.random_tokens(9, 512, 2)
    want = plain_gemma2.greedy(cfg, tensors, prompt, 20)
    eng = _engine(folder, "float32", ctx=64, cuda_graphs=graphs, page_size=4)
    a = eng.add_request(prompt, Sampling(temperature=0.0), max_tokens=20, ignore_eos=True)
    while len(eng.requests[a].output) < 5:
        eng.step()
    b = eng.fork(a, logprobs=2)
    c = eng.fork(b, sampling=Sampling(temperature=1.5, top_k=0, top_p=1.0), seed=9)
    while not eng.idle:
        eng.step()
    assert eng.requests[a].output == want and eng.requests[b].output == want
    assert eng.requests[c].output[:4] == want[:4] and len(eng.requests[c].output) == 20
    eng.runner.cache.check()
    assert eng.runner.cache.n_live == 0


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("how", [dict(beams=4, max_tokens=9), dict(beams=3, max_tokens=8, length_penalty=0.8),
                                 dict(beams=5, max_tokens=6, eos=tuple(range(0, 512, 5)))])
def test_beams(models, how, graphs):
    """Everything together: alternatives of every open answer, forks, copies, pages that come back, replayed decode steps."""
    folder, cfg, tensors = models["A"]
    eng = _engine(folder, "float32", ctx=64, cuda_graphs=graphs, page_size=4)
    got = sc.check_beams(eng, cfg, tensors, 8 * TOL["float32"], **how)
    scores = eng.score([helpers.random_tokens(9, 512, 4) + b.tokens for b in got])      # the search's sums are the answers' scores
    for b, s in zip(got, scores):
        assert abs(sum(t.logprob for t in s[8:]) - b.logprob) < 9 * TOL["float32"]


def test_beams_of_the_tensor_core_path(models):
    """bfloat16: the same search twice gives the same answers, and their sums are what the fused head scores."""
    folder, cfg, _ = models["E"]
    eng = _engine(folder, "bfloat16", ctx=1024, batch=512, page_size=64)
    prompt = helpers.random_tokens(150, cfg["vocab_size"], 4)
    got = eng.beam_search(prompt, beams=6, max_tokens=12, ignore_eos=True)
    again = eng.beam_search(prompt, beams=6, max_tokens=12, ignore_eos=True)
    assert [(b.tokens, b.logprob) for b in got] == [(b.tokens, b.logprob) for b in again]
    assert all(a.logprob >= b.logprob for a, b in zip(got, got[1:])) and len({tuple(b.tokens) for b in got}) == 6
    for b, s in zip(got, eng.score([prompt + b.tokens for b in got])):
        assert abs(sum(t.logprob for t in s[149:]) - b.logprob) < 12 * TOL["bfloat16"]
    eng.runner.cache.check()


def test_programs(models):
    folder, cfg, tensors = models["A"]
    ids = helpers.random_tokens(12, 512, 3)

    def run(*args):
        p = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "kungfu"), *args, "--model", folder, "--ids", json.dumps(ids), "--dtype", "float32",
                            "--ctx", "64"], capture_output=True, text=True, timeout=600)
        assert p.returncode == 0, p.stderr[-2000:]
        return json.loads(p.stdout)

    doc = run("score", "--logprobs", "--topk", "2")
    want = sc.plain_scores(cfg, tensors, ids)
    assert abs(doc["logprob"] - sum(w[0] for w in want)) < 11 * TOL["float32"] and len(doc["scores"]) == 11
    assert all(s["rank"] == w[2] and len(s["top"]) == 2 for s, w in zip(doc["scores"], want))
    doc = run("generate", "--max-tokens", "5", "--ignore-eos", "--logprobs", "1")
    assert doc["generated"] == plain_gemma2.greedy(cfg, tensors, ids, 5) and [s["token"] for s in doc["scores"]] == doc["generated"]
    doc = run("generate", "--max-tokens", "4", "--ignore-eos", "--beams", "3")
    want = sc.plain_beams(cfg, tensors, ids, 3, 4)
    assert [b["generated"] for b in doc["beams"]] == [t for t, _, _ in want]
