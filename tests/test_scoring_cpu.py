"""Forks of requests, scores of tokens and beam search: the host's part, the kernels replaced by the CPU stand-in."""
import random

import pytest
import torch

import helpers
import plain_gemma2
import scoring_cases as sc
from kungfu_b200 import api
from kungfu_b200.cache import CacheError, CacheManager, OutOfPages
from kungfu_b200.engine.engine import Engine
from kungfu_b200.engine.step import StepEntry, StepError
from kungfu_b200.parts import FixedState, PagedKV
from kungfu_b200.sampling import Sampling


def make_cache(n_pages=16, page=4, window=8, max_requests=4, max_context=64):
    needs = [PagedKV(2, 8, window), PagedKV(2, 8, None), PagedKV(1, 16, window), FixedState((3,), torch.float32), FixedState((1,), torch.int32)]
    return CacheManager(needs, page_size=page, n_pages=n_pages, max_requests=max_requests, max_context=max_context,
                        dtype=torch.float32, device="cpu")


# ---- the cache manager ---------------------------------------------------------------------------------------------

def test_a_fork_shares_full_pages_and_copies_the_last_and_the_states(cpu_ops):
    c = make_cache()
    c.add_request("a")
    c.reserve("a", 6)
    c.commit("a", 6)
    for g in range(2):
        for p in c.block_table(g, "a"):
            for s in c.groups[g].slots:
                c.storage[s][p] = float(10 * s + p + 1)
    c.storage[3][c.state_slot("a")] = 7.0
    c.storage[4][c.state_slot("a")] = 5
    c.fork("a", "b")
    c.check()
    assert c.length("b") == 6 and c.state_slot("b") != c.state_slot("a")
    for g in range(2):
        ta, tb = c.block_table(g, "a"), c.block_table(g, "b")
        assert ta[0] == tb[0] and ta[1] != tb[1]
        for s in c.groups[g].slots:
            assert torch.equal(c.storage[s][ta[1]], c.storage[s][tb[1]])
        assert c.free_pages()[g] == 16 - 3
    assert float(c.storage[3][c.state_slot("b")].min()) == 7.0 and int(c.storage[4][c.state_slot("b")]) == 5
    c.release("a")                                            # the shared page stays with the fork
    c.check()
    assert c.free_pages() == [14, 14]
    c.release("b")
    assert c.free_pages() == [16, 16]
    c.check()


def test_a_fork_at_a_page_boundary_copies_no_page(cpu_ops):
    c = make_cache()
    c.add_request("a")
    c.reserve("a", 8)
    c.commit("a", 8)
    c.fork("a", "b")
    assert c.block_table(1, "a") == c.block_table(1, "b") and c.free_pages()[1] == 14
    for r in ("a", "b"):                                      # each goes on in a page of its own
        c.reserve(r, 1)
        c.commit(r, 1)
    assert c.block_table(1, "a")[2] != c.block_table(1, "b")[2]
    c.check()


def test_a_fork_of_an_empty_request(cpu_ops):
    c = make_cache()
    c.add_request("a")
    c.fork("a", "b")
    assert c.length("b") == 0 and c.free_pages() == [16, 16]
    c.check()


def test_windows_let_shared_pages_go_one_by_one(cpu_ops):
    c = make_cache()
    c.add_request("a")
    c.reserve("a", 10)
    c.commit("a", 10)
    c.fork("a", "b")
    free = c.free_pages()[0]
    c.reserve("a", 1)
    c.commit("a", 1)                                          # the parent has passed page 0, the fork has not
    assert c.block_table(0, "a")[0] == -1 and c.block_table(0, "b")[0] >= 0 and c.free_pages()[0] == free
    c.check()
    c.reserve("b", 1)
    c.commit("b", 1)
    assert c.free_pages()[0] == free + 1
    c.check()


def test_forks_that_are_refused_change_nothing(cpu_ops):
    c = make_cache(n_pages=4, max_requests=4)
    c.add_request("a")
    c.reserve("a", 6)
    with pytest.raises(CacheError):
        c.fork("a", "b")                                      # tokens reserved, not committed
    c.commit("a", 6)
    for parent, child in (("x", "b"), ("a", "a")):
        with pytest.raises(CacheError):
            c.fork(parent, child)
    with pytest.raises(CacheError):
        c.fork_all([("a", "b"), ("a", "b")])
    with pytest.raises(CacheError):
        c.fork_all([("a", "b"), ("b", "c")])                  # a child cannot be forked before it is there
    with pytest.raises(OutOfPages):
        c.fork_all([("a", "b"), ("a", "c"), ("a", "d")])      # two pages are free in each group, three wanted
    assert c.n_live == 1 and c.free_pages() == [2, 2]
    c.check()
    c.fork("a", "b")
    with pytest.raises(CacheError):
        c.fork("a", "b")
    c.add_request("c")
    c.add_request("d")
    with pytest.raises(CacheError):
        c.fork("a", "e")                                      # no state slot
    c.check()
    assert c.n_live == 4


def test_a_copy_that_fails_takes_the_forks_back(cpu_ops, monkeypatch):
    from kungfu_b200 import ops
    c = make_cache()
    c.add_request("a")
    c.reserve("a", 3)
    c.commit("a", 3)

    def fails(*_a):
        raise ops.KernelError("no")
    monkeypatch.setattr(ops, "copy_pages", fails)
    with pytest.raises(ops.KernelError):
        c.fork("a", "b")
    assert c.n_live == 1 and c.free_pages() == [15, 15]
    c.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_lives_keep_the_accounts(cpu_ops, seed):
    """Requests are admitted, grow, are forked and released in any order; what each holds is told by a number written with every token."""
    rng = random.Random(seed)
    c = make_cache(n_pages=40, max_requests=6, max_context=60)
    told: dict = {}                                           # request -> the number of each of its tokens
    nth = 0
    for _ in range(300):
        what = rng.random()
        if what < 0.25 and c.n_live < 6:
            c.add_request(nth)
            told[nth] = []
            nth += 1
        elif what < 0.45 and told and c.n_live < 6:
            parent = rng.choice(list(told))
            try:
                c.fork(parent, nth)
                told[nth] = list(told[parent])
                nth += 1
            except OutOfPages:
                pass
        elif what < 0.6 and told:
            r = rng.choice(list(told))
            c.release(r)
            del told[r]
        elif told:
            r, n = rng.choice(list(told)), rng.randint(1, 7)
            try:
                c.reserve(r, n)
            except OutOfPages:
                continue
            for _ in range(n):
                at, value = len(told[r]), rng.random()
                told[r].append(value)
                for g in range(2):
                    page = c.block_table(g, r)[at // 4]
                    for s in c.groups[g].slots:
                        c.storage[s][page, :, :, at % 4] = value
            c.commit(r, n)
        c.check()
        for r, values in told.items():
            table = c.block_table(1, r)                       # the group without a window
            got = [float(c.storage[1][table[i // 4], 0, 0, i % 4, 0]) for i in range(len(values))]
            assert got == pytest.approx(values)
    for r in list(told):
        c.release(r)
    assert c.free_pages() == [40, 40]


@pytest.mark.parametrize("name", list(sc.ARCHITECTURES))
@pytest.mark.parametrize("prompt_len", [1, 4, 23])
def test_forks_of_every_architecture(tmp_path, cpu_ops, name, prompt_len):
    cfg, write = sc.ARCHITECTURES[name]
    run = sc.runner(write(str(tmp_path / "m")), dtype="float32", device="cpu")
    sc.check_forks(run, cfg.get("vocab_size", cfg.get("vocab")), prompt_len)


# ---- the engine ------------------------------------------------------------------------------------------------------

def _engine(folder, cfg_dict, *, page=4, pool_tokens=256, batch=16, parallel=4, pipeline=True):
    cfg, model = api.load_model(folder, dtype="float32", device="cpu")
    runner = api.make_runner(cfg, model, dtype="float32", device="cpu", page_size=page, max_tokens=pool_tokens, max_requests=parallel,
                             max_context=cfg_dict["max_position_embeddings"])
    return Engine(runner=runner, batch=batch, parallel=parallel, pipeline=pipeline)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    cfg = helpers.TINY_A
    folder = helpers.write_model(str(tmp_path_factory.mktemp("scoring") / "m"), cfg, seed=4, dtype=torch.float32, draw="loud")
    return folder, cfg, helpers.read_tensors(folder)


TOL = 2e-4                                                    # of a log probability: what the engine's tests allow a logit


@pytest.mark.parametrize("top", [0, 3])
def test_scores_of_prompts(model, cpu_ops, top):
    folder, cfg, tensors = model
    eng = _engine(folder, cfg, pool_tokens=96)                # fewer pages than all the prompts want at a time
    prompts = [helpers.random_tokens(n, cfg["vocab_size"], 7 + n) for n in (1, 2, 17, 40, 33, 5)] + [[]]
    got = eng.score(prompts, top=top)
    assert [len(g) for g in got] == [max(len(p) - 1, 0) for p in prompts]
    for p, scores in zip(prompts, got):
        want = sc.plain_scores(cfg, tensors, p) if len(p) > 1 else []
        for s, t, (lp, ent, rank, row) in zip(scores, p[1:], want):
            assert s.token == t and abs(s.logprob - lp) < TOL and abs(s.entropy - ent) < 10 * TOL
            assert s.rank == (rank if top else None) and len(s.top) == top
            best = torch.sort(row, descending=True, stable=True).indices[:top].tolist()
            assert [i for i, _ in s.top] == best and all(abs(v - float(row[i])) < TOL for i, v in s.top)
    assert eng.runner.cache.n_live == 0


def test_scores_that_are_refused(model, cpu_ops):
    folder, cfg, _ = model
    eng = _engine(folder, cfg)
    for prompts, how in (([[1, 600]], {}), ([[1] * 65], {}), ([[1, 2]], dict(top=65)), ([[1, 2]], dict(top=-1))):
        with pytest.raises(ValueError):
            eng.score(prompts, **how)
    with pytest.raises(ValueError):
        eng.add_request([1, 2], logprobs=65)
    run = eng.runner
    run.cache.add_request("x")
    for entries, targets in (([StepEntry("x", [1, 2], [0])], [[1, 2]]), ([StepEntry("x", [1], [0])], [[512]]), ([StepEntry("x", [1], [])], [[]])):
        with pytest.raises(StepError):
            run.score(entries, targets)
    assert run.cache.length("x") == 0
    tight = _engine(folder, cfg, pool_tokens=24)              # 6 pages: a prompt of 40 tokens cannot be held
    with pytest.raises(OutOfPages):
        tight.score([helpers.random_tokens(40, 512, 1)])
    assert tight.runner.cache.n_live == 0


@pytest.mark.parametrize("pipeline", [True, False])
def test_scores_of_produced_tokens(model, cpu_ops, pipeline):
    folder, cfg, tensors = model
    eng = _engine(folder, cfg, pipeline=pipeline, pool_tokens=36)       # 9 pages: somebody is preempted and recomputed
    prompts = [helpers.random_tokens(n, 512, 30 + n) for n in (5, 7, 6)]
    ids = [eng.add_request(p, Sampling(temperature=t), max_tokens=9, logprobs=k) for p, t, k in zip(prompts, (0.0, 0.9, 0.0), (2, 0, None))]
    while not eng.idle:
        eng.step()
    assert eng.scheduler.n_preemptions > 0
    for i, p, k in zip(ids, prompts, (2, 0, None)):
        r = eng.requests[i]
        assert len(r.output) == 9
        if k is None:
            assert r.scores == []
            continue
        want = sc.plain_scores(cfg, tensors, p + r.output)[len(p) - 1:]
        assert len(r.scores) == 9
        for s, t, (lp, ent, rank, _row) in zip(r.scores, r.output, want):
            assert s.token == t and abs(s.logprob - lp) < TOL and abs(s.entropy - ent) < 10 * TOL and s.rank == rank and len(s.top) == k


@pytest.mark.parametrize("pipeline", [True, False])
def test_a_forked_request_goes_on_by_itself(model, cpu_ops, pipeline):
    folder, cfg, tensors = model
    prompt = helpers.random_tokens(9, 512, 2)
    want = plain_gemma2.greedy(cfg, tensors, prompt, 10)
    eng = _engine(folder, cfg, pipeline=pipeline)
    a = eng.add_request(prompt, Sampling(temperature=0.0), max_tokens=10, ignore_eos=True, logprobs=0)
    with pytest.raises(ValueError):
        eng.fork(a)                                           # nothing produced yet
    events = []
    while len(eng.requests[a].output) < 4:
        events += eng.step()
    n = len(eng.requests[a].output)
    b = eng.fork(a, max_tokens=8)
    c = eng.fork(a, sampling=Sampling(temperature=1.5, top_k=0, top_p=1.0), seed=9, logprobs=2)
    with pytest.raises(ValueError):
        eng.fork(a, max_tokens=2)
    with pytest.raises(ValueError):
        eng.fork(a, new_id=b)
    while not eng.idle:
        events += eng.step()
    assert eng.requests[a].output == want and eng.requests[b].output == want[:8]
    assert eng.requests[c].output[:4] == want[:4] and len(eng.requests[c].output) == 10
    assert [t for i, t, _ in events if i == a] == want        # no event was lost to the flush inside fork
    assert len(eng.requests[c].scores) == 10 and len(eng.requests[c].scores[-1].top) == 2 and len(eng.requests[b].scores) == 8
    assert n <= 8 and eng.runner.cache.n_live == 0
    eng.runner.cache.check()
    with pytest.raises(ValueError):
        eng.fork(a)                                           # finished


def test_forks_that_outgrow_the_pool_are_preempted_and_recomputed(model, cpu_ops):
    folder, cfg, tensors = model
    prompt = helpers.random_tokens(5, 512, 8)
    want = plain_gemma2.greedy(cfg, tensors, prompt, 12)
    eng = _engine(folder, cfg, pool_tokens=36, batch=16)      # nine pages: four requests of 17 tokens want up to twenty
    a = eng.add_request(prompt, Sampling(temperature=0.0), max_tokens=12, ignore_eos=True, logprobs=0)
    while len(eng.requests[a].output) < 2:
        eng.step()
    ids = [a, eng.fork(a), eng.fork(a), eng.fork(a)]
    while not eng.idle:
        eng.step()
        eng.runner.cache.check()
    assert eng.scheduler.n_preemptions > 0
    for i in ids:
        assert eng.requests[i].output == want and len(eng.requests[i].scores) == 12
    assert eng.runner.cache.free_pages() == [9, 9]


def test_a_cancelled_parent_leaves_its_forks_alone(model, cpu_ops):
    folder, cfg, tensors = model
    prompt = helpers.random_tokens(10, 512, 9)
    want = plain_gemma2.greedy(cfg, tensors, prompt, 8)
    eng = _engine(folder, cfg)
    a = eng.add_request(prompt, Sampling(temperature=0.0), max_tokens=8, ignore_eos=True)
    while len(eng.requests[a].output) < 3:
        eng.step()
    b = eng.fork(a)
    events = eng.cancel(a)
    assert (a, None, "cancelled") in events
    other = eng.add_request(helpers.random_tokens(30, 512, 1), Sampling(temperature=0.0), max_tokens=4, ignore_eos=True)    # takes what came back
    while not eng.idle:
        eng.step()
    assert eng.requests[b].output == want and len(eng.requests[other].output) == 4
    eng.runner.cache.check()


@pytest.mark.parametrize("pipeline", [True, False])
def test_scoring_and_searching_beside_running_requests(model, cpu_ops, pipeline):
    folder, cfg, tensors = model
    prompt, text = helpers.random_tokens(9, 512, 2), helpers.random_tokens(21, 512, 5)
    want = plain_gemma2.greedy(cfg, tensors, prompt, 10)
    eng = _engine(folder, cfg, pipeline=pipeline, parallel=6)
    a = eng.add_request(prompt, Sampling(temperature=0.0), max_tokens=10, ignore_eos=True)
    events = eng.step() + eng.step() + eng.step()
    scores = eng.score([text])[0]
    assert all(abs(s.logprob - w[0]) < TOL for s, w in zip(scores, sc.plain_scores(cfg, tensors, text)))
    events += eng.step() + eng.step()
    found = eng.beam_search(text, beams=4, max_tokens=4, ignore_eos=True)
    assert [b.tokens for b in found] == [t for t, _, _ in sc.plain_beams(cfg, tensors, text, 4, 4)]
    while not eng.idle:
        events += eng.step()
    assert eng.requests[a].output == want and [t for i, t, _ in events if i == a] == want


def test_forks_without_a_slot_are_refused(model, cpu_ops):
    folder, cfg, _ = model
    eng = _engine(folder, cfg, parallel=2)
    a = eng.add_request([1, 2, 3], Sampling(temperature=0.0), max_tokens=12, ignore_eos=True)
    while not eng.requests[a].output:
        eng.step()
    eng.fork(a)
    with pytest.raises(CacheError):
        eng.fork(a)
    assert len(eng.scheduler.running) == 2


@pytest.mark.parametrize("how", [dict(beams=1, max_tokens=6), dict(beams=4, max_tokens=7), dict(beams=3, max_tokens=6, length_penalty=0.8),
                                 dict(beams=5, max_tokens=5, eos=tuple(range(0, 512, 5)))])
def test_beams(model, cpu_ops, how):
    folder, cfg, tensors = model
    sc.check_beams(_engine(folder, cfg, parallel=8), cfg, tensors, 8 * TOL, **how)


def test_beams_reach_the_context_and_are_refused(model, cpu_ops):
    folder, cfg, _ = model
    eng = _engine(folder, cfg, parallel=3)
    got = eng.beam_search(helpers.random_tokens(60, 512, 3), beams=3, max_tokens=30, ignore_eos=True)
    assert len(got) == 3 and all(len(b.tokens) == 4 and b.finish_reason == "context" for b in got)
    for prompt, how in (([], {}), ([512], {}), ([1] * 64, {}), ([1], dict(beams=0)), ([1], dict(beams=33)), ([1], dict(max_tokens=0))):
        with pytest.raises(ValueError):
            eng.beam_search(prompt, **how)
    with pytest.raises(CacheError):
        eng.beam_search([1], beams=4)
    tight = _engine(folder, cfg, parallel=4, pool_tokens=12)   # three pages
    with pytest.raises(OutOfPages):
        tight.beam_search(helpers.random_tokens(7, 512, 1), beams=4, max_tokens=20, ignore_eos=True)
    assert tight.runner.cache.n_live == 0 and tight.runner.cache.free_pages() == [3, 3]
