"""What the tests of scoring, forks and beams share: every architecture's small model, and the same computed by the plain Gemma 2."""
import math

import torch

import bolonex_cases
import fovosun_cases
import helpers
import lurisun_cases
import nukelix_cases
import petanex_cases
import pimodra_cases
import plain_gemma2
from kungfu_b200 import api

# architecture -> (configuration, writer of a model folder): windows, chunks, kept first tokens, latents, recurrent states, convolution tails,
# the token before
ARCHITECTURES = {
    "gemma2": (helpers.TINY_A, lambda f: helpers.write_model(f, helpers.TINY_A, seed=3, dtype=torch.float32, draw="loud")),
    "bolonex": (bolonex_cases.BX_A, lambda f: bolonex_cases.write_model(f, bolonex_cases.BX_A, 3)),
    "petanex": (petanex_cases.PX_A, lambda f: petanex_cases.write_model(f, petanex_cases.PX_A, 3)),
    "pimodra": (pimodra_cases.PM_A, lambda f: pimodra_cases.write_model(f, pimodra_cases.PM_A, 3)),
    "nukelix": (nukelix_cases.NK_A, lambda f: nukelix_cases.write_model(f, nukelix_cases.NK_A, 3)),
    "lurisun": (lurisun_cases.LU_A, lambda f: lurisun_cases.write_model(f, lurisun_cases.LU_A, 3)),
    "fovosun": (fovosun_cases.FO_A, lambda f: fovosun_cases.write_model(f, fovosun_cases.FO_A, 3)),
}


def runner(folder, *, dtype, device, page=4, max_requests=6, max_tokens=512, max_context=64):
    cfg, model = api.load_model(folder, dtype=dtype, device=device)
    return api.make_runner(cfg, model, dtype=dtype, device=device, page_size=page, max_tokens=max_tokens, max_requests=max_requests,
                           max_context=max_context, cuda_graphs=False)


def check_forks(run, vocab, prompt_len):
    """A parent and its forks go on with different tokens; each gives, bit for bit, the logits of a request that was fed the same tokens and
    never forked (every step holds one request, so that nothing but the pages differs)."""
    from kungfu_b200.engine.step import StepEntry
    prompt = helpers.random_tokens(prompt_len, vocab, 5 + prompt_len)
    more = {name: helpers.random_tokens(7, vocab, 50 + i) for i, name in enumerate(("a", "b", "c"))}

    def feed(name, tokens):
        return run.step([StepEntry(name, tokens, [len(tokens) - 1])]).clone()

    cache = run.cache
    cache.add_request("a")
    feed("a", prompt)
    cache.fork("a", "b")
    got = {"a": [feed("a", [t]) for t in more["a"][:3]]}       # the parent writes on while the fork waits
    cache.check()
    cache.fork("b", "c")
    got["b"] = [feed("b", [t]) for t in more["b"]]
    got["c"] = [feed("c", [t]) for t in more["c"]]
    got["a"] += [feed("a", [t]) for t in more["a"][3:]]
    cache.check()
    cache.release("a")
    cache.release("c")
    cache.check()
    for name in ("a", "b", "c"):
        cache.add_request("fresh")
        feed("fresh", prompt)
        want = [feed("fresh", [t]) for t in more[name]]
        assert all(torch.equal(x, y) for x, y in zip(got[name], want)), name
        cache.release("fresh")
    cache.release("b")
    cache.check()
    assert cache.n_live == 0 and all(f == g.pool.n_pages for f, g in zip(cache.free_pages(), cache.groups))


def plain_scores(cfg, tensors, prompt):
    """(log probability, entropy, rank, whole log softmax) of every token of the prompt but the first."""
    logp = torch.log_softmax(plain_gemma2.forward(cfg, tensors, prompt).double(), dim=-1)
    out = []
    for i, t in enumerate(prompt[1:]):
        row = logp[i]
        out.append((float(row[t]), float(-(row.exp() * row).sum()), int((row > row[t]).sum()), row))
    return out


def plain_beams(cfg, tensors, prompt, beams, max_tokens, eos=(), length_penalty=0.0):
    """Beam search by whole recomputation, every continuation of every open answer looked at."""
    live, done = [([], 0.0)], []
    value = lambda lp, n: lp / n ** length_penalty  # noqa: E731
    for n in range(1, max_tokens + 1):
        found = []
        for toks, lp in live:
            row = torch.log_softmax(plain_gemma2.forward(cfg, tensors, list(prompt) + toks)[-1].double(), dim=-1)
            found += [(toks + [t], lp + float(row[t])) for t in range(row.numel())]
        found.sort(key=lambda f: -value(f[1], n))
        nxt = []
        for place, (toks, lp) in enumerate(found):
            if toks[-1] in eos:
                if place < beams:
                    done.append((toks, lp, "eos"))
            else:
                nxt.append((toks, lp))
            if len(nxt) == beams:
                break
        if n == max_tokens:
            done += [(t, lp, "length") for t, lp in nxt]
        done = sorted(done, key=lambda d: -value(d[1], len(d[0])))[:beams]
        live = nxt
        if not live or (length_penalty == 0.0 and len(done) == beams and max(lp for _, lp in live) <= done[-1][1]):
            break
    return done


def check_beams(engine, cfg, tensors, tol, **how):
    prompt = helpers.random_tokens(how.pop("prompt_len", 9), cfg["vocab_size"], 4)
    want = plain_beams(cfg, tensors, prompt, how.get("beams", 4), how["max_tokens"], how.get("eos", ()), how.get("length_penalty", 0.0))
    got = engine.beam_search(prompt, **how)
    assert [b.tokens for b in got] == [t for t, _, _ in want]
    assert [b.finish_reason for b in got] == [r for _, _, r in want]
    assert all(math.isclose(b.logprob, lp, abs_tol=tol) for b, (_, lp, _) in zip(got, want))
    assert engine.runner.cache.n_live == 0
    engine.runner.cache.check()
    return got
