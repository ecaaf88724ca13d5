"""Operators around a step's last product and its cache, with their inputs, their plain forms and the exact answers.

  tokens   log probabilities of given tokens, their ranks, the rows' entropies and the best alternatives, from stored logits
           (what a served reply reports for every token, and what a beam search chooses from)
  head     log probabilities and entropies straight from the rows that enter the output head: product, cap and reduction in
           one, logits never stored (scoring a prompt, perplexity)
  copy     pages of a cache, or rows of per-request states, copied in every store of the cache at once (a forked request's last
           page and states, a context moved as a whole)

Sizes are those of this repository's configurations and benchmark: a vocabulary of 256,000 over a width of 2304 with
logits capped at 30, 26 layers of pages of 64 tokens, the eight-layer models' pages and states, and the tests' small models; the odd
sizes are generic.
"""
from __future__ import annotations

import math

import torch

own = False

_BF16, _F32 = "bfloat16", "float32"


# ---- cases -----------------------------------------------------------------------------------------------------------

def _tokens(rows, vocab, top, dtype, masked):
    return {"op": "tokens", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "masked": masked}


def _head(rows, width, vocab, softcap, dtype):
    return {"op": "head", "rows": rows, "width": width, "vocab": vocab, "softcap": softcap, "dtype": dtype}


def _copy(stores, pages, unit, pairs, dtype):
    return {"op": "copy", "stores": stores, "pages": pages, "unit": unit, "pairs": pairs, "dtype": dtype}


def listed():
    return [
        # one user's decode step that reports five alternatives: nothing but latency
        dict(_tokens(1, 256000, 5, _F32, 0.0), name="reply-1"),
        # a busy server's decode step, twenty alternatives a token
        dict(_tokens(64, 256000, 20, _F32, 0.0), name="reply-64"),
        # a portion of a prompt whose logits the program keeps anyway: ranks and entropies, no alternatives
        dict(_tokens(512, 256000, 0, _F32, 0.0), name="kept-512"),
        # replies under a grammar that forbids a third of an odd vocabulary, 16-bit logits, the most alternatives
        dict(_tokens(301, 32003, 64, _BF16, 0.3), name="grammar-301"),
        # the tests' small model on the 32-bit path
        dict(_head(97, 512, 3000, 30.0, _F32), name="score-small-fp32"),
        # the replies of forty requests, scored without keeping their logits
        dict(_head(40, 2304, 256000, 30.0, _BF16), name="score-40"),
        # an odd number of rows, a width that ends inside a tile, an odd vocabulary, no cap
        dict(_head(701, 1000, 32003, 0.0, _BF16), name="score-odd"),
        # a document scored in one portion: the largest product of the benchmark's model
        dict(_head(2048, 2304, 256000, 30.0, _BF16), name="score-2048"),
        # a fork of one request of the tests' small model: pages of 16 tokens, two layers
        dict(_copy(2, 8, 2 * 2 * 16 * 128, 1, _F32), name="fork-small"),
        # a beam search of eight forks its beams: the last page of each, in 26 layers of 2 x 4 heads x 64 tokens x 256
        dict(_copy(26, 64, 2 * 4 * 64 * 256, 8, _BF16), name="fork-beams"),
        # recurrent states of forked requests: 64 heads of 64 x 128 numbers in 32 bits, six layers, an odd tail
        dict(_copy(6, 16, 64 * 64 * 128 + 3, 7, _F32), name="fork-states"),
        # whole contexts moved, sixteen thousand tokens in eight layers
        dict(_copy(8, 512, 2 * 4 * 64 * 128, 256, _BF16), name="move-long"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tokens", "head", "copy"])
    dtype = rng.choice([_F32, _BF16])
    if op == "tokens":
        vocab = _log_uniform(rng, 1000, 256000)
        rows = _log_uniform(rng, 1, min(2048, 512 * 256000 // vocab))
        return _tokens(rows, vocab, rng.choice([0, rng.randint(1, 64)]), dtype, rng.choice([0.0, 0.0, 0.3, 0.9]))
    if op == "head":
        width, vocab = 8 * _log_uniform(rng, 16, 288), _log_uniform(rng, 1000, 256000)
        most = 2048 if dtype == _BF16 else max(1, min(2048, 20_000_000_000 // (width * vocab)))
        return _head(_log_uniform(rng, 1, most), width, vocab, rng.choice([0.0, 30.0]), dtype)
    stores, unit = _log_uniform(rng, 1, 42), _log_uniform(rng, 500, 131072)
    unit = unit if rng.random() < 0.3 else -(-unit // 64) * 64
    size = 4 if dtype == _F32 else 2
    pairs = _log_uniform(rng, 1, max(1, min(256, 268_000_000 // (stores * unit * size))))
    return _copy(stores, 2 * pairs + rng.randint(0, 9), unit, pairs, dtype)


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _dtype(case):
    return torch.bfloat16 if case["dtype"] == _BF16 else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def whole(high, n):
        return torch.randint(0, high, (n,), generator=g, device="cuda")

    dtype = _dtype(case)
    if case["op"] == "copy":
        n, shape = case["pairs"], (case["pages"], case["unit"])
        order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed))[:2 * n].tolist()
        return {"case": case, "stores": [normal(*shape, dtype=dtype) for _ in range(case["stores"])], "src": order[:n], "dst": order[n:]}
    rows, vocab = case["rows"], case["vocab"]
    tokens = whole(vocab, rows)
    at = torch.arange(rows, device="cuda")
    # a model is sure of some tokens and surprised by others: the given token's logit stands up to six spreads above the rest
    lift = 6.0 * torch.rand(rows, generator=g, device="cuda")
    if case["op"] == "tokens":
        logits = normal(rows, vocab).mul_(2.5)
        logits[at, tokens] += 2.5 * lift
        if case["masked"] > 0.0:
            masked = torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"]
            masked[at, tokens] = False
            logits.masked_fill_(masked, float("-inf"))
            del masked
        return {"case": case, "logits": logits.to(dtype), "tokens": tokens.to(torch.int32)}
    width = case["width"]
    weight = normal(vocab, width).mul_(2.5 / math.sqrt(width)).to(dtype)
    x = normal(rows, width)
    x += weight[tokens].float() * (lift / 2.5)[:, None]
    return {"case": case, "x": x.to(dtype), "weight": weight, "tokens": tokens.to(torch.int32)}


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "copy":
        src, dst = (torch.tensor(state[k], device="cuda") for k in ("src", "dst"))
        return [store.index_copy_(0, dst, store.index_select(0, src)) for store in state["stores"]]
    tokens = state["tokens"].long()[:, None]
    if case["op"] == "head":
        logits = state["x"].float() @ state["weight"].float().T
        if case["softcap"] > 0.0:
            logits = (logits / case["softcap"]).tanh_().mul_(case["softcap"])
        logprob, entropy, _ = _plain(logits, tokens)
        return {"logprob": logprob, "entropy": entropy}
    logits = state["logits"].float()
    logprob, entropy, shift = _plain(logits, tokens)
    given = logits.gather(1, tokens)
    column = torch.arange(case["vocab"], device="cuda")
    rank = ((logits > given) | ((logits == given) & (column < tokens))).sum(1, dtype=torch.int32)
    out = {"logprob": logprob, "entropy": entropy, "rank": rank}
    if case["top"]:
        values, ids = torch.sort(logits, dim=1, descending=True, stable=True)
        out["top_ids"] = ids[:, :case["top"]].to(torch.int32)
        out["top_logprobs"] = values[:, :case["top"]] - shift
    return out


def _plain(logits, tokens):
    """(log probability of the tokens, entropy, log of the sum of exponentials) of every row."""
    largest = logits.amax(1, keepdim=True)
    below = logits - largest
    weight = below.exp()
    total = weight.sum(1, keepdim=True)
    entropy = total.log() - (weight * below.clamp(min=-1e4)).sum(1, keepdim=True) / total
    return (below.gather(1, tokens) - total.log())[:, 0], entropy[:, 0], largest + total.log()


def _run_own(case, state):
    from kungfu_b200 import ops
    if case["op"] == "copy":
        ops.copy_pages(state["stores"], state["src"], state["dst"])
        return state["stores"]
    rows = case["rows"]
    logprob = torch.empty(rows, device="cuda")
    out = {"logprob": logprob, "entropy": torch.empty_like(logprob)}
    if case["op"] == "head":
        ops.head_logprobs(state["x"], state["weight"], state["tokens"], logprob, out_entropy=out["entropy"], softcap=case["softcap"])
        return out
    out["rank"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    if case["top"]:
        out["top_ids"] = torch.empty(rows, case["top"], dtype=torch.int32, device="cuda")
        out["top_logprobs"] = torch.empty(rows, case["top"], device="cuda")
    ops.token_logprobs(state["logits"], state["tokens"], logprob, out_entropy=out["entropy"], out_rank=out["rank"],
                       out_top_ids=out.get("top_ids"), out_top_logprobs=out.get("top_logprobs"))
    return out


# ---- what a pass cannot do without, and the exact answer ----------------------------------------------------------------------

def work(case):
    size = 2 if case["dtype"] == _BF16 else 4
    if case["op"] == "copy":
        return {"bytes": 2 * case["stores"] * case["pairs"] * case["unit"] * size, "flops": 0}
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "tokens":                              # per logit: maximum, scaling, exponential, two sums, rank
        return {"bytes": rows * (vocab * size + 16 + 8 * case["top"]), "flops": 8 * rows * vocab}
    return {"bytes": (rows + vocab) * case["width"] * size + 12 * rows, "flops": 2 * rows * vocab * case["width"]}


def exact(case, seed):
    """In 64 bits, the vocabulary in pieces: Z = sum exp(x - c), S = sum x exp(x - c) with c the largest logit."""
    if case["op"] == "copy":
        return None                                         # nothing is computed
    state = prepare(case, seed)
    rows, vocab, tokens = case["rows"], case["vocab"], state["tokens"].to(torch.int64)
    step = max(1, min(vocab, 64_000_000 // rows, 16384 if case["op"] == "head" else vocab))
    x64 = state["x"].to(torch.float64) if case["op"] == "head" else None

    def piece(a):
        if x64 is None:
            return state["logits"][:, a:a + step].to(torch.float64)
        raw = torch.einsum("rk,vk->rv", x64, state["weight"][a:a + step].to(torch.float64))
        cap = case["softcap"]
        return cap * torch.tanh(raw / cap) if cap > 0.0 else raw

    c = torch.full((rows,), -math.inf, dtype=torch.float64, device="cuda")
    z, s, given = torch.zeros_like(c), torch.zeros_like(c), torch.zeros_like(c)
    best = None
    for a in range(0, vocab, step):
        v = piece(a)
        new = torch.maximum(c, v.max(dim=1).values)
        old = torch.where(torch.isinf(c), torch.zeros_like(c), torch.exp(c - new))
        e = torch.exp(v - new[:, None])
        z = z * old + e.sum(dim=1)
        s = s * old + torch.where(e > 0, v * e, torch.zeros_like(e)).sum(dim=1)
        c = new
        here = (tokens >= a) & (tokens < a + v.shape[1])
        given = torch.where(here, v[torch.arange(rows, device="cuda"), (tokens - a).clamp(0, v.shape[1] - 1)], given)
        if case.get("top"):
            v = torch.topk(v, min(case["top"], v.shape[1]), dim=1).values
            best = v if best is None else torch.topk(torch.cat([best, v], 1), min(case["top"], best.shape[1] + v.shape[1]), dim=1).values
    lse = c + torch.log(z)
    out = {"logprob": given - lse, "entropy": lse - s / z}
    if case["op"] == "tokens":
        out["rank"] = None
        if case["top"]:
            out["top_ids"], out["top_logprobs"] = None, best - lse[:, None]
    return out
