"""Log probabilities, ranks, entropies and alternatives of stored logits, against the same formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 2.0 ** -24


def plain(x, tokens, top):
    """(logprob, entropy, rank, ids, logprobs of the alternatives) of rows in 64 bits; tokens inside the row."""
    x = x.double().cpu()
    t = tokens.long().cpu()[:, None]
    m = x.max(1, keepdim=True).values
    d = torch.where(torch.isinf(m), torch.where(torch.isinf(x), -math.inf, x), x - m)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    log_s = torch.where(torch.isinf(m), 0.0, torch.log(s))   # kept apart from m: beside m = -3e38 it would be lost even in 64 bits
    given = x.gather(1, t)
    entropy = torch.where(s > 0, torch.log(s) - torch.where(e > 0, d * e, 0.0).sum(1, keepdim=True) / s, 0.0)
    rank = ((x > given) | ((x == given) & (torch.arange(x.shape[1]) < t))).sum(1)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return (d.gather(1, t) - log_s)[:, 0], entropy[:, 0], rank, ids, d.gather(1, ids) - log_s


def run(logits, tokens, top, fill=7):
    from kungfu_b200 import ops
    R = logits.shape[0]
    out = [torch.full((R,), float(fill), device=DEV), torch.full((R,), float(fill), device=DEV),
           torch.full((R,), fill, dtype=torch.int32, device=DEV)]
    ids = torch.full((R, top), fill, dtype=torch.int32, device=DEV) if top else None
    lps = torch.full((R, top), float(fill), device=DEV) if top else None
    ops.token_logprobs(logits, tokens, out[0], out_entropy=out[1], out_rank=out[2], out_top_ids=ids, out_top_logprobs=lps)
    return out + [ids, lps]


def bound(x, V):
    """How far log s may be off: every term's exponential (its argument rounded once or twice, then within 2^-22), summed in chains
    whose length together stays under V / 1024 additions and under 64 more in trees: (V / 1024 + 96) units; a term's argument counts
    with its own size, and the weighted mean of |d| is at most log V <= 13, two roundings each: 26 more."""
    return (V / 1024 + 96 + 26) * UNIT


def check(logits, tokens, top):
    got = run(logits, tokens, top)
    V = logits.shape[1]
    want = plain(logits, tokens, top)
    tol = bound(logits, V)
    for g, w, scale in ((got[0], want[0], 1.0), (got[1], want[1], 1.0), (got[4], want[4], 1.0) if top else (got[0], want[0], 1.0)):
        g = g.double().cpu()
        finite = torch.isfinite(w)
        assert torch.equal(torch.isfinite(g), finite) and torch.equal(g[~finite], w[~finite])
        # besides log s: the difference to the maximum and the two subtractions, each rounded; the entropy's quotient (as far off as s)
        slack = tol * (1.0 + w[finite].abs()) + 4 * UNIT * w[finite].abs()
        assert bool(((g[finite] - w[finite]).abs() <= slack).all()), float(((g[finite] - w[finite]).abs() / slack).max())
    assert torch.equal(got[2].cpu().long(), want[2])
    if top:
        assert torch.equal(got[3].cpu().long(), want[3])


SIZES = [(1, 1), (2, 2), (3, 31), (4, 64), (2, 257), (5, 1000), (3, 4099), (2, 8191), (2, 8192), (2, 8193), (2, 16385), (7, 32003), (1, 65536),
         (3, 131071), (2, 256000), (700, 300), (1300, 77)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("R,V", SIZES)
def test_rows_of_any_length(R, V, top, dtype):
    g = torch.Generator().manual_seed(R * 7 + V + top)
    x = (3.0 * torch.randn(R, V, generator=g)).to(dtype).to(DEV)
    tokens = torch.randint(0, V, (R,), generator=g).to(torch.int32).to(DEV)
    tokens[0] = 0
    tokens[-1] = V - 1
    check(x, tokens, min(top, V))


def _shapes(V, g):
    """Rows of one kind each: what a mask, a tie or a sure model can make of a row."""
    r = 3.0 * torch.randn(V, generator=g)
    inf = float("inf")
    yield "equal", torch.full((V,), 2.5)
    yield "zeros of both signs", torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    yield "rising", torch.arange(V).float() / V * 20
    yield "falling", -torch.arange(V).float() / V * 20
    yield "steps", (torch.arange(V) // 3).float() / V * 30
    yield "saw", (torch.arange(V) * 37 % 101).float() * 0.25
    yield "masked but one", torch.where(torch.arange(V) == V // 2, 1.0, -inf)
    yield "masked but three", torch.where(torch.arange(V) % (V // 3 + 1) == 0, r, torch.tensor(-inf))
    yield "masked first half", torch.where(torch.arange(V) < V // 2, torch.tensor(-inf), r)
    yield "masked last half", torch.where(torch.arange(V) >= V // 2, torch.tensor(-inf), r)
    yield "all masked", torch.full((V,), -inf)
    yield "lowest value", torch.where(torch.arange(V) % 2 == 0, r, torch.tensor(torch.finfo(torch.bfloat16).min))
    yield "only the lowest value", torch.full((V,), torch.finfo(torch.bfloat16).min)
    yield "huge", r * 1e4
    yield "sure", torch.where(torch.arange(V) == V - 1, 60.0, r)
    yield "far below zero", r - 3e4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [67, 5001, 40000])
@pytest.mark.parametrize("top", [0, 3, 64])
def test_masks_ties_and_extremes(V, top, dtype):
    g = torch.Generator().manual_seed(V + top)
    rows = [r for _, r in _shapes(V, g)]
    x = torch.stack(rows).to(dtype).to(DEV)
    for at in (0, V // 2, V - 1):
        check(x, torch.full((len(rows),), at, dtype=torch.int32, device=DEV), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,skip", [(1, 0), (3, 1), (5, 3), (8, 0), (120, 7)])
def test_rows_that_lie_apart(pad, skip, dtype):
    g = torch.Generator().manual_seed(pad)
    wide = torch.full((9, 1003 + pad), 1e30).to(dtype).to(DEV)
    x = wide[:, skip:skip + 1003]
    x.copy_(torch.randn(9, 1003, generator=g))
    check(x, torch.randint(0, 1003, (9,), generator=g).to(torch.int32).to(DEV), 11)
    one = x[4:5].expand(6, 1003)                              # one row read six times
    check(one, torch.arange(6, dtype=torch.int32, device=DEV) * 200, 4)


def test_padding_rows_stay_as_they_are_and_strange_tokens_are_told():
    V, top = 5000, 6
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, V, generator=g).to(DEV)
    tokens = torch.tensor([4, -1, V, 2 ** 31 - 1, -(2 ** 31), 17], dtype=torch.int32, device=DEV)
    lp, ent, rank, ids, lps = run(x, tokens, top)
    inside = torch.tensor([4, 0, 0, 0, 0, 17], dtype=torch.int32)
    want = plain(x, inside, top)
    for r in (1, 4):
        assert float(lp[r]) == float(ent[r]) == float(rank[r]) == 7.0 and bool((ids[r] == 7).all()) and bool((lps[r] == 7).all())
    for r in (2, 3):
        assert math.isnan(float(lp[r])) and int(rank[r]) == -1
    for r in (0, 2, 3, 5):
        assert torch.equal(ids[r].cpu().long(), want[3][r])
        assert abs(float(ent[r]) - float(want[1][r])) < bound(x, V) * (1 + float(want[1][r]))
    for r in (0, 5):
        assert int(rank[r]) == int(want[2][r])


def test_padding_rows_of_clusters():
    """Few long rows are shared by clusters of blocks: a row of padding between others, and one alone."""
    V, top = 120000, 9
    x = torch.randn(5, V, generator=torch.Generator().manual_seed(6)).to(DEV)
    tokens = torch.tensor([3, -1, V - 1, -5, V + 2], dtype=torch.int32, device=DEV)
    lp, ent, rank, ids, lps = run(x, tokens, top)
    want = plain(x, tokens.clamp(0, V - 1), top)
    for r in (1, 3):
        assert float(lp[r]) == float(ent[r]) == float(rank[r]) == 7.0 and bool((ids[r] == 7).all()) and bool((lps[r] == 7).all())
    for r in (0, 2):
        assert abs(float(lp[r]) - float(want[0][r])) < 14 * bound(x, V) and int(rank[r]) == int(want[2][r])
    assert math.isnan(float(lp[4])) and int(rank[4]) == -1
    for r in (0, 2, 4):
        assert torch.equal(ids[r].cpu().long(), want[3][r]) and abs(float(ent[r]) - float(want[1][r])) < 14 * bound(x, V)
    one = run(x[1:2], tokens[1:2], top)
    assert float(one[0][0]) == 7.0 and bool((one[3] == 7).all())


def test_rows_that_are_no_numbers():
    V = 9000
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, V, generator=g)
    x[0, 8500] = float("nan")
    x[1, 3] = float("inf")
    x[2, :] = float("nan")
    lp, ent, rank, ids, lps = run(x.to(DEV), torch.tensor([1, 1, 1, 1], dtype=torch.int32, device=DEV), 5)
    assert bool(torch.isnan(lp[:3]).all()) and bool(torch.isnan(ent[:3]).all()) and bool(torch.isnan(lps[:3]).all())
    assert math.isfinite(float(lp[3])) and math.isfinite(float(ent[3]))
    assert int(ids[1, 0]) == 3 and 8500 not in ids[0].tolist()
    assert ids[2].tolist() == [0, 1, 2, 3, 4]
    few = torch.full((1, V), float("-inf"))                   # NaN comes behind -inf
    few[0, :3] = float("nan")
    few[0, V - 1] = 1.0
    ids = run(few.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV), 4)[3]
    assert ids[0].tolist() == [V - 1, 3, 4, 5]


def test_alternatives_alone_and_no_rows():
    from kungfu_b200 import ops
    x = torch.randn(3, 700, generator=torch.Generator().manual_seed(1)).to(DEV)
    ids = torch.empty(3, 4, dtype=torch.int32, device=DEV)
    ops.token_logprobs(x, None, None, out_top_ids=ids)
    assert torch.equal(ids.cpu().long(), torch.sort(x.cpu(), dim=1, descending=True, stable=True).indices[:, :4])
    ops.token_logprobs(x[:0], torch.empty(0, dtype=torch.int32, device=DEV), torch.empty(0, device=DEV))


def test_offsets_beyond_32_bits():
    V, R = 262144, 9000                                       # 2.36e9 elements of bfloat16: the last rows start past 2^32 bytes and 2^31 elements
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    x[R - 1, 5] = 3.0
    x[8190, V - 1] = 2.0
    tokens = torch.full((R,), -1, dtype=torch.int32, device=DEV)
    tokens[R - 1], tokens[8190] = 5, V - 1
    lp, _, rank, ids, _ = run(x, tokens, 2)
    for r, v, first in ((R - 1, 3.0, 5), (8190, 2.0, V - 1)):
        assert abs(float(lp[r]) - (v - math.log(V - 1 + math.exp(v)))) < bound(x, V) * 14
        assert int(rank[r]) == 0 and ids[r].tolist() == [first, 0]
    assert float(lp[0]) == 7.0


def test_streams_and_graphs():
    """Two streams at a time, and a graph captured once and replayed on new logits, give what one call after another gives."""
    from kungfu_b200 import ops
    V, R, top = 50000, 6, 8
    g = torch.Generator().manual_seed(8)
    xs = [torch.randn(R, V, generator=g).to(DEV) for _ in range(2)]
    tok = torch.randint(0, V, (R,), generator=g).to(torch.int32).to(DEV)
    want = [run(x, tok, top) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(xs[i], tok, top)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    held = xs[0].clone()
    lp, ids = torch.empty(R, device=DEV), torch.empty(R, top, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    ops.token_logprobs(held, tok, lp, out_top_ids=ids)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.token_logprobs(held, tok, lp, out_top_ids=ids)
    for i in (1, 0, 1):
        held.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lp, want[i][0]) and torch.equal(ids, want[i][3])
