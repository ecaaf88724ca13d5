"""Rows of several chunks a block whose length or start is no multiple of 16 bytes: ties across their ends, lists of keys that grow too long,
masks of the lowest number, and tokens whose logit is none."""
import math

import pytest
import torch

from test_gpu_token_logprobs import DEV, _shapes, check, run

pytestmark = pytest.mark.gpu

# one block a row (more rows than multiprocessors; above twice as many, rows of up to four chunks take the form without loads ahead), blocks that
# share a row, sixteen blocks of two chunks
SIZES = [(200, 32003), (160, 45005), (320, 24581), (100, 49157), (1, 256001), (3, 256003)]


def _apart(rows, skip, dtype):
    """The rows in a buffer of which each starts `skip` elements behind a 16-byte boundary, between columns that would win."""
    R, V = rows.shape
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    wide = torch.full((R, -(-(V + skip) // per) * per), 1e30).to(dtype).to(DEV)
    x = wide[:, skip:skip + V]
    x.copy_(rows)
    return x


def _ends(V, skip, dtype):
    """How many columns stand before the first whole 16 bytes of a row, and behind the last."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    head = min(V, -skip % per)
    return head, (V - head) % per


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top,skip", [(1, 0), (1, 3), (3, 1), (64, 0), (64, 7)])
@pytest.mark.parametrize("R,V", SIZES)
def test_ties_between_a_row_and_its_ends(R, V, top, skip, dtype):
    """top - 1 columns of the first chunk lead; the last place goes to the first of equal ones in the head, in any chunk and in the tail."""
    g = torch.Generator().manual_seed(V + top + skip)
    head, tail = _ends(V, skip, dtype)
    rows = torch.zeros(R, V)
    for r in range(R):
        kind = r % 4
        lead = head + torch.randperm(8000, generator=g)[:top - 1]
        if tail:
            rows[r, V - tail:] = 5.0
        if head and kind == 3:
            rows[r, :head] = 5.0
        if kind != 2:                                         # (kind 2: only the tail holds the value)
            rows[r, int(torch.randint(head + 8192, V - tail, (1,), generator=g)) if R > 3 else head + 9000] = 5.0
        rows[r, lead] = 6.0 + 0.5 * (torch.arange(top - 1) % 7)
    tokens = torch.randint(0, V, (R,), generator=g)
    tokens[::2] = V - 1
    check(_apart(rows, skip, dtype), tokens.to(torch.int32).to(DEV), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top,skip", [(1, 0), (20, 5), (64, 3)])
@pytest.mark.parametrize("R,V", SIZES[:4])
def test_values_of_few_kinds(R, V, top, skip, dtype):
    """Random rows of so few values that every place is shared."""
    g = torch.Generator().manual_seed(V + top + skip)
    rows = torch.randint(0, 4, (R, V), generator=g).float()
    rows[:, : V // 2] -= 1.0 * (torch.arange(R)[:, None] % 3)
    top_value = torch.rand(R, V, generator=g) < 20.0 / V      # about twenty of the highest
    rows[top_value] = 4.0
    check(_apart(rows, skip, dtype), torch.randint(0, V, (R,), generator=g).to(torch.int32).to(DEV), top)


def _stairs(V):
    """What makes the list of keys too long in a later chunk of 8,192 columns, once, twice, or while it is still short."""
    inf, i = float("inf"), torch.arange(V)
    yield "equal within a chunk, higher in the next", (i // 8192).float()
    yield "rising within a chunk, higher in the next", i.float() / V * 9 + (i // 8192).float()
    yield "one value behind a masked chunk", torch.where(i < 8200, torch.tensor(-inf), torch.tensor(2.0))
    yield "few behind a masked chunk", torch.where((i < 8200) | (i % 997 != 5), torch.tensor(-inf), (i % 13).float())
    yield "all in the ends", torch.where((i < 3) | (i >= V - 3), (i % 3).float(), torch.tensor(-inf))
    yield "the ends highest", torch.where((i < 3) | (i >= V - 3), torch.tensor(7.0), (i % 50).float() * 0.125)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top,skip", [(1, 3), (20, 0), (64, 5)])
@pytest.mark.parametrize("R,V", SIZES[:4])
def test_shapes_in_rows_of_several_chunks(R, V, top, skip, dtype):
    g = torch.Generator().manual_seed(V + top)
    kinds = [r for _, r in _shapes(V, g)] + [r for _, r in _stairs(V)]
    rows = torch.stack([kinds[r % len(kinds)] for r in range(R)])
    tokens = torch.tensor([(0, V // 2, V - 1, 8192 + 3)[r // len(kinds) % 4] for r in range(R)], dtype=torch.int32)
    check(_apart(rows, skip, dtype), tokens.to(DEV), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", ["lowest", -3e38, -1e38])
@pytest.mark.parametrize("R,V", [(7, 5001), (7, 40000), (1, 256003), (160, 32003), (320, 24581)])
def test_masks_of_the_lowest_number_over_ranges(R, V, low, dtype):
    """A mask of finite numbers whose sum over a thread's columns is none: its range first, last, all but one column, by chunks and by stripes."""
    low = torch.finfo(dtype).min if low == "lowest" else low
    g = torch.Generator().manual_seed(V)
    r, i = 3.0 * torch.randn(V, generator=g), torch.arange(V)
    masks = [i < V // 2, i >= V // 2, i != V // 2, i != V - 1, i < 8192, i // 8192 % 2 == 0, i // 32 % 2 == 0]
    rows = torch.stack([torch.where(masks[n % len(masks)], torch.tensor(low), r) for n in range(max(R, len(masks)))])
    for a in range(0, rows.shape[0], R):                      # (one row at a time where a row is shared by a cluster)
        x = _apart(rows[a:a + R], 0, dtype)
        check(x, torch.full((x.shape[0],), V // 3, dtype=torch.int32, device=DEV), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(6, 37), (6, 5001), (6, 120000), (160, 32003)])
def test_a_token_whose_logit_is_no_number_has_no_rank(R, V, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(R, V, generator=g).to(dtype)
    tokens = torch.randint(0, V, (R,), generator=g)
    x[torch.arange(0, R, 2), tokens[::2]] = float("nan")
    lp, ent, rank, _, _ = run(x.to(DEV), tokens.to(torch.int32).to(DEV), 2)
    assert rank[::2].tolist() == [-1] * len(tokens[::2])
    assert bool(torch.isnan(lp[::2]).all()) and bool(torch.isnan(ent[::2]).all())
    assert int(rank[1::2].min()) >= 0 and math.isfinite(float(lp[1::2].sum()))
