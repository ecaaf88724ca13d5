"""Pages copied in every store of a cache at once: the bytes of the destinations, and of everything else."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(stores, src, dst):
    from kungfu_b200 import ops
    want = [t.clone() for t in stores]
    for t in want:
        if src:
            t[dst] = t[src]
    ops.copy_pages(stores, src, dst)
    torch.cuda.synchronize()
    for a, b in zip(stores, want):
        bits = {torch.bfloat16: torch.int16, torch.float32: torch.int32}.get(a.dtype, a.dtype)
        assert torch.equal(a.view(bits), b.view(bits))


def _store(g, n, shape, dtype):
    return torch.randint(-30000, 30000, (n, *shape), generator=g).to(dtype).to(DEV)


# pages whose bytes are a multiple of 16, of 4, of 2 and odd, of one element and of many, above and below a block's share
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int32, torch.uint8])
@pytest.mark.parametrize("shape", [(1,), (3,), (7, 5), (2, 2, 16, 128), (1001,), (4097,), (2, 4, 64, 256), (16384 * 3 + 1,)])
def test_pages_of_any_size(shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    stores = [_store(g, 9, shape, dtype) for _ in range(3)]
    check(stores, [2], [7])
    check(stores, [0, 8, 3], [1, 4, 6])


def test_stores_of_several_sizes_and_types_in_one_call():
    g = torch.Generator().manual_seed(2)
    stores = [_store(g, 12, (2, 2, 16, 128), torch.bfloat16), _store(g, 12, (5,), torch.float32), _store(g, 40, (1,), torch.int32),
              _store(g, 12, (3, 7), torch.uint8), torch.empty(12, 0, device=DEV)]
    check(stores, [11, 0], [3, 5])


def test_one_source_for_many_and_more_pairs_and_stores_than_one_launch_takes():
    g = torch.Generator().manual_seed(3)
    check([_store(g, 700, (24,), torch.float32)], [5] * 600, [i for i in range(700) if i != 5][:600])
    order = torch.randperm(1300, generator=g).tolist()
    check([_store(g, 1300, (8,), torch.float32)], order[:650], order[650:])
    check([_store(g, 4, (6 + i,), torch.bfloat16) for i in range(150)], [0, 1], [3, 2])


def test_a_base_that_is_not_aligned():
    g = torch.Generator().manual_seed(4)
    flat = torch.randint(0, 255, (4001,), generator=g).to(torch.uint8).to(DEV)
    for off, n in ((1, 32), (2, 32), (4, 48), (8, 16)):
        before = flat.clone()
        check([flat[off:off + 10 * n].view(10, n)], [0, 9], [4, 5])
        assert torch.equal(flat[:off], before[:off]) and torch.equal(flat[off + 10 * n:], before[off + 10 * n:])


def test_every_phase_of_sixteen_bytes():
    """Sources and copies at every pair of phases, of pages with and without a whole vector between their ends; the bytes around them stay."""
    g = torch.Generator().manual_seed(9)
    flat = torch.randint(0, 255, (16 + 33 * 40000,), generator=g).to(torch.uint8).to(DEV)
    for n in (1, 2, 15, 16, 17, 30, 31, 33, 47, 48, 49, 63, 65, 95, 16384 + 16 + 1, 16384 + 47):
        for off in (0, 1, 2, 4, 7, 8, 12, 15):
            before = flat.clone()
            check([flat[off:off + 33 * n].view(33, n)], list(range(16)), list(range(16, 32)))
            assert torch.equal(flat[:off], before[:off]) and torch.equal(flat[off + 33 * n:], before[off + 33 * n:])
    for dtype, size in ((torch.bfloat16, 2), (torch.float32, 4)):
        for n in (1, 3, 9, 13, 8197, 8191):
            check([_store(g, 33, (n,), dtype), flat[:33 * n * size + size].view(dtype)[1:1 + 33 * n].view(33, n)], list(range(16)), list(range(16, 32)))


def test_nothing_to_copy():
    from kungfu_b200 import ops
    t = torch.ones(3, 4, device=DEV)
    ops.copy_pages([t], [], [])
    ops.copy_pages([], [0], [1])
    assert float(t.sum()) == 12.0


def test_offsets_beyond_32_bits():
    from kungfu_b200 import ops
    t = torch.zeros(5, 1 << 30, dtype=torch.uint8, device=DEV)
    t[4, -5:] = 9
    ops.copy_pages([t], [4], [3])
    assert t[3, -6:].tolist() == [0, 9, 9, 9, 9, 9] and int(t[2].max()) == 0


def test_streams_and_graphs():
    from kungfu_b200 import ops
    g = torch.Generator().manual_seed(6)
    a, b = _store(g, 8, (4096,), torch.float32), _store(g, 8, (4096,), torch.float32)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for t, st in zip((a, b), streams):
        with torch.cuda.stream(st):
            ops.copy_pages([t], [1, 2], [5, 6])
            ops.copy_pages([t], [5], [7])                     # a page copied on from the copy just made
    torch.cuda.synchronize()
    for t in (a, b):
        assert torch.equal(t[7], t[1]) and torch.equal(t[6], t[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages([a], [0], [3])
    a[0] = 4.0
    graph.replay()
    torch.cuda.synchronize()
    assert float(a[3].min()) == float(a[3].max()) == 4.0
