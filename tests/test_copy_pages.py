"""Copies of cache pages, bit for bit, and what they refuse."""
import pytest
import torch

from tokenizer_b200.kernels import ops
from tokenizer_b200.kernels.build import load_library


def plain_copy(pool, page, pairs):
    for source, target, rows in pairs:
        pool[..., target * page:target * page + rows, :, :] = pool[..., source * page:source * page + rows, :, :].clone()
    return pool


def check(pairs, pages, page):
    flat = ops._flat_pairs(pairs)
    return load_library("pages.cu").tokb200_copy_pages_check(
        ops.ctypes.c_void_p(flat.buffer_info()[0]), len(pairs), ops._ll(pages), page)


def test_pairs_that_have_an_order_are_refused_before_a_launch():
    assert check([(0, 1, 4), (0, 2, 0), (7, 3, 1)], 8, 4) == 0
    for pairs in ([(0, 8, 4)], [(8, 0, 4)], [(-1, 0, 4)], [(0, -1, 4)], [(0, 1, 5)], [(0, 1, -1)], [(0, 1, 4), (2, 1, 4)],
                  [(0, 1, 4), (1, 2, 4)], [(3, 3, 4)]):
        assert check(pairs, 8, 4) == -1
        with pytest.raises(ValueError, match="copy_pages"):
            ops._explain_pairs(pairs, 8, 4)
    for pairs in ([(0, 1)], [(0, 1, 2, 3)], [(0, 1), (2, 3, 4, 5)], [(0.0, 1, 2)], [(0, 1 << 31, 2)], [5]):
        with pytest.raises(ValueError, match="copy_pages"):
            ops._flat_pairs(pairs)


def test_a_pool_on_the_host_is_an_error():
    with pytest.raises(ops.KernelError):
        ops.copy_pages(torch.zeros(1, 2, 8, 1, 4), 4, [(0, 1, 4)])


@pytest.mark.gpu
@pytest.mark.parametrize("planes", [(1, 1), (3, 2), (28, 2)])
@pytest.mark.parametrize("heads, d, page", [(1, 1, 1), (2, 64, 16), (4, 128, 16), (1, 3, 5), (3, 5, 7), (2, 48, 21)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
def test_copies(planes, heads, d, page, dtype):
    g = torch.Generator().manual_seed(heads * d + page)
    pages = 30
    pool = torch.randint(0, 255, (*planes, pages * page, heads, d), generator=g).to(dtype).cuda()
    order = torch.randperm(pages, generator=g).tolist()
    pairs = [(order[i % 4], order[4 + i], int(torch.randint(0, page + 1, (1,), generator=g))) for i in range(20)]
    want = plain_copy(pool.clone(), page, pairs)
    ops.copy_pages(pool, page, pairs)
    assert torch.equal(pool, want)


@pytest.mark.gpu
def test_many_pairs_and_none():
    pool = torch.randn(2, 2, 1500 * 2, 1, 8).cuda()
    pairs = [(i % 7, 7 + i, 1 + i % 2) for i in range(1300)]
    want = plain_copy(pool.clone(), 2, pairs)
    ops.copy_pages(pool, 2, [])
    ops.copy_pages(pool, 2, (p for p in pairs))
    assert torch.equal(pool, want)


@pytest.mark.gpu
def test_a_pool_that_begins_inside_an_allocation():
    """A view that is aligned to 2 bytes only."""
    whole = torch.randn(1 + 2 * 8 * 8).to(torch.bfloat16).cuda()
    pool = whole[1:].view(1, 2, 8, 1, 8)
    want = plain_copy(pool.clone(), 4, [(0, 1, 3)])
    ops.copy_pages(pool, 4, [(0, 1, 3)])
    assert torch.equal(pool, want)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A pool of 5 GB, copies at its far end."""
    pool = torch.zeros(5, 1, 1 << 17, 4, 1024, dtype=torch.bfloat16, device="cuda")
    page = 64
    pages = (1 << 17) // page
    pool[:, :, -page:] = torch.randn(5, 1, page, 4, 1024).to(torch.bfloat16).cuda()
    ops.copy_pages(pool, page, [(pages - 1, pages - 2, 63), (pages - 1, 0, 1)])
    far = pool[:, :, -page:]
    assert torch.equal(pool[:, :, -2 * page:-page - 1], far[:, :, :63]) and torch.equal(pool[:, :, :1], far[:, :, :1])
    assert not pool[:, :, -page - 1:-page].any() and not pool[:, :, 1:page].any()


@pytest.mark.gpu
def test_captured():
    pool = torch.randn(2, 2, 64, 2, 64).cuda()
    ops.copy_pages(pool, 16, [])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    pairs = [(0, 2, 9)]
    with torch.cuda.graph(graph):
        ops.copy_pages(pool, 16, pairs)
    pairs[0] = (0, 3, 16)                     # the graph keeps what it was captured with
    pool.normal_()
    want = plain_copy(pool.clone(), 16, [(0, 2, 9)])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool, want)


@pytest.mark.gpu
def test_refusals():
    pool = torch.zeros(1, 2, 32, 2, 8).cuda()
    for bad in ([(0, 4, 8)], [(0, 1, 9)], [(0, 1, 8), (0, 1, 8)], [(0, 1, 8), (1, 2, 8)], [(0, 1)]):
        with pytest.raises(ValueError, match="copy_pages"):
            ops.copy_pages(pool, 8, bad)
    for page in (0, 5):
        with pytest.raises(ValueError, match="copy_pages"):
            ops.copy_pages(pool, page, [(0, 1, 1)])
    with pytest.raises(ValueError, match="contiguous"):
        ops.copy_pages(pool[:, :, :, :1], 8, [(0, 1, 1)])
    assert not pool.any()
