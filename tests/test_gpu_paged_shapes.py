"""The paged operators at the ends of their ranges: the largest pages, the largest groups, more heads than a round has blocks,
an append of many rows. Inputs in which every 16 keys show (paged_dense.telling); tolerance: test_gpu_paged.py's (check)."""
import pytest
import torch

from oracle import paged as OP
from paged_dense import values
from test_gpu_paged import back, dev                                    # noqa: F401  (dev: the fixture)
from test_gpu_paged_tiles import both_ways

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [256, 512, 1024])
@pytest.mark.parametrize("d,mx", [(64, False), (128, True), (256, False), (256, True)])
def test_large_pages(dev, page, d, mx):                                    # noqa: F811
    both_ways(dev, 4, 2, d, page, mx, [1, 2, 1], [2300, 1025, 1023], (900,))
    both_ways(dev, 4, 2, d, page, mx, [80, 2], [2300, 1025])


@pytest.mark.parametrize("hq,hkv,d", [(64, 1, 256), (128, 2, 128), (64, 1, 64)])
@pytest.mark.parametrize("mx", [False, True])
def test_large_groups(dev, hq, hkv, d, mx):                                # noqa: F811
    """64 query heads a K / V head: a query fills four blocks of few rows, two of them 128 rows of a chunk's."""
    both_ways(dev, hq, hkv, d, 16, mx, [1, 1], [2100, 30])
    both_ways(dev, hq, hkv, d, 16, mx, [3, 1, 5], [2100, 30, 4])


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hkv", [256, 300, 520])
def test_many_heads(dev, hkv, mx):                                         # noqa: F811
    """As many K / V heads as a round has blocks, and more."""
    both_ways(dev, hkv, hkv, 64, 16, mx, [1, 1], [2100, 30])
    if hkv < 512:
        both_ways(dev, hkv, hkv, 64, 16, mx, [100, 3], [2100, 30], kws=(dict(),))


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_an_append_of_many_rows(dev, kind):                                # noqa: F811
    """70003 rows of two sequences into pages of 1024 tokens through their table, every row and no other slot; read back."""
    from rfill import ops
    from rfill.paged import Pages
    hkv, d, page, rows = 1, 64, 1024, [70000, 3]
    lens = [70000, 2049]
    g = torch.Generator().manual_seed(1)
    n_pages = 75
    table = torch.randperm(n_pages, generator=g)[:72].to(torch.int32)
    table = torch.stack((table, table.roll(-69)))                          # sequence 1: three pages that sequence 0 does not reach
    pages = Pages.empty(n_pages, hkv, page, d, kind, dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)         # noqa: E731
    slots, pos = ops.paged_slots(table.to(dev), i32(lens), i32([0, 70000, 70003]), 70003, pages)
    at = torch.cat((torch.arange(70000), torch.arange(2046, 2049)))
    which = torch.cat((torch.zeros(70000, dtype=torch.long), torch.ones(3, dtype=torch.long)))
    assert torch.equal(pos.cpu(), at)
    want_slots = table[which, at // page].long() * page + at % page
    assert torch.equal(slots.cpu(), want_slots)
    k, v = (torch.randn(70003, hkv, d, generator=g).to(torch.bfloat16) for _ in "kv")
    ops.paged_append(k.to(dev), v.to(dev), slots, pages)
    pools = back(pages, OP.Pools(1, hkv, page, d, kind == "mx4"))
    for pool, x in zip(values(pools), (k, v)):
        if kind == "mx4":
            x = OP.mx4_decode(*OP.mx4_encode(x.float())).float()
        want = torch.zeros(n_pages * page, hkv, d, dtype=torch.float64)
        want[want_slots] = x.double()
        assert torch.equal(pool.transpose(1, 2).reshape(n_pages * page, hkv, d), want)
    for got, pool in zip(ops.paged_read(pages, slots), values(pools)):
        assert torch.equal(got.cpu().double(), pool.transpose(1, 2).reshape(n_pages * page, hkv, d)[want_slots])
