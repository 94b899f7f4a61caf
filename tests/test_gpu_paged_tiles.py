"""Attention over pages where every 16 keys show in the outputs (paged_dense.telling; test_paged_dense_host.py shows that they
do): windows of table entries, runs and splits of the keys, several rounds of blocks, many sequences, pages that are none beside
the windows' edges. Tolerance: test_gpu_paged.py's (check), and bit for bit the same from run to run."""
import pytest
import torch

from paged_dense import attend as dense, telling
from test_gpu_paged import check, dev, layout, run                         # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


def both_ways(dev, hq, hkv, d, page, mx, rows, lens, holes=(), kws=(dict(), dict(workspace=None))):   # noqa: F811
    """holes: keys of every sequence whose pages are none."""
    table, n_pages = layout(lens, page, d + len(rows))
    for i, key in enumerate(holes):
        for b, n in enumerate(lens):
            if key < n:
                table[b, key // page] = (-1, n_pages, 1 << 30)[i % 3]
    for down in (False, True):
        pools, q = telling(hq, hkv, d, page, mx, rows, lens, table, n_pages, down)
        want, size = dense(pools, table, n_pages, q, rows, lens, hq, 1.0)
        for kw in kws:
            got = run(dev, pools, table, q, rows, lens, hq, 1.0, **kw)
            check(got, want, size, (rows, lens, down, kw))
            assert torch.equal(got, run(dev, pools, table, q, rows, lens, hq, 1.0, **kw)), "run to run"


KINDS = [(64, False), (128, False), (256, False), (64, True), (128, True), (256, True)]


@pytest.mark.parametrize("holes", [(), (1008, 1030), (2040, 2050, 3071)])
@pytest.mark.parametrize("d,mx", KINDS)
def test_chunks_over_windows(dev, d, mx, holes):                           # noqa: F811
    """Chunks of 70 and 33 rows over up to five windows of 1024 keys, unsplit and split, beside a short sequence."""
    both_ways(dev, 4, 2, d, 16, mx, [70, 33, 2], [2600, 4700, 40], holes)


@pytest.mark.parametrize("d,mx", KINDS)
def test_chunks_over_pages_of_several_tiles(dev, d, mx):                   # noqa: F811
    """Pages of 128 tokens: a tile's halves on one page, windows' edges inside the pages' run."""
    both_ways(dev, 4, 1, d, 128, mx, [40], [3000], (2 * 1024 - 1,))


@pytest.mark.parametrize("holes", [(), (4090, 4100)])
@pytest.mark.parametrize("d,mx", KINDS)
def test_few_rows_over_windows(dev, d, mx, holes):                         # noqa: F811
    """Single tokens and a few over more tiles than a wave's window of 32 holds (4096 keys a block), unsplit, and in runs."""
    both_ways(dev, 4, 2, d, 16, mx, [1, 3, 1], [9001, 4700, 77], holes)
    both_ways(dev, 2, 1, d, 64, mx, [1], [8300], holes)


@pytest.mark.parametrize("d,mx", [(64, False), (128, False), (64, True), (128, True)])
def test_chunks_in_several_rounds(dev, d, mx):                             # noqa: F811
    """More row blocks than one round of blocks: splits by the estimated time, of unequal sequences."""
    both_ways(dev, 32, 16, d, 64, mx, [300, 280, 301, 260], [2100, 2700, 400, 2500], kws=(dict(),))


@pytest.mark.parametrize("hkv", [2, 4])
@pytest.mark.parametrize("d,mx", [(64, False), (128, True)])
def test_chunks_of_many_sequences(dev, d, mx, hkv):                        # noqa: F811
    """75 sequences of chunks, more than a wave looks at at once; one long, some empty. hkv 4: several rounds."""
    g = torch.Generator().manual_seed(75)
    lens = torch.randint(60, 300, (75,), generator=g).tolist()
    rows = [min(n, 9 + 5 * (i % 11)) if i % 7 else 0 for i, n in enumerate(lens)]
    lens[70], rows[70] = 2600, 60
    both_ways(dev, 2 * hkv, hkv, d, 16, mx, rows, lens)


@pytest.mark.parametrize("mx", [False, True])
def test_runs_of_single_tokens(dev, mx):                                   # noqa: F811
    """70 sequences of one token, some long: runs that end inside a sequence and hold several."""
    g = torch.Generator().manual_seed(70)
    lens = torch.randint(1, 400, (70,), generator=g).tolist()
    lens[3], lens[40], lens[69] = 5000, 3333, 2500
    both_ways(dev, 16, 8, 64, 16, mx, [1] * 70, lens, (100,))
