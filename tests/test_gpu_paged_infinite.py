"""4-bit pages whose scales take values past bfloat16's range: bytes 253 and 254 make infinities of some codes, 255 makes NaN
of all. Attention by both kernels (few rows a sequence, chunks), where such values are hidden and where they are seen, and the
rows read back. Tolerance: test_gpu_paged.py's (check)."""
import pytest
import torch

from oracle import paged as OP
from paged_dense import attend as dense, values
from test_gpu_paged import batch, check, dev, run                       # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu

# new rows and lengths of two sequences: single tokens, a few, a chunk (k_paged_many at head_dim 64 and 128)
SHAPES = (([1, 1], [21, 37]), ([6, 3], [21, 40]), ([90, 70], [101, 75]))


def spoil(pools, page, token, g, byte=None):
    """Random codes under scale bytes 253 to 255 (or `byte`) at a token of a page, in keys and values."""
    d, hkv = pools.d, pools.hkv
    codes = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)          # noqa: E731
    pools.k[page, :, token], pools.v[page, :, token // 8, :, token % 8] = codes(hkv, d // 2), codes(hkv, 16, d // 32)
    for t in (pools.ks, pools.vs):
        t[page, :, token // 8, :, token % 8] = (torch.randint(253, 256, (hkv, d // 32), generator=g, dtype=torch.uint8)
                                                if byte is None else byte)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_hidden_scales_do_not_matter(dev, d):                              # noqa: F811
    """Such bytes in slots past a sequence's end, in later tokens of the same call and on page 0 behind a table entry that is
    none: the rows that do not see them keep their outputs bit for bit."""
    hq, hkv, page = 4, 2, 16
    for rows, lens in SHAPES:
        pools, table, n_pages, q = batch(hq, hkv, d, page, True, rows, lens, d + rows[0])
        spare = next(p for p in range(n_pages) if p and not bool((table == p).any()))
        for t in (pools.k, pools.v, pools.ks, pools.vs):                   # page 0 belongs to no sequence
            t[spare] = t[0]
        table[table == 0] = spare
        table[1, 0] = n_pages
        base = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
        split = run(dev, pools, table, q, rows, lens, hq, d ** -0.5, max_keys=1 << 16)
        want, size = dense(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
        check(base, want, size, "clean")
        check(split, want, size, "clean, split")
        g = torch.Generator().manual_seed(d)
        used = {(int(table[b, j // page]), j % page) for b in range(2) for j in range(lens[b])}
        for byte in (253, 254, None):
            for p in range(n_pages):
                for t in range(page):
                    if (p, t) not in used:
                        spoil(pools, p, t, g, byte)
            got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
            assert torch.equal(base, got), (rows, byte)
            got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5, max_keys=1 << 16)
            assert torch.equal(split, got), (rows, byte, "split")
        if rows[0] == 1:
            continue
        first = rows[0] - rows[0] // 2                                     # the rows that see none of the spoiled tokens
        for byte in (253, 254, None):
            for j in range(lens[0] - rows[0] // 2, lens[0]):
                spoil(pools, int(table[0, j // page]), j % page, g, byte)
            for kw, ref in ((dict(), base), (dict(max_keys=1 << 16), split)):
                got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5, **kw)
                assert torch.equal(ref[:first], got[:first]) and torch.equal(ref[rows[0]:], got[rows[0]:]), (rows, byte, kw)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_seen_scales(dev, d):                                              # noqa: F811
    """Infinite values in sight reach their columns with their sign, whatever else their tile holds (a block that reads as NaN
    in a seen slot of other columns, or in a hidden one), NaN where both signs meet; other columns stay finite and right."""
    hq, hkv, page = 4, 2, 16
    inf_codes = torch.tensor([4, 5, 6, 7, 12, 13, 14, 15], dtype=torch.uint8)            # under byte 254: 2 to 6 times 2^127
    for rows, lens in SHAPES:
        pools, table, n_pages, q = batch(hq, hkv, d, page, True, rows, lens, 3 * d + rows[0])
        g = torch.Generator().manual_seed(7 * d)
        n = lens[0]
        for j, mode in ((3, "all"), (n - 2, "some"), (n - 1, "some"), (n - 2 - rows[0] // 2, "all")):
            p, t = int(table[0, j // page]), j % page
            codes = inf_codes[torch.randint(0, 8, (hkv, d), generator=g)]
            keep = torch.rand(hkv, d, generator=g) < (0.1 if mode == "all" else 0.3)
            codes = torch.where(keep, codes, 0)
            pools.v[p, :, t // 8, :, t % 8] = (codes[:, 0::2] | (codes[:, 1::2] << 4)).view(hkv, 16, -1)
            pools.vs[p, :, t // 8, :, t % 8] = 254
        p, t = int(table[0, (n - 1) // page]), (n - 1) % page
        pools.vs[p, 0, t // 8, 1, t % 8] = 255                             # head 0, columns 32 .. 63 of the last token
        last = int(table[1, (lens[1] - 1) // page])
        for t in range((lens[1] - 1) % page + 1, page):                    # sequence 1: hidden ones only
            spoil(pools, last, t, g)
        want, size = dense(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
        assert bool((want == float("inf")).any()) and bool((want == float("-inf")).any()) and bool(want.isnan().any())
        for kw in (dict(), dict(max_keys=1 << 16), dict(max_keys=1 << 16, workspace=None)):
            got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5, **kw).cpu().double()
            assert torch.equal(got.isnan(), want.isnan()), (rows, kw)
            odd = ~want.isfinite()
            same = odd & ~want.isnan()
            assert torch.equal(got[same], want[same]), (rows, kw)
            check(got.masked_fill(odd, 0), want.masked_fill(odd, 0), size, (rows, kw))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_beyond_bfloat16(dev, d):                                     # noqa: F811
    """What an append makes of magnitudes above 1.75 2^127 (byte 253, a code of 4: 2^128), and what blocks of every byte from 248
    on read as: values beyond bfloat16 are infinities, byte 255 is NaN."""
    from rfill import ops
    from rfill.paged import Pages
    hkv, page, n_pages = 2, 16, 2
    top = torch.finfo(torch.bfloat16).max
    x = torch.zeros(4, hkv, d, dtype=torch.bfloat16)
    x[0], x[1, :, ::2], x[1, :, 1::2] = top, -top, 1.0
    x[2] = 1.5 * 2.0 ** 127
    x[3] = -1.75 * 2.0 ** 127                                             # the largest that still rounds into range: to 1.5 2^127
    pages = Pages.empty(n_pages, hkv, page, d, "mx4", dev)
    slots = torch.tensor([0, 5, 17, 31], device=dev)
    ops.paged_append(x.to(dev), x.flip(0).to(dev), slots, pages)
    want = torch.where(x.double().abs() > 1.75 * 2.0 ** 127, float("inf"), 1.5 * 2.0 ** 127).copysign(x.double())
    want[1, :, 1::2] = 0
    rk, rv = (t.cpu().double() for t in ops.paged_read(pages, slots))
    assert torch.equal(rk, want) and torch.equal(rv, want.flip(0))
    pools = OP.Pools(n_pages, hkv, page, d, True)
    g = torch.Generator().manual_seed(d)
    for t in (pools.k, pools.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (pools.ks, pools.vs):
        t.copy_(torch.randint(248, 256, t.shape, generator=g, dtype=torch.uint8))
    raw = Pages(*(t.to(dev) for t in (pools.k, pools.v, pools.ks, pools.vs)))
    at = torch.arange(n_pages * page)
    for got, want in zip(ops.paged_read(raw, at.to(dev)), values(pools)):
        want = want.transpose(1, 2).reshape(n_pages * page, hkv, d)
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan()) and bool((want == float("inf")).any())
        assert torch.equal(got.nan_to_num(7.0, float("inf"), float("-inf")), want.nan_to_num(7.0, float("inf"), float("-inf")))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_the_smallest_scales(dev, d):                              # noqa: F811
    """Blocks of bytes 0 to 8, 2^-127 to 2^-119: their codes' values down to 2^-128 are bfloat16 numbers, and read as such."""
    from rfill import ops
    from rfill.paged import Pages
    hkv, page, n_pages = 2, 16, 2
    pools = OP.Pools(n_pages, hkv, page, d, True)
    g = torch.Generator().manual_seed(d)
    for t in (pools.k, pools.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (pools.ks, pools.vs):
        t.copy_(torch.randint(0, 9, t.shape, generator=g, dtype=torch.uint8))
    raw = Pages(*(t.to(dev) for t in (pools.k, pools.v, pools.ks, pools.vs)))
    for got, want in zip(ops.paged_read(raw, torch.arange(n_pages * page, device=dev)), values(pools)):
        assert torch.equal(got.cpu().double(), want.transpose(1, 2).reshape(n_pages * page, hkv, d))
