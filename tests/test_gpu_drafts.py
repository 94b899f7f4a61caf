"""Answering by drafts on the GPU (rf_paged_tree, rf_attend_tree, rf_verify_drafts, rf_paged_keep) against the float64 oracle.

Tolerances. Attention: test_gpu_paged.py's (check). Slots, positions, bits, paths, tokens and kept rows are equal. (A verified
draw is compared in 64 bits on both sides, where a random number falls between the two sides' borders with a chance below
1e-6 a call: weights are within 3e-12, and there are at most some 1e5 borders.)"""
import random

import pytest
import torch

from oracle import drafts as OD, paged as OP
from test_gpu_paged import ATTN, batch, check, dev, layout, offsets, pages_on, back      # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu
i32 = lambda x, dev: torch.tensor(x, dtype=torch.int32, device=dev)                       # noqa: E731


def tree(n, seed, chain=False):
    r = random.Random(seed)
    return [-1] + [i - 1 if chain or r.random() < 0.4 else r.randint(0, i - 1) for i in range(1, n)] if n else []


# ------------------------------------------------------------------------------------------------ the plan

def plan_oracle(parents, lens, table, page, n_pages, words):
    slots, pos, seen = [], [], []
    for b, par in enumerate(parents):
        see, depth = OD.above(par)
        base = lens[b] - len(par)
        for i in range(len(par)):
            p = base + i
            pg = int(table[b, p // page]) if 0 <= p < table.shape[1] * page else -1
            slots.append(pg * page + p % page if 0 <= pg < n_pages else -1)
            pos.append(max(0, base + depth[i]))
        seen.append(OD.words(see, words))
    return slots, pos, torch.cat(seen)


def test_plan(dev):                                                                        # noqa: F811
    """Trees, chains of hundreds, forests, parents that do not come before their rows, sequences without rows, more rows than
    tokens, padded rows, pages outside the pool, words too few."""
    from rfill import ops
    from rfill.paged import Pages
    page = 16
    parents = [tree(7, 1), [], tree(300, 2, chain=True), tree(190, 3), [-1, 5, 1, 3, -7, 0, 2], tree(20, 4), tree(64, 5), tree(65, 6)]
    lens = [40, 9, 1200, 190, 100, 5, 64, 66]
    table, n_pages = layout([max(n, 1) for n in lens], page, 3)
    table[0, 2], table[3, 1] = 1 << 30, n_pages
    pages = Pages.empty(n_pages, 1, page, 64, "bf16", dev)
    counts = [len(p) for p in parents]
    T = sum(counts) + 5
    par = i32([x for p in parents for x in p] + [0] * 5, dev)
    for words in (5, 1):
        slots, pos, seen = ops.paged_tree(table.to(dev), i32(lens, dev), offsets(counts).to(dev), par, T, pages, 64 * words)
        ws, wp, wb = plan_oracle(parents, lens, table, page, n_pages, words)
        assert slots.tolist() == ws + [-1] * 5 and pos.tolist() == wp + [0] * 5
        assert torch.equal(seen.cpu(), torch.cat((wb, torch.zeros(5, words, dtype=torch.int64))))
    one = ops.paged_tree(table[:0].to(dev), i32([], dev), i32([0], dev), par[:3], 3, pages, 3)
    assert one[0].tolist() == [-1] * 3 and one[1].tolist() == [0] * 3 and one[2].tolist() == [[0]] * 3
    none = ops.paged_tree(table.to(dev), i32(lens, dev), offsets([0] * 8).to(dev), par[:0], 0, pages, 0)
    assert none[0].shape == (0,) and none[2].shape == (0, 1)


def test_plan_many_sequences(dev):                                                         # noqa: F811
    """More rows than a block, sequences across the blocks' borders, one of thousands of rows."""
    from rfill import ops
    from rfill.paged import Pages
    page = 64
    parents = [tree(1 + 13 * b % 60, b) for b in range(70)] + [tree(5000, 7)]
    lens = [200 + b for b in range(70)] + [5100]
    table, n_pages = layout(lens, page, 3)
    pages = Pages.empty(n_pages, 1, page, 64, "bf16", dev)
    counts = [len(p) for p in parents]
    got = ops.paged_tree(table.to(dev), i32(lens, dev), offsets(counts).to(dev), i32([x for p in parents for x in p], dev), sum(counts),
                         pages, 5000)
    see = [None] * 5000
    for i, p in enumerate(parents[70]):
        see[i] = (see[p] if p >= 0 else 0) | 1 << i
    want = [[(x >> 64 * w & (1 << 64) - 1) for w in range(79)] for x in see]
    want = torch.tensor([[x - (1 << 64) if x >> 63 else x for x in row] for row in want], dtype=torch.int64)
    assert torch.equal(got[2][-5000:].cpu(), want)
    ws, wp, wb = plan_oracle(parents[:70], lens, table, page, n_pages, 1)
    m = sum(counts) - 5000
    assert got[0][:m].tolist() == ws and got[1][:m].tolist() == wp and torch.equal(got[2][:m, :1].cpu(), wb)
    assert bool((got[2][:m, 1:] == 0).all())


# ------------------------------------------------------------------------------------------------ attention

def sees(parents):
    return [OD.above(p)[0] for p in parents]


def bits_of(see, words):
    return torch.cat([OD.words(s, words) for s in see])


def oracle(pools, table, n_pages, q, see, lens, hq, scale):
    out, size = (torch.zeros(q.shape[0], hq, pools.d, dtype=torch.float64) for _ in "os")
    at = 0
    for b, (s, n) in enumerate(zip(see, lens)):
        r = s.shape[0]
        if r:
            k, v, ok = OP.keys_of(pools, table[b], n, n_pages)
            out[at:at + r], size[at:at + r] = OD.attend(q[at:at + r].view(r, hq, pools.d), k, v, ok, s, scale)
        at += r
    return out.flatten(1), size.flatten(1)


def run(dev, pools, table, q, see, lens, hq, scale, bits=None, **kw):                      # noqa: F811
    from rfill import ops
    rows = [s.shape[0] for s in see]
    bits = bits_of(see, max(1, -(-max(rows) // 64))) if bits is None else bits
    return ops.attend_tree(q.to(dev), pages_on(pools, dev), table.to(dev), i32(lens, dev), offsets(rows).to(dev), bits.to(dev), hq, scale,
                           kw.pop("max_rows", max(rows)), kw.pop("max_keys", max(max(lens), 1)), **kw)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hq,hkv,d", ATTN)
def test_attend_trees(dev, hq, hkv, d, mx):                                                # noqa: F811
    """Trees of one to some hundred rows: over tiles' and pages' edges, with nothing before them, with more rows than tokens,
    none at all; split and not."""
    for counts, lens in (([6, 1, 0, 13, 4], [50, 1, 30, 77, 3]), ([31, 33, 2], [31, 160, 40]), ([70, 129], [133, 150])):
        see = sees([tree(n, 5 * n + d) for n in counts])
        pools, table, n_pages, q = batch(hq, hkv, d, 16, mx, counts, lens, 3 * d + counts[0])
        want, size = oracle(pools, table, n_pages, q, see, lens, hq, d ** -0.5)
        for kw in (dict(), dict(max_keys=1 << 20), dict(max_keys=1 << 20, workspace=None)):
            got = run(dev, pools, table, q, see, lens, hq, d ** -0.5, **kw)
            check(got, want, size, (counts, kw))


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_long(dev, d, mx):                                                          # noqa: F811
    """Splits of long sequences: trees at their end, whole splits before them, the same bits from run to run."""
    hq, hkv = 8, 2
    for counts, lens in (([3, 9, 1], [9001, 40, 5003]), ([70, 20], [4700, 3000])):
        see = sees([tree(n, n) for n in counts])
        pools, table, n_pages, q = batch(hq, hkv, d, 128, mx, counts, lens, 5)
        want, size = oracle(pools, table, n_pages, q, see, lens, hq, d ** -0.5)
        got = run(dev, pools, table, q, see, lens, hq, d ** -0.5)
        check(got, want, size, "split")
        assert torch.equal(got, run(dev, pools, table, q, see, lens, hq, d ** -0.5))
        check(run(dev, pools, table, q, see, lens, hq, d ** -0.5, workspace=None), want, size, "whole")


@pytest.mark.parametrize("hkv,rep", [(1, 4), (3, 2), (4, 4), (8, 4), (16, 2)])
@pytest.mark.parametrize("d", [128, 256])
def test_attend_row_blocks_beside_one_another(dev, d, hkv, rep):                           # noqa: F811
    """4-bit pages and several row blocks a sequence: any number of heads over the XCDs, few and many sequences, split and not."""
    for counts, lens in (([9, 20, 1, 30], [4000, 2500, 70, 300]), ([1 + i % 17 for i in range(70)], [20 + i for i in range(70)])):
        see = sees([tree(n, n) for n in counts])
        pools, table, n_pages, q = batch(hkv * rep, hkv, d, 64, True, counts, lens, hkv)
        want, size = oracle(pools, table, n_pages, q, see, lens, hkv * rep, d ** -0.5)
        for kw in (dict(), dict(max_keys=1 << 20), dict(max_keys=1 << 20, max_rows=32)):
            got = run(dev, pools, table, q, see, lens, hkv * rep, d ** -0.5, **kw)
            check(got, want, size, (hkv, kw))
            assert torch.equal(got, run(dev, pools, table, q, see, lens, hkv * rep, d ** -0.5, **kw))


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_any_bits(dev, d, mx):                                                      # noqa: F811
    """Bits that are no tree's: random ones, rows that do not see themselves, rows that see nothing (zeros where nothing comes
    before the new rows), bits past a row itself (not looked at), words of which only some rows' are used."""
    hq, hkv = 4, 2
    g = torch.Generator().manual_seed(d)
    for counts, lens in (([9, 20, 33], [9, 20, 90]), ([100, 70], [100, 171])):
        see = [torch.rand(n, n, generator=g) < 0.4 for n in counts]
        for s in see:
            s[3], s[-1] = False, False
        pools, table, n_pages, q = batch(hq, hkv, d, 32, mx, counts, lens, d)
        want, size = oracle(pools, table, n_pages, q, see, lens, hq, d ** -0.5)
        got = run(dev, pools, table, q, see, lens, hq, d ** -0.5, bits=bits_of(see, 4))
        check(got, want, size, counts)
        assert bool((got[3] == 0).all()) and bool((got[counts[0] - 1] == 0).all())


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_hidden_values_do_not_matter(dev, d, mx):                                   # noqa: F811
    """What a row does not see of its own tree may be NaN or infinite: rows beside it keep their bits, rows that see it get
    them."""
    hq, hkv, page = 4, 2, 16
    for n, length in ((7, 30), (80, 123)):
        counts, lens = [n, 5], [length, 21]
        see = sees([tree(n, 11), tree(5, 2)])
        pools, table, n_pages, q = batch(hq, hkv, d, page, mx, counts, lens, d)
        base = run(dev, pools, table, q, see, lens, hq, d ** -0.5)
        odd = [i for i in range(2, n) if i % 3 == 0]
        for x, i in enumerate(odd):
            p = length - n + i
            bad = torch.full((hkv, d), (float("nan"), float("inf"), float("-inf"))[x % 3], dtype=torch.float64)
            pools.write(int(table[0, p // page]) * page + p % page, bad, bad)
        got = run(dev, pools, table, q, see, lens, hq, d ** -0.5)
        reached = see[0][:, odd].any(1)
        assert 0 < int(reached.sum()) < n
        assert torch.equal(base[:n].cpu()[~reached], got[:n].cpu()[~reached]) and torch.equal(base[n:], got[n:])
        assert bool(got[:n].cpu()[reached].isnan().any(1).all())


@pytest.mark.parametrize("n", [6, 40])
def test_attend_infinite_values_by_row(dev, n):                                            # noqa: F811
    """An infinite value reaches its column in the rows that see it, and no other row or column."""
    hq, hkv, d, page = 4, 2, 128, 16
    see = sees([tree(n, 3)])
    pools, table, n_pages, q = batch(hq, hkv, d, page, False, [n], [n + 20], 4)
    base = run(dev, pools, table, q, see, [n + 20], hq, d ** -0.5).cpu().view(n, hq, d)
    p = 20 + 2
    pools.v[int(table[0, p // page]), 1, p % page, 9] = float("-inf")
    got = run(dev, pools, table, q, see, [n + 20], hq, d ** -0.5).cpu().view(n, hq, d)
    hit = see[0][:, 2]
    assert bool((got[hit][:, 2:, 9] == float("-inf")).all())
    got[:, 2:, 9], base[:, 2:, 9] = 0, 0
    # (the tile's other values enter the product as before)
    assert bool(got.isfinite().all()) and torch.equal(got[~hit], base[~hit])


@pytest.mark.parametrize("mx", [False, True])
def test_attend_chain_is_causal(dev, mx):                                                  # noqa: F811
    """A chain's bits give attend_paged's outputs (their tolerance apart, twice: tiles are cut elsewhere)."""
    from test_gpu_paged import run as causal
    hq, hkv, d = 8, 2, 128
    counts, lens = [8, 1, 70], [300, 17, 90]
    see = sees([tree(n, 0, chain=True) for n in counts])
    pools, table, n_pages, q = batch(hq, hkv, d, 32, mx, counts, lens, 8)
    want, size = oracle(pools, table, n_pages, q, see, lens, hq, d ** -0.5)
    check(run(dev, pools, table, q, see, lens, hq, d ** -0.5), want, size, "bits")
    check(causal(dev, pools, table, q, counts, lens, hq, d ** -0.5), want, size, "causal")


def test_attend_strides_and_rows_of_no_sequence(dev):                                      # noqa: F811
    """Queries, outputs and bits with strides of their own, rows after the last sequence left as they were."""
    from rfill import ops
    hq, hkv, d, page, counts, lens = 8, 2, 128, 16, [5, 3], [70, 33]
    see = sees([tree(5, 1), tree(3, 2)])
    pools, table, n_pages, q = batch(hq, hkv, d, page, False, counts, lens, 2)
    want, size = oracle(pools, table, n_pages, q, see, lens, hq, d ** -0.5)
    qs = torch.zeros(10, hq * d + 24, dtype=torch.bfloat16, device=dev)
    qs[:8, : hq * d] = q.to(dev)
    wide = torch.full((10, 5), -1, dtype=torch.int64, device=dev)
    wide[:8, 1:2] = bits_of(see, 1).to(dev)
    out = torch.full((10, hq * d + 8), 3.0, dtype=torch.bfloat16, device=dev)
    ops.attend_tree(qs[:, : hq * d], pages_on(pools, dev), table.to(dev), i32(lens, dev), offsets(counts).to(dev), wide[:, 1:2], hq,
                    d ** -0.5, 5, 70, out=out[:, : hq * d])
    check(out[:8, : hq * d], want, size, "strides")
    assert bool((out[8:] == 3).all()) and bool((out[:, hq * d:] == 3).all())


def test_attend_refusals(dev):                                                             # noqa: F811
    from rfill import ops
    hq, hkv, d = 4, 2, 64
    pools, table, n_pages, q = batch(hq, hkv, d, 16, False, [3], [20], 2)
    a = (q.to(dev), pages_on(pools, dev), table.to(dev), i32([20], dev), offsets([3]).to(dev))
    seen = torch.full((3, 1), -1, dtype=torch.int64, device=dev)
    ops.attend_tree(*a, seen, hq, 0.1, 3, 20)
    for bad, kind in ((seen.int(), ValueError), (seen[:2], ValueError), (seen.cpu(), ValueError), (None, TypeError),
                      (seen[:, :0], ValueError), (seen.expand(3, 1)[:1].expand(3, 1).t().contiguous().t(), ValueError),
                      (seen[:1].expand(3, 1), ValueError)):
        with pytest.raises(kind):
            ops.attend_tree(*a, bad, hq, 0.1, 3, 20)
    q2 = torch.zeros(70, hq * d, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        ops.attend_tree(q2, *a[1:], torch.zeros(70, 1, dtype=torch.int64, device=dev), hq, 0.1, 70, 20)
    with pytest.raises(ValueError):
        ops.paged_tree(*a[2:5], i32([-1, 0], dev), 3, a[1], 3)
    with pytest.raises(ValueError):
        ops.paged_tree(*a[2:5], i32([-1, 0, 0], dev), 3, a[1], -1)
    with pytest.raises(ValueError):
        ops.paged_tree(*a[2:5], torch.tensor([-1, 0, 0], dtype=torch.int32), 3, a[1], 3)


# ------------------------------------------------------------------------------------------------ verification

def case(V, counts, seed, draft=False, temps=(0.0, 0.7, 1.0, 1.3), chain=False, peak=8.0):
    """Logits with a few likely tokens a row, trees whose children are likely tokens or drawn from the draft's shares."""
    g = torch.Generator().manual_seed(seed)
    T = sum(counts)
    x = 2 * torch.randn(T, V, generator=g)
    x.scatter_(1, torch.randint(0, V, (T, min(4, V)), generator=g), peak + 2 * torch.randn(T, min(4, V), generator=g))
    q = torch.softmax(x + 0.5 * torch.randn(T, V, generator=g), 1) if draft else None
    parents = [tree(n, seed + i, chain) for i, n in enumerate(counts)]
    tokens, at = torch.zeros(T, dtype=torch.int64), 0
    for par in parents:
        for i, p in enumerate(par):
            if p >= 0:
                row = x[at + p] if q is None else q[at + p].log()
                noise = -torch.log(-torch.log(torch.rand(V, generator=g).clamp(1e-9, 1 - 1e-7)))
                tokens[at + i] = int((row + noise).argmax())
        at += len(par)
    temp = torch.tensor([temps[b % len(temps)] for b in range(len(counts))])
    return dict(x=x, q=q, parents=parents, tokens=tokens, counts=counts, temp=temp, u=torch.rand(T, generator=g),
                r=torch.rand(len(counts), generator=g))


def want_of(c, depth):
    paths, nxt, at = [], [], 0
    for b, par in enumerate(c["parents"]):
        n = len(par)
        s = slice(at, at + n)
        if n == 0:
            p, t = [], -1
        else:
            p, t = OD.verify(c["x"][s], c["tokens"][s], par, c["u"][s], c["r"][b], float(c["temp"][b]), depth,
                             None if c["q"] is None else c["q"][s])
        paths.append(p)
        nxt.append(t)
        at += n
    return paths, nxt


def verify(dev, c, depth, x=None, q="own", rows=None, **kw):                               # noqa: F811
    from rfill import ops
    up = lambda t: t.to(dev)                                                               # noqa: E731
    q = c["q"] if isinstance(q, str) else q
    x = up(c["x"]) if x is None else x
    pad = x.shape[0] - sum(c["counts"])
    z = lambda t: torch.cat((t, t.new_zeros(pad)))                                         # noqa: E731
    return ops.verify_drafts(x, up(z(c["tokens"])), i32([v for p in c["parents"] for v in p] + [0] * pad, dev), offsets(c["counts"]).to(dev),
                             up(z(c["u"])), up(c["r"]), up(c["temp"]), max(c["counts"]) if rows is None else rows, depth=depth,
                             draft=None if q is None else up(q), **kw)


def same(got, want, depth, name=""):
    paths, nxt = want
    assert got[1].tolist() == [len(p) for p in paths], (name, got[1].tolist(), [len(p) for p in paths])
    assert got[0].tolist() == [p + [-1] * (depth - len(p)) for p in paths], name
    assert got[2].tolist() == nxt, (name, got[2].tolist(), nxt)


@pytest.mark.parametrize("V", [1, 3, 130, 4095, 4096, 4097, 50257, 128256])
@pytest.mark.parametrize("form", ["likely", "f32", "bf16"])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_verify(dev, V, form, kind):                                                       # noqa: F811
    """Chains and trees, greedy and drawn, over vocabularies of one token and up, even and odd."""
    for seed, counts in ((1, [1]), (2, [6, 1, 0, 13]), (3, [30, 9, 2, 17])) if V < 60000 else ((4, [9, 5]),):
        for chain in (False, True):
            c = case(V, counts, seed + V, form != "likely", chain=chain)
            c["x"] = c["x"].to(kind)
            if form == "bf16":
                c["q"] = c["q"].to(torch.bfloat16)
            want = want_of(c, 20)
            same(verify(dev, c, 20), want, 20, (counts, chain))
            if V == 130:
                assert torch.equal(verify(dev, c, 20)[0], verify(dev, c, 20, workspace=torch.full((1 << 16,), 255, dtype=torch.uint8, device=dev))[0])


@pytest.mark.parametrize("draft", [False, True])
def test_verify_many_draws(dev, draft):                                                    # noqa: F811
    """Many sequences over few tokens: every kind of ending (no child accepted, a leaf, several rejected, the same token twice)."""
    counts = [1 + (7 * b) % 12 for b in range(300)]
    c = case(6, counts, 5, draft, peak=1.0)
    same(verify(dev, c, 12), want_of(c, 12), 12)
    flat = case(9000, counts[:60], 6, draft, peak=0.0)                                     # many borders
    same(verify(dev, flat, 12), want_of(flat, 12), 12)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_large_trees(dev, draft):                                                   # noqa: F811
    """As many rows as a sequence may have: a chain, a star (hundreds of rejections at one row), a random tree."""
    V = 5000
    for name, par in (("chain", tree(1024, 1, True)), ("star", [-1] + [0] * (199 if draft else 1023)), ("tree", tree(1024, 2))):
        n = len(par)
        c = case(V, [n], 9, draft, temps=(1.0,))
        c["parents"] = [par]
        if name == "star":
            c["tokens"][1:] = torch.randint(0, V, (n - 1,), generator=torch.Generator().manual_seed(1))
            c["tokens"][5] = c["tokens"][3]
        if name == "chain":                                                                # all accepted, down to the end
            c["u"].zero_()
            c["tokens"][1:] = c["x"][:-1].argmax(1)
        want = want_of(c, 1024)
        same(verify(dev, c, 1024), want, 1024, name)
        assert name != "chain" or len(want[0][0]) == 1024


def test_verify_edges(dev):                                                                # noqa: F811
    """Ties, NaN, rows of nothing, infinite logits and temperatures, r of 1, u of 0, tokens outside the vocabulary, the largest
    and smallest temperatures; in one chunk and over several."""
    inf, nan = float("inf"), float("nan")
    for V in (5, 9001):
        rows = torch.full((8, V), -inf)
        rows[0, :2], rows[0, V - 2:] = torch.tensor([3.0, 1.0]), torch.tensor([3.0, 2.0])
        rows[1, 0], rows[1, V - 1], rows[1, 2] = nan, 0.0, -1.0
        rows[2] = nan
        rows[4, 1], rows[4, V - 1], rows[4, 2] = inf, inf, 7.0
        rows[5] = torch.linspace(-3e38, 3e38, V, dtype=torch.float64).float()
        rows[6] = 0.0
        rows[7, 3] = -3e38
        for t in (0.0, 1.0, 1e-30, 1e-45, 1e30, inf, nan, -1.0):
            for r in (0.0, 0.3, 0.49, 0.5, 0.51, 0.999999, 1.0):
                tokens = torch.zeros(16, dtype=torch.int64)
                tokens[1::2] = torch.tensor([V - 2, V - 1, 0, V, V - 1, V - 1, 3, 3])
                c = dict(x=rows.repeat_interleave(2, 0), q=None, parents=[[-1, 0]] * 8, tokens=tokens, counts=[2] * 8,
                         temp=torch.full((8,), t), u=torch.full((16,), 0.4), r=torch.full((8,), r))
                same(verify(dev, c, 2), want_of(c, 2), 2, (V, t, r))
    # a draft with NaN, negative and infinite shares, and one that leaves nothing
    x = torch.tensor([[1.0, 2.0, 0.5, 0.0], [0.0, 0.0, 1.0, 0.0]])
    for q in ([nan, 0.5, -3.0, 0.5], [0.2, inf, 0.0, nan], [1.0, 1.0, 1.0, 1.0]):
        for u in (0.0, 0.3, 0.9):
            for tok in range(4):
                c = dict(x=x, q=torch.tensor([q, q]), parents=[[-1, 0]], tokens=torch.tensor([0, tok]), counts=[2],
                         temp=torch.ones(1), u=torch.tensor([0.0, u]), r=torch.tensor([0.5]))
                same(verify(dev, c, 2), want_of(c, 2), 2, (q, u, tok))


def test_verify_bounds_strides_and_padding(dev):                                           # noqa: F811
    """Rows with strides and at addresses of their own, rows of no sequence (NaN, never read into an answer), paths shorter than
    the trees, a bound below the rows; no temperature: all greedy."""
    from rfill import ops
    c = case(1003, [9, 4, 0, 12], 3, True)
    for kind in (torch.float32, torch.bfloat16):
        c["x"], q = c["x"].to(kind), c["q"].to(kind)
        c["q"] = q
        wide = torch.full((28, 1003 + 14), float("nan"), dtype=kind, device=dev)
        wq = wide.clone()
        for off in (0, 1, 3):
            wide[:25, off:off + 1003], wq[:25, off:off + 1003] = c["x"].to(dev), q.to(dev)
            same(verify(dev, c, 7, x=wide[:, off:off + 1003], q=wq[:, off:off + 1003]), want_of(c, 7), 7, (kind, off))
        for depth in (1, 2):
            same(verify(dev, c, depth), want_of(c, depth), depth, depth)
    less = dict(c, parents=[p[:5] for p in c["parents"]])
    full, at = [], 0
    for p in c["parents"]:
        full.append(list(range(at, at + min(5, len(p)))))
        at += len(p)
    pick = [i for f in full for i in f]
    short = dict(less, x=c["x"][pick], q=c["q"][pick], tokens=c["tokens"][pick], u=c["u"][pick], counts=[len(f) for f in full])
    same(verify(dev, c, 7, rows=5), want_of(short, 7), 7, "rows")
    par = i32([v for p in c["parents"] for v in p], dev)
    got = ops.verify_drafts(c["x"].to(dev), c["tokens"].to(dev), par, offsets(c["counts"]).to(dev), None, None, None, 12)
    assert got[0].shape == (4, 12)
    same(got, want_of(dict(c, temp=torch.zeros(4)), 12), 12, "greedy")
    nothing = ops.verify_drafts(c["x"].to(dev)[:0], c["tokens"].to(dev)[:0], par[:0], i32([0, 0], dev), None, None, None, 0)
    assert nothing[0].tolist() == [[-1]] and nothing[1].tolist() == [0] and nothing[2].tolist() == [-1]
    none = ops.verify_drafts(c["x"].to(dev)[:0], c["tokens"].to(dev)[:0], par[:0], i32([0], dev), None, None, None, 3)
    assert none[0].shape == (0, 3) and none[2].shape == (0,)


def test_verify_refusals(dev):                                                             # noqa: F811
    from rfill import _lib, ops
    x = torch.zeros(4, 50, device=dev)
    z = lambda n, t=torch.float32: torch.zeros(n, dtype=t, device=dev)                     # noqa: E731
    ok = dict(logits=x, tokens=z(4, torch.int64), parents=z(4, torch.int32), cu=i32([0, 4], dev), u=z(4), r=z(1), temperature=z(1),
              max_rows=4)
    ops.verify_drafts(**ok)
    for k, v in (("logits", x.double()), ("logits", x.cpu()), ("logits", x[:3]), ("logits", x[:1].expand(4, 50)), ("logits", x.t()),
                 ("tokens", z(4, torch.int32)), ("tokens", z(3, torch.int64)), ("parents", z(4, torch.int64)), ("parents", z(5, torch.int32)),
                 ("cu", i32([], dev)), ("cu", i32([0, 2, 4], dev)), ("u", z(3)), ("u", z(4, torch.float64)), ("r", z(2)),
                 ("temperature", z(2)), ("depth", 0), ("depth", 1025), ("draft", x[:, :49]), ("draft", x.half()), ("draft", x.cpu()),
                 ("workspace", z(8, torch.uint8)), ("workspace", z(4096)), ("max_rows", -1)):
        with pytest.raises(ValueError):
            ops.verify_drafts(**dict(ok, **{k: v}))
    for k, v in (("u", None), ("r", None)):
        with pytest.raises(TypeError):
            ops.verify_drafts(**dict(ok, **{k: v}))
    with pytest.raises(TypeError):
        ops.verify_drafts(**dict(ok, workspace=None))
    with pytest.raises(_lib.UnsupportedArchitecture):
        ops.verify_drafts(**dict(ok, max_rows=1025))


# ------------------------------------------------------------------------------------------------ kept rows

@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hkv,d,page", [(2, 64, 16), (8, 128, 64), (2, 256, 16), (17, 256, 32), (1, 128, 1024)])
def test_keep(dev, hkv, d, page, mx):                                                      # noqa: F811
    """Paths of every kind, in several layers of different memory: none moved, all, within a page and across pages, longer than
    a run of entries, ones that end early (an entry that does not rise, no row, a count beyond them), pages that are none, a
    sequence with more rows than tokens. Everything else keeps its bits."""
    from rfill import ops
    g = torch.Generator().manual_seed(d + page)
    rows = [8, 1, 0, 40, 600, 9, 9, 20, 30, 7]
    lens = [20, 1, 5, 75, 700, 9, 30, 52, 61, 5]
    long = sorted(random.Random(4).sample(range(600), 400))
    path = [[0, 3, 4, 7], [0], [], [0, 17, 30, 39], long, [0, 1, 2], [0, 5, 4, 8], [0, 2, 20, 21], [0, 8, 16, 25], [0, 3, 5, 6]]
    count = [4, 1, 3, 4, 400, 9, 4, 4, 4, 4]
    table, n_pages = layout([max(n, 7) for n in lens], page, 5)
    if page <= 32:
        table[8, 45 // page] = n_pages                         # (rows of sequence 8 begin at 31)
    layers = []
    for i in range(3):
        pools = OP.Pools(n_pages, hkv, page, d, mx)
        for t in (pools.k, pools.v, pools.ks, pools.vs):
            if t is not None:
                t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, dtype=torch.uint8))
        layers.append(pools)
    pages = [pages_on(p, dev) for p in layers]
    wide = torch.full((10, 403), -1, dtype=torch.int32)
    for b, p in enumerate(path):
        wide[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    assert ops.paged_keep(pages, table.to(dev), i32(lens, dev), offsets(rows).to(dev), wide.to(dev)[:, :401], i32(count, dev)) is None

    def spot(b, p):
        pg = int(table[b, p // page]) if p >= 0 else -1
        return (pg, p % page) if 0 <= pg < n_pages else None
    for pools, now in zip(layers, pages):
        moves = []
        for b in range(10):
            base = lens[b] - rows[b]
            moves += [(spot(b, base + i), spot(b, base + j)) for i, j in OD.keep(wide[b, :401].tolist(), count[b], rows[b])]
        moves = [(s, t) for s, t in moves if s and t]
        assert len(moves) > 400
        for name in ("k", "v", "ks", "vs"):
            x = getattr(pools, name)
            if x is None:
                continue
            old = x.clone()
            for (sp, so), (dp, do) in moves:
                if not mx or name == "k":
                    x[dp, :, do] = old[sp, :, so]
                else:
                    x[dp, :, do // 8, :, do % 8] = old[sp, :, so // 8, :, so % 8]
            equal = torch.equal(getattr(now, name).cpu().view(torch.uint8), x.view(torch.uint8))
            assert equal, name


def test_keep_many_layers(dev):                                                            # noqa: F811
    """More layers than a launch takes, pages of one buffer with strides of their own; a path on the table's last page."""
    from rfill import ops
    from rfill.paged import Pages
    buf = torch.randn(70, 4, 2, 2, 16, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)      # [layers, pages, k|v, ..]
    now = buf.to(dev)
    pools = [Pages(now[i, :, 0], now[i, :, 1]) for i in range(70)]
    table = torch.tensor([[3, 0], [1, 2]], dtype=torch.int32)
    ops.paged_keep(pools, table.to(dev), i32([32, 20], dev), i32([0, 6, 12], dev), i32([[0, 2, 5], [0, 1, 4]], dev), i32([3, 3], dev))
    want = buf.clone()
    for (sp, so), (dp, do) in (((0, 12), (0, 11)), ((0, 15), (0, 12)), ((2, 2), (2, 0))):
        want[:, dp, :, :, do] = buf[:, sp, :, :, so]
    assert torch.equal(now.cpu(), want)


def test_keep_refusals(dev):                                                               # noqa: F811
    from rfill import ops
    from rfill.paged import Pages
    p = [Pages.empty(2, 1, 16, 64, "bf16", dev) for _ in range(2)]
    a = dict(pools=p, table=i32([[0, 1]], dev), lens=i32([20], dev), cu=i32([0, 4], dev), path=i32([[0, 2]], dev), count=i32([2], dev))
    ops.paged_keep(**a)
    other = Pages.empty(2, 1, 16, 64, "mx4", dev), Pages.empty(2, 1, 32, 64, "bf16", dev), Pages.empty(2, 2, 16, 64, "bf16", dev)
    for k, v in [("pools", [])] + [("pools", [p[0], x]) for x in other] + [
            ("path", i32([[0, 2]], "cpu")), ("path", i32([0, 2], dev)), ("path", i32([[0], [2]], dev)), ("count", i32([2, 2], dev)),
            ("count", torch.tensor([2], device=dev)), ("path", i32([[0], [2]], dev).t()[:, :1].expand(1, 2))]:
        with pytest.raises(ValueError):
            ops.paged_keep(**dict(a, **{k: v}))
    ops.paged_keep(**dict(a, path=i32([[]], dev)))


# ------------------------------------------------------------------------------------------------ together

def test_together_captured_and_on_another_stream(dev):                                     # noqa: F811
    """Plan, append, attention, verification and kept rows as one captured step: replays follow new trees, lengths, tokens and
    random numbers, with the program's own work between them; on another stream the same."""
    from rfill import ops
    hq, hkv, d, page, V, most = 8, 2, 64, 16, 5000, 9
    pool_lens = [80, 64, 130]
    table, n_pages = layout(pool_lens, page, 9)
    for mx in (False, True):
        pools, _, _, _ = batch(hq, hkv, d, page, mx, [1, 1, 1], pool_lens, 4)
        pages = [pages_on(pools, dev) for _ in range(2)]
        T = 3 * most
        hold = dict(lens=i32([0] * 3, dev), cu=i32([0] * 4, dev), par=i32([-1] * T, dev), tok=torch.zeros(T, dtype=torch.int64, device=dev),
                    u=torch.zeros(T, device=dev), r=torch.zeros(3, device=dev), temp=torch.zeros(3, device=dev),
                    kv=torch.zeros(T, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=dev), x=torch.zeros(T, V, device=dev),
                    q=torch.zeros(T, V, device=dev))
        tb = table.to(dev)
        ws = torch.zeros(ops.verify_drafts_workspace_bytes(T, V, 3, most), dtype=torch.uint8, device=dev)
        aws = torch.zeros(max(16, ops.attend_tree_workspace_bytes(T, hq, hkv, d, pages[0].kind, 3, most, 130)), dtype=torch.uint8, device=dev)

        def step():
            h = hold
            slots, _, seen = ops.paged_tree(tb, h["lens"], h["cu"], h["par"], T, pages[0], most)
            k, v = (h["kv"][:, (hq + i * hkv) * d:(hq + (i + 1) * hkv) * d].unflatten(1, (hkv, d)) for i in (0, 1))
            for p in pages:
                ops.paged_append(k, v, slots, p)
            out = torch.zeros(T, hq * d, dtype=torch.bfloat16, device=dev)
            ops.attend_tree(h["kv"][:, :hq * d], pages[0], tb, h["lens"], h["cu"], seen, hq, d ** -0.5, most, 130, out=out, workspace=aws)
            got = ops.verify_drafts(h["x"], h["tok"], h["par"], h["cu"], h["u"], h["r"], h["temp"], most, depth=6, draft=h["q"], workspace=ws)
            ops.paged_keep(pages, tb, h["lens"], h["cu"], got[0], got[1])
            return [out, *got]

        def fill(seed):
            counts = [(0, 9, 5), (9, 1, 7), (3, 3, 0)][seed % 3]
            c = case(V, list(counts), seed, True, temps=(0.9, 0.0, 1.1))
            lens = [max(n, n + 11 * seed % 60) for n in counts]
            g = torch.Generator().manual_seed(seed)
            n = sum(counts)
            hold["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
            hold["cu"].copy_(offsets(list(counts)))
            for key, val in (("par", torch.tensor([x for p in c["parents"] for x in p], dtype=torch.int32)), ("tok", c["tokens"]), ("u", c["u"]),
                             ("x", c["x"]), ("q", c["q"])):
                hold[key].zero_()
                hold[key][:n] = val.to(dev)
            hold["r"].copy_(c["r"])
            hold["temp"].copy_(c["temp"])
            hold["kv"].copy_(torch.randn(hold["kv"].shape, generator=g).to(torch.bfloat16))
            return c

        def fresh():
            for p in pages:
                for now, was in ((p.k, pools.k), (p.v, pools.v), (p.ks, pools.ks), (p.vs, pools.vs)):
                    if was is not None:
                        now.copy_(was)

        fill(1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for seed in range(1, 7):
            c = fill(seed)
            fresh()
            want = step()
            held = [t.clone() for p in pages for t in (p.k, p.v, p.ks, p.vs) if t is not None]
            same([t.cpu() for t in want[1:]], want_of(c, 6), 6, seed)
            n = sum(c["counts"])
            fresh()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0][:n], want[0][:n]) and bool((outs[0][n:] == 0).all())
            assert all(torch.equal(a, b) for a, b in zip(outs[1:], want[1:])), seed
            assert all(torch.equal(a, b) for a, b in zip([t for p in pages for t in (p.k, p.v, p.ks, p.vs) if t is not None], held))
            fresh()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = step()
            torch.cuda.current_stream().wait_stream(side)
            assert all(torch.equal(a, b) for a, b in zip(other[1:], want[1:])) and torch.equal(other[0][:n], want[0][:n])


def test_two_verifications_at_once(dev):                                                   # noqa: F811
    """Calls on two streams with workspaces of their own."""
    cs = [case(50000, [9, 30, 4], s, s == 2) for s in (1, 2)]
    want = [want_of(c, 12) for c in cs]
    for c in cs:
        c["x"], c["q"] = c["x"].to(dev), None if c["q"] is None else c["q"].to(dev)
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for turn in range(3):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(verify(dev, c, 12, x=c["x"]))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        same(o, want[i % 2], 12, i)
