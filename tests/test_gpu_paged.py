"""The paged cache on the GPU (rf_paged_slots, rf_paged_append, rf_paged_read, rf_attend_paged) against the float64
oracle.

Tolerances. A rounding to bf16 is off by at most u = 2^-8 of the value, one in fp32 by 2^-24.
 - Appended bf16 rows and queries: u |y| + 8 2^-24 (|a c| + |b s|): at most 8 fp32 roundings before the last one (the
   statistic's r, two products of the norm for each of the pair, two of the rotation and the sum).
 - 4-bit rows: half the step around the value the code stands for, plus the same fp32 part; rows stored without norm and
   rotation are exact, so their codes and scales are the oracle's.
 - Attention: u |o| for the output, u A for the probabilities (A = sum p |v|), and a relative error of the probabilities
   from fp32 scores, exponentials and sums: scores sum d products, each at most 2^-24 d sum |q k| scale off; the inputs
   here keep scale sum |q k| below 128, so with d <= 256 that is below 2^-9, twice (a probability and the sum) 2^-8 in the
   worst case. In all u |o| + 2 u A + 2^-30."""
import pytest
import torch

from oracle import paged as OP

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
F = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from rfill import _lib
    _lib.load()
    return torch.device("cuda")


def pages_on(pools, dev):
    from rfill.paged import Pages
    return Pages(*(None if t is None else t.to(dev) for t in (pools.k, pools.v, pools.ks, pools.vs)))


def back(pages, pools):
    """The device pages as oracle pools."""
    got = OP.Pools(1, pools.hkv, pools.page, pools.d, pools.mx)
    for n in ("k", "v", "ks", "vs"):
        setattr(got, n, None if getattr(pages, n) is None else getattr(pages, n).cpu())
    return got


def layout(lens, page, seed, extra=2):
    """A table of shuffled pages for sequences of these lengths (unused entries -1) and the number of pages."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def offsets(rows):
    return torch.tensor([0] + torch.tensor(rows).cumsum(0).tolist(), dtype=torch.int32)


def test_slots(dev):
    """Ragged sequences, an empty one, a padded row, a page outside the pool, more rows than tokens, a short table."""
    from rfill import ops
    from rfill.paged import Pages
    page = 16
    pages = Pages.empty(7, 1, page, 64, "bf16", dev)
    table = torch.tensor([[3, 1, -1], [0, 99, 2], [4, -1, -1], [5, 6, 0], [2, 2, 2]], dtype=torch.int32)
    lens = torch.tensor([20, 40, 0, 2, 60], dtype=torch.int32)
    rows = [5, 30, 0, 4, 20]
    slots, pos = ops.paged_slots(table.to(dev), lens.to(dev), offsets(rows).to(dev), sum(rows) + 3, pages)
    want_s, want_p = [], []
    for b, r in enumerate(rows):
        for i in range(r):
            p = int(lens[b]) - r + i
            pg = int(table[b, p // page]) if 0 <= p < 3 * page else -1
            want_s.append(pg * page + p % page if 0 <= pg < 7 else -1)
            want_p.append(max(p, 0))
    assert slots.tolist() == want_s + [-1] * 3 and pos.tolist() == want_p + [0] * 3


HEADS = [(4, 2, 64, 64), (32, 8, 128, 128), (16, 2, 256, 64), (6, 2, 128, 32), (3, 1, 64, 8), (5, 5, 256, 256)]


def _rows_in(rows, hq, hkv, d, rot, seed, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, (hq + 2 * hkv) * d, generator=g)
    x[:, : (hq + hkv) * d] *= torch.exp(0.7 * torch.randn((hq + hkv) * d, generator=g))
    x = x.to(torch.bfloat16)
    ang = 300 * torch.rand(rows, rot // 2, generator=g)
    cs = torch.cat((ang.cos(), ang.sin()), 1).to(torch.bfloat16)
    gains = [None, None] if kind is None else [(0.2 * torch.randn(d, generator=g) + 1 - kind).to(torch.bfloat16) for _ in "qk"]
    return x, cs, gains


def _fp32_part(x, gain, kind, eps, cs):
    """sum of the magnitudes that an output's fp32 roundings are relative to."""
    y = OP.rows(x, gain, kind, eps).abs()
    if cs is None:
        return y
    h = cs.shape[1] // 2
    c, s = cs[:, None, :h].double().abs(), cs[:, None, h:].double().abs()
    a, b = y[..., :h], y[..., h:2 * h]
    return torch.cat((a * c + b * s, b * c + a * s, y[..., 2 * h:]), -1)


@pytest.mark.parametrize("kind", [None, 0, 1])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hq,hkv,d,rot", HEADS)
def test_append(dev, hq, hkv, d, rot, mx, kind):
    """New rows of every head layout into pages: keys, values and queries, in place and into another buffer, skipped rows,
    strided inputs; the other slots keep their bits."""
    from rfill import ops
    page, eps = 32, 1e-5
    for rows in (1, 19, 150):
        x, cs, (qn, kn) = _rows_in(rows, hq, hkv, d, rot, 17 * rows + d, kind)
        g = torch.Generator().manual_seed(rows)
        n_pages = rows // page + 3
        slots = torch.randperm(n_pages * page, generator=g)[:rows]
        if rows > 1:
            slots[rows // 2], slots[0] = -1, n_pages * page    # rows that are not written
        pools = OP.Pools(n_pages, hkv, page, d, mx)
        for t in (pools.k, pools.v, pools.ks, pools.vs):
            if t is not None:
                t.view(torch.uint8).copy_(torch.randint(0, 120, t.view(torch.uint8).shape, generator=g, dtype=torch.uint8))
        pages = pages_on(pools, dev)
        xd = x.to(dev)
        q = xd[:, : hq * d]
        k, v = (xd[:, (hq + i * hkv) * d:(hq + (i + 1) * hkv) * d].unflatten(1, (hkv, d)) for i in (0, 1))
        up = lambda t: None if t is None else t.to(dev)        # noqa: E731
        out = torch.full((rows, hq * d + 16), 7.0, dtype=torch.bfloat16, device=dev)
        got_q = ops.paged_append(k, v, slots.to(dev), pages, cs=cs.to(dev), q=q, out=out[:, : hq * d], qnorm=up(qn),
                                 knorm=up(kn), norm_kind=kind or 0, eps=eps)
        assert bool((out[:, hq * d:] == 7).all())
        again = ops.paged_append(k, v, slots.to(dev), pages, cs=cs.to(dev), q=q, out=q, qnorm=up(qn), knorm=up(kn),
                                 norm_kind=kind or 0, eps=eps)
        assert again.data_ptr() == xd.data_ptr() and torch.equal(got_q, again)
        xq, xk = x[:, : hq * d].view(rows, hq, d), x[:, hq * d:(hq + hkv) * d].view(rows, hkv, d)
        xv = x[:, (hq + hkv) * d:].view(rows, hkv, d).double()
        want, part = OP.rows(xq, qn, kind, eps, cs), _fp32_part(xq, qn, kind, eps, cs)
        err = (got_q.cpu().double().view(rows, hq, d) - want).abs()
        assert bool((err <= U * want.abs() + 8 * F * part).all()), float((err - U * want.abs()).max())
        wk, pk = OP.rows(xk, kn, kind, eps, cs), _fp32_part(xk, kn, kind, eps, cs)
        now = back(pages, pools)
        live = [(i, int(s)) for i, s in enumerate(slots) if 0 <= s < n_pages * page]
        for i, s in live:
            gk, gv = now.read(s)
            if not mx:
                assert torch.equal(gv, xv[i])
                assert bool(((gk - wk[i]).abs() <= U * wk[i].abs() + 8 * F * pk[i]).all())
                continue
            (_, kb), (vc, vb) = OP.mx4_encode(wk[i]), OP.mx4_encode(xv[i])
            assert torch.equal(gv, OP.mx4_decode(vc, vb))
            p, t = s // page, s % page
            a = wk[i].abs().reshape(hkv, -1, 32).amax(-1)
            edge = (a / torch.exp2(torch.floor(torch.log2(a))) - 1.75).abs() < 1e-5
            assert bool(((now.ks[p, :, t // 8, :, t % 8] == kb) | edge).all())
            sc = torch.exp2(now.ks[p, :, t // 8, :, t % 8].double() - 127).repeat_interleave(32, -1)
            m = gk.abs() / sc                                  # half a step around a level, 1 past the largest
            step = torch.where(m < 2, 0.25, torch.where(m < 4, 0.5, 1.0)) * sc
            assert bool(((gk - wk[i]).abs() <= step + 8 * F * pk[i]).all())
        for i, s in live:                                      # every other slot as it was
            z = torch.zeros(hkv, d, dtype=torch.float64)
            now.write(s, z, z)
            pools.write(s, z, z)
        for n in ("k", "v", "ks", "vs"):
            a, b = getattr(now, n), getattr(pools, n)
            same = a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert same, n


@pytest.mark.parametrize("d", [64, 128, 256])
def test_stored_rows_are_exact(dev, d):
    """Rows stored as they are, from a filled cache's views [hkv, cap, d]: the bits of bf16, the oracle's codes and scales
    in 4 bits, also for zeros, halfway values, the smallest and largest magnitudes, infinities and NaN; read back."""
    from rfill import ops
    from rfill.paged import Pages
    hkv, page, rows = 3, 16, 85
    g = torch.Generator().manual_seed(d)
    kb, vb = ((torch.randn(hkv, rows + 11, d, generator=g) * torch.exp(3 * torch.randn(hkv, rows + 11, 1, generator=g)))
              .to(torch.bfloat16) for _ in "kv")
    kb[:, 3] = 0
    kb[:, 4, ::2] = -0.0
    half = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    kb[0, 5, :32] = torch.cat((half, -half, half / 2, half * 0.875)).to(torch.bfloat16)
    kb[1, 5, :32] = torch.cat((half * 2.0 ** -100, -half, half / 4, half * 0.75)).to(torch.bfloat16)
    kb[:, 6] = torch.finfo(torch.bfloat16).max
    kb[:, 7] = 1e-39
    vb[0, 8, 5], vb[1, 8, 33], vb[2, 9, 0] = float("inf"), float("nan"), float("-inf")
    slots = torch.randperm((rows // page + 2) * page, generator=g)[:rows]
    k, v = (b[:, :rows].transpose(0, 1) for b in (kb.to(dev), vb.to(dev)))
    for kind in ("bf16", "mx4"):
        pages = Pages.empty(rows // page + 2, hkv, page, d, kind, dev)
        assert ops.paged_append(k, v, slots.to(dev), pages) is None
        pools = OP.Pools(rows // page + 2, hkv, page, d, kind == "mx4")
        for i, s in enumerate(slots.tolist()):
            pools.write(s, kb[:, i].double(), vb[:, i].double())
        for n in ("k", "v", "ks", "vs"):
            a, b = getattr(pages, n), getattr(pools, n)
            if a is not None:                                  # (which NaN it is is left open)
                a, nan = a.cpu(), b.isnan()
                assert torch.equal(a.isnan(), nan), (kind, n)
                a, b = (t.masked_fill(nan, 0).view(torch.uint8) for t in (a, b))
                same = torch.equal(a, b)
                assert same, (kind, n)
        ask = torch.cat((slots, torch.tensor([-1, (rows // page + 2) * page, 1 << 40])))
        rk, rv = ops.paged_read(pages, ask.to(dev))
        for got, at in ((rk, 0), (rv, 1)):
            want = torch.stack([pools.read(s)[at] for s in slots.tolist()]).to(torch.bfloat16)
            assert torch.equal(got[:rows].cpu().isnan(), want.isnan())
            assert torch.equal(got[:rows].cpu().nan_to_num(7), want.nan_to_num(7))
            assert bool((got[rows:] == 0).all())


def batch(hq, hkv, d, page, mx, rows, lens, seed, size=1.0):
    """Pools filled with random K / V for these sequences, their table, queries."""
    g = torch.Generator().manual_seed(seed)
    table, n_pages = layout(lens, page, seed)
    pools = OP.Pools(n_pages, hkv, page, d, mx)
    k = torch.randn(n_pages, hkv, page, d, generator=g) * torch.exp(0.4 * torch.randn(d, generator=g))
    v = torch.randn(n_pages, hkv, page, d, generator=g)
    if mx:
        (kc, kb), (vc, vb) = OP.mx4_encode(k), OP.mx4_encode(v)
        by = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)      # noqa: E731
        s8 = lambda b: b.view(n_pages, hkv, page // 8, 8, d // 32).transpose(3, 4).contiguous()   # noqa: E731
        pools.k, pools.ks, pools.vs = by(kc).contiguous(), s8(kb), s8(vb)
        pools.v = by(vc).view(n_pages, hkv, page // 8, 8, 16, d // 32).transpose(3, 4).contiguous()
    else:
        pools.k, pools.v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    q = (size * torch.randn(sum(rows), hq * d, generator=g)).to(torch.bfloat16)
    return pools, table, n_pages, q


def oracle_attend(pools, table, n_pages, q, rows, lens, hq, scale):
    out, size = (torch.zeros(q.shape[0], hq, pools.d, dtype=torch.float64) for _ in "os")
    at = 0
    for b, (r, n) in enumerate(zip(rows, lens)):
        if r:
            k, v, ok = OP.keys_of(pools, table[b], n, n_pages)
            out[at:at + r], size[at:at + r] = OP.attend(q[at:at + r].view(r, hq, pools.d), k, v, ok, scale)
        at += r
    return out.flatten(1), size.flatten(1)


def check(got, want, size, name):
    err = (got.cpu().double() - want).abs()
    bound = U * want.abs() + 2 * U * size + 2.0 ** -30
    assert bool((err <= bound).all()), (name, float((err / bound).max()))


def run(dev, pools, table, q, rows, lens, hq, scale, **kw):
    from rfill import ops
    pages = pages_on(pools, dev)
    return ops.attend_paged(q.to(dev), pages, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                            offsets(rows).to(dev), hq, scale, kw.pop("max_rows", max(rows)),
                            kw.pop("max_keys", max(max(lens), 1)), **kw)


ATTN = [(4, 2, 64), (32, 8, 128), (16, 2, 256), (6, 2, 128), (7, 1, 64), (3, 3, 256), (48, 1, 128), (64, 1, 64)]


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hq,hkv,d", ATTN)
def test_attend_single_tokens(dev, hq, hkv, d, mx):
    """One new token of each of several sequences: lengths of one, around the tiles and pages, none at all; split and not."""
    lens = [1, 15, 16, 17, 33, 0, 64, 130, 401]
    rows = [1, 1, 1, 1, 1, 0, 1, 1, 1]
    for page in (16, 64):
        pools, table, n_pages, q = batch(hq, hkv, d, page, mx, rows, lens, 3 * d + page)
        want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
        for kw in (dict(), dict(max_keys=1 << 20), dict(max_keys=1 << 20, workspace=None)):
            check(run(dev, pools, table, q, rows, lens, hq, d ** -0.5, **kw), want, size, (page, kw))


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (32, 8, 128), (16, 2, 256), (6, 2, 128), (48, 1, 128)])
def test_attend_some_rows(dev, hq, hkv, d, mx):
    """A few to some hundred new rows a sequence, ragged, one with more rows than tokens."""
    for rows, lens in (([2, 5, 0, 3], [2, 40, 9, 77]), ([9, 1, 12], [100, 33, 7]), ([131, 70], [131, 260])):
        pools, table, n_pages, q = batch(hq, hkv, d, 32, mx, rows, lens, d + len(lens))
        want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
        for kw in (dict(), dict(max_keys=1 << 20)):
            got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5, **kw)
            check(got, want, size, (rows, kw))


@pytest.mark.parametrize("mx", [False, True])
def test_attend_long_splits(dev, mx):
    """Splits of one long sequence beside short ones, at positions past several thousand; run to run the same bits."""
    hq, hkv, d, page = 8, 2, 128, 128
    rows, lens = [1, 1, 3], [9001, 40, 5003]
    pools, table, n_pages, q = batch(hq, hkv, d, page, mx, rows, lens, 5)
    want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
    check(got, want, size, "split")
    assert torch.equal(got, run(dev, pools, table, q, rows, lens, hq, d ** -0.5))
    check(run(dev, pools, table, q, rows, lens, hq, d ** -0.5, workspace=None), want, size, "whole")


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_hidden_values_do_not_matter(dev, d, mx):
    """Slots past a sequence's end, later tokens of the same call and pages outside the pool may hold NaN and infinities:
    the rows that do not see them keep their outputs, bit for bit."""
    hq, hkv, page = 4, 2, 16
    for rows, lens in (([1, 1], [21, 37]), ([6, 3], [21, 40]), ([90, 70], [101, 75])):
        pools, table, n_pages, q = batch(hq, hkv, d, page, mx, rows, lens, d + rows[0])
        base = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
        seen = int(lens[0]) - rows[0] // 2                     # keys that the first half of sequence 0's rows see
        used = {(int(table[b, j // page]), j % page) for b in range(2) for j in range(lens[b])}
        nan = torch.full((hkv, d), float("nan"), dtype=torch.float64)
        for p in range(n_pages):
            for t in range(page):
                if (p, t) not in used:
                    pools.write(p * page + t, nan, nan * -1)
        again = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
        assert torch.equal(base, again)
        if rows[0] > 1:
            for j in range(seen, lens[0]):
                bad = nan if j % 2 else torch.full_like(nan, float("inf"))
                pools.write(int(table[0, j // page]) * page + j % page, bad, bad)
            first = rows[0] - rows[0] // 2
            got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
            assert torch.equal(base[:first], got[:first]) and torch.equal(base[rows[0]:], got[rows[0]:])
            assert bool(got[first:rows[0]].isnan().any(1).all())
    # a page outside the pool: its keys are not there; a sequence of none but such pages gives zeros
    rows, lens = [1, 2, 1], [50, 60, 40]
    pools, table, n_pages, q = batch(hq, hkv, d, page, mx, rows, lens, 77)
    table[0, 1], table[1, 3], table[2, :3] = 1 << 30, -7, n_pages
    want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
    check(got, want, size, "bad pages")
    assert bool((got[3] == 0).all())


def test_attend_seen_nan_and_infinity(dev):
    """A NaN key or value in sight makes its rows NaN; an infinite value its column infinite."""
    hq, hkv, d, page, rows, lens = 4, 2, 64, 16, [1, 1, 1], [30, 30, 30]
    pools, table, n_pages, q = batch(hq, hkv, d, page, False, rows, lens, 11)
    base = run(dev, pools, table, q, rows, lens, hq, d ** -0.5)
    at = [(int(table[b, 0]), 5) for b in range(3)]
    pools.k[at[0][0], 0, 5, 3] = float("nan")
    pools.v[at[1][0], 1, 5, 9] = float("inf")
    got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5).cpu().view(3, hq, d)
    assert bool(got[0, :2].isnan().all()) and torch.equal(got[0, 2:], base.cpu().view(3, hq, d)[0, 2:])
    assert bool((got[1, 2:, 9] == float("inf")).all()) and bool(got[1, :, :9].isfinite().all())
    assert torch.equal(got[2], base.cpu().view(3, hq, d)[2])


def test_attend_strides_and_rows_of_no_sequence(dev):
    """Queries, outputs, tables and pages with strides of their own, K and V pages of one buffer, rows after the last
    sequence left as they were, bounds below the true sizes."""
    from rfill import ops
    from rfill.paged import Pages
    hq, hkv, d, page, rows, lens = 8, 2, 128, 16, [2, 1], [70, 33]
    pools, table, n_pages, q = batch(hq, hkv, d, page, False, rows, lens, 2)
    want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    both = torch.stack((pools.k, pools.v), 1).to(dev)          # [pages, 2, hkv, page, d]
    pages = Pages(both[:, 0], both[:, 1])
    wide = torch.full((2, table.shape[1] + 3), 12345, dtype=torch.int32, device=dev)
    wide[:, : table.shape[1]] = table.to(dev)
    qs = torch.zeros(5, hq * d + 24, dtype=torch.bfloat16, device=dev)
    qs[:3, : hq * d] = q.to(dev)
    out = torch.full((5, hq * d + 8), 3.0, dtype=torch.bfloat16, device=dev)
    ln, cu = torch.tensor(lens, dtype=torch.int32, device=dev), offsets(rows).to(dev)
    ops.attend_paged(qs[:, : hq * d], pages, wide[:, : table.shape[1]], ln, cu, hq, d ** -0.5, 2, 70, out=out[:, : hq * d])
    check(out[:3, : hq * d], want, size, "strides")
    assert bool((out[3:] == 3).all()) and bool((out[:, hq * d:] == 3).all())
    # max_keys below the lengths: that many keys are looked at; max_rows below the rows: the first ones
    got = ops.attend_paged(q.to(dev), pages, table.to(dev), ln, cu, hq, d ** -0.5, 2, 33)
    w2, s2 = oracle_attend(pools, table, n_pages, q, rows, [33, 33], hq, d ** -0.5)
    check(got, w2, s2, "max_keys")


def test_attend_other_streams_and_graph(dev):
    """On a stream of its own, and captured: replays follow new lengths, tables, queries and pages, with the program's own
    work between them."""
    from rfill import ops
    hq, hkv, d, page = 8, 2, 128, 16
    steps = [([1, 1, 1], [300, 17, 64]), ([1, 0, 1], [411, 0, 65]), ([1, 1, 1], [2, 700, 1])]
    pool_lens = [512, 704, 80]
    table, n_pages = layout(pool_lens, page, 9)
    pools, _, _, _ = batch(hq, hkv, d, page, True, [1, 1, 1], pool_lens, 4)
    pages = pages_on(pools, dev)
    tb = table.to(dev)
    ln, cu = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    q = torch.zeros(3, hq * d, dtype=torch.bfloat16, device=dev)
    out = torch.zeros(3, hq * d, dtype=torch.bfloat16, device=dev)
    for max_keys in (704, 1 << 16):
        args = (q, pages, tb, ln, cu, hq, d ** -0.5, 1, max_keys)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.attend_paged(*args, out=out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.attend_paged(*args, out=out)
        for turn in range(2):
            for i, (rows, lens) in enumerate(steps):
                g = torch.Generator().manual_seed(10 * turn + i)
                qi = torch.randn(sum(rows), hq * d, generator=g).to(torch.bfloat16)
                q.zero_()
                q[: sum(rows)] = qi.to(dev)
                ln.copy_(torch.tensor(lens, dtype=torch.int32))
                cu.copy_(offsets(rows))
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                want, size = oracle_attend(pools, table, n_pages, qi, rows, lens, hq, d ** -0.5)
                check(out[: sum(rows)], want, size, (max_keys, turn, i))
                assert torch.equal(out, ops.attend_paged(*args, out=torch.zeros_like(out)))


def test_append_then_attend_then_read(dev):
    """As they are used together: a chunk of each sequence, then single tokens, appended and attended step by step through
    one table, then a sequence read back; both kinds of pages."""
    from rfill import ops
    from rfill.paged import Pages
    hq, hkv, d, page = 8, 2, 64, 16
    final = [75, 33, 51]
    table, n_pages = layout(final, page, 21)
    tb = table.to(dev)
    for kind in ("bf16", "mx4"):
        pages = Pages.empty(n_pages, hkv, page, d, kind, dev)
        pools = OP.Pools(n_pages, hkv, page, d, kind == "mx4")
        lens = [0, 0, 0]
        g = torch.Generator().manual_seed(3)
        for rows in ([70, 30, 0], [1, 1, 48], [1, 0, 1], [3, 2, 2]):
            lens = [n + r for n, r in zip(lens, rows)]
            T = sum(rows)
            x = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16)
            ln, cu = torch.tensor(lens, dtype=torch.int32, device=dev), offsets(rows).to(dev)
            slots, pos = ops.paged_slots(tb, ln, cu, T, pages)
            cs = ops.rope_table(pos, ops.inv_freq_default(1e4, d).to(dev))
            xd = x.to(dev)
            k, v = (xd[:, (hq + i * hkv) * d:(hq + (i + 1) * hkv) * d].unflatten(1, (hkv, d)) for i in (0, 1))
            q = ops.paged_append(k, v, slots, pages, cs=cs, q=xd[:, : hq * d])
            got = ops.attend_paged(q, pages, tb, ln, cu, hq, d ** -0.5, max(rows), max(lens))
            # the oracle on the very pages (their rows are checked above) and the device's queries
            for n in ("k", "v", "ks", "vs"):
                t = getattr(pages, n)
                setattr(pools, n, None if t is None else t.cpu())
            want, size = oracle_attend(pools, table, n_pages, q.cpu(), rows, lens, hq, d ** -0.5)
            check(got, want, size, (kind, rows))
        at = torch.arange(lens[0])
        slots = table[0, at // page].long() * page + at % page
        rk, rv = ops.paged_read(pages, slots.to(dev))
        k, v, ok = OP.keys_of(pools, table[0], lens[0], n_pages)
        assert bool(ok.all()) and torch.equal(rk.cpu().double(), k) and torch.equal(rv.cpu().double(), v)


def test_pages_past_32_bit_offsets(dev):
    """Pages more than 2^32 bytes apart: written, read and attended to."""
    from rfill import ops
    from rfill.paged import Pages
    hq, hkv, d, page, n_pages = 4, 2, 64, 16, 3
    gap = (3 << 29) + 8 * 64                                   # elements: 3 GiB from a page to the next
    buf = torch.empty(2 * gap + hkv * page * d, dtype=torch.bfloat16, device=dev)
    vbuf = torch.empty_like(buf)
    view = lambda b: b.as_strided((n_pages, hkv, page, d), (gap, page * d, d, 1))   # noqa: E731
    pages = Pages(view(buf), view(vbuf))
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(40, hkv, d, generator=g).to(torch.bfloat16) for _ in "kv")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    at = torch.arange(40)
    slots = table[0, at // page].long() * page + at % page
    ops.paged_append(k.to(dev), v.to(dev), slots.to(dev), pages)
    rk, rv = ops.paged_read(pages, slots.to(dev))
    assert torch.equal(rk.cpu(), k) and torch.equal(rv.cpu(), v)
    q = torch.randn(1, hq * d, generator=g).to(torch.bfloat16)
    want, size = OP.attend(q.view(1, hq, d), k.double(), v.double(), torch.ones(40, dtype=torch.bool), d ** -0.5)
    got = ops.attend_paged(q.to(dev), pages, table.to(dev), torch.tensor([40], dtype=torch.int32, device=dev),
                           torch.tensor([0, 1], dtype=torch.int32, device=dev), hq, d ** -0.5, 1, 40)
    check(got, want.flatten(1), size.flatten(1), "far pages")


def test_far_four_bit_pages(dev):
    """The same of 4-bit pages, codes and scales, with one row and with a chunk."""
    from rfill import ops
    from rfill.paged import Pages
    hq, hkv, d, page, n_pages = 4, 2, 64, 16, 3
    far = lambda: torch.empty(2 * (3 << 30) + 4096, dtype=torch.uint8, device=dev)   # noqa: E731  3 GiB from page to page
    view = lambda *s: far().as_strided((n_pages, *s), (3 << 30, *torch.empty(s, device="meta").stride()))   # noqa: E731
    pages = Pages(view(hkv, page, d // 2), view(hkv, page // 8, 16, 8, d // 32), view(hkv, page // 8, d // 32, 8),
                  view(hkv, page // 8, d // 32, 8))
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(40, hkv, d, generator=g).to(torch.bfloat16) for _ in "kv")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    at = torch.arange(40)
    slots = (table[0, at // page].long() * page + at % page).to(dev)
    ops.paged_append(k.to(dev), v.to(dev), slots, pages)
    rk, rv = (x.cpu().double() for x in ops.paged_read(pages, slots))
    for x, y in ((k, rk), (v, rv)):
        code, scale = OP.mx4_encode(x.float())
        assert torch.equal(OP.mx4_decode(code, scale).double(), y)
    for rows in (1, 40):
        q = torch.randn(rows, hq * d, generator=g).to(torch.bfloat16)
        want, size = OP.attend(q.view(rows, hq, d), rk, rv, torch.ones(40, dtype=torch.bool), d ** -0.5)
        got = ops.attend_paged(q.to(dev), pages, table.to(dev), torch.tensor([40], dtype=torch.int32, device=dev),
                               torch.tensor([0, rows], dtype=torch.int32, device=dev), hq, d ** -0.5, rows, 40)
        check(got, want.flatten(1), size.flatten(1), rows)


@pytest.mark.parametrize("hq,hkv,d,mx", [(6, 2, 256, False), (12, 1, 256, True), (20, 1, 256, False), (7, 1, 64, False),
                                         (40, 2, 128, True), (64, 2, 64, True), (5, 1, 128, False)])
def test_row_blocks_within_a_query(dev, hq, hkv, d, mx):
    """Groups that do not divide a block of 16, 128 or 256 query rows: blocks begin and end among a query's heads."""
    for rows, lens in (([3, 1, 7, 11], [300, 5, 1000, 64]), ([1, 1], [2100, 31]), ([60, 33], [60, 150])):
        pools, table, n_pages, q = batch(hq, hkv, d, 16, mx, rows, lens, d + hq)
        want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
        for kw in (dict(), dict(max_keys=1 << 20), dict(max_rows=1 << 20)):
            check(run(dev, pools, table, q, rows, lens, hq, d ** -0.5, **kw), want, size, (rows, kw))


@pytest.mark.parametrize("mx", [False, True])
def test_runs_over_sequences(dev, mx):
    """Runs of tiles that hold the end of one sequence, all of some and the beginning of another; a value that is NaN in one
    of them reaches that sequence's column alone."""
    hq = hkv = 32
    d, page = 64, 16
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(1, 700, (40,), generator=g).tolist()
    lens[11], lens[12], lens[20] = 5000, 1, 0
    rows = [min(n, 1) for n in lens]
    pools, table, n_pages, q = batch(hq, hkv, d, page, mx, rows, lens, 4)
    want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    check(run(dev, pools, table, q, rows, lens, hq, d ** -0.5, max_keys=1 << 20), want, size, "runs")
    at = (lens[5] - 1) % page                                  # the last token of sequence 5, head 0
    last = int(table[5, (lens[5] - 1) // page])
    if mx:
        pools.vs[last, 0, at // 8, 1, at % 8] = 255            # its second block of 32 columns
        hit = slice(32, 64)
    else:
        pools.v[last, 0, at, 7] = float("nan")
        hit = slice(7, 8)
    got = run(dev, pools, table, q, rows, lens, hq, d ** -0.5, max_keys=1 << 20).cpu()
    row = sum(rows[:5])
    assert bool(got[row, hit].isnan().all())
    got[row, hit], want[row, hit] = 0, 0
    check(got, want, size, "with a NaN")


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("max_rows", [3, 200])
def test_sizes_that_contradict_each_other(dev, mx, max_rows):
    """Offsets that fall, lengths below zero and past the table, pages that are none: rows of sound sequences stay right."""
    from rfill import ops
    hq, hkv, d, page = 8, 2, 128, 16
    pools, table, n_pages, q = batch(hq, hkv, d, page, mx, [3, 1, 1], [50, 20, 33], 9)
    want, size = oracle_attend(pools, table, n_pages, q[:3], [3], [50], hq, d ** -0.5)
    t = torch.cat((table, table.flip(0)))[:5].contiguous()
    t[3:] = torch.tensor(1 << 30)
    pages = pages_on(pools, dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    for keys in (64, 1 << 20):
        lens, cu = i32([50, -4, 1 << 30, 7, -(1 << 31)]), i32([0, 3, 3, -5, (1 << 31) - 1, 4])
        ops.attend_paged(q.to(dev), pages, t.to(dev), lens, cu, hq, d ** -0.5, max_rows, keys)
        torch.cuda.synchronize()
        slots, pos = ops.paged_slots(t.to(dev), lens, cu, 5, pages)
        assert bool(((slots >= -1) & (slots < n_pages * page)).all())
        cu = i32([0, 3, 3, 3, 3, 3])
        got = ops.attend_paged(q.to(dev), pages, t.to(dev), lens, cu, hq, d ** -0.5, max_rows, keys)
        check(got[:3], want, size, keys)


def test_many_sequences(dev):
    """More sequences than a wave looks at at once, most of them empty."""
    hq, hkv, d, page = 4, 2, 64, 16
    g = torch.Generator().manual_seed(6)
    lens = [int(n) if i % 3 else 0 for i, n in enumerate(torch.randint(1, 60, (150,), generator=g))]
    rows = [min(1 + i % 2, n) for i, n in enumerate(lens)]
    pools, table, n_pages, q = batch(hq, hkv, d, page, True, rows, lens, 8)
    want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    for kw in (dict(), dict(max_keys=1 << 18)):
        check(run(dev, pools, table, q, rows, lens, hq, d ** -0.5, **kw), want, size, kw)


def test_refusals(dev):
    from rfill import ops
    from rfill._lib import UnsupportedArchitecture
    from rfill.paged import Pages
    with pytest.raises(ValueError):
        Pages.empty(4, 2, 24, 64, "bf16", dev)
    with pytest.raises(UnsupportedArchitecture):
        Pages.empty(4, 2, 16, 96, "mx4", dev)
    with pytest.raises(ValueError):
        Pages.empty(4, 2, 16, 64, "int4", dev)
    p = Pages.empty(4, 2, 16, 64, "mx4", dev)
    with pytest.raises(ValueError):
        Pages(p.k, p.v)
    with pytest.raises(ValueError):
        Pages(p.k, p.v.transpose(3, 4), p.ks, p.vs)
    with pytest.raises(ValueError):
        Pages(p.k.cpu(), p.v, p.ks, p.vs)
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=dev)   # noqa: E731
    k, slots = z(3, 2, 64), z(3, t=torch.int64)
    with pytest.raises(ValueError):
        ops.paged_append(z(3, 1, 64), k, slots, p)
    with pytest.raises(ValueError):
        ops.paged_append(k, k, slots[:2], p)
    with pytest.raises(ValueError):
        ops.paged_append(k, k, slots.int(), p)
    with pytest.raises(ValueError):
        ops.paged_append(k, k, slots, p, qnorm=z(64))
    with pytest.raises(ValueError):
        ops.paged_append(k, k, slots, p, knorm=z(64), norm_kind=2)
    with pytest.raises(UnsupportedArchitecture):
        ops.paged_append(k, k, slots, p, cs=z(3, 12))
    with pytest.raises(UnsupportedArchitecture):
        ops.paged_append(k, k, slots, p, cs=z(3, 128))
    with pytest.raises(ValueError):
        ops.paged_append(z(4, 2, 65)[:3, :, 1:], k, slots, p)
    with pytest.raises(ValueError):
        ops.paged_append(k.cpu(), k, slots, p)
    table, ln, cu = z(2, 3, t=torch.int32), z(2, t=torch.int32), z(3, t=torch.int32)
    with pytest.raises(ValueError):
        ops.attend_paged(z(3, 256), p, table, ln[:1], cu, 4, 0.1, 1, 10)
    with pytest.raises(ValueError):
        ops.attend_paged(z(3, 128), p, table, ln, cu, 4, 0.1, 1, 10)
    with pytest.raises(UnsupportedArchitecture):
        ops.attend_paged(z(3, 192), p, table, ln, cu, 3, 0.1, 1, 10)
    with pytest.raises(UnsupportedArchitecture):
        ops.attend_paged(z(3, 130 * 64), p, table, ln, cu, 130, 0.1, 1, 10)
    with pytest.raises(ValueError):
        ops.attend_paged(z(3, 256), p, table, ln, cu, 4, 0.0, 1, 10)
    with pytest.raises(ValueError):
        ops.attend_paged(z(3, 256), p, table.long(), ln, cu, 4, 0.1, 1, 10)
    with pytest.raises(ValueError):
        ops.paged_read(p, slots, k_out=z(2, 2, 64))
    # nothing to do
    assert ops.attend_paged(z(0, 256), p, table, ln, cu, 4, 0.1, 1, 10).shape == (0, 256)
    assert ops.paged_read(p, slots[:0])[0].shape == (0, 2, 64)
    ops.paged_append(k[:0], k[:0], slots[:0], p)
    torch.cuda.synchronize()


def test_expanded_tensors_are_refused(dev):
    """Rows that share memory (expand): a stride below a row's width is refused, never read past; one row may have any."""
    from rfill import ops
    from rfill.paged import Pages
    p = Pages.empty(4, 2, 16, 64, "bf16", dev)
    bf = dict(dtype=torch.bfloat16, device=dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
    slots, kv = torch.arange(3, device=dev), torch.ones(3, 2, 64, **bf)
    table, lens, cu = i32([[0], [1], [2]]), i32([4, 4, 4]), i32([0, 1, 2, 3])
    q = torch.ones(3, 256, **bf)
    attend = lambda q=q, table=table, **kw: ops.attend_paged(q, p, table, lens, cu, 4, 0.1, 1, 16, **kw)   # noqa: E731
    append = lambda k=kv, v=kv, **kw: ops.paged_append(k, v, slots, p, **kw)   # noqa: E731
    append(q=q)
    attend()
    for call in (lambda: attend(q=q[:1].expand(3, -1)), lambda: attend(table=table[:1].expand(3, -1)[:, :1].repeat(1, 2)[:1].expand(3, -1)),
                 lambda: attend(out=torch.empty(1, 256, **bf).expand(3, -1)), lambda: append(k=kv[:1].expand(3, -1, -1)),
                 lambda: append(v=kv[:, :1].expand(-1, 2, -1)), lambda: append(q=q[:1].expand(3, -1)),
                 lambda: append(q=q, out=torch.empty(1, 256, **bf).expand(3, -1)),
                 lambda: ops.paged_read(p, slots, k_out=torch.empty(1, 2, 64, **bf).expand(3, -1, -1)),
                 lambda: ops.paged_slots(table[:1].expand(3, -1), lens, cu, 3, p)):
        with pytest.raises(ValueError):
            call()
    one = torch.empty(1, 512, **bf)[:, ::2]
    with pytest.raises(ValueError):
        ops.attend_paged(one, p, table[:1], lens[:1], cu[:2], 4, 0.1, 1, 16)       # last dim not contiguous


@pytest.mark.parametrize("mx", [False, True])
def test_two_graphs_on_one_workspace(dev, mx):
    """A step (slots, append, attention) of few rows and one of a chunk, captured apart over the same pages and the same
    workspace, replayed in turn; then both kinds at once on two streams with a workspace each."""
    from rfill import ops
    hq, hkv, d, page = 8, 2, 128, 16
    lens0 = [3000, 40, 1200]
    table, n_pages = layout([n + 400 for n in lens0], page, 12)
    pools, _, _, _ = batch(hq, hkv, d, page, mx, [1, 1, 1], [n + 400 for n in lens0], 13)
    pages, tb = pages_on(pools, dev), table.to(dev)
    g = torch.Generator().manual_seed(14)
    inv = ops.inv_freq_default(1e4, d).to(dev)
    keys = 1 << 14
    steps = []
    for rows in ([1, 1, 1], [90, 40, 130]):
        T = sum(rows)
        x = torch.randn(T, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16).to(dev)
        lens = torch.tensor([n + r for n, r in zip(lens0, rows)], dtype=torch.int32, device=dev)
        steps.append(dict(rows=rows, T=T, x=x, lens=lens, cu=offsets(rows).to(dev)))
    need = max(ops.attend_paged_workspace_bytes(s["T"], hq, hkv, d, pages.kind, 3, max(s["rows"]), keys) for s in steps)
    shared = torch.empty(need, dtype=torch.uint8, device=dev)

    def step(s, ws):
        slots, pos = ops.paged_slots(tb, s["lens"], s["cu"], s["T"], pages)
        k, v = (s["x"][:, (hq + i * hkv) * d:(hq + (i + 1) * hkv) * d].unflatten(1, (hkv, d)) for i in (0, 1))
        q = ops.paged_append(k, v, slots, pages, cs=ops.rope_table(pos, inv), q=s["x"][:, : hq * d])
        return q, ops.attend_paged(q, pages, tb, s["lens"], s["cu"], hq, d ** -0.5, max(s["rows"]), keys, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in steps:
            step(s, shared)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step(s, shared)))
    for turn in range(3):
        for s, (graph, (q, out)) in zip(steps, graphs):
            s["x"].copy_(torch.randn(s["x"].shape, generator=g).to(torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            for n in ("k", "v", "ks", "vs"):
                t = getattr(pages, n)
                setattr(pools, n, None if t is None else t.cpu())
            lens = s["lens"].tolist()
            want, size = oracle_attend(pools, table, n_pages, q.cpu(), s["rows"], lens, hq, d ** -0.5)
            check(got, want, size, (turn, s["rows"]))
            q2, eager = step(s, torch.full_like(shared, 0xff))
            assert torch.equal(q2, q) and torch.equal(eager, got)
    # at once: the pages hold the last step's rows now; both only read them
    one = [ops.attend_paged(q, pages, tb, s["lens"], s["cu"], hq, d ** -0.5, max(s["rows"]), keys) for s, (_, (q, _)) in
           zip(steps, graphs)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in steps], [None, None]
    for _ in range(3):
        for i, (s, (_, (q, _))) in enumerate(zip(steps, graphs)):
            with torch.cuda.stream(streams[i]):
                outs[i] = ops.attend_paged(q, pages, tb, s["lens"], s["cu"], hq, d ** -0.5, max(s["rows"]), keys)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], one[0]) and torch.equal(outs[1], one[1])
