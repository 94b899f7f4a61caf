"""A paged pool's rows and the attention over them in float64, all rows of a sequence at once (oracle.paged goes row by row;
this is for longer sequences and for values beyond bfloat16)."""
import torch

from oracle import paged as OP


def values(pools):
    """K, V [pages, hkv, page, d] float64 of the pools; values beyond bfloat16's range as the infinities they read as."""
    if not pools.mx:
        return pools.k.double(), pools.v.double()
    n, h, page, d = pools.k.shape[0], pools.hkv, pools.page, pools.d
    out = []
    for c, s in ((pools.k, pools.ks), (pools.v.transpose(3, 4).reshape(n, h, page, d // 2), pools.vs)):
        byte = s.transpose(3, 4).reshape(n, h, page, d // 32)
        out.append(OP.mx4_decode(torch.stack((c & 15, c >> 4), -1).reshape(n, h, page, d), byte).to(torch.bfloat16).double())
    return out


def attend(pools, table, n_pages, q, rows, lens, hq, scale):
    """Outputs and sum p |v| (finite values) [sum rows, hq d] of sequences with these new rows and lengths."""
    hkv, d, page = pools.hkv, pools.d, pools.page
    rep = hq // hkv
    kp, vp = values(pools)
    out, size = (torch.zeros(q.shape[0], hq, d, dtype=torch.float64) for _ in "os")
    at = 0
    for b, (r, n) in enumerate(zip(rows, lens)):
        if r and n:
            ids = table[b, torch.arange(n) // page].long()
            here = (ids >= 0) & (ids < n_pages)
            ids, tok = torch.where(here, ids, 0), torch.arange(n) % page
            see = here & (torch.arange(n) <= torch.arange(n - r, n)[:, None])          # [r, n]
            for h in range(hkv):
                k, v = kp[ids, h, tok], vp[ids, h, tok]                                   # [n, d]
                fine = v.isfinite()
                x = q[at:at + r].view(r, hq, d)[:, h * rep:(h + 1) * rep].double()
                s = (x.reshape(-1, d) @ torch.where(here[:, None], k, 0.0).T).view(r, rep, n) * scale
                s = s.masked_fill(~see[:, None], float("-inf"))
                top = s.amax(-1, keepdim=True)
                p = torch.where(see[:, None], torch.exp(s - torch.where(top == float("-inf"), 0.0, top)), 0.0)
                p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
                vf = torch.where(fine, v, 0.0)
                o, a = p @ vf, p @ vf.abs()
                if not bool(fine.all()):
                    seen = (p > 0).double()
                    up, down, nan = ((seen @ m.double()) > 0 for m in (v == float("inf"), v == float("-inf"), v.isnan()))
                    o = torch.where(up, float("inf"), torch.where(down, float("-inf"), o))
                    o = torch.where(nan | (up & down), float("nan"), o)
                out[at:at + r, h * rep:(h + 1) * rep], size[at:at + r, h * rep:(h + 1) * rep] = o, a
        at += r
    return out.flatten(1), size.flatten(1)


def pools_of(k, v, mx):
    """Pools that hold K / V [pages, hkv, page, d], rounded to bfloat16 or 4 bits."""
    n, h, page, d = k.shape
    pools = OP.Pools(n, h, page, d, mx)
    if not mx:
        pools.k, pools.v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        return pools
    (kc, kb), (vc, vb) = OP.mx4_encode(k), OP.mx4_encode(v)
    by = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)          # noqa: E731
    s8 = lambda b: b.view(n, h, page // 8, 8, d // 32).transpose(3, 4).contiguous()    # noqa: E731
    pools.k, pools.ks, pools.vs = by(kc).contiguous(), s8(kb), s8(vb)
    pools.v = by(vc).view(n, h, page // 8, 8, 16, d // 32).transpose(3, 4).contiguous()
    return pools


def telling(hq, hkv, d, page, mx, rows, lens, table, n_pages, down=False):
    """Pools and queries in which every 16 keys show. Of sequence b and K / V head h, keys 16 t .. have one value that is not
    zero, in column (t + 7 h + 3 b) % d: 1 in K, 2^(t // d) in V (down: the powers fall). Columns' scores (scale 1) are
    multiples of 1 / 8 below 8, so each output column is its own keys' weight, and 16 keys left out, taken twice, or taken
    from elsewhere change one by an eighth of a part in seven or more (up to five groups of d x 16 keys, in one of the two
    directions). What no sequence holds is far off: 1 in K's first column, 2^12 in all of V. All of it is exact in bfloat16
    and in 4 bits."""
    k, v = torch.zeros(n_pages, hkv, page, d), torch.full((n_pages, hkv, page, d), 2.0 ** 12)
    k[..., 0] = 1
    for b, n in enumerate(lens):
        j = torch.arange(n)
        ids = table[b, j // page].long()
        here = (ids >= 0) & (ids < n_pages)
        j, ids = j[here], ids[here]
        t, groups = j // 16, (n - 1) // (16 * d)
        for h in range(hkv):
            k[ids, h, j % page], v[ids, h, j % page] = 0, 0
            col = (t + 7 * h + 3 * b) % d
            k[ids, h, j % page, col] = 1
            v[ids, h, j % page, col] = torch.exp2((groups - t // d if down else t // d).float())
    g = torch.Generator().manual_seed(d + sum(rows))
    q = torch.stack([torch.randperm(d, generator=g) % 64 for _ in range(sum(rows) * hq)]) / 8
    return pools_of(k, v, mx), q.view(sum(rows), hq * d).to(torch.bfloat16)
