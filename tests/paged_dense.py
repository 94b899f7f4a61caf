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
