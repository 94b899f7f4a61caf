"""The paged cache in float64, from the definitions: 4-bit blocks, page layouts, norm and rotation of new rows, causal
attention of several sequences. Slow and plain (loops over rows and sequences); CPU tensors."""
import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mx4_encode(x):
    """Codes (uint8, one a value) and scale bytes of x [..., d]: blocks of 32 along d. With 2^n <= a < 2^(n + 1) for a
    block's largest magnitude a the scale is 2^(n - 2), or 2^(n - 1) when a > 1.75 2^n; the byte is clamped to [1, 254],
    255 for a block with a NaN or an infinity (codes 0). Codes: the nearest level, halfway to the even code, at most 6."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    a = b.abs().amax(-1)
    fine = torch.isfinite(b).all(-1)
    m, e = torch.frexp(torch.where(fine, a, 1.0))              # a = m 2^e, 0.5 <= m < 1
    byte = torch.where(a == 0, 1, (e - 1 - 2 + (m > 0.875).long() + 127).clamp(1, 254))
    y = torch.where(fine[..., None], b, 0.0) * torch.exp2(127.0 - byte.double())[..., None]
    lv = torch.tensor(LEVELS, dtype=torch.float64)
    mid = (lv[1:] + lv[:-1]) / 2
    t = y.abs()
    c = (t[..., None] > mid).sum(-1)                           # halfway: the lower code ...
    tie = (t[..., None] == mid).any(-1)
    c = torch.where(tie & (c % 2 == 1), c + 1, c)              # ... unless the upper one is even
    neg = torch.signbit(y)
    code = torch.where(fine[..., None], c + 8 * neg, 0).to(torch.uint8)
    return code.reshape(x.shape), torch.where(fine, byte, 255).to(torch.uint8)


def mx4_decode(code, byte):
    """float64 values of codes [..., d] with scale bytes [..., d / 32]."""
    lv = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64)
    sc = torch.where(byte == 255, float("nan"), torch.exp2(byte.double() - 127))
    return lv[code.long()] * sc.repeat_interleave(32, -1)


class Pools:
    """One layer's pages on the CPU in the library's layout."""

    def __init__(self, n_pages, hkv, page, d, mx):
        self.page, self.hkv, self.d, self.mx = page, hkv, d, mx
        if mx:
            z = lambda *s: torch.zeros(n_pages, hkv, *s, dtype=torch.uint8)   # noqa: E731
            self.k, self.v = z(page, d // 2), z(page // 8, 16, 8, d // 32)
            self.ks, self.vs = z(page // 8, d // 32, 8), z(page // 8, d // 32, 8)
        else:
            self.k, self.v = (torch.zeros(n_pages, hkv, page, d, dtype=torch.bfloat16) for _ in range(2))
            self.ks = self.vs = None

    def write(self, slot, k, v):
        """Row k, v [hkv, d] (float64; bf16 pages round them) into a slot."""
        p, t = slot // self.page, slot % self.page
        if not self.mx:
            self.k[p, :, t], self.v[p, :, t] = k.to(torch.bfloat16), v.to(torch.bfloat16)
            return
        (kc, kb), (vc, vb) = mx4_encode(k), mx4_encode(v)
        self.k[p, :, t] = kc[:, 0::2] | (kc[:, 1::2] << 4)
        self.v[p, :, t // 8, :, t % 8] = (vc[:, 0::2] | (vc[:, 1::2] << 4)).view(self.hkv, 16, -1)
        self.ks[p, :, t // 8, :, t % 8], self.vs[p, :, t // 8, :, t % 8] = kb, vb

    def read(self, slot):
        """K, V [hkv, d] float64 at a slot."""
        p, t = slot // self.page, slot % self.page
        if not self.mx:
            return self.k[p, :, t].double(), self.v[p, :, t].double()
        out = []
        for c, b in ((self.k[p, :, t], self.ks[p, :, t // 8, :, t % 8]),
                     (self.v[p, :, t // 8, :, t % 8].reshape(self.hkv, -1), self.vs[p, :, t // 8, :, t % 8])):
            out.append(mx4_decode(torch.stack((c & 15, c >> 4), -1).reshape(self.hkv, -1), b))
        return out


def rows(x, gain=None, kind=0, eps=0.0, cs=None):
    """x [rows, heads, d] normed per head (x / rms (gain or 1 + gain)) and its first cs.shape[1] dims rotated by halves."""
    x = x.double()
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (gain.double() + kind)
    if cs is None:
        return x
    h = cs.shape[1] // 2
    c, s = cs[:, None, :h].double(), cs[:, None, h:].double()
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * h:]), -1)


def keys_of(pools, table, length, n_pages):
    """K, V [length, hkv, d] float64 of one sequence and which of its keys lie on pages of the pool."""
    k = torch.zeros(length, pools.hkv, pools.d, dtype=torch.float64)
    v, ok = torch.zeros_like(k), torch.zeros(length, dtype=torch.bool)
    for j in range(length):
        pg = int(table[j // pools.page])
        if 0 <= pg < n_pages:
            k[j], v[j] = pools.read(pg * pools.page + j % pools.page)
            ok[j] = True
    return k, v, ok


def attend(q, k, v, ok, scale):
    """q [rows, hq, d]: the last rows of a sequence with keys k, v [length, hkv, d], of which ok are there. Returns the
    outputs [rows, hq, d] and sum_j p_j |v_j| of each (what the rounding of the probabilities is relative to)."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    size = torch.zeros_like(out)
    for i in range(n):
        see = torch.arange(length)[ok & (torch.arange(length) <= length - n + i)]
        if not len(see):
            continue
        for h in range(hq):
            kk, vv = k[see, h // (hq // hkv)], v[see, h // (hq // hkv)]
            p = torch.softmax(kk @ q[i, h].double() * scale, 0)
            out[i, h] = p @ vv
            size[i, h] = p @ vv.abs()
    return out, size
