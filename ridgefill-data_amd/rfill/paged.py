"""A paged K / V cache for several sequences: answering from filled caches, a token or a chunk at a time.

Pages: the pools of one layer as the kernels read them (ops.paged_append, paged_read, attend_paged), in bfloat16 or in 4
bits (17 / 32 byte a value: E2M1 codes with a power-of-two scale for each 32 values; include/rfill.h has the layout).
"""
import ctypes

import torch

from . import _lib

BF16, MX4 = 0, 1                        # kinds of pages (RF_PAGES_BF16, RF_PAGES_MX4)
KINDS = {"bf16": BF16, "mx4": MX4}


class Pages:
    """The pages of one layer. bf16: k, v [pages, hkv, page, d]. 4 bits: k [pages, hkv, page, d / 2], v [pages, hkv,
    page / 8, 16, 8, d / 32], ks, vs [pages, hkv, page / 8, d / 32, 8], all uint8. The tensors may be views with a stride
    of their own between pages (K and V of one buffer), contiguous within a page."""

    def __init__(self, k, v, ks=None, vs=None):
        if not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor):
            raise TypeError("Pages: k and v are tensors")
        if k.dtype == torch.bfloat16:
            if ks is not None or vs is not None:
                raise ValueError("Pages: bfloat16 pages have no scales")
            self.kind = BF16
            if k.dim() != 4 or k.shape != v.shape:
                raise ValueError(f"Pages: k {tuple(k.shape)}, v {tuple(v.shape)}, expected [pages, hkv, page, d] both")
            self.n_pages, self.hkv, self.page, self.d = k.shape
            parts = [("k", k), ("v", v)]
        else:
            self.kind = MX4
            if k.dim() != 4:
                raise ValueError(f"Pages: k {tuple(k.shape)}, expected [pages, hkv, page, d / 2]")
            self.n_pages, self.hkv, self.page, self.d = *k.shape[:3], 2 * k.shape[3]
            n, h, p8, g = self.n_pages, self.hkv, self.page // 8, self.d // 32
            for name, t, shape in (("v", v, (n, h, p8, 16, 8, g)), ("ks", ks, (n, h, p8, g, 8)), ("vs", vs, (n, h, p8, g, 8))):
                if t is None or tuple(t.shape) != shape:
                    raise ValueError(f"Pages: {name} {None if t is None else tuple(t.shape)}, expected {shape}")
            parts = [("k", k), ("v", v), ("ks", ks), ("vs", vs)]
        if self.n_pages == 0:
            raise ValueError("Pages: no pages")
        for name, t in parts:
            want = torch.bfloat16 if self.kind == BF16 else torch.uint8
            if t.dtype != want:
                raise ValueError(f"Pages: {name} dtype {t.dtype}, expected {want}")
            if t.device.type != "cuda" or t.device != k.device:
                raise ValueError(f"Pages: {name} must be on k's GPU (got {t.device})")
            if not t[0].is_contiguous():
                raise ValueError(f"Pages: {name} must be contiguous within a page")
        strides = [(t.stride(0) if self.n_pages > 1 else t[0].numel()) * t.element_size() for _, t in parts]
        if strides[0] != strides[1] or strides[2:3] != strides[3:]:
            raise ValueError(f"Pages: strides between pages {strides} bytes differ")
        self.k, self.v, self.ks, self.vs = k, v, ks, vs
        self._struct = _lib.RfPages(k.data_ptr(), v.data_ptr(), ks.data_ptr() if ks is not None else None,
                                    vs.data_ptr() if vs is not None else None, self.n_pages, strides[0],
                                    strides[2] if ks is not None else 0, self.kind, self.hkv, self.d, self.page)
        self.handle = ctypes.addressof(self._struct)

    @classmethod
    def empty(cls, n_pages, hkv, page, d, kind="bf16", device="cuda"):
        """New pools of n_pages pages of `page` tokens, hkv heads of d values; kind "bf16" or "mx4"."""
        if kind not in KINDS:
            raise ValueError(f"kind {kind!r} of pages (bf16, mx4)")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError(f"{page} tokens a page (a power of two from 16 to 1024)")
        if d not in (64, 128, 256):
            raise _lib.UnsupportedArchitecture(f"head_dim {d} (the kernels take 64, 128, 256)")
        if kind == "bf16":
            return cls(*(torch.zeros(n_pages, hkv, page, d, dtype=torch.bfloat16, device=device) for _ in range(2)))
        u8 = lambda *s: torch.zeros(n_pages, hkv, *s, dtype=torch.uint8, device=device)   # noqa: E731
        return cls(u8(page, d // 2), u8(page // 8, 16, 8, d // 32), u8(page // 8, d // 32, 8), u8(page // 8, d // 32, 8))

    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.ks, self.vs) if t is not None)
