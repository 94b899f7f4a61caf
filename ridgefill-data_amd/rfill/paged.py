"""A paged K / V cache for several sequences: answering from filled caches, a token or a chunk at a time.

Pages: the pools of one layer as the kernels read them (ops.paged_append, paged_read, attend_paged), in bfloat16 or in 4
bits (17 / 32 byte a value: E2M1 codes with a power-of-two scale for each 32 values; include/rfill.h has the layout).
PagedCache: the pages of every attention layer of a FillModel and the states of its GDN layers, for sequences that come
(empty, or with a cache that finish() or forward_exact() filled), grow (plan(), then FillModel.layer_paged of each layer;
FillModel.forward_paged does both) and go. Tokens that a cheaper model drafted, in a row or as trees, grow a sequence at once
and are then cut to those that were accepted (plan(parents=), accept(); FillModel.verify_paged does it all).
"""
import ctypes
from dataclasses import dataclass, field

import torch

from . import _lib, ops

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
        want, dev = torch.bfloat16 if self.kind == BF16 else torch.uint8, k.get_device()
        for name, t in parts:
            if t.dtype != want:
                raise ValueError(f"Pages: {name} dtype {t.dtype}, expected {want}")
            if not t.is_cuda or t.get_device() != dev:
                raise ValueError(f"Pages: {name} must be on k's GPU (got {t.device})")
            if not (t.is_contiguous() or t[0].is_contiguous()):
                raise ValueError(f"Pages: {name} must be contiguous within a page")
        size = 2 if self.kind == BF16 else 1
        strides = [(t.stride(0) if self.n_pages > 1 else t[0].numel()) * size for _, t in parts]
        if strides[0] != strides[1] or strides[2:3] != strides[3:]:
            raise ValueError(f"Pages: strides between pages {strides} bytes differ")
        self.k, self.v, self.ks, self.vs = k, v, ks, vs
        self.form = (self.kind, self.hkv, self.d, self.page, dev)
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


@dataclass
class Step:
    """New tokens of several sequences (PagedCache.plan): sequence b's rows are [cu[b], cu[b + 1]) and become its last
    tokens. On the device: table (its pages), lens (its tokens with them), cu, and of each row the slot, the position and
    the RoPE table row. moved: the sequences whose GDN states have taken rows of it. Trees: seen, the bits of the new rows that
    each row sees (ops.paged_tree), the positions by depth, and on the host parents, a list for each sequence. mark: what its
    sequences hold as long as it is their last plan; before: what they held until then."""
    seqs: list
    counts: list
    table: torch.Tensor
    lens: torch.Tensor
    cu: torch.Tensor
    slots: torch.Tensor
    pos: torch.Tensor
    cs: torch.Tensor
    max_rows: int
    max_keys: int
    ends: list = None                       # tokens of each sequence with the new ones
    moved: set = field(default_factory=set)
    seen: torch.Tensor = None
    parents: list = None
    mark: object = None
    before: list = None

    @property
    def rows(self):
        return sum(self.counts)


class _Sequence:
    def __init__(self):
        self.tokens = 0
        self.pages = []
        self.states = {}                    # GDN layers: conv, rec (own tensors, updated in place)
        self.lost = False                   # a step failed after its GDN states had moved (undo)
        self.mark = None                    # Step.mark of the last plan, of which tokens may go back (None: of none)


class PagedCache:
    """n_pages pages of `page` tokens (kind "bf16" or "mx4") in every packed attention layer of model; a page number means
    the same tokens in each of them. Sequences are named by the integers that add() returns."""

    def __init__(self, model, n_pages, page=64, kind="bf16"):
        self.model, self.page, self.kind = model, page, kind
        self.layers = [i for i in range(model.n_layers) if model.W[i] is not None]
        self.pools = {i: Pages.empty(n_pages, model.n_kv, page, model.head_dim, kind, model.device)
                      for i in self.layers if model.layer_types[i] == "attn"}
        self.n_pages = n_pages
        self._free = list(range(n_pages - 1, -1, -1))
        self._seqs = {}
        self._next = 0

    def __contains__(self, seq):
        return seq in self._seqs

    @property
    def free_pages(self):
        return len(self._free)

    def nbytes(self):
        return sum(p.nbytes() for p in self.pools.values())

    def _of(self, seq):
        if seq not in self._seqs:
            raise KeyError(f"no sequence {seq!r} in this cache")
        if self._seqs[seq].lost:
            raise RuntimeError(f"sequence {seq!r} was lost in a step that failed: remove() it")
        return self._seqs[seq]

    def tokens(self, seq):
        return self._of(seq).tokens

    def states(self, seq, i):
        """GDN layer i's states of the sequence (conv and rec; None before its first token)."""
        return self._of(seq).states.setdefault(i, dict(conv=None, rec=None))

    def add(self, cache=None):
        """A new sequence, empty or with the tokens of `cache` (one dict a layer, as FillModel.new_cache: every packed
        layer filled with as many tokens): K and V are copied into pages, in 4 bits rounded. Returns its name."""
        s = _Sequence()
        n = 0
        if cache is not None:
            counts = {i: cache[i].get("n" if self.model.layer_types[i] == "attn" else "len", 0) for i in self.layers}
            n = max(counts.values(), default=0)
            if any(c != n for c in counts.values()):
                raise ValueError(f"add: the cache's layers hold {sorted(set(counts.values()))} tokens")
        self._grow([(s, n)])
        if n:
            try:
                step = self._step([s], [n])
                for i in self.layers:
                    c = cache[i]
                    if i in self.pools:
                        ops.paged_append(c["kbuf"][:, :n].transpose(0, 1), c["vbuf"][:, :n].transpose(0, 1), step.slots,
                                         self.pools[i])
                    else:
                        s.states[i] = dict(conv=c["conv"].clone(), rec=c["rec"].float().contiguous().clone())
            except Exception:
                self._free += reversed(s.pages)
                raise
        name = self._next
        self._next += 1
        self._seqs[name] = s
        return name

    def remove(self, seq):
        """Forget a sequence; its pages are free for the next plan() or add(). (Work that reads them must have been queued
        on the stream that writes them next.)"""
        s = self._seqs[seq] if seq in self._seqs else self._of(seq)
        del self._seqs[seq]
        self._free += reversed(s.pages)

    def plan(self, seqs, counts, parents=None):
        """Room for counts[b] new tokens of each sequence seqs[b]: the Step that layer_paged of every layer takes. The
        sequences count the tokens from now on; undo() takes that back. Raises MemoryError when the pages do not suffice.
        Nothing is changed when it raises.
        parents: the new tokens are nodes of trees, parents[b][i] the place among the sequence's new ones of the token that
        token i follows (an earlier one; -1: it follows the tokens before the new ones). A token sees those above it, and its
        position is its depth's. GDN layers take their rows in order: UnsupportedArchitecture."""
        if len(seqs) != len(counts) or not len(seqs):
            raise ValueError(f"plan: {len(seqs)} sequences, {len(counts)} counts")
        if len(set(seqs)) != len(seqs):
            raise ValueError("plan: a sequence is named twice")
        if any(int(c) < 1 for c in counts):
            raise ValueError(f"plan: counts {list(counts)} (at least one token each)")
        ss, counts = [self._of(q) for q in seqs], [int(c) for c in counts]
        trees = ()
        if parents is not None:
            self._all_attention("trees of new tokens")
            parents = [[int(p) for p in x] for x in parents]
            if [len(x) for x in parents] != counts:
                raise ValueError(f"plan: parents of {[len(x) for x in parents]} tokens, counts {counts}")
            if any(not -1 <= p < i for x in parents for i, p in enumerate(x)):
                raise ValueError("plan: a token's parent is an earlier one of its sequence's new tokens, or -1")
            trees = (parents,)
        self._grow(list(zip(ss, counts)))
        try:
            step = self._step(ss, counts, list(seqs), *trees)
        except BaseException:
            self._shrink(list(zip(ss, counts)))
            raise
        step.mark, step.before = object(), [s.mark for s in ss]
        for s in ss:
            s.mark = step.mark
        return step

    def _last(self, step, what):
        """The step's sequences, if it is the last plan of each and none of its tokens have gone back or were kept yet. (Their
        counts would not tell: another plan may have brought them to the same ones, on other pages.)"""
        ss = [self._of(q) for q in step.seqs]
        if step.mark is None or any(s.mark is not step.mark for s in ss):
            raise ValueError(f"{what}: not the last plan of its sequences")
        return ss

    def undo(self, step):
        """Take back a plan() whose rows did not get through every layer, the last one of its sequences: they lose its tokens,
        and the pages that it took are free again. (remove()'s note on queued work holds.) A sequence whose GDN states have
        taken rows of the step cannot go back and is lost: every call on it but remove() raises RuntimeError."""
        ss = self._last(step, "undo")
        self._shrink([(s, n) for q, s, n in zip(step.seqs, ss, step.counts) if q not in step.moved])
        for q, s, mark in zip(step.seqs, ss, step.before):
            s.lost, s.mark = q in step.moved, mark

    def accept(self, step, path, count):
        """Keep of each sequence's new tokens those on a path: of a plan() whose rows are through every layer, the last one of
        its sequences, token path[b, j] becomes the j-th new one for j < count[b], in every layer's pages (path int32 [n,
        depth], count int32 [n] on the device, as ops.verify_drafts gives them). The sequences lose the others, and pages
        without tokens are free again (remove()'s note on queued work holds). A path goes from a token without a parent down,
        a child each; of a plan() without parents it is the first tokens. Returns the paths as lists; a step is accepted once.
        Nothing is changed when it raises."""
        self._all_attention("dropping tokens")
        ss = self._last(step, "accept")
        ops._need(path, "path", torch.int32, 2)
        ops._need(count, "count", torch.int32, 1)
        if path.shape[0] != len(ss) or count.shape[0] != len(ss):
            raise ValueError(f"accept: path {tuple(path.shape)}, count {tuple(count.shape)} of {len(ss)} sequences")
        kept = []
        for n, b, row in zip(step.counts, range(len(ss)), torch.cat((count[:, None], path), 1).tolist()):
            m, row = row[0], row[1:]
            above = range(-1, n - 1) if step.parents is None else step.parents[b]
            if not 0 <= m <= min(n, len(row)) or any(not 0 <= i < n or above[i] != (row[j - 1] if j else -1)
                                                     for j, i in enumerate(row[:m])):
                raise ValueError(f"accept: {m} tokens {row[:max(0, m)]} of {n} new ones are no path")
            kept.append(row[:m])
        if self.pools and any(i != j for row in kept for j, i in enumerate(row)):
            ops.paged_keep(list(self.pools.values()), step.table, step.lens, step.cu, path, count)
        self._shrink([(s, n - len(row)) for s, n, row in zip(ss, step.counts, kept)])
        for s, row, mark in zip(ss, kept, step.before):
            s.mark = None if row else mark
        return kept

    def _all_attention(self, what):
        if any(self.model.layer_types[i] != "attn" for i in self.layers):
            raise _lib.UnsupportedArchitecture(f"{what}: GDN layers take their rows in order, and none back")

    def _grow(self, wants):
        need = [-(-(s.tokens + n) // self.page) - len(s.pages) for s, n in wants]
        if sum(need) > len(self._free):
            raise MemoryError(f"{sum(need)} pages wanted, {len(self._free)} of {self.n_pages} free")
        for (s, n), m in zip(wants, need):
            s.pages += [self._free.pop() for _ in range(m)]
            s.tokens += n

    def _shrink(self, wants):               # _grow taken back
        for s, n in reversed(wants):
            s.tokens -= n
            keep = -(-s.tokens // self.page)
            self._free += reversed(s.pages[keep:])
            del s.pages[keep:]

    def _step(self, ss, counts, seqs=None, parents=None):
        dev = self.model.device
        width = max(1, max(len(s.pages) for s in ss))
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)   # noqa: E731
        table = i32([s.pages + [-1] * (width - len(s.pages)) for s in ss])
        lens, cu = i32([s.tokens for s in ss]), i32(cu)
        slots = pos = cs = seen = None
        if self.pools:                      # (GDN layers alone: no slots)
            pool = next(iter(self.pools.values()))
            if parents is None:
                slots, pos = ops.paged_slots(table, lens, cu, sum(counts), pool)
            else:
                slots, pos, seen = ops.paged_tree(table, lens, cu, i32([p for x in parents for p in x]), sum(counts), pool,
                                                  max(counts))
            cs = self.model.rope_table(pos)
        ends = [s.tokens for s in ss]
        return Step(seqs, counts, table, lens, cu, slots, pos, cs, max(counts), max(ends), ends, seen=seen, parents=parents)

    def read(self, seq):
        """The sequence's cache as FillModel.new_cache lays it out (bf16 buffers of its own; of 4-bit pages what they hold). The
        rows of a plan() must have run through the layers."""
        s = self._of(seq)
        out = self.model.new_cache()
        step = self._step([s], [s.tokens]) if s.tokens else None
        for i in self.layers:
            if step is None:
                continue
            if i in self.pools:
                c, n = out[i], s.tokens
                self.model.reserve(c, n, self.model.n_kv, self.model.head_dim, self.model.device)
                k, v = ops.paged_read(self.pools[i], step.slots)
                c["kbuf"][:, :n].copy_(k.transpose(0, 1))
                c["vbuf"][:, :n].copy_(v.transpose(0, 1))
                self.model.commit(c, n)
            else:
                st = self.states(seq, i)
                if st["conv"] is None or st["rec"] is None:
                    raise RuntimeError(f"read: the planned tokens of sequence {seq!r} have not run through layer {i}")
                out[i].update(conv=st["conv"].clone(), rec=st["rec"].clone(), len=s.tokens)
        return out
