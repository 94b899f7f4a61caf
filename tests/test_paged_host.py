"""The paged cache's host side without a GPU: the library's refusals (every one before a launch), the workspace rule, and
the oracle's 4-bit form against hand values."""
import ctypes

import pytest
import torch

from oracle import paged as OP


def _pages(**kw):
    from rfill import _lib
    p = dict(k=1 << 20, v=2 << 20, ks=3 << 20, vs=4 << 20, n_pages=8, page_stride=2 * 16 * 64, scale_stride=2 * 16 * 2, kind=1,
             hkv=2, d=64, page=16)
    p.update(kw)
    return _lib.RfPages(**p)


def _append(pages, **kw):
    from rfill import _lib
    a = dict(k=1 << 20, ld_k=128, head_k=64, v=1 << 20, ld_v=128, head_v=64, T=0, slots=1 << 20, cs=None, rot=0, q=None, ld_q=0,
             hq=0, q_out=None, ld_qo=0, qnorm=None, knorm=None, kind=0, eps=0.0)
    a.update(kw)
    _lib.call("rf_paged_append", a["k"], a["ld_k"], a["head_k"], a["v"], a["ld_v"], a["head_v"], a["T"], a["slots"],
              ctypes.byref(pages) if pages else None, a["cs"], a["rot"], a["q"], a["ld_q"], a["hq"], a["q_out"], a["ld_qo"],
              a["qnorm"], a["knorm"], a["kind"], a["eps"], None)


def _attend(pages, **kw):
    from rfill import _lib
    a = dict(q=1 << 20, ldq=256, T=0, hq=4, table=1 << 20, ldt=4, width=4, lens=1 << 20, cu=1 << 20, n=2, rows=1, keys=64,
             scale=0.125, out=1 << 20, ldo=256, ws=None, wb=0)
    a.update(kw)
    _lib.call("rf_attend_paged", a["q"], a["ldq"], a["T"], a["hq"], ctypes.byref(pages), a["table"], a["ldt"], a["width"],
              a["lens"], a["cu"], a["n"], a["rows"], a["keys"], a["scale"], a["out"], a["ldo"], a["ws"], a["wb"], None)


def test_bad_pages_are_refused():
    from rfill._lib import UnsupportedArchitecture
    _append(_pages())                                          # no rows: accepted, nothing launched
    _append(_pages(kind=0, page_stride=2 * 16 * 128, ks=None, vs=None))
    for bad in (dict(page=24), dict(page=8), dict(page=2048), dict(kind=2), dict(k=None), dict(ks=None), dict(vs=None),
                dict(n_pages=0), dict(n_pages=1 << 31), dict(hkv=0), dict(page_stride=2 * 16 * 32 - 16),
                dict(page_stride=2 * 16 * 32 + 8), dict(scale_stride=2 * 16 * 2 - 8), dict(scale_stride=2 * 16 * 2 + 4),
                dict(k=(1 << 20) + 8), dict(vs=(1 << 20) + 4)):
        for call in (_append, _attend):
            with pytest.raises(ValueError):
                call(_pages(**bad))
    with pytest.raises(UnsupportedArchitecture):
        _append(_pages(d=96))
    with pytest.raises(ValueError):
        _append(None)


def test_bad_appends_are_refused():
    from rfill._lib import UnsupportedArchitecture
    for bad in (dict(k=None), dict(slots=None), dict(T=-1), dict(ld_k=124), dict(head_k=56), dict(head_v=68), dict(q=1 << 20),
                dict(hq=4), dict(q=1 << 20, hq=4, ld_q=256, ld_qo=256), dict(q=1 << 20, hq=4, ld_q=248, q_out=1 << 20, ld_qo=256),
                dict(knorm=1 << 20, kind=2), dict(qnorm=1 << 20), dict(eps=-1.0), dict(eps=float("nan")), dict(k=(1 << 20) + 8),
                dict(cs=(1 << 20) + 8, rot=64)):
        with pytest.raises(ValueError):
            _append(_pages(), **bad)
    for rot in (0, 12, 20, 63, 66, 128):
        with pytest.raises(UnsupportedArchitecture):
            _append(_pages(), cs=1 << 20, rot=rot)
    for rot in (8, 16, 48, 64):
        _append(_pages(), cs=1 << 20, rot=rot)


def test_bad_attention_is_refused():
    from rfill._lib import UnsupportedArchitecture
    _attend(_pages())
    for bad in (dict(q=None), dict(lens=None), dict(cu=None), dict(table=None), dict(out=None), dict(T=-1), dict(ldq=252),
                dict(ldq=248), dict(ldo=255), dict(width=-1), dict(ldt=3), dict(n=-1), dict(rows=-1), dict(keys=-1),
                dict(keys=(1 << 27) + 1), dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=(1 << 20) + 8),
                dict(out=(1 << 20) + 4), dict(ws=(1 << 20) + 8)):
        with pytest.raises(ValueError):
            _attend(_pages(), **bad)
    for hq in (0, 3, 130):
        with pytest.raises(UnsupportedArchitecture):
            _attend(_pages(), hq=hq, ldq=8192 * 2, ldo=8192 * 2)


def test_bad_slots_and_reads_are_refused():
    from rfill import _lib
    p = 1 << 20

    def slots(table=p, ld=4, width=4, lens=p, cu=p, n=2, pages=8, page=16, T=0, out=p):
        _lib.call("rf_paged_slots", table, ld, width, lens, cu, n, pages, page, T, out, out, None)

    slots()
    for bad in (dict(table=None), dict(lens=None), dict(cu=None), dict(out=None), dict(ld=3), dict(width=-1), dict(n=-1),
                dict(page=24), dict(T=-1), dict(T=1 << 31), dict(pages=-1)):
        with pytest.raises(ValueError):
            slots(**bad)

    def read(pages=None, at=p, T=0, k=p, lk=128, v=p, lv=128):
        _lib.call("rf_paged_read", ctypes.byref(pages or _pages()), at, T, k, lk, v, lv, None)

    read()
    for bad in (dict(at=None), dict(k=None), dict(lk=120), dict(lv=132), dict(v=p + 8), dict(T=-1), dict(pages=_pages(page=20))):
        with pytest.raises(ValueError):
            read(**bad)


def test_workspace_rule():
    """Nothing for short sequences; room for one round of parts for few rows a sequence, whatever their number; for chunks it
    grows with the rows."""
    from rfill import ops
    f = ops.attend_paged_workspace_bytes
    assert f(1, 32, 8, 128, 0, 1, 1, 500) == 0
    one, many = f(1, 32, 8, 128, 0, 1, 1, 100000), f(64, 32, 8, 128, 0, 64, 1, 100000)
    assert 0 < one == many < (1 << 28)
    assert many < f(2048, 32, 8, 128, 0, 1, 2048, 100000) < f(16384, 32, 8, 128, 0, 8, 2048, 100000) < (1 << 32)
    assert f(0, 32, 8, 128, 0, 4, 1, 100000) == 0
    with pytest.raises(ValueError):
        f(1, 32, 7, 128, 0, 1, 1, 500)


def test_oracle_four_bit_values():
    """Levels, halfway cases to the even code, the scale's step at 7 / 4, zeros, infinities."""
    x = torch.zeros(1, 32)
    x[0, :12] = torch.tensor([6.0, 5.0, 4.99, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 0.26, -0.25, -7.0])
    c, b = OP.mx4_encode(x)
    assert int(b) == 127 and c[0, :12].tolist() == [7, 6, 6, 6, 4, 4, 2, 2, 0, 1, 8, 15]
    x[0, 0] = 7.01
    assert int(OP.mx4_encode(x)[1]) == 128
    z, b = OP.mx4_encode(torch.zeros(1, 64))
    assert b.tolist() == [[1, 1]] and int(z.sum()) == 0
    x[0, 3] = float("inf")
    c, b = OP.mx4_encode(x)
    assert int(b) == 255 and bool(OP.mx4_decode(c, b).isnan().all())


class _Stub:
    """What PagedCache asks of a model; GDN layers alone need no pools on a GPU."""
    n_layers, n_kv, head_dim, layer_types, device = 2, 1, 64, ["gdn", "gdn"], torch.device("cpu")
    W = [dict(kind="gdn"), dict(kind="gdn")]

    def new_cache(self):
        return [dict() for _ in range(self.n_layers)]


def test_page_accounting():
    """Pages come and go with the sequences; a plan that cannot be met or is malformed changes nothing."""
    from rfill.paged import PagedCache
    c = PagedCache(_Stub(), 10, page=16)
    a, b = c.add(), c.add()
    step = c.plan([a, b], [17, 16])
    assert c.free_pages == 7 and c.tokens(a) == 17 and step.rows == 33 and step.max_rows == 17 and step.max_keys == 17
    assert step.cu.tolist() == [0, 17, 33] and step.lens.tolist() == [17, 16]
    assert step.table.tolist() == [[0, 1], [2, -1]]
    step = c.plan([b], [1])
    assert step.table.tolist() == [[2, 3]] and step.lens.tolist() == [17] and step.max_rows == 1
    for seqs, counts, error in (([a, b], [100, 100], MemoryError), ([a, a], [1, 1], ValueError), ([a], [0], ValueError),
                                ([a], [1, 1], ValueError), ([], [], ValueError), ([a, 99], [1, 1], KeyError)):
        with pytest.raises(error):
            c.plan(seqs, counts)
        assert c.free_pages == 6 and c.tokens(a) == c.tokens(b) == 17
    c.remove(a)
    assert c.free_pages == 8 and a not in c and b in c
    with pytest.raises(KeyError):
        c.tokens(a)
    state = dict(conv=torch.zeros(3, 8), rec=torch.ones(1, 4, 4), len=20)
    d = c.add([dict(state), dict(state)])
    assert c.tokens(d) == 20 and c.free_pages == 6 and d not in (a, b)
    c.states(d, 0)["rec"].zero_()
    assert float(state["rec"].sum()) == 16                    # the sequence has states of its own
    with pytest.raises(ValueError):
        c.add([dict(state), dict(state, len=21)])
    with pytest.raises(MemoryError):
        c.add([dict(state, len=200), dict(state, len=200)])
    with pytest.raises(KeyError):
        c.add([dict(len=20), dict(len=20)])                    # no states: its pages are given back
    assert c.free_pages == 6
