"""Drafted tokens on the paged cache's host side, without a GPU: plans of trees and what they refuse, the tokens and pages of
sequences of which a path is kept."""
import pytest
import torch

from test_paged_host import _Stub


class _Attention(_Stub):
    """No packed layers: the cache counts tokens and pages, the pools are elsewhere."""
    layer_types, W = ["attn", "attn"], [None, None]


def _cache(monkeypatch, stub=_Attention, pages=12):
    from rfill import ops
    from rfill.paged import PagedCache
    monkeypatch.setattr(ops, "_need", lambda t, *a: None)      # (tensors of this test are on the host)
    return PagedCache(stub(), pages, page=16)


def _state(c):
    return (list(c._free), {q: (s.tokens, list(s.pages)) for q, s in c._seqs.items()})


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_plans_of_trees(monkeypatch):
    c = _cache(monkeypatch)
    a, b = c.add(), c.add()
    c.plan([a], [17])
    before = _state(c)
    for parents in ([[-1, 0]], [[-1, 0], [-1]], [[-1, 1, 0], [-1]], [[0, 0, 1], [-1]], [[-1, 0, -2], [-1]], [[-1, 0, 3], [-1]]):
        with pytest.raises(ValueError):
            c.plan([a, b], [3, 1], parents)
        assert _state(c) == before
    with pytest.raises(MemoryError):
        c.plan([a, b], [3, 200], [[-1, 0, 0], list(range(-1, 199))])
    assert _state(c) == before
    step = c.plan([a, b], [3, 2], [[-1, 0, 0], torch.tensor([-1, -1])])
    assert step.parents == [[-1, 0, 0], [-1, -1]] and step.ends == [20, 2] and c.plan([a], [1]).parents is None


def test_gdn_layers_refuse_trees_and_drops(monkeypatch):
    from rfill._lib import UnsupportedArchitecture
    c = _cache(monkeypatch, _Stub)
    a = c.add()
    before = _state(c)
    with pytest.raises(UnsupportedArchitecture):
        c.plan([a], [2], [[-1, 0]])
    assert _state(c) == before
    step = c.plan([a], [3])
    with pytest.raises(UnsupportedArchitecture):
        c.accept(step, _i32([[0]]), _i32([1]))
    assert c.tokens(a) == 3


def test_accept(monkeypatch):
    """The sequences keep their paths' tokens; pages behind them are free; what is no path changes nothing."""
    c = _cache(monkeypatch)
    a, b = c.add(), c.add()
    first = c.plan([a, b], [15, 16])
    step = c.plan([b, a], [20, 4], [list(range(-1, 19)), [-1, 0, 0, 2]])
    assert c.free_pages == 12 - 2 - 3
    before = _state(c)
    for path, count in (([[0, 1], [0, 3]], [2, 2]), ([[0, 1], [1, 2]], [2, 2]), ([[0, 2], [0, 2]], [2, 2]),
                        ([[0, 20], [0, 2]], [2, 1]), ([[0, -1], [0, 2]], [2, 2]), ([[0, 1], [0, 2]], [3, 1]),
                        ([[0, 1], [0, 2]], [-1, 1]), ([[0, 1]], [2, 2]), ([[0, 1], [0, 2]], [1])):
        with pytest.raises(ValueError):
            c.accept(step, _i32(path), _i32(count))
        assert _state(c) == before
    with pytest.raises(ValueError):
        c.accept(first, _i32([[0], [0]]), _i32([1, 1]))        # not their last plan
    assert c.accept(step, _i32([[0, -1, -1], [0, 2, 3]]), _i32([1, 3])) == [[0], [0, 2, 3]]
    assert c.tokens(b) == 17 and c.tokens(a) == 18 and c.free_pages == 12 - 4
    with pytest.raises(ValueError):
        c.accept(step, _i32([[0], [0]]), _i32([1, 1]))
    with pytest.raises(ValueError):
        c.undo(step)
    row = c.plan([a], [5])
    assert c.accept(row, _i32([[0, 1, 9]]), _i32([2])) == [[0, 1]] and c.tokens(a) == 20
    row = c.plan([a], [30])
    with pytest.raises(ValueError):
        c.accept(row, _i32([[0, 2]]), _i32([2]))               # a row of tokens, of which one was left out
    assert c.accept(row, _i32([[0]]), _i32([0])) == [[]] and c.tokens(a) == 20 and c.free_pages == 12 - 4


def test_keep_refuses_the_same_pages_twice():
    """In the library, before any launch: two blocks would move the same rows at once."""
    import ctypes
    from rfill import _lib
    from test_paged_host import _pages
    pages = [_pages(), _pages(k=5 << 20), _pages()]
    for which, n in ((pages, 0), (pages[:2], 1)):
        handles = (ctypes.c_void_p * len(which))(*(ctypes.addressof(p) for p in which))
        if n:                                                  # others: accepted, and of no sequences nothing is launched
            _lib.call("rf_paged_keep", handles, len(which), 1 << 20, 4, 4, 1 << 20, 1 << 20, 0, 1 << 20, 3, 3, 1 << 20, None)
            continue
        with pytest.raises(ValueError, match="same pages"):
            _lib.call("rf_paged_keep", handles, len(which), 1 << 20, 4, 4, 1 << 20, 1 << 20, 0, 1 << 20, 3, 3, 1 << 20, None)
