"""Steps of the paged cache that are no longer their sequences' last ones, on the host: accept() and undo() refuse them, whatever
the sequences count by now."""
import pytest
import torch

from test_drafts_host import _cache, _i32, _state


def _refused(c, step, path, count):
    before = _state(c)
    with pytest.raises(ValueError, match="last plan"):
        c.accept(step, _i32(path), _i32(count))
    with pytest.raises(ValueError, match="last plan"):
        c.undo(step)
    assert _state(c) == before


def test_a_step_that_was_undone(monkeypatch):
    """Another plan of the same size, on pages that an other sequence has taken meanwhile: the first step's table is stale."""
    c = _cache(monkeypatch)
    a, b = c.add(), c.add()
    c.plan([a], [14])
    first = c.plan([a], [5], [[-1, 0, 0, 1, 2]])
    c.undo(first)
    c.plan([b], [3])
    again = c.plan([a], [5], [[-1, 0, 1, 2, 3]])
    assert first.ends == again.ends and first.table.tolist() != again.table.tolist()
    _refused(c, first, [[0, 2, 4]], [3])
    assert c.accept(again, _i32([[0, 1, 2]]), _i32([3])) == [[0, 1, 2]] and c.tokens(a) == 17


def test_a_step_that_was_accepted(monkeypatch):
    """All rows, some of them with as many planned again, none: a step is accepted once."""
    c = _cache(monkeypatch)
    a, b = c.add(), c.add()
    step = c.plan([a, b], [3, 2])
    assert c.accept(step, _i32([[0, 1, 2], [0, 1, -1]]), _i32([3, 2])) == [[0, 1, 2], [0, 1]]
    assert c.tokens(a) == 3 and c.tokens(b) == 2
    _refused(c, step, [[0, 1, 2], [0, 1, -1]], [3, 2])
    step = c.plan([b, a], [4, 4])
    c.accept(step, _i32([[0], [0]]), _i32([1, 1]))
    later = c.plan([a, b], [3, 3])
    assert [c.tokens(q) for q in step.seqs] == step.ends
    _refused(c, step, [[0], [0]], [1, 1])
    c.accept(later, _i32([[0], [0]]), _i32([0, 0]))
    _refused(c, later, [[0], [0]], [0, 0])


def test_steps_in_turn(monkeypatch):
    """A step that is taken back, or of which nothing was kept, leaves the one before it the last; one of another cache never is."""
    c = _cache(monkeypatch)
    a, b = c.add(), c.add()
    first = c.plan([a], [5])
    second = c.plan([a, b], [2, 1])
    with pytest.raises(ValueError):
        c.undo(first)
    c.undo(second)
    third = c.plan([b, a], [1, 3])
    assert c.accept(third, _i32([[0], [0]]), _i32([0, 0])) == [[], []] and c.tokens(a) == 5
    fourth = c.plan([a], [4])
    assert c.accept(fourth, _i32([[0, 1]]), _i32([2])) == [[0, 1]]
    with pytest.raises(ValueError):
        c.undo(first)                                          # (tokens behind it were kept)
    other = _cache(monkeypatch)
    x = other.add()
    theirs = other.plan([x], [7])
    assert x == a and other.tokens(x) == c.tokens(a)
    with pytest.raises(ValueError, match="last plan"):
        c.undo(theirs)
    e = c.add()
    last = c.plan([e], [4])
    c.undo(last)
    assert c.tokens(e) == 0
    with pytest.raises(ValueError, match="last plan"):
        c.undo(last)


def test_a_plan_that_raises_leaves_the_last_one(monkeypatch):
    c = _cache(monkeypatch)
    a = c.add()
    step = c.plan([a], [5])
    with pytest.raises(MemoryError):
        c.plan([a], [1000])
    with monkeypatch.context() as m:
        m.setattr(c, "_step", lambda *args: (_ for _ in ()).throw(RuntimeError()))
        with pytest.raises(RuntimeError):
            c.plan([a], [2])
    with pytest.raises(ValueError):
        c.accept(step, _i32([[1]]), _i32([1]))                 # no path: nothing is changed
    c.undo(step)
    assert c.tokens(a) == 0 and c.free_pages == 12
    assert torch.is_tensor(step.table)
