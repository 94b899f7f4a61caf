"""Steps of the paged cache that fail, without a GPU: a plan whose tensors cannot be made, a layer that raises. The sequences
keep the tokens and pages they had; those whose GDN states moved are lost and say so."""
from types import SimpleNamespace

import pytest
import torch

from test_paged_host import _Stub


def _cache(pages=12):
    from rfill.paged import PagedCache
    return PagedCache(_Stub(), pages, page=16)


def _state(c):
    return (list(c._free), {q: (s.tokens, list(s.pages)) for q, s in c._seqs.items()})


def test_a_plan_that_raises_changes_nothing(monkeypatch):
    c = _cache()
    a, b = c.add(), c.add()
    c.plan([a, b], [17, 5])
    before = _state(c)

    def fails(*args):
        raise RuntimeError("no memory")

    with monkeypatch.context() as m:
        m.setattr(c, "_step", fails)
        with pytest.raises(RuntimeError, match="no memory"):
            c.plan([b, a], [40, 33])
    assert _state(c) == before
    assert c.plan([b, a], [40, 33]).ends == [45, 50]


def test_undo():
    c = _cache()
    a, b, d = c.add(), c.add(), c.add()
    first = c.plan([a, b], [17, 16])
    before = _state(c)
    step = c.plan([b, a, d], [1, 15, 40])
    with pytest.raises(ValueError):
        c.undo(first)                                          # not the last plan of a and b
    assert c.tokens(a) == 32
    c.undo(step)
    assert _state(c) == before and c.tokens(d) == 0
    with pytest.raises(ValueError):
        c.undo(step)                                           # taken back already
    again = c.plan([b, a, d], [1, 15, 40])
    assert again.table.tolist() == step.table.tolist() and again.ends == [17, 32, 40]


def test_lost_sequences():
    """Sequences whose states took rows of a step that failed: only remove() takes them; the others go back."""
    c = _cache()
    a, b = c.add(), c.add()
    c.plan([a, b], [17, 16])
    free = c.free_pages
    step = c.plan([a, b], [30, 1])
    step.moved.add(a)
    c.undo(step)
    assert c.tokens(b) == 16 and a in c
    for call in (lambda: c.tokens(a), lambda: c.plan([a], [1]), lambda: c.read(a), lambda: c.states(a, 0),
                 lambda: c.plan([b, a], [1, 1])):
        with pytest.raises(RuntimeError, match="lost"):
            call()
    assert c.tokens(b) == 16 and c.free_pages == free - 1      # (a: 47 tokens in three pages)
    c.remove(a)
    assert a not in c and c.free_pages == free + 2
    with pytest.raises(KeyError):
        c.remove(a)


def test_read_before_the_layers_ran():
    c = _cache()
    a = c.add()
    c.plan([a], [3])
    with pytest.raises(RuntimeError, match="not run"):
        c.read(a)


@pytest.mark.parametrize("moved", [(), (1,)])
@pytest.mark.parametrize("where", ["layer", "logits"])
def test_forward_paged_takes_its_step_back(where, moved):
    """FillModel.forward_paged over layers of its own that raise after the first one."""
    from rfill.model import FillModel
    from rfill.paged import PagedCache
    stub = _Stub()

    def layer_paged(i, h, step, cache, ssq=None):
        step.moved |= {step.seqs[j] for j in moved}
        if i == 1 and where == "layer":
            raise MemoryError("workspace")
        return h, ssq

    def embed(ids):
        return torch.zeros(ids.numel(), 4), torch.zeros(ids.numel(), 1)

    c = PagedCache(stub, 12, page=16)
    a, b = c.add(), c.add()
    c.plan([a, b], [17, 16])
    before = _state(c)
    # (on the CPU the gather of the last rows raises by itself)
    model = SimpleNamespace(n_layers=2, device=stub.device, embed=embed, layer_paged=layer_paged, logits=None)
    c.model = model
    with pytest.raises((MemoryError, ValueError, TypeError)):
        FillModel.forward_paged(model, c, [a, b], [[1, 2, 3], list(range(20))])
    if not moved:
        assert _state(c) == before
    else:
        assert c.tokens(a) == 17
        with pytest.raises(RuntimeError, match="lost"):
            c.tokens(b)
