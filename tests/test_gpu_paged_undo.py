"""A step of forward_paged that raises in a layer, on the GPU: given the same tokens again, the sequences answer as ones that
never saw the failure, bit for bit; hybrid sequences whose GDN states moved are lost, the cache's others are not."""
import pytest
import torch

from fill_cases import case, hybrid_config, hybrid_tensors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from rfill import _lib
    _lib.load()
    return torch.device("cuda")


class _Fails(Exception):
    pass


def _fail_in(monkeypatch, m, layer):
    """Layer `layer` of m raises before it attends (its workspace cannot be had, say)."""
    whole = m.layer_paged

    def layer_paged(i, *args, **kw):
        if i == layer:
            raise _Fails
        return whole(i, *args, **kw)

    monkeypatch.setattr(m, "layer_paged", layer_paged)


def _ids(seed, counts, vocab=64):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in counts]


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_a_failed_step_leaves_no_trace(dev, monkeypatch, kind):
    """Prompts, a step that fails in the last layer (the first ones have written their rows), other tokens, then the step's."""
    from rfill.model import FillModel
    from rfill.paged import PagedCache
    cfg = hybrid_config(["attn"] * 3)
    m = FillModel(cfg, hybrid_tensors(cfg, seed=4), dev)
    prompts, other, more = _ids(1, (30, 61)), _ids(2, (20, 3)), _ids(3, (1, 5))
    runs = []
    for fails in (False, True):
        cache = PagedCache(m, 32, page=16, kind=kind)
        seqs = [cache.add() for _ in prompts]
        m.forward_paged(cache, seqs, prompts)
        if fails:
            free, list0 = cache.free_pages, list(cache._free)
            with monkeypatch.context() as mp:
                _fail_in(mp, m, 2)
                with pytest.raises(_Fails):
                    m.forward_paged(cache, seqs, other)
            assert [cache.tokens(s) for s in seqs] == [30, 61] and cache.free_pages == free and cache._free == list0
        first = m.forward_paged(cache, seqs, more)
        runs.append((first, m.forward_paged(cache, seqs, _ids(5, (1, 1))), [cache.read(s) for s in seqs]))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    for a, b in zip(runs[0][2], runs[1][2]):
        for x, y in zip(a, b):
            assert x["n"] == y["n"] and torch.equal(x["k"], y["k"]) and torch.equal(x["v"], y["v"])


def test_hybrid_sequences_of_a_failed_step(dev, monkeypatch):
    """A failure behind a GDN layer: the step's sequences are lost, a third one goes on; a failure before any GDN layer ran
    loses none."""
    from rfill.model import FillModel
    from rfill.paged import PagedCache
    cfg = hybrid_config(["attn", "gdn", "attn"])
    m = FillModel(cfg, hybrid_tensors(cfg, seed=6), dev)
    ids = _ids(7, (40, 17, 9))
    cache, alone = PagedCache(m, 32, page=16), PagedCache(m, 32, page=16)
    seqs = [cache.add() for _ in ids]
    m.forward_paged(cache, seqs, ids)
    with monkeypatch.context() as mp:
        _fail_in(mp, m, 1)
        with pytest.raises(_Fails):
            m.forward_paged(cache, seqs, _ids(8, (1, 1, 1)))
    assert [cache.tokens(s) for s in seqs] == [40, 17, 9]
    with monkeypatch.context() as mp:
        _fail_in(mp, m, 2)
        with pytest.raises(_Fails):
            m.forward_paged(cache, seqs[:2], _ids(9, (1, 30)))
    for s in seqs[:2]:
        with pytest.raises(RuntimeError, match="lost"):
            m.forward_paged(cache, [s, seqs[2]], _ids(10, (1, 1)))
    twin = alone.add()
    m.forward_paged(alone, [twin], ids[2:])
    last = _ids(11, (2,))
    got, want = m.forward_paged(cache, seqs[2:], last), m.forward_paged(alone, [twin], last)
    assert float((got - want).norm() / want.norm()) < 8e-2     # (test_gpu_paged_model.py's bar: one of three, and alone)
    for s in seqs[:2]:
        cache.remove(s)
    assert cache.free_pages == 32 - 1
    again = cache.add()
    m.forward_paged(cache, [again], ids[:1])
    assert cache.tokens(again) == 40
