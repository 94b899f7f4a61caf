"""FillModel.verify_paged refuses what verification cannot take before any layer runs, and the sequences are as they were."""
import pytest
import torch

from test_gpu_drafts_model import _ids, _model, dev      # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


def test_refused_before_the_layers(dev, monkeypatch):                                      # noqa: F811
    from rfill import ops
    from rfill._lib import UnsupportedArchitecture
    from rfill.paged import PagedCache
    cfg, m = _model("llama_c1", dev)
    cache = PagedCache(m, 100, page=16)
    seqs = [cache.add() for _ in range(2)]
    m.forward_paged(cache, seqs, _ids(1, (30, 61)))
    ids, tree = _ids(2, (4, 3)), [[-1, 0, 0, 1], [-1, 0, 1]]
    state = list(cache._free), [(s.tokens, list(s.pages), s.mark) for s in cache._seqs.values()]
    z = lambda *n, t=torch.float32, d=dev: torch.zeros(*n, dtype=t, device=d)              # noqa: E731

    def runs(*args, **kw):
        raise AssertionError("a layer ran")

    with monkeypatch.context() as mp:
        mp.setattr(m, "layer_paged", runs)
        mp.setattr(ops, "attend_tree", runs)
        for bad in (dict(u=z(6)), dict(u=z(7, t=torch.float64)), dict(u=z(7, d="cpu")), dict(u=z(7, 1)), dict(r=z(3)), dict(r=z(2, d="cpu")),
                    dict(r=z(2, t=torch.bfloat16)), dict(draft=z(7, 63)), dict(draft=z(6, 64)), dict(draft=z(7, 64, t=torch.float16)),
                    dict(draft=z(7, 64, d="cpu")), dict(draft=z(64, 7).t()), dict(draft=z(1, 64).expand(7, 64))):
            with pytest.raises(ValueError):
                m.verify_paged(cache, seqs, ids, tree, temperature=1.0, **bad)
        for long in ([0] * 1025, list(range(1025))):
            with pytest.raises(UnsupportedArchitecture, match="1025 rows"):
                m.verify_paged(cache, seqs[:1], [[1] * 1025], [[-1] + long[:1024]] if long[1] == 0 else None)
        assert state == (list(cache._free), [(s.tokens, list(s.pages), s.mark) for s in cache._seqs.values()])
    u = z(7)
    accepted, after = m.verify_paged(cache, seqs, ids, tree, temperature=1.0, u=u, r=z(2), draft=z(7, 64, t=torch.bfloat16))
    assert len(accepted) == 2 and len(after) == 2
    # as many rows as there may be, in a row and as a star
    for parents in (None, [[-1] + [0] * 1023]):
        n = cache.tokens(seqs[0])
        accepted, _ = m.verify_paged(cache, seqs[:1], _ids(5, (1024,)), parents)
        assert cache.tokens(seqs[0]) == n + 1 + len(accepted[0])
