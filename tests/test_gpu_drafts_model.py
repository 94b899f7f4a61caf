"""Drafted tokens under a FillModel: layers of a step of trees (PagedCache.plan(parents=), FillModel.layer_paged) against the same
tokens in a row, and FillModel.verify_paged against the oracle's choice from the logits that the model gave.

Bars: layer outputs as in test_gpu_paged_model.py, each within 1e-2 of the oracle's (its update within 2e-2), so two of them
within 2e-2 and 4e-2; logits behind L layers within L times 2e-2. Moved rows keep their bits."""
import pytest
import torch

from fill_cases import case, hybrid_config, hybrid_tensors, inputs, rel_err
from oracle import drafts as OD

pytestmark = pytest.mark.gpu
TOL = 2e-2


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from rfill import _lib
    _lib.load()
    return torch.device("cuda")


def _model(name, dev, layers=2):
    from rfill.model import FillModel
    cfg, t = case(name, layers=layers)
    return cfg, FillModel(cfg, t, dev)


def _ids(seed, counts, vocab=64):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in counts]


TREES = [[-1, 0, 0, 1, 2, 2, 4, 0], [-1], [-1] + [max(0, i // 2 - 1) for i in range(1, 70)]]


def _paths(parents):
    """The paths from row 0 to every row without children."""
    out = []
    for i in set(range(len(parents))) - set(parents):
        path = []
        while i >= 0:
            path.insert(0, i)
            i = parents[i]
        out.append(path)
    return out


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
@pytest.mark.parametrize("name", ["llama_c1", "llama3_scaled", "qwen3_knorm", "qwen35_attn"])
def test_layers_of_trees(dev, name, kind):
    """Every path's rows as a chunk of that path alone. In 4 bits both read what the pages hold: from the same inputs their rows
    have the same keys and values but for the products' rounding, which moves few codes: out of the bars' reach."""
    from rfill.paged import PagedCache
    cfg, m = _model(name, dev)
    cache = PagedCache(m, 60, page=16, kind=kind)
    prompts = _ids(3, (150, 20, 33))
    seqs = [cache.add() for _ in prompts]
    m.forward_paged(cache, seqs, prompts)
    counts = [len(x) for x in TREES]
    step = cache.plan(seqs, counts, TREES)
    hs, ssq = [inputs(sum(counts), cfg["hidden_size"], seed=7).to(dev)], None
    for i in range(m.n_layers):
        out, ssq = m.layer_paged(i, hs[-1], step, cache, ssq=ssq)
        hs.append(out)
    cache.undo(step)
    ok, r = True, 0
    for b, tree in enumerate(TREES):
        for path in _paths(tree)[:6]:
            rows = torch.tensor(path, device=dev) + r
            alone = cache.plan([seqs[b]], [len(path)])
            for i in range(m.n_layers):
                h = hs[i][rows].contiguous()
                want, _ = m.layer_paged(i, h, alone, cache)
                got = hs[i + 1][rows]
                err, ed = rel_err(got, want), rel_err(got.float() - h.float(), want.float() - h.float())
                ok &= err < TOL and ed < 2 * TOL
                if not ok:
                    print(f"{name} layer {i} sequence {b} path {path}: out {err:.2e}, update {ed:.2e}", flush=True)
            cache.undo(alone)
        r += len(tree)
    assert ok


class _Seen:
    """What verify_paged gave ops.verify_drafts, and the step's rows before and after they moved."""

    def __init__(self, monkeypatch, cache):
        from rfill import ops
        self.cache, verify, accept = cache, ops.verify_drafts, cache.accept

        def spy(logits, tokens, parents, cu, u, r, temperature, max_rows, **kw):
            self.args = [None if x is None else x.detach().cpu() for x in (logits, tokens, parents, cu, u, r, temperature, kw.get("draft"))]
            return verify(logits, tokens, parents, cu, u, r, temperature, max_rows, **kw)

        def watch(step, path, count):
            self.step, self.before = step, self._rows(step)
            return accept(step, path, count)

        monkeypatch.setattr(ops, "verify_drafts", spy)
        monkeypatch.setattr(cache, "accept", watch)

    def _rows(self, step):
        from rfill import ops
        return {i: ops.paged_read(p, step.slots) for i, p in self.cache.pools.items()}

    def want(self):
        logits, tokens, parents, cu, u, r, t, draft = self.args
        out = []
        for b in range(len(cu) - 1):
            s = slice(int(cu[b]), int(cu[b + 1]))
            path, nxt = OD.verify(logits[s].float(), tokens[s], parents[s].tolist(), None if u is None else u[s],
                                  None if r is None else r[b], 0.0 if t is None else float(t[b]), 1 << 20,
                                  None if draft is None else draft[s])
            out.append((path, [int(tokens[s][i]) for i in path[1:]], nxt))
        return out

    def check(self, got, lens):
        accepted, after = got
        want = self.want()
        assert accepted == [x[1] for x in want] and after == [x[2] for x in want]
        now, r = self._rows(self.step), 0
        for b, (path, _, _) in enumerate(want):
            assert self.cache.tokens(self.step.seqs[b]) == lens[b] + len(path)
            for i in now:
                for x, y in zip(now[i], self.before[i]):
                    assert torch.equal(x[r:r + len(path)], y[torch.tensor(path, device=y.device) + r])
            r += self.step.counts[b]
        return want


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
@pytest.mark.parametrize("trees", [False, True])
def test_greedy_answers(dev, monkeypatch, kind, trees):
    """Prompts, then steps of drafts of which some are the model's own next tokens: the oracle's paths, their rows' bits; and in
    bfloat16 pages a cache that got the accepted tokens one after the other holds the same and answers the same."""
    from rfill.paged import PagedCache
    cfg, m = _model("llama_c1", dev, layers=3)
    cache, plain = PagedCache(m, 64, page=16, kind=kind), PagedCache(m, 64, page=16, kind=kind)
    prompts = _ids(11, (61, 16, 130))
    seqs, twins = [cache.add() for _ in prompts], [plain.add() for _ in prompts]
    first = m.forward_paged(cache, seqs, prompts)
    m.forward_paged(plain, twins, prompts)
    roots, lens, moved, taken = first.argmax(1).tolist(), [61, 16, 130], 0, 0
    for turn in range(3):
        own = [[x] for x in roots]                             # the model's own tokens, a token at a time
        scout = PagedCache(m, 64, page=16, kind=kind)
        scouts = [scout.add(cache.read(s)) for s in seqs]
        for _ in range(4):
            for x, y in zip(own, m.forward_paged(scout, scouts, [x[-1:] for x in own]).argmax(1).tolist()):
                x.append(y)
        g, ids, parents = torch.Generator().manual_seed(turn), [], []
        for b, x in enumerate(own):
            if trees:                                          # a wrong token and its child before each right one
                row, par, last = [x[0]], [-1], 0
                for y in x[1:3 + b]:
                    row += [(y + 1 + int(torch.randint(0, 60, (1,), generator=g))) % 64, 5, y]
                    par += [last, len(row) - 3, last]
                    last = len(row) - 1
                ids.append(row)
                parents.append(par)
            else:                                              # wrong from the third token on, or not at all
                ids.append([y if i < 3 - b or b == 2 else (y + 1) % 64 for i, y in enumerate(x)])
        with monkeypatch.context() as mp:
            seen = _Seen(mp, cache)
            got = m.verify_paged(cache, seqs, ids, parents if trees else None)
            want = seen.check(got, lens)
        m.forward_paged(plain, twins, [[x] + a for x, a in zip(roots, got[0])])
        lens, roots = [n + len(p) for n, (p, _, _) in zip(lens, want)], got[1]
        taken += sum(len(a) for a in got[0])
        moved += any(i != j for p, _, _ in want for j, i in enumerate(p))
        used = sum(-(-n // 16) for n in lens)
        assert cache.free_pages == 64 - used and [cache.tokens(s) for s in seqs] == lens
    print(f"{taken} drafted tokens taken, {moved} of 3 steps moved rows")
    assert taken >= 6 and (moved > 0) == trees
    if kind == "bf16":
        for s, t in zip(seqs, twins):
            for x, y in zip(cache.read(s), plain.read(t)):
                assert x["n"] == y["n"] and rel_err(x["k"], y["k"]) < TOL * m.n_layers and rel_err(x["v"], y["v"]) < TOL * m.n_layers
        a, b = m.forward_paged(cache, seqs, [[x] for x in roots]), m.forward_paged(plain, twins, [[x] for x in roots])
        assert rel_err(a, b) < TOL * m.n_layers


@pytest.mark.parametrize("drawn", [False, True])
def test_drawn_answers(dev, monkeypatch, drawn):
    """Temperatures of each sequence, given random numbers, with and without a draft's shares."""
    from rfill.paged import PagedCache
    cfg, m = _model("qwen3_knorm", dev)
    cache = PagedCache(m, 64, page=32)
    prompts = _ids(21, (40, 9, 70))
    seqs = [cache.add() for _ in prompts]
    m.forward_paged(cache, seqs, prompts)
    lens, taken = [40, 9, 70], 0
    counts = [len(x) for x in TREES]
    for turn in range(6):                                      # (of the first turns' few random tokens none need be taken)
        g = torch.Generator().manual_seed(30 + turn)
        u, r = torch.rand(sum(counts), generator=g).to(dev), torch.rand(3, generator=g).to(dev)
        u = u if turn < 3 else u * 2 ** -6
        draft = torch.softmax(torch.randn(sum(counts), 64, generator=g), -1).to(dev) if drawn else None
        with monkeypatch.context() as mp:
            seen = _Seen(mp, cache)
            want = seen.check(m.verify_paged(cache, seqs, _ids(50 + turn, counts), TREES, [1.0, 0.0, 2.5], u, r, draft), lens)
        lens = [n + len(p) for n, (p, _, _) in zip(lens, want)]
        taken += sum(len(a) for _, a, _ in want)
    assert taken > 0
    torch.manual_seed(5)                                       # torch's random numbers: the same seed, the same answer
    step = [cache.read(s) for s in seqs]
    answers = []
    for _ in range(2):
        torch.manual_seed(5)
        again = PagedCache(m, 64, page=32)
        answers.append(m.verify_paged(again, [again.add(x) for x in step], _ids(60, (4, 4, 4)), temperature=0.7))
    assert answers[0] == answers[1]


def test_failures_leave_no_trace(dev, monkeypatch):
    """A verification that raises, and calls that are refused: tokens and pages as before, and the same answer afterwards."""
    from rfill import ops
    from rfill._lib import UnsupportedArchitecture
    from rfill.model import FillModel
    from rfill.paged import PagedCache
    cfg, m = _model("llama_c1", dev)
    prompts, ids, tree = _ids(1, (30, 61)), _ids(2, (4, 3)), [[-1, 0, 0, 1], [-1, 0, 1]]
    answers = []
    for fails in (False, True):
        cache = PagedCache(m, 32, page=16)
        seqs = [cache.add() for _ in prompts]
        m.forward_paged(cache, seqs, prompts)
        if fails:
            state = list(cache._free), [(s.tokens, list(s.pages)) for s in cache._seqs.values()]

            def raises(*args, **kw):
                raise MemoryError

            for module, name in ((ops, "verify_drafts"), (cache, "accept"), (ops, "attend_tree")):
                with monkeypatch.context() as mp:
                    mp.setattr(module, name, raises)
                    with pytest.raises(MemoryError):
                        m.verify_paged(cache, seqs, ids, tree)
            for bad in (dict(parents=[[-1, 0, 0, 1], [-1, -1, 1]]), dict(parents=[[-1, 0, 0], [-1, 0, 1]]), dict(temperature=[1.0] * 3),
                        dict(parents=[[-1, 0, 2, 1], [-1, 0, 1]]), dict(temperature=1.0, u=torch.zeros(6, device=dev)),
                        dict(temperature=1.0, draft=torch.zeros(7, 63, device=dev)), dict(temperature=1.0, r=torch.zeros(2))):
                with pytest.raises(ValueError):
                    m.verify_paged(cache, seqs, ids, **{"parents": tree, **bad})
            for q, x in (([seqs[0]] * 2, ids), (seqs, [ids[0], ids[1][:0]]), (seqs, [ids[0] + 64, ids[1]]), (seqs[:1], ids), ([], [])):
                with pytest.raises(ValueError):
                    m.verify_paged(cache, q, x)
            assert state == (list(cache._free), [(s.tokens, list(s.pages)) for s in cache._seqs.values()])
        answers.append((m.verify_paged(cache, seqs, ids, tree), [cache.read(s) for s in seqs]))
    assert answers[0][0] == answers[1][0]
    for a, b in zip(answers[0][1], answers[1][1]):
        for x, y in zip(a, b):
            assert x["n"] == y["n"] and torch.equal(x["k"], y["k"]) and torch.equal(x["v"], y["v"])
    cfg = hybrid_config(["attn", "gdn"])
    h = FillModel(cfg, hybrid_tensors(cfg, seed=1), dev)
    cache = PagedCache(h, 8, page=16)
    s = cache.add()
    with pytest.raises(UnsupportedArchitecture):
        h.verify_paged(cache, [s], [[1, 2]])
    assert cache.tokens(s) == 0 and cache.free_pages == 8
