"""The paged cache under a FillModel: exact layers of new tokens of several sequences (FillModel.layer_paged, forward_paged)
against FillModel.layer of each sequence alone over its contiguous cache, which other tests hold against the oracle.

Bars: a layer's output is within 1e-2 (relative Frobenius) of the oracle's and its update (output - input) within 2e-2 there;
two such outputs are within the sum, 2e-2 and 4e-2. With 4-bit pages the contiguous cache holds what the pages hold, read
back, so that the bars stay the same."""
import pytest
import torch

from fill_cases import case, hybrid_config, hybrid_tensors, inputs, rel_err

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
    if name == "hybrid":
        cfg = hybrid_config(["gdn", "attn", "gdn", "attn"])
        return cfg, FillModel(cfg, hybrid_tensors(cfg, seed=9), dev)
    cfg, t = case(name, layers=layers)
    return cfg, FillModel(cfg, t, dev)


def _close(got, want, h, what):
    err, ed = rel_err(got, want), rel_err(got.float() - h.float(), want.float() - h.float())
    print(f"{what}: out {err:.2e}, update {ed:.2e}")
    return err < TOL and ed < 2 * TOL


@pytest.mark.parametrize("name", ["llama_c1", "llama3_scaled", "qwen3_knorm", "qwen35_attn", "hybrid"])
def test_layers_of_several_sequences(dev, name):
    """Filled prompts of several lengths and an empty sequence; then a step of a chunk, a token and a few tokens, and one of a
    token each: every layer's output per sequence against layer() alone, and the pages' rows against its cache."""
    from rfill.paged import PagedCache
    cfg, m = _model(name, dev)
    H = cfg["hidden_size"]
    lens = [150, 0, 33]
    prompts = [inputs(n, H, seed=60 + n).to(dev) for n in lens]
    alone = [m.new_cache() for _ in lens]
    for c, h in zip(alone, prompts):
        for i in range(m.n_layers):
            if h.shape[0]:
                h, _ = m.layer(i, h, torch.arange(h.shape[0], device=dev), c)
    cache = PagedCache(m, 40, page=16)
    seqs = [cache.add(c if n else None) for c, n in zip(alone, lens)]
    assert [cache.tokens(s) for s in seqs] == lens and cache.free_pages == 40 - 10 - 3
    ok = True
    for counts in ([1, 40, 5], [1, 1, 1]):
        step = cache.plan(seqs, counts)
        h = inputs(sum(counts), H, seed=70 + sum(counts)).to(dev)
        ssq = None
        for i in range(m.n_layers):
            out, ssq = m.layer_paged(i, h, step, cache, ssq=ssq)
            r = 0
            for b, n in enumerate(counts):
                p0 = cache.tokens(seqs[b]) - n
                want, _ = m.layer(i, h[r:r + n], torch.arange(p0, p0 + n, device=dev), alone[b])
                ok &= _close(out[r:r + n], want, h[r:r + n], f"{name} layer {i} sequence {b}")
                r += n
            h = out
    assert ok
    for b, s in enumerate(seqs):
        back = cache.read(s)
        for i in range(m.n_layers):
            if m.layer_types[i] == "attn":
                assert back[i]["n"] == alone[b][i]["n"]
                assert rel_err(back[i]["k"], alone[b][i]["k"]) < TOL and rel_err(back[i]["v"], alone[b][i]["v"]) < TOL
                n = lens[b]                                    # the rows that add() brought are bit for bit the filled ones
                assert torch.equal(back[i]["k"][:, :n], alone[b][i]["k"][:, :n])
            else:
                assert rel_err(back[i]["rec"], alone[b][i]["rec"]) < TOL


@pytest.mark.parametrize("name", ["llama3_scaled", "qwen35_attn"])
def test_four_bit_pages(dev, name):
    """layer_paged over 4-bit pages against the layer's own steps over what the pages hold after it."""
    from rfill import ops
    from rfill.paged import PagedCache
    cfg, m = _model(name, dev, layers=1)
    H = cfg["hidden_size"]
    w = m._pack_rows(0)
    cache = PagedCache(m, 60, page=32, kind="mx4")
    seqs, lens = [], [300, 77]
    for n in lens:
        c = m.new_cache()
        m.fill(0, inputs(n, H, seed=n).to(dev), torch.arange(n, device=dev), c)
        seqs.append(cache.add(c))
        # in units of the block's scale the largest value a lies in (3.5, 7], levels 4 and 6 are 2 apart and those below 4 at
        # most 1: a value v is off by at most 1 / 2 below 4 (a / 7), by v - 4 <= v / 5 up to 5, by 1 <= v / 5 from there on
        back, amax = cache.read(seqs[-1])[0], c[0]["v"].unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).float()
        off = (back["v"].float() - c[0]["v"].float()).unflatten(-1, (-1, 32)).abs()
        assert bool((off <= amax / 5 * (1 + 2 ** -20)).all())
    counts = [1, 6]
    step = cache.plan(seqs, counts)
    h = inputs(7, H, seed=5).to(dev)
    ssq = ops.row_ssq(h)
    got, _ = m.layer_paged(0, h, step, cache)
    ok, r = True, 0
    for b, n in enumerate(counts):
        c = cache.read(seqs[b])[0]
        assert c["n"] == lens[b] + n
        x, s = h[r:r + n], ssq[r:r + n]
        pos = torch.arange(lens[b], lens[b] + n, device=dev)
        q = ops.norm_q(x, s, m.eps, w["wq"], m.n_heads, m.head_dim, w.get("q_norm"), m.knorm_kind, m.rope_table(pos),
                       torch.arange(n, device=dev))
        o = ops.attend_rows(q, pos, c["kbuf"], c["vbuf"], c["n"], m.n_heads, m.scale)
        want = m._out_mlp(w, x, m._gate(w, x, s, o))[0]
        ok &= _close(got[r:r + n], want, x, f"{name} sequence {b}")
        r += n
    assert ok


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_finish_then_answer(dev, kind):
    """A prompt filled by finish() moves into the paged cache beside another one and both answer: late layers only."""
    from rfill.kva import Arm, finish
    from rfill.model import FillModel
    from rfill.paged import PagedCache
    cfg, t = case("llama_c1", layers=4)
    m = FillModel(cfg, t, dev, layers=[2, 3])
    H = cfg["hidden_size"]
    cache = PagedCache(m, 64, page=16, kind=kind)
    caches, seqs = [], []
    for n in (301, 120):
        h = inputs(n, H, seed=n).to(dev)
        _, c, _ = finish(m, torch.zeros(n, dtype=torch.long), h, None, Arm("id", split=2, tail=40, fill="identity"), 1)
        seqs.append(cache.add(c))
        caches.append(c if kind == "bf16" else cache.read(seqs[-1]))
    ok = True
    for turn in range(3):
        step = cache.plan(seqs, [1, 1])
        h = inputs(2, H, seed=80 + turn).to(dev)
        for i in (2, 3):
            out, _ = m.layer_paged(i, h, step, cache)
            for b in (0, 1):
                if kind == "mx4":                              # what the pages hold, the new row included
                    continue
                p = cache.tokens(seqs[b]) - 1
                want, _ = m.layer(i, h[b:b + 1], torch.tensor([p], device=dev), caches[b])
                ok &= _close(out[b:b + 1], want, h[b:b + 1], f"turn {turn} layer {i} sequence {b}")
            assert bool(torch.isfinite(out.float()).all())
            h = out
    assert ok
    free = cache.free_pages
    cache.remove(seqs[0])
    assert cache.free_pages == free + 19 and seqs[0] not in cache     # 304 tokens in pages of 16
    again = cache.add(caches[1])                               # its pages hold old rows: only the new ones count
    k = cache.read(again)[2]["k"]
    assert kind == "mx4" or torch.equal(k, caches[1][2]["k"])
    with pytest.raises(KeyError):
        cache.plan([seqs[0]], [1])


def test_forward_paged(dev):
    """Whole models: prompts in one call, then tokens, give forward_exact's logits; the same calls give the same bits."""
    from rfill.model import FillModel
    from rfill.paged import PagedCache
    cfg = hybrid_config(["gdn", "attn", "gdn", "attn"])
    m = FillModel(cfg, hybrid_tensors(cfg, seed=2), dev)
    g = torch.Generator().manual_seed(1)
    ids = [torch.randint(0, 64, (n,), generator=g) for n in (90, 41, 64)]
    runs = []
    for _ in range(2):
        cache = PagedCache(m, 64, page=16)
        seqs = [cache.add() for _ in ids]
        first = m.forward_paged(cache, seqs, [x[:-2] for x in ids])
        m.forward_paged(cache, seqs[::-1], [x[-2:-1] for x in ids[::-1]])
        runs.append((first, m.forward_paged(cache, seqs, [x[-1:] for x in ids])))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    ok = True
    for b, x in enumerate(ids):
        n = x.numel()
        want, _ = m.forward_exact(x, keep=[n - 3, n - 1])
        for got, y in ((runs[0][0][b], want[0]), (runs[0][1][b], want[1])):
            err = rel_err(got, y)
            print(f"sequence {b}: logits {err:.2e}")
            # the layers' outputs differ by up to 2e-2 each from the same input, four of them
            ok &= err < 4 * TOL
    assert ok
    with pytest.raises(ValueError):
        m.forward_paged(cache, seqs, [x[:0] for x in ids])
    with pytest.raises(ValueError):
        m.forward_paged(cache, [seqs[0], seqs[0]], [ids[0], ids[1]])
    assert cache.tokens(seqs[0]) == 90
