"""Verification without a draft's shares next to its borders: a child's test against the sum of a row's weights that are left.

The oracle decides in float64. Bounds: a weight is within 3e-12 of itself, so the two sides of u Z < w are within 1e-10 of theirs; every
random number here lies 5e-8 (relative) or more from its border (2^-24 = 6e-8 where the largest meets a last token), so paths and tokens
are equal."""
import numpy as np
import pytest
import torch

from oracle import drafts as OD
from test_gpu_drafts import dev, i32, offsets, same, verify, want_of      # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu
LOG2 = 0.6931471805599453
MOST = 1 - 2.0 ** -24                      # the largest random number below 1


def batch(rows, tokens, parents, temps, u, r):
    """Sequences of their own rows of logits."""
    return dict(x=torch.cat(rows), q=None, parents=parents, tokens=torch.cat(tokens), counts=[len(p) for p in parents],
                temp=torch.tensor(temps), u=torch.cat(u), r=torch.tensor(r))


def far(c, depth):
    """Whether every test that the oracle meets lies 5e-8 or more from its border."""
    at = 0
    for b, par in enumerate(c["parents"]):
        path = OD.verify(c["x"][at:at + len(par)], c["tokens"][at:at + len(par)], par, c["u"][at:at + len(par)], c["r"][b],
                         float(c["temp"][b]), depth)[0]
        for j, node in enumerate(path):
            left = OD.softmax(c["x"][at + node], float(c["temp"][b]))
            for i in (k for k in range(node + 1, len(par)) if par[k] == node):
                tok = int(c["tokens"][at + i])
                if not 0 <= tok < len(left):
                    continue
                p, total = float(left[tok]), float(left.sum())
                if p > 0 and abs(float(c["u"][at + i]) * total / p - 1) < 5e-8:
                    return False
                if j + 1 < len(path) and i == path[j + 1]:
                    break
                left[tok] = 0
        at += len(par)
    return True


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [4096, 9001])
def test_sums_behind_a_low_beginning(dev, V, kind):                                        # noqa: F811
    """The first logits that a wave reads lie 10, 30, 60 and 63 powers of two below the likely ones: the sums' reference is then far
    from the largest weights. Random numbers a few 1e-7 on either side of w / Z."""
    rows, tokens, parents, temps, u, r = [], [], [], [], [], []
    for gap in (10.0, 30.0, 60.0, 63.0):
        for t in (0.31, 0.7, 0.83, 1.0, 1.37):
            for d in (-3e-6, -1e-6, -3e-7, 3e-7, 1e-6, 3e-6):
                x = torch.full((2, V), float("-inf"))
                t32 = float(np.float32(t))
                x[0, 5] = x[0, 300] = -7.3
                x[0, 2000], x[0, 3500] = -7.3 + gap * LOG2 * t32, -7.4 + gap * LOG2 * t32
                x[0, V - 1] = -9.0
                x[1, 3] = 1.0
                x = x.to(kind).float()
                p = float(OD.softmax(x[0], t32)[2000])
                rows.append(x)
                tokens.append(torch.tensor([0, 2000]))
                parents.append([-1, 0])
                temps.append(t32)
                u.append(torch.tensor([0.0, float(np.float32(p * (1 + d)))]))
                r.append(0.5)
    c = batch(rows, tokens, parents, temps, u, r)
    assert far(c, 2)
    want = want_of(c, 2)
    assert {len(p) for p in want[0]} == {1, 2}
    c["x"] = c["x"].to(kind)
    same(verify(dev, c, 2), want, 2, (V, kind))


def filtered(V, shares, seed):
    """A row whose logits are -infinity but for len(shares) tokens of these shares; the tokens."""
    g = torch.Generator().manual_seed(seed)
    toks = torch.randperm(V, generator=g)[: len(shares)]
    x = torch.full((V,), float("-inf"))
    x[toks] = torch.tensor(shares, dtype=torch.float64).log().float()
    return x, toks


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_the_last_token_of_a_filtered_row(dev, kind):                                      # noqa: F811
    """A row's children are all of its tokens and all but the last are rejected: the last one is accepted, whatever its share was,
    and the walk goes on below it (in the last case to a second such row)."""
    V = 9001
    for shares in ([1.0, 1e-3], [1.0, 1e-4], [1.0, 1e-5], [1.0, 2e-6], [0.5, 0.3, 0.2, 3e-5], [1.0, 1e-3, 1e-6, 1e-9], [1.0, 1e-2, 1e-7, 1e-12],
                   [1.0] + [1e-5 * 0.9 ** i for i in range(1, 40)]):
        rows, tokens, parents, u = [], [], [], []
        for seed in range(8):
            x, toks = filtered(V, shares, seed)
            y, more = filtered(V, shares[::-1] if seed % 2 else shares, 100 + seed)
            n = len(shares)
            par = [-1] + [0] * n + [n] * n                     # (the second row's children: below the last of the first's)
            every = torch.zeros(len(par), V)
            every[0], every[n] = x, y
            every = every.to(kind).float()
            rows.append(every)
            tokens.append(torch.cat((torch.zeros(1, dtype=torch.int64), toks, more)))
            parents.append(par)
            u.append(torch.full((len(par),), MOST))
        c = batch(rows, tokens, parents, [1.0] * 8, u, [0.5] * 8)
        want = want_of(c, 5)
        assert all(p[:2] == [0, len(shares)] for p in want[0])
        c["x"] = c["x"].to(kind)
        same(verify(dev, c, 5), want, 5, shares)


def test_what_is_left_beside_rejected_tokens(dev):                                         # noqa: F811
    """Likely tokens are rejected, one of them twice, with tokens outside the vocabulary between them; a small rest is tested further,
    and drawn from where every child is rejected; over several chunks."""
    V = 50257
    g = torch.Generator().manual_seed(3)
    rows, tokens, parents, temps, u, r = [], [], [], [], [], []
    for b in range(24):
        x = torch.full((9, V), float("-inf"))
        rest = torch.randperm(V, generator=g)[:50]
        x[:, rest] = -12.0 + torch.rand(9, 50, generator=g)
        top = torch.randperm(V, generator=g)[:2]
        x[0, top] = torch.tensor([3.0, 1.0])
        tokens.append(torch.tensor([0, int(top[0]), -1, int(top[1]), int(top[0]), V, *rest[:3].tolist()]))
        parents.append([-1] + [0] * 8)
        v = torch.full((9,), MOST)
        v[6:] = torch.rand(3, generator=g) * (0.06 if b % 2 else 1)
        rows.append(x)
        u.append(v)
        temps.append([1.0, 0.9, 1.2][b % 3])
        r.append(float(torch.rand(1, generator=g)))
    c = batch(rows, tokens, parents, temps, u, r)
    assert far(c, 3)
    want = want_of(c, 3)
    assert {len(p) for p in want[0]} == {1, 2}
    got = verify(dev, c, 3)
    same(got, want, 3)
    again = verify(dev, c, 3)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_captured_and_on_another_stream(dev):                                              # noqa: F811
    """Replays follow new logits, tokens and random numbers, some of which leave tests open; another stream gives the same."""
    from rfill import ops
    V, n = 9001, 6
    parents = [-1] + [0] * 4 + [4]
    hold = dict(x=torch.zeros(3 * n, V, device=dev), tok=torch.zeros(3 * n, dtype=torch.int64, device=dev), u=torch.zeros(3 * n, device=dev),
                r=torch.zeros(3, device=dev), t=torch.zeros(3, device=dev))
    par, cu = i32(parents * 3, dev), offsets([n] * 3).to(dev)
    ws = torch.zeros(ops.verify_drafts_workspace_bytes(3 * n, V, 3, n), dtype=torch.uint8, device=dev)

    def step():
        return ops.verify_drafts(hold["x"], hold["tok"], par, cu, hold["u"], hold["r"], hold["t"], n, workspace=ws)

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(3 * n, V, generator=g)
        tok = torch.zeros(3 * n, dtype=torch.int64)
        u = torch.rand(3 * n, generator=g)
        for b in range(3):
            row, toks = filtered(V, [[1.0, 1e-4, 1e-8, 1e-9], [0.5, 0.3, 0.2, 1e-6], [0.25] * 4][(b + seed) % 3], 10 * seed + b)
            x[b * n] = row
            tok[b * n + 1:b * n + 5] = toks
            if b != 2:
                u[b * n + 1:b * n + 5] = MOST
        c = dict(x=x, q=None, parents=[parents] * 3, tokens=tok, counts=[n] * 3, temp=torch.tensor([1.0, 1.0, 1.1 - 0.1 * (seed % 2)]), u=u,
                 r=torch.rand(3, generator=g))
        for key, name in (("x", "x"), ("tok", "tokens"), ("u", "u"), ("r", "r"), ("t", "temp")):
            hold[key].copy_(c[name])
        return c

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(1, 6):
        c = fill(seed)
        assert far(c, n)
        want = want_of(c, n)
        ws.fill_(255)
        same(step(), want, n, seed)
        ws.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same(outs, want, n, seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        same(other, want, n, seed)
