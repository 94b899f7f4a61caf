"""The oracle of drafted tokens (oracle.drafts) against what verification is for: whatever the drafts, the tokens that come out
are distributed as the target's. And the refusals that need no GPU."""
import pytest
import torch

from oracle import drafts as OD


def test_above():
    see, depth = OD.above([-1, 0, 0, 2, 1, 3, -1, 9])
    rows = [[0], [0, 1], [0, 2], [0, 2, 3], [0, 1, 4], [0, 2, 3, 5], [6], [7]]
    assert [r.nonzero().flatten().tolist() for r in see] == rows and depth == [0, 1, 1, 2, 2, 3, 0, 0]
    w = OD.words(torch.ones(1, 130, dtype=torch.bool), 3)
    assert w.tolist() == [[-1, -1, 3]]


@pytest.mark.parametrize("form", ["likely", "drawn"])
def test_tokens_are_the_targets(form):
    """A tree of two tokens and one below the first, of a vocabulary of 5: over 20000 random numbers the first token's share
    is the target's, and the second's given the first. 20000 draws: a share's standard deviation is at most 0.0036; given the
    first (at least 5 % of them, 1000) 0.016; five of them."""
    g = torch.Generator().manual_seed(3)
    V, n = 5, 20000
    logits = torch.randn(4, V, generator=g)
    q = torch.softmax(logits + torch.randn(4, V, generator=g), 1)
    p = torch.softmax(logits.double() / 0.8, 1)
    parents = [-1, 0, 0, 1]
    if form == "likely":
        draws = torch.tensor([[3, 1, 4]]).expand(n, 3)
    else:
        draws = torch.cat((torch.multinomial(q[0].expand(n, V), 2, replacement=True, generator=g),
                           torch.multinomial(q[1].expand(n, V), 1, generator=g)), 1)
    u, r = torch.rand(n, 4, generator=g), torch.rand(n, generator=g)
    first, second = torch.zeros(V), torch.zeros(V)
    for i in range(n):
        toks = [0] + draws[i].tolist()
        path, nxt = OD.verify(logits, toks, parents, u[i], r[i], 0.8, 4, q if form == "drawn" else None)
        out = [toks[x] for x in path[1:]] + [nxt]
        first[out[0]] += 1
        if len(path) > 1 and path[1] == 1:
            second[out[1]] += 1
    assert bool(((first / n - p[0]).abs() < 0.018).all()), first / n - p[0]
    assert second.sum() > 1000 and bool(((second / second.sum() - p[1]).abs() < 0.08).all())


def test_verify_edges():
    """Ties, NaN, rows of nothing, infinities, the depth, tokens outside the vocabulary."""
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[1.0, 3.0, 3.0], [nan, -inf, 0.0], [-inf, nan, -inf], [0.0, inf, inf]])
    one = lambda row, **kw: OD.verify(x[row:row + 1], [0], [-1], [0.0], kw.pop("r", 0.0), kw.pop("t", 1.0), 4)   # noqa: E731
    assert one(0, t=0.0) == ([0], 1) and one(1, t=0.0) == ([0], 2) and one(2, t=0.0) == ([0], -1)
    assert one(1, r=0.999) == ([0], 2) and one(2) == ([0], -1) and one(3, r=0.4) == ([0], 1) and one(3, r=0.6) == ([0], 2)
    assert one(0, t=inf, r=0.2) == ([0], 0)
    assert OD.verify(x[[0, 0]], [0, 7], [-1, 0], [0, 0], 0.99, 1.0, 4) == ([0], 2)
    assert OD.verify(x[[0, 0]], [0, 1], [-1, 0], [0, 0.0], 0.0, 1.0, 1) == ([0], 0)
    assert OD.verify(x[[0, 0]], [0, 1], [-1, 0], [0, 0.0], 0.0, 1.0, 2) == ([0, 1], 0)


def test_keep():
    assert OD.keep([0, 2, 5], 3, 6) == [(0, 0), (2, 1), (5, 2)]
    assert OD.keep([0, 2, 2], 3, 6) == [(0, 0), (2, 1)] and OD.keep([0, 9], 2, 6) == [(0, 0)] and OD.keep([-1], 1, 6) == []
    assert OD.keep([0, 1, 2], 2, 6) == [(0, 0), (1, 1)]


def test_workspace_sizes_and_refusals():
    """Host-only size rule: 16 bytes a row and share of it (a share a 4096 logits, 8192 in all but at least one a row), 128 a
    (sequence, 4096 logits), 64 a sequence and four a row of each."""
    from rfill import _lib, ops
    size = ops.verify_drafts_workspace_bytes
    assert size(10, 4096, 2, 8) == 10 * 16 + 2 * (128 + 64 + 4 * 8) and size(10, 4097, 5, 80) == 20 * 16 + 5 * (256 + 64 + 4 * 10)
    assert size(5000, 40960, 1, 8) == 5000 * 16 + 1280 + 64 + 32 and size(9000, 40960, 1, 8) == 9000 * 16 + 1280 + 64 + 32
    assert size(0, 100, 3, 8) == 0 and size(5, 100, 0, 8) == 0
    for rows, vocab, n, most in ((1, (1 << 19) + 1, 1, 1), (1, 0, 1, 1), (1, 100, 1, 1025)):
        with pytest.raises(_lib.UnsupportedArchitecture):
            size(rows, vocab, n, most)
    with pytest.raises(ValueError):
        size((1 << 30) + 1, 1 << 19, 1, 1)
    with pytest.raises(ValueError):
        size(1, 100, -1, 1)
