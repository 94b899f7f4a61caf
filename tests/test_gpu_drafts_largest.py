"""Verification at the largest vocabulary and tree that it takes at once: 2^19 tokens, 1024 rows."""
import pytest
import torch

from oracle import drafts as OD
from test_gpu_drafts import dev, i32      # noqa: F401  (dev: the fixture)
from test_gpu_drafts_sums import MOST

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draft", [False, True])
def test_largest(dev, draft):                                                              # noqa: F811
    """A star of 1000 children whose first ones are rejected (without shares down to one that the row's sum leaves open: likely tokens
    are gone and little is left; with shares a pass over the row each), then a chain below the accepted one, then a draw."""
    from rfill import ops
    V, n, wide = 1 << 19, 1024, 1000
    g = torch.Generator().manual_seed(6 + draft)
    toks = torch.randperm(V, generator=g)[: n]
    parents = [-1] + [0] * wide + [4] + list(range(wide + 1, n - 1))
    tokens = torch.zeros(n, dtype=torch.int64)
    tokens[1:] = toks[1:]
    x = torch.zeros(n, V, dtype=torch.bfloat16)
    x[0] = -9.0
    x[0, toks[1:4]] = torch.tensor([12.0, 9.0, 8.0]).to(torch.bfloat16)       # (the rest: 6e-4 of it)
    x[0, toks[4:6]] = 4.0
    u = torch.full((n,), MOST)
    u[4] = 0.1
    for i in range(4, n):                                                      # a chain whose tokens are likely
        nxt = wide + 1 if i == 4 else i + 1 if i > wide else None
        if nxt is not None and nxt < n:
            x[i, tokens[nxt]] = 30.0
    u[wide + 1:] = 0.5
    q = None
    if draft:                                                                  # (the shares have the first tokens above p)
        q = torch.full((n, V), 2.0 ** -21, dtype=torch.bfloat16)
        q[0, toks[1:4]] = torch.tensor([1.0, 0.5, 0.25]).to(torch.bfloat16)
        q[0, toks[4]] = 2.0 ** -16
    r, t = 0.37, 1.0
    want = OD.verify(x, tokens, parents, u, r, t, n, q)
    assert want[0][:2] == [0, 4] and len(want[0]) == n - wide + 1
    up = lambda z: z.to(dev)                                                   # noqa: E731
    got = ops.verify_drafts(up(x), up(tokens), i32(parents, dev), i32([0, n], dev), up(u), torch.tensor([r], device=dev),
                            torch.tensor([t], device=dev), n, draft=None if q is None else up(q))
    assert got[1].tolist() == [len(want[0])] and got[0][0, :len(want[0])].tolist() == want[0] and got[2].tolist() == [want[1]]
