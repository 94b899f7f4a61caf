"""Attention at the smallest scales it takes (down to the least positive float), where 8 / (scale log2 e), the softmax's headroom
in units of the scores, is past the floats: each output is the mean of the values in sight. Paged attention of few rows and
of chunks, and attend_causal; unsplit and split. Tolerances: test_gpu_paged.py's (check)."""
import pytest
import torch

from paged_dense import attend as dense
from test_gpu_paged import batch, check, dev, run                       # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu
TINY = [1e-45, 1e-39, 2e-38, 1e-37]


@pytest.mark.parametrize("scale", TINY)
@pytest.mark.parametrize("d,mx", [(64, False), (128, False), (256, False), (64, True), (128, True), (256, True)])
def test_paged(dev, d, mx, scale):                                         # noqa: F811
    hq, hkv = 4, 2
    for rows, lens in (([1, 3], [1300, 70]), ([90, 1], [1300, 40])):
        pools, table, n_pages, q = batch(hq, hkv, d, 16, mx, rows, lens, d)
        want, size = dense(pools, table, n_pages, q, rows, lens, hq, scale)
        for kw in (dict(), dict(max_keys=1 << 16), dict(max_keys=1 << 16, workspace=None)):
            check(run(dev, pools, table, q, rows, lens, hq, scale, **kw), want, size, (rows, kw))


@pytest.mark.parametrize("scale", TINY)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_causal(dev, d, scale):                                            # noqa: F811
    from rfill import ops
    hq, hkv, n, nq = 4, 2, 5000, 40
    g = torch.Generator().manual_seed(d)
    q = torch.randn(nq, hq * d, generator=g).to(torch.bfloat16)
    k, v = (torch.randn(hkv, n, d, generator=g).to(torch.bfloat16) for _ in "kv")
    got = ops.attend_causal(q.to(dev), n - nq, k.to(dev), v.to(dev), n, hq, scale).cpu().double().view(nq, hq, d)
    upto = torch.arange(n - nq, n)
    mean = (v.double().cumsum(1) / torch.arange(1, n + 1)[:, None])[:, upto]            # [hkv, nq, d]
    size = (v.double().abs().cumsum(1) / torch.arange(1, n + 1)[:, None])[:, upto]
    by = lambda t: t.transpose(0, 1).repeat_interleave(hq // hkv, 1)                      # noqa: E731
    check(got, by(mean), by(size), d)
