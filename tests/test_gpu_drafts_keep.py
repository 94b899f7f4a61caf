"""Kept rows where the layers' pages lie between one another's: one buffer of pages, each with every layer's K and V. (Layers that share
memory are refused: test_drafts_keep_host.py.)"""
import pytest
import torch

from test_gpu_drafts import dev, i32      # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [1, 5, 40])
def test_layers_of_one_buffer(dev, layers):                                                # noqa: F811
    from rfill import ops
    from rfill.paged import Pages
    buf = torch.randn(4, layers, 2, 2, 16, 64, generator=torch.Generator().manual_seed(layers)).to(torch.bfloat16)   # [pages, layers, k|v, ..]
    now = buf.to(dev)
    pools = [Pages(now[:, i, 0], now[:, i, 1]) for i in range(layers)]
    args = i32([[3, 0], [1, 2]], dev), i32([32, 20], dev), i32([0, 6, 12], dev), i32([[0, 2, 5], [0, 1, 4]], dev), i32([3, 3], dev)
    ops.paged_keep(pools, *args)
    want = buf.clone()
    for (sp, so), (dp, do) in (((0, 12), (0, 11)), ((0, 15), (0, 12)), ((2, 2), (2, 0))):
        want[dp, :, :, :, do] = buf[sp, :, :, :, so]
    assert torch.equal(now.cpu(), want)
    with pytest.raises(ValueError, match="overlap"):
        ops.paged_keep(pools + [Pages(now[:, 0, 1], torch.zeros_like(now)[:, 0, 1])], *args)
    assert torch.equal(now.cpu(), want)
