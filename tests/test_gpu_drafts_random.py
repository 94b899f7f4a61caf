"""FillModel.verify_paged's own random numbers."""
import pytest
import torch

from test_gpu_drafts_model import _ids, _model, dev      # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


def test_random_numbers_under_another_default_type(dev):                                   # noqa: F811
    """torch's random numbers are 32-bit ones whatever torch.get_default_dtype() says."""
    from rfill.paged import PagedCache
    cfg, m = _model("llama_c1", dev)
    answers = []
    for t in (torch.float32, torch.bfloat16, torch.float64):
        cache = PagedCache(m, 20, page=16)
        s = cache.add()
        m.forward_paged(cache, [s], _ids(1, (30,)))
        torch.manual_seed(3)
        torch.set_default_dtype(t)
        try:
            answers.append(m.verify_paged(cache, [s], _ids(2, (5,)), temperature=0.8))
        finally:
            torch.set_default_dtype(torch.float32)
    assert answers[0] == answers[1] == answers[2]
