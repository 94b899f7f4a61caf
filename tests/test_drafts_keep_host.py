"""rf_paged_keep and layers whose pages share memory, without a GPU: refused in the library before any launch (two blocks would move the
same bytes at once). Layers that lie between one another's pages are none of these; nothing refuses them by name here (the launch
that follows finds no GPU)."""
import ctypes

import pytest
import torch

from test_paged_host import _pages

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: without a GPU only")
PAGE, HEADS = 2 * 16 * 64, 2 * 16 * 32     # _pages(): 4 bits, 2 heads of 64, 16 tokens: from a page to the next, and its codes


def _keep(pages, n_seq=1):
    from rfill import _lib
    handles = (ctypes.c_void_p * len(pages))(*(ctypes.addressof(p) for p in pages))
    _lib.call("rf_paged_keep", handles, len(pages), 1 << 20, 4, 4, 1 << 20, 1 << 20, n_seq, 1 << 20, 3, 3, 1 << 20, None)


def _layer(at, **kw):
    at <<= 20
    return _pages(**{**dict(k=at, v=at + (1 << 18), ks=at + (2 << 18), vs=at + (3 << 18)), **kw})


def _mib(x):
    return x << 20


@pytest.mark.parametrize("name", ["v", "ks", "vs"])
def test_a_pool_that_two_layers_share(name):
    a, b, c = _layer(1), _layer(2), _layer(3)
    setattr(c, name, getattr(a, name))
    with pytest.raises(ValueError, match="layers 0 and 2"):
        _keep([a, b, c])


@pytest.mark.parametrize("kw", [
    dict(v=_mib(1)),                                           # its values are the first layer's keys
    dict(k=_mib(1) + 3 * PAGE),                                # the first layer's keys from the fourth page on
    dict(k=_mib(1) + HEADS - 16),                              # every page over the end of the first's by 16 bytes
    dict(k=_mib(1) - HEADS + 16),                              # ... over its beginning
    dict(k=_mib(1) + 7 * PAGE),                                # its last page alone
    dict(ks=_mib(1) + 5 * PAGE + 64),                          # scales where codes are
    dict(k=_mib(1) + HEADS, page_stride=5 * HEADS, v=_mib(9)), # another stride: between the first's pages, then over them
])
def test_pools_that_overlap(kw):
    for pages in ([_layer(1), _layer(2, **kw)], [_layer(2, **kw), _layer(1)]):
        with pytest.raises(ValueError, match="layers [01] and [01]"):
            _keep(pages)


def test_keys_and_values_of_a_layer_overlap():
    for kw in (dict(v=_mib(1)), dict(v=_mib(1) + PAGE), dict(vs=_mib(1) + (2 << 18))):
        with pytest.raises(ValueError, match="layers 1 and 1"):
            _keep([_layer(5), _layer(1, **kw), _layer(6)])


def test_many_layers():
    """Beyond what a launch takes."""
    layers = [_layer(1 + i) for i in range(70)]
    layers[69].vs = layers[3].ks + 7 * PAGE // 32
    with pytest.raises(ValueError, match="layers 3 and 69"):
        _keep(layers)


def test_of_no_sequences_nothing_is_moved():
    _keep([_layer(1), _layer(2, v=_layer(1).v)], n_seq=0)


def test_layers_between_one_another():
    """K and V of one buffer, layers of one buffer: pages alternate, and the refusal is that of a machine without a GPU, if any."""
    at = _mib(1)
    beside = [
        [_layer(1, v=at + HEADS), _layer(2, v=_mib(2) + HEADS)],
        [_layer(1), _layer(2, k=at + HEADS)],                  # layer 1's keys in the gaps of layer 0's
        [_layer(1, page_stride=4 * HEADS, v=at + HEADS), _layer(2, page_stride=4 * HEADS, k=at + 2 * HEADS, v=at + 3 * HEADS)],
        [_layer(1, page_stride=4 * HEADS, v=at + HEADS), _layer(2, k=at + 2 * HEADS, v=_mib(9), page_stride=4 * HEADS, n_pages=3)],
        [_layer(1, page_stride=2 * HEADS, n_pages=1), _layer(2, k=at + HEADS, v=_mib(9), page_stride=5 * HEADS)],
        [_layer(1, page_stride=4 * HEADS, n_pages=4), _layer(2, k=at + HEADS, v=_mib(9), page_stride=8 * HEADS, n_pages=2)],
        [_layer(1), _layer(2, k=at + 8 * PAGE)],               # right behind
    ]
    for pages in beside:
        try:
            _keep(pages)
        except ValueError as e:
            pytest.fail(str(e))
        except Exception:                                      # (the launch's)
            pass
