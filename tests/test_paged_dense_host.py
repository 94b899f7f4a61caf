"""paged_dense's attention against the oracle's, and what its telling() inputs tell: a mistake of 16 keys anywhere, planted in
the oracle, is outside the bound that the GPU tests use."""
import pytest
import torch

from oracle import paged as OP
from paged_dense import attend, telling, values
from test_gpu_paged import U, batch, layout, oracle_attend


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (6, 2, 128), (3, 1, 256)])
def test_dense_attention_is_the_oracle_s(hq, hkv, d, mx):
    rows, lens = [5, 1, 0, 9, 2], [40, 17, 3, 7, 33]
    pools, table, n_pages, q = batch(hq, hkv, d, 16, mx, rows, lens, d)
    table[0, 1], table[4, :3] = -3, n_pages
    want, size = oracle_attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    got, a = attend(pools, table, n_pages, q, rows, lens, hq, d ** -0.5)
    assert float((got - want).abs().max()) < 1e-12 and float((a - size).abs().max()) < 1e-12
    k, v = values(pools)
    for s in range(0, n_pages * 16, 7):
        rk, rv = pools.read(s)
        assert torch.equal(k[s // 16, :, s % 16], rk) and torch.equal(v[s // 16, :, s % 16], rv)


def _outside(got, want, size):
    return bool(((got - want).abs() > U * want.abs() + 2 * U * size + 2.0 ** -30).any())


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d,n", [(64, 4700), (64, 2600), (256, 2600), (128, 9001)])
def test_every_sixteen_keys_tell(d, n, mx):
    hq, hkv, page, rows, lens = 2, 1, 16, [1], [n]
    table, n_pages = layout(lens, page, 3)
    sides = [telling(hq, hkv, d, page, mx, rows, lens, table, n_pages, down) for down in (False, True)]
    wants = [attend(p, table, n_pages, q, rows, lens, hq, 1.0) for p, q in sides]
    last = -(-n // page) - 1
    for t in list(range(0, last, 37)) + [63, 64, last]:
        told = []
        for (p, q), want in zip(sides, wants):
            gone, wrong = table.clone(), table.clone()
            gone[0, t] = -1                                    # left out
            wrong[0, t] = table[0, (t + 1) % last]             # another's in their place
            for bad in (gone, wrong):
                told.append(_outside(attend(p, bad, n_pages, q, rows, lens, hq, 1.0)[0], *want))
            keys = OP.Pools(n_pages, hkv, page, d, mx)         # K of another page, V their own
            keys.v, keys.vs = p.v, p.vs
            keys.k = p.k.clone()
            keys.k[int(table[0, t])] = p.k[int(table[0, (t + 1) % last])]
            if mx:
                keys.ks = p.ks.clone()
                keys.ks[int(table[0, t])] = p.ks[int(table[0, (t + 1) % last])]
            told.append(_outside(attend(keys, table, n_pages, q, rows, lens, hq, 1.0)[0], *want))
        assert (told[0] or told[3]) and (told[1] or told[4]) and (told[2] or told[5]), (t, told)
