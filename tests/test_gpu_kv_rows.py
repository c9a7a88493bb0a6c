"""Rows of a ragged batch (qr_kv_pool_store / _load / _attention of
include/qr_hip.h): rows without a page, and batches of more sequences than one
step of the rows' search holds."""
import numpy as np
import pytest

import kv_pool_ref as R

pytestmark = pytest.mark.gpu


def pool_of(lens, page=16, kv_heads=1, hd=32, n_layers=1, seed=1):
    """Sequences of the given lengths over shuffled pages, what they hold random."""
    rng = np.random.default_rng(seed)
    need = int(sum(-(-n // page) for n in lens))
    p = R.Pool(n_layers, need + 3, page, kv_heads, hd, len(lens), max(1, -(-max(lens) // page)) + 1,
               seed)
    p.data[:] = rng.integers(-127, 128, p.data.shape, dtype=np.int8)
    p.scale[:] = 0.02 * np.exp(rng.normal(0, 0.5, p.scale.shape))
    order, at = rng.permutation(p.n_pages), 0
    for s, n in enumerate(lens):
        k = -(-int(n) // page)
        p.table[s, :k], p.len[s] = order[at:at + k], n
        p.refs[order[at:at + k]] = 1
        at += k
    return p


def test_rows_without_a_page_load_as_positive_zeros(dev):
    p = pool_of([40, 5], kv_heads=2, hd=64)
    p.data[0, 0] = -1  # the layer's first page
    p.table[0, 1] = -1
    d = R.DevPool(dev, p)
    k, v = d.load(0, [0, 1], np.array([0, 40, 47], np.int32), 47)
    for x in (k, v):
        for rows in (x[16:32], x[40:42]):  # no page, before position 0
            assert (rows.view(np.uint32) == 0).all()
        assert (x[:16] != 0).any() and (x[32:40] != 0).any() and (x[42:] != 0).any()
