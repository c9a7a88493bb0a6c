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


@pytest.mark.parametrize("n,most", [(65, 40), (300, 30), (300, 1), (4500, 1), (4500, 3)])
def test_batches_of_many_sequences(dev, n, most):
    """The rows' search takes a step for each factor of 64: two from 65 sequences on, three from 4097.
    Sequences without rows among them, first and last too; store, load and attention."""
    rng = np.random.default_rng(n + most)
    lens = rng.integers(1, 60 if n < 1000 else 20, n)
    counts = np.minimum(rng.integers(0 if most > 1 else 1, most + 1, n), lens)
    counts[rng.random(n) < 0.2] = 0
    counts[[0, n - 1, n // 2]] = 0, 0, 1
    p = pool_of(lens.tolist(), seed=n)
    d = R.DevPool(dev, p)
    seqs = rng.permutation(n).tolist()
    counts = np.minimum(counts, lens[seqs])
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    T = int(start[-1]) + 2
    k, v = (rng.normal(0, 1, (T, 32)).astype(np.float32) for _ in range(2))
    p.store(0, seqs, start, k, v)
    d.store(0, seqs, start, k, v)
    R.assert_same(d, p)
    got = d.load(0, seqs, start, T)
    for i, s in enumerate(seqs):
        vals = p.values(s, 0)
        for side in (0, 1):
            want = vals[side][int(p.len[s]) - int(counts[i]):].astype(np.float32)
            np.testing.assert_array_equal(got[side][start[i]:start[i + 1]], want)
    for x in got:
        assert (x[start[-1]:] == 7).all()
    q = rng.normal(0, 1, (T, 2 * 32)).astype(np.float32)
    out = d.attention(0, seqs, start, q, 2, max_len=int(lens.max()))
    want = p.attention(0, seqs, start, q, 2)
    bound = R.attention_bound(p, 0, seqs, start, q, 2)
    own = slice(0, int(start[-1]))
    assert (np.abs(out[own] - want[own]) <= bound[own]).all()
    assert (out[start[-1]:] == 7).all()
