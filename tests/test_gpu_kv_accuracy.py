"""qr_kv_pool_attention (include/qr_hip.h) where fp32 accuracy is hard to keep:
against the formula in 64 bits, to bounds that an fp32 evaluation meets."""
import numpy as np
import pytest

import kv_pool_ref as R

pytestmark = pytest.mark.gpu


def long_pool(seed, n, hd, page=65536):
    """One sequence of n tokens of one kv head, its pages in order."""
    rng = np.random.default_rng(seed)
    n_pages = -(-n // page)
    p = R.Pool(1, n_pages, page, 1, hd, 1, n_pages, seed)
    p.table[0], p.len[0], p.refs[:] = np.arange(n_pages), n, 1
    p.data[:] = np.clip(np.rint(rng.normal(0, 42, p.data.shape)), -127, 127)
    p.scale[:] = 0.02 * np.exp(rng.normal(0, 0.5, p.scale.shape))
    return p


@pytest.mark.parametrize("n", [300001, 700001])
def test_long_sequences_in_one_part(dev, n):
    """Thousands of rounds of one workgroup (the bound on the lengths is far too small): what
    the sums stand against does not drift."""
    hd = 32
    p = long_pool(1, n, hd)
    q = np.random.default_rng(2).normal(0, 1, (2, 2 * hd)).astype(np.float32)
    start = np.array([0, 2], np.int32)
    d = R.DevPool(dev, p)
    got = d.attention(0, [0], start, q, 2, max_len=64)
    want = p.attention(0, [0], start, q, 2)
    bound = R.attention_bound(p, 0, [0], start, q, 2)
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), "off by %.3g over a bound of %.3g" % (np.abs(got - want).max(), bound.max())
