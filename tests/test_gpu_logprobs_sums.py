"""The sums of qr_logprobs (include/qr_hip.h) over long rows of small terms beside
a large one, against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", [-17.0, -18.5])
def test_small_terms_beside_a_large_one(dev, low):
    """One logit of 0 among V of `low`, whose e^low is below half of the last place of 1: they
    count all the same.  1024 rows, so that a row is one workgroup's."""
    rows, V = 1024, 40001
    x = np.full((rows, V), low, np.float32)
    hot = np.random.default_rng(1).integers(0, V, rows).astype(np.int32)
    x[np.arange(rows), hot] = 0
    xd, td = dev.upload(x), dev.upload(hot)
    lp, ent = dev.alloc(rows * 4), dev.alloc(rows * 4)
    dev.logprobs(xd.ptr, rows, V, td.ptr, lp.ptr, ent.ptr, None)
    p = np.exp(np.float64(low))
    S = 1 + (V - 1) * p
    want, entropy = -np.log(S), np.log(S) - (V - 1) * p * low / S
    # e = 2^-24.  A lane takes 16 logits a step, and a workgroup 4096: a rounding of e of the
    # lane's sum for each of V / 4096 + 1 steps, of e of 16 small terms inside one, ten of joining
    # the lanes and waves, exp2's 2^-22 and 4 e |low| of each small term, a few of the logarithm.
    e = 2.0 ** -24
    share = (V - 1) * p
    off = (V // 4096 + 1 + 10 + 5) * e + share * (16 * e + 2.0 ** -22 + 4 * e * -low)
    got = dev.download(lp, (rows,), np.float32)
    assert np.abs(got - want).max() <= off
    got = dev.download(ent, (rows,), np.float32)
    # U's terms are low times those of S
    assert np.abs(got - entropy).max() <= off + share * -low * (16 + 10 + V // 4096 + 8) * e
