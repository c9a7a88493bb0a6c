"""qr_logprobs (include/qr_hip.h) against its definition in 64 bits
(kv_pool_ref.logprobs): ranks and alternatives equal, the rest to a derived bound."""
import numpy as np
import pytest

import kv_pool_ref as R

pytestmark = pytest.mark.gpu


def run_logprobs(dev, x, V, targets, n, off=0):
    """qr_logprobs on rows whose first logit lies `off` floats into a buffer."""
    rows, stride = x.shape
    flat = np.concatenate([np.full(off, 9, np.float32), x.reshape(-1)])
    xd, td = dev.upload(flat), dev.upload(np.asarray(targets, np.int32))
    lp, ent, rank, tid, tlp = (dev.alloc(max(16, rows * max(1, k) * 4)) for k in (1, 1, 1, n, n))
    dev.logprobs(xd.offset(4 * off), rows, V, td.ptr, lp.ptr, ent.ptr, rank.ptr, n, tid.ptr, tlp.ptr,
                 stride=stride)
    return (dev.download(lp, (rows,), np.float32), dev.download(ent, (rows,), np.float32),
            dev.download(rank, (rows,), np.int32), dev.download(tid, (rows, n), np.int32),
            dev.download(tlp, (rows, n), np.float32))


def near(got, want, bound, what):
    ok = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid="ignore"):
        ok |= np.abs(got - want) <= bound
    assert ok.all(), "%s: %s" % (what, [(got[i], want[i]) for i in zip(*np.nonzero(~ok))][:4])


def check_logprobs(dev, x, V, targets, n, off=0):
    """x - m is rounded to e = 2^-24 of it, its product with log2 e twice more, exp2 to 2^-22;
    a term's share p of the sums is off by p (3 e |d| + 2^-22), each of the V / 64 + 200 adds by e
    of the sum at most: log S by (3 e 200 + 2^-22 + (V / 64 + 200) e), its own rounding and the
    last differences by 3 e (|lp| + |log S| + |d|)."""
    e = 2.0 ** -24
    got = run_logprobs(dev, x, V, targets, n, off)
    want = R.logprobs(x[:, :V], targets, n)
    np.testing.assert_array_equal(got[2], want[2])
    np.testing.assert_array_equal(got[3], want[3])
    fin = x[:, :V].astype(np.float64)
    fin = np.where(np.isfinite(fin), fin, -np.inf)
    m = fin.max(1, keepdims=True)
    d = np.where(fin > -np.inf, np.where(m > -np.inf, m, 0) - fin, 0)
    p = np.where(fin > -np.inf, np.exp(-d), 0)
    total = np.maximum(p.sum(1), 1e-300)
    share = (p * d).sum(1) / total
    base = 3 * e * share + 2.0 ** -22 + (V / 64 + 200) * e
    base = base + 3 * e * (np.log(V) + 1)
    near(got[0], want[0], base + 4 * e * np.nan_to_num(np.abs(want[0]), posinf=0), "lp")
    near(got[4], want[4], base[:, None] + 4 * e * np.nan_to_num(np.abs(want[4]), posinf=0), "top_lp")
    share2 = (p * d * d).sum(1) / total
    near(got[1], want[1], base * (2 + share) + 4 * e * (share + share2), "entropy")


@pytest.mark.parametrize("rows,V,n", [(1, 1, 1), (3, 2, 5), (2, 63, 64), (1, 1023, 20), (5, 1024, 1),
                                      (2, 4097, 7), (1, 32000, 20), (3, 151936, 64), (9, 50001, 0),
                                      (300, 5000, 3), (1100, 4200, 2), (2, 600001, 20), (2, 300000, 64),
                                      (1, 4300001, 33)])
def test_logprobs_sizes(dev, rows, V, n):
    rng = np.random.default_rng(V + n)
    x = (rng.normal(0, 3, (rows, V + rows % 5))).astype(np.float32)
    t = rng.integers(0, V, rows)
    t[::3] = [-1, V, 0][rows % 3]
    check_logprobs(dev, x, V, t, n)


@pytest.mark.parametrize("off,pad", [(0, 0), (1, 0), (0, 1), (3, 2), (4, 4)])
def test_logprobs_alignment_and_strides(dev, off, pad):
    rng = np.random.default_rng(off + 7)
    x = rng.normal(0, 3, (4, 9000 + pad)).astype(np.float32)
    x[:, 9000:] = np.nan  # never read
    check_logprobs(dev, x, 9000, rng.integers(0, 9000, 4), 10, off)


def test_logprobs_orders(dev):
    """Equal logits, rising and falling rows, few distinct values, zeros of both signs."""
    V = 20000
    rng = np.random.default_rng(8)
    up = np.linspace(-5, 5, V).astype(np.float32)
    x = np.stack([np.zeros(V), up, up[::-1], rng.integers(0, 3, V), rng.choice([0.0, -0.0], V),
                  np.where(np.arange(V) == V - 1, 9, 0), rng.normal(0, 1e-6, V),
                  1e4 * rng.normal(0, 1, V)]).astype(np.float32)
    for t in (0, 1, V // 2, V - 1):
        check_logprobs(dev, x, V, [t] * 8, 33)


def test_logprobs_of_masked_and_broken_rows(dev):
    V = 9001
    rng = np.random.default_rng(9)
    x = rng.normal(0, 2, (9, V)).astype(np.float32)
    x[0] = -np.inf
    x[1, 5:] = -np.inf       # fewer left than alternatives
    x[2, :-1] = -np.inf
    x[3, 77] = np.nan
    x[4, 78] = np.inf
    x[5] = np.nan
    x[6] = np.finfo(np.float32).min
    x[7, ::2] = -np.inf
    x[8] = np.finfo(np.float32).max
    for t in (0, 77, V - 1):
        check_logprobs(dev, x, V, [t] * 9, 20)


def test_logprobs_optional_outputs(dev):
    V = 5000
    rng = np.random.default_rng(10)
    x = rng.normal(0, 2, (3, V)).astype(np.float32)
    t = np.array([1, 2, 3], np.int32)
    full = run_logprobs(dev, x, V, t, 4)
    xd, td = dev.upload(x), dev.upload(t)
    for keep in ((1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 0), (0, 0, 0, 1, 0), (0, 0, 0, 0, 1)):
        out = [dev.alloc(64) if k else None for k in keep]
        ptr = [b.ptr if b else None for b in out]
        dev.logprobs(xd.ptr, 3, V, td.ptr if keep[0] or keep[2] else None, ptr[0], ptr[1], ptr[2], 4,
                     ptr[3], ptr[4])
        i = keep.index(1)
        np.testing.assert_array_equal(dev.download(out[i], full[i].shape, full[i].dtype), full[i])


