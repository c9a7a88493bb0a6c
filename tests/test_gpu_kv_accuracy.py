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


def fp32_bound(p, layer, seqs, start, q, n_heads, window=0, scale=0.0):
    """How far an fp32 evaluation may be off per output, from the terms that are there (no largest
    value of others stands in): [rows][n_heads][hd].  e = 2^-24.

    Both products sum exact products of two fp16 pieces of an fp32 number with int8, 32 to a matrix
    instruction, whose sum is off by at most 10 e of its largest term or of what it adds to (probed:
    7.4), the second pieces adding less than a tenth: a score by dz = 11 e c (hd / 32) sum |q_j k_tj|,
    and by 10 e |z| + (4 + |ev|) e of its exponent's roundings, V's 2^ev in it; its weight by that and
    exp2's 2^-22.
    A value's sums take 8 such instructions for 256 tokens and a rounding for each 256: (82 + n / 256) e of
    sum w |v|; the denominator (n / 64 + 40) e of itself, the quotient 3 e.
    The pieces: the nearest fp16 leaves half of 2^-10 of a number, 2048 times that is held to half
    of 2^-10 again: 2^-22 of the number; or, where 2048 times what is left lies below the smallest
    normal fp16, to half of 2^-24 / 2048 = 2^-36, the largest standing between 2^14 and 2^15: 2^-50 of
    the largest weight with its V scale (of q: of the row's largest)."""
    out = np.zeros((q.shape[0], n_heads, p.hd))
    c = scale if scale > 0 else 1.0 / np.sqrt(p.hd)
    e = 2.0 ** -24
    steps = -(-p.hd // 64) * 2
    for i, s in enumerate(seqs):
        k, v = p.values(s, layer)
        m, n = int(start[i + 1] - start[i]), int(p.len[s])
        vs = np.array([[p.scale[layer, p.table[s, t // p.page], h, t % p.page // 16, 1]
                        for h in range(p.kv_heads)] for t in range(n)], np.float64)
        vq = v / vs[:, :, None]
        ev = np.abs(np.log2(vs)) + 1
        for r in range(m):
            pos = n - m + r
            lo = max(0, pos - window + 1) if window else 0
            for h in range(n_heads if pos >= 0 else 0):
                kh = h * p.kv_heads // n_heads
                row = q[start[i] + r, h * p.hd:(h + 1) * p.hd].astype(np.float64)
                kk, vv = k[lo:pos + 1, kh], v[lo:pos + 1, kh]
                z = kk @ row * c
                d = (11 * e * steps + 2.0 ** -22) * c * (np.abs(kk) @ np.abs(row))
                d += 2.0 ** -50 * c * np.abs(row).max() * np.abs(kk).sum(1)
                d += 10 * e * np.abs(z) + (4 + ev[lo:pos + 1, kh]) * e + 2.0 ** -22
                w = np.exp(z - z.max())
                L = w.sum()
                least = 2.0 ** -50 * (w * vs[lo:pos + 1, kh]).max()
                num = (w * (d + 2.0 ** -22)) @ np.abs(vv) + least * np.abs(vq[lo:pos + 1, kh]).sum(0)
                num += (82 + n / 256) * e * (w @ np.abs(vv))
                den = w @ d + (n / 64 + 40) * e * L
                mean = np.abs(w @ vv) / L
                out[start[i] + r, h] = num / L + mean * (den / L + 3 * e)
    return out


def check(d, p, seqs, counts, q, n_heads, **how):
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    got = d.attention(0, seqs, start, q, n_heads, **how)
    how.pop("max_len", None)
    want = p.attention(0, seqs, start, q, n_heads, **how)
    off = np.abs(got - want) / (fp32_bound(p, 0, seqs, start, q, n_heads, **how) + 2.0 ** -149)
    assert off.max() <= 1, "off by %.3g times what fp32 may be" % off.max()
    return off.max()


def pool_with(seed, n, hd, page=32, kv_heads=1):
    """One sequence of n ordinary tokens, its pages in order."""
    rng = np.random.default_rng(seed)
    n_pages = -(-n // page)
    p = R.Pool(1, n_pages, page, kv_heads, hd, 1, n_pages, seed)
    p.table[0], p.len[0], p.refs[:] = np.arange(n_pages), n, 1
    p.data[:] = np.clip(np.rint(rng.normal(0, 42, p.data.shape)), -127, 127)
    p.scale[:] = 0.02 * np.exp(rng.normal(0, 0.5, p.scale.shape))
    return p


def token(p, t, side):
    """The int8 values of a token (kv head 0), to be written."""
    b = p.data[0, p.table[0, t // p.page], 0, t % p.page // 16, side]
    return b.reshape(16, p.hd)[t % 16] if side == 0 else b.reshape(p.hd, 16)[:, t % 16]


@pytest.mark.parametrize("hd,rows", [(64, 1), (64, 40), (128, 1), (128, 40), (32, 3), (96, 2), (256, 1),
                                     (224, 5)])
@pytest.mark.parametrize("own", [0, 1])
def test_sinks_of_small_values_in_ordinary_blocks(dev, hd, rows, own):
    """A token that takes half to 0.99999 of the first row's weight and whose values are 0 (or 1 of 127) in a
    block that its neighbours scale: the output is the others', to fp32 accuracy."""
    n, heads = 1201, 2
    rng = np.random.default_rng(hd + rows)
    for at in (0, 700, 1200 - rows):
        p = pool_with(hd, n, hd)
        p.scale[:, :, :, :, 0] = 0.02
        u = rng.choice([-1.0, 1.0], hd)
        token(p, at, 0)[:] = 127 * u
        token(p, at, 1)[:] = own
        q = (np.tile(u, heads) + rng.normal(0, 1, (rows, heads * hd))).astype(np.float32)
        k = p.values(0, 0)[0][:, 0]
        z = k[:n - rows + 1] @ q[0, :hd].astype(np.float64)
        d = R.DevPool(dev, p)
        for share in (0.5, 0.97, 0.997, 0.9999, 0.99999):
            lo, hi = 1e-3, 50.0  # the scale that gives the first row this share
            for _ in range(60):
                c = (lo + hi) / 2
                w = np.exp(c * (z - z.max()))
                lo, hi = (c, hi) if w[at] / w.sum() < share else (lo, c)
            assert abs(w[at] / w.sum() - share) < 1e-6 * share
            check(d, p, [0], [rows], q, heads, scale=float(np.float32(c)), max_len=n)


@pytest.mark.parametrize("hd,rows", [(64, 1), (64, 40), (128, 3), (128, 40), (32, 2), (96, 1), (160, 2),
                                     (256, 5)])
@pytest.mark.parametrize("size", [60.0, 1e4, 1e6])
def test_outlier_channels_of_q(dev, hd, rows, size):
    """A channel of q far above the others where K is small or 0: the others count all the same."""
    n, heads = 500, 2
    rng = np.random.default_rng(hd + rows)
    p = pool_with(hd, n, hd)
    for j, least in ((hd - 1, 0), (5, 0), (17, 1 if size < 100 else 0)):
        for t in range(n):
            token(p, t, 0)[j] = least * rng.integers(-1, 2)
    q = rng.normal(0, 1.5, (rows, heads * hd)).astype(np.float32)
    for h in range(heads):
        q[:, h * hd + rng.choice([hd - 1, 5, 17])] = size * rng.choice([-1, 1], rows)
    check(R.DevPool(dev, p), p, [0], [rows], q, heads, max_len=n)


def test_ordinary_rows_to_the_same_bound(dev):
    for hd, heads, rows, n in ((64, 8, 1, 702), (128, 8, 64, 900), (96, 4, 5, 300), (192, 1, 2, 150)):
        p = pool_with(hd + 1, n, hd)
        q = np.random.default_rng(n).normal(0, 1.5, (rows, heads * hd)).astype(np.float32)
        check(R.DevPool(dev, p), p, [0], [rows], q, heads, max_len=n)
        check(R.DevPool(dev, p), p, [0], [rows], q, heads, max_len=n, window=77)


@pytest.mark.parametrize("size", [1e-37, 1e-33, 1e-30, 1e-25, 1e-20, 1e-10, 1e10, 1e20, 1e30, 1e35])
def test_values_of_any_size(dev, size):
    """V small or large everywhere, down to the least normal scales: held as well as ordinary ones."""
    for hd, heads, rows, n in ((64, 8, 1, 300), (128, 2, 40, 600), (96, 4, 5, 70)):
        p = pool_with(hd + 2, n, hd)
        p.scale[:, :, :, :, 1] *= np.float32(size)
        q = np.random.default_rng(n).normal(0, 1, (rows, heads * hd)).astype(np.float32)
        check(R.DevPool(dev, p), p, [0], [rows], q, heads, max_len=n)
