"""A shared 8-bit KV pool (qr_kv_pool_* of include/qr_hip.h) against its
definitions in 64 bits (kv_pool_ref.py): page operations, 8-bit values and
scales bit for bit, attention to a bound derived there."""
import ctypes as C

import numpy as np
import pytest

import kv_pool_ref as R
import quantr_amd as Q

pytestmark = pytest.mark.gpu


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def filled(seed, lens, page=32, kv_heads=2, hd=64, n_layers=1, spare=2, shuffle=True):
    """A pool whose sequences hold random values of the given lengths."""
    rng = np.random.default_rng(seed)
    need = sum(-(-n // page) for n in lens)
    p = R.Pool(n_layers, max(1, need + spare), page, kv_heads, hd, len(lens),
               max(1, max(-(-n // page) for n in lens)) + 1, seed)
    order = rng.permutation(p.n_pages) if shuffle else np.arange(p.n_pages)
    at = 0
    for s, n in enumerate(lens):
        k = -(-n // page)
        p.table[s, :k] = order[at:at + k]
        p.len[s] = n
        at += k
        for g in p.table[s, :k]:
            p.refs[g] = 1
        for b in range(-(-n // R.BLOCK)):  # the blocks that hold tokens have values and scales
            g, bb = p.table[s, b * R.BLOCK // page], b * R.BLOCK % page // R.BLOCK
            p.data[:, g, :, bb] = np.clip(np.rint(rng.normal(0, 42, p.data[:, g, :, bb].shape)),
                                          -127, 127)
            p.scale[:, g, :, bb] = 0.02 * np.exp(rng.normal(0, 0.5, p.scale[:, g, :, bb].shape))
    return p


# ---- pages ------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed,page,kv_heads,hd,layers,n_pages", [
    (1, 16, 1, 32, 1, 40), (2, 32, 2, 64, 3, 24), (3, 256, 4, 128, 2, 12), (4, 64, 3, 96, 1, 9)])
def test_page_operations_follow_the_reference(dev, seed, page, kv_heads, hd, layers, n_pages):
    """A random program of extend, assign, trim and compact: every state equal."""
    rng = np.random.default_rng(seed)
    p = R.Pool(layers, n_pages, page, kv_heads, hd, 7, 6, seed)
    d = R.DevPool(dev, p)
    seen = set()
    for step in range(40):
        op = rng.choice(["extend", "extend", "extend", "assign", "trim", "compact"])
        n = int(rng.integers(1, 8))
        seqs = rng.permutation(7)[:n].tolist()
        if op == "extend":
            add = rng.choice([0, 1, int(rng.integers(1, 2 * page)), page], n).tolist()
            want, got = p.extend(seqs, add), d.extend(seqs, add)
        elif op == "assign":
            src = rng.integers(0, 7, n).tolist()
            want, got = p.assign(seqs, src), d.assign(seqs, src)
        elif op == "trim":
            keep = rng.choice([0, 1, page - 1, page, 3 * page], n).tolist()
            want, got = p.trim(seqs, keep), d.trim(seqs, keep)
        else:
            want, got = p.compact(), d.compact()
            np.testing.assert_array_equal(got[0], want[0])
            want, got = want[1], got[1]
        assert got == want, (step, op, seqs)
        seen.add((op, want if op != "compact" else 0))
        R.assert_same(d, p, "step %d %s" % (step, op))
    assert ("extend", R.OK) in seen


@pytest.mark.parametrize("listed", [[1, 2], [2, 1, 0], [0], [3, 2, 1, 0]])
def test_shared_last_page_is_copied_until_one_holder_is_left(dev, listed):
    p = filled(5, [37, 0, 0, 0], page=32, n_layers=2, spare=9)
    d = R.DevPool(dev, p)
    assert p.assign([1, 2, 3], [0, 0, 0]) == d.assign([1, 2, 3], [0, 0, 0]) == 0
    assert p.extend(listed, [1] * len(listed)) == d.extend(listed, [1] * len(listed)) == 0
    R.assert_same(d, p)
    tails = [p.table[s, 1] for s in range(4)]
    assert len(set(tails)) == (4 if len(listed) >= 3 else 1 + len(listed))


def test_extend_refuses_what_cannot_be(dev):
    p = filled(6, [37, 5, 0], page=32, spare=2)
    d = R.DevPool(dev, p)
    cap = p.max_pages * p.page
    for seqs, add, want in ([[0, 3], [1, 1], -1], [[0, -1], [1, 1], -1], [[1, 1], [1, 1], -1],
                            [[0], [-1], -1], [[1], [cap - 4], -1], [[1], [2 ** 31 - 1], -1],
                            [[0, 1, 2], [27, 28, 65], -3], [[0, 1, 2], [59, 60, 1], -3], [[0], [60], -1]):
        assert p.extend(seqs, add) == d.extend(seqs, add) == want, (seqs, add)
        R.assert_same(d, p, str(seqs))
    assert p.extend([2, 0], [1, 59]) == d.extend([2, 0], [1, 59]) == 0
    R.assert_same(d, p)


def test_lists_refuse_sequences_that_do_not_exist(dev):
    p = filled(7, [37, 5, 0], page=32)
    d = R.DevPool(dev, p)
    for dst, src in ([[0], [3]], [[3], [0]], [[-1], [0]], [[2, 2], [0, 1]]):
        assert p.assign(dst, src) == d.assign(dst, src) == -1
    for seqs, keep in ([[3], [0]], [[-1], [0]], [[0], [-1]]):
        assert p.trim(seqs, keep) == d.trim(seqs, keep) == -1
    R.assert_same(d, p)
    assert p.trim([0, 0, 1], [20, 33, 0]) == d.trim([0, 0, 1], [20, 33, 0]) == 0
    R.assert_same(d, p, "listed twice")
    for call in (p.extend, d.extend, p.assign, d.assign, p.trim, d.trim):
        assert call([], []) == 0
    R.assert_same(d, p, "empty lists")


def test_assign_reorders_in_place(dev):
    """A beam's step: every sequence is a source and a destination."""
    lens = [70, 40, 3, 0, 64, 33]
    p = filled(8, lens, page=16)
    d = R.DevPool(dev, p)
    dst, src = [0, 1, 2, 3, 4, 5], [5, 5, 0, 1, 2, 3]
    assert p.assign(dst, src) == d.assign(dst, src) == 0
    R.assert_same(d, p)


def test_many_sequences_in_one_list(dev):
    """Lists longer than a workgroup, a table wider than a pass."""
    n = 1500
    p = R.Pool(1, 5000, 16, 1, 32, n, 4, 1)
    d = R.DevPool(dev, p)
    rng = np.random.default_rng(2)
    order = rng.permutation(n).tolist()
    add = rng.integers(0, 50, n).tolist()
    assert p.extend(order, add) == d.extend(order, add) == 0
    R.assert_same(d, p)
    src = rng.integers(0, n, n).tolist()
    assert p.assign(order, src) == d.assign(order, src) == 0
    R.assert_same(d, p)
    add = rng.integers(0, 2, n).tolist()
    assert p.extend(order, add) == d.extend(order, add) == 0
    R.assert_same(d, p)
    got, want = d.compact(), p.compact()
    np.testing.assert_array_equal(got[0], want[0])
    assert got[1] == want[1]
    R.assert_same(d, p)


def test_large_extends(dev):
    """More free pages than fit the plan's LDS, reference counts beyond it."""
    p = R.Pool(1, 9000, 16, 1, 32, 5, 3000, 1)
    d = R.DevPool(dev, p)
    for seqs, add in (([3], [40000]), ([0, 1], [1, 16 * 2100 + 5]), ([4, 3, 0], [17, 3, 40]),
                      ([2], [16 * 2999]), ([2], [16 * 1700])):
        assert p.extend(seqs, add) == d.extend(seqs, add)
        R.assert_same(d, p, str(seqs))
    assert p.trim([3, 1], [900, 16 * 1500]) == d.trim([3, 1], [900, 16 * 1500])
    assert p.assign([2, 4], [1, 0]) == d.assign([2, 4], [1, 0]) == 0
    assert p.extend([2, 1, 4], [9, 9, 1]) == d.extend([2, 1, 4], [9, 9, 1])
    R.assert_same(d, p)


def test_reset_and_optional_outputs(dev):
    p = filled(9, [37, 5], page=32)
    d = R.DevPool(dev, p)
    dev.kv_pool_compact(d.h)
    p.compact()
    R.assert_same(d, p)
    s, k = d.list([0]), d.list([3])
    dev.kv_pool_trim(d.h, s.ptr, k.ptr, 1)
    p.trim([0], [3])
    R.assert_same(d, p)
    dev.kv_pool_reset(d.h)
    p.table[:], p.len[:], p.refs[:] = -1, 0, 0
    R.assert_same(d, p)


# ---- store and load -----------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page,old,new", [
    (16, [0, 1, 15, 16, 17, 40], [1, 1, 1, 1, 1, 1]),
    (64, [0, 5, 33, 16, 0, 70], [37, 0, 16, 15, 64, 3]),
    (256, [300, 0], [41, 290])])
def test_store_and_load(dev, hd, page, old, new):
    rng = np.random.default_rng(hd + page)
    kv = 3 if hd == 96 else 2
    p = filled(10, [o + m for o, m in zip(old, new)], page=page, kv_heads=kv, hd=hd, n_layers=2)
    d = R.DevPool(dev, p)
    seqs = rng.permutation(len(old)).tolist()
    m = [new[s] for s in seqs]
    start = starts(m)
    T = int(start[-1]) + 3  # rows behind the last sequence
    w = kv * hd
    k, v = (rng.normal(0, 1, (T, w + 8)).astype(np.float32) *
            np.exp(rng.normal(0, 1.5, (T, 1))).astype(np.float32) for _ in range(2))
    p.store(1, seqs, start, k, v)
    d.store(1, seqs, start, k, v)
    R.assert_same(d, p)
    # read back with the tokens before the new ones
    back = [min(int(p.len[s]), x + 20) for s, x in zip(seqs, m)]
    st = starts(back)
    T = int(st[-1]) + 2
    got = d.load(1, seqs, st, T)
    for i, s in enumerate(seqs):
        vals = p.values(s, 1)
        for side in (0, 1):
            want = vals[side][int(p.len[s]) - back[i]:].astype(np.float32)
            np.testing.assert_array_equal(got[side][st[i]:st[i + 1]], want)
    for side in (0, 1):
        assert (got[side][st[-1]:] == 7).all()


def test_store_halves_growth_and_extremes(dev):
    """Values on the rounding border, scales that grow over older values, zero
    blocks, the smallest and largest floats, NaN and infinities."""
    hd = 32
    p = filled(11, [40], page=32, kv_heads=1, hd=hd)
    d = R.DevPool(dev, p)
    rng = np.random.default_rng(3)

    def both(k, v):
        st = starts([k.shape[0]])
        with np.errstate(all="ignore"):
            p.store(0, [0], st, k, v)
        d.store(0, [0], st, k, v)
        R.assert_same(d, p)

    half = (rng.integers(-127, 127, (24, hd)) + 0.5).astype(np.float32)
    half[:, 0] = 127.0  # scale 1: every other value a tie
    both(half, half * np.float32(3.0))
    both(half[:3] * np.float32(1.7), half[:3] * np.float32(0.1))  # K grows, V does not
    both(half[:9] * np.float32(64), half[:9] * np.float32(1e30))
    both(np.zeros((40, hd), np.float32), np.zeros((40, hd), np.float32))
    tiny = (rng.integers(-300, 300, (17, hd)) * 2.0 ** -149).astype(np.float32)
    both(tiny, tiny * np.float32(1000))
    both(tiny[:1] * np.float32(2 ** 20), tiny[:1])
    big = (rng.normal(0, 1, (23, hd)) * 3e37).astype(np.float32)
    big[0, 0] = np.finfo(np.float32).max
    both(big, -big)
    odd = rng.normal(0, 1, (5, hd)).astype(np.float32)
    odd[0, :4] = [np.nan, np.inf, -np.inf, -np.nan]
    both(np.ascontiguousarray(odd), odd[::-1].copy())
    both(np.full((33, hd), np.nan, np.float32), np.full((33, hd), -np.inf, np.float32))


def test_rows_without_tokens(dev):
    """More rows than tokens, an empty sequence, one that does not exist, a table
    without a page: store skips, load gives zeros, attention zeros."""
    p = filled(12, [5, 0, 40], page=16, kv_heads=2, hd=64)
    p.table[2, 1] = -1
    d = R.DevPool(dev, p)
    rng = np.random.default_rng(4)
    seqs, m = [0, 1, 9, 2, -3], [9, 2, 3, 40, 1]
    st = starts(m)
    T = int(st[-1])
    k = rng.normal(0, 1, (T, 128)).astype(np.float32)
    d.store(0, seqs, st, k, k)
    want = p.copy()
    rows = np.concatenate([k[4:9], k[14:30], k[46:54]])
    want.store(0, [0], starts([5]), rows[:5], rows[:5])
    # sequence 2 page by page, the page that is missing left out
    full = filled(12, [5, 0, 40], page=16, kv_heads=2, hd=64)
    full.store(0, [2], starts([40]), k[14:54], k[14:54])
    g = [int(full.table[2, 0]), int(full.table[2, 2])]
    want.data[0, g], want.scale[0, g] = full.data[0, g], full.scale[0, g]
    np.testing.assert_array_equal(d.get("data"), want.data)
    np.testing.assert_array_equal(d.get("scale").view(np.uint32), want.scale.view(np.uint32))
    got = d.load(0, seqs, st, T)
    for x in got:
        assert (x[:4] == 0).all() and (x[9:14] == 0).all() and (x[-1] == 0).all()
        assert (x[14 + 16:14 + 32] == 0).all() and (x[14:30] != 0).any() and (x[4:9] != 0).any()
    q = rng.normal(0, 1, (T, 256)).astype(np.float32)
    out = d.attention(0, seqs, st, q, 4)
    assert (out[:4] == 0).all() and (out[9:14] == 0).all() and (out[-1] == 0).all()
    assert np.isfinite(out).all()
    # the tokens of the missing page are not seen: as if they were not there
    t, w = want.values(2, 0)[0], want.values(2, 0)[1]
    seen = np.r_[0:16, 32:40]
    for h in range(4):
        z = t[seen, h // 2] @ q[53, 64 * h:64 * h + 64].astype(np.float64) / 8
        e = np.exp(z - z.max())
        exp = e @ w[seen, h // 2] / e.sum()
        # scores of |z| < 40 in fp32 and the sum of 24: (10 * 40 + 64 + 24) 2^-24 of the values
        assert np.abs(out[53, h] - exp).max() <= 2 * 500 * 2.0 ** -24 * np.abs(w[seen]).max()


# ---- attention ------------------------------------------------------------------------------------
def check(d, p, seqs, counts, n_heads, seed, window=0, scale=0.0, max_len=0, pad=0, std=1.0, layer=0):
    rng = np.random.default_rng(seed)
    st = starts(counts)
    T = int(st[-1]) + pad
    q = (std * rng.normal(0, 1, (T, n_heads * p.hd + 4 * (pad > 0)))).astype(np.float32)
    got = d.attention(layer, seqs, st, q, n_heads, window=window, scale=scale, max_len=max_len)
    want = p.attention(layer, seqs, st, q, n_heads, window, scale)
    bound = R.attention_bound(p, layer, seqs, st, q, n_heads, window, scale)
    rows = int(st[-1])
    off = np.abs(got[:rows] - want[:rows]) - bound[:rows] - 2.0 ** -149
    assert (off <= 0).all(), "off by %.3g over a bound of %.3g at %s" % (
        np.abs(got[:rows] - want[:rows]).max(), bound.max(),
        np.unravel_index(off.argmax(), off.shape))
    assert (got[rows:] == 7).all()
    return got


@pytest.mark.parametrize("heads,kv,hd", [
    (8, 2, 64), (1, 1, 32), (6, 2, 96), (5, 1, 128), (16, 1, 64), (17, 1, 32), (40, 2, 32),
    (2, 2, 160), (3, 1, 192), (8, 1, 224), (4, 2, 256), (7, 7, 64)])
def test_attention_head_layouts(dev, heads, kv, hd):
    lens = [1, 70, 16, 129]
    p = filled(heads * hd, lens, page=32, kv_heads=kv, hd=hd)
    d = R.DevPool(dev, p)
    check(d, p, [3, 0, 1, 2], [1, 1, 1, 1], heads, 1)
    check(d, p, [2, 3], [5, 19], heads, 2, pad=3)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_attention_lengths_and_pages(dev, page):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700]
    p = filled(20 + page, lens, page=page, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    check(d, p, list(range(len(lens))), [1] * len(lens), 4, 1)


@pytest.mark.parametrize("counts", [[0, 3, 0, 129, 1], [64, 64, 64, 64, 64], [1, 2, 3, 5, 100]])
@pytest.mark.parametrize("window", [0, 1, 17, 64, 100])
def test_attention_of_several_rows_and_windows(dev, counts, window):
    lens = [300, 65, 64, 140, 101]
    p = filled(30, lens, page=16, kv_heads=1, hd=64)
    d = R.DevPool(dev, p)
    check(d, p, list(range(5)), counts, 4, window + 1, window=window)


def test_attention_of_long_sequences_in_parts(dev):
    """A token's work cut into parts, with a bound on the lengths that is right, loose and
    too small."""
    lens = [3001, 40, 1500]
    p = filled(31, lens, page=64, kv_heads=2, hd=64, n_layers=2)
    d = R.DevPool(dev, p)
    a = check(d, p, [0, 1, 2], [1, 1, 1], 16, 1, max_len=3001, layer=1)
    check(d, p, [0, 1, 2], [1, 1, 1], 16, 1, layer=1)
    check(d, p, [0, 1, 2], [1, 1, 1], 16, 1, max_len=64, layer=1)
    check(d, p, [2, 0], [1, 3], 16, 2, max_len=3001, window=700, layer=1)
    again = check(d, p, [0, 1, 2], [1, 1, 1], 16, 1, max_len=3001, layer=1)
    np.testing.assert_array_equal(a.view(np.uint32), again.view(np.uint32))


def test_attention_of_more_rounds_than_pages_are_held(dev):
    """A part of over 16384 tokens (the bound on the lengths is far too small),
    alone and behind a window."""
    p = filled(36, [17001, 40], page=16, kv_heads=1, hd=32)
    d = R.DevPool(dev, p)
    check(d, p, [0, 1], [1, 1], 2, 1, max_len=64)
    check(d, p, [1, 0], [2, 3], 2, 2, max_len=64, window=16900)


def test_rows_before_the_first_sequence(dev):
    """start[0] > 0: rows of nobody before the first sequence stay, others are found."""
    p = filled(37, [50, 7, 90], page=32, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    rng = np.random.default_rng(5)
    for st in ([5, 6, 7, 8], [21, 23, 23, 40], [3, 3, 3, 4]):
        st = np.array(st, np.int32)
        q = rng.normal(0, 1, (45, 4 * 64)).astype(np.float32)
        got = d.attention(0, [0, 1, 2], st, q, 4)
        want = p.attention(0, [0, 1, 2], st, q, 4)
        bound = R.attention_bound(p, 0, [0, 1, 2], st, q, 4)
        own = slice(st[0], st[-1])
        assert (np.abs(got[own] - want[own]) <= bound[own]).all()
        assert (got[:st[0]] == 7).all() and (got[st[-1]:] == 7).all()
        k = rng.normal(0, 1, (45, 128)).astype(np.float32)
        p.store(0, [0, 1, 2], st, k, -k)
        d.store(0, [0, 1, 2], st, k, -k)
        R.assert_same(d, p)
        back = d.load(0, [0, 1, 2], st, 45)
        for x in back:
            assert (x[:st[0]] == 7).all() and (x[st[-1]:] == 7).all()


def test_windows_beyond_any_length(dev):
    """The largest windows, with more rows than tokens, are no window."""
    p = filled(41, [2, 300, 0], page=16, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    none = check(d, p, [0, 1, 2], [5, 3, 2], 8, 3)
    assert (none[:3] == 0).all() and (none[3:8] != 0).any() and (none[8:] == 0).all()
    for window in (2 ** 31 - 1, 2 ** 30, 320, 319):
        got = check(d, p, [0, 1, 2], [5, 3, 2], 8, 3, window=window)
        np.testing.assert_array_equal(got.view(np.uint32), none.view(np.uint32))


def test_a_sequence_listed_twice_is_read_twice(dev):
    p = filled(42, [70, 45], page=32, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    check(d, p, [0, 1, 0, 0], [3, 2, 1, 40], 4, 4)
    k, v = d.load(0, [1, 1], starts([4, 2]), 6)
    for got in (k, v):
        np.testing.assert_array_equal(got[2:4], got[4:6])


def test_many_sequences_under_a_loose_bound(dev):
    """More tiles than parts are worth to, of a table for far longer sequences."""
    rng = np.random.default_rng(43)
    p = filled(43, [int(x) for x in rng.integers(0, 60, 300)], page=16, kv_heads=4, hd=32)
    p.table = np.concatenate([p.table, np.full((300, 4096 - p.max_pages), -1, np.int32)], 1)
    p.max_pages = 4096
    check(R.DevPool(dev, p), p, list(range(300)), [1] * 300, 4, 6)


def test_starts_that_are_not_ascending(dev):
    """Whatever `start` holds, no row that is not there is read or written."""
    p = filled(44, [90, 20, 40, 33], page=32, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    rng = np.random.default_rng(7)
    T, pad = 30, 4
    x = rng.normal(0, 1, (T + pad, 4 * 64)).astype(np.float32)
    for st in ([0, 20, 10, 2 ** 31 - 1, 5], [-2 ** 31, 30, -7, 12, 99], [31, 30, 29, 28, 27], [9] * 5,
               [0, 30, 0, 30, 0]):
        seqs, start = d.list([0, 1, 2, 3]), d.list(st)
        q, kv = dev.upload(x), dev.upload(x[:, :128].copy())
        out = dev.upload(np.full((T + pad, 256), 7, np.float32))
        back = [dev.upload(np.full((T + pad, 128), 7, np.float32)) for _ in range(2)]
        for max_len in (0, 16):
            dev.kv_pool_attention(d.h, 0, seqs.ptr, start.ptr, 4, T, 4, q.ptr, out.ptr,
                                  max_len=max_len)
        dev.kv_pool_store(d.h, 0, seqs.ptr, start.ptr, 4, T, kv.ptr, kv.ptr)
        dev.kv_pool_load(d.h, 0, seqs.ptr, start.ptr, 4, T, back[0].ptr, back[1].ptr)
        got = dev.download(out, (T + pad, 256), np.float32)
        assert np.isfinite(got).all() and (got[T:] == 7).all()
        for b in back:
            got = dev.download(b, (T + pad, 128), np.float32)
            assert np.isfinite(got).all() and (got[T:] == 7).all()


def test_attention_of_peaked_and_flat_scores(dev):
    p = filled(32, [500, 333], page=32, kv_heads=2, hd=128)
    d = R.DevPool(dev, p)
    for std, scale in ((0.0, 0.0), (1e-20, 0.0), (8.0, 0.0), (60.0, 0.0), (1.0, 1e-6), (1.0, 3.0),
                       (1e30, 1e-30)):
        check(d, p, [0, 1], [2, 1], 8, 5, std=std, scale=scale)


@pytest.mark.parametrize("std", [3e4, 4e5, 3e6, 2e7, 1e8, 3e9, 1e12, 1e30])
def test_attention_of_huge_scores(dev, std):
    """Scores far apart for fp32's spacing at their size: the leading token's values, V's
    scales unlike."""
    p = filled(46, [700, 300], page=32, kv_heads=2, hd=64)
    p.scale[:, :, :, :, 1] *= np.exp2(np.random.default_rng(2).integers(
        -12, 13, p.scale[:, :, :, :, 1].shape)).astype(np.float32)
    seqs, counts, heads = [0, 1], [3, 1], 8
    q = (std * np.random.default_rng(8).normal(0, 1, (4, heads * 64))).astype(np.float32)
    d = R.DevPool(dev, p)
    for window in (0, 500):
        got = d.attention(0, seqs, starts(counts), q, heads, window=window, max_len=700)
        for r, (s, pos) in enumerate(((0, 697), (0, 698), (0, 699), (1, 299))):
            k, v = p.values(s, 0)
            lo = max(0, pos - window + 1) if window else 0
            for h in range(heads):
                row = q[r, 64 * h:64 * h + 64].astype(np.float64)
                z = k[lo:pos + 1, h // 4] @ row / 8
                best, top = np.argmax(z), np.sort(z)[-2:]
                # a score is off by 3 e max |q| sum |k| and 10 e of itself (e = 2^-24)
                far = 2 * 2.0 ** -24 * (10 * np.abs(z).max() + 3 * np.abs(row).max() *
                                        np.abs(k[lo:pos + 1, h // 4]).sum(1).max() / 8)
                # beyond that, 40 more leave others e^-40, times V's 2^24 or so: below 2^-33
                if top[1] - top[0] < far + 40:
                    continue
                want = v[lo + best, h // 4]
                # exact digits: 2^-23 of the weight, few roundings of 2^-24, exp2's 2^-22
                assert np.abs(got[r, h] - want).max() <= 2.0 ** -20 * np.abs(want).max()


def test_attention_of_sinks(dev):
    """A token whose score leads all others by 2^5 to 2^90, first, last or amid rounds
    of 256 others, whose values are far smaller or larger than its own."""
    hd = 64
    for at, lead, own in ((0, 4.0, 1.0), (0, 20.0, 1.0), (0, 60.0, 1.0), (1200, 20.0, 1.0),
                          (700, 12.0, 1e-6), (0, 14.0, 1e-9), (300, 40.0, 1e-30), (0, 20.0, 1e6)):
        p = filled(45, [1201], page=32, kv_heads=1, hd=hd)
        q = np.random.default_rng(9).normal(0, 1, (1, 2 * hd)).astype(np.float32)
        g, b = p.table[0, at // 32], at // 16 % 2
        k = np.rint(127 * q[0, :hd] / np.abs(q[0, :hd]).max())
        p.data[0, g, 0, b, 0].reshape(16, hd)[at % 16] = k
        # the scale that gives it a score of lead + 4 (times ln 2 or so) for the first head
        p.scale[0, g, 0, b, 0] = (lead + 4) * np.sqrt(hd) / float(k @ q[0, :hd])
        p.scale[0, g, 0, b, 1] = 0.02 * own
        check(R.DevPool(dev, p), p, [0], [1], 2, 9)


def test_attention_of_unlike_blocks(dev):
    """Blocks of zeros, of the smallest and of large values beside ordinary ones."""
    p = filled(33, [200], page=32, kv_heads=1, hd=64)
    d0 = p.data.copy()
    for b, s in enumerate((0.0, 1e-3, 1e-30, 0.0, 1e3, 1e-12, 2e4, 1.0, 1e-3, 0.0, 1e-2, 1e-2, 0.0)):
        g, bb = p.table[0, b * 16 // 32], b % 2
        p.scale[0, g, 0, bb, 1] = s
        if s == 0:
            p.data[0, g, 0, bb, 1] = 0
    assert d0.shape == p.data.shape
    d = R.DevPool(dev, p)
    check(d, p, [0], [1], 4, 1)
    check(d, p, [0], [33], 4, 2)
    # tiny or no values before, beside and behind ones near the largest float
    for scales in ((0.0, 1e36, 1e-3, 0.0) * 3 + (0.0,), (1e36,) * 2 + (1e-36,) * 11,
                   (1e-38,) * 9 + (1e30,) * 4, (1e-44, 1e36) * 6 + (1e-44,)):
        for b, s in enumerate(scales):
            g, bb = p.table[0, b * 16 // 32], b % 2
            p.scale[0, g, 0, bb, 1] = s
        p.data[:] = d0
        d = R.DevPool(dev, p)
        check(d, p, [0], [1], 4, 3)
        check(d, p, [0], [40], 4, 4)
    for b in range(13):  # and nothing but zeros
        g, bb = p.table[0, b * 16 // 32], b % 2
        p.scale[0, g, 0, bb] = 0
        p.data[0, g, 0, bb] = 0
    assert (R.DevPool(dev, p).attention(0, [0], starts([1]), np.ones((1, 256), np.float32), 4) == 0).all()


def test_attention_of_rows_that_are_not_finite(dev):
    p = filled(34, [90], page=32, kv_heads=1, hd=64)
    d = R.DevPool(dev, p)
    q = np.random.default_rng(1).normal(0, 1, (6, 2 * 64)).astype(np.float32)
    good = d.attention(0, [0], starts([6]), q, 2)
    q[1, 3], q[2, 70], q[4, 127] = np.nan, np.inf, -np.inf
    out = d.attention(0, [0], starts([6]), q, 2)
    bad = np.zeros((6, 2), bool)
    bad[1, 0] = bad[2, 1] = bad[4, 1] = True
    assert np.isnan(out[bad]).all()
    np.testing.assert_array_equal(out[~bad], good[~bad])


def test_attention_reads_64_bit_offsets(dev):
    """A pool whose last page lies beyond 4 GiB."""
    hd, page = 64, 65536
    n_pages = 520  # of 8.4 MB: 4.4 GB
    page_bytes = page * 2 * hd
    data, scale = dev.alloc(n_pages * page_bytes), dev.alloc(n_pages * page // 16 * 8)
    p = filled(35, [100], page=128, kv_heads=1, hd=hd, spare=0)
    table, ln, refs = (dev.upload(np.full(1, v, np.int32)) for v in (n_pages - 1, 100, 1))
    refs = dev.upload(np.zeros(n_pages, np.int32))
    small = R.DevPool(dev, p)
    h = Q.KvPool(n_layers=1, n_pages=n_pages, page=page, n_kv_heads=1, head_dim=hd, n_seqs=1,
                 max_pages=1, data=data.ptr, scale=scale.ptr, table=table.ptr, len=ln.ptr,
                 refs=refs.ptr)
    rng = np.random.default_rng(5)
    k, v = (rng.normal(0, 1, (100, hd)).astype(np.float32) for _ in range(2))
    st, kd, vd = dev.upload(starts([100])), dev.upload(k), dev.upload(v)
    q = dev.upload(rng.normal(0, 1, (100, hd)).astype(np.float32))
    outs = []
    for pool in (h, small.h):
        out = dev.alloc(100 * hd * 4)
        dev.kv_pool_store(pool, 0, None, st.ptr, 1, 100, kd.ptr, vd.ptr)
        dev.kv_pool_attention(pool, 0, None, st.ptr, 1, 100, 1, q.ptr, out.ptr, max_len=100)
        outs.append(dev.download(out, (100, hd), np.float32))
    np.testing.assert_array_equal(outs[0], outs[1])


# ---- together -----------------------------------------------------------------------------------------
def test_a_search_step_by_step_and_captured(dev):
    """Beams over one prompt: prompt stored and attended, then steps of reorder,
    extend, store, attention, log probabilities of the outputs as logits -- the same
    results eager, and as one graph replayed three times with eager work
    between."""
    hd, heads, kv, beams, V = 64, 8, 2, 4, 512
    rng = np.random.default_rng(11)
    p = R.Pool(1, 40, 16, kv, hd, beams, 8, 3)
    d = R.DevPool(dev, p)
    w = kv * hd
    P = 37
    assert p.extend([0], [P]) == d.extend([0], [P]) == 0
    k, v = (rng.normal(0, 1, (P, w)).astype(np.float32) for _ in range(2))
    p.store(0, [0], starts([P]), k, v)
    d.store(0, [0], starts([P]), k, v)
    check(d, p, [0], [P], heads, 12)
    assert p.assign([1, 2, 3], [0, 0, 0]) == d.assign([1, 2, 3], [0, 0, 0]) == 0
    R.assert_same(d, p)

    rows = [rng.normal(0, 1, (beams, w)).astype(np.float32) for _ in range(2)]
    q = rng.normal(0, 1, (beams, heads * hd)).astype(np.float32)
    bufs = dict(dst=d.list(range(beams)), src=d.list([0, 0, 2, 1]), add=d.list([1] * beams),
                start=d.list(range(beams + 1)), k=dev.upload(rows[0]), v=dev.upload(rows[1]),
                q=dev.upload(q), out=dev.alloc(beams * V * 4), t=d.list([3, 500, 77, 0]),
                lp=dev.alloc(64), ent=dev.alloc(64), rank=dev.alloc(64), tid=dev.alloc(64),
                tlp=dev.alloc(64), st=d.list([5, 5]))

    def step():
        b = {n: x.ptr for n, x in bufs.items()}
        dev.kv_pool_assign(d.h, b["dst"], b["src"], beams, b["st"])
        dev.kv_pool_extend(d.h, b["dst"], b["add"], beams, b["st"] + 4)
        dev.kv_pool_store(d.h, 0, b["dst"], b["start"], beams, beams, b["k"], b["v"])
        dev.kv_pool_attention(d.h, 0, b["dst"], b["start"], beams, beams, heads, b["q"], b["out"],
                              max_len=8 * 16)
        dev.logprobs(b["out"], beams, V, b["t"], b["lp"], b["ent"], b["rank"], 2, b["tid"], b["tlp"])
        dev.kv_pool_compact(d.h)

    def verify():
        assert p.assign([0, 1, 2, 3], [0, 0, 2, 1]) == 0
        assert p.extend([0, 1, 2, 3], [1] * 4) == 0
        p.store(0, range(beams), starts([1] * beams), *rows)
        want = p.attention(0, range(beams), starts([1] * beams), q, heads)
        bound = R.attention_bound(p, 0, range(beams), starts([1] * beams), q, heads)
        p.compact()
        dev.sync()
        R.assert_same(d, p)
        got = dev.download(bufs["out"], (beams, heads, hd), np.float32)
        assert (np.abs(got - want) <= bound).all()
        lp = R.logprobs(got.reshape(beams, V), [3, 500, 77, 0], 2)
        assert np.abs(dev.download(bufs["lp"], (beams,), np.float32) - lp[0]).max() < 1e-4
        np.testing.assert_array_equal(dev.download(bufs["rank"], (beams,), np.int32), lp[2])
        np.testing.assert_array_equal(dev.download(bufs["tid"], (beams, 2), np.int32), lp[3])
        np.testing.assert_array_equal(dev.download(bufs["st"], (2,), np.int32), [0, 0])

    step()
    verify()
    g = dev.capture(step)
    try:
        for _ in range(3):
            dev.graph_launch(g)
            verify()
            check(d, p, [1, 3], [2, 1], heads, 13)
            dev.sync()
    finally:
        dev.graph_destroy(g)


def test_parts_captured_and_replayed(dev):
    """Calls whose work is cut into parts share the context's scratch: one after the other in
    a graph, replayed with eager calls of other sizes between."""
    p = filled(47, [3001, 90, 700], page=64, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    rng = np.random.default_rng(3)
    q = rng.normal(0, 1, (3, 8 * 64)).astype(np.float32)
    x = rng.normal(0, 3, (2, 60000)).astype(np.float32)
    seqs, start = d.list([0, 1, 2]), d.list([0, 1, 2, 3])
    dq, dx, t = dev.upload(q), dev.upload(x), d.list([77, 59999])
    add, none = d.list([0, 0, 0]), d.list([9])
    outs = [dev.alloc(3 * 512 * 4), dev.alloc(8), dev.alloc(8), dev.alloc(2 * 20 * 4)]

    def step():
        dev.kv_pool_extend(d.h, seqs.ptr, add.ptr, 3, none.ptr)
        dev.kv_pool_attention(d.h, 0, seqs.ptr, start.ptr, 3, 3, 8, dq.ptr, outs[0].ptr, max_len=3001)
        dev.logprobs(dx.ptr, 2, 60000, t.ptr, outs[1].ptr, None, outs[2].ptr, 20, outs[3].ptr)

    def results():
        dev.sync()
        return [dev.download(b, (n,), np.uint32) for b, n in zip(outs, (3 * 512, 2, 2, 40))]

    step()
    want = results()
    exact = p.attention(0, [0, 1, 2], starts([1, 1, 1]), q, 8)
    bound = R.attention_bound(p, 0, [0, 1, 2], starts([1, 1, 1]), q, 8)
    assert (np.abs(want[0].view(np.float32).reshape(3, 8, 64) - exact) <= bound).all()
    np.testing.assert_array_equal(want[3].view(np.int32).reshape(2, 20),
                                  np.argsort(-x, 1, kind="stable")[:, :20])
    g = dev.capture(step)
    try:
        for i in range(3):
            dev.graph_launch(g)
            for got, w in zip(results(), want):
                np.testing.assert_array_equal(got, w)
            check(d, p, [2, 0], [1 + i, 2], 8, 30 + i)
            dev.logprobs(dx.ptr, 1, 50000 + i, t.ptr, outs[1].ptr, None, outs[2].ptr, 20, outs[3].ptr)
            dev.sync()
    finally:
        dev.graph_destroy(g)


def test_another_stream_and_context(dev):
    """Two contexts on one device, one of them on the other's stream, share a pool."""
    p = filled(40, [77, 130], page=32, kv_heads=2, hd=64)
    d = R.DevPool(dev, p)
    other = Q.Device(0)
    try:
        other.set_stream(dev.lib.qr_ctx_get_stream(dev.ctx))
        e = R.DevPool(dev, p)
        e.dev = other
        e.h = d.h
        check(e, p, [0, 1], [1, 3], 4, 1)
        assert p.extend([0], [60]) == e.extend([0], [60])
        R.assert_same(d, p)
        other.set_stream(None)
        assert dev.lib.qr_ctx_get_stream(C.c_void_p(other.ctx)) != dev.lib.qr_ctx_get_stream(
            C.c_void_p(dev.ctx))
    finally:
        other.close()
