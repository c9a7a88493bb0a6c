"""A shared 8-bit KV pool and log probabilities from their definitions, in 64
bits and one step at a time, and the same pool on the device."""
import math

import numpy as np

import quantr_amd as Q

BLOCK = 16
OK, INVALID, NOMEM = 0, -1, -3


class Pool:
    """The state of a pool as numpy arrays; the operations list entry by list
    entry, page by page."""

    def __init__(self, n_layers=1, n_pages=16, page=32, kv_heads=2, hd=64, n_seqs=4, max_pages=8,
                 seed=0):
        self.n_layers, self.n_pages, self.page = n_layers, n_pages, page
        self.kv_heads, self.hd, self.n_seqs, self.max_pages = kv_heads, hd, n_seqs, max_pages
        rng = np.random.default_rng(seed)
        shape = (n_layers, n_pages, kv_heads, page // BLOCK, 2)
        # what no call has written holds anything
        self.data = rng.integers(-128, 128, shape + (BLOCK * hd,), dtype=np.int8)
        self.scale = np.where(rng.random(shape) < 0.5, np.nan, 1e30).astype(np.float32)
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        self.len = np.zeros(n_seqs, np.int32)
        self.refs = np.zeros(n_pages, np.int32)

    def copy(self):
        p = object.__new__(Pool)
        p.__dict__.update({k: v.copy() if isinstance(v, np.ndarray) else v
                           for k, v in self.__dict__.items()})
        return p

    def pages(self, tokens):
        return -(-int(tokens) // self.page)

    # ---- pages
    def extend(self, seqs, add):
        if len(set(seqs)) < len(seqs):
            return INVALID
        for s, a in zip(seqs, add):
            if not 0 <= s < self.n_seqs or a < 0:
                return INVALID
            if int(self.len[s]) + a > self.max_pages * self.page:
                return INVALID
        p = self.copy()
        free = [i for i in range(p.n_pages) if p.refs[i] == 0]
        for s, a in zip(seqs, add):
            n = int(p.len[s])
            if a > 0 and n % p.page:
                old = p.table[s, n // p.page]
                if p.refs[old] > 1:
                    if not free:
                        return NOMEM
                    new = free.pop(0)
                    p.data[:, new], p.scale[:, new] = p.data[:, old], p.scale[:, old]
                    p.refs[old] -= 1
                    p.refs[new] = 1
                    p.table[s, n // p.page] = new
            for c in range(p.pages(n), p.pages(n + a)):
                if not free:
                    return NOMEM
                p.table[s, c] = free.pop(0)
                p.refs[p.table[s, c]] = 1
            p.len[s] = n + a
        self.__dict__.update(p.__dict__)
        return OK

    def assign(self, dst, src):
        if len(set(dst)) < len(dst) or not all(0 <= s < self.n_seqs for s in list(dst) + list(src)):
            return INVALID
        rows, lens = self.table.copy(), self.len.copy()
        for d, s in zip(dst, src):
            for g in self.table[d]:
                if g >= 0:
                    self.refs[g] -= 1
            for g in rows[s]:
                if g >= 0:
                    self.refs[g] += 1
            self.table[d], self.len[d] = rows[s], lens[s]
        return OK

    def trim(self, seqs, keep):
        if not all(0 <= s < self.n_seqs for s in seqs) or not all(k >= 0 for k in keep):
            return INVALID
        for s, k in zip(seqs, keep):
            self.len[s] = min(self.len[s], k)
            for c in range(self.pages(self.len[s]), self.max_pages):
                if self.table[s, c] >= 0:
                    self.refs[self.table[s, c]] -= 1
                    self.table[s, c] = -1
        return OK

    def compact(self):
        live = int((self.refs > 0).sum())
        to = np.where(self.refs > 0, np.arange(self.n_pages), -1).astype(np.int32)
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, self.n_pages) if self.refs[i] > 0]
        for src, dst in zip(movers, holes):
            self.data[:, dst], self.scale[:, dst] = self.data[:, src], self.scale[:, src]
            self.refs[dst], self.refs[src] = self.refs[src], 0
            to[src] = dst
        for e in np.ndindex(self.table.shape):
            if self.table[e] >= 0:
                self.table[e] = to[self.table[e]]
        return to, live

    # ---- values
    def place(self, s, pos, kvh, layer, side):
        """Where a token's values lie: an index of data and one of scale."""
        g = self.table[s, pos // self.page]
        b, t = pos % self.page // BLOCK, pos % BLOCK
        vals = slice(t * self.hd, (t + 1) * self.hd) if side == 0 else slice(t, None, BLOCK)
        return (layer, g, kvh, b, side, vals), (layer, g, kvh, b, side)

    def values(self, s, layer):
        """K and V of a sequence, float64 [2][len][kv head][hd]."""
        n, hd = int(self.len[s]), self.hd
        out = np.zeros((2, n, self.kv_heads, hd))
        for t0 in range(0, n, BLOCK):
            g, b = self.table[s, t0 // self.page], t0 % self.page // BLOCK
            for h in range(self.kv_heads):
                d, sc = self.data[layer, g, h, b].astype(np.float64), self.scale[layer, g, h, b]
                k, v = d[0].reshape(BLOCK, hd), d[1].reshape(hd, BLOCK).T
                used = min(BLOCK, n - t0)
                out[0, t0:t0 + used, h] = k[:used] * np.float64(sc[0])
                out[1, t0:t0 + used, h] = v[:used] * np.float64(sc[1])
        return out

    def store(self, layer, seqs, start, k, v):
        for i, s in enumerate(seqs):
            m, n = start[i + 1] - start[i], int(self.len[s])
            for b in range(max(0, n - m) // BLOCK, (n - 1) // BLOCK + 1 if n and m else 0):
                new = [t for t in range(b * BLOCK, min(n, b * BLOCK + BLOCK)) if t >= n - m]
                old = [t for t in range(b * BLOCK, n - m)]
                for h in range(self.kv_heads):
                    for side, rows in ((0, k), (1, v)):
                        x = np.stack([rows[start[i] + t - (n - m), h * self.hd:(h + 1) * self.hd]
                                      for t in new])
                        self._block(layer, s, h, side, old, new, x)

    def _block(self, layer, s, h, side, old, new, x):
        sc = self.place(s, new[0], h, layer, side)[1]
        before = self.scale[sc] if old else np.float32(0)
        a = np.abs(x[np.isfinite(x)])
        top = np.float32(np.float64(a.max() if a.size else 0) / 127.0)
        after = max(before, top)
        if after > before:
            for t in old:
                at = self.place(s, t, h, layer, side)[0]
                q = self.data[at].astype(np.float64) * np.float64(before)
                self.data[at] = np.rint(q / np.float64(after))
        for t, row in zip(new, x):
            with np.errstate(all="ignore"):
                q = np.rint(row.astype(np.float64) / np.float64(after)) if after > 0 else (
                    np.zeros(self.hd))
            q = np.clip(np.where(np.isnan(row), 0, np.where(np.isinf(row), np.sign(row) * 127, q)),
                        -127, 127)
            self.data[self.place(s, t, h, layer, side)[0]] = q if after > 0 else 0
        self.scale[sc] = after

    def attention(self, layer, seqs, start, q, n_heads, window=0, scale=0.0):
        """float64 [rows][n_heads][hd]; rows that no sequence owns are NaN."""
        out = np.full((q.shape[0], n_heads, self.hd), np.nan)
        c = scale if scale > 0 else 1.0 / math.sqrt(self.hd)
        for i, s in enumerate(seqs):
            k, v = self.values(s, layer)
            m, n = start[i + 1] - start[i], int(self.len[s])
            for r in range(m):
                pos = n - m + r
                lo = max(0, pos - window + 1) if window else 0
                for h in range(n_heads):
                    kh = h * self.kv_heads // n_heads
                    if pos < 0:
                        out[start[i] + r, h] = 0
                        continue
                    row = q[start[i] + r, h * self.hd:(h + 1) * self.hd].astype(np.float64)
                    z = k[lo:pos + 1, kh] @ row * c
                    w = np.exp(z - z.max())
                    out[start[i] + r, h] = (w @ v[lo:pos + 1, kh]) / w.sum()
        return out


class DevPool:
    """A copy of a Pool's state on the device."""

    def __init__(self, dev, p):
        self.dev, self.p = dev, p
        self.bufs = {k: dev.upload(getattr(p, k)) for k in ("data", "scale", "table", "len", "refs")}
        self.h = Q.KvPool(n_layers=p.n_layers, n_pages=p.n_pages, page=p.page,
                          n_kv_heads=p.kv_heads, head_dim=p.hd, n_seqs=p.n_seqs,
                          max_pages=p.max_pages, **{k: b.ptr for k, b in self.bufs.items()})
        self.status = dev.upload(np.full(4, 77, np.int32))

    def list(self, v):
        return self.dev.upload(np.asarray(v, np.int32).reshape(-1)) if len(v) else self.status

    def get(self, name):
        a = getattr(self.p, name)
        return self.dev.download(self.bufs[name], a.shape, a.dtype)

    def status_of(self, call, a, b):
        a_, b_ = self.list(a), self.list(b)
        call(self.h, a_.ptr, b_.ptr, len(a), self.status.ptr)
        return int(self.dev.download(self.status, (1,), np.int32)[0])

    def extend(self, seqs, add):
        return self.status_of(self.dev.kv_pool_extend, seqs, add)

    def assign(self, dst, src):
        return self.status_of(self.dev.kv_pool_assign, dst, src)

    def trim(self, seqs, keep):
        return self.status_of(self.dev.kv_pool_trim, seqs, keep)

    def compact(self):
        to = self.dev.upload(np.zeros(self.p.n_pages, np.int32))
        self.dev.kv_pool_compact(self.h, to.ptr, self.status.ptr)
        return (self.dev.download(to, (self.p.n_pages,), np.int32),
                int(self.dev.download(self.status, (1,), np.int32)[0]))

    def store(self, layer, seqs, start, k, v):
        s, st, kd, vd = self.list(seqs), self.list(start), self.dev.upload(k), self.dev.upload(v)
        self.dev.kv_pool_store(self.h, layer, s.ptr, st.ptr, len(seqs), k.shape[0], kd.ptr, vd.ptr,
                               stride=k.shape[1])
        self.dev.sync()

    def load(self, layer, seqs, start, T):
        w = self.p.kv_heads * self.p.hd
        s, st = self.list(seqs), self.list(start)
        k = self.dev.upload(np.full((T, w), 7, np.float32))
        v = self.dev.upload(np.full((T, w), 7, np.float32))
        self.dev.kv_pool_load(self.h, layer, s.ptr, st.ptr, len(seqs), T, k.ptr, v.ptr)
        return [self.dev.download(b, (T, self.p.kv_heads, self.p.hd), np.float32) for b in (k, v)]

    def attention(self, layer, seqs, start, q, n_heads, window=0, scale=0.0, max_len=0, fill=7.0):
        T = q.shape[0]
        s, st, qd = self.list(seqs), self.list(start), self.dev.upload(q)
        out = self.dev.upload(np.full((T, n_heads * self.p.hd), fill, np.float32))
        self.dev.kv_pool_attention(self.h, layer, s.ptr, st.ptr, len(seqs), T, n_heads, qd.ptr,
                                   out.ptr, max_len=max_len, window=window, scale=scale,
                                   q_stride=q.shape[1])
        return self.dev.download(out, (T, n_heads, self.p.hd), np.float32)


def assert_same(d, p, what=""):
    """The device pool holds the reference's state, bit for bit."""
    for name in ("table", "len", "refs", "data"):
        np.testing.assert_array_equal(d.get(name), getattr(p, name), err_msg="%s %s" % (what, name))
    np.testing.assert_array_equal(d.get("scale").view(np.uint32), p.scale.view(np.uint32),
                                  err_msg="%s scale" % what)


def attention_bound(p, layer, seqs, start, q, n_heads, window=0, scale=0.0):
    """How far the 8-bit products' attention may be off per output element:
    [rows][n_heads][hd].  e = 2^-24, c the scale, z the scores.

    q is held to half a step of its row's largest value / 8355711, after two
    roundings of up to a step: 3 e max |q| each, so a score to 3 e c max |q| sum |k_j|.
    The integer products are exact; joining them, the factors and the exponent's
    sums round z seven times, its power of two (with V's, |ev| <= 60) three times: dz =
    that + 10 e |z| + 64 e.  exp2 is good to 2^-22.  A weight off by the factor 1 + x moves
    an output by up to 2 x sum w |v| / sum w (numerator and denominator).  fp32 sums add
    (n / 64 + 40) e of sum w |v| / sum w.  A weight is rounded to half of 1 / 4177800 of the
    largest weight with its V scale: n 2^-23 max(w 127 vs) / sum w."""
    out = np.zeros((q.shape[0], n_heads, p.hd))
    c = scale if scale > 0 else 1.0 / math.sqrt(p.hd)
    e = 2.0 ** -24
    for i, s in enumerate(seqs):
        k, v = p.values(s, layer)
        m, n = start[i + 1] - start[i], int(p.len[s])
        vs = np.array([[p.scale[layer, p.table[s, t // p.page], h, t % p.page // BLOCK, 1]
                        for h in range(p.kv_heads)] for t in range(n)], np.float64)
        for r in range(m):
            pos = n - m + r
            lo = max(0, pos - window + 1) if window else 0
            for h in range(n_heads if pos >= 0 else 0):
                kh = h * p.kv_heads // n_heads
                row = q[start[i] + r, h * p.hd:(h + 1) * p.hd].astype(np.float64)
                kk, vv = k[lo:pos + 1, kh], np.abs(v[lo:pos + 1, kh])
                z = kk @ row * c
                dz = 3 * e * c * np.abs(row).max() * np.abs(kk).sum(1) + 10 * e * np.abs(z) + 64 * e
                w = np.exp(z - z.max())
                mean = (w @ vv) / w.sum()
                out[start[i] + r, h] = mean * (2 * dz.max() + 2 * 2.0 ** -22 + (n / 64 + 40) * e)
                out[start[i] + r, h] += (n * 2.0 ** -23 * 127 *
                                         (w * vs[lo:pos + 1, kh]).max() / w.sum())
    return out


def logprobs(x, targets, n_top):
    """lp, entropy, rank, top_id, top_lp of rows, in 64 bits."""
    R, V = x.shape
    lp, ent, rank = np.zeros(R), np.zeros(R), np.full(R, -1, np.int32)
    tid, tlp = np.full((R, n_top), -1, np.int32), np.full((R, n_top), -np.inf)
    for r in range(R):
        row = x[r].astype(np.float64)
        bad = bool((np.isnan(row) | (row == np.inf)).any())
        key = np.where(np.isnan(row), -np.inf, row)
        order = np.lexsort((np.arange(V), -key))
        m = key.max()
        with np.errstate(all="ignore"):
            if m == -np.inf:
                z = np.full(V, -np.inf)
            else:
                z = row - m - np.log(np.exp(row - m).sum())
            p = np.exp(z)
            ent[r] = np.nan if bad else -np.where(p > 0, p * z, 0).sum()
        t = int(targets[r])
        if 0 <= t < V:
            lp[r] = np.nan if bad else z[t]
            rank[r] = int((key > key[t]).sum() + (key[:t] == key[t]).sum())
        k = min(n_top, V)
        tid[r, :k] = order[:k]
        tlp[r, :k] = np.nan if bad else z[order[:k]]
    return lp, ent, rank, tid, tlp
