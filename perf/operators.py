"""Serving several sequences from one cache: the page operations of a pool that sequences share
(take pages, fork, cut back, compact), the pool's 8-bit rows with one scale per 16 tokens and head
(store, load, attention of a ragged batch), and the log probabilities by which continuations are
chosen.

`run` makes the library's calls where `own` is true and computes the same in elementary torch
operations otherwise; `exact` computes them from their definitions in 64 bits.

The pool: data int8 [layer][page][kv head][page / 16][2][16 * head_dim], a block of 16 tokens as its
K rows [16][head_dim] and then its V columns [head_dim][16]; scale fp32 [layer][page][kv head]
[page / 16][2]; table int32 [sequence][max_pages] (-1: no page), len int32 [sequence], refs int32
[page], the table entries that name a page.  A cached value is q * scale.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 16

# (heads, kv heads, head_dim): the two models of this repository's benchmark, then generic layouts
SHAPES = {"moe": (32, 4, 128), "dense": (32, 4, 64)}
GENERIC = [(32, 4, 128), (32, 4, 64), (40, 8, 128), (16, 2, 256), (8, 8, 96), (20, 5, 64),
           (32, 1, 64), (24, 8, 128), (48, 8, 32)]


def _att(name, shape, page, n, max_len, new, window=0, fused=False):
    h, kh, hd = shape
    return dict(name=name, kind="attention", heads=h, kv_heads=kh, hd=hd, page=page, n=n,
                max_len=max_len, new=new, window=window, fused=fused)


def listed():
    return [
        # one sequence of a dense model decodes mid-conversation: launch and latency
        _att("attend_1x702_hd64", SHAPES["dense"], 256, 1, 702, 1),
        # a batch of 32 conversations of mixed lengths decodes one token each
        _att("attend_32x4096_hd128", SHAPES["moe"], 256, 32, 4096, 1, fused=True),
        # one long document: the work of one token split over its length
        _att("attend_1x32768_hd128", SHAPES["moe"], 256, 1, 32768, 1),
        # speculative verification: up to five tokens of each of 24 sequences, sliding window,
        # small pages
        _att("verify_24x2047_window", SHAPES["dense"], 16, 24, 2047, 5, window=1000),
        # a 512-token prompt chunk far into its cache, an odd length
        _att("prompt_512_at_1501", SHAPES["moe"], 256, 1, 2013, 512, fused=True),
        # the step of a 64-sequence batch stores one token of each sequence
        dict(name="store_64x1", kind="store", kv_heads=4, hd=128, page=256, n=64, max_len=2048,
             new=1),
        # four prompts of up to 512 tokens stored, odd tails
        dict(name="store_4x509", kind="store", kv_heads=4, hd=128, page=64, n=4, max_len=1501,
             new=509),
        # best-of-8 from each of 8 prompts: the children of the last step cut back, forked again,
        # and given room (their shared last pages copied)
        dict(name="fork_8x8", kind="pages", parents=8, children=8, length=1001, add=7, page=256,
             layers=4, kv_heads=4, hd=128, spare=16),
        # a pool with holes after many sequences ended, compacted over 8 layers
        dict(name="compact_400", kind="compact", n_pages=400, n=24, live=0.6, page=256, layers=8,
             kv_heads=4, hd=128),
        # one decoded token of a large vocabulary with its 20 best alternatives
        dict(name="logprobs_1x151936", kind="logprobs", rows=1, vocab=151936, top=20, masked=0.0,
             pad=0),
        # a batch's logits of a small vocabulary, half of it masked out by a grammar, padded rows
        dict(name="logprobs_17x32000_masked", kind="logprobs", rows=17, vocab=32000, top=5,
             masked=0.5, pad=13),
        # every position of a 512-token prompt scored
        dict(name="logprobs_512x151936", kind="logprobs", rows=512, vocab=151936, top=20,
             masked=0.0, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "store", "pages", "compact",
                       "logprobs", "logprobs"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "attention":
        h, kh, hd = rng.choice(GENERIC)
        new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
        n = _log(rng, 1, 48) if new < 9 else rng.randint(1, 3)
        # at most the cached values of the largest listed batch, or the products of its prompt
        most = 32 * 4096 * 4 * 128 // (n * kh * hd)
        most = min(most, 512 * 2013 * 32 * 128 // (n * new * h * hd), 32768)
        max_len = max(new, _log(rng, 1, max(2, most)))
        return dict(kind=kind, heads=h, kv_heads=kh, hd=hd, page=page, n=n, max_len=max_len,
                    new=new, window=rng.choice([0, 0, 0, _log(rng, 1, 2048)]),
                    fused=rng.random() < 0.5)
    if kind == "store":
        _, kh, hd = rng.choice(GENERIC)
        new = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 509)])
        n = _log(rng, 1, 64) if new < 9 else rng.randint(1, 4)
        return dict(kind=kind, kv_heads=kh, hd=hd, page=page, n=n,
                    max_len=max(new, _log(rng, 1, 2048)), new=new)
    if kind == "pages":
        return dict(kind=kind, parents=rng.randint(1, 8), children=rng.randint(1, 8),
                    length=_log(rng, 1, 1500), add=_log(rng, 1, 300), page=page,
                    layers=rng.randint(1, 4), kv_heads=rng.choice([1, 2, 4]),
                    hd=rng.choice([64, 96, 128]), spare=rng.randint(0, 40))
    if kind == "compact":
        return dict(kind=kind, n_pages=_log(rng, 5, 400), n=rng.randint(1, 24),
                    live=round(rng.uniform(0.05, 0.95), 2), page=page, layers=rng.randint(1, 8),
                    kv_heads=rng.choice([1, 2, 4]), hd=rng.choice([64, 96, 128]))
    vocab = _log(rng, 100, 151936)
    return dict(kind=kind, rows=_log(rng, 1, 512), vocab=vocab,
                top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                masked=rng.choice([0.0, 0.0, 0.5, 0.99]), pad=rng.choice([0, rng.randint(1, 40)]))


# ---- what a program has in hand -----------------------------------------------------------------
_STREAM = []
_DEV = []


def _stream():
    """The program's one stream, which torch and the library share."""
    if not _STREAM:
        _STREAM.append(torch.cuda.Stream())
    if torch.cuda.current_stream() != _STREAM[0]:
        torch.cuda.set_stream(_STREAM[0])


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "quantr-in-c_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import quantr_amd
    return quantr_amd


def _dev():
    if not _DEV:
        _DEV.append(_lib().Device(0))
        _DEV[0].set_stream(_STREAM[0].cuda_stream)
    return _DEV[0]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(case):
    """Each sequence's tokens in the cache (the first has the most) and its new ones among them."""
    r = random.Random(case["n"] * 1000003 + case["max_len"] * 101 + case["new"])
    lens, news = [case["max_len"]], [case["new"]]
    for _ in range(case["n"] - 1):
        n = _log(r, max(1, case["max_len"] / 8), case["max_len"])
        lens.append(n)
        news.append(min(n, r.randint(max(1, case["new"] // 2), case["new"])))
    return lens, news


def _starts(counts):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return s


def _pool(g, layers, n_pages, kh, page, hd):
    data = (torch.randn((layers, n_pages, kh, page // BLOCK, 2, BLOCK * hd), device="cuda",
                        generator=g) * 42).round_().clamp_(-127, 127).to(torch.int8)
    scale = 0.02 * torch.exp(0.4 * torch.randn((layers, n_pages, kh, page // BLOCK, 2),
                                               device="cuda", generator=g))
    return data, scale


def _owned(g, lens, page, n_pages, max_pages):
    """A table over randomly ordered pages, the lengths and the reference counts."""
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        k = -(-n // page)
        table[i, :k] = order[at:at + k]
        at += k
    refs[order[:at].long()] = 1
    return table, _i32(lens), refs


def _prepare_cache(case, seed):
    g = _gen(seed)
    lens, news = _lengths(case)
    page, kh, hd, n = case["page"], case["kv_heads"], case["hd"], case["n"]
    n_pages = sum(-(-x // page) for x in lens) + 3
    data, scale = _pool(g, 2, n_pages, kh, page, hd)
    table, length, refs = _owned(g, lens, page, n_pages, -(-max(lens) // page) + 1)
    s = dict(case=case, data=data, scale=scale, table=table, len=length, refs=refs, layer=1,
             seqs=_i32(random.Random(seed).sample(range(n), n)), max_len=max(lens))
    order = s["seqs"].tolist()
    s["news"] = [news[i] for i in order]
    s["start"] = _i32(_starts(s["news"]))
    T = sum(news)
    if case["kind"] == "attention":
        qd = case["heads"] * hd
        # with `fused`, the q columns of a fused projection's rows
        s["qrow"] = torch.randn((T, qd + (2 * kh * hd if case["fused"] else 0)), device="cuda",
                                generator=g) * 1.5
        s["out"] = torch.zeros((T, qd), device="cuda")
        return s
    kv = torch.randn((2, T, kh * hd), device="cuda", generator=g)
    kv *= torch.exp(0.7 * torch.randn((2, 1, kh * hd), device="cuda", generator=g))
    s["k"], s["v"] = kv[0], kv[1]
    # the rows read back: the new ones and those before them that share a block
    back = [min(lens[i], m + BLOCK - 1) for i, m in zip(order, s["news"])]
    s["back"], s["back_start"] = back, _i32(_starts(back))
    s["k_out"] = torch.zeros((sum(back), kh * hd), device="cuda")
    s["v_out"] = torch.zeros_like(s["k_out"])
    return s


def _prepare_pages(case, seed):
    g = _gen(seed)
    page, P, C = case["page"], case["parents"], case["children"]
    r = random.Random(case["length"] * 1009 + case["add"])
    lens = [max(1, case["length"] - r.randint(0, min(case["length"] - 1, page))) for _ in range(P)]
    lens[0] = case["length"]
    most = -(-(case["length"] + case["add"]) // page)
    n_pages = sum(-(-x // page) for x in lens) + P * C * (-(-case["add"] // page) + 1) + (
        case["spare"])
    data, scale = _pool(g, case["layers"], n_pages, case["kv_heads"], page, case["hd"])
    table, length, refs = _owned(g, lens + [0] * (P * C), page, n_pages, most + 1)
    kids = list(range(P, P + P * C))
    return dict(case=case, data=data, scale=scale, table=table, len=length, refs=refs,
                kids=_i32(kids), parent=_i32([i // C for i in range(P * C)]),
                zero=_i32([0] * (P * C)), add=_i32([r.randint(1, case["add"]) for _ in kids]),
                status=_i32([0, 0, 0]))


def _prepare_compact(case, seed):
    g = _gen(seed)
    page, N, n = case["page"], case["n_pages"], case["n"]
    data, scale = _pool(g, case["layers"], N, case["kv_heads"], page, case["hd"])
    live = max(1, int(N * case["live"]))
    each = [live // n + (i < live % n) for i in range(n)]
    table, length, refs = _owned(g, [max(0, k * page - 3) for k in each], page, N, max(each) + 1)
    return dict(case=case, data=data, scale=scale, table=table, len=length, refs=refs,
                table0=table.clone(), refs0=refs.clone(), live=_i32([0]),
                map=torch.zeros(N, dtype=torch.int32, device="cuda"))


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    R, V = case["rows"], case["vocab"]
    x = torch.randn((R, V + case["pad"]), device="cuda", generator=g) * 2.5
    hot = torch.randint(0, V, (R, 24), device="cuda", generator=g)
    x.scatter_add_(1, hot, 14 * torch.rand((R, 24), device="cuda", generator=g))
    if case["masked"]:
        x[:, :V].masked_fill_(torch.rand((R, V), device="cuda", generator=g) < case["masked"],
                              -math.inf)
    t = hot[:, 0].to(torch.int32)
    if case["pad"]:
        t[::7] = -1  # rows of padding have no token
        x[:, V:] = math.nan  # and the columns behind the vocabulary hold nothing
    top = case["top"]
    return dict(case=case, x=x, targets=t, lp=torch.zeros(R, device="cuda"),
                entropy=torch.zeros(R, device="cuda"),
                rank=torch.zeros(R, dtype=torch.int32, device="cuda"),
                top_id=torch.zeros((R, top), dtype=torch.int32, device="cuda"),
                top_lp=torch.zeros((R, top), device="cuda"))


def prepare(case, seed):
    _stream()
    if case["kind"] in ("attention", "store"):
        return _prepare_cache(case, seed)
    if case["kind"] == "pages":
        return _prepare_pages(case, seed)
    if case["kind"] == "compact":
        return _prepare_compact(case, seed)
    return _prepare_logprobs(case, seed)


# ---- the library's calls ------------------------------------------------------------------------
def _handle(s):
    """The pool as the library takes it; a program keeps it as long as the pool."""
    if "handle" not in s:
        c = s["case"]
        s["handle"] = _lib().KvPool(
            n_layers=s["data"].shape[0], n_pages=s["data"].shape[1], page=c["page"],
            n_kv_heads=c["kv_heads"], head_dim=c["hd"], n_seqs=s["table"].shape[0],
            max_pages=s["table"].shape[1], data=s["data"].data_ptr(), scale=s["scale"].data_ptr(),
            table=s["table"].data_ptr(), len=s["len"].data_ptr(), refs=s["refs"].data_ptr())
    return s["handle"]


def _run_own(s):
    c, dev = s["case"], _dev()
    if c["kind"] == "attention":
        dev.kv_pool_attention(_handle(s), s["layer"], s["seqs"].data_ptr(), s["start"].data_ptr(),
                              c["n"], s["qrow"].shape[0], c["heads"], s["qrow"].data_ptr(),
                              s["out"].data_ptr(), max_len=s["max_len"], window=c["window"],
                              q_stride=s["qrow"].shape[1])
        return s["out"]
    if c["kind"] == "store":
        p = _handle(s)
        dev.kv_pool_store(p, s["layer"], s["seqs"].data_ptr(), s["start"].data_ptr(), c["n"],
                          s["k"].shape[0], s["k"].data_ptr(), s["v"].data_ptr())
        dev.kv_pool_load(p, s["layer"], s["seqs"].data_ptr(), s["back_start"].data_ptr(), c["n"],
                         s["k_out"].shape[0], s["k_out"].data_ptr(), s["v_out"].data_ptr())
        return dict(k=s["k_out"], v=s["v_out"], scale=s["scale"])
    if c["kind"] == "pages":
        p, n, st = _handle(s), s["kids"].shape[0], s["status"].data_ptr()
        dev.kv_pool_trim(p, s["kids"].data_ptr(), s["zero"].data_ptr(), n, st)
        dev.kv_pool_assign(p, s["kids"].data_ptr(), s["parent"].data_ptr(), n, st + 4)
        dev.kv_pool_extend(p, s["kids"].data_ptr(), s["add"].data_ptr(), n, st + 8)
        return _pages_out(s, status=s["status"])
    if c["kind"] == "compact":
        s["table"].copy_(s["table0"])  # the holes again
        s["refs"].copy_(s["refs0"])
        dev.kv_pool_compact(_handle(s), s["map"].data_ptr(), s["live"].data_ptr())
        return _pages_out(s, live=s["live"], map=s["map"])
    dev.logprobs(s["x"].data_ptr(), c["rows"], c["vocab"], s["targets"].data_ptr(),
                 s["lp"].data_ptr(), s["entropy"].data_ptr(), s["rank"].data_ptr(), c["top"],
                 s["top_id"].data_ptr(), s["top_lp"].data_ptr(), stride=s["x"].shape[1])
    return _logprobs_out(s)


def _pages_out(s, **more):
    # the page operations move the cache's bytes unread: they come back as bytes
    return dict(table=s["table"], len=s["len"], refs=s["refs"], data=s["data"], scale=s["scale"],
                **more)


def _logprobs_out(s):
    out = dict(lp=s["lp"], entropy=s["entropy"], rank=s["rank"])
    if s["case"]["top"]:
        out.update(top_id=s["top_id"], top_lp=s["top_lp"])
    return out


# ---- the plain forms ------------------------------------------------------------------------------
def _sequences(s, count):
    """The cached values of the batch's sequences, fp32 [n][kv head][count tokens][head_dim]."""
    c = s["case"]
    n, kh, hd, page = c["n"], c["kv_heads"], c["hd"], c["page"]
    pages = s["table"][s["seqs"].long(), :-(-count // page)].long().clamp(min=0)
    mp = pages.shape[1]
    d, sc = s["data"][s["layer"]][pages], s["scale"][s["layer"]][pages]
    k = d[..., 0, :].view(n, mp, kh, page // BLOCK, BLOCK, hd).float() * sc[..., 0, None, None]
    v = d[..., 1, :].view(n, mp, kh, page // BLOCK, hd, BLOCK).float() * sc[..., 1, None, None]
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(n, kh, mp * page, hd)
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(n, kh, mp * page, hd)
    return k[:, :, :count], v[:, :, :count]


def _rows(start, T):
    """Each row's sequence and its place among that sequence's rows."""
    t = torch.arange(T, dtype=torch.int32, device="cuda")
    i = torch.searchsorted(start[1:].contiguous(), t, right=True)
    return i, (t - start[i]).long()


def _plain_attention(s):
    c = s["case"]
    n, H, kh, hd, G = c["n"], c["heads"], c["kv_heads"], c["hd"], c["heads"] // c["kv_heads"]
    T, L, M = s["qrow"].shape[0], s["max_len"], max(s["news"])
    k, v = _sequences(s, L)
    m = (s["start"][1:] - s["start"][:-1])[:, None]
    j = torch.arange(M, device="cuda")[None]
    row = (s["start"][:-1, None] + j).clamp(max=T - 1).long()
    q = s["qrow"][row, :H * hd].view(n, M, kh, G, hd).permute(0, 2, 3, 1, 4).reshape(n, kh, G * M, hd)
    a = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hd))
    pos = (s["len"][s["seqs"].long()][:, None] - m + j)[:, None, None, :, None]
    t = torch.arange(L, device="cuda")
    seen = t <= pos
    if c["window"]:
        seen = seen & (t > pos - c["window"])
    a = a.view(n, kh, G, M, L).masked_fill(~seen, -math.inf)
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(top == -math.inf, 0.0, top))
    o = torch.matmul(e.view(n, kh, G * M, L), v.contiguous()).view(n, kh, G, M, hd)
    den = e.sum(-1)[..., None]
    o = torch.where(den > 0, o / den, 0.0).permute(0, 3, 1, 2, 4).reshape(n, M, H * hd)
    i, at = _rows(s["start"], T)
    s["out"].copy_(o[i, at])
    return s["out"]


def _quantize(new, old, fresh, held, s_old):
    """A block's 8-bit values and scale; axes (token, column) last, fresh / held: the new and the
    older tokens."""
    x = torch.where(fresh, new, 0.0)
    amax = torch.where(torch.isfinite(x), x.abs(), 0.0).amax((-1, -2))
    had = held.any(-2)[..., 0]
    sc = torch.maximum(torch.where(had, s_old, 0.0), (amax.double() / 127.0).float())
    d = sc.double()[..., None, None]
    q_new = torch.nan_to_num(torch.round(x.double() / d), 0.0, 127.0, -127.0).clamp(-127, 127)
    grown = torch.round(old.double() * s_old.double()[..., None, None] / d)
    q_old = torch.where((sc > s_old)[..., None, None], torch.nan_to_num(grown, 0.0), old.double())
    q_new = torch.where(d > 0, q_new, 0.0)
    return torch.where(fresh, q_new, torch.where(held, q_old, old.double())).to(torch.int8), sc


def _plain_store(s):
    c = s["case"]
    n, kh, hd, page, layer = c["n"], c["kv_heads"], c["hd"], c["page"], s["layer"]
    seqs, T = s["seqs"].long(), s["k"].shape[0]
    length = s["len"][seqs].long()[:, None]
    m = (s["start"][1:] - s["start"][:-1]).long()[:, None]
    first, last = (length - m) // BLOCK, (length - 1) // BLOCK
    b = torch.arange((max(s["news"]) + 2 * BLOCK - 2) // BLOCK, device="cuda")[None]
    blk = torch.minimum(first + b, last)  # [n][b]; a place behind the last block repeats it
    pos = blk[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    fresh = (pos >= (length - m)[..., None]) & (pos < length[..., None])
    held = pos < (length - m)[..., None]
    row = (s["start"][:-1].long()[:, None, None] + pos - (length - m)[..., None]).clamp(0, T - 1)
    at = (torch.gather(s["table"][seqs], 1, blk * BLOCK // page).long(), blk % (page // BLOCK))
    at = (at[0][..., None], torch.arange(kh, device="cuda"), at[1][..., None])  # [n][b][kh]
    old, s_old = s["data"][layer][at], s["scale"][layer][at]  # [n][b][kh][2][...], [n][b][kh][2]
    f, h = fresh[:, :, None, :, None], held[:, :, None, :, None]

    def rows(x):
        return x[row].view(n, -1, BLOCK, kh, hd).permute(0, 1, 3, 2, 4)

    kq, ks = _quantize(rows(s["k"]), old[..., 0, :].unflatten(-1, (BLOCK, hd)), f, h, s_old[..., 0])
    vq, vs = _quantize(rows(s["v"]), old[..., 1, :].unflatten(-1, (hd, BLOCK)).transpose(-1, -2),
                       f, h, s_old[..., 1])
    s["data"][layer][at] = torch.stack([kq.flatten(-2), vq.transpose(-1, -2).flatten(-2)], -2)
    s["scale"][layer][at] = torch.stack([ks, vs], -1)
    # read back
    T2 = s["k_out"].shape[0]
    i, j = _rows(s["back_start"], T2)
    count = (s["back_start"][1:] - s["back_start"][:-1]).long()
    pos = (length[:, 0] - count)[i] + j
    pg = s["table"][seqs[i], pos // page].long()
    d = s["data"][layer][pg, :, pos % page // BLOCK]  # [T2][kh][2][...]
    sc = s["scale"][layer][pg, :, pos % page // BLOCK]
    t = torch.arange(T2, device="cuda")
    k = d[:, :, 0].unflatten(-1, (BLOCK, hd))[t, :, pos % BLOCK].float() * sc[..., 0, None]
    v = d[:, :, 1].unflatten(-1, (hd, BLOCK))[t, :, :, pos % BLOCK].float() * sc[..., 1, None]
    s["k_out"].copy_(k.flatten(1))
    s["v_out"].copy_(v.flatten(1))
    return dict(k=s["k_out"], v=s["v_out"], scale=s["scale"])


def _count(refs, pages, by):
    """refs[page] += by for each listed page (-1: none)."""
    refs.index_add_(0, pages.clamp(min=0).flatten().long(),
                    torch.where(pages >= 0, by, 0).flatten().to(torch.int32))


def _plain_pages(s):
    c = s["case"]
    page, table, length, refs = c["page"], s["table"], s["len"], s["refs"]
    kids, parent = s["kids"].long(), s["parent"].long()
    n, N = kids.shape[0], refs.shape[0]
    col = torch.arange(table.shape[1], device="cuda")[None]
    # cut back
    keep = torch.minimum(length[kids], s["zero"])
    rows = table[kids]
    drop = (col >= (keep[:, None] + page - 1) // page) & (rows >= 0)
    _count(refs, torch.where(drop, rows, -1), -1)
    table[kids] = torch.where(drop, -1, rows)
    length[kids] = keep
    # fork
    old, new = table[kids], table[parent]
    _count(refs, old, -1)
    _count(refs, new, 1)
    table[kids] = new
    length[kids] = length[parent]
    # make room: each last page that others hold too is copied, then the further pages
    L = length[kids].long()
    have, want = (L + page - 1) // page, (L + s["add"] + page - 1) // page
    last = torch.gather(new, 1, (have - 1).clamp(min=0)[:, None]).long()[:, 0]
    part = (L % page != 0) & (s["add"] > 0)
    same = (last[:, None] == last[None]) & part[:, None] & part[None]
    earlier = torch.tril(same, -1).sum(1)
    copy = part & (earlier < refs[last.clamp(min=0)] - 1)
    need = copy + want - have
    base = torch.cumsum(need, 0) - need
    free = torch.sort((refs > 0).to(torch.int8), stable=True).indices
    total = need.sum()
    slot = base[:, None] + copy[:, None] + col - have[:, None]
    more = (col >= have[:, None]) & (col < want[:, None])
    rows = torch.where(more, free[slot.clamp(0, N - 1)].to(torch.int32), new)
    fresh = free[base.clamp(max=N - 1)]
    moved = copy[:, None] & (col == (have - 1)[:, None])
    table[kids] = torch.where(moved, fresh[:, None].to(torch.int32), rows)
    _count(refs, torch.where(copy, last, -1), -1)
    refs[free] = torch.where(torch.arange(N, device="cuda") < total, 1, refs[free])
    length[kids] += s["add"]
    # where nothing is copied, the page in use onto itself: no other child writes it
    dst = torch.where(copy, fresh, last)
    s["data"][:, dst] = s["data"][:, last]
    s["scale"][:, dst] = s["scale"][:, last]
    s["status"].zero_()
    return _pages_out(s, status=s["status"])


def _plain_compact(s):
    s["table"].copy_(s["table0"])  # the holes again
    s["refs"].copy_(s["refs0"])
    table, refs = s["table"], s["refs"]
    live = refs > 0
    n_live = live.sum()
    at = torch.arange(refs.shape[0], device="cuda")
    src = (live & (at >= n_live)).nonzero()[:, 0]
    dst = (~live & (at < n_live)).nonzero()[:, 0]
    to = torch.where(live, at, -1).to(torch.int32)
    to[src] = dst.to(torch.int32)
    s["data"][:, dst] = s["data"][:, src]
    s["scale"][:, dst] = s["scale"][:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    s["map"].copy_(to)
    s["live"].copy_(n_live[None])
    return _pages_out(s, live=s["live"], map=s["map"])


def _plain_logprobs(s):
    c = s["case"]
    x = s["x"][:, :c["vocab"]]
    top = x.amax(-1, keepdim=True)
    d = x - torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(d)
    total = e.sum(-1)
    total = torch.where(total == 0, 1.0, total)  # a row with nothing left: -inf, and no entropy
    s["entropy"].copy_(torch.log(total) - torch.where(e > 0, e * d, 0.0).sum(-1) / total)
    t = s["targets"].long()[:, None]
    xt = torch.gather(x, 1, t.clamp(min=0))
    lp = torch.gather(d, 1, t.clamp(min=0))[:, 0] - torch.log(total)
    s["lp"].copy_(torch.where(t[:, 0] >= 0, lp, 0.0))
    at = torch.arange(c["vocab"], device="cuda")
    better = (x > xt) | ((x == xt) & (at < t))
    s["rank"].copy_(torch.where(t[:, 0] >= 0, better.sum(-1), -1))
    if c["top"]:
        # a number's place in the order of its value, then of the lower index
        b = (x + 0.0).view(torch.int32)
        b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
        key = torch.topk((b << 32) | (0x7FFFFFFF - at), c["top"], dim=-1).values
        pick = 0x7FFFFFFF - (key & 0xFFFFFFFF)
        s["top_id"].copy_(pick)
        s["top_lp"].copy_(torch.gather(d, 1, pick) - torch.log(total)[:, None])
    return _logprobs_out(s)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "attention":
        return _plain_attention(state)
    if kind == "store":
        return _plain_store(state)
    if kind == "pages":
        return _plain_pages(state)
    if kind == "compact":
        return _plain_compact(state)
    return _plain_logprobs(state)


# ---- bytes and operations -------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "attention":
        lens, news = _lengths(case)
        w = case["window"] or (1 << 30)
        seen = read = 0
        for n, m in zip(lens, news):
            seen += sum(min(p + 1, w) for p in range(n - m, n))
            read += min(n, w + m - 1)
        row = case["heads"] * case["hd"]
        return {"bytes": read * case["kv_heads"] * (2 * case["hd"] + 8 / BLOCK) + 8 * sum(news) * row,
                "flops": 4.0 * seen * row}
    if kind == "store":
        lens, news = _lengths(case)
        T, row = sum(news), case["kv_heads"] * case["hd"]
        back = sum(min(n, m + BLOCK - 1) for n, m in zip(lens, news))
        blocks = sum((n - 1) // BLOCK - (n - m) // BLOCK + 1 for n, m in zip(lens, news))
        return {"bytes": T * row * (8 + 2) + back * row * (2 + 8) + 16 * blocks * case["kv_heads"],
                "flops": 4.0 * T * row}
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (16 + 8 * case["top"]), "flops": 6.0 * n}
    whole = case["layers"] * case["kv_heads"] * case["page"] * (2 * case["hd"] + 8 / BLOCK)
    if kind == "pages":
        kids = case["parents"] * case["children"]
        copies = kids if case["length"] % case["page"] else 0
        return {"bytes": 2 * copies * whole + 16 * kids * (case["length"] // case["page"] + 2),
                "flops": 0.0}
    live = max(1, int(case["n_pages"] * case["live"]))
    moved = live * (case["n_pages"] - live) / case["n_pages"]  # as many as holes, on average
    return {"bytes": 2 * moved * whole + 16 * case["n_pages"], "flops": 0.0}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _tokens64(s, seq, layer):
    """One sequence's cached K and V, float64 [tokens][kv head][head_dim], block by block."""
    c = s["case"]
    length, page, hd = int(s["len"][seq]), c["page"], c["hd"]
    k = torch.empty((length, c["kv_heads"], hd), dtype=torch.float64, device="cuda")
    v = torch.empty_like(k)
    pages = s["table"][seq].tolist()
    for at in range(0, length, page):
        d, sc = s["data"][layer, pages[at // page]], s["scale"][layer, pages[at // page]].double()
        used = min(page, length - at)
        kk = d[:, :, 0].reshape(-1, page, hd).double() * sc[:, :, 0].repeat_interleave(BLOCK, 1)[..., None]
        vv = d[:, :, 1].reshape(-1, page // BLOCK, hd, BLOCK).double() * sc[:, :, 1, None, None]
        vv = vv.transpose(2, 3).reshape(-1, page, hd)
        k[at:at + used], v[at:at + used] = kk[:, :used].transpose(0, 1), vv[:, :used].transpose(0, 1)
    return k, v


def _exact_attention(case, seed):
    s = prepare(case, seed)
    H, kh, hd = case["heads"], case["kv_heads"], case["hd"]
    out = torch.empty((s["qrow"].shape[0], H, hd), dtype=torch.float64, device="cuda")
    at = 0
    for seq, m in zip(s["seqs"].tolist(), s["news"]):
        k, v = _tokens64(s, seq, s["layer"])
        n = k.shape[0]
        far = torch.arange(n - m, n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None]
        hide = (far < 0) | (far >= (case["window"] or n + 1))
        for h in range(H):
            q = s["qrow"][at:at + m, h * hd:(h + 1) * hd].double()
            z = (q @ k[:, h * kh // H].T) / math.sqrt(hd)
            out[at:at + m, h] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ v[:, h * kh // H]
        at += m
    return out.flatten(1)


def _exact_store(case, seed):
    s = prepare(case, seed)
    kh, hd, layer = case["kv_heads"], case["hd"], s["layer"]
    scale = s["scale"].double()
    outs = ([], [])
    at = 0
    for seq, m, back in zip(s["seqs"].tolist(), s["news"], s["back"]):
        length = int(s["len"][seq])
        kept = _tokens64(s, seq, layer)
        for side, (x, vals) in enumerate(zip((s["k"], s["v"]), kept)):
            x64 = x[at:at + m].double().view(m, kh, hd)
            for b in range((length - m) // BLOCK, (length - 1) // BLOCK + 1):
                lo, hi = b * BLOCK, min(length, b * BLOCK + BLOCK)
                cut = max(lo, length - m)
                page = int(s["table"][seq, lo // case["page"]])
                place = (layer, page, slice(None), lo % case["page"] // BLOCK, side)
                before = scale[place] if cut > lo else torch.zeros_like(scale[place])
                add = x64[cut - (length - m):hi - (length - m)]
                # the scale is a 32-bit number
                after = torch.maximum(before, (add.abs().amax((0, 2)) / 127).float().double())
                vals[cut:hi] = torch.round(add / after[:, None]) * after[:, None]
                if cut > lo:
                    grown = torch.round(vals[lo:cut] / after[:, None]) * after[:, None]
                    vals[lo:cut] = torch.where((after > before)[:, None], grown, vals[lo:cut])
                scale[place] = after
            outs[side].append(vals[length - back:].flatten(1))
        at += m
    return dict(k=torch.cat(outs[0]), v=torch.cat(outs[1]), scale=scale)


def _exact_logprobs(case, seed):
    s = prepare(case, seed)
    lp, entropy, top_lp = [], [], []
    for x, t in zip(s["x"][:, :case["vocab"]].split(64), s["targets"].long().split(64)):
        z = x.double()
        z = z - torch.logsumexp(z, -1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(z)
        entropy.append(-(torch.where(p > 0, z, 0.0) * p).sum(-1))
        lp.append(torch.where(t >= 0, z.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0))
        top_lp.append(z.topk(case["top"], -1).values)
    out = dict(lp=torch.cat(lp), entropy=torch.cat(entropy), rank=None)
    if case["top"]:
        out.update(top_id=None, top_lp=torch.cat(top_lp))
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "attention":
        return _exact_attention(case, seed)
    if kind == "store":
        return _exact_store(case, seed)
    if kind in ("pages", "compact"):
        return None  # whole numbers and moved bytes: nothing is computed
    return _exact_logprobs(case, seed)
