"""Refused arguments of qr_kv_pool_* and qr_logprobs: a status and a message
before anything is launched (the context is never looked at, so no device is
needed)."""
import ctypes as C

import pytest

import quantr_amd as Q

_mem = C.create_string_buffer(1 << 16)
BASE = (C.addressof(_mem) + 4095) & ~4095
CTX = BASE  # never dereferenced: every call here is refused first


def pool(**change):
    a = dict(n_layers=2, n_pages=8, page=32, n_kv_heads=2, head_dim=64, n_seqs=4, max_pages=4,
             data=BASE, scale=BASE, table=BASE, len=BASE, refs=BASE)
    a.update(change)
    return Q.KvPool(**a)


def refused(name, *args, code=-1, says=""):
    lib = Q.load()
    rc = getattr(lib, name)(*args)
    assert rc == code, (rc, lib.qr_last_error())
    assert name.encode() in lib.qr_last_error() and says.encode() in lib.qr_last_error()


CALLS = {
    "qr_kv_pool_reset": lambda c, p: (c, p),
    "qr_kv_pool_extend": lambda c, p: (c, p, BASE, BASE, 1, None),
    "qr_kv_pool_assign": lambda c, p: (c, p, BASE, BASE, 1, None),
    "qr_kv_pool_trim": lambda c, p: (c, p, BASE, BASE, 1, None),
    "qr_kv_pool_compact": lambda c, p: (c, p, None, None),
    "qr_kv_pool_store": lambda c, p: (c, p, 0, None, BASE, 1, 1, BASE, BASE, 128),
    "qr_kv_pool_load": lambda c, p: (c, p, 0, None, BASE, 1, 1, BASE, BASE, 128),
    "qr_kv_pool_attention": lambda c, p: (c, p, 0, None, BASE, 1, 1, 4, BASE, 256, BASE, 256, 0, 0,
                                          0.0),
}


@pytest.mark.parametrize("name", CALLS)
def test_pools_that_cannot_be(name):
    args = CALLS[name]
    refused(name, *args(None, pool()), says="null ctx")
    refused(name, *args(CTX, None), says="null pool")
    for change, says in (
            (dict(page=24), "page"), (dict(page=8), "page"), (dict(page=0), "page"),
            (dict(page=131072), "page"), (dict(head_dim=48), "head_dim"),
            (dict(head_dim=288), "head_dim"), (dict(head_dim=0), "head_dim"),
            (dict(n_layers=0), "layers"), (dict(n_pages=-1), "pages"), (dict(n_kv_heads=0), "heads"),
            (dict(n_kv_heads=1025), "heads"), (dict(n_seqs=0), "table"),
            (dict(n_seqs=65537), "table"), (dict(max_pages=0), "table"),
            (dict(max_pages=(1 << 25) + 1), "2^30"), (dict(n_pages=(1 << 29) + 1, page=32), "2^31"),
            (dict(data=None), "null"), (dict(scale=None), "null"),
            (dict(table=None), "null"), (dict(len=None), "null"), (dict(refs=None), "null"),
            (dict(data=BASE + 8), "alignment"), (dict(scale=BASE + 4), "alignment"),
            (dict(table=BASE + 2), "alignment")):
        refused(name, *args(CTX, pool(**change)), says=says)


@pytest.mark.parametrize("name", ["qr_kv_pool_extend", "qr_kv_pool_assign", "qr_kv_pool_trim"])
def test_lists_that_cannot_be(name):
    p = pool()
    refused(name, CTX, p, None, BASE, 1, None, says="null list")
    refused(name, CTX, p, BASE, None, 1, None, says="null list")
    refused(name, CTX, p, BASE, BASE, -1, None, says="list of")
    refused(name, CTX, p, BASE, BASE, 4097, None, says="list of")


@pytest.mark.parametrize("name", ["qr_kv_pool_store", "qr_kv_pool_load"])
def test_rows_that_cannot_be(name):
    p = pool()
    refused(name, CTX, p, 2, None, BASE, 1, 1, BASE, BASE, 128, says="layer")
    refused(name, CTX, p, -1, None, BASE, 1, 1, BASE, BASE, 128, says="layer")
    refused(name, CTX, p, 0, None, None, 1, 1, BASE, BASE, 128, says="start")
    refused(name, CTX, p, 0, None, BASE, -1, 1, BASE, BASE, 128, says="sequences")
    refused(name, CTX, p, 0, None, BASE, 65537, 1, BASE, BASE, 128, says="sequences")
    refused(name, CTX, p, 0, None, BASE, 1, -1, BASE, BASE, 128, says="rows")
    refused(name, CTX, p, 0, None, BASE, 1, (1 << 22) + 1, BASE, BASE, 128, says="rows")
    refused(name, CTX, p, 0, None, BASE, 1, 1, None, BASE, 128, says="null rows")
    refused(name, CTX, p, 0, None, BASE, 1, 1, BASE, None, 128, says="null rows")
    refused(name, CTX, p, 0, None, BASE, 1, 1, BASE + 4, BASE, 128, says="aligned")
    refused(name, CTX, p, 0, None, BASE, 1, 1, BASE, BASE, 124, says="stride")
    refused(name, CTX, p, 0, None, BASE, 1, 1, BASE, BASE, 130, says="stride")


def test_attention_that_cannot_be():
    def call(says, heads=4, q=BASE, qs=256, out=BASE, os=256, max_len=0, window=0, scale=0.0, p=None):
        refused("qr_kv_pool_attention", CTX, p or pool(), 0, None, BASE, 1, 1, heads, q, qs, out, os,
                max_len, window, scale, says=says)

    call("heads", heads=3)
    call("heads", heads=0)
    call("heads", heads=16386)
    call("null rows", q=None)
    call("null rows", out=None)
    call("aligned", q=BASE + 4)
    call("aligned", out=BASE + 8)
    call("stride", qs=252)
    call("stride", os=257)
    call("max_len", max_len=-1)
    call("window", window=-1)
    call("scale", scale=float("nan"))
    call("scale", scale=float("inf"))


def test_logprobs_that_cannot_be():
    def call(says, ctx=CTX, x=BASE, stride=100, rows=1, vocab=100, t=BASE, lp=BASE, n=0):
        refused("qr_logprobs", ctx, x, stride, rows, vocab, t, lp, None, None, n, None, None, says=says)

    call("null ctx", ctx=None)
    call("null logits", x=None)
    call("null targets", t=None)
    call("stride", stride=99)
    call("logits", rows=-1)
    call("logits", vocab=0)
    call("n_top", n=65)
    call("n_top", n=-1)
    call("alignment", x=BASE + 2)
