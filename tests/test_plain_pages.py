"""The plain form of the page operations (perf/operators.py) against the pool's
definition, entry by entry, on the CPU."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import kv_pool_ref as R

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf",
                    "operators.py")


class OnHost:
    """torch, with its tensors made in host memory."""

    def __getattr__(self, name):
        f = getattr(torch, name)
        if name not in ("arange", "tensor", "zeros", "full"):
            return f
        return lambda *a, **k: f(*a, **{**k, "device": "cpu"})


@pytest.fixture(scope="module")
def ops():
    spec = importlib.util.spec_from_file_location("plain_operators", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.torch = OnHost()
    return m


# lengths of the parents: whole pages, partly filled ones, both in either order
@pytest.mark.parametrize("lens", [[48, 37], [37, 48], [48, 32], [1, 16, 33, 16], [16, 1, 32, 40],
                                  [5, 5, 5]])
@pytest.mark.parametrize("children,add,spare", [(2, 7, 5), (3, 40, 0), (1, 16, 1)])
def test_fork_of_mixed_parents(ops, lens, children, add, spare):
    page, P = 16, len(lens)
    n, rng = P * children, np.random.default_rng(sum(lens) + add)
    adds = rng.integers(1, add + 1, n).tolist()
    held = sum(-(-x // page) for x in lens)
    p = R.Pool(2, held + n * (-(-add // page) + 1) + spare, page, 2, 32, P + n,
               -(-(max(lens) + add) // page) + 1, 1)
    p.scale[:] = rng.random(p.scale.shape)  # numbers, so that states compare
    order, at = rng.permutation(p.n_pages), 0
    for s, x in enumerate(lens):
        k = -(-x // page)
        p.table[s, :k], p.len[s] = order[at:at + k], x
        p.refs[order[at:at + k]] = 1
        at += k
    kids, parent = list(range(P, P + n)), [i // children for i in range(n)]
    names = ("table", "len", "refs", "data", "scale")
    s = {k: torch.from_numpy(getattr(p, k).copy()) for k in names}
    i32 = dict(dtype=torch.int32)
    s.update(case=dict(page=page), kids=torch.tensor(kids, **i32), parent=torch.tensor(parent, **i32),
             zero=torch.zeros(n, **i32), add=torch.tensor(adds, **i32), status=torch.ones(3, **i32))
    for turn in range(2):  # children of nothing, then the last turn's
        assert p.trim(kids, [0] * n) == p.assign(kids, parent) == p.extend(kids, adds) == 0
        out = ops._plain_pages(s)
        for k in names:
            np.testing.assert_array_equal(out[k].numpy(), getattr(p, k), err_msg="%d %s" % (turn, k))
        assert out["status"].tolist() == [0, 0, 0]
