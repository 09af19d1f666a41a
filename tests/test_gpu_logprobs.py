"""Token log probabilities on the device against numpy in 64 bits."""
import numpy as np
import pytest

from spirv_inference_b200 import _lib
from spirv_inference_b200.graph import Graph

pytestmark = pytest.mark.gpu


@pytest.fixture
def g(gpu):
    with Graph(gpu) as graph:
        yield graph


def _run(g, x, ids, k, ld=None):
    rows, cols = x.shape
    ld = cols if ld is None else ld
    host = np.full((rows, ld), 1e30, np.float32)       # what lies between rows is not read
    host[:, :cols] = x
    lp, ent, rank = g.alloc((rows,)), g.alloc((rows,)), g.alloc((rows,), np.int32)
    top = dict(top_k=k, top_ids=g.alloc((rows, k), np.int32), top_logprobs=g.alloc((rows, k))) \
        if k else {}
    g.token_logprobs(g.tensor(host), ld, rows, cols, g.tensor(ids, np.int32), lp, entropy=ent,
                     rank=rank, **top)
    out = [t.download() for t in (lp, ent, rank)]
    return out + ([top["top_ids"].download(), top["top_logprobs"].download()] if k else [])


def _ref(x, ids, k):
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        l = e.sum(1, keepdims=True)
        p = x - m - np.log(l)
        ent = -np.nansum(np.where(e > 0, e / l * p, 0), axis=1)
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    r = np.arange(len(x))
    return p[r, ids], ent, 1 + (x > x[r, ids][:, None]).sum(1), order, \
        np.take_along_axis(p, order, 1)


def _check(got, want, x, k):
    # x - m and log l are rounded once each, the sum over n terms of a tree of
    # partial sums to about 2^-20, and e^d to |d| 2^-23: 2^-19 (1 + |result|)
    tol = 2.0 ** -19
    for i in (0, 1):
        assert np.all(np.abs(got[i] - want[i]) <= tol * (1 + np.abs(want[i]))), i
    assert np.array_equal(got[2], want[2])
    if k:
        assert np.array_equal(got[3], want[3])
        assert np.all(np.abs(got[4] - want[4]) <= tol * (1 + np.abs(want[4])))


@pytest.mark.parametrize("rows,cols,k,ld", [
    (1, 1, 1, None), (1, 2, 2, None), (3, 31, 5, 40), (2, 1000, 0, None), (5, 1001, 20, 1003),
    (1, 32000, 5, None), (64, 32000, 20, None), (7, 4097, 64, 4100), (300, 513, 3, None),
    (2, 50257, 1, None), (1, 200003, 20, None), (3, 128256, 64, 128260), (700, 9000, 5, None), (2500, 1003, 7, 1003),
    (2400, 700, 64, None)])
def test_random_rows(g, rows, cols, k, ld):
    rng = np.random.default_rng(rows + cols)
    x = (rng.standard_normal((rows, cols)) * 3).astype(np.float32)
    ids = rng.integers(0, cols, rows).astype(np.int32)
    ids[0] = np.argmax(x[0])
    _check(_run(g, x, ids, k, ld), _ref(x, ids, k), x, k)


@pytest.mark.parametrize("cols", [70, 1000, 32000, 100000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "steps", "one thread's"])
def test_orders_that_fill_the_candidates(g, cols, kind):
    """Rows in which very many values tie or lie above any early threshold."""
    k = 20
    j = np.arange(cols)
    x = {"equal": np.zeros(cols), "rising": j / cols, "falling": -j / cols,
         "steps": (j // 7 % 50).astype(float),
         "one thread's": np.where(j % 512 == 3, 5.0 + j / cols, -1.0)}[kind].astype(np.float32)
    x = np.stack([x, -x])
    ids = np.array([cols - 1, cols // 2], np.int32)
    _check(_run(g, x, ids, k), _ref(x, ids, k), x, k)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "masked"])
def test_orders_many_rows(g, kind):
    """The same with rows enough for each warp to have its own."""
    cols, rows, k = 1500, 2400, 40
    j = np.arange(cols)
    x = {"equal": np.zeros(cols), "rising": j / cols, "falling": -j / cols,
         "masked": np.where(j % 300 == 7, 1.0 + j, -np.inf)}[kind].astype(np.float32)
    x = np.tile(x, (rows, 1))
    ids = np.full(rows, 7, np.int32)
    got, want = _run(g, x, ids, k), _ref(x[:1], ids[:1], k)
    if kind == "masked":
        assert np.array_equal(got[3][:, :5], np.tile(want[3][:, :5], (rows, 1)))
        rest = [i for i in range(k) if i % 300 != 7][:k - 5]
        assert np.array_equal(got[3][:, 5:], np.tile(rest, (rows, 1)))
        assert np.all(np.isneginf(got[4][:, 5:]))
    else:
        assert np.array_equal(got[3], np.tile(want[3], (rows, 1)))
    assert np.all(got[2] == want[2][0])
    for i in (0, 1):
        assert np.abs(got[i] - want[i][0]).max() <= 2.0 ** -19 * (1 + abs(want[i][0]))


@pytest.mark.parametrize("cols", [40, 5000, 40000])
def test_masked_and_special_rows(g, cols):
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((8, cols)).astype(np.float32)
    x[0, rng.permutation(cols)[:cols - 3]] = -np.inf      # three tokens left
    x[1] = -np.inf                                        # nothing left
    x[2, 1:] = np.finfo(np.float32).min                   # masked by the lowest number
    x[3, 7] = np.nan
    x[4, 9] = np.inf
    x[5] = 1e38 * np.sign(x[5])                           # large, finite
    x[6, 4] = 3e38
    ids = np.array([int(np.argmax(x[0])), 2, 0, 1, 1, 5, 4, -1], np.int32)
    k = 5
    lp, ent, rank, top, tlp = _run(g, x, ids, k)
    want = _ref(x, np.maximum(ids, 0), k)
    for r in (0, 2, 5, 6):
        assert abs(lp[r] - want[0][r]) <= 1e-5 * (1 + abs(want[0][r])), r
        assert abs(ent[r] - want[1][r]) <= 1e-5 * (1 + want[1][r]), r
        assert rank[r] == want[2][r]
        assert np.array_equal(top[r], want[3][r])
    assert np.all(np.isneginf(tlp[0, 3:])) and np.isfinite(tlp[0, :3]).all()
    assert np.isneginf(lp[1]) and ent[1] == 0 and rank[1] == 1
    assert top[1].tolist() == list(range(k)) and np.all(np.isneginf(tlp[1]))
    assert np.isnan(lp[3]) and np.isnan(ent[3]) and 7 not in top[3]
    assert np.isnan(lp[4]) and np.isnan(ent[4]) and top[4, 0] == 9
    assert lp[7] == 0 and rank[7] == 0 and abs(ent[7] - want[1][7]) <= 1e-5 * (1 + want[1][7])
    x[3] = np.nan
    top = _run(g, x, np.full(8, cols, np.int32), k)
    assert np.isnan(top[0]).all() and np.all(top[2] == 0)      # an id past the columns
    assert top[3][3].tolist() == list(range(k))


def test_optional_outputs_and_refusals(g):
    x = np.random.default_rng(0).standard_normal((4, 300)).astype(np.float32)
    d, ids = g.tensor(x), g.tensor(np.arange(4), np.int32)
    ent, lp, one = g.alloc((4,)), g.alloc((4,)), g.alloc((4, 2), np.int32)
    g.token_logprobs(d, 300, 4, 300, None, None, entropy=ent)
    want = _ref(x, np.arange(4), 0)
    assert np.abs(ent.download() - want[1]).max() <= 1e-5
    g.token_logprobs(d, 300, 4, 300, ids, lp)
    assert np.abs(lp.download() - want[0]).max() <= 1e-5
    for call in (lambda: g.token_logprobs(d, 299, 4, 300, ids, lp),
                 lambda: g.token_logprobs(d, 300, 0, 300, ids, lp),
                 lambda: g.token_logprobs(d, 300, 4, 0, ids, lp),
                 lambda: g.token_logprobs(d, 300, 4, 300, None, lp),
                 lambda: g.token_logprobs(d, 300, 4, 300, ids, lp, top_k=2, top_ids=one),
                 lambda: g.token_logprobs(d, 300, 4, 300, ids, lp, top_k=65, top_ids=one,
                                          top_logprobs=lp),
                 lambda: g.token_logprobs(d, 300, 4, 1, ids, lp, top_k=2, top_ids=one,
                                          top_logprobs=lp)):
        with pytest.raises(_lib.SpxError) as e:
            call()
        assert e.value.code == _lib.SPX_ERR_INVALID_ARGUMENT


def test_runs_are_equal_to_the_bit(g):
    x = np.random.default_rng(1).standard_normal((33, 32000)).astype(np.float32)
    ids = np.arange(33, dtype=np.int32)
    a = _run(g, x, ids, 20)
    for _ in range(3):
        assert all(np.array_equal(u, v) for u, v in zip(a, _run(g, x, ids, 20)))
