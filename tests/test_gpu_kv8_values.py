"""Attention over the 8-bit cache on values of unlike sizes, each row against
bounds of its own: what a row does not see, or hardly weighs, takes no part in
its accuracy."""
import numpy as np
import pytest

import _kv8_np as N
from spirv_inference_b200.graph import Graph
from test_gpu_kv8 import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture
def g(gpu):
    with Graph(gpu) as graph:
        yield graph


def _filled(g, lens, T, change, *, Hkv=2, G=8, D=64, S=512, blk=32, seed=0, new=None):
    """A cache of lens[b] tokens and the queries of T new ones.  `change` edits
    the tokens [B][max(lens) + T][heads q, k, v][D]; sequence b has slot i of them
    at i."""
    B = len(lens)
    s = Setup(g, B, Hkv, G, D, S, blk, seed=seed)
    x = s.rng.standard_normal((B, max(lens) + T, Hkv * (G + 2), D)).astype(np.float32)
    change(x, Hkv * G, Hkv)
    if max(lens):
        s.append(max(lens), lens, qkv=np.ascontiguousarray(x[:, :max(lens)]).reshape(B, -1, x[0, 0].size))
        s.advance(max(lens), lens)
    last = np.stack([x[b, n:n + T] for b, n in enumerate(lens)])
    d_q, q = s.append(T, new, qkv=np.ascontiguousarray(last).reshape(B, T, -1))
    return s, d_q, q


def _bounds(q, K, V, tops, vtops, open_rows, len0, scale):
    """What the rows q [T][G][D] may be off by: out, lse, weights.  K, V [n][D],
    tops, vtops [n]: the largest value of a slot's closed block, or of an open slot;
    open_rows [n]: which are open.

    A score: an element of q, or of an open key, has 22 bits (both of them, and
    the product of their last halves left out: 3 2^-22) or, with few rows, 2^-30 of
    the row's largest; D + 8 sums that may be cut, 2^-23 each of sum |q k|; a
    key of a block may carry 2^-30 of the row's largest times the block's.  An
    exponent: the score, the largest score and their difference rounded.  A
    weight: that, exp2 and two halves of 11 bits (2^-20).  It is multiplied by
    2^15 s / r, s its block's scale and r the largest that the row sees, and its
    low half is a multiple of 2^-24: off by 2^-25, which times an int8 of at most
    127 and r / 2^15 is 2^-40 of 127 r, the largest that a value of that block can
    be (its own values may be smaller: they are only known to r / 2).  An open
    row beside closed ones in a tile is held at 2^10 to 2^11 where those are 127, so
    that its weight, in the same unit, is 2^11 where theirs is 2^15: 2^-36 of its
    largest.  Sums: 64 cut ones of a tile, and one a tile.  A row that sees a block closed around a key
    1e18 times the others' has, by the block's term, scores to 1e9: no bound."""
    T, G, D = q.shape
    n = len(K)
    q, aK, aV = q.astype(np.float64), np.abs(K), np.abs(V)
    sc = np.einsum("tgd,sd->tgs", q, K) * scale
    qk = np.einsum("tgd,sd->tgs", np.abs(q), aK)
    ds = abs(scale) * (qk * (3 * 2.0 ** -22 + (D + 8) * 2.0 ** -23)
                       + np.abs(q).max(-1)[..., None] * (aK.sum(-1) + tops) * 2.0 ** -30)
    out, lse, w = np.zeros((T, G, D)), np.zeros((T, G)), np.zeros(n)
    for t in range(T):
        m = len0 + t + 1
        s, d, v = sc[t, :, :m], ds[t, :, :m], aV[:m]
        top = s.max(-1, keepdims=True)
        e = np.exp(s - top)
        p = e / e.sum(-1, keepdims=True)
        z = top[:, 0] + np.log(e.sum(-1))
        d = np.expm1(np.minimum(d + (np.abs(s) + np.abs(top)) * 2.0 ** -22, 1.0))
        all_d = (p * d).sum(-1, keepdims=True) + (m / 16 + 64) * 2.0 ** -24
        with np.errstate(invalid="ignore"):
            all_d = np.where(all_d < 0.1, all_d / (1 - all_d), np.inf)
        rel = d * 1.12 + all_d + 2.0 ** -20        # (1 / 0.9 < 1.12)
        out[t] = (p * (rel + 64 * 2.0 ** -23 + (m / 16) * 2.0 ** -24)) @ v
        out[t] += (m * 2.0 ** -40 * max(v.max(), vtops[:m].max())
                   + (open_rows[:m] * vtops[:m]).sum() * 2.0 ** -36 + 2.0 ** -140)
        lse[t] = all_d[:, 0] + 2.0 ** -21 * (1 + np.abs(z))
        w[:m] += (p * (rel + np.abs(z)[:, None] * 2.0 ** -22)).sum(0) + G * 2.0 ** -120
    return out, lse, w


def _check(s, d_q, q, len0, scale=None, skip=0):
    """skip: this many of a sequence's last rows are not looked at (nor weights)."""
    B, T, G, D, Hq, S = s.B, s.T, s.G, s.D, s.Hq, s.S
    scale = D ** -0.5 if scale is None else scale
    out, lse = s.g.tensor(np.zeros((B * T, Hq, D), np.float32)), s.g.tensor(
        np.zeros((B * T, Hq), np.float32))
    w0 = s.rng.uniform(0, 1, (B, s.Hkv, S)).astype(np.float32)
    w = s.g.tensor(w0)
    s.g.attention_kv8(d_q, s.cache, out, q_len=T, q_heads=Hq, scale=scale, new_lens=s.d_new,
                      lse=lse, weights=w)
    o, z, wd = out.download().reshape(B, T, Hq, D), lse.download().reshape(B, T, Hq), w.download()
    looked_at = of_all = 0
    for b in range(B):
        n = s.new[b] - skip
        if n == 0:
            assert np.array_equal(wd[b], w0[b])
            continue
        for h in range(s.Hkv):
            hs = slice(h * G, (h + 1) * G)
            K, V = (c.values()[:len0[b] + n] for c in s.np[b][h])
            tops = [127 * c.row_scales().astype(np.float64)[:len0[b] + n] for c in s.np[b][h]]
            ro, rz, rw = N.attend(q[b, :n, hs], K, V, len0[b], scale)
            is_open = np.arange(len(K)) >= s.np[b][h][0].n // s.blk * s.blk
            bo, bz, bw = _bounds(q[b, :n, hs], K, V, *tops, is_open, len0[b], scale)
            looked_at += np.isfinite(bz).sum()
            of_all += bz.size
            for what, err, bound in (("out", np.abs(o[b, :n, hs] - ro), bo),
                                     ("lse", np.abs(z[b, :n, hs] - rz), bz)):
                worst = np.unravel_index(np.argmax(np.where(np.isnan(err), np.inf, err / bound)),
                                         err.shape)
                assert np.all(err <= bound), (what, b, h, worst, err[worst], bound[worst])
            if skip:
                continue
            total = len(K)
            want = np.where(np.arange(total) < len0[b], w0[b, h, :total], 0) + rw
            err = np.abs(wd[b, h, :total] - want)
            bw = bw + want * 2.0 ** -22 + n * G * 2.0 ** -24 * rw
            assert np.all(err <= bw), ("weights", b, h, np.argmax(err / bw))
    assert looked_at > 0.8 * of_all or not of_all
    return o, z, wd


ROWS = [(1, 1), (1, 8), (2, 8), (5, 8), (16, 8), (24, 8)]   # new tokens, heads of a group


def _zero(x, q, kv):
    x[:, :, q + kv:] = 0


def _zero_late(x, q, kv):          # the open block and what closed before it
    x[:, 20:, q + kv:] = 0


def _zero_early(x, q, kv):         # a zero start, in an open block too
    x[:, :40, q + kv:] = 0


def _zero_head(x, q, kv):
    x[:, :, q + kv] = 0


def _tiny(size):
    def change(x, q, kv):
        x[:, :, q + kv:] *= np.float32(size)
    return change


def _tiny_beside(x, q, kv):        # blocks of 1e-33, of 1 and of 1e-37 in turn
    at = np.arange(x.shape[1]) // 32 % 3
    x[:, :, q + kv:] *= np.array([1e-33, 1, 1e-37], np.float32)[at][None, :, None, None]


small = pytest.mark.parametrize(
    "change", [_zero, _zero_late, _zero_early, _zero_head, _tiny(1e-33), _tiny(3e-35), _tiny(1e-37),
               _tiny_beside],
    ids=["zero", "late", "early", "head", "1e-33", "3e-35", "1e-37", "beside"])


@small
@pytest.mark.parametrize("T,G", [r for r in ROWS if r[0] * r[1] < 80])
@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_over_zero_and_tiny_values(g, D, T, G, change):
    """Values that are zero, or so small that 2^15 over them passes fp32."""
    lens = [0, 37, 96, 300]
    s, d_q, q = _filled(g, lens, T, change, G=G, D=D)
    _check(s, d_q, q, lens)


@small
@pytest.mark.parametrize("T,G", [r for r in ROWS if r[0] * r[1] >= 80])
@pytest.mark.parametrize("D", [64, 128])
def test_many_rows_over_zero_and_tiny_values(g, D, T, G, change):
    lens = [0, 37, 96, 300]
    s, d_q, q = _filled(g, lens, T, change, G=G, D=D)
    _check(s, d_q, q, lens)


def _wide(ratio):
    """q with a channel `ratio` times the others, where the keys are zero (one
    pair, which the rotation turns into itself)."""
    def change(x, q, kv):
        half = x.shape[-1] // 2
        x[:, :, :q, [0, half]] *= np.float32(ratio)
        x[:, :, q:q + kv, 0] = x[:, :, q:q + kv, half] = 0
    return change


@pytest.mark.parametrize("ratio", [300, 30000])
@pytest.mark.parametrize("T,G", [(40, 4), (100, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_rows_of_queries_with_a_wide_channel(g, D, T, G, ratio):
    """The first rows see a key or two, so that a score's error shows as it is."""
    lens = [0, 37, 300]
    s, d_q, q = _filled(g, lens, T, _wide(ratio), G=G, D=D)
    _check(s, d_q, q, lens)


def _uneven(x, q, kv):             # neighbours of very different sizes
    rng = np.random.default_rng(7)
    x[:, :, q:q + kv] *= (10.0 ** rng.integers(-6, 1, x.shape[:2] + (kv, 1))).astype(np.float32)
    x[:, :, q + kv:] *= (10.0 ** rng.integers(-9, 9, x.shape[:2] + (kv, 1))).astype(np.float32)


def _giants(T, lens, first, factor, at=-1):
    """Heads `first` (k 0, v 1) of a sequence's new tokens from `at` on times `factor`."""
    def change(x, q, kv):
        for b, n in enumerate(lens):
            x[b, n + at % T:, q + first * kv:q + (first + 1) * kv] *= np.float32(factor)
    return change


@pytest.mark.parametrize("ratio", [300, 30000])
@pytest.mark.parametrize("T,G", [(40, 1), (70, 1), (3, 8), (1, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_of_queries_with_a_wide_channel(g, D, T, G, ratio):
    """Lengths of 0 and 40 or more: the first rows see a key or two of a closed
    block."""
    lens = [0, 37, 300]
    s, d_q, q = _filled(g, lens, T, _wide(ratio), G=G, D=D)
    _check(s, d_q, q, lens)


@pytest.mark.parametrize("T", [3, 40])
def test_rows_of_queries_of_any_size(g, T):
    """Each row with scores of size 1: queries of 1e-30 to 1e30 as they come, by
    a scale that suits them."""
    lens = [0, 37]
    for power in (-30, -12, 0, 12, 24):
        def change(x, q, kv, f=np.float32(10.0) ** power):
            x[:, :, :q] *= f
        s, d_q, q = _filled(g, lens, T, change, G=2)
        _check(s, d_q, q, lens, scale=float(np.float32(0.1) / np.float32(10.0) ** power))


FEW_OPEN = [(5, 8, 64), (5, 8, 128), (2, 8, 64), (8, 1, 64), (8, 1, 128), (9, 7, 64)]


@pytest.mark.parametrize("T,G,D", FEW_OPEN)
def test_few_rows_over_an_open_block_of_unlike_rows(g, T, G, D):
    """What a later token holds does not reach the rows before it; rows next to
    each other keep their own bits."""
    lens = [0, 37, 96, 300, 20]
    for change, skip in ((_uneven, 0), (_giants(T, lens, 1, 1e25), 0),
                         (_giants(T, lens, 0, 1e18), 1)):
        s, d_q, q = _filled(g, lens, T, change, G=G, D=D)
        _check(s, d_q, q, lens, skip=skip)


@pytest.mark.parametrize("T,G,D,blk", [(16, 8, 64, 32), (16, 8, 128, 32), (40, 2, 64, 64),
                                       (33, 8, 64, 16), (100, 1, 128, 16), (150, 4, 64, 128)])
def test_many_rows_over_an_open_block_of_unlike_rows(g, T, G, D, blk):
    """The same; and later blocks that have closed, next to those that a row sees."""
    lens = [0, 37, 96, 300, 20]
    for change, skip in ((_uneven, 0), (_giants(T, lens, 1, 1e25), 0),
                         (_giants(T, lens, 1, 1e25, T // 2), 0), (_giants(T, lens, 0, 1e18), 1)):
        s, d_q, q = _filled(g, lens, T, change, G=G, D=D, blk=blk)
        _check(s, d_q, q, lens, skip=skip)


@pytest.mark.parametrize("T", [1, 3, 24])
@pytest.mark.parametrize("closed", [False, True])
def test_where_a_nan_goes(g, T, closed):
    """In q or K: to output, lse and weights of the rows that see it; in V: to
    their outputs alone."""
    for part in ("q", "k", "v"):
        n0 = 96 - T if closed else 100

        def change(x, q, kv):
            first = {"q": 0, "k": q, "v": q + kv}[part]
            x[0, n0 + T - 1, first, 5] = np.nan
        s, d_q, q = _filled(g, [n0], T, change, Hkv=1, G=8)
        out, lse, w = g.alloc((T, 8, 64)), g.alloc((T, 8)), g.tensor(np.zeros((1, 1, 512), np.float32))
        g.attention_kv8(d_q, s.cache, out, q_len=T, q_heads=8, scale=0.125, lse=lse, weights=w)
        o, z, w = np.isnan(out.download()), np.isnan(lse.download()), np.isnan(w.download()[0, 0])
        # rotation spreads one element over a pair; a closed block is all NaN
        late = (np.arange(n0, n0 + T) >= 64) if closed and part != "q" else np.arange(T) == T - 1
        want = np.repeat(late[:, None], 8, 1)
        if part == "q":
            want[T - 1, 1:] = False
        assert np.array_equal(o.all(-1), want) and np.array_equal(o.any(-1), want), part
        assert np.array_equal(z, want & (part != "v")), part
        assert w[:n0 + T].all() == (part != "v") and w.any() == (part != "v"), part


@pytest.mark.parametrize("T,G", [(5, 1), (8, 2), (9, 8), (24, 8)])
def test_rows_behind_the_new_tokens_have_no_part(g, T, G):
    lens, new = [0, 37, 96], [T - 3, 0, 1]
    s, d_q, q = _filled(g, lens, T, lambda x, a, b: None, G=G, new=new)
    got = []
    for junk in (0.0, np.nan, np.inf, 3e38):
        x = q.copy()
        for b, n in enumerate(new):
            x[b, n:] = junk
        d_q.upload(x.reshape(d_q.shape))
        got.append(_check(s, d_q, q, lens))
        s.rng = np.random.default_rng(1)
    for other in got[2:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[1], other))


def _zero_keys(x, q, kv):
    x[:, :, q] = 0                      # kv head 0: all keys; kv head 1: some
    x[:, 5::3, q + 1:q + kv] = 0


def _zero_queries(x, q, kv):
    x[:, :, 0] = 0
    x[:, -1, :q] = 0


def _tiny_keys(x, q, kv):
    x[:, :, q:q + kv] *= np.float32(1e-36)
    x[:, ::7, q:q + kv] = 0


@pytest.mark.parametrize("change", [_zero_keys, _zero_queries, _tiny_keys])
@pytest.mark.parametrize("T,G,D", [(1, 8, 64), (2, 8, 64), (5, 8, 128), (16, 8, 64), (20, 8, 128)])
def test_zero_and_tiny_keys_and_queries(g, T, G, D, change):
    lens = [0, 37, 96, 300]
    s, d_q, q = _filled(g, lens, T, change, G=G, D=D)
    for scale in (None, -0.3, 0.0):
        _check(s, d_q, q, lens, scale=scale)


def _light_open(x, q, kv):
    """Closed values in one channel and with all the weight; open ones, of the same
    size, in the others and with 2^-20 of it (scores by the pair of channels that
    hardly turns)."""
    half = x.shape[-1] // 2
    x[:, :, :q + kv] = 0
    x[:, :, :q, half - 1] = 10
    x[:, 16:, q:q + kv, half - 1] = -1.4 * x.shape[-1] ** 0.5
    x[:, :16, q + kv:] = 0
    x[:, :, q + kv:, 0] = 0
    x[:, :16, q + kv:, 0] = 1


@pytest.mark.parametrize("T,G,D", [(24, 8, 64), (31, 4, 128), (24, 1, 64)])
def test_light_open_values_beside_heavy_closed_ones(g, T, G, D):
    s, d_q, q = _filled(g, [0], T, _light_open, G=G, D=D, S=64, blk=16)
    o, _, _ = _check(s, d_q, q, [0])
    assert 0 < np.abs(o[0, 16:, :, 1:]).max() < 1e-4
