"""The 8-bit key / value cache on the device against its 64-bit restatement:
append (exact), read-back, attention with its softmax sums and gathered
weights, eviction (exact), bookkeeping, the operators in a row as one captured
step, and the decoder that uses them."""
from dataclasses import replace

import numpy as np
import pytest

import _kv8_np as N
from spirv_inference_b200 import _lib, llama
from spirv_inference_b200.graph import Graph, Kv8Cache

pytestmark = pytest.mark.gpu


@pytest.fixture
def g(gpu):
    with Graph(gpu) as graph:
        yield graph


def _rope(S, D):
    inv = 1.0 / (10000.0 ** (np.arange(0, D, 2, dtype=np.float32) / D))
    f = np.outer(np.arange(S, dtype=np.float32), inv)
    f = np.concatenate([f, f], -1)
    return np.cos(f).astype(np.float32), np.sin(f).astype(np.float32)


class Setup:
    """A device cache and its restatement, filled by appends."""

    def __init__(self, g, B, Hkv, G, D, S, blk, seed=0, lens=None):
        self.g, self.B, self.Hkv, self.G, self.D, self.S, self.blk = g, B, Hkv, G, D, S, blk
        self.Hq = Hkv * G
        self.rng = np.random.default_rng(seed)
        self.cache = g.kv8_cache(B, Hkv, S, D, block=blk)
        # garbage behind the ends must not matter
        for t in (self.cache.k_scale, self.cache.v_scale, self.cache.k_tail, self.cache.v_tail):
            t.upload(np.full(t.shape, np.nan, np.float32))
        for t in (self.cache.k, self.cache.v):
            t.upload(self.rng.integers(-128, 128, t.shape).astype(np.int8))
        self.np = [[(N.Cache(S, blk, D), N.Cache(S, blk, D)) for _ in range(Hkv)]
                   for _ in range(B)]
        self.rows = S + 64
        self.tables = _rope(self.rows, D)
        self.cos, self.sin = (g.tensor(t) for t in self.tables)
        self.pos = g.tensor(np.zeros(B, np.int32), np.int32)
        if lens is not None and max(lens):
            self.append(max(lens), lens)
            self.advance(max(lens), lens)

    def append(self, T, new=None, qkv=None, pad=0):
        """Appends new[b] of T rows on both sides; returns q on both sides."""
        B, Hq, Hkv, D = self.B, self.Hq, self.Hkv, self.D
        ld = (Hq + 2 * Hkv) * D + pad
        if qkv is None:
            qkv = self.rng.standard_normal((B, T, ld)).astype(np.float32)
        new = [T] * B if new is None else list(new)
        d_new = self.g.tensor(np.array(new, np.int32), np.int32)
        d_q = self.g.tensor(np.full((B * T, Hq, D), 7.0, np.float32))
        pos = self.pos.download()
        self.g.rope_kv8_append(self.g.tensor(qkv), ld, self.cos, self.sin, self.pos, d_q,
                               self.cache, q_len=T, q_heads=Hq, new_lens=d_new)
        q = np.full((B, T, Hq, D), 7.0, np.float32)
        for b in range(B):
            n = min(max(new[b], 0), T)
            x = qkv[b, :n, :(Hq + 2 * Hkv) * D].reshape(n, Hq + 2 * Hkv, D)
            c, s = (t[pos[b]:pos[b] + n, None] for t in self.tables)
            with np.errstate(invalid="ignore"):
                r = N.rotate(x[:, :Hq + Hkv], c, s)
            q[b, :n] = r[:, :Hq]
            for h in range(Hkv):
                self.np[b][h][0].append(r[:, Hq + h])
                self.np[b][h][1].append(x[:, Hq + Hkv + h])
        self.new, self.T, self.d_new = new, T, d_new
        return d_q, q

    def advance(self, T, new=None):
        d_new = self.g.tensor(np.array([T] * self.B if new is None else new, np.int32), np.int32)
        self.g.kv8_advance(self.cache, self.pos, q_len=T, new_lens=d_new)

    def check_cache(self):
        c = self.cache
        dev = [[t.download() for t in ts] for ts in ((c.k, c.k_scale, c.k_tail),
                                                     (c.v, c.v_scale, c.v_tail))]
        for b in range(self.B):
            for h in range(self.Hkv):
                for i in (0, 1):
                    n = self.np[b][h][i]
                    full = n.n // self.blk
                    q8, sc, tail = (t[b, h] for t in dev[i])
                    assert np.array_equal(sc[:full], n.scale[:full], equal_nan=True), (b, h, i)
                    assert np.array_equal(q8[:full * self.blk], n.q8[:full * self.blk])
                    left = n.n - full * self.blk
                    assert np.array_equal(tail[:left], n.tail[:left], equal_nan=True)

    def check_attention(self, d_q, q, len0, scale=None, with_weights=True, finite=True):
        """len0: tokens before the last append."""
        B, T, Hq, D, G, S = self.B, self.T, self.Hq, self.D, self.G, self.S
        scale = D ** -0.5 if scale is None else scale
        out, lse = self.g.tensor(np.full((B * T, Hq, D), 5.0, np.float32)), self.g.tensor(
            np.full((B * T, Hq), 5.0, np.float32))
        w0 = self.rng.uniform(0, 1, (B, self.Hkv, S)).astype(np.float32)
        if len0[0] < S:
            w0[0, 0, -1] = np.nan                # not in use, or a new token's
        w = self.g.tensor(w0)
        self.g.attention_kv8(d_q, self.cache, out, q_len=T, q_heads=Hq, scale=scale,
                             new_lens=self.d_new, lse=lse, weights=w if with_weights else None)
        o, z, wd = out.download().reshape(B, T, Hq, D), lse.download().reshape(B, T, Hq), \
            w.download()
        for b in range(B):
            n = min(max(self.new[b], 0), T)
            assert np.all(o[b, n:] == 5.0) and np.all(z[b, n:] == 5.0)
            for h in range(self.Hkv):
                K, V = (c.values() for c in self.np[b][h])
                hs = slice(h * G, (h + 1) * G)
                if n == 0:
                    assert np.array_equal(wd[b, h], w0[b, h], equal_nan=True)
                    continue
                ro, rz, rw = N.attend(q[b, :n, hs], K, V, len0[b], scale)
                if not finite:
                    assert np.array_equal(np.isnan(o[b, :n, hs]), np.isnan(ro))
                    continue
                # Error of a score: q and its products in two 11-bit halves
                # (2^-22 each of the row's largest term), D + 8 roundings of
                # 2^-24 of sum |q k|; of exp: that, and 4 roundings.
                qk = np.abs(q[b, :n, hs]).astype(np.float64).max(-1) * np.abs(K).sum(-1).max()
                ds = abs(scale) * qk.max() * (2.0 ** -21 + (D + 8) * 2.0 ** -24)
                dp = 2 * ds + 2.0 ** -20
                assert np.abs(o[b, :n, hs] - ro).max() <= np.abs(V).max() * dp, (b, h)
                assert np.all(np.abs(z[b, :n, hs] - rz) <= ds + 2.0 ** -21 * (1 + np.abs(rz)))
                if not with_weights:
                    continue
                total = len(K)
                want = np.where(np.arange(total) < len0[b], w0[b, h, :total], 0) + rw
                assert np.all(np.abs(wd[b, h, :total] - want)
                              <= want * dp + n * G * 2.0 ** -22), (b, h)
                assert np.array_equal(wd[b, h, total:], w0[b, h, total:], equal_nan=True)
        return o, z, wd


@pytest.mark.parametrize("B,Hkv,G,D,S,blk,lens,T,new", [
    (1, 4, 8, 64, 64, 32, [0], 1, [1]),                # the first token
    (1, 1, 1, 64, 64, 16, [15], 1, [1]),               # closes a block
    (1, 1, 1, 128, 128, 64, [63], 2, [2]),             # closes one and opens the next
    (3, 2, 4, 64, 96, 32, [31, 0, 40], 33, [33, 1, 0]),
    (2, 2, 7, 128, 160, 16, [5, 77], 70, [70, 69]),    # several blocks at once
    (2, 1, 2, 64, 128, 128, [100, 127], 28, [28, 1]),
    (2, 1, 3, 64, 64, 32, [60, 64], 9, [9, 9]),        # past the end
    (1, 2, 2, 64, 64, 32, [10], 40, [500]),            # new_lens above q_len
    (2, 1, 1, 64, 64, 32, [20, 3], 5, [-3, 5])])
def test_append_read_attend(g, B, Hkv, G, D, S, blk, lens, T, new):
    s = Setup(g, B, Hkv, G, D, S, blk, lens=lens)
    d_q, q = s.append(T, new, pad=8)
    assert np.array_equal(d_q.download().reshape(q.shape), q)
    s.check_cache()
    # read-back before the advance, from uneven starts
    starts = np.array([max(0, n - 5) - (0 if i else 2) for i, n in enumerate(lens)], np.int32)
    count = T + 9
    k_out, v_out = (g.alloc((B, Hkv, count, D)) for _ in range(2))
    g.kv8_read(s.cache, k_out, v_out, count=count, starts=g.tensor(starts, np.int32), q_len=T,
               new_lens=s.d_new)
    for i, got in enumerate((k_out.download(), v_out.download())):
        for b in range(B):
            for h in range(Hkv):
                x = s.np[b][h][i].values()
                for r in range(count):
                    at = starts[b] + r
                    want = x[at].astype(np.float32) if 0 <= at < len(x) else 0
                    assert np.array_equal(got[b, h, r], np.broadcast_to(want, (D,))), (b, h, r)
    s.check_attention(d_q, q, lens)
    s.advance(T, new)
    n = [min(max(v, 0), T) for v in new]
    assert s.cache.lens.download().tolist() == [min(a + b, S) for a, b in zip(lens, n)]
    assert s.pos.download().tolist() == [a + b for a, b in zip(lens, n)]


def test_contents_do_not_depend_on_the_calls(g):
    B, Hkv, G, D, S, blk = 2, 2, 2, 64, 128, 32
    a = Setup(g, B, Hkv, G, D, S, blk)
    x = a.rng.standard_normal((B, 100, (G + 2) * Hkv * D)).astype(np.float32)
    a.append(100, qkv=x)
    b = Setup(g, B, Hkv, G, D, S, blk)
    for lo, hi in ((0, 1), (1, 32), (32, 63), (63, 65), (65, 100)):
        b.append(hi - lo, qkv=np.ascontiguousarray(x[:, lo:hi]))
        b.advance(hi - lo)
    for s in (a, b):
        s.check_cache()
    assert np.array_equal(a.cache.k.download()[:, :, :96], b.cache.k.download()[:, :, :96])
    assert np.array_equal(a.cache.v_tail.download()[:, :, :4], b.cache.v_tail.download()[:, :, :4])


def test_append_rounding_edges(g):
    """Values on and next to halves of a step, zeros, tiny, huge, NaN, inf."""
    D, blk = 64, 16
    s = Setup(g, 1, 1, 1, D, 128, blk)
    x = np.zeros((1, 112, 3 * D), np.float32)
    rng = np.random.default_rng(3)
    half = (np.arange(blk * D) % 255 - 127) * np.float32(0.5)
    x[0, :16, 2 * D:] = (half * np.float32(127 / 63.5)).reshape(blk, D) / 2   # exact halves
    x[0, :16, 2 * D] = 127.0
    x[0, 16:32, 2 * D:] = np.nextafter(x[0, :16, 2 * D:], np.float32(np.inf))
    x[0, 32:48, 2 * D:] = rng.uniform(-1e-37, 1e-37, (blk, D))                # held as zero
    x[0, 48:64, 2 * D:] = rng.uniform(-3e38, 3e38, (blk, D))
    x[0, 64:80, 2 * D:] = rng.standard_normal((blk, D))
    x[0, 70, 2 * D + 3] = np.inf
    x[0, 80:96, 2 * D:] = rng.standard_normal((blk, D))
    x[0, 95, 2 * D + 63] = np.nan
    x[0, 96:112, 2 * D:] = rng.standard_normal((blk, D)) * 10.0 ** rng.integers(-6, 6, (blk, 1))
    s.append(112, qkv=x)
    # the largest magnitude of an infinite block is its scale
    s.check_cache()


def test_position_outside_the_tables_is_nan(g):
    s = Setup(g, 1, 1, 1, 64, 64, 32)
    s.pos.upload(np.array([s.rows - 1], np.int32))
    d_q = g.alloc((2, 1, 64))
    x = g.tensor(np.ones((2, 192), np.float32))
    g.rope_kv8_append(x, 192, s.cos, s.sin, s.pos, d_q, s.cache, q_len=2, q_heads=1)
    q = d_q.download()
    assert np.isfinite(q[0]).all() and np.isnan(q[1]).all()


@pytest.mark.parametrize("G", [1, 2, 3, 7, 8, 12, 32])
@pytest.mark.parametrize("D,blk", [(64, 32), (128, 16)])
def test_attend_one_token_lengths(g, G, D, blk):
    """Decode: history lengths around every tile and block border."""
    lens = [0, 1, 15, 16, 17, 31, 63, 64, 65, 127, 128, 300, 511]
    s = Setup(g, len(lens), 2, G, D, 512, blk, seed=G, lens=lens)
    d_q, q = s.append(1)
    s.check_attention(d_q, q, lens)


@pytest.mark.parametrize("T,G,D,blk,lens", [
    (2, 4, 64, 32, [0, 33]), (5, 8, 64, 16, [100, 3]), (16, 8, 64, 64, [64, 200]),
    (17, 1, 128, 32, [0, 31]), (64, 2, 64, 32, [0, 150]), (130, 3, 64, 128, [5, 300]),
    (200, 8, 64, 32, [7, 250]), (129, 4, 128, 64, [1, 260])])
def test_attend_many_tokens(g, T, G, D, blk, lens):
    s = Setup(g, 2, 2, G, D, 512, blk, seed=T, lens=lens)
    d_q, q = s.append(T, [T, max(1, T - 3)])
    s.check_attention(d_q, q, lens)


@pytest.mark.parametrize("B,Hkv,G,D,T,lens", [
    (1, 1, 8, 64, 1, [8000]), (1, 2, 4, 128, 1, [7777]), (1, 2, 5, 64, 3, [6000]),
    (2, 4, 2, 128, 1, [8100, 37]), (3, 3, 1, 64, 2, [0, 8190, 4097])])
def test_attend_few_long_sequences(g, B, Hkv, G, D, T, lens):
    """Keys of a sequence over large clusters, of sizes that do not divide the rows."""
    s = Setup(g, B, Hkv, G, D, 8192, 64, seed=D, lens=lens)
    d_q, q = s.append(T)
    s.check_attention(d_q, q, lens)


@pytest.mark.parametrize("T,G", [(79, 1), (80, 1), (9, 8), (10, 8), (20, 4), (27, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_from_few_rows_to_many(g, T, G, D):
    s = Setup(g, 2, 1, G, D, 512, 32, seed=T, lens=[370, 33])
    d_q, q = s.append(T, [T, T - 1])
    s.check_attention(d_q, q, [370, 33])


@pytest.mark.parametrize("T,G,D,blk,lens,scale", [
    (300, 1, 64, 128, [0, 200], None), (400, 2, 64, 16, [3, 100], -0.1),
    (150, 6, 128, 32, [350, 0], -0.07), (64, 2, 64, 64, [440, 448], 0.0)])
def test_attend_many_tokens_scales(g, T, G, D, blk, lens, scale):
    """Row tiles dealt to a cluster, keys that only some of them see, scales of any sign."""
    s = Setup(g, 2, 2, G, D, 512, blk, seed=T, lens=lens)
    d_q, q = s.append(T)
    s.check_attention(d_q, q, lens, scale=scale)


@pytest.mark.parametrize("B,Hkv,G,D,T,S,lens", [
    (1, 1, 8, 64, 16, 4096, [4000]), (2, 1, 4, 128, 40, 2048, [1999, 1]),
    (3, 2, 16, 64, 17, 2048, [0, 64, 2031]), (1, 1, 1, 128, 260, 1024, [700]),
    (2, 2, 32, 64, 4, 512, [508, 100])])
def test_attend_rows_split_over_keys(g, B, Hkv, G, D, T, S, lens):
    """Few row tiles: their keys over a cluster, some CTAs of which have none."""
    s = Setup(g, B, Hkv, G, D, S, 32, seed=T, lens=lens)
    d_q, q = s.append(T, [T] + [max(1, T - 5)] * (B - 1))
    s.check_attention(d_q, q, lens)


@pytest.mark.parametrize("T", [1, 24])
def test_nan_rows_and_values_over_clusters(g, T):
    """A NaN in a query or in an open V reaches the rows that see it, no others."""
    s = Setup(g, 1, 2, 8, 64, 4096, 32, lens=[3000])
    x = s.rng.standard_normal((1, T, 20 * 64)).astype(np.float32)
    x[0, T - 1, 18 * 64 + 3] = np.nan       # V of kv head 0 of the last token
    x[0, 0, 9 * 64] = np.nan                # q of head 9 (kv head 1) of the first
    d_q, q = s.append(T, qkv=x)
    out, lse = g.tensor(np.zeros((T, 16, 64), np.float32)), g.tensor(
        np.zeros((T, 16), np.float32))
    g.attention_kv8(d_q, s.cache, out, q_len=T, q_heads=16, scale=0.125, lse=lse)
    o = out.download().reshape(T, 16, 64)
    bad = np.zeros((T, 16), bool)
    bad[T - 1, :8] = True
    bad[0, 9] = True
    assert np.isnan(o[bad]).all(axis=-1).all() and np.isfinite(o[~bad]).all()
    assert np.isnan(lse.download().reshape(T, 16)[0, 9])


def test_attend_sharp_and_flat(g):
    """Scores of +-100 and of 0: one slot takes everything; all are equal."""
    s = Setup(g, 1, 2, 4, 64, 256, 32, lens=[200])
    d_q, q = s.append(1)
    s.check_attention(d_q, q, [200], scale=12.0)
    s.check_attention(d_q, q, [200], scale=0.0)


def test_nan_in_a_block_is_seen_and_behind_the_end_is_not(g):
    s = Setup(g, 1, 1, 2, 64, 128, 32)
    x = s.rng.standard_normal((1, 70, 4 * 64)).astype(np.float32)
    x[0, 40, 3 * 64 + 5] = np.nan          # V of slot 40: block 1
    d_q, q = s.append(70, qkv=x)
    o, _, _ = s.check_attention(d_q, q, [0], finite=False)
    assert np.isfinite(o[0, :32]).all() and np.isnan(o[0, 32:]).any()


def test_long_cache_offsets_pass_32_bits(g):
    """The last sequence's rows lie more than 2^31 values into the cache."""
    B, Hkv, D, S, blk = 3, 8, 128, 1 << 20, 32
    lens = [3, 40, 90]
    s = Setup.__new__(Setup)
    s.g, s.B, s.Hkv, s.G, s.D, s.S, s.blk, s.Hq = g, B, Hkv, 1, D, S, blk, Hkv
    s.rng = np.random.default_rng(1)
    s.cache = g.kv8_cache(B, Hkv, S, D, block=blk)
    assert s.cache.k.size > 2 ** 31
    s.np = [[(N.Cache(128, blk, D), N.Cache(128, blk, D)) for _ in range(Hkv)] for _ in range(B)]
    s.rows, s.tables = 256, _rope(256, D)
    s.cos, s.sin = (g.tensor(t) for t in s.tables)
    s.pos = g.tensor(np.zeros(B, np.int32), np.int32)
    s.append(90, lens)
    s.advance(90, lens)
    d_q, q = s.append(1)
    out = g.alloc((B, Hkv, D))
    g.attention_kv8(d_q, s.cache, out, q_len=1, q_heads=Hkv, scale=0.1)
    o = out.download()
    for b in range(B):
        for h in range(Hkv):
            K, V = (c.values() for c in s.np[b][h])
            want, _, _ = N.attend(q[b, :, h:h + 1], K, V, lens[b], 0.1)
            assert np.abs(o[b, h] - want[0, 0]).max() <= 1e-5


def test_long_cache_offsets_many_rows(g):
    """The same, for the chunk itself: its attention, weights and read-back."""
    B, Hkv, D, S, blk, T = 3, 8, 128, 1 << 20, 32, 100
    new = [100, 3, 95]
    s = Setup.__new__(Setup)
    s.g, s.B, s.Hkv, s.G, s.D, s.S, s.blk, s.Hq = g, B, Hkv, 1, D, S, blk, Hkv
    s.rng = np.random.default_rng(2)
    s.cache = g.kv8_cache(B, Hkv, S, D, block=blk)
    s.np = [[(N.Cache(128, blk, D), N.Cache(128, blk, D)) for _ in range(Hkv)] for _ in range(B)]
    s.rows, s.tables = 256, _rope(256, D)
    s.cos, s.sin = (g.tensor(t) for t in s.tables)
    s.pos = g.tensor(np.zeros(B, np.int32), np.int32)
    d_q, q = s.append(T, new)
    out, lse, w = g.alloc((B * T, Hkv, D)), g.alloc((B * T, Hkv)), g.alloc((B, Hkv, S))
    g.attention_kv8(d_q, s.cache, out, q_len=T, q_heads=Hkv, scale=0.1, new_lens=s.d_new, lse=lse,
                    weights=w)
    k, v = g.alloc((B, Hkv, 96, D)), g.alloc((B, Hkv, 96, D))
    g.kv8_read(s.cache, k, v, count=96, q_len=T, new_lens=s.d_new)
    o, got_k = out.download().reshape(B, T, Hkv, D), k.download()
    last = w.view((S,), (B * Hkv - 1) * S).download()
    for b in range(B):
        n = new[b]
        for h in range(Hkv):
            K, V = (c.values() for c in s.np[b][h])
            want, _, weights = N.attend(q[b, :n, h:h + 1], K, V, 0, 0.1)
            assert np.abs(o[b, :n, h] - want[:, 0]).max() <= 1e-5
            assert np.array_equal(got_k[b, h, :min(n, 96)], K[:96].astype(np.float32))
    assert np.abs(last[:new[-1]] - weights).max() <= 1e-4


def test_runs_are_equal_to_the_bit(g):
    for T in (1, 40):
        s = Setup(g, 4, 2, 8, 64, 1024, 32, lens=[900, 10, 512, 333])
        d_q, q = s.append(T)
        got = []
        for _ in range(3):
            out, lse = g.alloc((4 * T, 16, 64)), g.alloc((4 * T, 16))
            w = g.alloc((4, 2, 1024))
            g.zero(w)
            g.attention_kv8(d_q, s.cache, out, q_len=T, q_heads=16, scale=0.125, lse=lse,
                            weights=w)
            got.append([t.download() for t in (out, lse, w)])
        for other in got[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(got[0], other))


# -- eviction -----------------------------------------------------------------
def _evict_check(s, w, keep, recent, sink, idx, caches, w_out):
    """The device's choice and the moved contents against the restatement."""
    got = idx.download()
    for b in range(s.B):
        for h in range(s.Hkv):
            n = s.np[b][h][0].n
            want = N.choose(w[b, h], n, keep, recent, sink)
            assert np.array_equal(got[b, h, :len(want)], want), (b, h)
            assert np.all(got[b, h, len(want):] == -1)
            assert np.array_equal(w_out[b, h, :len(want)], w[b, h, want], equal_nan=True)
            for i in (0, 1):
                r = s.np[b][h][i].cut(want)
                q8, sc, tail = (t[b, h] for t in caches[i])
                full = r.n // s.blk
                assert np.array_equal(sc[:full], r.scale[:full], equal_nan=True), (b, h, i)
                assert np.array_equal(q8[:full * s.blk], r.q8[:full * s.blk]), (b, h, i)
                assert np.array_equal(tail[:r.n - full * s.blk], r.tail[:r.n - full * s.blk],
                                      equal_nan=True)


@pytest.mark.parametrize("S,blk,D,lens,keep,recent,sink", [
    (64, 32, 64, [64, 33, 20], 32, 16, 4), (64, 16, 128, [64, 1, 0], 33, 1, 0),
    (256, 32, 64, [256, 255, 129], 128, 0, 0), (256, 64, 64, [256, 200, 97], 96, 96, 0),
    (512, 16, 64, [512, 500, 17], 300, 100, 4), (512, 128, 128, [400, 512, 511], 257, 30, 2),
    (64, 32, 64, [64, 40, 2], 1, 0, 0), (64, 32, 64, [64, 40, 2], 1, 0, 1),
    (2048, 32, 64, [2048, 1999, 1500], 1500, 512, 4), (64, 32, 64, [64, 64, 64], 64, 0, 0)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(g, S, blk, D, lens, keep, recent, sink, in_place):
    B, Hkv = len(lens), 2
    s = Setup(g, B, Hkv, 1, D, S, blk, seed=keep, lens=lens)
    w = np.exp(2 * s.rng.standard_normal((B, Hkv, S))).astype(np.float32)
    w[:, 1] = np.round(w[:, 1])                     # many ties
    w[0, 0, 3::7] = [np.nan, -np.inf, np.inf, -0.0, 0.0, 1e-40][keep % 6]
    dw = g.tensor(w)
    idx = g.alloc((B, Hkv, keep), np.int32)
    if in_place:
        c, dw2 = s.cache, dw
        g.kv8_evict(c, dw, keep, idx=idx, recent=recent, sink=sink)
    else:
        S2 = -(-keep // blk) * blk
        before = [t.download() for t in (s.cache.k, s.cache.v_scale, s.cache.k_tail)]
        c = g.kv8_cache(B, Hkv, S2, D, block=blk)
        dw2 = g.alloc((B, Hkv, S2))
        g.kv8_evict(s.cache, dw, keep, idx=idx, recent=recent, sink=sink, into=c,
                    into_weights=dw2)
        for t, x in zip((s.cache.k, s.cache.v_scale, s.cache.k_tail), before):
            assert np.array_equal(t.download(), x, equal_nan=True)
        assert np.array_equal(dw.download(), w, equal_nan=True)
    caches = [[t.download() for t in ts] for ts in ((c.k, c.k_scale, c.k_tail),
                                                    (c.v, c.v_scale, c.v_tail))]
    _evict_check(s, w, keep, recent, sink, idx, caches, dw2.download())
    if in_place:      # lens follows by the advance, and the cache goes on from there
        g.kv8_advance(s.cache, limit=keep)
        assert s.cache.lens.download().tolist() == [min(n, keep) for n in lens]
        for b in range(B):
            for h in range(Hkv):
                at = N.choose(w[b, h], s.np[b][h][0].n, keep, recent, sink)
                s.np[b][h] = tuple(x.cut(at) for x in s.np[b][h])
        now = [min(n, keep) for n in lens]
        d_q, q = s.append(3)
        s.check_cache()
        s.check_attention(d_q, q, now)


def test_evict_equal_scales_keep_their_bits(g):
    """Rows of one magnitude: nothing is rounded again, however often."""
    S, blk, D = 256, 32, 64
    s = Setup(g, 1, 1, 1, D, S, blk)
    x = s.rng.uniform(-1, 1, (1, S, 3 * D)).astype(np.float32)
    x[:, :, 2 * D] = 1.0
    s.append(S, qkv=x)
    s.advance(S)
    v0 = s.cache.v.download()[0, 0]
    w = s.rng.uniform(0, 1, (1, 1, S)).astype(np.float32)
    idx = g.alloc((1, 1, 192), np.int32)
    g.kv8_evict(s.cache, g.tensor(w), 192, idx=idx)
    at = idx.download()[0, 0]
    assert np.array_equal(s.cache.v.download()[0, 0, :192], v0[at])


def test_refusals(g):
    s = Setup(g, 2, 2, 2, 64, 64, 32)
    q, out = g.alloc((2, 4, 64)), g.alloc((2, 4, 64))
    idx, w = g.alloc((2, 2, 64), np.int32), g.alloc((2, 2, 64))
    other = g.kv8_cache(2, 2, 64, 64, block=16)
    shifted = Kv8Cache(s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale, s.cache.k_tail,
                       g.alloc((2, 2, 32, 64)), s.cache.lens, block=32)
    calls = [
        lambda: g.attention_kv8(q, s.cache, out, q_len=0, q_heads=4, scale=1.0),
        lambda: g.attention_kv8(q, s.cache, out, q_len=1, q_heads=3, scale=1.0),
        lambda: g.attention_kv8(q, s.cache, out, q_len=1, q_heads=4, scale=1.0, weights=w),
        lambda: g.attention_kv8(q.view((1,), 1), s.cache, out, q_len=1, q_heads=4, scale=1.0),
        lambda: g.rope_kv8_append(q, 511, s.cos, s.sin, s.pos, out, s.cache, q_len=1, q_heads=4),
        lambda: g.rope_kv8_append(q, 512, s.cos, s.sin, s.pos, out, s.cache, q_len=0, q_heads=4),
        lambda: g.kv8_read(s.cache, q, out, count=0),
        lambda: g.kv8_read(s.cache, q, out, count=1, q_len=-1),
        lambda: g.kv8_evict(s.cache, w, 0, idx=idx),
        lambda: g.kv8_evict(s.cache, w, 65, idx=idx),
        lambda: g.kv8_evict(s.cache, w, 8, idx=idx, recent=6, sink=3),
        lambda: g.kv8_evict(s.cache, w, 8, idx=idx, recent=-1),
        lambda: g.kv8_evict(s.cache, w, 8, idx=idx, into=other, into_weights=w),
        lambda: g.kv8_evict(s.cache, w, 8, idx=idx, into=shifted, into_weights=w),
        lambda: g.kv8_evict(s.cache, w, 8, idx=idx, into=s.cache,
                            into_weights=g.alloc((2, 2, 64))),
        lambda: g.kv8_advance(s.cache, s.pos, q_len=-1),
        lambda: g.kv8_advance(s.cache, s.pos, q_len=1, limit=0),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(_lib.SpxError) as e:
            call()
        assert e.value.code == _lib.SPX_ERR_INVALID_ARGUMENT, i
    with pytest.raises(ValueError):
        g.kv8_evict(s.cache, w, 8, idx=idx, into=s.cache)
    g.sync()


def test_queries_and_outputs_apart(g):
    """What a row writes, another may still have to read."""
    s = Setup(g, 1, 1, 2, 64, 64, 32)
    both = g.alloc((4, 2, 64))
    for at in (0, 2 * 64):
        with pytest.raises(_lib.SpxError) as e:
            g.attention_kv8(both, s.cache, both.view((2, 2, 64), at), q_len=2, q_heads=2, scale=1.0)
        assert e.value.code == _lib.SPX_ERR_INVALID_ARGUMENT
    s.append(2)
    g.attention_kv8(both, s.cache, both.view((2, 2, 64), 4 * 64), q_len=2, q_heads=2, scale=1.0)
    g.sync()


# -- together -----------------------------------------------------------------
def test_captured_step(g):
    """Append, attention with weights, log probabilities of a made-up head and
    the advance as one captured graph, replayed over block borders, equal to
    the same calls run one by one."""
    B, Hkv, G, D, S, blk, V = 3, 2, 4, 64, 128, 16, 500
    Hq = Hkv * G
    rng = np.random.default_rng(5)
    xs = rng.standard_normal((40, B, (Hq + 2 * Hkv) * D)).astype(np.float32)
    results = []
    for captured in (True, False):
        s = Setup(g, B, Hkv, G, D, S, blk, lens=[14, 0, 31], seed=9)
        qkv, q, out = g.alloc((B, (Hq + 2 * Hkv) * D)), g.alloc((B, Hq, D)), g.alloc((B, Hq, D))
        lse, w = g.alloc((B, Hq)), g.alloc((B, Hkv, S))
        ids = g.tensor(np.array([3, 499, 100], np.int32), np.int32)
        lp, ent = g.alloc((B,)), g.alloc((B,))
        g.zero(w)

        def step():
            g.rope_kv8_append(qkv, (Hq + 2 * Hkv) * D, s.cos, s.sin, s.pos, q, s.cache, q_len=1,
                              q_heads=Hq)
            g.attention_kv8(q, s.cache, out, q_len=1, q_heads=Hq, scale=0.125, lse=lse, weights=w)
            g.token_logprobs(out.view((B, V)), Hq * D, B, V, ids, lp, entropy=ent)
            g.kv8_advance(s.cache, s.pos, q_len=1)

        if captured:
            g.capture_begin()
            step()
            g.capture_end()
        got = []
        for x in xs:
            qkv.upload(x)
            g.replay() if captured else step()
            got.append([t.download() for t in (out, lse, lp, ent)])
        results.append((got, [t.download() for t in (s.cache.k, s.cache.k_tail, w, s.pos)]))
    for a, b in zip(results[0][0], results[1][0]):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
    for x, y in zip(results[0][1], results[1][1]):
        assert np.array_equal(x, y, equal_nan=True)


def test_two_graphs_on_their_own_streams(gpu):
    """Two graphs with their own caches, calls interleaved, neither waiting."""
    alone, both = [], []
    for seed in (1, 2):
        with Graph(gpu) as g:
            s = Setup(g, 2, 2, 4, 64, 512, 32, lens=[400, 123], seed=seed)
            alone.append(_attend_steps(s))
    with Graph(gpu) as g1, Graph(gpu) as g2:
        ss = [Setup(x, 2, 2, 4, 64, 512, 32, lens=[400, 123], seed=seed)
              for x, seed in ((g1, 1), (g2, 2))]
        qs = [s.append(1)[0] for s in ss]
        outs = [s.g.alloc((2, 8, 64)) for s in ss]
        for _ in range(20):
            for s, q, o in zip(ss, qs, outs):
                s.g.attention_kv8(q, s.cache, o, q_len=1, q_heads=8, scale=0.125)
        both = [o.download() for o in outs]
    for a, b in zip(alone, both):
        assert np.array_equal(a, b)


def _attend_steps(s):
    q, out = s.append(1)[0], s.g.alloc((2, 8, 64))
    s.g.attention_kv8(q, s.cache, out, q_len=1, q_heads=8, scale=0.125)
    return out.download()


def test_chunks_captured_on_two_streams(gpu):
    """Prompts taken in chunks of many rows: two graphs at once, of 64 and 128
    values a head, each a captured chunk replayed while its lengths grow, equal
    to the same calls one by one."""
    T, S, Hkv, G = 24, 512, 2, 8
    Hq = Hkv * G

    class Run:
        def __init__(self, g, D):
            self.s, self.D = Setup(g, 2, Hkv, G, D, S, 32, lens=[5, 130], seed=D), D
            ld = (Hq + 2 * Hkv) * D
            self.qkv, self.q, self.out = (g.alloc((2 * T, n)) for n in (ld, Hq * D, Hq * D))
            self.lse, self.w = g.alloc((2 * T, Hq)), g.alloc((2, Hkv, S))
            g.zero(self.w)
            self.xs = np.random.default_rng(D).standard_normal((6, 2 * T, ld)).astype(np.float32)

        def step(self):
            s, g = self.s, self.s.g
            g.rope_kv8_append(self.qkv, self.qkv.shape[1], s.cos, s.sin, s.pos, self.q, s.cache,
                              q_len=T, q_heads=Hq)
            g.attention_kv8(self.q, s.cache, self.out, q_len=T, q_heads=Hq, scale=self.D ** -0.5,
                            lse=self.lse, weights=self.w)
            g.kv8_advance(s.cache, s.pos, q_len=T)

        def results(self):
            return [t.download() for t in (self.out, self.lse, self.w, self.s.cache.lens)]

    alone = []
    for D in (64, 128):
        with Graph(gpu) as g:
            r = Run(g, D)
            for x in r.xs:
                r.qkv.upload(x)
                r.step()
            alone.append(r.results())
    with Graph(gpu) as g1, Graph(gpu) as g2:
        runs = [Run(g1, 64), Run(g2, 128)]
        for r in runs:
            r.s.g.capture_begin()
            r.step()
            r.s.g.capture_end()
        for i in range(6):
            for r in runs:
                r.qkv.upload(r.xs[i])
            for r in runs:
                r.s.g.replay()
        for r, want in zip(runs, alone):
            for x, y in zip(r.results(), want):
                assert np.isfinite(y).all() and np.array_equal(x, y)


# -- decoder ------------------------------------------------------------------
def _logits_match(dec, cfg, W, prompt, toks, blk, **kw):
    rope = llama.rope_tables(cfg, max(cfg.max_seq, prompt.shape[1] + toks.shape[1]))
    last = dec.last_logits()
    for b in range(prompt.shape[0]):
        cut = kw["cut"](b) if "cut" in kw else None
        logits = N.decode(cfg, W, prompt[b], toks[b], rope, blk, cut=cut)
        for i, t in enumerate(toks[b]):
            top2 = np.sort(logits[i])[-2:]
            assert int(np.argmax(logits[i])) == int(t) or top2[1] - top2[0] < 1e-3, (b, i)
        assert np.abs(last[b] - logits[-1]).max() <= 1e-3 * np.abs(logits[-1]).max()


@pytest.mark.parametrize("batch,blk", [(1, 32), (2, 16), (12, 32)])
def test_decoder_int8(gpu, batch, blk):
    cfg = llama.TINY_TEST
    W = llama.make_weights(cfg, 0)
    prompt = llama.make_prompt(cfg, batch, 30)
    for capture in (True, False):
        dec = llama.LlamaDecoder(cfg, W, batch, 30, 20, device=gpu, kv_cache="int8", kv_block=blk,
                                 capture=capture)
        try:
            toks = dec.generate(prompt)
            assert np.array_equal(toks, dec.generate(prompt))     # starts afresh
            if capture:
                first = toks
                _logits_match(dec, cfg, W, prompt[:2], toks[:2], blk)
        finally:
            dec.close()
    assert np.array_equal(first, toks)


def test_decoder_with_eviction(gpu):
    """A cache of 48 slots cut to 24 twice while 45 tokens follow a prompt of
    30: the contents follow the slots that the device chose, and each choice is
    the heaviest by the restatement's weights, near-ties aside."""
    cfg = replace(llama.TINY_TEST, max_seq=48)
    W = llama.make_weights(cfg, 4)
    prompt = llama.make_prompt(cfg, 2, 30)
    dec = llama.LlamaDecoder(cfg, W, 2, 30, 45, device=gpu, kv_cache="int8", kv_block=16,
                             kv_keep=24, kv_recent=8, kv_sink=2)
    kept = []
    evict = dec.g.kv8_evict

    def spy(cache, w, keep, **kw):
        evict(cache, w, keep, **kw)
        kept.append(kw["idx"].download())

    dec.g.kv8_evict = spy
    try:
        toks = dec.generate(prompt)
        assert len(kept) == 2 * cfg.layers

        def cut(b):
            seen = {}

            def choose(li, h, w, n):
                i = seen[li, h] = seen.get((li, h), -1) + 1
                idx = kept[i * cfg.layers + li][b, h]
                assert n == 48 and np.all(np.diff(idx) > 0)
                assert idx[:2].tolist() == [0, 1] and idx[-8:].tolist() == list(range(40, 48))
                mid = np.zeros(48, bool)
                mid[2:40] = True
                stay = np.zeros(48, bool)
                stay[idx] = True
                assert w[mid & stay].min() >= w[mid & ~stay].max() - 1e-3
                return idx
            return choose

        _logits_match(dec, cfg, W, prompt, toks, 16, cut=cut)
    finally:
        dec.close()


@pytest.mark.parametrize("kv_cache", ["fp32", "int8"])
def test_decoder_logprobs_and_score(gpu, kv_cache):
    """score() of a text that the decoder generated gives the log probabilities
    that it noted when it generated it."""
    cfg = llama.TINY_TEST
    W = llama.make_weights(cfg, 2)
    prompt = llama.make_prompt(cfg, 3, 20)
    dec = llama.LlamaDecoder(cfg, W, 3, 20, 12, device=gpu, logprobs=4, kv_cache=kv_cache,
                             kv_block=64)
    try:
        toks = dec.generate(prompt)
        lp = dec.token_logprobs()
        logits = dec.last_logits().astype(np.float64)
    finally:
        dec.close()
    assert lp["top_ids"].shape == (3, 12, 4) and np.all(lp["rank"] == 1)
    assert np.array_equal(lp["top_ids"][:, :, 0], toks)
    assert np.array_equal(lp["top_logprobs"][:, :, 0], lp["logprobs"])
    z = logits - logits.max(1, keepdims=True)
    z -= np.log(np.exp(z).sum(1, keepdims=True))
    assert np.abs(lp["entropy"][:, -1] + (np.exp(z) * z).sum(1)).max() <= 1e-5
    text = np.concatenate([prompt, toks], 1)
    dec = llama.LlamaDecoder(cfg, W, 3, 32, 1, device=gpu, kv_cache=kv_cache, kv_block=64)
    try:
        with pytest.raises(ValueError):
            dec.token_logprobs()
        sc = dec.score(text, top_k=2)
        assert sc["logprobs"].shape == (3, 31) and sc["top_ids"].shape == (3, 31, 2)
        # one pass over 32 positions and 12 single steps sum in another order;
        # logits agree to 1e-3 of their size (about 1)
        assert np.abs(sc["logprobs"][:, 19:] - lp["logprobs"]).max() <= 2e-3
        assert np.abs(sc["entropy"][:, 19:] - lp["entropy"]).max() <= 2e-3
        again = dec.score(text)
        assert set(again) == {"logprobs", "entropy", "rank"}
        assert np.array_equal(again["logprobs"], sc["logprobs"])
    finally:
        dec.close()
