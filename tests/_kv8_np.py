"""numpy restatement, in 64 bits, of the 8-bit key / value cache: what its
blocks hold, attention over it, the weights it gathers, eviction, and a decoder
that uses it.  Scales and rotated keys are rounded to fp32, as they are held."""
import numpy as np

from oracle import llama_ref as R

TINY = 127.0 * 2.0 ** -126


def scale_of(amax):
    a = np.float32(amax)
    if not np.isfinite(a):
        return a
    return np.float32(0) if a < TINY else np.float32(np.float64(a) / 127.0)


def quantise(x, s=None):
    """fp32 [rows][D] -> (int8 [rows][D], fp32 scale); s: a given scale."""
    x = np.asarray(x, np.float64)
    if s is None:
        m = np.abs(x).max()
        s = scale_of(np.nan if np.isnan(x).any() else m)
    if not np.isfinite(s) or s == 0:
        return np.zeros(x.shape, np.int8), s
    return np.clip(np.rint(x / np.float64(s)), -127, 127).astype(np.int8), s


class Cache:
    """One kv head of one sequence, K or V."""

    def __init__(self, S, blk, D):
        self.S, self.blk, self.D, self.n = S, blk, D, 0
        self.q8 = np.zeros((S, D), np.int8)
        self.scale = np.zeros(S // blk, np.float32)
        self.tail = np.zeros((blk, D), np.float32)

    def append(self, rows):
        for x in rows:
            if self.n >= self.S:
                return
            self.tail[self.n % self.blk] = x
            self.n += 1
            if self.n % self.blk == 0:
                i = self.n // self.blk - 1
                self.q8[self.n - self.blk:self.n], self.scale[i] = quantise(self.tail)

    def row_scales(self):
        closed = self.n // self.blk * self.blk
        return np.concatenate([np.repeat(self.scale[:closed // self.blk], self.blk),
                               [scale_of(np.abs(r).max()) for r in self.tail[:self.n - closed]]])

    def values(self):
        closed = self.n // self.blk * self.blk
        with np.errstate(invalid="ignore"):
            q = self.q8[:closed].astype(np.float64) * np.repeat(
                self.scale[:closed // self.blk].astype(np.float64), self.blk)[:, None]
        return np.concatenate([q, self.tail[:self.n - closed].astype(np.float64)])

    def cut(self, idx):
        """The rows idx, in a cache of their own."""
        out = Cache(self.S, self.blk, self.D)
        x, sc, blk = self.values()[idx], self.row_scales()[idx], self.blk
        out.n = len(idx)
        for i in range(out.n // blk):
            rows = slice(i * blk, (i + 1) * blk)
            out.q8[rows], out.scale[i] = quantise(x[rows], np.float32(sc[rows].max()))
        closed = out.n // blk * blk
        out.tail[:out.n - closed] = x[closed:].astype(np.float32)
        return out


def rotate(x, cos, sin):
    """fp32 RoPE with each product and the sum rounded once."""
    return x * cos + R.rotate_half(x) * sin


def attend(q, K, V, len0, scale):
    """q [T][G][D] at slots len0 + t over K, V [n][D]: out [T][G][D], lse
    [T][G], weights [n]."""
    T, n = q.shape[0], len(K)
    s = np.einsum("tgd,sd->tgs", q.astype(np.float64), K) * scale
    late = np.arange(n)[None, :] > len0 + np.arange(T)[:, None]
    s[np.broadcast_to(late[:, None, :], s.shape)] = -np.inf
    m = s.max(-1, keepdims=True)
    e = np.exp(s - m)
    l = e.sum(-1, keepdims=True)
    p = e / l
    # a masked slot takes no part, whatever it holds
    out = np.stack([p[t, :, :len0 + t + 1] @ V[:len0 + t + 1] for t in range(T)])
    return out, (m + np.log(l))[..., 0], p.sum((0, 1))


def choose(w, n, keep, recent, sink):
    """Slots of the n held that stay, by weight w."""
    if n <= keep:
        return np.arange(n)
    score = np.asarray(w[:n], np.float64)          # argsort puts NaN last
    mid = np.arange(sink, n - recent)
    order = mid[np.argsort(-score[mid], kind="stable")][:keep - sink - recent]
    return np.sort(np.concatenate([np.arange(sink), order, np.arange(n - recent, n)])).astype(int)


def decode(cfg, W, prompt, forced, rope, blk, cut=None, slots=None):
    """Logits [len(forced)][vocab] of a decoder on the 8-bit cache, teacher
    forced.  cut(li, h, w, n) -> the slots to keep of layer li and kv head h,
    called when the cache of `slots` is full."""
    D, Hq, Hkv = cfg.head_dim, cfg.heads, cfg.kv_heads
    G, S = Hq // Hkv, slots or -(-cfg.max_seq // blk) * blk
    caches = [[(Cache(S, blk, D), Cache(S, blk, D)) for _ in range(Hkv)] for _ in W["layers"]]
    weights = [[np.zeros(S) for _ in range(Hkv)] for _ in W["layers"]]
    scale = 1.0 / np.sqrt(D)

    def block(ids, pos0):
        T = len(ids)
        x = W["embed"][ids].astype(np.float32)
        cos, sin = rope[0][pos0:pos0 + T, None], rope[1][pos0:pos0 + T, None]
        for li, L in enumerate(W["layers"]):
            h = R.rms_norm(x, L["ln"], cfg.eps)
            q = rotate((h @ L["q"]).reshape(T, Hq, D), cos, sin)
            k = rotate((h @ L["k"]).reshape(T, Hkv, D), cos, sin)
            v = (h @ L["v"]).reshape(T, Hkv, D)
            att = np.zeros((T, Hq, D))
            for i in range(Hkv):
                kc, vc = caches[li][i]
                n0 = kc.n
                kc.append(k[:, i])
                vc.append(v[:, i])
                att[:, i * G:(i + 1) * G], _, w = attend(q[:, i * G:(i + 1) * G], kc.values(),
                                                         vc.values(), n0, scale)
                acc = weights[li][i]
                acc[n0:kc.n] = 0
                acc[:kc.n] += w
            x = x + (att.reshape(T, Hq * D).astype(np.float32) @ L["o"])
            x = R._mlp_block(cfg, L, x)
        return R.rms_norm(x[-1:], W["final_ln"], cfg.eps) @ W["lm_head"]

    logits = [block([int(t) for t in prompt], 0)[0]]
    pos = len(prompt)
    for i in range(len(forced) - 1):
        if caches[0][0][0].n + 1 > S:
            for li in range(len(caches)):
                for h in range(Hkv):
                    idx = cut(li, h, weights[li][h], caches[li][h][0].n)
                    caches[li][h] = tuple(c.cut(idx) for c in caches[li][h])
                    weights[li][h][:len(idx)] = weights[li][h][idx]
        logits.append(block([int(forced[i])], pos)[0])
        pos += 1
    return np.stack(logits)
