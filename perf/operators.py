"""The serving operators around the 8-bit key/value cache, and what a pass of each one does.

Four paths, named by a case's "op":

  append    rotary embedding of new tokens, and their keys and values taken into a cache that
            holds a full block of tokens as int8 with one scale for each block and head, and
            the block that is still open in fp32; then the blocks that it touched, read back
  attend    causal grouped-query attention of new tokens over that cache, with the log of each
            softmax sum and, on request, the attention weight that each slot has received
  evict     the slots with the most accumulated weight (and the first and the last ones) kept,
            in order, in another cache; then that cache, read back
  logprobs  of a row of logits: the log probability and the rank of a given token, the entropy,
            and the top alternatives

With `own` false, `run` computes a pass with elementary torch operations in fp32; with `own`
true, with the framework's operators.
"""
import math

import torch

own = False

TINY_AMAX = 127.0 * 2.0 ** -126   # a block of smaller values is held as zero


# -- cases --------------------------------------------------------------------
def listed():
    return [
        # One sequence, one token: the latency of a decode step's append.
        dict(name="append_one", op="append", batch=1, tokens=1, old_lo=37, old_hi=37, new_lo=1,
             heads=32, kv_heads=4, dim=64, cap=64, block=32),
        # A batch of prompts of different lengths, some with an earlier part in the cache.
        dict(name="append_prompts", op="append", batch=16, tokens=1000, old_lo=0, old_hi=531,
             new_lo=117, heads=32, kv_heads=4, dim=64, cap=1536, block=32),
        # One token over the decoder's default window of 64 slots.
        dict(name="attend_one_short", op="attend", batch=1, tokens=1, old_lo=45, old_hi=45,
             new_lo=1, heads=32, kv_heads=4, dim=64, cap=64, block=32, weights=False),
        # A full decode batch over uneven histories, weights gathered for a later eviction.
        dict(name="attend_batch", op="attend", batch=64, tokens=1, old_lo=611, old_hi=4095,
             new_lo=1, heads=32, kv_heads=4, dim=64, cap=4096, block=32, weights=True),
        # One sequence with a very long history, wide heads.
        dict(name="attend_one_long", op="attend", batch=1, tokens=1, old_lo=131007, old_hi=131007,
             new_lo=1, heads=32, kv_heads=8, dim=128, cap=131072, block=64, weights=False),
        # A few drafted tokens a sequence, verified together.
        dict(name="attend_draft", op="attend", batch=16, tokens=5, old_lo=300, old_hi=1500,
             new_lo=3, heads=32, kv_heads=4, dim=64, cap=1536, block=32, weights=True),
        # Prompts of uneven lengths behind a cached part of uneven lengths.
        dict(name="attend_prompts", op="attend", batch=4, tokens=1024, old_lo=0, old_hi=1000,
             new_lo=777, heads=32, kv_heads=4, dim=64, cap=2048, block=32, weights=True),
        # One sequence's window cut to half.
        dict(name="evict_one", op="evict", batch=1, old_lo=512, old_hi=512, kv_heads=4, dim=64,
             cap=512, keep=256, recent=64, sink=4, block=32),
        # A decode batch whose caches have filled up.
        dict(name="evict_batch", op="evict", batch=64, old_lo=1500, old_hi=4096, kv_heads=4,
             dim=64, cap=4096, keep=2048, recent=512, sink=4, block=32),
        # One answer's token.
        dict(name="logprobs_one", op="logprobs", rows=1, cols=32000, top=5),
        # A decode batch's tokens.
        dict(name="logprobs_batch", op="logprobs", rows=64, cols=32000, top=20),
        # Every token of a batch of prompts scored.
        dict(name="logprobs_prompts", op="logprobs", rows=4096, cols=32000, top=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cache_shape(rng):
    kv = rng.choice([1, 2, 4, 8])
    return dict(kv_heads=kv, heads=kv * rng.choice([1, 4, 7, 8]), dim=rng.choice([64, 64, 128]),
                block=rng.choice([16, 32, 64]))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "logprobs"])
    if op == "logprobs":
        cols = _log_int(rng, 1000, 200000)
        return dict(op=op, rows=_log_int(rng, 1, max(1, 40000000 // cols)), cols=cols,
                    top=rng.choice([1, 3, 5, 20]))
    c = dict(op=op, **_cache_shape(rng))
    per_slot = c["kv_heads"] * c["dim"]
    if op == "evict":
        cap = _log_int(rng, 8, 8192)
        cap = -(-cap // c["block"]) * c["block"]
        keep = rng.randint(1, cap)
        recent = rng.randint(0, keep)
        del c["heads"]
        return dict(c, batch=_log_int(rng, 1, max(1, 40000000 // (cap * per_slot))), cap=cap,
                    keep=keep, recent=recent, sink=rng.randint(0, min(4, keep - recent)),
                    old_lo=rng.randint(0, cap), old_hi=cap)
    kind = rng.choice(["step", "draft", "prompt"])
    tokens = {"step": 1, "draft": rng.randint(2, 8), "prompt": _log_int(rng, 9, 1024)}[kind]
    old = _log_int(rng, 1, 1024 if kind == "prompt" else 16384)
    cap = -(-(old + tokens) // c["block"]) * c["block"]
    room = 40000000 // (cap * per_slot)
    if kind == "prompt":
        room = min(room, 100000000 // (cap * tokens * c["heads"]))
    c = dict(c, batch=_log_int(rng, 1, max(1, min(64, room))), tokens=tokens,
             old_lo=rng.randint(0, old), old_hi=old, new_lo=rng.randint(1, tokens), cap=cap)
    return dict(c, weights=rng.random() < 0.5) if op == "attend" else c


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, both taken where n allows, in no order."""
    return [hi] if n == 1 else [lo + (hi - lo) * ((i * 37 + 11) % n) // (n - 1) for i in range(n)]


def _lengths(c):
    """(tokens in the cache, new tokens) of each sequence."""
    old = _spread(c["batch"], c["old_lo"], c["old_hi"])
    if c["op"] == "evict":
        return old, [0] * c["batch"]
    return old, _spread(c["batch"], c["new_lo"], c["tokens"])[::-1]


def work(c):
    if c["op"] == "logprobs":
        n = c["rows"] * c["cols"]
        return {"bytes": 4 * n + c["rows"] * (16 + 8 * c["top"]), "flops": 6 * n}
    old, new = _lengths(c)
    h, d, blk = c["kv_heads"], c["dim"], c["block"]

    def held(n):   # bytes of the keys and values of n slots
        closed = n // blk
        return h * (closed * (2 * blk * d + 8) + (n - closed * blk) * 8 * d)

    if c["op"] == "evict":
        kept = [min(n, c["keep"]) for n in old]
        rows = sum(kept)
        # every score, the kept rows in and out, their slots and scores, and the rows read back
        return {"bytes": 4 * h * sum(old) + 2 * sum(held(n) for n in kept) + 8 * h * rows
                + sum(held(n) for n in kept) + 8 * h * d * c["batch"] * c["keep"],
                "flops": 4 * h * d * rows}
    rows = sum(new)
    if c["op"] == "append":
        touched = [o + n - o // blk * blk for o, n in zip(old, new)]
        return {"bytes": 4 * rows * (2 * c["heads"] + 2 * h) * d
                + 2 * sum(held(n) for n in touched)
                + 8 * h * d * c["batch"] * _window(c),
                "flops": rows * (c["heads"] + 3 * h) * 3 * d}
    seen = sum(n * o + n * (n + 1) // 2 for o, n in zip(old, new))
    b = sum(held(o + n) for o, n in zip(old, new)) + 8 * rows * c["heads"] * d
    b += 4 * rows * c["heads"]
    if c["weights"]:
        b += 8 * h * sum(o + n for o, n in zip(old, new))
    return {"bytes": b, "flops": 4 * d * c["heads"] * seen}


def _window(c):
    """Slots that an append may touch, from the start of the open block on."""
    return -(-(c["tokens"] + c["block"] - 1) // c["block"]) * c["block"]


# -- inputs -------------------------------------------------------------------
def _scale(amax):
    """The scale of a block (or of a row on its own) whose largest magnitude is amax."""
    amax = torch.where(amax < TINY_AMAX, torch.zeros_like(amax), amax)
    return amax / torch.full_like(amax, 127.0)   # by a tensor: rounded as a division is


def _to_blocks(x, blk):
    """fp32 [B][H][S][D] -> int8 values [B][H][S][D] and scales [B][H][S/blk]."""
    b, h, s, d = x.shape
    x = x.view(b, h, s // blk, blk, d)
    amax = x.abs().amax((3, 4))
    scale = _scale(amax)
    # in 64 bits: a quotient next to a half has to fall on its own side
    step = torch.where(scale > 0, scale, math.inf).double()
    q = torch.round(x.double() / step[..., None, None]).to(torch.int8)
    return q.view(b, h, s, d), scale


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed((seed * 1000003 + 17) % 2 ** 63)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = {"case": c}
    if c["op"] == "logprobs":
        rows, cols = c["rows"], c["cols"]
        # a model's logits: a broad floor, and a handful of likely tokens
        x = normal(rows, cols, std=2.0)
        at = torch.randint(0, cols, (rows, 40), generator=gen, device="cuda")
        x.scatter_add_(1, at, 4.0 + 3.0 * torch.randn(at.shape, generator=gen, device="cuda"))
        s["logits"] = x
        likely = torch.rand(rows, generator=gen, device="cuda") < 0.7
        s["ids"] = torch.where(likely, x.argmax(1),
                               torch.randint(0, cols, (rows,), generator=gen, device="cuda")).int()
        s["out"] = dict(logprobs=torch.zeros(rows, device="cuda"),
                        entropy=torch.zeros(rows, device="cuda"),
                        rank=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                        top_ids=torch.zeros(rows, c["top"], dtype=torch.int32, device="cuda"),
                        top_logprobs=torch.zeros(rows, c["top"], device="cuda"))
        return _handle(s)
    b, h, d, cap, blk = c["batch"], c["kv_heads"], c["dim"], c["cap"], c["block"]
    old, new = _lengths(c)
    s["lens"], s["new"] = ints(old), ints(new)
    # keys have a few wide channels, as a model's do; what lies behind a
    # sequence's end is left from an earlier one
    wide = torch.where(torch.rand(h, 1, d, generator=gen, device="cuda") < 0.06, 3.0, 1.0)
    s["k"], s["ks"] = _to_blocks(normal(b, h, cap, d) * wide, blk)
    s["v"], s["vs"] = _to_blocks(normal(b, h, cap, d), blk)
    s["kt"], s["vt"] = normal(b, h, blk, d) * wide, normal(b, h, blk, d)
    if c["op"] == "append":
        t, hq = c["tokens"], c["heads"]
        s["qkv"] = normal(b * t, (hq + 2 * h) * d)
        s["pos"] = s["lens"].clone()
        freq = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        ang = torch.arange(cap, dtype=torch.float64, device="cuda")[:, None] * freq
        ang = torch.cat([ang, ang], 1)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["start"] = s["lens"] // blk * blk
        s["kt0"], s["vt0"] = s["kt"].clone(), s["vt"].clone()
        s["q"] = torch.zeros(b * t, hq, d, device="cuda")
        s["k_read"] = torch.zeros(b, h, _window(c), d, device="cuda")
        s["v_read"] = torch.zeros_like(s["k_read"])
    elif c["op"] == "attend":
        t, hq = c["tokens"], c["heads"]
        s["q"] = normal(b * t, hq, d, std=1.3)
        s["out"] = torch.zeros(b * t, hq, d, device="cuda")
        s["lse"] = torch.zeros(b * t, hq, device="cuda")
        if c["weights"]:
            s["w0"] = torch.rand(b, h, cap, generator=gen, device="cuda")
            s["w"] = s["w0"].clone()
    else:
        keep = c["keep"]
        # a few slots get most of the attention
        s["w"] = normal(b, h, cap, std=2.0).exp()
        cap2 = -(-keep // blk) * blk
        s["cap2"] = cap2
        s["lens2"] = torch.clamp(s["lens"], max=keep)
        s["k2"] = torch.zeros(b, h, cap2, d, dtype=torch.int8, device="cuda")
        s["v2"] = torch.zeros_like(s["k2"])
        s["ks2"] = torch.zeros(b, h, cap2 // blk, device="cuda")
        s["vs2"] = torch.zeros_like(s["ks2"])
        s["kt2"], s["vt2"] = torch.zeros_like(s["kt"]), torch.zeros_like(s["vt"])
        s["w2"] = torch.zeros(b, h, cap2, device="cuda")
        s["idx"] = torch.zeros(b, h, keep, dtype=torch.int32, device="cuda")
        s["k_read"] = torch.zeros(b, h, keep, d, device="cuda")
        s["v_read"] = torch.zeros_like(s["k_read"])
    return _handle(s)


def _handle(s):
    """What a program that uses the framework keeps: its graph, and the buffers as it names them."""
    if own:
        import numpy as np
        from spirv_inference_b200.graph import DeviceTensor, Graph, Kv8Cache
        c = s["case"]
        g = s["graph"] = Graph(0)
        types = {torch.float32: np.float32, torch.int32: np.int32, torch.int8: np.int8}

        def dev(x):
            return DeviceTensor(x.data_ptr(), tuple(x.shape), np.dtype(types[x.dtype]), g)

        s["dev"] = {n: dev(x) for n, x in s.items() if isinstance(x, torch.Tensor)}
        if c["op"] == "logprobs":
            s["dev"].update({n: dev(x) for n, x in s["out"].items()})
        else:
            t = s["dev"]
            s["cache"] = Kv8Cache(t["k"], t["v"], t["ks"], t["vs"], t["kt"], t["vt"], t["lens"],
                                  block=c["block"])
            if c["op"] == "evict":
                s["cache2"] = Kv8Cache(t["k2"], t["v2"], t["ks2"], t["vs2"], t["kt2"], t["vt2"],
                                       t["lens2"], block=c["block"])
    return s


# -- one pass -----------------------------------------------------------------
def run(s):
    return {"append": _append, "attend": _attend, "evict": _evict,
            "logprobs": _logprobs}[s["case"]["op"]](s)


def _append(s):
    c = s["case"]
    b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    cap, blk, n = c["cap"], c["block"], _window(c)
    if own:
        g, v = s["graph"], s["dev"]
        if t > 1:   # the open block as the call before left it
            g.copy_d2d(v["kt"], v["kt0"].ptr, v["kt"].nbytes)
            g.copy_d2d(v["vt"], v["vt0"].ptr, v["vt"].nbytes)
        g.rope_kv8_append(v["qkv"], (hq + 2 * h) * d, v["cos"], v["sin"], v["pos"], v["q"],
                          s["cache"], q_len=t, q_heads=hq, new_lens=v["new"])
        g.kv8_read(s["cache"], v["k_read"], v["v_read"], count=n, starts=v["start"], q_len=t,
                   new_lens=v["new"])
        return [s["q"], s["k_read"], s["v_read"]]
    lens, new = s["lens"].long(), s["new"].long()
    step = torch.arange(t, device="cuda")
    ok = step[None] < new[:, None]                                        # [B][T]
    x = s["qkv"].view(b, t, hq + 2 * h, d)
    at = (s["pos"].long()[:, None] + step).clamp(max=cap - 1)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    r = x[:, :, :hq + h]
    turned = torch.cat([-r[..., d // 2:], r[..., :d // 2]], -1)
    r = r * cos + turned * sin
    q = torch.where(ok[..., None, None], r[:, :, :hq], 0.0).reshape(b * t, hq, d)
    # the window of slots from the open block's first on: what the open block
    # holds, then the new tokens
    at_w = torch.arange(n, device="cuda")
    before = lens % blk
    total = (before + new).clamp(max=n)
    src = (at_w[None] - before[:, None]).clamp(0, t - 1)                  # [B][n]
    read = []
    for fresh, tail, out8, outs in ((r[:, :, hq:], s["kt0"], s["k"], s["ks"]),
                                    (x[:, :, hq + h:], s["vt0"], s["v"], s["vs"])):
        fresh = torch.take_along_dim(fresh.transpose(1, 2), src[:, None, :, None], 2)
        held = torch.nn.functional.pad(tail, (0, 0, 0, n - blk))
        w = torch.where((at_w[None] < before[:, None])[:, None, :, None], held, fresh)
        w = torch.where((at_w[None] < total[:, None])[:, None, :, None], w, 0.0)
        q8, sc = _to_blocks(w, blk)
        full = (at_w[::blk] + blk)[None] <= total[:, None]                # [B][n/blk]
        slot = (s["start"].long()[:, None] + at_w)
        hit = full.repeat_interleave(blk, 1) & (slot < cap)
        bi, wi = hit.nonzero(as_tuple=True)
        out8[bi, :, slot[bi, wi]] = q8.transpose(1, 2)[bi, wi]
        bj, wj = full.nonzero(as_tuple=True)
        outs[bj, :, slot[bj, wj * blk] // blk] = sc.transpose(1, 2)[bj, wj]
        values = q8.float() * sc.repeat_interleave(blk, 2)[..., None]
        read.append(torch.where(full.repeat_interleave(blk, 1)[:, None, :, None], values, w))
    return [q, *read]


def _values(s, x8, xs, tail, lens):
    """A cache's slots as fp32 [B][H][S][D]; `lens` the tokens of each sequence."""
    c = s["case"]
    b, h, cap, d = x8.shape
    blk = c["block"]
    x = x8.to(xs.dtype).view(b, h, cap // blk, blk, d) * xs[..., None, None]
    x = x.view(b, h, cap, d)
    j = torch.arange(cap, device="cuda")
    is_open = (j // blk)[None] == (lens // blk)[:, None]
    return torch.where(is_open[:, None, :, None], tail[:, :, j % blk], x)


def _attend(s):
    c = s["case"]
    b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    scale = d ** -0.5
    if own:
        g, v = s["graph"], s["dev"]
        if not c["weights"]:
            g.attention_kv8(v["q"], s["cache"], v["out"], q_len=t, q_heads=hq, scale=scale,
                            new_lens=v["new"], lse=v["lse"])
            return [s["out"], s["lse"]]
        g.copy_d2d(v["w"], v["w0"].ptr, v["w"].nbytes)
        g.attention_kv8(v["q"], s["cache"], v["out"], q_len=t, q_heads=hq, scale=scale,
                        new_lens=v["new"], lse=v["lse"], weights=v["w"])
        return [s["out"], s["lse"], s["w"]]
    lens, new = s["lens"].long(), s["new"].long()
    total = lens + new
    k = _values(s, s["k"], s["ks"], s["kt"], total)
    v = _values(s, s["v"], s["vs"], s["vt"], total)
    j, step = torch.arange(c["cap"], device="cuda"), torch.arange(t, device="cuda")
    ok = step[None] < new[:, None]                                        # [B][T]
    seen = j[None, None] <= (lens[:, None] + step)[..., None]             # [B][T][S]
    g = hq // h
    q = s["q"].view(b, t, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * g, d)
    x = (q @ k.transpose(2, 3)).mul_(scale).view(b, h, t, g, c["cap"])
    x.masked_fill_(~seen[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    p = p.div_(l)
    out = (p.view(b, h, t * g, c["cap"]) @ v).view(b, h, t, g, d)
    out = torch.where(ok[:, None, :, None, None], out, 0.0)
    lse = torch.where(ok[:, None, :, None], (m + l.log())[..., 0], 0.0)
    out = out.permute(0, 2, 1, 3, 4).reshape(b * t, hq, d)
    lse = lse.permute(0, 2, 1, 3).reshape(b * t, hq)
    if not c["weights"]:
        return [out, lse]
    got = torch.where(ok[:, None, :, None, None], p, 0.0).sum((2, 3))
    had = torch.where((j[None] < lens[:, None])[:, None], s["w0"], 0.0)
    return [out, lse, torch.where((j[None] < total[:, None])[:, None], had + got, s["w0"])]


def _evict(s):
    c = s["case"]
    b, h, d, cap, blk, keep = (c[n] for n in ("batch", "kv_heads", "dim", "cap", "block", "keep"))
    if own:
        g, v = s["graph"], s["dev"]
        g.kv8_evict(s["cache"], v["w"], keep, recent=c["recent"], sink=c["sink"], idx=v["idx"],
                    into=s["cache2"], into_weights=v["w2"])
        g.kv8_read(s["cache2"], v["k_read"], v["v_read"], count=keep)
        return [s["idx"], s["w2"], s["k_read"], s["v_read"]]
    lens = s["lens"].long()
    j = torch.arange(cap, device="cuda")
    n = lens.clamp(max=keep)                                              # kept
    safe = (j[None] < c["sink"]) | (j[None] >= lens[:, None] - c["recent"])
    score = torch.where(safe[:, None], math.inf, s["w"])
    score = torch.where((j[None] < lens[:, None])[:, None], score, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    i = torch.arange(keep, device="cuda")
    there = (i[None] < n[:, None])[:, None]                               # [B][1][keep]
    idx = torch.where(there, best, cap).sort(-1).values
    src = idx.clamp(max=cap - 1)
    closed = lens // blk * blk
    from_tail = src >= closed[:, None, None]
    full = (i[None] // blk * blk + blk) <= n[:, None]                     # [B][keep]
    pad = -keep % blk
    read = []
    for x8, xs, tail in ((s["k"], s["ks"], s["kt"]), (s["v"], s["vs"], s["vt"])):
        ts = _scale(tail.abs().amax(-1))
        x = _values(s, x8, xs.double(), tail.double(), lens)
        x = torch.take_along_dim(x, src[..., None], 2)
        sc = torch.where(from_tail, torch.take_along_dim(ts, src % blk, 2),
                         torch.take_along_dim(xs, src // blk, 2))
        sc = torch.nn.functional.pad(torch.where(there, sc, 0.0), (0, pad))
        sc = sc.view(b, h, -1, blk).amax(-1)
        sc = sc.repeat_interleave(blk, 2)[..., :keep, None]
        q8 = torch.round(x / torch.where(sc > 0, sc, math.inf).double())
        x = torch.where(full[:, None, :, None], q8.float() * sc, x.float())
        read.append(torch.where(there[..., None], x, 0.0))
    w = torch.where(there, torch.take_along_dim(s["w"], src, 2), 0.0)
    w = torch.nn.functional.pad(w, (0, s["cap2"] - keep))
    return [torch.where(there, idx, -1).int(), w, *read]


def _logprobs(s):
    c = s["case"]
    if own:
        v = s["dev"]
        s["graph"].token_logprobs(v["logits"], c["cols"], c["rows"], c["cols"], v["ids"],
                                  v["logprobs"], entropy=v["entropy"], rank=v["rank"],
                                  top_k=c["top"], top_ids=v["top_ids"],
                                  top_logprobs=v["top_logprobs"])
        return s["out"]
    x = s["logits"]
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    l = e.sum(1, keepdim=True)
    entropy = l.log()[:, 0] - (e * (x - m)).sum(1) / l[:, 0]
    one = torch.take_along_dim(x, s["ids"].long()[:, None], 1)
    rank = 1 + (x > one).sum(1)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    top = best[:, :c["top"]]
    return dict(logprobs=(one - m - l.log())[:, 0], entropy=entropy, rank=rank.int(),
                top_ids=at[:, :c["top"]].int(), top_logprobs=top - m - l.log())


# -- the same from the definitions, in 64 bits ----------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict,
            "logprobs": _exact_logprobs}[c["op"]](c, s)


def _held64(q8, scale, tail, n, blk):
    """The first n slots of one sequence, [H][n][D]."""
    closed = n // blk * blk
    part = q8[:, :closed].double() * scale[:, :closed // blk].double().repeat_interleave(blk, 1)[
        ..., None]
    return torch.cat([part, tail[:, :n - closed].double()], 1)


def _block64(x):
    """What a full block [H][blk][D] reads back as; its scale is held in fp32."""
    step = (x.abs().amax((1, 2), keepdim=True) / 127.0).float().double()
    return torch.where(step > 0, torch.round(x / step.clamp(min=1e-300)) * step, 0.0)


def _exact_append(c, s):
    b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    blk, n = c["block"], _window(c)
    old, new = _lengths(c)
    q = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    k = torch.zeros(b, h, n, d, dtype=torch.float64, device="cuda")
    v = torch.zeros_like(k)
    x = s["qkv"].view(b, t, hq + 2 * h, d).double()
    half = d // 2

    def held(v):   # a rotated value and its two products are each rounded to fp32, as defined
        return v.float().double()

    for i in range(b):
        cos = s["cos"][old[i]:old[i] + new[i]].double()[:, None]
        sin = s["sin"][old[i]:old[i] + new[i]].double()[:, None]
        y = x[i, :new[i]]
        lo, hi = y[:, :hq + h, :half], y[:, :hq + h, half:]
        y[:, :hq + h] = torch.cat(
            [held(held(lo * cos[..., :half]) - held(hi * sin[..., :half])),
             held(held(hi * cos[..., half:]) + held(lo * sin[..., half:]))], -1)
        q[i, :new[i]] = y[:, :hq]
        began = old[i] % blk
        for out, tail, fresh in ((k, s["kt0"], y[:, hq:hq + h]), (v, s["vt0"], y[:, hq + h:])):
            row = torch.cat([tail[i, :, :began].double(), fresh.transpose(0, 1)], 1)
            for at in range(0, row.shape[1] // blk * blk, blk):
                row[:, at:at + blk] = _block64(row[:, at:at + blk])
            out[i, :, :row.shape[1]] = row
    return [q.view(b * t, hq, d), k, v]


def _exact_attend(c, s):
    b, t, hq, h, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    blk, g = c["block"], c["heads"] // c["kv_heads"]
    old, new = _lengths(c)
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(b, t, hq, dtype=torch.float64, device="cuda")
    w = s["w0"].double() if c["weights"] else None
    for i in range(b):
        n = old[i] + new[i]
        k = _held64(s["k"][i], s["ks"][i], s["kt"][i], n, blk)
        v = _held64(s["v"][i], s["vs"][i], s["vt"][i], n, blk)
        q = s["q"].view(b, t, h, g, d)[i, :new[i]].double()
        x = torch.einsum("thgd,hsd->thgs", q, k) / math.sqrt(d)
        late = torch.arange(n, device="cuda")[None] > (
            old[i] + torch.arange(new[i], device="cuda"))[:, None]
        x.masked_fill_(late[:, None, None], -math.inf)
        z = torch.logsumexp(x, -1, keepdim=True)
        p = (x - z).exp()
        out[i, :new[i]] = torch.einsum("thgs,hsd->thgd", p, v).reshape(new[i], hq, d)
        lse[i, :new[i]] = z[..., 0].reshape(new[i], hq)
        if w is not None:
            w[i, :, old[i]:n] = 0
            w[i, :, :n] += p.sum((0, 2))
    got = [out.view(b * t, hq, d), lse.view(b * t, hq)]
    return got if w is None else got + [w]


def _exact_evict(c, s):
    b, h, d, blk, keep = (c[n] for n in ("batch", "kv_heads", "dim", "block", "keep"))
    old, _ = _lengths(c)
    if b * h * keep > 600000:
        return None
    w2 = torch.zeros(b, h, s["cap2"], dtype=torch.float64, device="cuda")
    read = [torch.zeros(b, h, keep, d, dtype=torch.float64, device="cuda") for _ in range(2)]
    for i in range(b):
        n = old[i]
        score = s["w"][i, :, :n].double()
        score[:, :c["sink"]] = math.inf
        score[:, max(0, n - c["recent"]):] = math.inf
        at = torch.argsort(score, dim=-1, descending=True, stable=True)
        at = at[:, :keep].sort(-1).values                                 # [H][m]
        m = at.shape[1]
        w2[i, :, :m] = s["w"][i].double().gather(1, at)
        for out, x8, xs, tail in ((read[0], s["k"], s["ks"], s["kt"]),
                                  (read[1], s["v"], s["vs"], s["vt"])):
            x = _held64(x8[i], xs[i], tail[i], n, blk).gather(1, at[..., None].expand(h, m, d))
            steps = torch.cat([xs[i, :, :n // blk].double().repeat_interleave(blk, 1),
                               (tail[i, :, :n % blk].double().abs().amax(-1) / 127.0).float().double()], 1)
            steps = steps.gather(1, at)
            for a in range(0, m // blk * blk, blk):
                step = steps[:, a:a + blk].amax(1)[:, None, None]
                x[:, a:a + blk] = torch.where(
                    step > 0, torch.round(x[:, a:a + blk] / step.clamp(min=1e-300)) * step, 0.0)
            out[i, :, :m] = x
    return [None, w2, *read]


def _exact_logprobs(c, s):
    if c["rows"] * c["cols"] > 150000000:
        return None
    x = s["logits"].double()
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    top = lp.topk(c["top"], 1).values
    return dict(logprobs=lp.gather(1, s["ids"].long()[:, None])[:, 0],
                entropy=-(lp.exp() * lp).sum(1), rank=None, top_ids=None, top_logprobs=top)
