"""The operators that make a long context smaller, as timed cases.

Five kinds, on a ``PagedKVCache`` of 8-bit pages (``kv_bits=8``) or of FP16
ones:

* ``append``   K/V rows written into the 8-bit cache and read back as the
  values it holds (``append_rows``, ``read_rows``);
* ``decode``   attention of one new token per sequence over the 8-bit cache;
* ``prefill``  causal attention of a prompt chunk over the 8-bit cache;
* ``weights``  the softmax weights that a step's last tokens give each cached
  row, summed per KV head onto decayed earlier ones (``attn_weights``);
* ``evict``    the rows of largest weight kept, per layer and KV head, in
  pages of another sequence (``evict``), and read back.

The 8-bit cache holds a full 16-row page of one KV head, K and V apart, as
codes c in [-127, 127] and a scale s; a value is c s.  s is the smallest
m 2^e with m in 8..15 and e >= -24 for which 127 s covers the page's largest
magnitude, at most 512, and c = x / s rounded to the nearest, ties to even.  A
sequence's last page stays in FP16 until its sixteenth row arrives.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 256
PAGE = 16


def _case(kind, seqs, ctx_lo, ctx_hi, new_lo=1, new_hi=1, layers=1, heads=24, kv_heads=4, bits=8, gate=False, obs=1,
          keep_lo=0, keep_hi=0, decay=1.0, ragged=0):
    """ctx: rows of a sequence before its new ones; evict keeps keep_lo..keep_hi of them."""
    return {"kind": kind, "seqs": seqs, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "new_lo": new_lo, "new_hi": new_hi,
            "layers": layers, "heads": heads, "kv_heads": kv_heads, "bits": bits, "gate": gate, "obs": obs,
            "keep_lo": keep_lo, "keep_hi": keep_hi, "decay": decay, "ragged": ragged}


def listed():
    return [
        # The new rows of a serving batch's decode step.
        dict(_case("append", 32, 100, 8000, ragged=1), name="append_b32"),
        # A restored or freshly prefilled prompt's rows.
        dict(_case("append", 4, 0, 100, 1500, 2048, ragged=2), name="append_4x2k"),
        # One user near the start of a conversation: launches and latency.
        dict(_case("decode", 1, 255, 255), name="decode_b1_256"),
        # The serving batch of the benchmark: 32 ragged contexts of 1k to 8k.
        dict(_case("decode", 32, 1024, 8192, gate=True, ragged=3), name="decode_b32_8k"),
        # Many long documents at once.
        dict(_case("decode", 48, 4096, 32768, ragged=4), name="decode_b48_32k"),
        # A short prompt into an empty cache.
        dict(_case("prefill", 1, 0, 0, 181, 181, gate=True), name="prefill_181"),
        # The chunks of four prompts at several depths.
        dict(_case("prefill", 4, 0, 2048, 512, 512, gate=True, ragged=5), name="prefill_4x512"),
        # A chunk late in a long prompt.
        dict(_case("prefill", 1, 16400, 16400, 2048, 2048), name="prefill_2k_at_16k"),
        # Weights followed during decode, step by step, for a batch.
        dict(_case("weights", 32, 1024, 8192, decay=0.9, ragged=6), name="weights_b32_8k"),
        # The last 32 tokens of prompts vote on what to keep of them.
        dict(_case("weights", 4, 3000, 16000, 32, 32, bits=16, obs=32, decay=0.0, ragged=7), name="weights_4x32_16k"),
        # One conversation cut to a third.
        dict(_case("evict", 1, 1500, 1500, layers=4, keep_lo=512, keep_hi=512), name="evict_1500_512"),
        # Long prompts cut before decoding starts.
        dict(_case("evict", 8, 4096, 16384, layers=4, bits=16, keep_lo=1024, keep_hi=2100, ragged=8),
             name="evict_8x16k_2k"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "weights", "weights", "evict"])
    heads, kv_heads = rng.choice([(24, 4), (24, 4), (12, 2), (6, 1), (16, 4), (8, 8), (8, 1), (6, 3)])
    ragged = rng.randrange(1, 1 << 20)
    more = {"heads": heads, "kv_heads": kv_heads, "ragged": ragged}
    if kind == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 8192 // seqs)
        hi = _log(rng, 1, min(8000, 200000 // seqs))
        return _case(kind, seqs, int(hi * rng.random()), hi, max(1, int(new * rng.uniform(0.3, 1.0))), new, **more)
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, min(32768, 850000 // seqs))
        return _case(kind, seqs, int(hi * rng.uniform(0.1, 1.0)), hi, gate=rng.random() < 0.5, **more)
    if kind == "prefill":
        seqs = rng.choice([1, 1, 2, 4, 7])
        new = _log(rng, 2, 2048 // seqs)
        hi = rng.choice([0, _log(rng, 1, 16000 // seqs)])
        return _case(kind, seqs, int(hi * rng.random()), hi, max(1, int(new * rng.uniform(0.5, 1.0))), new,
                     gate=rng.random() < 0.5, **more)
    if kind == "weights":
        obs = rng.choice([1, 1, _log(rng, 1, 32), 32])
        new = 1 if obs == 1 else rng.choice([obs, _log(rng, 1, 200)])
        seqs = _log(rng, 1, 32)
        hi = _log(rng, 1, min(16000, (150000 if obs == 1 else 40000) // seqs))
        return _case(kind, seqs, int(hi * rng.uniform(0.1, 1.0)), hi, max(1, int(new * rng.uniform(0.5, 1.0))), new,
                     bits=rng.choice([8, 16]), obs=obs, decay=rng.choice([0.0, 0.9, 1.0]), **more)
    seqs = _log(rng, 1, 16)
    hi = _log(rng, 24, min(16384, 80000 // seqs))
    lo = max(24, int(hi * rng.uniform(0.3, 1.0)))
    keep = _log(rng, 20, lo)
    return _case(kind, seqs, lo, hi, layers=rng.choice([1, 2, 4]), bits=rng.choice([8, 16]),
                 keep_lo=max(20, int(keep * rng.uniform(0.5, 1.0))), keep_hi=keep, **more)


#: Rows that an eviction never drops: the first ones and the latest.
FIRST, RECENT = 4, 16


class _Plan:
    """What a case's sizes come to: lengths, new rows, pages, and the places of everything."""

    def __init__(self, case):
        self.c = case
        self.kind, self.bits = case["kind"], case["bits"]
        self.L, self.H, self.KV, self.B = case["layers"], case["heads"], case["kv_heads"], case["seqs"]
        self.G = self.H // self.KV
        r = np.random.default_rng(case["ragged"])
        draw_ = lambda lo, hi: r.integers(lo, hi + 1, self.B).astype(np.int64)  # noqa: E731
        self.base = draw_(case["ctx_lo"], case["ctx_hi"])
        self.new = draw_(case["new_lo"], case["new_hi"]) if self.kind != "evict" else np.zeros(self.B, np.int64)
        self.keep = draw_(case["keep_lo"], case["keep_hi"])
        self.ctx = self.base + self.new
        self.T, self.R = int(self.new.sum()), int(self.ctx.sum())
        self.n_pages = -(-self.ctx // PAGE)
        self.pages, self.widest = int(self.n_pages.sum()), int(self.n_pages.max())
        self.width = self.widest * PAGE  # rows of a sequence, padded to the longest one's pages
        self.max_new = int(self.new.max())


def _put(x):
    return torch.as_tensor(x, device="cuda")


def _rows(p, seed):
    """Every sequence's K and V rows, [layer, row, KV, D] packed in sequence
    order: normalised keys with a few strong channels, values with heads of
    unlike size."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.empty(p.L, p.R, p.KV, D, dtype=torch.float16, device="cuda").normal_(generator=g)
    v = torch.empty_like(k).normal_(generator=g)
    strong = torch.ones(D, device="cuda")
    strong[torch.randperm(D, generator=g, device="cuda")[:6]] = 3.0
    size = torch.empty(p.KV, 1, device="cuda").uniform_(0.2, 2.0, generator=g)
    return k.mul_(strong.half()), v.mul_(size.half()), g


def _weights(p, g):
    """Weights gathered before: [seq, KV, row] of one layer, about a step's
    own in size, or for an eviction [layer, seq, KV, row], a few large ones
    over many small, with ties at zero (rows that no token looked at)."""
    if p.kind == "weights":
        w = torch.empty(p.B, p.KV, p.width, device="cuda").exponential_(generator=g)
        return w * (p.G * p.c["obs"] / p.width)
    w = torch.empty(p.L, p.B, p.KV, p.width, device="cuda").exponential_(generator=g) ** 3
    return w * (torch.rand(w.shape, device="cuda", generator=g) < 0.8)


class _State:
    pass


def prepare(case, seed):
    s = _State()
    p = s.p = _Plan(case)
    k, v, g = _rows(p, seed)
    half = lambda *shape: torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)  # noqa: E731
    s.k, s.v = k, v
    if p.kind in ("decode", "prefill", "weights"):
        s.q = half(p.T, p.H, D)
        s.gate = half(p.T, p.H, D) if case["gate"] else None
    if p.kind in ("weights", "evict"):
        s.w = _weights(p, g)
    order = np.random.default_rng(seed).permutation(p.pages).astype(np.int32)
    s.blocks = np.split(order, np.cumsum(p.n_pages)[:-1])
    at = np.concatenate([np.arange(b, c) + o for b, c, o in zip(p.base, p.ctx, np.cumsum(p.ctx) - p.ctx)])
    s.at = _put(at)  # the new rows among the packed ones
    s.lens = _put(p.ctx)
    s.row_seq = _put(np.repeat(np.arange(p.B), p.ctx))
    s.row_at = _put(np.concatenate([np.arange(c) for c in p.ctx]))
    if p.kind == "append":
        s.k_new, s.v_new = k[0, s.at].contiguous(), v[0, s.at].contiguous()
    if own:
        _own_cache(s)
    else:
        _plain_cache(s)
    torch.cuda.synchronize()
    return s


# ---- the framework's side ---------------------------------------------------

def _own_cache(s):
    """The cache that a user's program holds: the rows before the step in its
    pages, the step begun."""
    from mi50grad_amd.kv_cache import PagedKVCache

    p = s.p
    step = 32768
    extra = int((-(-p.keep // PAGE)).sum()) if p.kind == "evict" else 0
    slots = 2 * p.B if p.kind == "evict" else p.B
    s.cache = PagedKVCache(n_layers=p.L, max_seqs=slots, max_blocks=p.pages + extra, max_blocks_per_seq=p.widest,
                           max_step_tokens=max(step, p.T) + 16 * p.B, num_heads=p.H, num_kv_heads=p.KV, kv_bits=p.bits)
    s.seqs = list(range(p.B))
    for b, ids in enumerate(s.blocks):
        s.cache.set_blocks(b, ids)
    start = np.cumsum(p.ctx) - p.ctx
    done, goal = np.zeros(p.B, np.int64), p.ctx if p.kind != "append" else p.base
    if p.kind in ("decode", "prefill", "weights"):
        goal = p.base
    share = max(PAGE, step // p.B // PAGE * PAGE)
    while (done < goal).any():
        n = np.minimum(goal - done, share)
        rows = _put(np.concatenate([np.arange(d, d + m) + o for d, m, o in zip(done, n, start)]))
        s.cache.begin_step(s.seqs, n)
        for i in range(p.L):
            k, v = s.k[i, rows], s.v[i, rows]
            s.cache.append_rows(i, k.data_ptr(), v.data_ptr())
            torch.cuda.synchronize()  # before k and v go
        done += n
    if p.kind == "evict":
        s.first, s.second = s.seqs, [p.B + b for b in s.seqs]
        s.kept = torch.empty(p.L, p.B, p.KV, int(p.keep.max()), dtype=torch.int32, device="cuda")
        s.w_out = torch.empty_like(s.w)
        s.rows = int(p.keep.sum())
        s.zeros, s.keep = [0] * p.B, [int(x) for x in p.keep]
        s.out = [torch.empty(p.L, s.rows, p.KV, D, dtype=torch.float16, device="cuda") for _ in "kv"]
        return
    s.cache.begin_step(s.seqs, p.new)
    if p.kind == "append":
        s.out = [torch.empty_like(s.k_new), torch.empty_like(s.v_new)]
        s.base, s.new = [int(x) for x in p.base], [int(x) for x in p.new]
        return
    k, v = s.k[0, s.at], s.v[0, s.at]
    s.cache.append_rows(0, k.data_ptr(), v.data_ptr())
    torch.cuda.synchronize()  # before k and v go
    s.out = torch.empty_like(s.q)


def _own_run(s):
    p, cache = s.p, s.cache
    if p.kind == "append":
        cache.append_rows(0, s.k_new.data_ptr(), s.v_new.data_ptr())
        cache.read_rows(0, s.seqs, s.base, s.new, s.out[0].data_ptr(), s.out[1].data_ptr())
        return {"k": s.out[0], "v": s.out[1]}
    if p.kind in ("decode", "prefill"):
        call = cache.decode if p.kind == "decode" else cache.prefill
        call(0, s.q.data_ptr(), s.out.data_ptr(), gate=s.gate.data_ptr() if s.gate is not None else None)
        return {"out": s.out}
    if p.kind == "weights":
        w = s.w.clone()
        cache.attn_weights(0, s.q.data_ptr(), w.data_ptr(), p.width, n_obs=p.c["obs"], decay=p.c["decay"])
        return {"w": w}
    cache.evict(s.first, s.keep, s.w.data_ptr(), p.width, s.kept.data_ptr(), s.kept.shape[-1], first=FIRST,
                recent=RECENT, dst_ids=s.second, weights_out=s.w_out.data_ptr())
    for i in range(p.L):
        cache.read_rows(i, s.second, s.zeros, s.keep, s.out[0][i].data_ptr(), s.out[1][i].data_ptr())
    return {"kept": s.kept, "w": s.w_out, "k": s.out[0], "v": s.out[1]}


# ---- the plain forms ----------------------------------------------------------

def _scale(amax):
    """The 8-bit scale of a page whose largest magnitude is amax (in 64 bits:
    the border between two scales is where a quotient of small whole numbers lies)."""
    m, e = torch.frexp(amax.double() / 127.0)  # m in [1/2, 1)
    up = torch.ldexp(torch.ceil(m * 16.0) / 16.0, e)
    return up.clamp(2.0 ** -21, 512.0)


def _quantise(x):
    """x [..., row, D], whole pages: codes (as floats) and scale [..., 1, 1]."""
    s = _scale(x.abs().amax((-1, -2), keepdim=True)).float()
    return torch.clamp(torch.round(x.float() / s), -127, 127), s


def _paged(rows, blocks, p):
    """Packed rows [layer, R, KV, D] in a pool [layer, page, KV, 16, D], zeros
    behind a sequence's last one."""
    at = np.concatenate([ids[np.arange(c) // PAGE].astype(np.int64) * PAGE + np.arange(c) % PAGE
                         for ids, c in zip(blocks, p.ctx)])
    pool = torch.zeros(p.L, p.pages * PAGE, p.KV, D, dtype=torch.float16, device="cuda")
    pool[:, _put(at)] = rows
    return pool.view(p.L, p.pages, PAGE, p.KV, D).transpose(2, 3).contiguous()


def _plain_cache(s):
    """Pools of pages behind a block table: FP16, or codes with their scales
    and each sequence's last, open page in FP16."""
    p = s.p
    table = np.zeros((p.B, p.widest), np.int64)
    for b, ids in enumerate(s.blocks):
        table[b, :len(ids)] = ids
    s.table = _put(table)
    s.pools = [_paged(x, s.blocks, p) for x in (s.k, s.v)]
    if p.bits == 16:
        return
    s.open_at = (s.lens // PAGE).clamp(max=p.widest - 1)
    s.is_open = (s.lens % PAGE > 0)
    s.last = [x[:, s.table[torch.arange(p.B, device="cuda"), s.open_at]].contiguous() for x in s.pools]
    s.scales = []
    for i, x in enumerate(s.pools):
        codes = torch.empty(x.shape, dtype=torch.int8, device="cuda")
        scales = torch.empty(p.L, p.pages, p.KV, 1, 1, device="cuda")
        for j in range(0, p.pages, 4096):
            c, scales[:, j:j + 4096] = _quantise(x[:, j:j + 4096])
            codes[:, j:j + 4096] = c.to(torch.int8)
        s.pools[i] = codes
        s.scales.append(scales)


def _dense(s, which):
    """K (0) or V (1) of every sequence, [layer, seq, KV, row, D] in 32 bits, padded to the longest."""
    p = s.p
    x = s.pools[which][:, s.table].float()  # [layer, seq, page, KV, 16, D]
    if p.bits == 8:
        x *= s.scales[which][:, s.table]
        here = torch.arange(p.B, device="cuda")
        x[:, here, s.open_at] = torch.where(s.is_open[:, None, None, None], s.last[which].float(), x[:, here, s.open_at])
    return x.transpose(2, 3).reshape(p.L, p.B, p.KV, p.width, D)


def _padded(s, x):
    """Per-token rows [T, ...] as [seq, longest, ...], zeros behind a sequence's last."""
    p = s.p
    if not hasattr(s, "tok"):
        s.tok = _put(np.concatenate([np.arange(n) + b * p.max_new for b, n in enumerate(p.new)]))
    y = torch.zeros((p.B * p.max_new,) + x.shape[1:], dtype=x.dtype, device="cuda")
    y[s.tok] = x
    return y.view((p.B, p.max_new) + x.shape[1:])


def _probabilities(s, q, k):
    """Softmax over the rows that each new token sees: q [seq, token, H, D],
    k [seq, KV, row, D]; [seq, KV, token * G, row]."""
    p = s.p
    n = q.shape[1]
    q = q.float().view(p.B, n, p.KV, p.G, D).permute(0, 2, 1, 3, 4).reshape(p.B, p.KV, n * p.G, D)
    sc = torch.matmul(q / 16.0, k.transpose(-1, -2)).view(p.B, p.KV, n, p.G, p.width)
    # token i of a sequence sees rows up to its own
    own_row = _put(p.base)[:, None] + torch.arange(n, device="cuda")
    seen = torch.arange(p.width, device="cuda") <= own_row[..., None]
    sc.masked_fill_(~seen[:, None, :, None], float("-inf"))
    sc = torch.exp(sc - sc.amax(-1, keepdim=True))
    return (sc / sc.sum(-1, keepdim=True)).view(p.B, p.KV, n * p.G, p.width)


def _plain_append(s):
    """The new rows as the 8-bit cache holds them: pages that are full now in
    codes, the open page's rows as they came."""
    p = s.p
    got = []
    for new, pool in ((s.k_new, 0), (s.v_new, 1)):
        # The step's pages: rows from before it that share the first one, then the new rows.
        if not hasattr(s, "touched"):
            first = p.base // PAGE * PAGE
            n = -(-(p.ctx - first) // PAGE) * PAGE
            o = np.cumsum(n) - n
            s.touched = int(n.sum())
            s.old_to = _put(np.concatenate([np.arange(b - f) + i for b, f, i in zip(p.base, first, o)]).astype(np.int64))
            s.old_at = _put(np.concatenate([np.arange(f, b) + c for b, f, c in
                                            zip(p.base, first, np.cumsum(p.ctx) - p.ctx)]).astype(np.int64))
            s.new_to = _put(np.concatenate([np.arange(m) + b - f + i for m, b, f, i in zip(p.new, p.base, first, o)]))
            s.full = _put(np.concatenate([np.arange(m) // PAGE * PAGE + PAGE <= c - f
                                          for m, c, f in zip(n, p.ctx, first)]))
        x = torch.zeros(s.touched, p.KV, D, dtype=torch.float16, device="cuda")
        x[s.old_to] = (s.k, s.v)[pool][0, s.old_at]
        x[s.new_to] = new
        c, sc = _quantise(x.view(-1, PAGE, p.KV, D).transpose(1, 2))
        held = (c * sc).transpose(1, 2).reshape(s.touched, p.KV, D).half()
        got.append(torch.where(s.full[:, None, None], held, x)[s.new_to])
    return {"k": got[0], "v": got[1]}


def _plain_attention(s):
    p = s.p
    pr = _probabilities(s, _padded(s, s.q), _dense(s, 0)[0])
    out = torch.matmul(pr, _dense(s, 1)[0])
    out = out.view(p.B, p.KV, p.max_new, p.G, D).permute(0, 2, 1, 3, 4).reshape(p.B * p.max_new, p.H, D)[s.tok]
    if s.gate is not None:
        out = out * (1.0 / (1.0 + torch.exp(-s.gate.float())))
    return {"out": out.half()}


def _plain_weights(s):
    p = s.p
    pr = _probabilities(s, _padded(s, s.q), _dense(s, 0)[0]).view(p.B, p.KV, p.max_new, p.G, p.width)
    i = torch.arange(p.max_new, device="cuda")
    new = _put(p.new)[:, None]
    counts = (i < new) & (i >= new - p.c["obs"])
    got = torch.where(counts[:, None, :, None, None], pr, pr.new_zeros(())).sum((2, 3))
    if p.c["decay"]:
        got = got + p.c["decay"] * s.w
    return {"w": torch.where((torch.arange(p.width, device="cuda") < s.lens[:, None])[:, None], got, s.w)}


def _kept(p, w, lens):
    """Places of the rows that stay, ascending, -1 behind them: [layer, seq,
    KV, most]; rows of equal weight stay from the lowest place on."""
    at = torch.arange(p.width, device="cuda")
    keep, lens = _put(p.keep)[None, :, None, None], lens[None, :, None, None]
    held = (at < FIRST) | (at >= lens - RECENT)
    rank = torch.where(held, float("inf"), w)
    rank = torch.where(at < lens, rank, float("-inf"))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    stay = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, best, (at < keep).expand_as(rank))
    most = int(p.keep.max())
    order = torch.where(stay, at, p.width).sort(-1).values[..., :most]
    return torch.where(order < p.width, order, -1).to(torch.int32)


def _plain_evict(s):
    p = s.p
    kept = _kept(p, s.w, s.lens)
    most, at = kept.shape[-1], kept.clamp(min=0).long()
    w = torch.zeros_like(s.w)
    w[..., :most] = torch.where(kept >= 0, s.w.gather(-1, at), s.w.new_zeros(()))
    here = torch.arange(p.B, device="cuda")
    n = _put(p.keep)
    out = {"kept": kept, "w": w}
    full = -(-most // PAGE) * PAGE
    for name, which in (("k", 0), ("v", 1)):
        x = _dense(s, which).gather(3, at[..., None].expand(-1, -1, -1, -1, D))
        x = torch.where((kept >= 0)[..., None], x, x.new_zeros(()))
        if p.bits == 8:
            x = torch.nn.functional.pad(x, (0, 0, 0, full - most)).view(p.L, p.B, p.KV, full // PAGE, PAGE, D)
            c, sc = _quantise(x)
            shut = torch.arange(PAGE, full + 1, PAGE, device="cuda") <= n[:, None]  # [seq, page]
            x = torch.where(shut[None, :, None, :, None, None], c * sc, x).view(p.L, p.B, p.KV, full, D)[..., :most, :]
        valid = torch.arange(most, device="cuda") < n[here][:, None]
        out[name] = x.half().transpose(2, 3).reshape(p.L, p.B * most, p.KV, D)[:, valid.reshape(-1)]
    return out


def run(s):
    if own:
        return _own_run(s)
    kind = s.p.kind
    if kind == "append":
        return _plain_append(s)
    if kind == "weights":
        return _plain_weights(s)
    return _plain_evict(s) if kind == "evict" else _plain_attention(s)


# ---- the work, and the definition in 64 bits ------------------------------------

def work(case):
    p = _Plan(case)
    e = 1 if p.bits == 8 else 2
    scale = 4.0 / PAGE if p.bits == 8 else 0.0  # of one row of a head's K or V
    row = D * e + scale
    seen = float(np.sum(p.base * p.new + p.new * (p.new + 1) // 2))
    if p.kind == "append":
        return {"bytes": 2.0 * p.T * p.KV * (2 * D + row) + 2.0 * p.T * p.KV * (row + 2 * D), "flops": 0.0}
    if p.kind in ("decode", "prefill"):
        rows = (3 if case["gate"] else 2) * p.T * p.H * D * 2
        return {"bytes": 2.0 * p.R * p.KV * row + rows, "flops": 4.0 * p.H * D * seen}
    if p.kind == "weights":
        obs = np.minimum(p.new, case["obs"])
        seen = float(np.sum(obs * (p.ctx - obs) + obs * (obs + 1) // 2))
        w = (2 if case["decay"] else 1) * 4.0 * p.KV * p.R
        return {"bytes": p.R * p.KV * row + float(obs.sum()) * p.H * D * 2 + w, "flops": 2.0 * p.H * D * seen}
    kept = float(p.keep.sum()) * p.L * p.KV
    return {"bytes": 4.0 * p.L * p.KV * float(p.base.sum()) + kept * (4 + 2 * 4) + kept * 2 * (2 * row + row + 2 * D),
            "flops": 0.0}


def _page_values(x):
    """The 64-bit values that the 8-bit cache has for the FP16 rows x [rows,
    KV, D] of one sequence: whole pages rounded to their scales, the rest as it is."""
    n = x.shape[0] // PAGE * PAGE
    y = x[:n].double().view(-1, PAGE, x.shape[1], D)
    top = y.abs().amax((1, 3), keepdim=True).clamp(min=2.0 ** -30) / 127.0
    unit = torch.exp2(torch.floor(torch.log2(top)) - 3)  # a power of two (or twice it) below top / 8
    unit = torch.where(top / unit >= 16, unit * 2, unit)
    unit = torch.where(top / unit < 8, unit / 2, unit)
    step = (torch.ceil(top / unit) * unit).clamp(min=2.0 ** -21, max=512.0)
    y = torch.round(y / step).clamp(-127, 127) * step
    return torch.cat([y.view(n, x.shape[1], D), x[n:].double()])


def exact(case, seed):
    p = _Plan(case)
    k, v, g = _rows(p, seed)
    half = lambda *shape: torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)  # noqa: E731
    ends = np.cumsum(p.ctx)
    held = (lambda x: _page_values(x)) if p.bits == 8 else (lambda x: x.double())
    of = lambda x, i, b: held(x[i, ends[b] - p.ctx[b]:ends[b]])  # noqa: E731
    if p.kind == "append":
        return {n: torch.cat([of(x, 0, b)[p.base[b]:] for b in range(p.B)]) for n, x in (("k", k), ("v", v))}
    if p.kind == "evict":
        w = _weights(p, g)
        most = int(p.keep.max())
        kept = torch.full((p.L, p.B, p.KV, most), -1, dtype=torch.int32, device="cuda")
        w_out = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        rows = {"k": [], "v": []}
        for i in range(p.L):
            for b in range(p.B):
                n, m = int(p.ctx[b]), int(p.keep[b])
                places = []
                for h in range(p.KV):
                    wt = w[i, b, h, :n].double().cpu().numpy()
                    inner = np.arange(FIRST, n - RECENT)
                    inner = inner[np.lexsort((inner, -wt[inner]))][:max(0, m - FIRST - RECENT)]
                    at = np.sort(np.concatenate([np.arange(FIRST), inner, np.arange(n - RECENT, n)]))
                    kept[i, b, h, :m] = _put(at.astype(np.int32))
                    w_out[i, b, h, :m] = _put(wt[at])
                    places.append(_put(at))
                places = torch.stack(places, 1)
                for name, x in (("k", k), ("v", v)):
                    y = of(x, i, b).gather(0, places[..., None].expand(-1, -1, D))
                    rows[name].append(held(y))
        return {"kept": kept, "w": w_out, **{n: torch.cat(r).view(p.L, -1, p.KV, D) for n, r in rows.items()}}
    q = half(p.T, p.H, D).double()
    gate = half(p.T, p.H, D).double() if case["gate"] else None
    out = torch.empty_like(q)
    if p.kind == "weights":
        w = _weights(p, g).double()
    t = 0
    for b in range(p.B):
        n, c = int(p.new[b]), int(p.ctx[b])
        kb, vb = of(k, 0, b), of(v, 0, b) if p.kind != "weights" else None
        m = min(n, case["obs"]) if p.kind == "weights" else n  # the last m tokens are looked at
        qb = q[t + n - m:t + n]
        shut = torch.arange(c, device="cuda") > torch.arange(c - m, c, device="cuda")[:, None]
        if p.kind == "weights":
            w[b, :, :c] *= case["decay"]
        for h in range(p.H):
            j = h // p.G
            sc = qb[:, h].contiguous() @ kb[:, j].t().contiguous() / 16.0
            pr = torch.softmax(sc.masked_fill_(shut, float("-inf")), -1)
            if p.kind == "weights":
                w[b, j, :c] += pr.sum(0)
            else:
                out[t:t + n, h] = pr @ vb[:, j].contiguous()
        t += n
    if p.kind == "weights":
        return {"w": w}
    return {"out": out if gate is None else out * torch.sigmoid(gate)}
