"""GPU: attention weights gathered over both kinds of cache, and eviction by
them, against plain float64 forms."""
import numpy as np
import pytest

from cache8_helpers import D, held, make, put, rows, same_bits, within
from gpu_helpers import Tables, expected_norm, say
from mi50grad_amd._lib import KvaError
from oracle import kvattn_oracle as orc

pytestmark = pytest.mark.gpu
F32 = np.finfo(np.float32).eps / 2


def _values(bits, k, v):
    return orc.int8_rows(k, v) if bits == 8 else (k.astype(np.float64), v.astype(np.float64))


def _weights(q, k, ctx, m, G):
    """Sum of the softmax weights of the last m tokens of q [n, H, D] over k
    [ctx, kv, D]: [kv, ctx], and how far float32 may be off: a score's error (sum of
    256 products, scaled) counts twice, in the weight and in the row's sum."""
    kv = k.shape[1]
    out, tol = np.zeros((kv, ctx)), np.zeros((kv, ctx))
    q = q[len(q) - m:].astype(np.float64)
    see = np.arange(ctx)[None] <= ctx - m + np.arange(m)[:, None]
    for h in range(kv * G):
        s = q[:, h] @ k[:, h // G].T / 16.0
        size = (np.abs(q[:, h]) @ np.nan_to_num(np.abs(k[:, h // G])).T / 16.0).max() if m else 0.0
        s = np.where(see, s, -np.inf)
        with np.errstate(invalid="ignore"):
            p = np.exp(s - s.max(-1, keepdims=True))
        p = np.where(see, p / p.sum(-1, keepdims=True), 0.0)
        out[h // G] += p.sum(0)
        tol[h // G] += p.sum(0) * (2 * (D + 16) * F32 * size + 128 * F32)
    return out, tol + 1e-37


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("heads,kv", [(24, 4), (6, 1), (8, 8), (8, 1), (6, 3)])
@pytest.mark.parametrize("base,new,obs", [([0, 15, 300, 2100], [1, 1, 1, 1], 1), ([40, 0, 1000], [3, 40, 33], 32),
                                          ([17, 500], [20, 2], 5), ([5000], [1], 7), ([33, 64], [0, 9], 9)], ids=str)
def test_weights(device, bits, heads, kv, base, new, obs):
    say(f"weights {bits} {heads}/{kv} {base} {new} {obs}")
    rng = np.random.default_rng(heads + obs)
    lens = [b + n for b, n in zip(base, new)]
    cache = make(lens, heads=heads, kv=kv, bits=bits)
    seqs = list(range(len(lens)))
    data = [rows(rng, n, kv) for n in lens]
    put(device, cache, seqs, [d[0][:b] for d, b in zip(data, base)], [d[1][:b] for d, b in zip(data, base)])
    put(device, cache, seqs, [d[0][b:] for d, b in zip(data, base)], [d[1][b:] for d, b in zip(data, base)])
    q = (rng.standard_normal((max(1, sum(new)), heads, D)) * 1.5).astype(np.float16)
    width = max(lens) + 3
    for decay in (0.0, 0.75, 1.0):
        old = rng.exponential(size=(len(lens), kv, width)).astype(np.float32)
        old[0, 0, 0] = np.nan if decay == 0 else old[0, 0, 0]
        w = device.array(old)
        cache.attn_weights(0, device.array(q), w, width, n_obs=obs, decay=decay)
        device.synchronize()
        got, t = w.numpy().astype(np.float64), 0
        for b, (n, c) in enumerate(zip(new, lens)):
            want, tol = _weights(q[t:t + n], _values(bits, *data[b])[0], c, min(n, obs), heads // kv)
            if decay:
                before = decay * old[b, :, :c].astype(np.float64)
                want, tol = want + before, tol + 2 * F32 * (want + before)
            within(got[b, :, :c], want, tol + F32 * np.abs(want))
            assert np.array_equal(got[b, :, c:], old[b, :, c:].astype(np.float64)), "rows behind the sequence"
            t += n
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
def test_weights_of_rows_not_finite(device, bits):
    """A NaN key gives NaN to every row that the tokens which see it weigh."""
    say("weights nan")
    rng = np.random.default_rng(2)
    k, v = rows(rng, 70, 2)
    k[40, 0, 3] = np.nan
    cache = make([70], heads=2, kv=2, bits=bits)
    put(device, cache, [0], [k], [v])
    q = rng.standard_normal((70, 2, D)).astype(np.float16)
    w = device.array(np.zeros((1, 2, 70), np.float32))
    cache.attn_weights(0, device.array(q), w, 70, n_obs=4)
    device.synchronize()
    got = w.numpy()[0]
    assert np.isnan(got[0]).all()
    want, tol = _weights(q[:, 1:], _values(bits, k, v)[0][:, 1:], 70, 4, 1)
    within(got[1:], want, tol + F32 * want)
    cache.destroy()


def _not_finite(q, k, ctx, m, G):
    """_weights with scores that are not finite: q [n, H, D], k [ctx, kv, D] in
    float64.  The tolerance's score size is that of the finite ones."""
    kv = k.shape[1]
    out, tol = np.zeros((kv, ctx)), np.zeros((kv, ctx))
    q = q[len(q) - m:].astype(np.float64)
    see = np.arange(ctx)[None] <= ctx - m + np.arange(m)[:, None]
    finite = lambda x: np.where(np.isfinite(x), np.abs(x), 0.0)  # noqa: E731
    with np.errstate(invalid="ignore"):
        for h in range(kv * G):
            s = np.where(see, q[:, h] @ k[:, h // G].T / 16.0, -np.inf)
            size = (finite(q[:, h]) @ finite(k[:, h // G]).T / 16.0).max()
            p = np.exp(s - s.max(-1, keepdims=True))
            p = np.where(see, p / p.sum(-1, keepdims=True), 0.0)
            out[h // G] += p.sum(0)
            tol[h // G] += np.nan_to_num(p).sum(0) * (2 * (D + 16) * F32 * size + 128 * F32)
    return out, tol + 1e-37


@pytest.mark.parametrize("obs", [1, 3, 5, 32])
@pytest.mark.parametrize("heads,kv", [(24, 4), (6, 2)])
@pytest.mark.parametrize("what", ["lowest and highest", "query", "all lowest"])
def test_weights_of_infinite_scores(device, what, heads, kv, obs):
    """A score of -inf is a score: where its row's sum is NaN (a score of +inf
    elsewhere, or none but -inf), so is its weight.  Rows that a token does not
    see get nothing of it."""
    say(f"infinite scores: {what} {heads}/{kv} {obs}")
    rng = np.random.default_rng(obs + heads)
    for bits in (16, 8) if what == "query" else (16,):
        n = 333
        k, v = rows(rng, n, kv)
        q = rng.standard_normal((obs, heads, D)).astype(np.float16)
        if what == "query":  # a token's every score: infinite, of both signs
            q[0, ::2, 7] = np.inf
        elif what == "all lowest":
            q[0, :, 7] = np.abs(q[0, :, 7]) + np.float16(0.5)
            q[1:, :, 7] = -np.abs(q[1:, :, 7]) - np.float16(0.5)
            k[:, 0, 7] = -np.inf
        else:  # a score of -inf for every query row of a head, and one of +inf that only the last token sees
            q[:, :, 7] = np.abs(q[:, :, 7]) + np.float16(0.5)
            k[100, 0, 7] = -np.inf
            k[n - 1, 0, 7] = np.inf
        cache = make([n], heads=heads, kv=kv, bits=bits)
        put(device, cache, [0], [k[:n - obs]], [v[:n - obs]])
        put(device, cache, [0], [k[n - obs:]], [v[n - obs:]])
        w = device.array(np.full((1, kv, n), 3.0, np.float32))
        cache.attn_weights(0, device.array(q), w, n, n_obs=obs, decay=0.0)
        device.synchronize()
        want, tol = _not_finite(q, _values(bits, k, v)[0], n, obs, heads // kv)
        within(w.numpy()[0], want, tol + F32 * np.abs(want))
        cache.destroy()


@pytest.mark.parametrize("obs", [1, 3, 5, 32])
@pytest.mark.parametrize("heads,kv", [(24, 4), (6, 2), (6, 1)])
def test_weights_of_a_key_that_no_token_weighs(device, heads, kv, obs):
    """A key with scores of -inf only weighs nothing, also where the token and
    head pairs do not fill the tiles of 16 that they are multiplied in."""
    say(f"a key of -inf {heads}/{kv} {obs}")
    rng = np.random.default_rng(obs + heads)
    n = 333
    k, v = rows(rng, n, kv)
    q = rng.standard_normal((obs, heads, D)).astype(np.float16)
    q[:, :, 7] = np.abs(q[:, :, 7]) + np.float16(0.5)
    k[[100, 301], :, 7] = -np.inf
    cache = make([n], heads=heads, kv=kv, bits=16)
    put(device, cache, [0], [k[:n - obs]], [v[:n - obs]])
    put(device, cache, [0], [k[n - obs:]], [v[n - obs:]])
    w = device.array(np.full((1, kv, n), 3.0, np.float32))
    cache.attn_weights(0, device.array(q), w, n, n_obs=obs, decay=0.0)
    device.synchronize()
    want, tol = _not_finite(q, k.astype(np.float64), n, obs, heads // kv)
    assert (want[:, [100, 301]] == 0).all()
    within(w.numpy()[0], want, tol + F32 * want)
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
def test_weights_without_rows(device, bits):
    """Sequences without rows, and without new ones, beside others and alone."""
    say(f"weights without rows {bits}")
    rng = np.random.default_rng(5)
    k, v = rows(rng, 40, 2)
    cache = make([40, 16, 16], heads=4, kv=2, bits=bits)
    q = device.array(rng.standard_normal((40, 4, D)).astype(np.float16))
    old = rng.exponential(size=(3, 2, 48)).astype(np.float32)
    w = device.array(old)
    cache.begin_step([1, 2], [0, 0])
    cache.attn_weights(0, q, w, 48, decay=0.5)
    device.synchronize()
    assert np.array_equal(w.numpy(), old)
    cache.begin_step([1, 0, 2], [0, 40, 0])
    cache.append_rows(0, device.array(k), device.array(v))
    cache.attn_weights(0, q, w, 48, n_obs=3, decay=0.5)
    device.synchronize()
    got = w.numpy()
    assert np.array_equal(got[[0, 2]], old[[0, 2]]) and np.array_equal(got[1, :, 40:], old[1, :, 40:])
    want, tol = _weights(q.numpy()[:40], _values(bits, k, v)[0], 40, 3, 2)
    want = want + 0.5 * old[1, :, :40].astype(np.float64)
    within(got[1, :, :40], want, tol + 3 * F32 * want)
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
def test_weights_whose_scores_do_not_fit(device, bits):
    """One tile of query rows over so many pages that K is read twice: the same
    8192 rows over and over, so each of their weights is the same in every turn."""
    say(f"weights of many pages {bits}")
    rng = np.random.default_rng(6)
    kv, each, turns, obs = 8, 8192, 34, 16
    n = each * turns + obs
    cache = make([n], heads=kv, kv=kv, bits=bits, step=each)
    k, v = rows(rng, each, kv)
    last = rows(rng, obs, kv)
    dk, dv = device.array(k), device.array(v)
    for _ in range(turns):
        cache.begin_step([0], [each])
        cache.append_rows(0, dk, dv)
    put(device, cache, [0], [last[0]], [last[1]])
    q = rng.standard_normal((obs, kv, D)).astype(np.float16)
    w = device.array(np.zeros((1, kv, n), np.float32))
    cache.attn_weights(0, device.array(q), w, n, n_obs=obs, decay=0.0)
    device.synchronize()
    got = w.numpy()[0].astype(np.float64)
    kd, kl = _values(bits, k, v)[0], _values(bits, *last)[0]
    see = np.arange(obs)[None] <= np.arange(obs)[:, None]
    for h in range(kv):
        x = q[:, h].astype(np.float64)
        s, sl = x @ kd[:, h].T / 16.0, np.where(see, x @ kl[:, h].T / 16.0, -np.inf)
        m = np.maximum(s.max(-1), sl.max(-1))[:, None]
        p, pl = np.exp(s - m), np.exp(sl - m)
        total = turns * p.sum(-1, keepdims=True) + pl.sum(-1, keepdims=True)
        want = np.concatenate([np.tile((p / total).sum(0), turns), (pl / total).sum(0)])
        size = (np.abs(x) @ np.abs(kd[:, h]).T / 16.0).max()
        # as in _weights; a lane's running sum takes n / 1024 terms at most here
        within(got[h], want, want * (2 * (D + 16) * F32 * size + 512 * F32) + 1e-37)
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
def test_more_sequences_than_lanes(device, bits):
    """150 sequences, some without rows: weights, eviction in place and as copies
    (their sizes go to the kernels 64 at a time), reading and decode."""
    say(f"150 sequences {bits}")
    rng = np.random.default_rng(10)
    B, H, kv, keep, first, recent = 150, 4, 2, 24, 2, 8
    lens = [int(x) for x in rng.integers(1, 70, B)]
    for b in (0, 63, 64, 149):
        lens[b] = 16 * (b % 3 + 1)
    cache = make(lens, heads=H, kv=kv, bits=bits, spare=400, slots=2 * B, extra=16)
    data = [rows(rng, n + 1, kv) for n in lens]
    seqs = [int(x) for x in rng.permutation(B)]
    put(device, cache, list(range(B)), [d[0][:-1] for d in data], [d[1][:-1] for d in data])
    put(device, cache, seqs, [data[s][0][-1:] for s in seqs], [data[s][1][-1:] for s in seqs])
    q = rng.standard_normal((B, H, D)).astype(np.float16)
    out, w = device.empty(q.shape, np.float16), device.array(np.zeros((1, B, kv, 80), np.float32))
    cache.decode(0, device.array(q), out)
    cache.attn_weights(0, device.array(q), w, 80, decay=0.0)
    device.synchronize()
    vals = [_values(bits, *d) for d in data]
    got = w.numpy()
    for i, s in enumerate(seqs):
        want, tol = _weights(q[i:i + 1], vals[s][0], lens[s] + 1, 1, H // kv)
        within(got[0, i, :, :lens[s] + 1], want, tol + F32 * want)
        within(out.numpy()[i:i + 1], *orc.attention_bound(q[i:i + 1], *vals[s]))
    for split in (32, 2048, 16384):  # shares of two pages, of some forty sequences, of all
        cache.set_decode_split(split)
        cache.decode(0, device.array(q), out)
        device.synchronize()
        for i, s in enumerate(seqs):
            within(out.numpy()[i:i + 1], *orc.attention_bound(q[i:i + 1], *vals[s]))
    dst = [s if i % 2 else B + i for i, s in enumerate(seqs)]
    kept = device.empty((1, B, kv, keep), np.int32)
    cache.evict(seqs, [keep] * B, w, 80, kept, keep, first=first, recent=recent, dst_ids=dst)
    have, o = held(device, cache, dst), 0
    for i, s in enumerate(seqs):
        n = lens[s] + 1
        m = min(n, keep)
        places = [_stay(got[0, i, h], n, keep, first, recent) for h in range(kv)]
        assert all(np.array_equal(kept.numpy()[0, i, h][:m], places[h]) for h in range(kv)), i
        want = vals[s] if dst[i] == s and m == n else _moved(bits, data[s], places)
        assert same_bits(have[0][o:o + m], want[0]) and same_bits(have[1][o:o + m], want[1]), i
        o += m
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n_short", [62, 70, 150])
def test_weights_of_a_long_sequence_among_short_ones(device, n_short, bits):
    """About as many sequences as workgroups run at once (64 of 192 query rows
    each per KV head) and more, one of them long: in several chunks, and right."""
    say(f"one long sequence, {n_short} short, {bits}")
    rng = np.random.default_rng(n_short + bits)
    H, kv, obs = 24, 4, 32
    lens = [int(x) for x in rng.integers(1, 60, n_short)]
    lens.insert(n_short // 2, 2500)
    new = [min(n, obs) for n in lens]
    cache = make(lens, heads=H, kv=kv, bits=bits)
    seqs = list(range(len(lens)))
    data = [rows(rng, n, kv) for n in lens]
    put(device, cache, seqs, [d[0][:len(d[0]) - n] for d, n in zip(data, new)],
        [d[1][:len(d[1]) - n] for d, n in zip(data, new)])
    put(device, cache, seqs, [d[0][len(d[0]) - n:] for d, n in zip(data, new)],
        [d[1][len(d[1]) - n:] for d, n in zip(data, new)])
    q = rng.standard_normal((sum(new), H, D)).astype(np.float16)
    old = rng.exponential(size=(len(lens), kv, 2500)).astype(np.float32)
    w = device.array(old)
    cache.attn_weights(0, device.array(q), w, 2500, n_obs=obs, decay=0.5)
    device.synchronize()
    assert cache.weights_plan()[0] < 40, "pages of the long sequence's 157 in one chunk"
    got, t = w.numpy().astype(np.float64), 0
    for b, (n, c) in enumerate(zip(new, lens)):
        want, tol = _weights(q[t:t + n], _values(bits, *data[b])[0], c, n, H // kv)
        before = 0.5 * old[b, :, :c].astype(np.float64)
        within(got[b, :, :c], want + before, tol + F32 * (2 * (want + before) + want))
        assert np.array_equal(got[b, :, c:], old[b, :, c:].astype(np.float64))
        t += n
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
def test_two_caches_on_two_streams(device, bits):
    """The same work on two caches at once, each on a stream of its own, gives
    what it gives alone."""
    from mi50grad_amd.device import Stream

    say(f"two caches {bits}")
    rng = np.random.default_rng(11)
    H, kv, lens, keep = 12, 2, [700, 129, 2000], [256, 100, 512]
    data = [rows(rng, n, kv) for n in lens]
    q = device.array(rng.standard_normal((3, H, D)).astype(np.float16))
    hold = [device.array(np.concatenate([d[j][:-1] for d in data])) for j in (0, 1)]
    tail = [device.array(np.concatenate([d[j][-1:] for d in data])) for j in (0, 1)]

    def work(cache, stream, out, w, kept):
        cache.begin_step([0, 1, 2], [n - 1 for n in lens], stream=stream)
        cache.append_rows(0, *hold, stream=stream)
        cache.begin_step([0, 1, 2], [1] * 3, stream=stream)
        cache.append_rows(0, *tail, stream=stream)
        for _ in range(4):
            cache.decode(0, q, out, stream=stream)
            cache.attn_weights(0, q, w, 2048, decay=0.5, stream=stream)
        cache.evict([0, 1, 2], keep, w, 2048, kept, 512, first=4, recent=16, stream=stream)

    streams = [Stream(), Stream()]
    caches = [make(lens, heads=H, kv=kv, bits=bits, spare=60) for _ in range(3)]
    outs = [[device.empty((3, H, D), np.float16), device.array(np.ones((1, 3, kv, 2048), np.float32)),
             device.array(np.full((1, 3, kv, 512), 7, np.int32))] for _ in range(3)]
    device.synchronize()
    work(caches[2], None, *outs[2])
    device.synchronize()
    for c, s, o in zip(caches, streams, outs):
        work(c, s.handle, *o)
    for s in streams:
        s.synchronize()
    want = held(device, caches[2], [0, 1, 2])
    for c, o in zip(caches[:2], outs):
        assert all(np.array_equal(x.numpy(), y.numpy()) for x, y in zip(o, outs[2]))
        got = held(device, c, [0, 1, 2])
        assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    for c in caches:
        c.destroy()
    for s in streams:
        s.destroy()


def test_weights_repeat_to_the_bit(device):
    say("weights repeat")
    rng = np.random.default_rng(3)
    lens = [900, 33, 2000]
    cache = make(lens)
    data = [rows(rng, n, 4) for n in lens]
    put(device, cache, [0, 1, 2], [d[0] for d in data], [d[1] for d in data])
    q = device.array(rng.standard_normal((sum(lens), 24, D)).astype(np.float16))
    got = []
    for _ in range(3):
        w = device.array(np.ones((3, 4, 2000), np.float32))
        cache.attn_weights(0, q, w, 2000, n_obs=32)
        device.synchronize()
        got.append(w.numpy())
    assert all(np.array_equal(g.view(np.uint32), got[0].view(np.uint32)) for g in got)
    cache.destroy()


def _stay(w, n, keep, first, recent):
    if keep >= n:
        return np.arange(n)
    w = np.where(np.isnan(w), -np.inf, w[...])[:n].astype(np.float64)
    inner = np.arange(first, n - recent)
    inner = inner[np.lexsort((inner, -w[inner]))][:keep - first - recent]
    return np.sort(np.concatenate([np.arange(first), inner, np.arange(n - recent, n)])).astype(int)


KINDS = {
    "spread": lambda r, n: r.exponential(size=n) ** 3,
    "ties": lambda r, n: r.integers(0, 4, n) * 0.25,
    "all_equal": lambda r, n: np.full(n, 0.5),
    "any_sign": lambda r, n: np.where(r.random(n) < 0.1, r.choice([0.0, -0.0, np.inf, -np.inf, np.nan], n), r.standard_normal(n)),
    "near": lambda r, n: 1 + r.integers(0, 50, n) * 2.0 ** -23,
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,keep,first,recent", [(1, 1, 0, 0), (1, 0, 0, 0), (40, 20, 4, 16), (40, 21, 4, 16),
                                                 (1000, 500, 0, 0), (1000, 999, 3, 0), (2000, 77, 0, 32),
                                                 (5000, 5000, 4, 16), (33, 100, 4, 16), (33000, 9000, 4, 64)], ids=str)
def test_which_rows_stay(device, kind, n, keep, first, recent):
    say(f"which stay {kind} {n} {keep}")
    rng = np.random.default_rng(n + keep)
    cache = make([n], heads=1, kv=1, bits=16, step=max(16, n), spare=min(n, keep) // 16 + 1, slots=2)
    put(device, cache, [0], [np.zeros((n, 1, D), np.float16)], [np.zeros((n, 1, D), np.float16)])
    width, most = n + 5, min(n, keep) + 3
    w = np.zeros((1, 1, 1, width), np.float32)
    w[..., :n] = KINDS[kind](rng, n)
    w[..., n:] = 1e30  # behind the sequence: never looked at
    kept = device.array(np.full((1, 1, 1, most), 99, np.int32))
    out = device.array(np.full(w.shape, 99, np.float32))
    cache.evict([0], [keep], device.array(w), width, kept, most, first=first, recent=recent, dst_ids=[1],
                weights_out=out)
    device.synchronize()
    want = _stay(w[0, 0, 0], n, keep, first, recent)
    got = kept.numpy()[0, 0, 0]
    assert np.array_equal(got[:len(want)], want) and (got[len(want):] == -1).all()
    back = out.numpy()[0, 0, 0]
    assert np.array_equal(back[:len(want)].view(np.uint32), w[0, 0, 0][want].view(np.uint32))
    assert (back[len(want):] == 0).all()
    assert cache.seq_len(1) == len(want) and cache.seq_len(0) == n
    cache.destroy()


def _filled(device, lens, heads, kv, layers, bits, rng, **kw):
    cache = make(lens, heads=heads, kv=kv, layers=layers, bits=bits, **kw)
    data = [[rows(rng, n, kv) for n in lens] for _ in range(layers)]
    for i in range(layers):
        put(device, cache, list(range(len(lens))), [d[0] for d in data[i]], [d[1] for d in data[i]], layer=i)
    return cache, data


def _moved(bits, d, places):
    """Rows d = (k, v) of a sequence, of each head those at places[h]."""
    got = [np.stack([x[places[h], h] for h in range(x.shape[1])], 1) for x in _values(bits, *d)]
    return _values(bits, got[0], got[1]) if bits == 8 else got


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("where", ["copy", "in_place", "in_place_tight", "mixed"])
def test_evict(device, bits, where):
    say(f"evict {bits} {where}")
    rng = np.random.default_rng(7)
    lens, keep, first, recent = [100, 17, 333, 64, 5], [37, 20, 128, 16, 5], 2, 9
    keep = [k if k >= first + recent or k >= n else first + recent for k, n in zip(keep, lens)]
    kv, heads, layers, B = 3, 6, 2, len(lens)
    # tight: room for the largest sequence's new blocks only
    spare = 8 if where == "in_place_tight" else 30
    cache, data = _filled(device, lens, heads, kv, layers, bits, rng, spare=spare, slots=2 * B)
    free = cache.free_block_count()
    dst = {"copy": [B + b for b in range(B)], "mixed": [0, B + 1, B + 2, 3, 4]}.get(where)
    w = rng.exponential(size=(layers, B, kv, max(lens))).astype(np.float32)
    kept = device.empty((layers, B, kv, max(keep)), np.int32)
    out = device.empty(w.shape, np.float32)
    before = [held(device, cache, list(range(B)), layer=i) for i in range(layers)]
    cache.evict(list(range(B)), keep, device.array(w), max(lens), kept, max(keep), first=first, recent=recent,
                dst_ids=dst, weights_out=out)
    device.synchronize()
    to = dst or list(range(B))
    m = [min(k, n) for k, n in zip(keep, lens)]
    assert [cache.seq_len(s) for s in to] == m
    for i in range(layers):
        got, o = held(device, cache, to, layer=i), 0
        for b in range(B):
            places = [_stay(w[i, b, h], lens[b], keep[b], first, recent) for h in range(kv)]
            assert all(np.array_equal(kept.numpy()[i, b, h][:m[b]], places[h]) for h in range(kv))
            same = to[b] == b and m[b] == lens[b]  # left as it is
            want = _values(bits, *data[i][b]) if same else _moved(bits, data[i][b], places)
            assert same_bits(got[0][o:o + m[b]], want[0]) and same_bits(got[1][o:o + m[b]], want[1]), (i, b)
            o += m[b]
        if where == "copy":
            now = held(device, cache, list(range(B)), layer=i)
            assert same_bits(now[0], before[i][0]) and same_bits(now[1], before[i][1]), "the sources stay"
    blocks = lambda ns: sum((n + 15) // 16 for n in ns)  # noqa: E731
    gone = sum((lens[b] + 15) // 16 for b in range(B) if to[b] == b)
    assert cache.free_block_count() == free + gone - blocks(m)
    # the copies again, over themselves: their own blocks come back first
    if where == "copy":
        cache.evict(list(range(B)), keep, device.array(w), max(lens), kept, max(keep), first=first, recent=recent,
                    dst_ids=dst)
        device.synchronize()
        assert cache.free_block_count() == free - blocks(m)
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("turn", [1, -1])
def test_evict_from_a_full_pool_in_any_order(device, bits, turn):
    """Two free blocks: sequences that need four, three and two of them, and a copy
    over a sequence that holds more than it gets, listed in either order."""
    say(f"evict from a full pool {bits} {turn}")
    rng = np.random.default_rng(18)
    lens, kv, heads, layers = [120, 100, 90, 50, 64], 2, 4, 2
    cache, data = _filled(device, lens, heads, kv, layers, bits, rng, spare=2)
    assert cache.free_block_count() == 2
    jobs = [(0, 0, 60), (1, 1, 40), (2, 2, 25), (3, 4, 20)][::turn]
    src, dst, keep = (list(x) for x in zip(*jobs))
    width, first, recent = max(lens), 3, 8
    w = rng.exponential(size=(layers, len(jobs), kv, width)).astype(np.float32)
    kept = device.empty((layers, len(jobs), kv, max(keep)), np.int32)
    cache.evict(src, keep, device.array(w), width, kept, max(keep), first=first, recent=recent, dst_ids=dst)
    device.synchronize()
    for i in range(layers):
        got, o = held(device, cache, dst, layer=i), 0
        for j, (s, _, m) in enumerate(jobs):
            places = [_stay(w[i, j, h], lens[s], m, first, recent) for h in range(kv)]
            want = _moved(bits, data[i][s], places)
            assert same_bits(got[0][o:o + m], want[0]) and same_bits(got[1][o:o + m], want[1]), (i, s)
            o += m
        stayed, want = held(device, cache, [3], layer=i), _values(bits, *data[i][3])
        assert same_bits(stayed[0], want[0]) and same_bits(stayed[1], want[1]), "a copy's source stays"
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 16])
def test_evict_then_go_on(device, bits):
    """A prompt, the weights its last tokens give, eviction in place, then decode
    steps at their true positions, with the weights followed: every output and
    every weight against float64 over what the cache holds, and a second eviction."""
    say(f"evict then go on {bits}")
    rng = np.random.default_rng(8)
    H, kv, layers, B = 6, 2, 2, 3
    lens, keep, first, recent = [200, 90, 47], [64, 50, 40], 4, 16
    tables = Tables(device, 512)
    ws = [device.array((1 + 0.02 * rng.standard_normal(D)).astype(np.float16)) for _ in range(2)]
    cache = make(lens, heads=H, kv=kv, layers=layers, bits=bits, extra=64, spare=16)
    width = 256
    w = device.array(np.full((layers, B, kv, width), np.nan, np.float32))  # decay 0 starts them
    w2 = device.empty((layers, B, kv, width), np.float32)
    T = sum(lens)
    cache.begin_step([0, 1, 2], lens)
    for i in range(layers):
        q = device.array(rng.standard_normal((T, H, D)).astype(np.float16))
        k, v = rows(rng, T, kv)
        cache.append(i, q, device.array(k), device.array(v), *ws, tables.d_cos, tables.d_sin, 512)
        cache.prefill(i, q, device.empty((T, H, D), np.float16))
        at = w.ptr + i * B * kv * width * 4
        cache.attn_weights(i, q, at, width, n_obs=16, decay=0.0)
        device.synchronize()
        qn, mine, t = q.numpy(), w.numpy()[i], 0
        hk, _ = held(device, cache, [0, 1, 2], layer=i)
        for b, n in enumerate(lens):
            want, tol = _weights(qn[t:t + n], hk[t:t + n].astype(np.float64), n, 16, H // kv)
            within(mine[b, :, :n], want, tol + F32 * want)
            t += n
    kept = device.empty((layers, B, kv, max(keep)), np.int32)
    pos = list(lens)
    for turn in range(2):
        n_before = [cache.seq_len(b) for b in range(B)]
        old = w.numpy()
        before = [held(device, cache, [0, 1, 2], layer=i) for i in range(layers)]
        cache.evict([0, 1, 2], keep, w, width, kept, max(keep), first=first, recent=recent, weights_out=w2)
        device.synchronize()
        for i in range(layers):
            got, o, p = held(device, cache, [0, 1, 2], layer=i), 0, 0
            for b in range(B):
                m = min(keep[b], n_before[b])
                places = [_stay(old[i, b, h], n_before[b], keep[b], first, recent) for h in range(kv)]
                rows_ = [np.stack([x[o:o + n_before[b]][places[h], h] for h in range(kv)], 1) for x in before[i]]
                want = _values(bits, *rows_)
                assert same_bits(got[0][p:p + m], want[0]) and same_bits(got[1][p:p + m], want[1]), (turn, i, b)
                o, p = o + n_before[b], p + m
        w, w2 = w2, w
        for step in range(18):
            cache.begin_step([0, 1, 2], [1, 1, 1], rope_pos=pos)
            for i in range(layers):
                q = rng.standard_normal((B, H, D)).astype(np.float16)
                k, v = rows(rng, B, kv)
                dq, out = device.array(q), device.empty((B, H, D), np.float16)
                cache.append_decode(i, dq, device.array(k), device.array(v), *ws, tables.d_cos, tables.d_sin, 512, out)
                at = w.ptr + i * B * kv * width * 4
                was = w.numpy()[i].astype(np.float64)
                cache.attn_weights(i, dq, at, width, decay=0.9)
                device.synchronize()
                now = w.numpy()[i].astype(np.float64)
                assert np.array_equal(dq.numpy().view(np.uint16),
                                      expected_norm(q, ws[0].numpy(), tables, pos).view(np.uint16))
                if step not in (0, 1, 15, 17):
                    continue
                n = [cache.seq_len(b) for b in range(B)]
                hk, hv = held(device, cache, [0, 1, 2], layer=i)
                o = 0
                for b in range(B):
                    kb, vb = hk[o:o + n[b]].astype(np.float64), hv[o:o + n[b]].astype(np.float64)
                    qb = dq.numpy()[b:b + 1]
                    within(out.numpy()[b:b + 1], *orc.attention_bound(qb, kb, vb))
                    want, tol = _weights(qb, kb, n[b], 1, H // kv)
                    more = 0.9 * was[b, :, :n[b]]
                    within(now[b, :, :n[b]], want + more, tol + 4 * F32 * (want + more))
                    o += n[b]
            pos = [p + 1 for p in pos]
    cache.destroy()


def test_evict_refuses(device):
    say("evict refuses")
    rng = np.random.default_rng(9)
    cache, _ = _filled(device, [100, 50], 2, 1, 1, 8, rng)  # no spare block
    w = device.array(np.zeros((1, 2, 1, 100), np.float32))
    kept = device.empty((1, 2, 1, 40), np.int32)
    with pytest.raises(KvaError) as e:
        cache.evict([0, 1], [40, 40], w, 100, kept, 40)
    assert e.value.code == -4 and cache.seq_len(0) == 100 and cache.free_block_count() == 0
    before = held(device, cache, [0, 1])
    cache.evict([0, 1], [100, 50], device.array(np.zeros((1, 2, 1, 100), np.float32)), 100,
                device.empty((1, 2, 1, 100), np.int32), 100)  # nothing moves: no block needed
    after = held(device, cache, [0, 1])
    assert same_bits(before[0], after[0]) and same_bits(before[1], after[1])
    with pytest.raises(KvaError):
        cache.evict([0], [40], w, 100, w, 40)  # kept over weights
    cache.destroy()
