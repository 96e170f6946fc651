"""GPU: the 8-bit cache.  What it holds is compared value for value with the
oracle's 8-bit rows; attention over it with float64 attention over those values,
within the bound of its roundings (attention_bound)."""
import numpy as np
import pytest

from cache8_helpers import D, held, make, put, rows, same_bits, within
from gpu_helpers import Tables, expected_norm, say
from oracle import kvattn_oracle as orc

pytestmark = pytest.mark.gpu


def _steps(n, how):
    """Row counts of the steps that bring n rows."""
    if how == "one":
        return [n]
    if how == "single":
        return [1] * n
    rng, out = np.random.default_rng(n), []
    while sum(out) < n:
        out.append(min(int(rng.integers(0, 40)), n - sum(out)))
    return out


@pytest.mark.parametrize("how", ["one", "single", "mixed"])
@pytest.mark.parametrize("kv", [1, 4])
def test_rows_held(device, kv, how):
    say(f"rows_held kv {kv} {how}")
    rng = np.random.default_rng(kv)
    lens = [1, 15, 16, 17, 31, 50, 64]
    cache = make(lens, heads=kv, kv=kv)
    data = [rows(rng, n, kv) for n in lens]
    plan = [_steps(n, how) for n in lens]
    done = [0] * len(lens)
    for i in range(max(len(p) for p in plan)):
        take = [p[i] if i < len(p) else 0 for p in plan]
        put(device, cache, list(range(len(lens))), [d[0][o:o + t] for d, o, t in zip(data, done, take)],
            [d[1][o:o + t] for d, o, t in zip(data, done, take)])
        done = [o + t for o, t in zip(done, take)]
    got = held(device, cache, list(range(len(lens))))
    want = [orc.int8_rows(*d) for d in data]
    assert same_bits(got[0], np.concatenate([w[0] for w in want]))
    assert same_bits(got[1], np.concatenate([w[1] for w in want]))
    # part of the rows, sequences out of order and twice
    got = held(device, cache, [5, 3, 5], [3, 16, 20], [40, 1, 0])
    assert same_bits(got[0], np.concatenate([want[5][0][3:43], want[3][0][16:17]]))
    assert same_bits(got[1], np.concatenate([want[5][1][3:43], want[3][1][16:17]]))
    cache.destroy()


def test_rows_that_close_the_open_page_and_open_another(device):
    """A sequence's open block is read for the page that closes and written for
    the page that is open then, in one step, for many sequences and heads at once."""
    say("close and open")
    rng = np.random.default_rng(14)
    kv, B = 8, 48
    old = [int(x) for x in rng.integers(1, 16, B)]
    new = [16 - o + 16 * int(p) + int(r) for o, p, r in zip(old, rng.integers(0, 3, B), rng.integers(1, 16, B))]
    cache = make([o + n for o, n in zip(old, new)], heads=kv, kv=kv)
    data = [rows(rng, o + n, kv) for o, n in zip(old, new)]
    seqs = list(range(B))
    put(device, cache, seqs, [d[0][:o] for d, o in zip(data, old)], [d[1][:o] for d, o in zip(data, old)])
    put(device, cache, seqs, [d[0][o:] for d, o in zip(data, old)], [d[1][o:] for d, o in zip(data, old)])
    got = held(device, cache, seqs)
    want = [orc.int8_rows(*d) for d in data]
    assert same_bits(got[0], np.concatenate([w[0] for w in want]))
    assert same_bits(got[1], np.concatenate([w[1] for w in want]))
    cache.destroy()


def test_append_again_in_a_step_gives_the_same(device):
    """Each append of a step may be called more than once: pages that close take
    their earlier rows as they were before the step."""
    say("append again")
    rng = np.random.default_rng(15)
    kv, lens, new = 3, [5, 20, 47, 16], [30, 29, 1, 9]
    cache = make([o + n for o, n in zip(lens, new)], heads=kv, kv=kv)
    data = [rows(rng, o + n, kv) for o, n in zip(lens, new)]
    seqs = list(range(4))
    put(device, cache, seqs, [d[0][:o] for d, o in zip(data, lens)], [d[1][:o] for d, o in zip(data, lens)])
    cache.begin_step(seqs, new)
    k, v = [device.array(np.concatenate([d[i][o:] for d, o in zip(data, lens)])) for i in range(2)]
    want = [orc.int8_rows(*d) for d in data]
    for _ in range(3):
        cache.append_rows(0, k, v)
        got = held(device, cache, seqs)
        assert same_bits(got[0], np.concatenate([w[0] for w in want]))
        assert same_bits(got[1], np.concatenate([w[1] for w in want]))
    cache.destroy()


def test_set_back_past_the_page_before(device):
    """Back into the page that was open before the present one: its FP16 rows
    are still there, up to those that came with the row that filled it."""
    say("set back past a page")
    rng = np.random.default_rng(16)
    for back, exact in ((19, True), (16, True), (20, True), (21, False), (31, False), (9, False)):
        k, v = rows(rng, 40, 2)
        cache = make([60], heads=2, kv=2)
        for lo, hi in ((0, 20), (20, 40)):
            put(device, cache, [0], [k[lo:hi]], [v[lo:hi]])
        cache.set_len(0, back)
        k1, v1 = rows(rng, 2, 2)
        full = [a.astype(np.float16) for a in orc.int8_rows(k, v)]
        p = back // 16 * 16
        before = (k[:back], v[:back]) if exact else [np.concatenate([x[:p], f[p:back]]) for x, f in zip((k, v), full)]
        put(device, cache, [0], [k1], [v1])
        got = held(device, cache, [0])
        want = orc.int8_rows(np.concatenate([before[0], k1]), np.concatenate([before[1], v1]))
        assert same_bits(got[0], want[0]) and same_bits(got[1], want[1]), back
        cache.destroy()


@pytest.mark.parametrize("what", ["zeros", "tiny", "huge", "halfway", "borders", "one_large"])
def test_rows_of_hard_values(device, what):
    """Magnitudes at the ends of the scales, values half-way between two codes,
    largest magnitudes at and next to a border between two scales."""
    say(f"hard values {what}")
    rng = np.random.default_rng(3)
    n, kv = 16 * 24, 2
    x = np.zeros((n, kv, D), np.float16)
    if what == "tiny":
        x = (rng.integers(-40, 41, x.shape) * 2.0 ** -24).astype(np.float16)
    elif what == "huge":
        x = rng.uniform(-65504, 65504, x.shape).astype(np.float16)
        x[::16, :, 0] = 65504
    elif what == "halfway":
        # multiples of half a step of the scale that 127 steps of s make
        s = rng.choice([m * 2.0 ** e for m in range(8, 16) for e in range(-9, -4)], (n // 16, 1, kv, 1))
        c = rng.integers(-253, 254, (n // 16, 16, kv, D)) / 2
        c[:, 0, :, 0] = 127
        x = (c * s).astype(np.float16).reshape(n, kv, D)
    elif what == "borders":
        s = np.array([(8 + i % 8) * 2.0 ** (i // 8 - 8) for i in range(24)]).reshape(24, 1, 1, 1)
        top = (127 * s).astype(np.float16)
        top = np.where(np.arange(2)[None, None, :, None], np.nextafter(top, np.float16(np.inf)), top)
        x = (rng.uniform(-1, 1, (24, 16, kv, D)) * top).astype(np.float16)
        x[:, 5, :, 7] = -top[:, 0, :, 0]
        x = x.reshape(n, kv, D)
    elif what == "one_large":
        x = (rng.standard_normal(x.shape) * 1e-3).astype(np.float16)
        x[::16, :, 9] = 900
    k, v = x, x[::-1].copy()
    cache = make([n], heads=kv, kv=kv)
    put(device, cache, [0], [k], [v])
    got, want = held(device, cache, [0]), orc.int8_rows(k, v)
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    cache.destroy()


def test_rows_not_finite(device):
    say("rows not finite")
    rng = np.random.default_rng(4)
    k, v = rows(rng, 40, 3)
    k[3, 0, 5], v[20, 1, 255], v[35, 2, 0], k[39, 0, 0] = np.inf, np.nan, -np.inf, np.nan
    cache = make([40], heads=3, kv=3)
    put(device, cache, [0], [k], [v])
    got, want = held(device, cache, [0]), orc.int8_rows(k, v)
    assert np.isnan(want[0][:16, 0]).all() and np.isfinite(want[0][16:32, 0]).all() and np.isnan(want[0][35, 2]).all()
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    cache.destroy()


@pytest.mark.parametrize("keep_k", [False, True])
def test_append_normalises_as_the_fp16_cache(device, keep_k):
    """append (and append_decode's, which leaves k alone): q and k the bits of
    the norm's exact order; the pages hold those k."""
    say(f"append norm {keep_k}")
    rng = np.random.default_rng(5)
    lens, new, H, kv = [0, 7, 30], ([1, 1, 1] if keep_k else [33, 9, 2]), 6, 3
    tables = Tables(device, 256)
    cache = make([n + m for n, m in zip(lens, new)], heads=H, kv=kv)
    old = [rows(rng, n, kv) for n in lens]
    put(device, cache, [0, 1, 2], [o[0] for o in old], [o[1] for o in old])
    T = sum(new)
    q = rng.standard_normal((T, H, D), dtype=np.float32).astype(np.float16)
    k, v = rows(rng, T, kv)
    qw, kw = [(1 + 0.02 * rng.standard_normal(D)).astype(np.float16) for _ in range(2)]
    pos = np.concatenate([np.arange(n, n + m) for n, m in zip(lens, new)]) + 11
    dq, dk = device.array(q), device.array(k)
    cache.begin_step([0, 1, 2], new, rope_pos=pos)
    args = (0, dq, dk, device.array(v), device.array(qw), device.array(kw), tables.d_cos, tables.d_sin, 256)
    if keep_k:
        cache.append_decode(*args, device.empty((T, H, D), np.float16))
    else:
        cache.append(*args)
    device.synchronize()
    kn = expected_norm(k, kw, tables, pos)
    assert np.array_equal(dq.numpy().view(np.uint16), expected_norm(q, qw, tables, pos).view(np.uint16))
    assert np.array_equal(dk.numpy().view(np.uint16), (k if keep_k else kn).view(np.uint16))
    got, o, t = held(device, cache, [0, 1, 2]), 0, 0
    for (ok, ov), m in zip(old, new):
        want = orc.int8_rows(np.concatenate([ok, kn[t:t + m]]), np.concatenate([ov, v[t:t + m]]))
        n = len(ok) + m
        assert same_bits(got[0][o:o + n], want[0]) and same_bits(got[1][o:o + n], want[1])
        o, t = o + n, t + m
    cache.destroy()


def test_project_append(device):
    """A projection onto the 8-bit cache leaves the rows that it leaves on an
    FP16 cache, in pages of codes."""
    say("project_append")
    H, kv, hidden = 6, 1, 512
    for new in ([1, 1, 1], [50, 17, 1]):
        rng = np.random.default_rng(6)
        tables = Tables(device, 256)
        T = sum(new)
        x = rng.standard_normal((T, hidden)).astype(np.float16)
        wq = (rng.standard_normal((2 * H * D, hidden)) / 20).astype(np.float16)
        wk = (rng.standard_normal((2 * kv * D, hidden)) / 20).astype(np.float16)
        qw, kw = [(1 + 0.02 * rng.standard_normal(D)).astype(np.float16) for _ in range(2)]
        lens, old = [15, 3, 16], None
        got, q = {}, {}
        for bits in (8, 16):
            cache = make([n + m for n, m in zip(lens, new)], heads=H, kv=kv, bits=bits)
            old = old or [rows(rng, n, kv) for n in lens]
            put(device, cache, [0, 1, 2], [o[0] for o in old], [o[1] for o in old])
            cache.begin_step([0, 1, 2], new)
            qo = device.empty((T, H, D), np.float16)
            cache.project_append(0, device.array(x), hidden, device.array(wq), device.array(wk), device.array(qw),
                                 device.array(kw), tables.d_cos, tables.d_sin, 256, qo)
            device.synchronize()
            got[bits], q[bits] = held(device, cache, [0, 1, 2]), qo.numpy()
            cache.destroy()
        assert np.array_equal(q[8].view(np.uint16), q[16].view(np.uint16))
        o = 0
        for n, m in zip(lens, new):
            want = orc.int8_rows(got[16][0][o:o + n + m], got[16][1][o:o + n + m])
            assert same_bits(got[8][0][o:o + n + m], want[0]) and same_bits(got[8][1][o:o + n + m], want[1])
            o += n + m


def _attend(cache_rows, q, base, gate=None):
    n = q.shape[0]
    k, v = orc.int8_rows(*cache_rows)
    seen = np.arange(k.shape[0])[None] <= base + np.arange(n)[:, None]
    return orc.attention_bound(q, k, v, seen, gate)


@pytest.mark.parametrize("heads,kv", [(24, 4), (6, 1), (8, 8), (8, 1), (6, 3), (10, 5), (40, 10)])
@pytest.mark.parametrize("lens", [[1], [16], [5, 17, 33, 300, 2, 1100], [4000], [300, 1, 129, 1024, 16, 1023]], ids=str)
def test_decode(device, heads, kv, lens):
    say(f"decode8 {heads}/{kv} {lens}")
    rng = np.random.default_rng(heads + kv)
    cache = make(lens, heads=heads, kv=kv)
    data = [rows(rng, n, kv) for n in lens]
    seqs = list(range(len(lens)))
    put(device, cache, seqs, [d[0][:-1] for d in data], [d[1][:-1] for d in data])
    put(device, cache, seqs, [d[0][-1:] for d in data], [d[1][-1:] for d in data])
    q = rng.standard_normal((len(lens), heads, D)).astype(np.float16)
    gate = rng.standard_normal((len(lens), 2 * heads, D)).astype(np.float16)
    out, gated = device.empty(q.shape, np.float16), device.empty(q.shape, np.float16)
    cache.decode(0, device.array(q), out)
    cache.decode(0, device.array(q), gated, gate=device.array(gate), gate_stride=2 * heads * D)
    device.synchronize()
    for b, n in enumerate(lens):
        within(out.numpy()[b:b + 1], *_attend(data[b], q[b:b + 1], n - 1))
        within(gated.numpy()[b:b + 1], *_attend(data[b], q[b:b + 1], n - 1, gate[b:b + 1, :heads]))
    cache.destroy()


# Shares of many pages that begin inside a sequence and go on over others, by
# whole pages and by their last rows: 0 is a workgroup per CU, 2048 shares of
# more pages than a wave has lanes.
@pytest.mark.parametrize("split", [0, 112, 2048])
@pytest.mark.parametrize("heads,kv", [(24, 4), (8, 1)])
def test_decode_of_long_shares(device, heads, kv, split):
    say(f"decode8 long shares {heads}/{kv} {split}")
    rng = np.random.default_rng(heads + split)
    lens = [3001, 9000, 16, 5007, 1, 4444, 2032]
    cache = make(lens, heads=heads, kv=kv, step=sum(lens))
    cache.set_decode_split(split)
    data = [rows(rng, n, kv) for n in lens]
    seqs = list(range(len(lens)))
    put(device, cache, seqs, [d[0][:-1] for d in data], [d[1][:-1] for d in data])
    put(device, cache, seqs, [d[0][-1:] for d in data], [d[1][-1:] for d in data])
    q = rng.standard_normal((len(lens), heads, D)).astype(np.float16)
    out = device.empty(q.shape, np.float16)
    cache.decode(0, device.array(q), out)
    device.synchronize()
    for b, n in enumerate(lens):
        within(out.numpy()[b:b + 1], *_attend(data[b], q[b:b + 1], n - 1))
    cache.destroy()


@pytest.mark.parametrize("heads,kv", [(24, 4), (6, 1), (8, 8), (8, 1), (6, 3), (16, 4)])
@pytest.mark.parametrize("base,new", [([0], [1]), ([0], [16]), ([0], [181]), ([5, 100, 0, 64], [3, 9, 2, 7]),
                                      ([1000, 0, 33], [200, 90, 15]), ([3000], [65])], ids=str)
def test_prefill(device, heads, kv, base, new):
    say(f"prefill8 {heads}/{kv} {base} {new}")
    rng = np.random.default_rng(heads * 10 + kv)
    lens = [b + n for b, n in zip(base, new)]
    cache = make(lens, heads=heads, kv=kv)
    data = [rows(rng, n, kv) for n in lens]
    seqs = list(range(len(lens)))
    put(device, cache, seqs, [d[0][:b] for d, b in zip(data, base)], [d[1][:b] for d, b in zip(data, base)])
    put(device, cache, seqs, [d[0][b:] for d, b in zip(data, base)], [d[1][b:] for d, b in zip(data, base)])
    T = sum(new)
    q = rng.standard_normal((T, heads, D)).astype(np.float16)
    gate = rng.standard_normal((T, heads, D)).astype(np.float16)
    out, gated = device.empty(q.shape, np.float16), device.empty(q.shape, np.float16)
    cache.prefill(0, device.array(q), out)
    cache.prefill(0, device.array(q), gated, gate=device.array(gate))
    device.synchronize()
    t = 0
    for b, n in zip(range(len(lens)), new):
        rows_ = slice(t, t + n)
        within(out.numpy()[rows_], *_attend(data[b], q[rows_], base[b]))
        within(gated.numpy()[rows_], *_attend(data[b], q[rows_], base[b], gate[rows_]))
        t += n
    cache.destroy()


# Steps long enough for two row tiles per wave (48 blocks of 64 keys for each of
# 256 workgroups), as in test_gpu_long_prefill.py; rows of whole tiles, of their
# ends and of a sequence without a past are looked at.
@pytest.mark.parametrize("heads,kv,base,new", [(24, 4, [16400, 16390, 7], [131, 85, 3]),
                                               (16, 2, [24600, 0], [257, 33])])
def test_prefill_of_two_row_tiles(device, heads, kv, base, new):
    say(f"prefill8 two tiles {heads}/{kv} {base} {new}")
    rng = np.random.default_rng(heads + sum(new))
    lens = [b + n for b, n in zip(base, new)]
    cache = make(lens, heads=heads, kv=kv, step=sum(base))
    data = [rows(rng, n, kv) for n in lens]
    seqs = list(range(len(lens)))
    put(device, cache, seqs, [d[0][:b] for d, b in zip(data, base)], [d[1][:b] for d, b in zip(data, base)])
    put(device, cache, seqs, [d[0][b:] for d, b in zip(data, base)], [d[1][b:] for d, b in zip(data, base)])
    tokens = 256 // (heads // kv)
    assert cache.query_tile() == (2, tokens)
    T = sum(new)
    q = rng.standard_normal((T, heads, D)).astype(np.float16)
    gate = rng.standard_normal((T, heads, D)).astype(np.float16)
    out, gated = device.empty(q.shape, np.float16), device.empty(q.shape, np.float16)
    cache.prefill(0, device.array(q), out)
    cache.prefill(0, device.array(q), gated, gate=device.array(gate))
    device.synchronize()
    t = 0
    for b, n in zip(range(len(lens)), new):
        k, v = orc.int8_rows(*data[b])
        for i in sorted({0, 1, tokens // 2, tokens - 1, tokens, n - 2, n - 1}):
            if 0 <= i < n:
                at = slice(t + i, t + i + 1)
                seen = np.arange(lens[b])[None] <= base[b] + i
                within(out.numpy()[at], *orc.attention_bound(q[at], k, v, seen))
                within(gated.numpy()[at], *orc.attention_bound(q[at], k, v, seen, gate[at]))
        t += n
    cache.destroy()


@pytest.mark.parametrize("heads,kv,base,new", [(24, 4, [0, 37, 300], [70, 9, 140]), (8, 8, [100, 7], [9, 5]),
                                               (8, 1, [31, 0], [1, 33]), (24, 4, [16400], [181])], ids=str)
@pytest.mark.parametrize("gated", [False, True])
def test_append_prefill(device, heads, kv, base, new, gated):
    """The one call against append and prefill, to the bit: output, query rows
    and what the cache holds; k is only read.  RoPE positions other than the slots."""
    say(f"append_prefill8 {heads}/{kv} {base} {new} {gated}")
    rng = np.random.default_rng(heads + sum(new))
    lens = [b + n for b, n in zip(base, new)]
    seqs, T = list(range(len(lens))), sum(new)
    tables = Tables(device, 32768)
    ws = [device.array((1 + 0.02 * rng.standard_normal(D)).astype(np.float16)) for _ in range(2)]
    before = [rows(rng, b, kv) for b in base]
    q = rng.standard_normal((T, heads, D)).astype(np.float16)
    k, v = rows(rng, T, kv)
    gate = device.array(rng.standard_normal((T, heads, D)).astype(np.float16)) if gated else None
    pos = [700 + p for b, n in zip(base, new) for p in range(b, b + n)]
    got = []
    for one in (False, True):
        cache = make(lens, heads=heads, kv=kv, step=max(8192, sum(base)))
        put(device, cache, seqs, [d[0] for d in before], [d[1] for d in before])
        cache.begin_step(seqs, new, rope_pos=pos)
        dq, dk, out = device.array(q), device.array(k), device.empty(q.shape, np.float16)
        args = (dq, dk, device.array(v), *ws, tables.d_cos, tables.d_sin, tables.rows)
        if one:
            cache.append_prefill(0, *args, out, gate=gate)
        else:
            cache.append(0, *args)
            cache.prefill(0, dq, out, gate=gate)
        device.synchronize()
        got.append([x.view(np.uint16) for x in (out.numpy(), dq.numpy(), *held(device, cache, seqs))])
        if one:
            assert np.array_equal(dk.numpy().view(np.uint16), k.view(np.uint16)), "k is only read"
        cache.destroy()
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_infinite_query(device):
    """A query head with an infinite value has scores of +inf, or none but -inf:
    its output is NaN, in every form of the decode and in a prefill, and no other's."""
    say("infinite query 8")
    rng = np.random.default_rng(19)
    H, kv = 12, 2
    for lens in ([5, 300, 16], [5, 1100, 4000], [20000, 31, 700]):
        cache = make(lens, heads=H, kv=kv, extra=3, step=32768)
        data = [rows(rng, n + 3, kv) for n in lens]
        put(device, cache, [0, 1, 2], [d[0][:-3] for d in data], [d[1][:-3] for d in data])
        for at, m in ((0, 1), (1, 2)):
            put(device, cache, [0, 1, 2], *([d[j][len(d[j]) - 3 + at:][:m] for d in data] for j in (0, 1)))
            q = rng.standard_normal((3 * m, H, D)).astype(np.float16)
            q[0, 1, 7], q[m, 9, 200], q[2 * m, 4, 0] = np.inf, -np.inf, np.inf
            out = device.empty(q.shape, np.float16)
            (cache.decode if m == 1 else cache.prefill)(0, device.array(q), out)
            device.synchronize()
            want = np.zeros(q.shape, bool)
            want[0, 1] = want[m, 9] = want[2 * m, 4] = True
            assert np.array_equal(np.isnan(out.numpy()), want), (lens, m)
        cache.destroy()


def test_what_is_not_finite_reaches_only_who_sees_it(device):
    say("not finite in attention")
    rng = np.random.default_rng(9)
    H, kv, base, new = 4, 2, 30, 40
    k, v = rows(rng, base + new, kv)
    v[41, 0, 3] = np.inf   # a full page when the chunk is in: rows 32..47 of head 0
    k[66, 1, 0] = np.nan   # in the open page
    cache = make([base + new + 1], heads=H, kv=kv)
    put(device, cache, [0], [k[:base]], [v[:base]])
    put(device, cache, [0], [k[base:]], [v[base:]])
    q = rng.standard_normal((new, H, D)).astype(np.float16)
    out = device.empty(q.shape, np.float16)
    cache.prefill(0, device.array(q), out)
    device.synchronize()
    want = _attend((k, v), q, base)
    assert np.isfinite(want[0][:2, :2]).all() and np.isnan(want[0][2:, :2]).all()
    assert np.isfinite(want[0][:36, 2:]).all() and np.isnan(want[0][36:, 2:]).all()
    within(out.numpy(), *want)
    # a decode step sees both
    k1, v1 = rows(rng, 1, kv)
    put(device, cache, [0], [k1], [v1])
    cache.decode(0, device.array(q[:1]), out)
    device.synchronize()
    assert np.isnan(out.numpy()[0]).all()
    cache.destroy()


def test_stale_rows_of_the_open_page_are_not_read(device):
    """A sequence starts over in a slot whose open page held NaN rows."""
    say("stale open rows")
    rng = np.random.default_rng(10)
    H, kv = 6, 2
    cache = make([16], heads=H, kv=kv, extra=16)
    k, v = rows(rng, 10, kv)
    k[:], v[:] = np.nan, np.inf
    put(device, cache, [0], [k], [v])
    cache.set_len(0, 0)
    k, v = rows(rng, 5, kv)
    put(device, cache, [0], [k[:4]], [v[:4]])
    q = rng.standard_normal((4, H, D)).astype(np.float16)
    out = device.empty(q.shape, np.float16)
    cache.prefill(0, device.array(q), out)
    device.synchronize()
    within(out.numpy(), *_attend((k[:4], v[:4]), q, 0))
    put(device, cache, [0], [k[4:]], [v[4:]])
    cache.decode(0, device.array(q[:1]), out)
    device.synchronize()
    within(out.numpy()[:1], *_attend((k, v), q[:1], 4))
    cache.destroy()


@pytest.mark.parametrize("layers", [1, 3])
def test_length_set_back(device, layers):
    """Back within the open page, to a page's end, and into full pages (whose
    values the open page then continues from); then on again."""
    say(f"set back {layers}")
    rng = np.random.default_rng(11)
    H, kv = 4, 2
    cache = make([80], heads=H, kv=kv, layers=layers)
    data = [rows(rng, 70, kv) for _ in range(layers)]

    def add(k, v):
        cache.begin_step([0], [len(k[0])])
        for i in range(layers):
            cache.append_rows(i, device.array(k[i]), device.array(v[i]))

    add([d[0] for d in data], [d[1] for d in data])
    model = [[np.array(a) for a in d] for d in data]  # rows as they went in, or as the open page continues from
    for back in (67, 64, 37, 36, 20):
        if back // 16 != len(model[0][0]) // 16 and back % 16:
            for m in model:
                full = [a.astype(np.float16) for a in orc.int8_rows(*m)]
                p = back // 16 * 16
                m[0][p:p + 16], m[1][p:p + 16] = full[0][p:p + 16], full[1][p:p + 16]
        cache.set_len(0, back)
        more = [rows(rng, 3, kv) for _ in range(layers)]
        add([m[0] for m in more], [m[1] for m in more])
        for i in range(layers):
            model[i] = [np.concatenate([a[:back], b]) for a, b in zip(model[i], more[i])]
            got, want = held(device, cache, [0], layer=i), orc.int8_rows(*model[i])
            assert same_bits(got[0], want[0]) and same_bits(got[1], want[1]), (back, i)
    q = rng.standard_normal((1, H, D)).astype(np.float16)
    more = [rows(rng, 1, kv) for _ in range(layers)]
    add([m[0] for m in more], [m[1] for m in more])
    out = device.empty(q.shape, np.float16)
    cache.decode(layers - 1, device.array(q), out)
    device.synchronize()
    last = [np.concatenate([a, b]) for a, b in zip(model[-1], more[-1])]
    within(out.numpy(), *_attend(last, q, len(last[0]) - 1))
    cache.destroy()


def test_blocks_that_change_places(device):
    """A full page reads as the block that it was given, also where the length
    goes back into it and rows follow; the last page stays with the sequence."""
    say("blocks change places")
    rng = np.random.default_rng(16)
    kv = 2
    k, v = rows(rng, 42, kv)
    cache = make([40], heads=2, kv=kv, extra=8)
    for a, b in ((0, 20), (20, 40)):  # page 1 is open once
        put(device, cache, [0], [k[a:b]], [v[a:b]])
    page = [orc.int8_rows(k[16 * p:16 * p + 16], v[16 * p:16 * p + 16]) for p in range(2)]
    b0, b1, b2 = cache.blocks(0)
    cache.set_blocks(0, [b1, b0, b2])
    swapped = [np.concatenate([page[1][i], page[0][i], x[32:40].astype(np.float64)]) for i, x in enumerate((k, v))]
    for n in (40, 18):
        cache.set_len(0, n)
        got = held(device, cache, [0])
        assert all(same_bits(g, w[:n]) for g, w in zip(got, swapped)), n
    put(device, cache, [0], [k[40:]], [v[40:]])
    got = held(device, cache, [0])
    for g, w, x in zip(got, swapped, (k, v)):
        assert same_bits(g[:18], w[:18]) and same_bits(g[18:], x[40:])
    cache.destroy()


def test_a_step_without_rows_leaves_the_sequence(device):
    """Listed with no new rows, a sequence that was set back keeps what lies
    behind its length, the open page's FP16 rows among it."""
    say("a step without rows")
    rng = np.random.default_rng(17)
    kv = 2
    k, v = rows(rng, 41, kv)
    cache = make([40, 10], heads=2, kv=kv, extra=8)
    for a, b in ((0, 20), (20, 40)):
        put(device, cache, [0], [k[a:b]], [v[a:b]])
    for back in (18, 9, 16, 0):  # pages held in FP16, in codes, none
        cache.set_len(0, back)
        put(device, cache, [0, 1], [k[:0], k[:2]], [v[:0], v[:2]])
        cache.set_len(0, 40)
        got, want = held(device, cache, [0]), orc.int8_rows(k[:40], v[:40])
        assert same_bits(got[0], want[0]) and same_bits(got[1], want[1]), back
    put(device, cache, [0], [k[40:]], [v[40:]])
    got, want = held(device, cache, [0]), orc.int8_rows(k, v)
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    cache.destroy()


def test_recorded_step(device):
    """A replayed step gives the eager bits while lengths grow over page ends,
    with eager work between the replays."""
    from mi50grad_amd.device import Stream

    say("recorded step 8")
    rng = np.random.default_rng(12)
    H, kv, lens = 6, 2, [14, 31, 2000, 100]
    tables = Tables(device, 4096)
    seqs = list(range(4))
    w = [device.array((1 + 0.02 * rng.standard_normal(D)).astype(np.float16)) for _ in range(2)]
    caches = [make(lens, heads=H, kv=kv, extra=32) for _ in range(2)]
    data = [rows(rng, n, kv) for n in lens]
    s = Stream()
    for c in caches:
        put(device, c, seqs, [d[0] for d in data], [d[1] for d in data])
    device.synchronize()
    dq, dk, dv, out, eager_q = [device.empty((4, h, D), np.float16) for h in (H, kv, kv, H, H)]
    graph = None
    for i in range(12):
        q = rng.standard_normal((4, H, D)).astype(np.float16)
        k, v = rows(rng, 4, kv)
        dk.copy_from(k)
        dv.copy_from(v)
        eager_q.copy_from(q)
        caches[0].begin_step(seqs, [1] * 4)
        want = device.empty(q.shape, np.float16)
        caches[0].append_decode(0, eager_q, dk, dv, *w, tables.d_cos, tables.d_sin, 4096, want)
        device.synchronize()
        dq.copy_from(q)
        caches[1].begin_step(seqs, [1] * 4, stream=s.handle)
        if graph is None:
            graph = caches[1].record_step(s.handle)
            caches[1].append_decode(0, dq, dk, dv, *w, tables.d_cos, tables.d_sin, 4096, out, stream=s.handle)
            graph.end()
        graph.launch()
        s.synchronize()
        assert np.array_equal(out.numpy().view(np.uint16), want.numpy().view(np.uint16)), i
    a, b = held(device, caches[0], seqs), held(device, caches[1], seqs)
    assert same_bits(a[0], b[0]) and same_bits(a[1], b[1])
    graph.destroy()
    for c in caches:
        c.destroy()
    s.destroy()


def test_recorded_short_step_of_sequences_grown(device):
    """A decode recorded in its form for short sequences, replayed when they
    have grown past what the step plan holds the pages of and past 512 pages."""
    from mi50grad_amd.device import Stream

    say("recorded short step 8")
    rng = np.random.default_rng(14)
    H, kv, seqs = 12, 2, [0, 1, 2]
    parts = [[1, 1000, 17], [1100, 0, 15], [0, 8200, 16]]
    data = [rows(rng, sum(n) + len(parts), kv) for n in zip(*parts)]
    cache = make([len(d[0]) for d in data], heads=H, kv=kv, step=9000)
    s = Stream()
    at = [0, 0, 0]

    def grow(n):
        ks = [d[0][a:a + m] for d, a, m in zip(data, at, n)]
        vs = [d[1][a:a + m] for d, a, m in zip(data, at, n)]
        put(device, cache, seqs, ks, vs, stream=s.handle)
        s.synchronize()
        for b, m in enumerate(n):
            at[b] += m

    dq, out = device.empty((3, H, D), np.float16), device.empty((3, H, D), np.float16)
    graph = None
    for n in parts:
        if any(n):
            grow(n)
        grow([1, 1, 1])
        q = rng.standard_normal((3, H, D)).astype(np.float16)
        dq.copy_from(q)
        device.synchronize()
        if graph is None:
            graph = cache.record_step(s.handle)
            cache.decode(0, dq, out, stream=s.handle)
            graph.end()
        graph.launch()
        s.synchronize()
        got = out.numpy()
        for b in seqs:
            within(got[b:b + 1], *_attend([x[:at[b]] for x in data[b]], q[b:b + 1], at[b] - 1))
    graph.destroy()
    cache.destroy()
    s.destroy()


def test_pages_past_32_bits(device):
    """Blocks whose codes lie more than 4 GiB into their pools."""
    from mi50grad_amd.kv_cache import PagedKVCache

    say("pages past 32 bits")
    rng = np.random.default_rng(15)
    H, kv, lens, blocks = 24, 4, [300, 1000], 270000  # 4.4 GB of K codes
    cache = PagedKVCache(n_layers=1, max_seqs=2, max_blocks=blocks, max_blocks_per_seq=64, max_step_tokens=1300,
                         num_heads=H, num_kv_heads=kv, kv_bits=8)
    assert blocks * 16 * kv * D > 2**32
    for b, at in enumerate((blocks - 19, blocks - 19 - 63)):
        cache.set_blocks(b, range(at, at + (lens[b] + 15) // 16))
    data = [rows(rng, n, kv) for n in lens]
    q = rng.standard_normal((9, H, D)).astype(np.float16)
    out, w = device.empty(q.shape, np.float16), device.empty((2, kv, 1000), np.float32)
    put(device, cache, [0, 1], [d[0][:-5] for d in data], [d[1][:-5] for d in data])
    put(device, cache, [0, 1], [d[0][-5:-1] for d in data], [d[1][-5:-1] for d in data])
    cache.prefill(0, device.array(q[:8]), out)
    device.synchronize()
    for b, n in enumerate(lens):
        at = slice(4 * b, 4 * b + 4)
        within(out.numpy()[at], *_attend([x[:-1] for x in data[b]], q[at], n - 5))
    put(device, cache, [0, 1], [d[0][-1:] for d in data], [d[1][-1:] for d in data])
    cache.decode(0, device.array(q[:2]), out)
    cache.attn_weights(0, device.array(q[:2]), w, 1000, decay=0.0)
    device.synchronize()
    got = held(device, cache, [0, 1])
    want = [np.concatenate(x) for x in zip(*(orc.int8_rows(*d) for d in data))]
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    for b, n in enumerate(lens):
        within(out.numpy()[b:b + 1], *_attend(data[b], q[b:b + 1], n - 1))
        assert np.abs(w.numpy()[b, :, :n].sum(-1) - H // kv).max() < 1e-3  # each head's weights sum to one
    cache.destroy()


def test_half_the_difference_of_a_step(device):
    """Against the FP16 rows themselves a value is off by half a step at most,
    and a step is at most 1/8 wider than 1/127 of the block's largest."""
    say("error of the codes")
    rng = np.random.default_rng(13)
    k, v = rows(rng, 160, 4)
    cache = make([160])
    put(device, cache, [0], [k], [v])
    for got, x in zip(held(device, cache, [0]), (k, v)):
        x = x.astype(np.float64).reshape(10, 16, 4, D)
        top = np.abs(x).max((1, 3), keepdims=True)
        assert (np.abs(got.reshape(x.shape) - x) <= top / 127 * 1.125 / 2).all()
    cache.destroy()
