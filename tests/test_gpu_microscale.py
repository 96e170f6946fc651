"""GPU: microscaled rows, the norm that makes them and the products of them,
against the oracle in 64 bits.

Quantisation, reading back and packing are exact.  Products are bit-exact on
inputs whose sums are exact in fp32 in any order, and on random ones within
half an fp16 step and the matrix unit's error: each instruction adds 64
products and the running sum, of which it may drop what lies below 2^-23 of the
largest, so K / 64 of them are off by at most K / 64 * 65 * 2^-23 of the largest
magnitude among the products and the running sums (twice the largest prefix
sum bounds those of any contiguous slice).
"""
import numpy as np
import pytest

from mi50grad_amd import microscale as ms
from mi50grad_amd.device import DeviceArray, Stream
from mi50grad_amd.kv_cache import PagedKVCache
from oracle import kvattn_oracle as orc
from oracle import microscale_oracle as mx

from gpu_helpers import D, Tables, build_cache, max_err, say

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _bits(a):
    return np.asarray(a).view(np.uint16)


def _rows(rng, rows, cols):
    """fp16 rows of unlike size, from subnormal to infinite, with zero blocks and signed zeros."""
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-22, 13, (rows, 1))
    x[:, ::7] *= 8
    x[rng.random((rows, cols)) < 0.1] = 0.0
    x[rng.random((rows, cols)) < 0.05] *= -0.0
    x[0, :32] = 0.0
    with np.errstate(over="ignore"):
        return x.astype(np.float16)


def _quantize(device, x, bits, stride=0):
    rows, cols = x.shape[0], x.shape[1] if not stride else x.shape[1] - stride
    guard = 64
    codes = device.array(np.full(rows * cols * bits // 8 + guard, 0xa5, np.uint8))
    scales = device.array(np.full(rows * cols // 32 + guard, 0xa5, np.uint8))
    ms.quantize(device.array(x), rows, cols, bits, codes, scales, x_stride=x.shape[1])
    device.synchronize()
    c, s = codes.numpy(), scales.numpy()
    assert (c[-guard:] == 0xa5).all() and (s[-guard:] == 0xa5).all()
    return c[:-guard].reshape(rows, -1), s[:-guard].reshape(rows, -1)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows,cols,stride", [(1, 32, 0), (3, 96, 8), (37, 512, 0), (5, 6144, 6144), (129, 352, 24)])
def test_quantize(device, bits, rows, cols, stride):
    say(f"quantize {rows} x {cols} to {bits} bits, stride {cols + stride}")
    rng = np.random.default_rng(rows + bits)
    x = _rows(rng, rows, cols + stride)
    c, s = _quantize(device, x, bits, stride)
    code, b = mx.encode(x[:, :cols], bits)
    assert np.array_equal(s, b)
    assert np.array_equal(mx.unpack_codes(c, bits), code)


@pytest.mark.parametrize("bits", [8, 4])
def test_quantize_every_value(device, bits):
    """Every finite fp16 value beside the largest of blocks of several sizes."""
    say(f"quantize every fp16 value to {bits} bits")
    v = np.arange(65536, dtype=np.uint16).view(np.float16)
    v = np.sort(v[np.isfinite(v)])
    v = np.concatenate([v, np.zeros(-len(v) % 31, np.float16)]).reshape(-1, 31)
    for top in (0.0, 1.0, 6.0, 447.0, 448.5, 65504.0, 2.0 ** -24):
        x = np.concatenate([v, np.full((len(v), 1), top, np.float16)], 1)
        c, s = _quantize(device, x, bits)
        code, b = mx.encode(x, bits)
        assert np.array_equal(s, b), top
        assert np.array_equal(mx.unpack_codes(c, bits), code), top


@pytest.mark.parametrize("bits", [8, 4])
def test_quantize_what_is_not_finite(device, bits):
    say(f"quantize infinities and NaN to {bits} bits")
    x = np.ones((3, 128), np.float16)
    x[0, 3], x[1, 40], x[2, 127] = np.inf, np.nan, -np.inf
    c, s = _quantize(device, x, bits)
    code, b = mx.encode(x, bits)
    assert np.array_equal(s, b) and (s == 255).sum() == 3
    assert np.array_equal(mx.unpack_codes(c, bits), code)


@pytest.mark.parametrize("bits", [8, 4])
def test_dequantize(device, bits):
    """Every code under every scale, those of other makers among them."""
    say(f"dequantize every {bits}-bit code under every scale")
    per = (1 << bits) if bits == 8 else 256
    codes = np.tile(np.arange(per, dtype=np.uint8), (256, 1))
    cols = 8 * per // bits
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], cols // 32, 1)
    y = device.empty((256, cols), np.float16)
    ms.dequantize(device.array(codes), device.array(scales), 256, cols, bits, y)
    device.synchronize()
    with np.errstate(over="ignore"):
        want = mx.decode(codes, scales, bits).astype(np.float16)
    got = y.numpy()
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(np.signbit(got) | np.isnan(got), np.signbit(want) | np.isnan(want))


@pytest.mark.parametrize("rows,cols", [(1, 512), (32, 512), (45, 1024), (336, 1536)])
def test_pack_weights(device, rows, cols):
    say(f"pack {rows} x {cols}")
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, cols // 32), dtype=np.uint8)
    n = ms.packed_bytes(rows, cols)
    packed = device.array(np.full(n + 64, 0xa5, np.uint8))
    ms.pack_weights(device.array(codes), device.array(scales), rows, cols, packed)
    device.synchronize()
    got = packed.numpy()
    assert np.array_equal(got[:n], mx.pack_weights(codes, scales)) and (got[n:] == 0xa5).all()


# ---- the norm ---------------------------------------------------------------

# The sum of n squares in fp32 (lanes of at most 32 terms one after another,
# then a tree and at most 16 more), the root, the quotient and two products:
# under 64 roundings of 2^-24.
FP32 = 2.0 ** -18


def _check_norm(total, want, got, bits):
    """`got`: fp16 rows, or (codes, scales)."""
    if bits == 16:
        slack = np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) + np.abs(want) * FP32
        assert (np.abs(got.astype(np.float64) - want) <= slack).all()
        return
    codes, scales = got
    top = mx.GRID[bits][-1]
    most = np.abs(want.reshape(want.shape[0], -1, 32)).max(-1)
    s = 2.0 ** (scales.astype(float) - 127)
    assert (most * (1 - FP32) <= top * s).all()
    assert ((most * (1 + FP32) > top * s / 2) | (scales == 1)).all()
    y = np.abs(want) / np.repeat(s, 32, 1)
    least, mant = {8: (-6, 3), 4: (0, 1)}[bits]
    e = np.maximum(np.floor(np.log2(np.maximum(y * (1 + FP32), 2.0 ** least))), least)
    slack = np.exp2(e - mant) / 2 * np.repeat(s, 32, 1) + np.abs(want) * FP32
    assert (np.abs(mx.decode(codes, scales, bits) - want) <= slack).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("n_tok,cols,delta", [(1, 5120, True), (3, 32, True), (2, 96, False), (67, 512, True),
                                              (5, 8192, True), (3, 8224, False), (2, 16416, True), (2, 32768, True)])
def test_norm(device, bits, n_tok, cols, delta):
    say(f"add_rmsnorm {n_tok} x {cols} to {bits} bits, delta {delta}")
    rng = np.random.default_rng(n_tok + cols + bits)
    h = rng.standard_normal((n_tok, cols)).astype(np.float16)
    h[:, ::41] *= 30
    d = rng.standard_normal((n_tok, cols)).astype(np.float16) if delta else None
    w = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float16)
    total, want = mx.add_rmsnorm(h, d, w, EPS)
    guard = np.full((1, cols), 77.0, np.float16)
    s_out = device.array(np.concatenate([h, guard])) if delta else None
    kw = dict(sum_out=s_out)
    if bits == 16:
        out = device.array(np.concatenate([h, guard]))
    else:
        out = device.array(np.full((n_tok + 1, cols * bits // 8), 0xa5, np.uint8))
        kw.update(scales=device.array(np.full((n_tok + 1, cols // 32), 0xa5, np.uint8)), bits=bits)
    ms.add_rmsnorm(device.array(h), device.array(d) if delta else None, device.array(w), n_tok, cols, EPS, out, **kw)
    device.synchronize()
    got = out.numpy()
    if delta:
        s = s_out.numpy()
        assert np.array_equal(_bits(s[:n_tok]), _bits(total)) and np.array_equal(_bits(s[n_tok:]), _bits(guard))
    if bits == 16:
        assert np.array_equal(_bits(got[n_tok:]), _bits(guard))
        _check_norm(total, want, got[:n_tok], bits)
    else:
        sc = kw["scales"].numpy()
        assert (got[n_tok:] == 0xa5).all() and (sc[n_tok:] == 0xa5).all()
        _check_norm(total, want, (got[:n_tok], sc[:n_tok]), bits)


def test_norm_in_place_and_edges(device):
    """The sum over either term; zeros, a tie that fp16 decides, infinities."""
    say("add_rmsnorm in place")
    rng = np.random.default_rng(5)
    n, cols = 6, 320
    h, d = (rng.standard_normal((n, cols)).astype(np.float16) for _ in "hd")
    h[1], d[1] = 0, 0
    h[2], d[2] = 2048, 1 + 2.0 ** -10
    h[3, 7] = np.inf
    h[4, 9], d[4, 9] = np.inf, -np.inf
    h[5] = 6e-8
    d[5] = 0
    w = np.ones(cols, np.float16)
    with np.errstate(invalid="ignore"):
        total, want = mx.add_rmsnorm(h, d, w, EPS)
    for over in ("hidden", "delta"):
        dh, dd, x = device.array(h), device.array(d), device.empty((n, cols), np.float16)
        ms.add_rmsnorm(dh, dd, device.array(w), n, cols, EPS, x, sum_out=dh if over == "hidden" else dd)
        codes, scales = device.empty((n, cols), np.uint8), device.empty((n, cols // 32), np.uint8)
        ms.add_rmsnorm(dh if over == "hidden" else dd, None, device.array(w), n, cols, EPS, codes, scales=scales, bits=8)
        device.synchronize()
        got = (dh if over == "hidden" else dd).numpy()
        assert np.array_equal(got, total, equal_nan=True)
        x, c, s = x.numpy(), codes.numpy(), scales.numpy()
        fine = [0, 1, 2, 5]
        _check_norm(total[fine], want[fine], x[fine], 16)
        _check_norm(total[fine], want[fine], (c[fine], s[fine]), 8)
        assert not x[1].any() and (s[1] == 1).all()
        # an infinite sum makes every other value 0 and itself NaN; a NaN one all NaN
        assert np.isnan(x[3, 7]) and not np.delete(x[3], 7).any() and np.isnan(x[4]).all()
        assert s[3].tolist() == [255] + [1] * 9 and (s[4] == 255).all()


# ---- the products -----------------------------------------------------------

def _exact_rows(rng, rows, cols, bits):
    """Codes and scales whose products have exact fp32 sums: elements of at most
    8 (6 in 4 bits) in halves, scales 2^-4 to 2^-2."""
    grid = mx.GRID[bits]
    small = np.flatnonzero((grid <= 8) & (grid * 2 == np.round(grid * 2)))
    code = small[rng.integers(0, len(small), (rows, cols))] + (rng.integers(0, 2, (rows, cols)) << (bits - 1))
    return mx.pack_codes(code.astype(np.uint8), bits), rng.integers(123, 126, (rows, cols // 32), dtype=np.uint8)


def _random_rows(rng, rows, cols, bits):
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-2, 3, (rows, 1))
    x[:, ::97] *= 10
    code, s = mx.encode(x, bits)
    return mx.pack_codes(code, bits), s


def _pack(device, w):
    rows, cols = w[0].shape[0], 2 * w[0].shape[1]
    packed = device.empty(ms.packed_bytes(rows, cols), np.uint8)
    ms.pack_weights(device.array(w[0]), device.array(w[1]), rows, cols, packed)
    device.synchronize()
    return packed


def _product(x, w):
    """y in 64 bits and how far the matrix unit's fp32 sums may be off."""
    terms = x.shape[1]
    y = x @ w.T
    run = np.zeros_like(y)
    most = np.zeros_like(y)
    for k in range(0, terms, 64):
        run += x[:, k:k + 64] @ w[:, k:k + 64].T
        most = np.maximum(most, np.abs(run))
    top = np.abs(x).max(1)[:, None] * np.abs(w).max(1)[None, :]
    return y, terms / 64 * 65 * 2.0 ** -23 * (2 * most + top)


def _half_step(y):
    return np.maximum(np.abs(y) * 2.0 ** -11, 2.0 ** -25)


def _any_cache():
    return build_cache([8], [[0]], extra_rows=[1])[0]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_tok,q_dim,n_out,res", [
    (1, 512, 16, False), (1, 6144, 5120, True), (5, 512, 48, True), (31, 1536, 336, False), (32, 6144, 5120, True),
    (33, 2048, 1040, True), (64, 1024, 512, True), (100, 4096, 2064, False), (181, 6144, 5120, True),
    (257, 512, 272, True), (700, 1536, 1040, True), (2048, 512, 5120, False), (1300, 2048, 2048, True)])
def test_out_project_exact(device, bits, n_tok, q_dim, n_out, res):
    rng = np.random.default_rng(n_tok + n_out + bits)
    say(f"mx_out_project exact {n_tok} tokens, {q_dim} -> {n_out}, {bits} bits")
    cache = _any_cache()
    x, w = _exact_rows(rng, n_tok, q_dim, bits), _exact_rows(rng, n_out, q_dim, 4)
    r = rng.integers(-8, 9, (n_tok, n_out)).astype(np.float16) if res else None
    guard = np.full((1, n_out), 77.0, np.float16)
    out = device.array(np.concatenate([r if res else np.zeros((n_tok, n_out), np.float16), guard]))
    cache.mx_out_project(device.array(x[0]), n_tok, q_dim, _pack(device, w), n_out, out,
                         residual=out if res else None, attn_scales=device.array(x[1]), bits=bits)
    device.synchronize()
    y = mx.decode(*x, bits) @ mx.decode(*w, 4).T
    want = (y + r if res else y).astype(np.float16)
    got = out.numpy()
    assert np.array_equal(got[:n_tok], want)
    assert np.array_equal(_bits(got[n_tok:]), _bits(guard))
    cache.destroy()


# Every tile by its plan, with token and row remainders.
@pytest.mark.parametrize("bits,n_tok,q_dim,n_out,tile,partial", [
    (8, 37, 512, 48, (64, 128), 0), (4, 37, 512, 48, (64, 128), 0), (8, 45, 4096, 16, (64, 128), 1),
    (4, 45, 4096, 16, (64, 128), 1), (8, 271, 512, 7184, (64, 256), 0), (4, 150, 1536, 14352, (64, 256), 0),
    (8, 8190, 1024, 336, (128, 128), 0), (4, 271, 512, 7184, (128, 128), 0), (8, 283, 512, 14352, (128, 256), 0),
    (4, 283, 512, 14352, (128, 256), 0), (8, 1310, 1536, 6160, (128, 320), 0), (4, 1310, 1536, 6160, (128, 320), 0),
    (8, 1510, 1536, 7184, (256, 256), 0), (4, 1510, 1536, 7184, (256, 256), 0)])
def test_out_project_each_tile(device, bits, n_tok, q_dim, n_out, tile, partial):
    rng = np.random.default_rng(n_tok + n_out + bits)
    say(f"mx_out_project tile {tile} partial={partial} {n_tok} tokens, {q_dim} -> {n_out}, {bits} bits")
    cache = _any_cache()
    x, w = _exact_rows(rng, n_tok, q_dim, bits), _exact_rows(rng, n_out, q_dim, 4)
    r = rng.integers(-8, 9, (n_tok, n_out)).astype(np.float16)
    guard = np.full((1, n_out), 77.0, np.float16)
    out = device.array(np.concatenate([r, guard]))
    cache.mx_out_project(device.array(x[0]), n_tok, q_dim, _pack(device, w), n_out, out, residual=out,
                         attn_scales=device.array(x[1]), bits=bits)
    device.synchronize()
    plan = cache.product_plan()
    assert (plan["tile_tokens"], plan["tile_rows"]) == tile and plan["partial"] == partial, plan
    got = out.numpy()
    assert np.array_equal(got[:n_tok], (mx.decode(*x, bits) @ mx.decode(*w, 4).T + r).astype(np.float16))
    assert np.array_equal(_bits(got[n_tok:]), _bits(guard))
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_tok,q_dim,n_out", [(1, 6144, 5120), (7, 2048, 1040), (8, 512, 16), (3, 1536, 8208),
                                               (9, 1024, 336), (32, 6144, 5120), (181, 6144, 1040),
                                               (520, 4096, 528)])
def test_out_project_quantises_fp16_rows(device, bits, n_tok, q_dim, n_out):
    """fp16 rows give the bits that their microscaled rows give, and both are
    the product to its rounding."""
    rng = np.random.default_rng(n_tok + n_out + bits)
    say(f"mx_out_project of fp16 rows {n_tok} tokens, {q_dim} -> {n_out}, {bits} bits")
    cache = _any_cache()
    x = (rng.standard_normal((n_tok, q_dim)) * 2.0 ** rng.integers(-3, 3, (n_tok, 1))).astype(np.float16)
    x[:, ::97] *= 10
    x[0, 32:64] = 0
    x[n_tok // 2, 64:96] *= 2.0 ** -14  # subnormal
    w = _random_rows(rng, n_out, q_dim, 4)
    r = rng.standard_normal((n_tok, n_out)).astype(np.float16)
    packed, dr = _pack(device, w), device.array(r)
    out, coded = device.empty((n_tok, n_out), np.float16), device.empty((n_tok, n_out), np.float16)
    cache.mx_out_project(device.array(x), n_tok, q_dim, packed, n_out, out, residual=dr, bits=bits)
    codes, scales = device.empty((n_tok, q_dim * bits // 8), np.uint8), device.empty((n_tok, q_dim // 32), np.uint8)
    ms.quantize(device.array(x), n_tok, q_dim, bits, codes, scales)
    cache.mx_out_project(codes, n_tok, q_dim, packed, n_out, coded, residual=dr, attn_scales=scales, bits=bits)
    device.synchronize()
    got = out.numpy()
    assert np.array_equal(_bits(got), _bits(coded.numpy()))
    y, off = _product(mx.quantized(x, bits), mx.decode(*w, 4))
    y = y + r
    assert (np.abs(got - y) <= _half_step(y) + off).all()
    cache.destroy()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_tok", [2, 8, 20])
def test_fp16_rows_that_are_not_finite(device, bits, n_tok):
    """A row with an infinity or NaN gives NaN, the others what they give without."""
    rng = np.random.default_rng(n_tok + bits)
    q_dim, n_out = 1024, 48
    say(f"mx_out_project of fp16 rows that are not finite, {n_tok} tokens, {bits} bits")
    cache = _any_cache()
    v = rng.integers(-3, 4, (n_tok, q_dim)).astype(np.float16)  # exact in 4 and 8 bits
    w = _exact_rows(rng, n_out, q_dim, 4)
    y = v.astype(np.float64) @ mx.decode(*w, 4).T
    v[0, 17], v[1, 1000] = np.nan, -np.inf
    y[:2] = np.nan
    out = device.empty((n_tok, n_out), np.float16)
    cache.mx_out_project(device.array(v), n_tok, q_dim, _pack(device, w), n_out, out, bits=bits)
    device.synchronize()
    assert np.array_equal(out.numpy(), y.astype(np.float16), equal_nan=True)
    cache.destroy()


def test_out_project_in_parts(device):
    """More rows than the workspace takes at once."""
    rng = np.random.default_rng(9)
    heads, n_tok, q_dim, n_out = 1, 3000, 1024, 1024
    say("mx_out_project in parts")
    cache = PagedKVCache(n_layers=1, max_seqs=1, max_blocks=1, max_blocks_per_seq=1, max_step_tokens=1,
                         num_heads=heads, num_kv_heads=1)
    v = rng.integers(-4, 5, (n_tok, q_dim)).astype(np.float16)  # exact in 8 bits
    w = _exact_rows(rng, n_out, q_dim, 4)
    out = device.empty((n_tok, n_out), np.float16)
    cache.mx_out_project(device.array(v), n_tok, q_dim, _pack(device, w), n_out, out)
    device.synchronize()
    assert np.array_equal(out.numpy(), (v.astype(np.float64) @ mx.decode(*w, 4).T).astype(np.float16))
    cache.destroy()


@pytest.mark.parametrize("n_tok", [3, 40, 300])
def test_products_keep_nan_in_its_row(device, n_tok):
    """A NaN block of a token makes its outputs NaN, one of a weight row that
    row's; the others are as they are without."""
    rng = np.random.default_rng(n_tok)
    q_dim, n_out = 1024, 1040
    say(f"mx_out_project with NaN, {n_tok} tokens")
    cache = _any_cache()
    x, w = _exact_rows(rng, n_tok, q_dim, 8), _exact_rows(rng, n_out, q_dim, 4)
    y = mx.decode(*x, 8) @ mx.decode(*w, 4).T
    x[1][1, 30] = 255
    w[1][1037, 0] = w[1][40, 31] = 255
    x[0][2, 17] = 0x7f  # an element that is NaN
    out = device.empty((n_tok, n_out), np.float16)
    cache.mx_out_project(device.array(x[0]), n_tok, q_dim, _pack(device, w), n_out, out,
                         attn_scales=device.array(x[1]))
    device.synchronize()
    got = out.numpy()
    y[1:3] = np.nan
    y[:, [40, 1037]] = np.nan
    assert np.array_equal(got, y.astype(np.float16), equal_nan=True)
    cache.destroy()


def _step(device, rng, heads, kv, hidden, lengths, n_new, bits, exact, fp16=False, rope_pos=None):
    """One step through mx_project_append, everything to check with it."""
    T = sum(n_new)
    pages = [(a + b + 15) // 16 for a, b in zip(lengths, n_new)]
    perm = [int(x) for x in rng.permutation(sum(pages))]
    ids = [[perm.pop() for _ in range(n)] for n in pages]
    cache, kr, vr = build_cache(lengths, ids, extra_rows=list(n_new), rng=rng, num_heads=heads, num_kv_heads=kv)
    rows = _exact_rows if exact else _random_rows
    wq, wkv = rows(rng, 2 * heads * D, hidden, 4), rows(rng, 2 * kv * D, hidden, 4)
    qw, kw = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float16) for _ in "qk")
    tables = Tables(device, 1024)
    pos = rope_pos or [a + i for a, b in zip(lengths, n_new) for i in range(b)]
    if fp16:
        x = rng.integers(-4, 5, (T, hidden)).astype(np.float16)
        xv, dx, dxs = mx.quantized(x, bits), device.array(x), None
    else:
        x = rows(rng, T, hidden, bits)
        xv, dx, dxs = mx.decode(*x, bits), device.array(x[0]), device.array(x[1])
    cache.begin_step(list(range(len(lengths))), list(n_new), rope_pos=rope_pos)
    guard = lambda *s: device.array(np.full((T + 1,) + s, 77.0, np.float16))  # noqa: E731
    d = dict(q=guard(heads, D), g=guard(heads, D), kv=guard(2, kv, D))
    cache.mx_project_append(0, dx, hidden, _pack(device, wq), _pack(device, wkv), device.array(qw), device.array(kw),
                            tables.d_cos, tables.d_sin, tables.rows, d["q"], d["g"], d["kv"], x_scales=dxs, bits=bits)
    device.synchronize()
    got = {k: v.numpy() for k, v in d.items()}
    for v in got.values():
        assert (v[T:] == 77).all()
    got = {k: v[:T] for k, v in got.items()}
    y, off = _product(xv, np.concatenate([mx.decode(*wq, 4), mx.decode(*wkv, 4)]))
    return cache, kr, vr, got, y.reshape(T, -1, D), off.reshape(T, -1, D), qw, kw, tables, pos


def _check_rotated(got, y, off, w, tables, pos):
    """Rows after norm and RoPE.  An error e of y (at most `off`) moves the norm
    x / rms by e / rms and, through rms, by |x| / rms times the rms of e over
    rms; both are at most max(off) / rms (1 + max|x| / rms), the rotation adds
    two such terms, and fp32 under 2^-18 of the two values turned."""
    y = y.astype(np.float64)
    rms = np.sqrt((y * y).mean(-1, keepdims=True) + EPS)
    n = y / rms * w.astype(np.float64)
    c, s = (t[pos].astype(np.float64)[:, None] for t in (tables.cos, tables.sin))
    want = n.copy()
    a, b = n[..., 0:64:2], n[..., 1:64:2]
    want[..., 0:64:2], want[..., 1:64:2] = a * c - b * s, a * s + b * c
    top = np.abs(y).max(-1, keepdims=True) / rms
    slack = 2 * np.abs(w.astype(np.float64)).max() * (off.max(-1, keepdims=True) / rms * (1 + top) + top * FP32)
    assert (np.abs(got - want) <= _half_step(want) + slack).all()


def _check_step(cache, kr, vr, got, y, off, qw, kw, tables, pos, heads, kv, lengths, n_new, exact):
    T = len(pos)
    if exact:
        want = y.astype(np.float16)
        assert np.array_equal(got["g"], want[:, heads:2 * heads])
        assert np.array_equal(got["kv"].reshape(T, 2 * kv, D), want[:, 2 * heads:])
        rope = lambda x, w, n: orc.qknorm_rope_f32(  # noqa: E731
            x.reshape(-1, D), w, np.repeat(tables.cos[pos], n, 0), np.repeat(tables.sin[pos], n, 0)).reshape(T, n, D)
        assert np.array_equal(_bits(got["q"]), _bits(rope(y[:, :heads], qw, heads)))
        kn = rope(y[:, 2 * heads:2 * heads + kv], kw, kv)
    else:
        tol = _half_step(y) + off
        assert (np.abs(got["g"] - y[:, heads:2 * heads]) <= tol[:, heads:2 * heads]).all()
        assert (np.abs(got["kv"].reshape(T, 2 * kv, D) - y[:, 2 * heads:]) <= tol[:, 2 * heads:]).all()
        kn = None
        _check_rotated(got["q"], y[:, :heads], off[:, :heads], qw, tables, pos)
    o = 0
    for b, (L, n) in enumerate(zip(lengths, n_new)):
        krow, vrow = cache.gather(0, b, L + n)
        assert np.array_equal(_bits(krow[:L]), _bits(kr[0][b])) and np.array_equal(_bits(vrow[:L]), _bits(vr[0][b]))
        at = slice(o, o + n)
        if kn is not None:
            assert np.array_equal(_bits(krow[L:]), _bits(kn[at]))
        else:
            of = slice(2 * heads, 2 * heads + kv)
            _check_rotated(krow[L:], y[at, of], off[at, of], kw, tables, pos[at])
        assert np.array_equal(_bits(vrow[L:]), _bits(got["kv"][at, 1]))
        o += n


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv,hidden,n_new", [
    (2, 1, 512, [1]), (24, 4, 5120, [1] * 32), (6, 3, 1024, [3, 1, 5]), (8, 1, 1536, [31]), (4, 4, 512, [20, 21]),
    (24, 4, 512, [64]), (6, 1, 2560, [100, 81]), (2, 1, 512, [700]), (24, 4, 1024, [257, 1]), (8, 8, 512, [2048]),
    (24, 4, 512, [1000, 100]), (8, 4, 512, [2900])])  # the last two: more tiles than CUs
def test_project_exact(device, bits, heads, kv, hidden, n_new):
    rng = np.random.default_rng(heads + hidden + sum(n_new) + bits)
    lengths = [int(x) for x in rng.integers(0, 60, len(n_new))]
    say(f"mx_project_append exact {heads}/{kv} heads, hidden {hidden}, new {n_new}, {bits} bits")
    rope = [int(x) for x in rng.integers(0, 1024, sum(n_new))]
    r = _step(device, rng, heads, kv, hidden, lengths, n_new, bits, True, rope_pos=rope)
    _check_step(*r, heads, kv, lengths, n_new, True)
    r[0].destroy()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv,n_tok,hidden,tile,partial", [
    (2, 1, 45, 2048, (64, 128), 1), (2, 1, 45, 512, (64, 256), 0), (24, 4, 283, 512, (128, 256), 0),
    (16, 4, 813, 512, (256, 256), 0)])
def test_project_each_tile(device, bits, heads, kv, n_tok, hidden, tile, partial):
    rng = np.random.default_rng(n_tok + hidden + bits)
    say(f"mx_project_append tile {tile} partial={partial} {n_tok} tokens, hidden {hidden}, {bits} bits")
    r = _step(device, rng, heads, kv, hidden, [37], [n_tok], bits, True)
    plan = r[0].product_plan()
    assert (plan["tile_tokens"], plan["tile_rows"]) == tile and plan["partial"] == partial, plan
    _check_step(*r, heads, kv, [37], [n_tok], True)
    r[0].destroy()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_new", [[1], [9, 9], [70, 60]])
def test_project_random(device, bits, n_new):
    rng = np.random.default_rng(sum(n_new) + bits)
    lengths = [int(x) for x in rng.integers(0, 60, len(n_new))]
    say(f"mx_project_append random, new {n_new}, {bits} bits")
    r = _step(device, rng, 6, 1, 2560, lengths, n_new, bits, False)
    _check_step(*r, 6, 1, lengths, n_new, False)
    r[0].destroy()


@pytest.mark.parametrize("n_new", [[2, 1], [40], [300]])
def test_project_of_fp16_rows(device, n_new):
    """fp16 rows whose values 8 bits hold exactly."""
    rng = np.random.default_rng(sum(n_new))
    lengths = [5] * len(n_new)
    say(f"mx_project_append of fp16 rows, new {n_new}")
    r = _step(device, rng, 6, 1, 1024, lengths, n_new, 8, True, fp16=True)
    _check_step(*r, 6, 1, lengths, n_new, True)
    r[0].destroy()


@pytest.mark.parametrize("rotary_dim", [0, 8, 72, 256])
@pytest.mark.parametrize("n_tok,hidden", [(3, 512), (45, 2048), (45, 512)])
def test_project_rotary_dims(device, rotary_dim, n_tok, hidden):
    """Streamed, in parts of hidden and in one tile, the optional outputs left out."""
    rng = np.random.default_rng(rotary_dim + n_tok)
    heads, kv = 2, 1
    say(f"mx_project_append rotary_dim {rotary_dim}, {n_tok} tokens, hidden {hidden}")
    wq, wkv = (_exact_rows(rng, 2 * n * D, hidden, 4) for n in (heads, kv))
    x = _exact_rows(rng, n_tok, hidden, 8)
    qw, kw = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float16) for _ in "qk")
    angle = rng.uniform(0, 2 * np.pi, (64, rotary_dim // 2))
    cos, sin = np.cos(angle).astype(np.float16), np.sin(angle).astype(np.float16)
    tabs = [device.array(t if rotary_dim else np.zeros(8, np.float16)) for t in (cos, sin)]
    cache = PagedKVCache(n_layers=1, max_seqs=1, max_blocks=8, max_blocks_per_seq=8, max_step_tokens=64,
                         num_heads=heads, num_kv_heads=kv, rotary_dim=rotary_dim)
    cache.reserve(0, n_tok)
    cache.begin_step([0], [n_tok])
    q = device.empty((n_tok, heads, D), np.float16)
    cache.mx_project_append(0, device.array(x[0]), hidden, _pack(device, wq), _pack(device, wkv), device.array(qw),
                            device.array(kw), *tabs, 64, q, x_scales=device.array(x[1]))
    device.synchronize()
    y = mx.decode(*x, 8) @ np.concatenate([mx.decode(*wq, 4), mx.decode(*wkv, 4)]).T
    y = y.reshape(n_tok, -1, D)
    rope = lambda v, w, n: orc.qknorm_rope_f32(  # noqa: E731
        v.reshape(-1, D), w, np.repeat(cos[:n_tok], n, 0), np.repeat(sin[:n_tok], n, 0)).reshape(n_tok, n, D)
    assert np.array_equal(_bits(q.numpy()), _bits(rope(y[:, :heads], qw, heads)))
    k, v = cache.gather(0, 0, n_tok)
    assert np.array_equal(_bits(k), _bits(rope(y[:, 2 * heads:2 * heads + kv], kw, kv)))
    assert np.array_equal(v, y[:, 2 * heads + kv:].astype(np.float16))
    cache.destroy()


@pytest.mark.parametrize("n_new", [[1, 1], [33, 20]])
def test_project_onto_the_8_bit_cache(device, n_new):
    """The rows that an 8-bit cache holds are those of an append of the fp16 cache's."""
    rng = np.random.default_rng(sum(n_new))
    heads, kv, hidden, T, B = 6, 3, 1024, sum(n_new), len(n_new)
    say(f"mx_project_append onto an 8-bit cache, new {n_new}")
    wq, wkv = (_pack(device, _exact_rows(rng, 2 * n * D, hidden, 4)) for n in (heads, kv))
    x = [device.array(a) for a in _exact_rows(rng, T, hidden, 8)]
    qw, kw = (device.array((1 + 0.1 * rng.standard_normal(D)).astype(np.float16)) for _ in "qk")
    tables = Tables(device, 64)
    got = []
    for bits in (16, 8, 8):
        cache = PagedKVCache(n_layers=1, max_seqs=B, max_blocks=16, max_blocks_per_seq=8, max_step_tokens=64,
                             num_heads=heads, num_kv_heads=kv, kv_bits=bits)
        for b, n in enumerate(n_new):
            cache.reserve(b, n)
        cache.begin_step(list(range(B)), n_new)
        q = device.empty((T, heads, D), np.float16)
        k, v = device.empty((T, kv, D), np.float16), device.empty((T, kv, D), np.float16)
        if len(got) < 2:
            cache.mx_project_append(0, x[0], hidden, wq, wkv, qw, kw, tables.d_cos, tables.d_sin, 64, q, x_scales=x[1])
        else:  # the fp16 cache's rows, appended
            cache.append_rows(0, device.array(got[0][1]), device.array(got[0][2]))
        cache.read_rows(0, list(range(B)), [0] * B, n_new, k, v)
        device.synchronize()
        got.append((q.numpy(), k.numpy(), v.numpy()))
        cache.destroy()
    assert np.array_equal(_bits(got[1][0]), _bits(got[0][0]))
    assert np.array_equal(_bits(got[1][1]), _bits(got[2][1])) and np.array_equal(_bits(got[1][2]), _bits(got[2][2]))


# ---- together ---------------------------------------------------------------

class _Layer:
    """A layer as a program runs it: norm, projection, attention, output projection."""

    def __init__(self, device, rng, heads, kv, hidden, B, width):
        self.dev, self.heads, self.kv, self.hidden, self.B = device, heads, kv, hidden, B
        self.w = [_random_rows(rng, n * D, hidden, 4) for n in (2 * heads, 2 * kv)]
        self.w[0][1][:] -= 5
        self.w[1][1][:] -= 5
        self.wo = _random_rows(rng, hidden, heads * D, 4)
        self.wo[1][:] -= 6
        self.packed = [_pack(device, w) for w in self.w + [self.wo]]
        self.norm, self.qw, self.kw = ((1 + 0.1 * rng.standard_normal(n)).astype(np.float16) for n in (hidden, D, D))
        self.d_norm, self.d_qw, self.d_kw = (device.array(a) for a in (self.norm, self.qw, self.kw))
        self.tables = Tables(device, 1024)
        self.delta = device.empty((B, hidden), np.float16)
        self.h = device.empty((B, hidden), np.float16)
        self.codes, self.scales = device.empty((B, hidden), np.uint8), device.empty((B, hidden // 32), np.uint8)
        self.q, self.gate, self.attn = (device.empty((B, heads, D), np.float16) for _ in "qga")

    def run(self, cache, stream=None):
        H = self.hidden
        ms.add_rmsnorm(self.h, self.delta, self.d_norm, self.B, H, EPS, self.codes, sum_out=self.h, scales=self.scales,
                       bits=8, stream=stream)
        cache.mx_project_append(0, self.codes, H, *self.packed[:2], self.d_qw, self.d_kw, self.tables.d_cos,
                                self.tables.d_sin, self.tables.rows, self.q, self.gate, x_scales=self.scales,
                                stream=stream)
        cache.decode(0, self.q, self.attn, gate=self.gate, stream=stream)
        cache.mx_out_project(self.attn, self.B, self.heads * D, self.packed[2], H, self.h, residual=self.h,
                             stream=stream)


def test_a_layer(device):
    """The four calls one after another, each against the oracle on what the
    one before it left."""
    rng = np.random.default_rng(21)
    lengths = [3, 40, 17, 130, 0]
    B, heads, kv, hidden = len(lengths), 6, 1, 1024
    say("a decode step of a layer in 4 bits")
    ids, at = [], 0
    for n in lengths:
        ids.append(list(range(at, at + n // 16 + 1)))
        at += n // 16 + 1
    cache, kr, vr = build_cache(lengths, ids, extra_rows=[1] * B, rng=rng, num_heads=heads, num_kv_heads=kv)
    lay = _Layer(device, rng, heads, kv, hidden, B, 1)
    h = rng.standard_normal((B, hidden)).astype(np.float16)
    d = rng.standard_normal((B, hidden)).astype(np.float16)
    lay.h.copy_from(h)
    lay.delta.copy_from(d)
    cache.begin_step(list(range(B)), [1] * B)
    lay.run(cache)
    device.synchronize()
    total, want = mx.add_rmsnorm(h, d, lay.norm, EPS)
    codes, scales = lay.codes.numpy(), lay.scales.numpy()
    _check_norm(total, want, (codes, scales), 8)
    y, off = _product(mx.decode(codes, scales, 8), np.concatenate([mx.decode(*w, 4) for w in lay.w]))
    y, tol = y.reshape(B, -1, D), (_half_step(y) + off).reshape(B, -1, D)
    gate = lay.gate.numpy()
    assert (np.abs(gate - y[:, heads:2 * heads]) <= tol[:, heads:2 * heads]).all()
    attn = lay.attn.numpy()
    q = lay.q.numpy()
    for b, L in enumerate(lengths):
        k, v = cache.gather(0, b, L + 1)
        assert (np.abs(v[L] - y[b, 2 * heads + kv:]) <= tol[b, 2 * heads + kv:]).all()
        ref = orc.attention_fp32(q[b:b + 1], k, v)[0].astype(np.float64) / (1 + np.exp(-gate[b].astype(np.float64)))
        # Rows of any size, not N(0, 1): a probability's rounding to fp16 moves a
        # weighted mean of v by 2^-11 of the largest |v| at most, the output's
        # and the gated output's roundings by 2^-11 of themselves, and an output
        # is no larger than the largest |v|; as much as one again for the scores.
        assert max_err(attn[b], ref) <= 4 * 2.0 ** -11 * np.abs(v.astype(np.float64)).max()
    y, off = _product(mx.quantized(attn.reshape(B, -1), 8), mx.decode(*lay.wo, 4))
    y = y + total
    assert (np.abs(lay.h.numpy() - y) <= _half_step(y) + off).all()
    cache.destroy()


def test_a_recorded_layer(device):
    """A recorded layer replayed, its own eager runs between: the eager bits."""
    rng = np.random.default_rng(22)
    B, heads, kv, hidden = 4, 6, 1, 1024
    say("a recorded layer in 4 bits")
    lay = _Layer(device, rng, heads, kv, hidden, B, 1)
    caches = [PagedKVCache(n_layers=1, max_seqs=B, max_blocks=64, max_blocks_per_seq=16, max_step_tokens=64,
                           num_heads=heads, num_kv_heads=kv) for _ in range(2)]
    for c in caches:
        for b in range(B):
            c.reserve(b, 40)
    stream = Stream()
    s = stream.handle
    graph = None
    for step in range(6):
        h, d = (rng.standard_normal((B, hidden)).astype(np.float16) for _ in "hd")
        got = []
        for i, c in enumerate(caches):
            lay.h.copy_from(h)
            lay.delta.copy_from(d)
            device.synchronize()
            c.begin_step(list(range(B)), [1] * B, stream=s)
            if i == 0:
                lay.run(c, stream=s)
            else:
                if graph is None:
                    graph = c.record_step(s)
                    lay.run(c, stream=s)
                    graph.end()
                graph.launch()
            stream.synchronize()
            got.append([a.numpy() for a in (lay.h, lay.q, lay.gate, lay.attn)])
        for a, b in zip(*got):
            assert np.array_equal(_bits(a), _bits(b)), step
    graph.destroy()
    for c in caches:
        c.destroy()
    stream.destroy()


def test_two_caches_on_two_streams(device):
    """Calls on two caches that overlap in time: each has its own workspace."""
    rng = np.random.default_rng(23)
    n_tok, q_dim, n_out = 300, 1536, 1040
    say("mx_out_project on two streams at once")
    caches, streams = [_any_cache() for _ in range(2)], [Stream() for _ in range(2)]
    xs = [rng.integers(-4, 5, (n_tok, q_dim)).astype(np.float16) for _ in range(2)]
    ws = [_exact_rows(rng, n_out, q_dim, 4) for _ in range(2)]
    dx, packed = [device.array(x) for x in xs], [_pack(device, w) for w in ws]
    outs = [device.empty((n_tok, n_out), np.float16) for _ in range(2)]
    device.synchronize()
    for _ in range(8):
        for i in range(2):
            caches[i].mx_out_project(dx[i], n_tok, q_dim, packed[i], n_out, outs[i], stream=streams[i].handle)
    for st in streams:
        st.synchronize()
    for i in range(2):
        assert np.array_equal(outs[i].numpy(), (xs[i].astype(np.float64) @ mx.decode(*ws[i], 4).T).astype(np.float16))
        caches[i].destroy()
        streams[i].destroy()


def _tail(a, shape, dtype, end=0):
    """The last shape of values before `end` bytes of a device array's end."""
    n = int(np.prod(shape)) * np.dtype(dtype).itemsize
    return DeviceArray(a.dev, shape, dtype, ptr=a.ptr + a.nbytes - end - n)


def test_rows_far_apart(device):
    """Strides whose bytes pass 32 bits."""
    rng = np.random.default_rng(31)
    rows, cols, stride = 3, 96, 2 ** 31 + 8
    say(f"quantize {rows} rows {stride} values apart")
    x = rng.standard_normal((rows, cols)).astype(np.float16)
    big = device.empty((rows - 1) * stride + cols, np.float16)
    for r in range(rows):
        DeviceArray(device, cols, np.float16, ptr=big.ptr + 2 * r * stride).copy_from(x[r])
    codes, scales = device.empty((rows, cols), np.uint8), device.empty((rows, cols // 32), np.uint8)
    ms.quantize(big, rows, cols, 8, codes, scales, x_stride=stride)
    device.synchronize()
    code, b = mx.encode(x, 8)
    assert np.array_equal(codes.numpy(), code) and np.array_equal(scales.numpy(), b)
    big.free()


def test_more_than_32_bits_of_values(device):
    """The last rows of 2^32 values and more: norm, quantise, and back."""
    rng = np.random.default_rng(32)
    cols, n = 2048, 2 ** 21 + 5
    say(f"{n} rows of {cols}")
    last = rng.standard_normal((5, cols)).astype(np.float16)
    w = rng.uniform(0.5, 1.5, cols).astype(np.float16)
    x = device.empty((n, cols), np.float16)
    x.zero()
    _tail(x, last.shape, np.float16).copy_from(last)
    codes, scales = device.empty((n, cols), np.uint8), device.empty((n, cols // 32), np.uint8)
    ms.quantize(x, n, cols, 8, codes, scales)
    device.synchronize()
    code, b = mx.encode(last, 8)
    got, got_b = _tail(codes, (6, cols), np.uint8).numpy(), _tail(scales, (6, cols // 32), np.uint8).numpy()
    assert np.array_equal(got[1:], code) and np.array_equal(got_b[1:], b)
    assert not got[0].any()
    ms.add_rmsnorm(x, None, device.array(w), n, cols, 1e-6, codes, scales=scales, bits=8)
    device.synchronize()
    norm = _tail(codes, (6, cols), np.uint8).numpy(), _tail(scales, (6, cols // 32), np.uint8).numpy()
    few = device.empty((5, cols), np.uint8), device.empty((5, cols // 32), np.uint8)
    ms.add_rmsnorm(device.array(last), None, device.array(w), 5, cols, 1e-6, few[0], scales=few[1], bits=8)
    device.synchronize()
    assert np.array_equal(norm[0][1:], few[0].numpy()) and np.array_equal(norm[1][1:], few[1].numpy())
    assert not norm[0][0].any()
    ms.dequantize(codes, scales, n, cols, 8, x)
    device.synchronize()
    y = _tail(x, (6, cols), np.float16).numpy()
    assert np.array_equal(y, mx.decode(*norm, 8).astype(np.float16))
    for a in (x, codes, scales):
        a.free()


def test_out_project_of_more_than_32_bits_of_codes(device):
    """2^23 tokens and 5 more of 512: 4 GB of codes."""
    rng = np.random.default_rng(33)
    n, q_dim, n_out = 2 ** 23 + 5, 512, 16
    say(f"mx_out_project of {n} rows")
    cache = _any_cache()
    codes, scales = device.empty((n, q_dim), np.uint8), device.empty((n, q_dim // 32), np.uint8)
    codes.zero()
    scales.zero()
    c, s = _exact_rows(rng, 5, q_dim, 8)
    _tail(codes, c.shape, np.uint8).copy_from(c)
    _tail(scales, s.shape, np.uint8).copy_from(s)
    w = _exact_rows(rng, n_out, q_dim, 4)
    out = device.empty((n, n_out), np.float16)
    cache.mx_out_project(codes, n, q_dim, _pack(device, w), n_out, out, attn_scales=scales)
    device.synchronize()
    y = _tail(out, (6, n_out), np.float16).numpy()
    assert np.array_equal(y[1:], (mx.decode(c, s, 8) @ mx.decode(*w, 4).T).astype(np.float16))
    assert not y[0].any()
    for a in (codes, scales, out):
        a.free()
    cache.destroy()


# ---- which path ran -----------------------------------------------------------

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_tok,hidden,path", [(1, 512, "kernels"), (32, 512, "kernels"), (33, 512, "prefill_gemm"),
                                               (45, 2048, "prefill_gemm"), (64, 512, "prefill_gemm"),
                                               (65, 512, "prefill_gemm")])
def test_project_path(device, bits, n_tok, hidden, path):
    """Streamed weights up to 32 tokens, tiles above, whether a finish kernel follows them or not."""
    say(f"project_path of {n_tok} tokens by 4-bit weights, hidden {hidden}, {bits} bits")
    rng, heads, kv = np.random.default_rng(n_tok), 2, 1
    cache = PagedKVCache(n_layers=1, max_seqs=1, max_blocks=8, max_blocks_per_seq=8, max_step_tokens=n_tok,
                         num_heads=heads, num_kv_heads=kv)
    cache.reserve(0, n_tok)
    wq, wkv = (_pack(device, _exact_rows(rng, 2 * n * D, hidden, 4)) for n in (heads, kv))
    tables, norm = Tables(device, n_tok), device.array(np.ones(D, np.float16))
    x = [device.array(a) for a in _exact_rows(rng, n_tok, hidden, bits)]
    cache.begin_step([0], [n_tok])
    cache.mx_project_append(0, x[0], hidden, wq, wkv, norm, norm, tables.d_cos, tables.d_sin, tables.rows,
                            device.empty((n_tok, heads, D), np.float16), x_scales=x[1], bits=bits)
    device.synchronize()
    assert cache.project_path() == path
    assert (cache.product_plan()["tile_tokens"] == 0) == (path == "kernels")
    cache.destroy()


# ---- fp16 rows into the projection, recorded steps of many tokens --------------

@pytest.mark.parametrize("n_new", [[2, 1], [40], [300]])
def test_project_of_fp16_rows_to_4_bits(device, n_new):
    """fp16 rows whose values 4 bits hold exactly."""
    rng = np.random.default_rng(sum(n_new) + 4)
    lengths = [5] * len(n_new)
    say(f"mx_project_append of fp16 rows to 4 bits, new {n_new}")
    r = _step(device, rng, 6, 1, 1024, lengths, n_new, 4, True, fp16=True)
    _check_step(*r, 6, 1, lengths, n_new, True)
    r[0].destroy()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_new", [[500, 295], [771], [398]])
def test_project_of_fp16_rows_in_parts(device, bits, n_new):
    """More fp16 rows than a launch takes: half of the workspace, 2 MB for one
    query and one KV head, holds 397 rows of 5280 bytes in 8 bits and 770 of 2720
    in 4.  Some end with a launch of 1 to 32 tokens, which streams the weights."""
    rng = np.random.default_rng(sum(n_new) + bits)
    lengths = [int(x) for x in rng.integers(0, 60, len(n_new))]
    say(f"mx_project_append of fp16 rows in parts, new {n_new}, {bits} bits")
    rope = [int(x) for x in rng.integers(0, 1024, sum(n_new))]
    r = _step(device, rng, 1, 1, 5120, lengths, n_new, bits, True, fp16=True, rope_pos=rope)
    _check_step(*r, 1, 1, lengths, n_new, True)
    r[0].destroy()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_new", [[2, 1], [33, 20], [500, 295]])
def test_project_of_fp16_rows_onto_the_8_bit_cache(device, bits, n_new):
    """In one launch and in parts: what the cache holds is an append of the fp16
    cache's rows, and every output the same."""
    rng = np.random.default_rng(sum(n_new) + bits)
    heads, kv, hidden, T, B = 1, 1, 5120, sum(n_new), len(n_new)
    say(f"mx_project_append of fp16 rows onto an 8-bit cache, new {n_new}, {bits} bits")
    wq, wkv = (_pack(device, _exact_rows(rng, 2 * n * D, hidden, 4)) for n in (heads, kv))
    x = device.array(rng.integers(-4, 5, (T, hidden)).astype(np.float16))
    qw, kw = (device.array((1 + 0.1 * rng.standard_normal(D)).astype(np.float16)) for _ in "qk")
    tables = Tables(device, 512)
    got = []
    for kv_bits in (16, 8, 8):
        cache = PagedKVCache(n_layers=1, max_seqs=B, max_blocks=64, max_blocks_per_seq=32, max_step_tokens=1024,
                             num_heads=heads, num_kv_heads=kv, kv_bits=kv_bits)
        for b, n in enumerate(n_new):
            cache.reserve(b, n)
        cache.begin_step(list(range(B)), n_new)
        out = [device.empty((T, n, D), np.float16) for n in (heads, heads, 2 * kv)]
        k, v = device.empty((T, kv, D), np.float16), device.empty((T, kv, D), np.float16)
        if len(got) < 2:
            cache.mx_project_append(0, x, hidden, wq, wkv, qw, kw, tables.d_cos, tables.d_sin, 512, *out, bits=bits)
        else:  # the fp16 cache's rows, appended
            cache.append_rows(0, device.array(got[0][3]), device.array(got[0][4]))
        cache.read_rows(0, list(range(B)), [0] * B, n_new, k, v)
        device.synchronize()
        got.append([a.numpy() for a in out + [k, v]])
        cache.destroy()
    for i in range(3):
        assert np.array_equal(_bits(got[1][i]), _bits(got[0][i]))
    for i in (3, 4):
        assert np.array_equal(_bits(got[1][i]), _bits(got[2][i]))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n_tok", [1, 9, 32, 45, 300])
def test_project_of_random_fp16_rows(device, bits, n_tok):
    """Rows that are rounded on the way: the product of what they are rounded
    to, as test_project_random checks coded ones."""
    rng = np.random.default_rng(n_tok + bits)
    heads, kv, hidden = 3, 1, 2560
    say(f"mx_project_append of random fp16 rows, {n_tok} tokens, {bits} bits")
    cache, kr, vr = build_cache([7], [list(range(n_tok // 16 + 2))], extra_rows=[n_tok], rng=rng, num_heads=heads,
                                num_kv_heads=kv)
    x = (rng.standard_normal((n_tok, hidden)) * 2.0 ** rng.integers(-3, 3, (n_tok, 1))).astype(np.float16)
    x[:, ::97] *= 10
    wq, wkv = _random_rows(rng, 2 * heads * D, hidden, 4), _random_rows(rng, 2 * kv * D, hidden, 4)
    qw, kw = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float16) for _ in "qk")
    tables = Tables(device, 1024)
    cache.begin_step([0], [n_tok])
    d = dict(q=device.empty((n_tok, heads, D), np.float16), g=device.empty((n_tok, heads, D), np.float16),
             kv=device.empty((n_tok, 2, kv, D), np.float16))
    cache.mx_project_append(0, device.array(x), hidden, _pack(device, wq), _pack(device, wkv), device.array(qw),
                            device.array(kw), tables.d_cos, tables.d_sin, tables.rows, *d.values(), bits=bits)
    device.synchronize()
    got = {k: v.numpy() for k, v in d.items()}
    y, off = _product(mx.quantized(x, bits), np.concatenate([mx.decode(*wq, 4), mx.decode(*wkv, 4)]))
    _check_step(cache, kr, vr, got, y.reshape(n_tok, -1, D), off.reshape(n_tok, -1, D), qw, kw, tables,
                list(range(7, 7 + n_tok)), heads, kv, [7], [n_tok], False)
    cache.destroy()


@pytest.mark.parametrize("coded", [True, False])
@pytest.mark.parametrize("heads,kv,hidden,n_new", [(2, 1, 512, [25, 20]), (2, 1, 2048, [25, 20]), (1, 1, 5120, [410])])
def test_a_recorded_prompt_step(device, heads, kv, hidden, n_new, coded):
    """Norm, projection and output projection (of the gates) of more than 32
    tokens, recorded and replayed, its own eager runs between: the eager bits.
    Tiles that finish their rows, parts of hidden with a finish kernel, and (fp16
    rows of 5120) more than one launch."""
    rng = np.random.default_rng(hidden + coded)
    B, T, steps = len(n_new), sum(n_new), 5
    say(f"a recorded step of {n_new} tokens in 4 bits, {heads}/{kv} heads, hidden {hidden}, coded {coded}")
    w = [_random_rows(rng, n * D, hidden, 4) for n in (2 * heads, 2 * kv)]
    w.append(_random_rows(rng, hidden, 512, 4))
    for a in w:
        a[1][:] -= 6
    packed = [_pack(device, a) for a in w]
    norm, qw, kw = (device.array((1 + 0.1 * rng.standard_normal(n)).astype(np.float16)) for n in (hidden, D, D))
    tables = Tables(device, 4096)
    empty = lambda *s, t=np.float16: device.empty(s, t)  # noqa: E731
    h, delta, x, gate, q = empty(T, hidden), empty(T, hidden), empty(T, hidden), empty(T, heads, D), empty(T, heads, D)
    codes, scales = empty(T, hidden, t=np.uint8), empty(T, hidden // 32, t=np.uint8)
    n_rows = T * heads * D // 512  # the gates as rows of 512
    caches = [PagedKVCache(n_layers=1, max_seqs=B, max_blocks=256, max_blocks_per_seq=160, max_step_tokens=512,
                           num_heads=heads, num_kv_heads=kv) for _ in range(2)]
    for c in caches:
        for b in range(B):
            c.reserve(b, steps * n_new[b])

    def run(cache, s):
        if coded:
            ms.add_rmsnorm(h, delta, norm, T, hidden, EPS, codes, sum_out=h, scales=scales, bits=8, stream=s)
            cache.mx_project_append(0, codes, hidden, *packed[:2], qw, kw, tables.d_cos, tables.d_sin, tables.rows, q,
                                    gate, x_scales=scales, stream=s)
        else:
            ms.add_rmsnorm(h, delta, norm, T, hidden, EPS, x, sum_out=h, stream=s)
            cache.mx_project_append(0, x, hidden, *packed[:2], qw, kw, tables.d_cos, tables.d_sin, tables.rows, q,
                                    gate, stream=s)
        cache.mx_out_project(gate, n_rows, 512, packed[2], hidden, h, residual=h, stream=s)

    stream = Stream()
    s = stream.handle
    graph = None
    for step in range(steps):
        h0, d0 = (rng.standard_normal((T, hidden)).astype(np.float16) for _ in "hd")
        got = []
        for i, c in enumerate(caches):
            h.copy_from(h0)
            delta.copy_from(d0)
            q.zero()
            gate.zero()
            device.synchronize()
            c.begin_step(list(range(B)), n_new, stream=s)
            if i == 0:
                run(c, s)
            else:
                if graph is None:
                    graph = c.record_step(s)
                    run(c, s)
                    graph.end()
                graph.launch()
            stream.synchronize()
            got.append([a.numpy() for a in (h, q, gate)])
        for a, b in zip(*got):
            assert np.isfinite(a).all() and a.any()
            assert np.array_equal(_bits(a), _bits(b)), step
    for b in range(B):
        for a, g in zip(*(c.gather(0, b, steps * n_new[b]) for c in caches)):
            assert np.array_equal(_bits(a), _bits(g))
    graph.destroy()
    for c in caches:
        c.destroy()
    stream.destroy()
