"""The oracle of microscaled rows, pinned: element lists against torch's own
8-bit type and against the 4-bit format's definition, the scale rule at its
borders, rounding at every tie, the packed order by a brute-force walk."""
import numpy as np
import pytest
import torch

from oracle import microscale_oracle as mx


def test_elements_are_the_formats_values():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).to(torch.float64).numpy()
    got = mx.decode(codes.reshape(8, 32), np.full((8, 1), 127, np.uint8), 8).reshape(-1)
    assert np.array_equal(got, want, equal_nan=True)
    for c in range(16):  # sign, two exponent bits of bias 1, one mantissa bit
        e, m = c >> 1 & 3, c & 1
        v = (1 + m / 2) * 2.0 ** (e - 1) if e else m * 0.5
        got = mx.decode(np.full((1, 16), c | c << 4, np.uint8), np.array([[127]], np.uint8), 4)
        assert np.array_equal(got, np.full((1, 32), -v if c & 8 else v)), c


@pytest.mark.parametrize("bits,most", [(8, 448.0), (4, 6.0)])
def test_scale_is_the_smallest_that_covers(bits, most):
    for e in (-126, -30, -1, 0, 5, 40):
        x = np.zeros((3, 32))
        x[0, 3], x[1, 31], x[2, 0] = most * 2.0 ** e, -np.nextafter(most * 2.0 ** e, np.inf), most * 2.0 ** (e - 1)
        got = mx.scale_bytes(x, bits)[:, 0].astype(int) - 127
        assert list(got) == [e, e + 1, max(e - 1, -126)], e
    assert mx.scale_bytes(np.zeros((1, 64)), bits).tolist() == [[1, 1]]
    x = np.zeros((1, 96))
    x[0, 5], x[0, 70] = np.inf, np.nan
    assert mx.scale_bytes(x, bits).tolist() == [[255, 1, 255]]
    assert not mx.encode(x, bits)[0].any()
    assert np.isnan(mx.quantized(x, bits)).reshape(3, 32).all(1).tolist() == [True, False, True]


@pytest.mark.parametrize("bits", [8, 4])
def test_elements_round_to_the_nearest_even(bits):
    grid = mx.GRID[bits]
    for i in range(len(grid) - 1):
        tie = (grid[i] + grid[i + 1]) / 2
        x = np.zeros((1, 32))
        x[0, :7] = [grid[-1], grid[i], tie, np.nextafter(tie, 0), np.nextafter(tie, 1e9), -tie, -grid[i + 1]]
        even = i if i % 2 == 0 else i + 1
        neg = 1 << (bits - 1)
        assert mx.encode(x, bits)[0][0, :7].tolist() == \
            [len(grid) - 1, i, even, i, i + 1, even + neg, i + 1 + neg], i


def test_eight_bits_agree_with_torch():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 128)) * 2.0 ** rng.integers(-9, 9, (64, 1))).astype(np.float16)
    code, b = mx.encode(x, 8)
    s = np.repeat(2.0 ** (b.astype(float) - 127), 32, axis=1)
    want = torch.from_numpy((x / s).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(code, want)


def test_a_second_quantisation_changes_nothing():
    rng = np.random.default_rng(2)
    for bits in (8, 4):
        y = mx.quantized(rng.standard_normal((16, 256)), bits)
        assert np.array_equal(mx.quantized(y, bits), y)


def test_packed_order():
    rng = np.random.default_rng(3)
    rows, cols = 45, 512
    codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, cols // 32), dtype=np.uint8)
    p = mx.pack_weights(codes, scales)
    assert p.size == 64 * (cols // 2 + cols // 32)
    base = 64 * cols // 2
    for row in (0, 31, 32, 44, 45, 63):
        for k in (0, 31, 32, 64, 200, 255, 256, 511):
            tile, lane, step = row // 32, row % 32 + 32 * (k // 32 % 2), k // 64
            got = p[(tile * (cols // 64) + step) * 1024 + 16 * lane + k % 32 // 2]
            assert got == (codes[row, k // 2] if row < rows else 0), (row, k)
            got = p[base + (tile * (cols // 256) + k // 256) * 256 + 4 * lane + k // 64 % 4]
            assert got == (scales[row, k // 32] if row < rows else 1), (row, k)


def test_norm_closed_forms():
    h = np.full((2, 64), 3.0, np.float16)
    w = np.linspace(0.5, 2.0, 64).astype(np.float16)
    total, x = mx.add_rmsnorm(h, None, w, 0.0)
    assert np.array_equal(total, h) and np.allclose(x, w.astype(float), rtol=1e-15)
    total, x = mx.add_rmsnorm(h, -h, w, 1e-6)
    assert not total.any() and not x.any()
    # the sum is rounded once: 2049 is a tie that the small term decides
    total, _ = mx.add_rmsnorm(np.full((1, 32), 2048, np.float16), np.full((1, 32), 1 + 2.0 ** -10, np.float16),
                              np.ones(32, np.float16), 0.0)
    assert (total == 2050).all()
