"""Shared by the tests of the 8-bit cache: rows, a cache that holds them, and
what it stands for."""
from __future__ import annotations

import numpy as np

from mi50grad_amd.kv_cache import PagedKVCache

D = 256


def rows(rng, n, kv, size=1.0):
    """K and V rows [n, kv, D]: strong channels in K, heads of unlike size in V."""
    k = rng.standard_normal((n, kv, D), dtype=np.float32)
    k[..., rng.permutation(D)[:5]] *= 4
    v = rng.standard_normal((n, kv, D), dtype=np.float32) * rng.uniform(0.1, 3.0, (1, kv, 1)).astype(np.float32)
    return (k * size).astype(np.float16), (v * size).astype(np.float16)


def make(lens, heads=24, kv=4, layers=1, bits=8, extra=0, step=8192, spare=0, slots=None):
    """A cache with a permuted block list per sequence, room for `extra` rows
    behind each length."""
    need = [(n + extra + 15) // 16 for n in lens]
    cache = PagedKVCache(n_layers=layers, max_seqs=slots or len(lens), max_blocks=max(1, sum(need)) + spare,
                         max_blocks_per_seq=max(1, max(need)), max_step_tokens=step, num_heads=heads,
                         num_kv_heads=kv, kv_bits=bits)
    ids = np.random.default_rng(sum(need)).permutation(sum(need))
    o = 0
    for b, n in enumerate(need):
        cache.set_blocks(b, ids[o:o + n])
        o += n
    return cache


def put(device, cache, seqs, ks, vs, layer=0, stream=None):
    """One step that appends ks[i], vs[i] to seqs[i] (layer 0 begins the step)."""
    if layer == 0:
        cache.begin_step(seqs, [len(k) for k in ks], stream=stream)
    if sum(len(k) for k in ks):
        cache.append_rows(layer, device.array(np.concatenate(ks)), device.array(np.concatenate(vs)), stream=stream)


def held(device, cache, seqs, first=None, count=None, layer=0):
    """What the cache holds of those rows, [sum, kv, D] each."""
    first = [0] * len(seqs) if first is None else first
    count = [cache.seq_len(s) - f for s, f in zip(seqs, first)] if count is None else count
    n = max(1, sum(count))
    out = [device.empty((n, cache.num_kv_heads, D), np.float16) for _ in range(2)]
    for o in out:
        o.copy_from(np.full(o.shape, 7.0, np.float16))
    cache.read_rows(layer, seqs, first, count, *out)
    device.synchronize()
    return [o.numpy()[:sum(count)] for o in out]


def same_bits(a, b):
    """Equal values; NaN equals NaN, and zeros of either sign."""
    return np.array_equal(np.asarray(a, np.float64), np.asarray(b, np.float64), equal_nan=True)


def within(got, want, tol):
    got = np.asarray(got, np.float64)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), "NaN in other places"
    off = np.abs(np.where(nan, 0.0, got - want)) - np.where(nan, 1.0, tol)
    assert (off <= 0).all(), f"{(off > 0).sum()} values off, by up to {np.nanmax(np.abs(got - want)):.3e}"
