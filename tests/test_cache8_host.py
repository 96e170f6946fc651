"""The 8-bit cache without a GPU: its oracle against exact arithmetic, and what
its calls refuse (a host-only cache reports every refusal)."""
from fractions import Fraction

import numpy as np
import pytest

from mi50grad_amd._lib import LIB_PATH, KvaError
from mi50grad_amd.kv_cache import PagedKVCache
from oracle import kvattn_oracle as orc

UNSUPPORTED, STATE, INVALID, NO_DEVICE, MISALIGNED, BAD_SEQ = -2, -8, -1, -3, -10, -6


def make(**kw):
    args = dict(n_layers=2, max_seqs=4, max_blocks=20, max_blocks_per_seq=8, max_step_tokens=64, host_only=True,
                kv_bits=8)
    args.update(kw)
    return PagedKVCache(**args)


def refused(code, call, *args, **kw):
    with pytest.raises(KvaError) as e:
        call(*args, **kw)
    assert e.value.code == code, e.value


def test_scale_is_the_smallest_of_its_kind():
    scales = sorted(m * 2.0 ** e for m in range(8, 16) for e in range(-24, 6)) + [512.0]
    rng = np.random.default_rng(0)
    tops = np.concatenate([[0.0, 2.0 ** -24, 65504.0, 65024.0, 1.0], np.exp(rng.uniform(-16, 11, 300))])
    for top in tops.astype(np.float16).astype(np.float64):
        want = next((s for s in scales if Fraction(127) * Fraction(s) >= Fraction(top)), 512.0)
        assert orc.int8_scale(top) == want


def test_values_are_fp16_numbers():
    """Codes of every scale times the scale: exact in fp16."""
    codes = np.arange(-127, 128, dtype=np.float64)
    for e in range(-24, 7):
        for m in range(8, 16):
            s = m * 2.0 ** e
            if s <= 512:
                assert np.array_equal((codes * s).astype(np.float16).astype(np.float64), codes * s)


def test_codes_do_not_depend_on_the_arithmetic():
    """x / s in float32 rounds to the code that exact arithmetic gives, for
    every fp16 magnitude of some binades and every significand of s."""
    for m in range(8, 16):
        s = m * 2.0 ** -9
        x = np.arange(0x0001, 0x7c00, dtype=np.uint16).view(np.float16)
        x = x[x.astype(np.float64) <= 127 * s]
        got = np.rint(x.astype(np.float32) / np.float32(s)).astype(int)
        num = [Fraction(float(v)) / Fraction(s) for v in x]
        want = [int(n) + (1 if n - int(n) > Fraction(1, 2) or (n - int(n) == Fraction(1, 2) and int(n) % 2) else 0)
                for n in num]
        assert np.array_equal(got, want)


def test_full_pages_only_are_rounded():
    rng = np.random.default_rng(1)
    k, v = [rng.standard_normal((20, 2, 256)).astype(np.float16) for _ in range(2)]
    gk, gv = orc.int8_rows(k, v)
    assert np.array_equal(gk[16:], k[16:]) and np.array_equal(gv[16:], v[16:])
    assert not np.array_equal(gk[:16], k[:16])
    assert np.array_equal(orc.int8_rows(k[:15], v[:15])[0], k[:15])


def test_attention_bound_is_attention():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((3, 6, 256)), rng.standard_normal((20, 2, 256)), rng.standard_normal((20, 2, 256))
    seen = orc.chunk_visibility(17, 3)
    out, tol = orc.attention_bound(q, k, v, seen)
    want = orc.attention_fp32(q.astype(np.float32), k, v, seen)
    assert np.abs(out - want).max() < 1e-5 and (tol > 0).all() and tol.max() < 5e-3


def test_addresses_and_moves_are_refused():
    c = make()
    c.reserve(0, 32)
    refused(NO_DEVICE, c.layer_pools, 0)
    refused(UNSUPPORTED, c.begin_step, [0], [2], tree_bits=[1, 3])
    c.begin_step([0], [20])
    refused(UNSUPPORTED, c.tree_verify, 0, 16, 16)
    refused(UNSUPPORTED, c.rollback, [0], [4], [[0, 2]])
    assert c.seq_len(0) == 20
    c.rollback([0], [4], [[0, 1, 2]])  # a prefix moves nothing
    assert c.seq_len(0) == 7


def test_length_goes_up_only_to_rows_written():
    c = make()
    c.reserve(0, 100)
    refused(STATE, c.set_len, 0, 1)
    c.begin_step([0], [40])
    c.set_len(0, 10)
    c.set_len(0, 40)
    c.set_len(0, 20)
    c.begin_step([0], [1])
    refused(STATE, c.set_len, 0, 22)
    c.free_seq(0)
    c.reserve(0, 100)
    refused(STATE, c.set_len, 0, 1)


def test_rows_go_with_their_blocks():
    """Rows behind the length whose page gets another block, or none, were not
    written any more."""
    c = make()
    c.set_blocks(0, [5, 6, 7])
    c.begin_step([0], [40])
    c.set_len(0, 10)
    c.set_blocks(0, [5, 6, 8])
    refused(STATE, c.set_len, 0, 33)
    c.set_len(0, 32)
    c.set_len(0, 10)
    c.set_blocks(0, [5])
    c.reserve(0, 100)
    refused(STATE, c.set_len, 0, 17)
    c.set_len(0, 16)
    c.set_len(0, 10)
    c.set_blocks(0, [9, 6])
    refused(STATE, c.set_len, 0, 11)


def test_a_step_without_rows_leaves_the_sequence():
    c = make()
    c.begin_step([0], [40])
    c.set_len(0, 20)
    c.begin_step([0, 1], [0, 3])
    c.set_len(0, 40)
    assert c.seq_len(0) == 40


@pytest.mark.parametrize("bits", [8, 16])
def test_append_rows_and_read_rows_refuse(bits):
    c = make(kv_bits=bits)
    refused(STATE, c.append_rows, 0, 16, 16)
    c.begin_step([1, 2], [3, 0])
    refused(INVALID, c.append_rows, 2, 16, 16)
    refused(INVALID, c.append_rows, 0, None, 16)
    refused(MISALIGNED, c.append_rows, 0, 16, 24)
    refused(NO_DEVICE, c.append_rows, 0, 16, 16)
    refused(BAD_SEQ, c.read_rows, 0, [4], [0], [0], 16, 16)
    refused(INVALID, c.read_rows, 0, [1], [1], [3], 16, 16)
    refused(INVALID, c.read_rows, 0, [1], [-1], [1], 16, 16)
    refused(INVALID, c.read_rows, 0, [1], [0], [-1], 16, 16)
    refused(INVALID, c.read_rows, -1, [1], [0], [1], 16, 16)
    refused(INVALID, c.read_rows, 0, [1], [0], [1], None, 16)
    refused(MISALIGNED, c.read_rows, 0, [1], [0], [1], 16, 20)
    refused(NO_DEVICE, c.read_rows, 0, [1], [0], [3], 16, 16)
    with pytest.raises(ValueError):
        c.read_rows(0, [1, 2], [0], [1], 16, 16)


def test_kinds_of_cache():
    with pytest.raises(ValueError):
        make(kv_bits=4)
    assert make().row_bytes * 2 == make(kv_bits=16).row_bytes


@pytest.mark.parametrize("bits", [8, 16])
def test_attn_weights_refuses(bits):
    c = make(kv_bits=bits)
    ok = (0, 16, 16, 100)
    refused(STATE, c.attn_weights, *ok)
    c.begin_step([1, 2], [30, 5])
    refused(NO_DEVICE, c.attn_weights, *ok, n_obs=32)
    refused(INVALID, c.attn_weights, 2, 16, 16, 100)
    refused(INVALID, c.attn_weights, 0, None, 16, 100)
    refused(INVALID, c.attn_weights, 0, 16, None, 100)
    refused(MISALIGNED, c.attn_weights, 0, 24, 16, 100)
    refused(MISALIGNED, c.attn_weights, 0, 16, 18, 100)
    refused(INVALID, c.attn_weights, 0, 16, 16, 29)
    for n in (0, -1, 33):
        refused(UNSUPPORTED, c.attn_weights, *ok, n_obs=n)
    for d in (float("nan"), float("inf")):
        refused(INVALID, c.attn_weights, *ok, decay=d)
    if bits == 16:
        c.begin_step([3], [1], tree_bits=[1])
        refused(STATE, c.attn_weights, *ok)


def long_ones(pages, heads, kv, obs):
    """Sequences of `pages` full pages less the obs rows of the next step."""
    c = make(n_layers=1, max_seqs=len(pages), max_blocks=sum(pages), max_blocks_per_seq=max(pages),
             max_step_tokens=16 * sum(pages), num_heads=heads, num_kv_heads=kv)
    c.begin_step(list(range(len(pages))), [16 * p - obs for p in pages])
    return c


@pytest.mark.parametrize("heads,kv,obs,slots", [(24, 4, 1, 192), (24, 4, 32, 64), (8, 8, 1, 96), (8, 8, 32, 96),
                                                (8, 1, 32, 256)])
@pytest.mark.parametrize("long,short", [(1000, 32), (2048, 10), (2000, 2), (47, 47)])
def test_weights_share_out_a_long_sequence(heads, kv, obs, slots, long, short):
    """A long sequence beside short ones, fewer, as many and more than there are
    workgroups at once: no chunk is longer than about two even shares of the
    rounds that the sequences make, and a workgroup's start (24 pages)."""
    for n_short in (1, slots // 2, slots - 2, slots - 1, slots, 2 * slots, 3 * slots):
        pages = [short] * n_short + [long]
        c = long_ones(pages, heads, kv, obs)
        c.begin_step(list(range(len(pages))), [obs] * len(pages))
        refused(NO_DEVICE, c.attn_weights, 0, 16, 16, 16 * long, n_obs=obs)
        chunk, n = c.weights_plan()
        assert n == sum(-(-p // chunk) for p in pages)
        rounds = -(-len(pages) // slots)
        share = -(-sum(pages) // (rounds * slots))
        assert min(chunk, long) <= 2 * max(share, 4) + 24, (n_short, chunk)


def test_evict_refuses():
    c = make()
    c.begin_step([0, 1], [40, 20])
    big = 1 << 20
    ok = dict(weights=16, w_stride=40, kept=big, kept_stride=20)
    call = lambda ids, keep, **kw: refused(kw.pop("code"), c.evict, ids, keep, **{**ok, **kw})  # noqa: E731
    call([0, 1], [20, 20], code=NO_DEVICE)
    call([0, 4], [20, 20], code=BAD_SEQ)
    call([0, 0], [20, 20], code=INVALID)
    call([0], [-1], code=INVALID)
    call([0], [10], first=4, recent=7, code=INVALID)
    call([0], [10], first=-1, code=INVALID)
    call([0], [10], recent=-1, code=INVALID)
    call([0, 1], [20, 20], dst_ids=[1, 0], code=INVALID)  # another's source
    call([0, 1], [20, 20], dst_ids=[2, 2], code=INVALID)
    call([0, 1], [20, 20], dst_ids=[2, 9], code=BAD_SEQ)
    call([0], [20], weights=None, code=INVALID)
    call([0], [20], kept=None, code=INVALID)
    call([0], [20], kept=big + 2, code=MISALIGNED)
    call([0], [20], w_stride=39, code=INVALID)
    call([0], [20], kept_stride=19, code=INVALID)
    call([0], [20], weights_out=16, code=INVALID)
    call([0], [20], kept=32, code=INVALID)
    with pytest.raises(ValueError):
        c.evict([0, 1], [20], **ok)
    assert c.seq_len(0) == 40 and c.seq_len(1) == 20
    tight = make(max_blocks=6, max_step_tokens=128)
    tight.begin_step([0, 1], [40, 40])
    refused(-4, tight.evict, [0], [20], **ok)
    refused(NO_DEVICE, tight.evict, [0, 1], [40, 40], 16, 40, big, 40)


def test_evict_does_not_depend_on_the_order_listed():
    """A sequence that finds its blocks free gives up more of them than it takes."""
    big = 1 << 20
    args = dict(weights=16, w_stride=64, kept=big, kept_stride=40)
    for seqs, keep in (([0, 1], [40, 20]), ([1, 0], [20, 40])):
        c = make(max_blocks=10, max_step_tokens=128)
        c.begin_step([0, 1], [64, 64])  # two blocks are free
        refused(NO_DEVICE, c.evict, seqs, keep, **args)
        refused(-4, c.evict, seqs, [40, 40], **args)
    for seqs, keep, dst in (([0, 1], [20, 10], [0, 2]), ([1, 0], [10, 20], [2, 0])):
        c = make(max_blocks=12, max_step_tokens=192)
        c.begin_step([0, 1, 2], [64, 64, 48])  # one is free, and the copy takes two fewer than sequence 2 holds
        refused(NO_DEVICE, c.evict, seqs, keep, dst_ids=dst, **args)
        refused(-4, c.evict, [0], [20], **args)
        c.begin_step([1], [1])  # none is free
        refused(-4, c.evict, seqs, [k + 16 for k in keep], dst_ids=dst, **args)


@pytest.mark.skipif(LIB_PATH.name == "libkvattn_san.so", reason="the sanitizer ends the process at such an allocation")
def test_out_of_host_memory_is_an_error():
    """Tables of 4 PiB: the call answers, it does not end the process."""
    with pytest.raises(KvaError) as e:
        make(max_seqs=2**30, max_blocks_per_seq=2**20)
    assert "out of host memory" in str(e.value)
