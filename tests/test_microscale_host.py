"""Refusals of the microscaled entry points (CPU: each is found before the
device is touched), and the sizes that they tell."""
import pytest

from mi50grad_amd import microscale as ms
from mi50grad_amd._lib import KvaError
from mi50grad_amd.kv_cache import PagedKVCache

INVALID, UNSUPPORTED, NO_DEVICE, STATE, MISALIGNED = -1, -2, -3, -8, -10
A, B, C, E = 1 << 40, 1 << 41, 1 << 42, 1 << 43  # far apart


def refused(code, call, *args, **kw):
    with pytest.raises(KvaError) as e:
        call(*args, **kw)
    assert e.value.code == code, e.value


def test_packed_bytes():
    assert ms.packed_bytes(64, 512) == 64 * (256 + 16)
    assert ms.packed_bytes(33, 1024) == 64 * (512 + 32)
    assert ms.packed_bytes(0, 512) == 0
    assert ms.packed_bytes(2 ** 31 - 1, 2 ** 31 - 512) > 1 << 61
    refused(INVALID, ms.packed_bytes, -1, 512)
    refused(INVALID, ms.packed_bytes, 32, 0)
    refused(INVALID, ms.packed_bytes, 32, 256)


def test_quantize_refusals():
    for bits in (0, 2, 6, 16):
        refused(UNSUPPORTED, ms.quantize, A, 4, 64, bits, B, C)
        refused(UNSUPPORTED, ms.dequantize, A, B, 4, 64, bits, C)
    refused(INVALID, ms.quantize, A, -1, 64, 8, B, C)
    for cols in (0, -32, 8, 33, 48):
        refused(INVALID, ms.quantize, A, 4, cols, 8, B, C, x_stride=64)
        refused(INVALID, ms.dequantize, A, B, 4, cols, 8, C)
    for stride in (32, 65, 68, -64):
        refused(INVALID, ms.quantize, A, 4, 64, 8, B, C, x_stride=stride)
    for args in ((None, B, C), (A, None, C), (A, B, None)):
        refused(INVALID, ms.quantize, args[0], 4, 64, 8, args[1], args[2])
        refused(INVALID, ms.dequantize, args[0], args[1], 4, 64, 8, args[2])
    for args in ((A + 8, B, C), (A, B + 4, C), (A, B, C + 1)):
        refused(MISALIGNED, ms.quantize, args[0], 4, 64, 8, args[1], args[2])
        refused(MISALIGNED, ms.dequantize, args[0], args[1], 4, 64, 8, args[2])
    # 4 rows of 64 at a stride of 128: 896 bytes of x
    refused(INVALID, ms.quantize, A, 4, 64, 8, A + 880, C, x_stride=128)
    refused(INVALID, ms.quantize, A, 4, 64, 8, B, A - 16 + 16, x_stride=128)
    refused(INVALID, ms.quantize, A, 4, 64, 8, B, B + 240)
    refused(INVALID, ms.dequantize, A, B, 4, 64, 8, A - 496)
    refused(INVALID, ms.dequantize, A, B, 4, 64, 8, B)
    # more values, or further apart, than a call takes
    refused(UNSUPPORTED, ms.quantize, A, 1 << 21, 64, 8, 1 << 60, 1 << 61, x_stride=(1 << 19) + 8)
    refused(UNSUPPORTED, ms.quantize, A, 1, 64, 8, B, C, x_stride=(1 << 40) + 8)
    refused(UNSUPPORTED, ms.quantize, A, 2 ** 31 - 1, 64, 8, B, C, x_stride=2 ** 63 - 8)
    refused(UNSUPPORTED, ms.dequantize, A, B, 2 ** 31 - 1, 1024, 8, C)
    refused(UNSUPPORTED, ms.pack_weights, A, B, 2 ** 31 - 1, 1024, C)
    ms.quantize(None, 0, 64, 8, None, None)  # nothing to do
    ms.dequantize(None, None, 0, 64, 8, None)


def test_pack_refusals():
    refused(INVALID, ms.pack_weights, A, B, -1, 512, C)
    refused(INVALID, ms.pack_weights, A, B, 32, 256, C)
    for args in ((None, B, C), (A, None, C), (A, B, None)):
        refused(INVALID, ms.pack_weights, args[0], args[1], 32, 512, args[2])
    for args in ((A + 8, B, C), (A, B + 4, C), (A, B, C + 1)):
        refused(MISALIGNED, ms.pack_weights, args[0], args[1], 32, 512, args[2])
    refused(INVALID, ms.pack_weights, A, B, 33, 512, A)
    refused(INVALID, ms.pack_weights, A, B, 33, 512, B - ms.packed_bytes(33, 512) + 16)
    ms.pack_weights(None, None, 0, 512, None)


def test_norm_refusals():
    norm = ms.add_rmsnorm
    for bits in (0, 2, 6, 32):
        refused(UNSUPPORTED, norm, A, None, B, 4, 64, 1e-6, C, scales=E, bits=bits)
    refused(INVALID, norm, A, None, B, -1, 64, 1e-6, C)
    for cols in (0, 8, 40, -32):
        refused(INVALID, norm, A, None, B, 4, cols, 1e-6, C)
    refused(UNSUPPORTED, norm, A, None, B, 4, 32768 + 32, 1e-6, C)
    for eps in (-1e-6, float("nan")):
        refused(INVALID, norm, A, None, B, 4, 64, eps, C)
    refused(INVALID, norm, None, None, B, 4, 64, 1e-6, C)
    refused(INVALID, norm, A, None, None, 4, 64, 1e-6, C)
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, None)
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, C, scales=E)  # fp16 rows have none
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, C, bits=8)
    refused(INVALID, norm, A, E, B, 4, 64, 1e-6, C)  # a delta without a place for the sum
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, C, sum_out=E)
    refused(MISALIGNED, norm, A + 8, None, B, 4, 64, 1e-6, C)
    refused(MISALIGNED, norm, A, None, B, 4, 64, 1e-6, C, scales=E + 8, bits=4)
    # 4 x 64 values: 512 bytes of fp16 rows, 256 of 8-bit codes
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, A + 496)
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, A)
    refused(INVALID, norm, A, E, B, 4, 64, 1e-6, C, sum_out=A + 16)
    refused(INVALID, norm, A, E, B, 4, 64, 1e-6, C, sum_out=C + 496)
    refused(INVALID, norm, A, E, B, 4, 64, 1e-6, E, sum_out=C)
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, C, scales=C + 240, bits=8)
    refused(INVALID, norm, A, None, B, 4, 64, 1e-6, B, scales=C, bits=8)
    norm(None, None, None, 0, 64, 1e-6, None)


def test_sizes_that_a_launch_cannot_count():
    """Lanes, eight values each, are counted in 32 bits."""
    rows, far = 1 << 20, (1 << 55, 1 << 56, 1 << 57)  # of 16384: 2^34 values
    for bits in (8, 4):
        refused(UNSUPPORTED, ms.quantize, far[0], rows + 1, 16384, bits, far[1], far[2])
        refused(MISALIGNED, ms.quantize, far[0] + 8, rows, 16384, bits, far[1], far[2])
        refused(UNSUPPORTED, ms.dequantize, far[0], far[1], rows + 1, 16384, bits, far[2])
        refused(MISALIGNED, ms.dequantize, far[0] + 8, far[1], rows, 16384, bits, far[2])
    refused(UNSUPPORTED, ms.pack_weights, far[0], far[1], rows + 1, 16384, far[2])
    refused(MISALIGNED, ms.pack_weights, far[0] + 8, far[1], rows, 16384, far[2])
    for cols in (32, 544, 5120, 32768):
        most = (1 << 34) // (cols + 512)
        refused(UNSUPPORTED, ms.add_rmsnorm, far[0], None, far[1], most + 1, cols, 1e-6, far[2])
        refused(MISALIGNED, ms.add_rmsnorm, far[0] + 8, None, far[1], most, cols, 1e-6, far[2])


def make(**kw):
    return PagedKVCache(n_layers=1, max_seqs=4, max_blocks=2048, max_blocks_per_seq=512,
                        max_step_tokens=kw.pop("max_step_tokens", 4096), host_only=True, **kw)


def project(c, layer=0, x=A, hidden=512, wq=B, wkv=C, norms=(1 << 44, 1 << 44), tabs=(1 << 45, 1 << 45), rows=4096,
            q=E, gate=None, kv=None, scales=None, bits=8):
    c.mx_project_append(layer, x, hidden, wq, wkv, *norms, *tabs, rows, q, gate, kv, x_scales=scales, bits=bits)


def test_project_refusals():
    c = make()
    refused(STATE, project, c)
    c.begin_step([0, 1], [3, 2])
    refused(NO_DEVICE, project, c)  # every check passed
    refused(NO_DEVICE, project, c, scales=1 << 46, gate=1 << 47, kv=1 << 48, bits=4)
    refused(INVALID, project, c, layer=1)
    for bits in (16, 6, 0):
        refused(UNSUPPORTED, project, c, bits=bits)
    for kw in (dict(x=None), dict(wq=None), dict(wkv=None), dict(q=None), dict(norms=(None, A)),
               dict(norms=(1 << 44, None)), dict(tabs=(None, 1 << 45)), dict(tabs=(1 << 45, None))):
        refused(INVALID, project, c, **kw)
    for kw in (dict(x=A + 8), dict(wq=B + 8), dict(wkv=C + 1), dict(q=E + 2), dict(gate=A - 8), dict(kv=A - 8),
               dict(scales=(1 << 46) + 4), dict(norms=((1 << 44) + 8, 1 << 44)), dict(tabs=((1 << 45) + 4, 1 << 45))):
        refused(MISALIGNED, project, c, **kw)
    for hidden in (0, -512, 256, 768, 513):
        refused(INVALID, project, c, hidden=hidden)
    refused(INVALID, project, c, rows=2)  # positions 0..2
    refused(INVALID, project, c, hidden=1 << 25)
    # outputs over operands: 5 tokens, x 5 x 512 values
    for kw in (dict(q=A), dict(q=A + 5 * 1024 - 16), dict(gate=A), dict(kv=A), dict(q=B), dict(kv=C + 16)):
        refused(INVALID, project, c, **kw)
    # norm weights of 512 bytes, tables of 4096 rows of 32, 5 tokens of 24 query heads and 8 K and V heads
    for at in (1 << 44, (1 << 44) + 496, (1 << 45) + 4096 * 64 - 16):
        for kw in (dict(q=at), dict(gate=at), dict(kv=at)):
            refused(INVALID, project, c, **kw)
    refused(NO_DEVICE, project, c, q=(1 << 44) + 512, gate=(1 << 45) + 4096 * 64)
    q_bytes, kv_bytes = 5 * 24 * 512, 5 * 8 * 512
    for kw in (dict(gate=E), dict(gate=E + q_bytes - 16), dict(kv=E + q_bytes - 16), dict(kv=E - kv_bytes + 16),
               dict(gate=1 << 47, kv=(1 << 47) + 16)):
        refused(INVALID, project, c, **kw)
    refused(NO_DEVICE, project, c, gate=E + q_bytes, kv=E - kv_bytes)
    refused(NO_DEVICE, project, c, q=A + 5 * 1024)
    refused(NO_DEVICE, project, c, q=A + 5 * 512, scales=1 << 46)
    refused(INVALID, project, c, q=A + 5 * 512, scales=A + 5 * 512 + 16)
    refused(INVALID, project, c, q=A + 5 * 256, scales=1 << 46)
    refused(NO_DEVICE, project, c, q=A + 5 * 256, scales=1 << 46, bits=4)
    c.begin_step([0], [0])
    refused(NO_DEVICE, project, c, x=None)  # a step without tokens asks for nothing
    c.destroy()


def test_project_without_rotary_dims():
    """Tables are named but not read: they overlap nothing."""
    c = make(rotary_dim=0)
    c.begin_step([0], [1])
    refused(NO_DEVICE, project, c, tabs=(E + 16, E + 32))
    c.destroy()


def out(c, x=A, n=5, q_dim=512, w=B, n_out=64, res=None, o=E, scales=None, bits=8):
    c.mx_out_project(x, n, q_dim, w, n_out, o, residual=res, attn_scales=scales, bits=bits)


def test_out_refusals():
    c = make()
    refused(NO_DEVICE, out, c)
    refused(NO_DEVICE, out, c, res=E)  # in place
    refused(NO_DEVICE, out, c, n=0, x=None)
    for bits in (16, 6, 0):
        refused(UNSUPPORTED, out, c, bits=bits)
    refused(INVALID, out, c, n=-1)
    for kw in (dict(x=None), dict(w=None), dict(o=None)):
        refused(INVALID, out, c, **kw)
    for kw in (dict(x=A + 8), dict(w=B + 8), dict(o=E + 2), dict(res=A - 8), dict(scales=A - 8)):
        refused(MISALIGNED, out, c, **kw)
    for q_dim in (0, -512, 256, 768):
        refused(INVALID, out, c, q_dim=q_dim)
    for n_out in (0, -16, 8, 40):
        refused(INVALID, out, c, n_out=n_out)
    refused(UNSUPPORTED, out, c, n_out=(1 << 20) + 16)
    refused(NO_DEVICE, out, c, n_out=1 << 20)
    refused(INVALID, out, c, n=1 << 20, n_out=4096)
    refused(INVALID, out, c, q_dim=1 << 25)
    for kw in (dict(o=A), dict(o=A + 5 * 1024 - 16), dict(o=B + 16), dict(o=E, res=E + 16), dict(o=E, res=E - 16)):
        refused(INVALID, out, c, **kw)
    refused(NO_DEVICE, out, c, o=E, res=E + 5 * 128)
    refused(INVALID, out, c, o=A + 5 * 512, scales=A + 5 * 512)
    c.destroy()


def test_out_beyond_the_workspace():
    """fp16 rows go through half of the workspace, a token at least."""
    c = make(num_heads=1, num_kv_heads=1, max_step_tokens=1)
    room = 4 * 64 * 4 * 256 * 4 // 2  # bytes, half of [4 splits][64 tokens][4 * 256 rows] floats
    fit = (room - 512) * 32 // 33 // 512 * 512
    refused(NO_DEVICE, out, c, n=3, q_dim=fit)
    refused(INVALID, out, c, n=3, q_dim=fit + 1024)
    refused(NO_DEVICE, out, c, n=3, q_dim=fit + 1024, scales=1 << 46)
    refused(NO_DEVICE, out, c, n=3, q_dim=fit + 1024, bits=4)
    c.destroy()


def test_rows_whose_distance_no_64_bits_hold():
    """Rows times stride past 2^63 (and past 2^64, where the product's low bits
    are small again) is refused like any distance above 2^40."""
    for rows in (2, 1 << 22, 1 << 23, 1 << 24, (1 << 24) + 1, 1 << 29):
        refused(UNSUPPORTED, ms.quantize, A, rows, 32, 8, B, C, x_stride=1 << 40)
    refused(UNSUPPORTED, ms.quantize, A, 1 << 29, 32, 4, B, C, x_stride=(1 << 35) + 8)
    far = (1 << 55, 1 << 56, (1 << 57) + 8)
    refused(MISALIGNED, ms.quantize, far[0], 1, 32, 8, far[1], far[2], x_stride=1 << 40)  # at the limit: the next check
    refused(MISALIGNED, ms.quantize, far[0], 1 << 20, 32, 8, far[1], far[2], x_stride=1 << 20)
    refused(UNSUPPORTED, ms.quantize, far[0], 1 << 20, 32, 8, far[1], far[2], x_stride=(1 << 20) + 8)


def test_a_refusal_names_the_sizes_it_was_given():
    for cols in (32, 5120):
        n = (1 << 34) // (cols + 512) + 1
        with pytest.raises(KvaError, match=rf"{n} rows of {cols} values, {cols} apart"):
            ms.add_rmsnorm(1 << 55, None, 1 << 56, n, cols, 1e-6, 1 << 57)
