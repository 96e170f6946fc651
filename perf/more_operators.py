"""The operators of a layer whose projections are held in 4 bits, as timed cases.

Four kinds.  A microscaled row is a row of blocks of 32 elements, each block
with one scale: 4-bit elements (sign, 2 exponent and 1 mantissa bit: 0, 0.5, 1,
1.5, 2, 3, 4, 6) or 8-bit ones (4 exponent and 3 mantissa bits, up to 448), and
a scale 2^(b - 127) held as the byte b.  The scale is the smallest power of two,
from 2^-126 on, for which the largest element value covers the block's largest
magnitude; an element is x / scale rounded to the nearest, ties to even.

* ``norm``      hidden += delta, and its root-mean-square norm as microscaled
  8-bit rows (read back) or in FP16 (``add_rmsnorm``, ``dequantize``);
* ``quantize``  FP16 rows as microscaled ones, read back (``quantize``,
  ``dequantize``);
* ``project``   the Q, gate, K and V projection of a step's tokens by 4-bit
  weights, with QK norm, RoPE and the append to the cache (``mx_project_append``);
* ``out``       the output projection of attention rows by 4-bit weights onto
  the residual; the rows come in FP16 and are quantised on the way
  (``mx_out_project``).

A product's value is the sum over k of the two elements' products, each times
both scales.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 256
PAGE = 16
BLOCK = 32
EPS = 1e-6
HALF_ROT = 32
THETA = 1e7
#: Largest element, its exponent, the least exponent of a normal one, mantissa bits.
FORMATS = {8: (448.0, 8, -6, 3), 4: (6.0, 2, 0, 1)}


def _case(kind, tokens, cols=0, rows=0, bits=8, heads=24, kv_heads=4, seqs=1, stride=0, delta=True, ragged=0):
    """cols: the axis summed over (or normalised, or quantised); rows: of a weight; stride: values between rows
    beyond cols."""
    return {"kind": kind, "tokens": tokens, "cols": cols, "rows": rows, "bits": bits, "heads": heads,
            "kv_heads": kv_heads, "seqs": seqs, "stride": stride, "delta": delta, "ragged": ragged}


def listed():
    return [
        # The norm before a layer's projections, one user.
        dict(_case("norm", 1, 5120), name="norm_b1"),
        # The same of a long batch of prompt chunks.
        dict(_case("norm", 8192, 5120), name="norm_8k"),
        # The last layer's rows, whose head is not in 8 bits.
        dict(_case("norm", 2048, 5120, bits=16), name="norm_2k_fp16"),
        # An output projection's weights taken to 4 bits.
        dict(_case("quantize", 5120, 6144, bits=4), name="quantize_w_o"),
        # The attention rows of a short prompt, cut from a wider buffer.
        dict(_case("quantize", 181, 6144, bits=8, stride=6144), name="quantize_181"),
        # One user's decode step.
        dict(_case("project", 1, 5120, ragged=1), name="project_b1"),
        # The decode step of the benchmark's serving batch.
        dict(_case("project", 32, 5120, seqs=32, ragged=2), name="project_b32"),
        # A prompt of odd length.
        dict(_case("project", 181, 5120, ragged=3), name="project_181"),
        # The chunks of four prompts, with 8-bit and with 4-bit activations.
        dict(_case("project", 2048, 5120, seqs=4, ragged=4), name="project_4x512"),
        dict(_case("project", 2048, 5120, bits=4, seqs=4, ragged=5), name="project_4x512_a4"),
        # The other end of the attention, for the batch and for the chunks.
        dict(_case("out", 32, 6144, 5120), name="out_b32"),
        dict(_case("out", 2048, 6144, 5120), name="out_4x512"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "project", "project", "project", "out", "out"])
    if kind == "norm":
        cols = 32 * _log(rng, 8, 256)
        return _case(kind, _log(rng, 1, 8192 * 5120 // max(cols, 5120)), cols, bits=rng.choice([8, 8, 16]),
                     delta=rng.random() < 0.7)
    if kind == "quantize":
        cols = 32 * _log(rng, 2, 256)
        return _case(kind, _log(rng, 1, min(16384, 30000000 // cols)), cols, bits=rng.choice([8, 4]),
                     stride=rng.choice([0, 0, 8 * rng.randrange(1, 800)]))
    heads, kv_heads = rng.choice([(24, 4), (24, 4), (16, 4), (8, 8), (8, 1), (6, 3), (6, 1)])
    tokens = rng.choice([_log(rng, 1, 48), _log(rng, 1, 2048)])
    if kind == "project":
        cols = rng.choice([512, 1024, 1536, 2048, 2560, 4096, 5120, 5120, 5120])
        return _case(kind, tokens, cols, bits=rng.choice([8, 8, 4]), heads=heads, kv_heads=kv_heads,
                     seqs=rng.choice([1, min(tokens, rng.randrange(1, 33)), min(tokens, 32)]),
                     ragged=rng.randrange(1, 1 << 20))
    rows = rng.choice([336, 1040, 2048, 2560, 5120, 5120])
    return _case(kind, tokens, heads * D, min(rows, 2 * (heads + kv_heads) * D), bits=rng.choice([8, 8, 4]),
                 heads=heads, kv_heads=kv_heads, delta=rng.random() < 0.8)


class _Plan:
    """A step's sequences: rows held, new tokens, pages, positions."""

    def __init__(self, case):
        r = np.random.default_rng(case["ragged"])
        n = case["seqs"]
        cut = np.sort(r.choice(np.arange(1, case["tokens"]), n - 1, replace=False)) if n > 1 else np.zeros(0, np.int64)
        self.new = np.diff(np.concatenate([[0], cut, [case["tokens"]]])).astype(np.int64)
        self.base = r.integers(0, 40, n)  # rows of the cache that are filled already
        self.n_pages = -(-(self.base + self.new) // PAGE)
        self.pages = int(self.n_pages.sum())
        order = r.permutation(self.pages).astype(np.int32)
        self.blocks = np.split(order, np.cumsum(self.n_pages)[:-1])
        start = r.integers(0, 30000, n)  # positions run ahead of the rows where earlier ones were evicted
        self.pos = np.concatenate([s + b + np.arange(m) for s, b, m in zip(start, self.base, self.new)])
        self.slot = np.concatenate([ids[(b + np.arange(m)) // PAGE].astype(np.int64) * PAGE + (b + np.arange(m)) % PAGE
                                    for ids, b, m in zip(self.blocks, self.base, self.new)])


def _put(x):
    return torch.as_tensor(x, device="cuda")


def _half(g, *shape):
    return torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)


def _weight_rows(g, rows, cols):
    """A projection's rows in FP16: of unlike size, a few strong columns."""
    w = _half(g, rows, cols)
    w *= (cols ** -0.5 * torch.empty(rows, 1, device="cuda").uniform_(0.5, 2.0, generator=g)).half()
    w[:, torch.randperm(cols, generator=g, device="cuda")[:4]] *= 4
    return w


def _hidden_rows(g, rows, cols):
    """A residual stream's rows: some channels far stronger than the rest."""
    x = _half(g, rows, cols)
    strong = torch.ones(cols, device="cuda")
    strong[torch.randperm(cols, generator=g, device="cuda")[:max(1, cols // 256)]] = 20.0
    return x.mul_(strong.half())


def _norm_weight(g, cols):
    return (1 + 0.02 * torch.empty(cols, device="cuda").normal_(generator=g)).half()


def _inputs(case, seed):
    """A case's inputs, from its seed alone, as FP16 tensors (a product's weights and activations before they are
    taken to 4 and 8 bits)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, n, cols = case["kind"], case["tokens"], case["cols"]
    if kind == "norm":
        return {"hidden": _hidden_rows(g, n, cols), "delta": _hidden_rows(g, n, cols) if case["delta"] else None,
                "w": _norm_weight(g, cols)}
    if kind == "quantize":
        x = _hidden_rows(g, n, cols + case["stride"])
        return {"x": x * torch.exp2(torch.randint(-12, 6, (n, 1), generator=g, device="cuda").float()).half()}
    if kind == "project":
        heads, kv = case["heads"], case["kv_heads"]
        return {"x": _hidden_rows(g, n, cols), "wq": _weight_rows(g, 2 * heads * D, cols),
                "wkv": _weight_rows(g, 2 * kv * D, cols), "q_norm": _norm_weight(g, D), "k_norm": _norm_weight(g, D)}
    size = torch.empty(case["heads"], 1, device="cuda").uniform_(0.05, 2.0, generator=g)  # heads of unlike size
    x = (_half(g, n, case["heads"], D).float() * size).half().view(n, cols)
    return {"x": x, "w": _weight_rows(g, case["rows"], cols), "res": _hidden_rows(g, n, case["rows"])
            if case["delta"] else None}


def _tables(case):
    """cos and sin of every position the case reaches, [rows, 32] FP16."""
    at = np.arange(int(_Plan(case).pos.max()) + 1, dtype=np.float64)[:, None]
    angle = at * THETA ** (-np.arange(HALF_ROT) / HALF_ROT)
    return _put(np.cos(angle).astype(np.float16)), _put(np.sin(angle).astype(np.float16))


# ---- microscaled rows, plainly -------------------------------------------------

def _scale_exponent(x, bits):
    """Exponent of the scale of each block of x [..., blocks, 32]."""
    most, top, _, _ = FORMATS[bits]
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1)
    e = e.int() - 1 - top + (m * 2 ** (top + 1) > most).int()
    return torch.where(amax > 0, e, -126).clamp(-126, 127)


def _elements(x, bits):
    """x [rows, cols] in 32 bits as elements and scale exponents, [rows, blocks, 32] and [rows, blocks]."""
    _, _, least, mant = FORMATS[bits]
    x = x.view(x.shape[0], -1, BLOCK)
    e = _scale_exponent(x, bits)
    y = torch.ldexp(x, -e[..., None])
    step = torch.ldexp(torch.ones((), device="cuda"), (torch.frexp(y)[1].int() - 1).clamp(min=least) - mant)
    return torch.round(y / step) * step, e


def _values(x, bits):
    y, e = _elements(x, bits)
    return torch.ldexp(y, e[..., None]).view(x.shape)


def _element_table(bits):
    """The value of every code."""
    _, _, least, mant = FORMATS[bits]
    c = torch.arange(1 << bits, device="cuda")
    mag = c & ((1 << (bits - 1)) - 1)
    e, m = mag >> mant, (mag & ((1 << mant) - 1)).float() / (1 << mant)
    v = torch.where(e > 0, torch.ldexp(1 + m, (e - 1 + least).int()), torch.ldexp(m, torch.full_like(e, least).int()))
    return torch.where(c >> (bits - 1) == 1, -v, v)


def _encode(x, bits):
    """FP16 rows as codes and scale bytes: [rows, cols * bits / 8] (the even element in the low half of a byte) and
    [rows, cols / 32]."""
    y, e = _elements(x.float(), bits)
    half = 1 << (bits - 1)
    code = torch.searchsorted(_element_table(bits)[:half].nan_to_num(posinf=1e9).contiguous(), y.abs().contiguous())
    code = (code + half * torch.signbit(y)).view(x.shape)
    if bits == 4:
        code = code[:, ::2] | code[:, 1::2] << 4
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def _decode(codes, scales, bits):
    """The values that codes stand for, in 32 bits."""
    t = _element_table(bits)
    v = t[codes.int()] if bits == 8 else torch.stack([t[(codes & 15).int()], t[(codes >> 4).int()]], -1)
    v = v.view(codes.shape[0], -1, BLOCK)
    return torch.ldexp(v, scales.int()[..., None] - 127).view(codes.shape[0], -1)


# ---- states ----------------------------------------------------------------------

class _State:
    pass


class _Memory:
    """Device memory that torch may see without a copy; a tensor made of it
    keeps it, and it its owner."""

    def __init__(self, owner, ptr, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": kind, "version": 3}


def prepare(case, seed):
    s = _State()
    s.c = case
    kind, n, cols, bits = case["kind"], case["tokens"], case["cols"], case["bits"]
    for k, v in _inputs(case, seed).items():
        setattr(s, k, v)
    if kind in ("project", "out"):  # the weights are held in 4 bits; a projection's rows come from a norm in `bits`
        for k in ("wq", "wkv") if kind == "project" else ("w",):
            setattr(s, k, _encode(getattr(s, k), 4))
    if kind == "project":
        s.x = _encode(s.x, bits)
        s.cos, s.sin = _tables(case)
        s.plan = _Plan(case)
    if own:
        _own_prepare(s)
    elif kind == "project":
        s.pos, s.slot = _put(s.plan.pos), _put(s.plan.slot)
        shape = (s.plan.pages * PAGE, case["kv_heads"], D)
        s.k, s.v = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in "kv")
    torch.cuda.synchronize()
    return s


# ---- the framework's side ----------------------------------------------------------

def _own_prepare(s):
    from mi50grad_amd import microscale
    from mi50grad_amd.kv_cache import PagedKVCache

    s.mx = microscale
    c = s.c
    n, cols, bits = c["tokens"], c["cols"], c["bits"]
    new = lambda *shape, t=torch.float16: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
    if c["kind"] in ("norm", "quantize"):
        s.out = new(n, cols)
        if c["kind"] == "norm" and s.delta is not None:
            s.sum = new(n, cols)
        if bits < 16:
            s.codes, s.scales = new(n, cols * bits // 8, t=torch.uint8), new(n, cols // BLOCK, t=torch.uint8)
        return

    def packed(w):  # the order that the products read, laid out once
        codes, scales = w
        rows = codes.shape[0]
        p = new(microscale.packed_bytes(rows, cols), t=torch.uint8)
        microscale.pack_weights(codes.data_ptr(), scales.data_ptr(), rows, cols, p.data_ptr())
        torch.cuda.synchronize()  # before codes and scales go
        return p

    heads, kv = c["heads"], c["kv_heads"]
    if c["kind"] == "out":
        s.w = packed(s.w)
        s.cache = PagedKVCache(n_layers=1, max_seqs=1, max_blocks=1, max_blocks_per_seq=1, max_step_tokens=max(n, 64),
                               num_heads=heads, num_kv_heads=kv)
        s.out = new(n, c["rows"])
        return
    s.wq, s.wkv = packed(s.wq), packed(s.wkv)
    p = s.plan
    s.cache = PagedKVCache(n_layers=1, max_seqs=len(p.new), max_blocks=p.pages, max_blocks_per_seq=int(p.n_pages.max()),
                           max_step_tokens=max(n, 64), num_heads=heads, num_kv_heads=kv, eps=EPS)
    for b, ids in enumerate(p.blocks):
        s.cache.set_blocks(b, ids)
        s.cache.set_len(b, int(p.base[b]))
    s.cache.begin_step(range(len(p.new)), p.new, rope_pos=p.pos)
    s.q, s.gate = new(n, heads, D), new(n, heads, D)
    s.k, s.v = (torch.as_tensor(_Memory(s.cache, x, (p.pages * PAGE, kv, D), "<f2"), device="cuda")
                for x in s.cache.layer_pools(0))


def _own_run(s):
    c, mx = s.c, s.mx
    n, cols, bits = c["tokens"], c["cols"], c["bits"]
    if c["kind"] == "norm":
        delta, total = (None, None) if s.delta is None else (s.delta.data_ptr(), s.sum.data_ptr())
        if bits == 16:
            mx.add_rmsnorm(s.hidden.data_ptr(), delta, s.w.data_ptr(), n, cols, EPS, s.out.data_ptr(), sum_out=total)
        else:
            mx.add_rmsnorm(s.hidden.data_ptr(), delta, s.w.data_ptr(), n, cols, EPS, s.codes.data_ptr(),
                           scales=s.scales.data_ptr(), bits=bits, sum_out=total)
            mx.dequantize(s.codes.data_ptr(), s.scales.data_ptr(), n, cols, bits, s.out.data_ptr())
        return {"x": s.out} if delta is None else {"hidden": s.sum, "x": s.out}
    if c["kind"] == "quantize":
        mx.quantize(s.x.data_ptr(), n, cols, bits, s.codes.data_ptr(), s.scales.data_ptr(),
                    x_stride=cols + c["stride"])
        mx.dequantize(s.codes.data_ptr(), s.scales.data_ptr(), n, cols, bits, s.out.data_ptr())
        return {"x": s.out}
    if c["kind"] == "project":
        s.cache.mx_project_append(0, s.x[0].data_ptr(), cols, s.wq.data_ptr(), s.wkv.data_ptr(), s.q_norm.data_ptr(),
                                  s.k_norm.data_ptr(), s.cos.data_ptr(), s.sin.data_ptr(), s.cos.shape[0],
                                  s.q.data_ptr(), s.gate.data_ptr(), x_scales=s.x[1].data_ptr(), bits=bits)
        return {"q": s.q, "gate": s.gate, "k": s.k, "v": s.v}
    s.cache.mx_out_project(s.x.data_ptr(), n, cols, s.w.data_ptr(), c["rows"], s.out.data_ptr(),
                           residual=s.res.data_ptr() if s.res is not None else None, bits=bits)
    return {"out": s.out}


# ---- the plain forms ------------------------------------------------------------------

def _rms(x, w):
    return x * (1.0 / torch.sqrt(torch.mean(x * x, -1, keepdim=True) + EPS)) * w.float()


def _rotated(x, s):
    """Norm and partial rotation of head rows [token, head, D]: interleaved pairs of the first 64 dims."""
    cos, sin = s.cos[s.pos].float()[:, None], s.sin[s.pos].float()[:, None]
    a, b = x[..., 0:2 * HALF_ROT:2], x[..., 1:2 * HALF_ROT:2]
    pair = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([pair, x[..., 2 * HALF_ROT:]], -1)


def _plain_run(s):
    c = s.c
    n, cols, bits = c["tokens"], c["cols"], c["bits"]
    if c["kind"] == "norm":
        hidden = s.hidden if s.delta is None else (s.hidden.float() + s.delta.float()).half()
        x = _rms(hidden.float(), s.w)
        x = (x if bits == 16 else _values(x, bits)).half()
        return {"x": x} if s.delta is None else {"hidden": hidden, "x": x}
    if c["kind"] == "quantize":
        return {"x": _values(s.x[:, :cols].float(), bits).half()}
    if c["kind"] == "project":
        heads, kv = c["heads"], c["kv_heads"]
        x = _decode(*s.x, bits)
        y = torch.matmul(x, _decode(*s.wq, 4).t()).view(n, 2 * heads, D)
        z = torch.matmul(x, _decode(*s.wkv, 4).t()).view(n, 2 * kv, D)
        s.k[s.slot] = _rotated(_rms(z[:, :kv], s.k_norm), s).half()
        s.v[s.slot] = z[:, kv:].half()
        return {"q": _rotated(_rms(y[:, :heads], s.q_norm), s).half(), "gate": y[:, heads:].half(), "k": s.k, "v": s.v}
    y = torch.matmul(_values(s.x.float(), bits), _decode(*s.w, 4).t())
    return {"out": (y if s.res is None else y + s.res.float()).half()}


def run(s):
    return _own_run(s) if own else _plain_run(s)


# ---- the work, and the definition in 64 bits ---------------------------------------------

def work(case):
    kind, n, cols, bits = case["kind"], case["tokens"], case["cols"], case["bits"]
    held = bits / 8 + (1 / BLOCK if bits < 16 else 0)  # bytes of a value
    back = held + 2 if bits < 16 else 0  # read back
    if kind == "norm":
        return {"bytes": n * cols * ((6 if case["delta"] else 2) + held + back) + 2 * cols, "flops": 6.0 * n * cols}
    if kind == "quantize":
        return {"bytes": n * cols * (2 + held + back), "flops": 0.0}
    heads, kv = case["heads"], case["kv_heads"]
    rows = 2 * (heads + kv) * D if kind == "project" else case["rows"]
    weights = rows * cols * (0.5 + 1 / BLOCK)
    if kind == "project":
        return {"bytes": weights + n * cols * held + n * rows * 2.0, "flops": 2.0 * n * rows * cols}
    return {"bytes": weights + n * cols * 2.0 + n * rows * (4.0 if case["delta"] else 2.0),
            "flops": 2.0 * n * rows * cols}


def _grid(bits):
    """An element's magnitudes, ascending, in 64 bits."""
    small = {4: [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
             8: [k / 512 for k in range(8)] + [(8 + k) / 8 * 2.0 ** e for e in range(-6, 9) for k in range(8)][:-1]}
    return torch.tensor(small[bits], dtype=torch.float64, device="cuda")


def _nearest(x, bits):
    """What microscaled rows hold of x, in 64 bits, by looking for the nearest element."""
    grid = _grid(bits)
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for i in range(0, x.shape[0], 1024):
        y = x[i:i + 1024].double().view(-1, x.shape[1] // BLOCK, BLOCK)
        most = y.abs().amax(-1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(most / grid[-1]).clamp(-126, 127)))
        unit = torch.where(most > grid[-1] * unit, unit * 2, unit)
        unit = torch.where((most <= grid[-1] * unit / 2) & (unit > 2.0 ** -126), unit / 2, unit)
        y = y / unit
        mag = y.abs().contiguous()
        hi = torch.searchsorted(grid, mag).clamp(max=len(grid) - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = grid[hi] - mag, mag - grid[lo]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        out[i:i + 1024] = (torch.copysign(grid[pick], y) * unit).view(-1, x.shape[1])
    return out


def exact(case, seed):
    i = _inputs(case, seed)
    kind, n, cols, bits = case["kind"], case["tokens"], case["cols"], case["bits"]
    if kind == "norm":
        hidden = i["hidden"] if i["delta"] is None else (i["hidden"].double() + i["delta"].double()).half()
        x = hidden.double()
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * i["w"].double()
        x = x if bits == 16 else _nearest(x, bits)
        return {"x": x} if i["delta"] is None else {"hidden": hidden.double(), "x": x}
    if kind == "quantize":
        return {"x": _nearest(i["x"][:, :cols], bits)}
    x = _nearest(i["x"], bits)
    if kind == "out":
        y = x @ _nearest(i["w"], 4).t().contiguous()
        return {"out": y if i["res"] is None else y + i["res"].double()}
    heads, kv = case["heads"], case["kv_heads"]
    p = _Plan(case)
    cos, sin = (t[_put(p.pos)].double()[:, None] for t in _tables(case))

    def normed(y, w):
        y = y * torch.rsqrt(y.square().sum(-1, keepdim=True) / D + EPS) * w.double()
        z = torch.view_as_complex(y[..., :2 * HALF_ROT].reshape(y.shape[:2] + (HALF_ROT, 2)))
        z = torch.view_as_real(z * torch.complex(cos, sin).expand(y.shape[:2] + (HALF_ROT,)))
        return torch.cat([z.flatten(-2), y[..., 2 * HALF_ROT:]], -1)

    y = (x @ _nearest(i["wq"], 4).t().contiguous()).view(n, 2 * heads, D)
    z = (x @ _nearest(i["wkv"], 4).t().contiguous()).view(n, 2 * kv, D)
    k, v = (torch.zeros(p.pages * PAGE, kv, D, dtype=torch.float64, device="cuda") for _ in "kv")
    k[_put(p.slot)] = normed(z[:, :kv], i["k_norm"])
    v[_put(p.slot)] = z[:, kv:]
    return {"q": normed(y[:, :heads], i["q_norm"]), "gate": y[:, heads:], "k": k, "v": v}
