"""MXFP4 quantisation, products and expert layers on the GPU (marked `gpu`)
against the 64-bit numpy restatement (oracle/mx_numpy.py).

Tolerances, fixed from the arithmetic before any run:
  * quantisation, decoding, unpacking, choices and plans: equal bit for bit;
  * a sum of n products in f32, in any order: n * 2^-24 * sum |a b|
    (products of MXFP4 with MXFP4 are exact, with f32 one more rounding); the
    matrix instructions may truncate where an f32 addition rounds: twice that;
  * silu(g) * u: the operands' own errors to first order (|silu'| <= 1.1), and
    8 ulp for exp, quotient and product;
  * f16 / bf16 outputs: half an ulp more (2^-11, 2^-8 relative).
"""
from __future__ import annotations

import sys

import numpy as np
import pytest

from oracle import mx_numpy as MX

pytestmark = pytest.mark.gpu

F32, F16, BF16, MXFP4 = 0, 1, 30, 39
U24, U23 = 2.0 ** -24, 2.0 ** -23


def _say(msg: str) -> None:
    print(msg, flush=True)
    sys.stdout.flush()


class Dev:
    """Device copies of arrays, freed together; an output's guard bytes are
    checked to be untouched."""

    def __init__(self, ctx):
        self.ctx, self.bufs = ctx, []

    def up(self, a, shift=0):
        a = np.ascontiguousarray(a)
        b = self.ctx.alloc(max(16, a.nbytes + shift))
        self.bufs.append(b)
        raw = np.zeros(a.nbytes + shift, dtype=np.uint8)
        raw[shift:] = a.reshape(-1).view(np.uint8)
        if raw.nbytes:
            self.ctx.upload(b, raw)
        return b.ptr + shift

    def out(self, nbytes):
        b = self.ctx.alloc(nbytes + 64)
        self.bufs.append(b)
        self.ctx.upload(b, np.full(nbytes + 64, 0xA5, dtype=np.uint8))
        return b.ptr

    def down(self, ptr, nbytes, dtype, shape):
        raw = np.frombuffer(self.ctx.download(ptr, nbytes + 64), dtype=np.uint8)
        assert (raw[nbytes:] == 0xA5).all(), "written past the end"
        return raw[:nbytes].view(dtype).reshape(shape).copy()

    def close(self):
        for b in self.bufs:
            b.close()


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    ctx.synchronize()
    d.close()


def bf16_bits(x):
    """f32 -> bf16 bit patterns, round to nearest even (NaN kept)."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def bf16_value(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def as_type(x, t):
    """(bytes to upload, the values they stand for) of f32 data in type t."""
    x = np.asarray(x, dtype=np.float32)
    if t == F32:
        return x, x
    if t == F16:
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float32)
    b = bf16_bits(x)
    return b, bf16_value(b)


def read_out(dev, ptr, t, shape):
    n = int(np.prod(shape))
    if t == F32:
        return dev.down(ptr, 4 * n, np.float32, shape).astype(np.float64)
    if t == F16:
        return dev.down(ptr, 2 * n, np.float16, shape).astype(np.float64)
    return bf16_value(dev.down(ptr, 2 * n, np.uint16, shape)).astype(np.float64)


SIZE = {F32: 4, F16: 2, BF16: 2}
ROUND = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def activations(seed, rows, cols):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[:, rng.random(cols) < 0.02] *= 12
    return x


# ---- quantisation ----------------------------------------------------------------
def edge_blocks():
    """Blocks whose rounding, scale or special values can go wrong."""
    f = np.float32
    rows = []
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0]
    for top in (4.0, 7.9, 6.0, 7.0):  # ties of a block whose scale is 1
        up = [np.nextafter(f(t), f(9)) for t in ties]
        down = [np.nextafter(f(t), f(0)) for t in ties]
        rows.append(ties + up + down + [top] + [-t for t in ties[:7]])
    tiny = float(np.finfo(np.float32).smallest_subnormal)
    rows.append([0.0] * 31 + [-0.0])
    rows.append([tiny] + [0.0] * 30 + [-tiny])
    rows.append([2.0 ** -126, 2.0 ** -127, -(2.0 ** -128)] + [0.0] * 29)
    rows.append([2.0 ** -125, -(2.0 ** -125) * 1.75] + [2.0 ** -127] * 30)
    rows.append([2.0 ** -124 * 1.999] + [2.0 ** -125] * 31)
    rows.append([3.4028235e38, -3.4028235e38, 1e38] + [1.0] * 29)
    rows.append([1.0] * 31 + [np.inf])
    rows.append([-np.inf] + [1.0] * 31)
    rows.append([np.nan] + [1e30] * 31)
    rows.append([1.0] * 16 + [np.nan] * 16)
    rows.append(list(np.float32(2.0) ** -np.arange(32)))
    return np.array(rows, dtype=np.float32)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_quantize_edge_blocks_bit_exact(ctx, dev, t):
    with np.errstate(over="ignore"):
        raw, x = as_type(edge_blocks(), t)
    rows = len(x)
    _say(f"quantize edge blocks type {t}")
    dc, ds = dev.out(rows * 16), dev.out(rows)
    ctx.mxfp4_quantize(dev.up(raw), dc, ds, rows, 32, t)
    ctx.synchronize()
    codes, scales = dev.down(dc, rows * 16, np.uint8, (rows, 16)), dev.down(ds, rows, np.uint8,
                                                                          (rows, 1))
    want_c, want_s = MX.quantize(x)
    assert np.array_equal(scales, want_s)
    assert np.array_equal(codes, want_c)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,stride", [(1, 32, 0), (1, 4096, 0), (7, 96, 0), (5, 1312, 0),
                                              (3, 416, 424), (65, 64, 1000), (257, 2048, 0),
                                              (4099, 4128, 4136)])
def test_quantize_rows_and_strides(ctx, dev, t, rows, cols, stride):
    _say(f"quantize {rows}x{cols} stride {stride} type {t}")
    step = stride or cols
    raw, x = as_type(activations(rows * cols, rows, step) * 3, t)
    dc, ds = dev.out(rows * cols // 2), dev.out(rows * cols // 32)
    ctx.mxfp4_quantize(dev.up(raw), dc, ds, rows, cols, t, stride)
    ctx.synchronize()
    want_c, want_s = MX.quantize(x[:, :cols])
    assert np.array_equal(dev.down(ds, rows * cols // 32, np.uint8, want_s.shape), want_s)
    assert np.array_equal(dev.down(dc, rows * cols // 2, np.uint8, want_c.shape), want_c)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_dequant_every_code_and_scale(ctx, dev, t):
    """Every byte of codes under every scale byte; what a type cannot hold is
    rounded (f16) or an infinity (scale byte 254 times 4 or 6 in f32 and bf16)."""
    n = 256 * 8
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (n // 16, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 8).reshape(n, 1)
    codes[1::2] = codes[1::2][:, ::-1]
    dw = dev.out(n * 32 * SIZE[t])
    ctx.mxfp4_dequant(dev.up(codes), dev.up(scales), dw, n, t)
    ctx.synchronize()
    w = read_out(dev, dw, t, (n, 32))
    want = MX.decode(codes, scales)
    with np.errstate(over="ignore", invalid="ignore"):
        want = want.astype(np.float32)
        want = (want.astype(np.float16) if t == F16 else want).astype(np.float64)
    assert np.array_equal(np.isnan(w), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.array_equal(w[fine], want[fine])
    assert np.array_equal(np.signbit(w[fine]), np.signbit(want[fine]))


def test_unpack_ggml_blocks(ctx, dev):
    codes, scales = MX.gen_weights(11, 37, 352)
    q = MX.to_ggml(codes, scales)
    n = scales.size
    dc, ds = dev.out(codes.nbytes), dev.out(n)
    ctx.mxfp4_unpack_ggml(dev.up(q, shift=1), dc, ds, n)
    ctx.synchronize()
    assert np.array_equal(dev.down(dc, codes.nbytes, np.uint8, codes.shape), codes)
    assert np.array_equal(dev.down(ds, n, np.uint8, scales.shape), scales)


# ---- products ----------------------------------------------------------------------
SHAPES = [(1, 32), (3, 64), (8, 512), (9, 544), (33, 1024), (100, 1056), (999, 1312), (130, 2048),
          (17, 2080), (64, 4096), (257, 14336), (5, 40000), (2000, 256), (70, 768)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_matvec(ctx, dev, rows, cols):
    _say(f"mxfp4 matvec {rows}x{cols}")
    codes, scales = MX.gen_weights(rows + cols, rows, cols)
    x = activations(cols, 1, cols)[0]
    dy = dev.out(rows * 4)
    ctx.mxfp4_matvec(dev.up(codes), dev.up(scales, shift=3), dev.up(x), dy, rows, cols)
    ctx.synchronize()
    y = dev.down(dy, rows * 4, np.float32, rows).astype(np.float64)
    w = MX.decode(codes, scales)
    bound = cols * U24 * (np.abs(w) @ np.abs(x.astype(np.float64)))
    assert (np.abs(y - w @ x.astype(np.float64)) <= bound).all()


def test_matvec_special_scales(ctx, dev):
    """Scale 255 makes its row NaN and no other; scale 0 is 2^-127."""
    codes, scales = MX.gen_weights(5, 40, 2080)
    scales[3, 64] = 255
    scales[4, :] = 0
    x = activations(6, 1, 2080)[0]
    x[:32] = 2.0 ** 120
    dy = dev.out(160)
    ctx.mxfp4_matvec(dev.up(codes), dev.up(scales), dev.up(x), dy, 40, 2080)
    ctx.synchronize()
    y = dev.down(dy, 160, np.float32, 40)
    assert np.isnan(y[3]) and np.isfinite(np.delete(y, 3)).all()
    w = MX.decode(codes, scales)[4]
    xd = x.astype(np.float64)
    # products below 2^-126 may lose bits of the smallest f32
    assert abs(y[4] - w @ xd) <= 2080 * U24 * (np.abs(w) @ np.abs(xd)) + 2080 * 2.0 ** -149


MATMULS = [(1, 32, 1), (3, 64, 2), (31, 224, 5), (33, 256, 32), (64, 288, 33), (100, 1312, 17),
           (129, 512, 64), (65, 544, 65), (128, 1024, 128), (300, 1056, 130), (1000, 96, 300),
           (257, 4096, 77), (2048, 2048, 16), (1025, 736, 513), (40, 10272, 20), (16500, 544, 33),
           (2100, 512, 130), (2100, 1600, 520), (1700, 544, 1800), (3900, 512, 3300)]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,batch", MATMULS)
def test_matmul(ctx, dev, axc, rows, cols, batch, t):
    _say(f"mxfp4 matmul {rows}x{cols}x{batch} type {t}: "
         f"{axc.mxfp4_matmul_kernel_name(rows, cols, batch, t)}")
    wc, ws = MX.gen_weights(rows + cols, rows, cols)
    xc, xs = MX.quantize(activations(batch, batch, cols))
    dy = dev.out(rows * batch * SIZE[t])
    ctx.mxfp4_matmul(dev.up(wc), dev.up(ws, shift=1), dev.up(xc), dev.up(xs, shift=2), dy, rows,
                     cols, batch, t)
    ctx.synchronize()
    y = read_out(dev, dy, t, (batch, rows))
    w, x = MX.decode(wc, ws), MX.decode(xc, xs)
    exact = x @ w.T
    bound = cols * U23 * (np.abs(x) @ np.abs(w).T) + ROUND[t] * np.abs(exact)
    assert (np.abs(y - exact) <= bound).all()


def test_matmul_of_many_tiles_is_that_of_few(ctx, dev, axc):
    """More workgroups than the chip holds at once, and a long K: every column is the
    one that calls with fewer columns, on other kernels, give."""
    rows, cols, batch = 8192, 8192, 1024
    _say(f"matmul {rows}x{cols} b{batch} in parts")
    rng = np.random.default_rng(5)
    wc = rng.integers(0, 256, rows * cols // 2, dtype=np.uint8)
    xc = rng.integers(0, 256, batch * cols // 2, dtype=np.uint8)
    ws = np.full(rows * cols // 32, 120, dtype=np.uint8)
    xs = np.full(batch * cols // 32, 127, dtype=np.uint8)
    dwc, dws, dxc, dxs = dev.up(wc), dev.up(ws), dev.up(xc), dev.up(xs)
    # products are multiples of 2^-9 and sums below 8192 * 36 * 2^-7 < 2^12: 21 bits, so
    # that every sum is exact, in whatever order
    whole, names = None, set()
    for part in (batch, 512, 256, 96, 64):
        names.add(axc.mxfp4_matmul_kernel_name(rows, cols, part))
        dy = dev.out(4 * rows * batch)
        for at in range(0, batch, part):
            n = min(part, batch - at)
            ctx.mxfp4_matmul(dwc, dws, dxc + at * cols // 2, dxs + at * cols // 32,
                             dy + 4 * at * rows, rows, cols, n)
        ctx.synchronize()
        y = dev.down(dy, 4 * rows * batch, np.float32, (batch, rows))
        whole = y if whole is None else whole
        assert np.array_equal(y, whole)
    assert len(names) >= 3


@pytest.mark.parametrize("rows,cols,batches", [(70, 1056, (66, 20, 160)), (1100, 544, (300,)),
                                               (2100, 512, (130,)), (700, 1600, (500,)),
                                               (16500, 544, (33,))])
def test_matmul_special_scales(ctx, dev, axc, rows, cols, batches):
    """A NaN block reaches its row (or column) only; blocks past a row's end are
    not multiplied with the next row's."""
    for b in batches:
        _say(f"{rows}x{cols}x{b}: {axc.mxfp4_matmul_kernel_name(rows, cols, b)}")
        wc, ws = MX.gen_weights(1, rows, cols)
        xc, xs = MX.quantize(activations(b, b, cols))
        ws[11, 0] = 255
        xs[9, -1] = 255
        dy = dev.out(rows * b * 4)
        ctx.mxfp4_matmul(dev.up(wc), dev.up(ws), dev.up(xc), dev.up(xs), dy, rows, cols, b)
        ctx.synchronize()
        y = read_out(dev, dy, F32, (b, rows))
        nan = np.zeros((b, rows), dtype=bool)
        nan[9, :] = True
        nan[:, 11] = True
        assert np.array_equal(np.isnan(y), nan), b


def test_matmul_one_hot_is_exact(ctx, dev):
    """Rows of X with one element of 1 pick the weights out, bit for bit."""
    rows, cols = 96, 288
    wc, ws = MX.gen_weights(2, rows, cols)
    xc, xs = MX.quantize(np.eye(cols, dtype=np.float32))
    for lo, n in ((0, cols), (100, 40), (250, 9)):
        dy = dev.out(rows * n * 4)
        ctx.mxfp4_matmul(dev.up(wc), dev.up(ws), dev.up(xc[lo:lo + n]), dev.up(xs[lo:lo + n]), dy,
                         rows, cols, n)
        ctx.synchronize()
        y = read_out(dev, dy, F32, (n, rows))
        assert np.array_equal(y, MX.decode(wc, ws).T[lo:lo + n])


# ---- routing -------------------------------------------------------------------------
# experts, cols, tokens: a wave a logit for few, then tiles of 16 x 16, 64 x 64 (257 and
# 1024 experts) and 32 x 32 (500)
LOGITS = [(1, 32, 1), (5, 96, 3), (64, 4096, 1), (7, 2080, 8), (256, 2048, 2), (1, 32, 9),
          (33, 544, 9), (32, 2048, 70), (128, 1312, 77), (1000, 96, 40), (257, 512, 2500),
          (1024, 288, 830), (500, 416, 401), (700, 32, 9),
          (5, 2080, 1300)]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,cols,tokens", LOGITS)
def test_expert_logits(ctx, dev, n, cols, tokens, t):
    _say(f"logits {n} x {cols}, {tokens} tokens, type {t}")
    rng = np.random.default_rng(n + cols)
    raw, w = as_type(rng.standard_normal((n, cols)).astype(np.float32) / 8, t)
    x = activations(41, tokens, cols)
    dw, dx, dy = dev.up(raw), dev.up(x), dev.out(tokens * n * 4)
    ctx.expert_logits(dw, dx, dy, n, cols, tokens, t)
    ctx.synchronize()
    y = dev.down(dy, tokens * n * 4, np.float32, (tokens, n)).astype(np.float64)
    x = x.astype(np.float64)
    w = w.astype(np.float64)
    assert (np.abs(y - x @ w.T) <= (cols + 1) * U23 * (np.abs(x) @ np.abs(w).T)).all()
    # a row with a single 1 takes one element, and a token's NaN stays its own
    k = (np.arange(n) * 37 + 5) % cols
    one = np.zeros((n, cols), dtype=np.float32)
    one[np.arange(n), k] = 1
    xs = activations(42, tokens, cols)
    dw, dx = dev.up(as_type(one, t)[0]), dev.up(xs)
    ctx.expert_logits(dw, dx, dy, n, cols, tokens, t)
    ctx.synchronize()
    y = dev.down(dy, tokens * n * 4, np.float32, (tokens, n))
    assert np.array_equal(y, xs[:, k])
    xs[tokens // 2, cols // 2] = np.nan
    dx = dev.up(xs)
    ctx.expert_logits(dw, dx, dy, n, cols, tokens, t)
    ctx.synchronize()
    nan = np.isnan(dev.down(dy, tokens * n * 4, np.float32, (tokens, n)))
    assert nan[tokens // 2].all() and nan.sum() == n


def test_expert_logits_refusals(ctx, dev, axc):
    p = dev.out(1 << 12)
    good = dict(w=p, x=p, y=p, n=4, cols=64, tokens=2, t=F32)

    def call(**k):
        a = good | k
        ctx.expert_logits(a["w"], a["x"], a["y"], a["n"], a["cols"], a["tokens"], a["t"])

    for k in (dict(w=None), dict(x=None), dict(y=None), dict(w=p + 8), dict(x=p + 4),
              dict(y=p + 2), dict(n=0), dict(n=1025), dict(cols=0), dict(cols=48),
              dict(cols=1 << 23), dict(tokens=1 << 31), dict(t=MXFP4), dict(t=2)):
        with pytest.raises(axc.DispatchError) as err:
            call(**k)
            pytest.fail(f"{k} was accepted")
        assert err.value.variant == "InvalidArgument", k
    call(tokens=0)
    ctx.synchronize()
    assert (dev.down(p, 1 << 12, np.uint8, (1 << 12,)) == 0xA5).all()


def _route(ctx, dev, axc, logits, bias=None, t=F32, **kw):
    tokens, n = logits.shape
    raw, values = as_type(logits, t)
    o = axc.RouteOptions(n_experts=n, **kw)
    de, dw = dev.out(tokens * o.top_k * 4), dev.out(tokens * o.top_k * 4)
    ctx.expert_route(dev.up(raw), dev.up(bias) if bias is not None else None, de, dw, tokens, o, t)
    ctx.synchronize()
    e = dev.down(de, tokens * o.top_k * 4, np.int32, (tokens, o.top_k))
    w = dev.down(dw, tokens * o.top_k * 4, np.float32, (tokens, o.top_k))
    return values, e, w


def _spread_logits(seed, tokens, n):
    """Distinct logits at least 2^-7 apart: no two scores or biased keys near
    each other relative to f32."""
    rng = np.random.default_rng(seed)
    return np.stack([rng.permutation(n) for _ in range(tokens)]).astype(np.float32) / 64 - n / 128


ROUTES = [
    (1, 32, dict(top_k=4)), (5, 8, dict(top_k=8)), (3, 1, dict(top_k=1)),
    (9, 33, dict(top_k=2, normalize=False)), (4, 1000, dict(top_k=64)),
    (66, 256, dict(top_k=8, score="sigmoid", scale=2.5)),
    (7, 128, dict(top_k=6, n_groups=8, groups_kept=3)),
    (7, 256, dict(top_k=8, score="sigmoid", n_groups=8, groups_kept=4, group_best=2)),
    (5, 96, dict(top_k=3, score="softmax", n_groups=3, groups_kept=1, group_best=2)),
    (5, 64, dict(top_k=2, score="sigmoid", n_groups=64, groups_kept=5, normalize=False)),
    (6, 160, dict(top_k=4, n_groups=5, groups_kept=5, group_best=1)),
]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(ROUTES)))
def test_route(ctx, dev, axc, case, t):
    tokens, n, kw = ROUTES[case]
    _say(f"route {tokens}x{n} {kw} type {t}")
    logits = _spread_logits(case, tokens, n)
    values, e, w = _route(ctx, dev, axc, logits, t=t, **kw)
    if t == BF16 and n > 512:  # bf16 rounds neighbours together: ties stay ties
        assert len(np.unique(values[0])) < n
    want_e, want_w = MX.route(values, **kw)
    assert np.array_equal(e, want_e)
    assert np.allclose(w, want_w, rtol=64 * U23, atol=1e-37)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_bias_orders_but_does_not_weigh(ctx, dev, axc, score):
    rng = np.random.default_rng(3)
    # keys a multiple of 2^-6 apart: bias on that grid, scores of one value
    logits = np.zeros((4, 64), dtype=np.float32)
    logits[:, ::2] = 8 if score == "sigmoid" else 0
    bias = (rng.permutation(64).astype(np.float32) - 32) / 64
    values, e, w = _route(ctx, dev, axc, logits, bias, score=score, top_k=5)
    want_e, want_w = MX.route(values, 5, score, bias)
    assert np.array_equal(e, want_e)
    assert np.allclose(w, want_w, rtol=64 * U23)


def test_route_ties_take_the_lowest_expert(ctx, dev, axc):
    logits = np.zeros((3, 200), dtype=np.float32)
    logits[1, 150:] = 1
    logits[2, [7, 70, 130]] = [2, 2, 2]
    logits[2, 3] = -0.0
    _, e, w = _route(ctx, dev, axc, logits, top_k=4)
    assert e.tolist() == [[0, 1, 2, 3], [150, 151, 152, 153], [7, 70, 130, 0]]
    assert np.allclose(w[0], 0.25)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masked_and_special_logits(ctx, dev, axc, score):
    """-inf and NaN are never chosen; rows with nothing, or too little, left;
    the lowest finite value is no mask; +inf takes the weight."""
    inf, low = np.inf, float(np.finfo(np.float32).min)
    logits = np.full((7, 70), -inf, dtype=np.float32)
    logits[1, 69] = 0
    logits[2, :] = np.nan
    logits[2, [5, 64]] = [1, 2]
    logits[3, :] = low
    logits[4, [3, 66]] = inf
    logits[4, 10] = 0
    logits[5, :] = np.nan
    logits[6, 2] = -200.0
    values, e, w = _route(ctx, dev, axc, logits, top_k=3, score=score)
    want_e, want_w = MX.route(values, 3, score)
    assert e[0].tolist() == [-1, -1, -1] and e[5].tolist() == [-1, -1, -1]
    assert e[3].tolist() == [0, 1, 2] and e[4].tolist() == [3, 66, 10]
    assert np.array_equal(e, want_e)
    assert np.allclose(w, want_w, rtol=64 * U23, atol=1e-37)
    assert np.isfinite(w).all()


def test_route_groups_with_masked_members(ctx, dev, axc):
    """A group with fewer than group_best candidates comes last, and a kept
    group with none gives no choice."""
    logits = np.full((3, 12), -np.inf, dtype=np.float32)
    logits[0, [0, 4, 5, 8]] = [9, 1, 2, 3]
    logits[1, [0]] = 5
    logits[2, [1, 2, 9, 10]] = [0.5, 1, 2, 3]
    for best in (1, 2):
        values, e, w = _route(ctx, dev, axc, logits, top_k=4, score="sigmoid", n_groups=3,
                              groups_kept=2, group_best=best)
        want_e, want_w = MX.route(values, 4, "sigmoid", None, 3, 2, best)
        assert np.array_equal(e, want_e), best
        assert np.allclose(w, want_w, rtol=64 * U23), best


# ---- expert layers ---------------------------------------------------------------------
def _choices(seed, tokens, top_k, n_experts, holes=True):
    rng = np.random.default_rng(seed)
    e = np.stack([rng.permutation(n_experts)[:top_k] for _ in range(tokens)]).astype(np.int32)
    if holes and tokens > 2:
        e[1, 0] = -1
        e[2, :] = -1
    return e


@pytest.mark.parametrize("tokens,top_k,n", [(1, 1, 1), (3, 2, 5), (100, 8, 64), (1000, 4, 33),
                                            (5, 1, 1024), (2500, 6, 128), (64, 2, 2),
                                            (40000, 8, 61)])
def test_plan(ctx, dev, axc, tokens, top_k, n):
    _say(f"plan {tokens}x{top_k} of {n}")
    e = _choices(tokens, tokens, top_k, n)
    if tokens > 50:
        e[40:45, 0] = n  # out of range: left out
    nbytes = axc.expert_plan_bytes(tokens, top_k, n)
    dp = dev.out(nbytes)
    ctx.expert_plan(dev.up(e), dp, tokens, top_k, n)
    ctx.synchronize()
    p = dev.down(dp, nbytes, np.uint32, nbytes // 4)
    offsets, order = MX.plan(e, n)
    assert np.array_equal(p[:n + 1], offsets)
    at = (n + 1 + 15) // 16 * 16
    assert np.array_equal(p[at:at + len(order)], order)


LAYERS = [(1, 1, 1, 64, 32), (1, 4, 8, 512, 256), (3, 2, 5, 1312, 736), (2, 8, 16, 2080, 96),
          (5, 3, 7, 96, 2208), (4, 2, 3, 4096, 1056)]


def _swiglu_bound(g, u, eg, eu):
    """First order in the operands' errors, and 8 ulp of the result."""
    s = np.abs(MX.swiglu(g, np.ones_like(g)))
    return 1.1 * eg * (np.abs(u) + eu) + s * eu + 8 * U23 * np.abs(MX.swiglu(g, u))


@pytest.mark.parametrize("tokens,top_k,n,hidden,ffn", LAYERS)
def test_expert_layer_for_few_tokens(ctx, dev, tokens, top_k, n, hidden, ffn):
    _say(f"expert decode {tokens} of {n} k{top_k} {hidden}/{ffn}")
    gc, gs = MX.gen_weights(1, n, ffn, hidden)
    uc, us = MX.gen_weights(2, n, ffn, hidden)
    wc, ws = MX.gen_weights(3, n, hidden, ffn)
    e = _choices(4, tokens, top_k, n)
    x = activations(5, tokens, hidden)
    weights = np.random.default_rng(6).random((tokens, top_k)).astype(np.float32)
    slots = tokens * top_k
    dh, dy = dev.out(slots * ffn * 4), dev.out(tokens * hidden * 4)
    de = dev.up(e)
    ctx.mxfp4_expert_gate_up(dev.up(gc), dev.up(gs), dev.up(uc), dev.up(us), dev.up(x), de, dh, ffn,
                             hidden, tokens, top_k, n)
    ctx.mxfp4_expert_down(dev.up(wc), dev.up(ws), dh, de, dev.up(weights), dy, hidden, ffn, tokens,
                          top_k, n)
    ctx.synchronize()
    h = dev.down(dh, slots * ffn * 4, np.float32, (tokens, top_k, ffn)).astype(np.float64)
    y = dev.down(dy, tokens * hidden * 4, np.float32, (tokens, hidden)).astype(np.float64)
    for t in range(tokens):
        want, bound = np.zeros(hidden), np.zeros(hidden)
        for k in range(top_k):
            if e[t, k] < 0:
                assert (h[t, k] == 0).all()
                continue
            xd = x[t].astype(np.float64)
            wg, wu = (MX.decode(c[e[t, k]], s[e[t, k]]) for c, s in ((gc, gs), (uc, us)))
            g, u = wg @ xd, wu @ xd
            eg, eu = (hidden * U24 * (np.abs(m) @ np.abs(xd)) for m in (wg, wu))
            assert (np.abs(h[t, k] - MX.swiglu(g, u)) <= _swiglu_bound(g, u, eg, eu)).all()
            wd = MX.decode(wc[e[t, k]], ws[e[t, k]])
            want += float(weights[t, k]) * (wd @ h[t, k])
            bound += (ffn + top_k + 1) * U24 * weights[t, k] * (np.abs(wd) @ np.abs(h[t, k]))
        assert (np.abs(y[t] - want) <= bound).all()


PROMPTS = [(1, 1, 1, 64, 32), (7, 2, 5, 288, 64), (40, 4, 8, 512, 256), (333, 6, 40, 416, 96),
           (300, 4, 4, 1312, 160), (700, 3, 8, 544, 288), (260, 1, 1, 256, 64),
           (333, 6, 40, 544, 544), (300, 2, 130, 544, 576), (2100, 1, 2, 544, 1056)]


@pytest.mark.parametrize("t", [F32, F16, BF16, MXFP4])
@pytest.mark.parametrize("tokens,top_k,n,hidden,ffn", PROMPTS)
def test_expert_products_for_prompts(ctx, dev, axc, tokens, top_k, n, hidden, ffn, t):
    """gate/up into every type of h, then the down product of what it holds."""
    _say(f"expert prompt {tokens} of {n} k{top_k} {hidden}/{ffn} type {t}")
    gc, gs = MX.gen_weights(1, n, ffn, hidden)
    uc, us = MX.gen_weights(2, n, ffn, hidden)
    e = _choices(4, tokens, top_k, n)
    xc, xs = MX.quantize(activations(5, tokens, hidden))
    slots = tokens * top_k
    dp = dev.out(axc.expert_plan_bytes(tokens, top_k, n))
    ctx.expert_plan(dev.up(e), dp, tokens, top_k, n)
    size = slots * ffn // 2 if t == MXFP4 else slots * ffn * SIZE[t]
    dh, ds = dev.out(size), dev.out(slots * ffn // 32)
    ctx.mxfp4_expert_gate_up_matmul(dev.up(gc), dev.up(gs), dev.up(uc), dev.up(us), dev.up(xc),
                                    dev.up(xs), dp, dh, ds if t == MXFP4 else None, ffn, hidden,
                                    tokens, top_k, n, t)
    ctx.synchronize()
    x = MX.decode(xc, xs)
    if t == MXFP4:
        hc = dev.down(dh, size, np.uint8, (slots, ffn // 2))
        hs = dev.down(ds, slots * ffn // 32, np.uint8, (slots, ffn // 32))
    else:
        h = read_out(dev, dh, t, (slots, ffn))
    flat = e.reshape(-1)
    for ex in range(n):
        mine = np.nonzero(flat == ex)[0]
        if not len(mine):
            continue
        xm = x[mine // top_k]
        wg, wu = MX.decode(gc[ex], gs[ex]), MX.decode(uc[ex], us[ex])
        g, u = xm @ wg.T, xm @ wu.T
        eg, eu = (hidden * U23 * (np.abs(xm) @ np.abs(m).T) for m in (wg, wu))
        want, bound = MX.swiglu(g, u), _swiglu_bound(g, u, eg, eu)
        if t != MXFP4:
            assert (np.abs(h[mine] - want) <= bound + ROUND[t] * (np.abs(want) + bound) + (
                2.0 ** -25 if t == F16 else 0)).all()
            continue
        # the scale may be the next one where the maximum is next to a power of
        # two; an element is within half a step of what its own scale allows
        block = want.reshape(len(mine), -1, 32)
        eb = bound.reshape(block.shape)
        lo, hi = (MX.quantize(np.maximum(np.abs(block) + s * eb, 0).reshape(len(mine), -1))[1]
                  for s in (-1, 1))
        got_s = hs[mine]
        assert ((got_s >= lo) & (got_s <= hi)).all()
        a = np.abs(block) / np.exp2(got_s.astype(np.float64) - 127)[..., None]
        step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
        scale = np.exp2(got_s.astype(np.float64) - 127)[..., None]
        got = MX.decode(hc[mine], got_s).reshape(block.shape)
        # (values near 2 and 4 may take the step of either side; 8 saturates to 6)
        assert (np.abs(got - block) <= step * scale * (1 + 1e-5) + eb).all()
        near = np.abs(got - block) > 0.5 * step * scale + eb
        assert not (near & (a < 6)).any()
    left = np.nonzero(flat < 0)[0]
    if t == MXFP4 and len(left):
        assert (hc[left] == 0xA5).all() and (hs[left] == 0xA5).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,top_k,n,hidden,ffn", PROMPTS)
def test_expert_down_and_combine(ctx, dev, axc, tokens, top_k, n, hidden, ffn, t):
    _say(f"expert down {tokens} of {n} k{top_k} {hidden}/{ffn} type {t}")
    wc, ws = MX.gen_weights(3, n, hidden, ffn)
    e = _choices(4, tokens, top_k, n)
    slots = tokens * top_k
    hc, hs = MX.quantize(activations(7, slots, ffn))
    weights = np.random.default_rng(6).random((tokens, top_k)).astype(np.float32)
    dp = dev.out(axc.expert_plan_bytes(tokens, top_k, n))
    de = dev.up(e)
    ctx.expert_plan(de, dp, tokens, top_k, n)
    d_slots, dy = dev.out(slots * hidden * SIZE[t]), dev.out(tokens * hidden * SIZE[t])
    ctx.mxfp4_expert_matmul(dev.up(wc), dev.up(ws), dev.up(hc), dev.up(hs), dp, d_slots, hidden,
                            ffn, tokens, top_k, n, t)
    ctx.expert_combine(d_slots, de, dev.up(weights), dy, hidden, tokens, top_k, t)
    ctx.synchronize()
    got = read_out(dev, d_slots, t, (tokens, top_k, hidden))
    y = read_out(dev, dy, t, (tokens, hidden))
    h = MX.decode(hc, hs).reshape(tokens, top_k, ffn)
    exact, bound = np.zeros(got.shape), np.zeros(got.shape)
    for ex in range(n):
        at = np.nonzero(e == ex)
        if not len(at[0]):
            continue
        w = MX.decode(wc[ex], ws[ex])
        exact[at] = h[at] @ w.T
        bound[at] = ffn * U23 * (np.abs(h[at]) @ np.abs(w).T)
    real = (e >= 0)[..., None]
    bound += ROUND[t] * (np.abs(exact) + bound) + (2.0 ** -25 if t == F16 else 0)
    assert (np.abs(np.where(real, got, 0) - exact) <= bound).all()
    wd = weights.astype(np.float64)[..., None]
    got = np.where(real, got, 0)
    want = (wd * got).sum(axis=1)
    most = (wd * np.abs(got)).sum(axis=1)
    assert (np.abs(y - want) <= (top_k * U24 + ROUND[t]) * most * 1.01 + (
        2.0 ** -25 if t == F16 else 0)).all()


# rows of fewer than 16 blocks through the 128 x 128 tiles: matrices, prompts, blocks 1 to 15
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,batch", [(2000, 32, 1700), (1801, 256, 1665), (2000, 288, 1700),
                                             (3500, 480, 900)])
def test_matmul_short_rows(ctx, dev, axc, rows, cols, batch, t):
    assert "_t128x128n_" in axc.mxfp4_matmul_kernel_name(rows, cols, batch, t)
    test_matmul(ctx, dev, axc, rows, cols, batch, t)


@pytest.mark.parametrize("t", [F32, F16, BF16, MXFP4])
@pytest.mark.parametrize("tokens,top_k,n,hidden,ffn", [(700, 2, 8, 96, 160), (400, 3, 5, 480, 32),
                                                       (260, 1, 3, 256, 288)])
def test_expert_products_short_rows(ctx, dev, axc, tokens, top_k, n, hidden, ffn, t):
    test_expert_products_for_prompts(ctx, dev, axc, tokens, top_k, n, hidden, ffn, t)
    if t != MXFP4:
        test_expert_down_and_combine(ctx, dev, axc, tokens, top_k, n, hidden, ffn, t)


@pytest.mark.parametrize("cols", [1, 7, 33, 2049, 4096])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_combine_odd_columns(ctx, dev, cols, t):
    tokens, top_k = 5, 3
    raw, v = as_type(activations(cols, tokens * top_k, cols), t)
    e = np.array([[0, 1, 2], [3, -1, 0], [-1, -1, -1], [9, 1, 0], [1, 1, 1]], dtype=np.int32)
    w = np.random.default_rng(1).random((tokens, top_k)).astype(np.float32)
    dy = dev.out(tokens * cols * SIZE[t])
    ctx.expert_combine(dev.up(raw), dev.up(e), dev.up(w), dy, cols, tokens, top_k, t, n_experts=9)
    ctx.synchronize()
    y = read_out(dev, dy, t, (tokens, cols))
    use = ((e >= 0) & (e < 9))[..., None] * w.astype(np.float64)[..., None]
    v = v.astype(np.float64).reshape(tokens, top_k, cols)
    want, most = (use * v).sum(axis=1), (use * np.abs(v)).sum(axis=1)
    assert (y[2] == 0).all()
    assert (np.abs(y - want) <= (top_k * U24 + ROUND[t]) * most * 1.01 + (
        2.0 ** -25 if t == F16 else 0)).all()


def test_calls_on_another_stream_and_in_a_graph(ctx, dev, axc):
    """One MXFP4 linear layer on another stream, and recorded in a graph, replay
    after replay with eager work between, gives the eager result."""
    rows, cols, batch = 160, 544, 40
    wc, ws = MX.gen_weights(1, rows, cols)
    x = activations(2, batch, cols)
    dx, dwc, dws = dev.up(x), dev.up(wc), dev.up(ws)
    dc, ds, dy = dev.out(batch * cols // 2), dev.out(batch * cols // 32), dev.out(rows * batch * 4)

    def step(stream=None):
        ctx.mxfp4_quantize(dx, dc, ds, batch, cols, stream=stream)
        ctx.mxfp4_matmul(dwc, dws, dc, ds, dy, rows, cols, batch, stream=stream)

    step()
    ctx.synchronize()
    eager = dev.down(dy, rows * batch * 4, np.float32, (batch, rows))
    other = axc.HipContext.new()
    ctx.upload(dy, np.zeros(rows * batch * 4, dtype=np.uint8))
    step(other.stream)
    ctx.synchronize(other.stream)
    assert np.array_equal(dev.down(dy, rows * batch * 4, np.float32, (batch, rows)), eager)
    other.close()
    g = ctx.capture(step)
    assert g.node_count == 2
    for _ in range(3):
        ctx.upload(dy, np.zeros(rows * batch * 4, dtype=np.uint8))
        g.launch()
        ctx.synchronize()
        assert np.array_equal(dev.down(dy, rows * batch * 4, np.float32, (batch, rows)), eager)
        step()
        ctx.synchronize()
    g.close()


# ---- an expert layer from a file -----------------------------------------------------------
def _layer_file(axc, path, n, hidden, ffn, bias):
    """Writes the layer blk.3 and returns its matrices, in 64 bits."""
    gg, out, tensors = axc.gguf, {}, []
    for i, (name, rows, cols) in enumerate((("ffn_gate_inp", (n,), hidden),
                                            ("ffn_gate_exps", (n, ffn), hidden),
                                            ("ffn_up_exps", (n, ffn), hidden),
                                            ("ffn_down_exps", (n, hidden), ffn))):
        c, s = MX.gen_weights(20 + i, *rows, cols)
        out[name] = MX.decode(c, s)
        tensors.append((f"blk.3.{name}.weight", MXFP4, (cols,) + rows[::-1],
                        MX.to_ggml(c, s).tobytes()))
    if bias is not None:
        tensors.append(("blk.3.exp_probs_b.bias", F32, (n,), bias.tobytes()))
    gg.write_gguf(path, [], tensors)
    return out


@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 70])
def test_expert_layer_from_a_file(ctx, dev, axc, tmp_path, tokens):
    """Each step of a layer's run against the formulas on the step before it, and
    three replays of it in a graph."""
    n, k, hidden, ffn = 12, 3, 544, 576
    _say(f"expert layer, {tokens} tokens")
    bias = np.linspace(-0.2, 0.2, n, dtype=np.float32)
    w = _layer_file(axc, tmp_path / "layer.gguf", n, hidden, ffn, bias)
    options = axc.RouteOptions(n_experts=n, top_k=k, score="sigmoid")
    with axc.gguf.GgufFile(tmp_path / "layer.gguf") as f:
        layer = axc.experts.ExpertLayer(ctx, f, "blk.3", options, max_tokens=70)
    x = activations(30, tokens, hidden)
    dx, dy = dev.up(x), dev.out(tokens * hidden * 4)
    layer.run(dx, dy, tokens)
    ctx.synchronize()
    y = dev.down(dy, tokens * hidden * 4, np.float32, (tokens, hidden))

    def get(buf, dtype, shape):
        nbytes = int(np.prod(shape)) * np.dtype(dtype).itemsize
        return np.frombuffer(ctx.download(buf, nbytes), dtype=dtype).reshape(shape)

    few = tokens <= layer.few_tokens
    xq = MX.decode(*MX.quantize(x))
    xr = x.astype(np.float64) if tokens == 1 else xq
    logits = get(layer.logits, np.float32, (tokens, n)).astype(np.float64)
    bound = hidden * U23 * (np.abs(xr) @ np.abs(w["ffn_gate_inp"]).T)
    assert (np.abs(logits - xr @ w["ffn_gate_inp"].T) <= bound).all()
    e, wt = MX.route(logits, k, "sigmoid", bias=bias)
    assert np.array_equal(get(layer.experts, np.int32, (tokens, k)), e)
    got = get(layer.weights, np.float32, (tokens, k)).astype(np.float64)
    assert (np.abs(got - wt) <= 64 * U23 * np.abs(wt)).all()
    if few:
        h = get(layer.h, np.float32, (tokens, k, ffn)).astype(np.float64)
    else:
        h = MX.decode(get(layer.h_codes, np.uint8, (tokens, k, ffn // 2)),
                      get(layer.h_scales, np.uint8, (tokens, k, ffn // 32)))
    for t in range(tokens):
        want, bound = np.zeros(hidden), np.zeros(hidden)
        for i in range(k):
            xt = x[t].astype(np.float64) if few else xq[t]
            wg, wu = w["ffn_gate_exps"][e[t, i]], w["ffn_up_exps"][e[t, i]]
            exact = MX.swiglu(wg @ xt, wu @ xt)
            ulp = _swiglu_bound(wg @ xt, wu @ xt, *(hidden * U23 * (np.abs(m) @ np.abs(xt))
                                                    for m in (wg, wu)))
            # MXFP4: half a step, or what is cut off above 6, is at most a quarter of the
            # block's largest magnitude
            step = 0 if few else np.repeat(np.abs(exact).reshape(-1, 32).max(axis=1) / 4, 32)
            assert (np.abs(h[t, i] - exact) <= ulp + step).all()
            wd = w["ffn_down_exps"][e[t, i]]
            want += got[t, i] * (wd @ h[t, i])
            bound += (2 * ffn + k + 1) * U24 * got[t, i] * (np.abs(wd) @ np.abs(h[t, i]))
        assert (np.abs(y[t] - want) <= bound).all()
    g = ctx.capture(lambda: layer.run(dx, dy, tokens))
    for _ in range(3):
        ctx.upload(dy, np.zeros(tokens * hidden * 4, dtype=np.uint8))
        g.launch()
        ctx.synchronize()
        assert np.array_equal(dev.down(dy, tokens * hidden * 4, np.float32, y.shape), y)
        layer.run(dx, dy, tokens)
        ctx.synchronize()
    g.close()
    layer.close()


def test_expert_layer_refuses_a_router_of_another_type(ctx, axc, tmp_path):
    n, hidden, path = 4, 64, tmp_path / "layer.gguf"
    _layer_file(axc, path, n, hidden, 32, None)
    with axc.gguf.GgufFile(path) as f:
        rest = [(name, s.type, tuple(s.shape), f.tensor_bytes(name))
                for name, s in f.tensors.items() if "gate_inp" not in name]
    axc.gguf.write_gguf(path, [], [("blk.3.ffn_gate_inp.weight", 2, (hidden, n),
                                    bytes(n * hidden // 32 * 18))] + rest)
    with axc.gguf.GgufFile(path) as f, pytest.raises(ValueError, match="is of type 2"):
        axc.experts.ExpertLayer(ctx, f, "blk.3", axc.RouteOptions(n_experts=n, top_k=1),
                                max_tokens=8)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [1, 3, 70])
def test_expert_layer_with_a_router_of_floats(ctx, dev, axc, tmp_path, tokens, t):
    """The layer is the calls one after another, with the router's product in f32."""
    n, k, hidden, ffn = 12, 3, 544, 576
    _say(f"expert layer, router of type {t}, {tokens} tokens")
    path = tmp_path / "layer.gguf"
    _layer_file(axc, path, n, hidden, ffn, None)
    rng = np.random.default_rng(50)
    raw, w = as_type(rng.standard_normal((n, hidden)).astype(np.float32) / 16, t)
    with axc.gguf.GgufFile(path) as f:
        rest = [(name, s.type, tuple(s.shape), f.tensor_bytes(name))
                for name, s in f.tensors.items() if "gate_inp" not in name]
    axc.gguf.write_gguf(path, [], [("blk.3.ffn_gate_inp.weight", t, (hidden, n),
                                    raw.tobytes())] + rest)
    options = axc.RouteOptions(n_experts=n, top_k=k)
    with axc.gguf.GgufFile(path) as f:
        layer = axc.experts.ExpertLayer(ctx, f, "blk.3", options, max_tokens=70, few_tokens=4)
    x = activations(51, tokens, hidden)
    dx, dy = dev.up(x), dev.out(tokens * hidden * 4)
    layer.run(dx, dy, tokens)
    ctx.synchronize()
    y = dev.down(dy, tokens * hidden * 4, np.float32, (tokens, hidden))
    logits = np.frombuffer(ctx.download(layer.logits, tokens * n * 4), dtype=np.float32)
    logits = logits.reshape(tokens, n).astype(np.float64)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    assert (np.abs(logits - x64 @ w64.T)
            <= (hidden + 1) * U23 * (np.abs(x64) @ np.abs(w64).T)).all()
    chosen = np.frombuffer(ctx.download(layer.experts, tokens * k * 4), dtype=np.int32)
    assert np.array_equal(chosen.reshape(tokens, k), MX.route(logits, k)[0])
    again = dev.out(tokens * hidden * 4)
    g, u, d = layer.gate, layer.up, layer.down
    if tokens <= 4:
        ctx.mxfp4_expert_gate_up(g.codes, g.scales, u.codes, u.scales, dx, layer.experts, layer.h,
                                 ffn, hidden, tokens, k, n)
        ctx.mxfp4_expert_down(d.codes, d.scales, layer.h, layer.experts, layer.weights, again,
                              hidden, ffn, tokens, k, n)
    else:
        ctx.mxfp4_quantize(dx, layer.x_codes, layer.x_scales, tokens, hidden)
        ctx.expert_plan(layer.experts, layer.plan, tokens, k, n)
        ctx.mxfp4_expert_gate_up_matmul(g.codes, g.scales, u.codes, u.scales, layer.x_codes,
                                        layer.x_scales, layer.plan, layer.h_codes, layer.h_scales,
                                        ffn, hidden, tokens, k, n)
        ctx.mxfp4_expert_matmul(d.codes, d.scales, layer.h_codes, layer.h_scales, layer.plan,
                                layer.slots, hidden, ffn, tokens, k, n)
        ctx.expert_combine(layer.slots, layer.experts, layer.weights, again, hidden, tokens, k,
                           n_experts=n)
    ctx.synchronize()
    assert np.array_equal(dev.down(again, tokens * hidden * 4, np.float32, y.shape), y)
    graph = ctx.capture(lambda: layer.run(dx, dy, tokens))
    for _ in range(3):
        ctx.upload(dy, np.zeros(tokens * hidden * 4, dtype=np.uint8))
        graph.launch()
        ctx.synchronize()
        assert np.array_equal(dev.down(dy, tokens * hidden * 4, np.float32, y.shape), y)
    graph.close()
    layer.close()


def test_expert_layer_refusals(ctx, axc, tmp_path):
    _layer_file(axc, tmp_path / "layer.gguf", 4, 64, 32, np.zeros(4, dtype=np.float32))
    with axc.gguf.GgufFile(tmp_path / "layer.gguf") as f:
        make = axc.experts.ExpertLayer
        for prefix, n, t in (("blk.4", 4, 8), ("blk.3", 5, 8), ("blk.3", 4, 0)):
            with pytest.raises(ValueError):
                make(ctx, f, prefix, axc.RouteOptions(n_experts=n, top_k=1), max_tokens=t)
        layer = make(ctx, f, "blk.3", axc.RouteOptions(n_experts=4, top_k=1), max_tokens=8)
    with pytest.raises(ValueError):
        layer.run(layer.slots, layer.slots, 9)
    layer.run(layer.slots, layer.slots, 0)
    layer.close()


# ---- refusals ------------------------------------------------------------------------------
def test_refusals(ctx, dev, axc):
    """Every bad argument is a typed error before any launch: buffers stay as
    they were."""
    p = dev.out(1 << 16)
    R = axc.RouteOptions

    def q(**k):
        a = dict(x=p, codes=p, scales=p, rows=2, cols=64, x_type=F32, x_stride=0) | k
        ctx.mxfp4_quantize(a["x"], a["codes"], a["scales"], a["rows"], a["cols"], a["x_type"],
                           a["x_stride"])

    def mm(**k):
        a = dict(w=p, ws=p, x=p, xs=p, y=p, rows=2, cols=64, batch=2, t=F32) | k
        ctx.mxfp4_matmul(a["w"], a["ws"], a["x"], a["xs"], a["y"], a["rows"], a["cols"],
                         a["batch"], a["t"])

    def mv(**k):
        a = dict(w=p, ws=p, x=p, y=p, rows=2, cols=64) | k
        ctx.mxfp4_matvec(a["w"], a["ws"], a["x"], a["y"], a["rows"], a["cols"])

    def route(o, l=p, b=None, e=p, w=p, t=F32):
        ctx.expert_route(l, b, e, w, 3, o, t)

    def gu(**k):
        a = dict(w=p, ws=p, x=p, e=p, h=p, rows=2, cols=64, tokens=2, k=2, n=4) | k
        ctx.mxfp4_expert_gate_up(a["w"], a["ws"], p, p, a["x"], a["e"], a["h"], a["rows"],
                                 a["cols"], a["tokens"], a["k"], a["n"])

    def down(**k):
        a = dict(w=p, h=p, e=p, wt=p, y=p, rows=2, cols=64, tokens=2, k=2, n=4) | k
        ctx.mxfp4_expert_down(a["w"], p, a["h"], a["e"], a["wt"], a["y"], a["rows"], a["cols"],
                              a["tokens"], a["k"], a["n"])

    def gum(**k):
        a = dict(w=p, x=p, plan=p, h=p, hs=p, rows=32, cols=64, tokens=2, k=2, n=4, t=MXFP4) | k
        ctx.mxfp4_expert_gate_up_matmul(a["w"], p, p, p, a["x"], p, a["plan"], a["h"], a["hs"],
                                        a["rows"], a["cols"], a["tokens"], a["k"], a["n"], a["t"])

    def em(**k):
        a = dict(w=p, x=p, plan=p, y=p, rows=32, cols=64, tokens=2, k=2, n=4, t=F32) | k
        ctx.mxfp4_expert_matmul(a["w"], p, a["x"], p, a["plan"], a["y"], a["rows"], a["cols"],
                                a["tokens"], a["k"], a["n"], a["t"])

    def comb(**k):
        a = dict(s=p, e=p, w=p, y=p, rows=8, tokens=2, k=2, t=F32) | k
        ctx.expert_combine(a["s"], a["e"], a["w"], a["y"], a["rows"], a["tokens"], a["k"], a["t"])

    bad = [
        *(lambda f=f, c=c: f(cols=c) for f in (q, mm, mv, gu, down, gum, em)
          for c in (0, 16, 33, 1 << 23)),
        *(lambda n=n: q(**{n: None}) for n in ("x", "codes", "scales")),
        lambda: q(x=p + 8), lambda: q(codes=p + 4), lambda: q(x_type=MXFP4), lambda: q(x_type=2),
        lambda: q(x_stride=63), lambda: q(x_stride=66), lambda: q(x_type=F16, x_stride=68),
        lambda: q(rows=1 << 31, cols=1 << 22),
        *(lambda n=n: mm(**{n: None}) for n in ("w", "ws", "x", "xs", "y")),
        lambda: mm(w=p + 8), lambda: mm(x=p + 8), lambda: mm(y=p + 2), lambda: mm(t=MXFP4),
        lambda: mm(y=p + 1, t=BF16),
        *(lambda n=n: mv(**{n: None}) for n in ("w", "ws", "x", "y")),
        lambda: mv(w=p + 8), lambda: mv(x=p + 4), lambda: mv(y=p + 2),
        lambda: route(R(0, 1)), lambda: route(R(1025, 1)), lambda: route(R(8, 0)),
        lambda: route(R(8, 9)), lambda: route(R(200, 65)), lambda: route(R(8, 2, n_groups=3)),
        lambda: route(R(8, 2, n_groups=2, groups_kept=0)),
        lambda: route(R(8, 2, n_groups=2, groups_kept=3)),
        lambda: route(R(8, 5, n_groups=2, groups_kept=1)),
        lambda: route(R(8, 2, n_groups=2, group_best=3)),
        lambda: route(R(130, 2, n_groups=65, groups_kept=2)),
        lambda: route(R(8, 2, scale=float("nan"))), lambda: route(R(8, 2, scale=float("inf"))),
        lambda: route(R(8, 2), l=None), lambda: route(R(8, 2), e=None),
        lambda: route(R(8, 2), w=None), lambda: route(R(8, 2), l=p + 2),
        lambda: route(R(8, 2), b=p + 2), lambda: route(R(8, 2), t=MXFP4),
        *(lambda f=f, n=n: f(n=n) for f in (gu, down, gum, em) for n in (0, 1025)),
        *(lambda f=f, k=k: f(k=k) for f in (gu, down, gum, em, comb) for k in (0, 65)),
        *(lambda f=f: f(tokens=1 << 31) for f in (gu, down, gum, em)),
        lambda: gu(tokens=40000), lambda: down(tokens=40000),
        *(lambda n=n: gu(**{n: None}) for n in ("w", "ws", "x", "e", "h")),
        lambda: gu(x=p + 4), lambda: gu(w=p + 8), lambda: gu(rows=1 << 16, cols=1 << 20),
        *(lambda n=n: down(**{n: None}) for n in ("w", "h", "e", "wt", "y")),
        lambda: down(h=p + 4), lambda: down(y=p + 2),
        *(lambda n=n: gum(**{n: None}) for n in ("w", "x", "plan", "h", "hs")),
        lambda: gum(rows=33), lambda: gum(t=2), lambda: gum(h=p + 8), lambda: gum(plan=p + 2),
        lambda: gum(x=p + 8), lambda: gum(tokens=1 << 12, cols=1 << 20, k=1),
        *(lambda n=n: em(**{n: None}) for n in ("w", "x", "plan", "y")),
        lambda: em(t=MXFP4), lambda: em(y=p + 2), lambda: em(x=p + 8),
        lambda: em(tokens=1 << 12, cols=1 << 20, k=1),
        *(lambda n=n: comb(**{n: None}) for n in ("s", "e", "w", "y")),
        lambda: comb(t=MXFP4), lambda: comb(s=p + 8), lambda: comb(y=p + 4),
        lambda: ctx.mxfp4_dequant(p, p, p, 1, MXFP4), lambda: ctx.mxfp4_dequant(None, p, p, 1),
        lambda: ctx.mxfp4_dequant(p + 2, p, p, 1), lambda: ctx.mxfp4_dequant(p, p, p + 4, 1),
        lambda: ctx.mxfp4_dequant(p, p, p, 1 << 30),
        lambda: ctx.mxfp4_unpack_ggml(None, p, p, 1), lambda: ctx.mxfp4_unpack_ggml(p, p + 1, p, 1),
        lambda: ctx.expert_plan(None, p, 1, 1, 1), lambda: ctx.expert_plan(p, p + 2, 1, 1, 1),
        lambda: ctx.expert_plan(p, p, 1, 1, 0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(axc.DispatchError) as err:
            call()
            pytest.fail(f"call {i} was accepted")
        assert err.value.variant == "InvalidArgument", i
    # nothing to do
    q(rows=0), mm(rows=0), mm(batch=0), mv(rows=0), gu(rows=0), gu(tokens=0), down(tokens=0)
    gum(tokens=0), em(rows=0), comb(tokens=0), comb(rows=0)
    ctx.expert_route(None, None, None, None, 0, R(8, 2))
    ctx.mxfp4_dequant(None, None, None, 0)
    ctx.expert_plan(None, None, 0, 1, 1)
    ctx.synchronize()
    assert (dev.down(p, 1 << 16, np.uint8, (1 << 16,)) == 0xA5).all()
