"""MXFP4 products and expert layers on the GPU (marked `gpu`) where values are not ordinary:
NaN blocks in every kernel, and gates over the whole range of silu.

NaN: a scale byte of 255 reaches the outputs that its row (column, expert) is part of and no
other, and these are, bit for bit, those of the same call without it.
Gates: g and u are sums of a few powers of two, exact in f32 in any order.  silu(g) * u is
within 8 ulp; below g = -87.3, where the reciprocal may be 0, silu(g) is within 2e-36."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import mx_numpy as MX
import test_gpu_mx
from test_gpu_mx import BF16, F16, F32, MXFP4, U23, Dev, _choices, _say, activations

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    ctx.synchronize()
    d.close()


def _plant(scales, rows):
    """NaN blocks in rows of (..., rows, blocks) scales, taken as one array of rows: in the last
    block of the array, in the first of its neighbours, and in first, last and middle blocks."""
    flat = scales.reshape(-1, scales.shape[-1])
    n, blocks = flat.shape
    out = np.zeros(n, dtype=bool)
    for row, block in ((n - 1, blocks - 1), (0, 0), (rows // 2, blocks - 1),
                       (min(rows // 2 + 2, n - 1), 0), (rows - 1, blocks // 2),
                       (min(rows, n - 1), blocks - 1)):
        flat[row, block] = 255
        out[row] = True
    return out.reshape(scales.shape[:-1])


# rows, cols, batch, kernel; rows of 1, 8, 9 and 15 blocks for the tiles of short rows
DENSE = [(2000, 32, 1665, "t128x128n"), (2000, 256, 1665, "t128x128n"),
         (2000, 288, 1665, "t128x128n"), (2000, 480, 1665, "t128x128n"),
         (1999, 96, 1601, "t128x128n"), (2100, 544, 520, "t64x128"), (1700, 544, 1800, "t128x128"),
         (1700, 1056, 1800, "t128x128"), (3900, 512, 3300, "t256x256"),
         (3900, 800, 3300, "t256x256"), (40, 10272, 20, "k16"), (70, 224, 20, "k32"),
         (70, 288, 20, "k32"), (1100, 736, 300, "t64x64s2"), (16500, 544, 33, "t64x64")]


@pytest.mark.parametrize("rows,cols,batch,kernel", DENSE)
def test_nan_blocks_of_a_product_stay_in_their_rows(ctx, dev, axc, rows, cols, batch, kernel):
    assert f"_{kernel}_" in axc.mxfp4_matmul_kernel_name(rows, cols, batch)
    _say(f"NaN blocks, {kernel} {rows}x{cols}x{batch}")
    wc, ws = MX.gen_weights(1, rows, cols)
    xc, xs = MX.quantize(activations(2, batch, cols))
    dwc, dxc, dy = dev.up(wc), dev.up(xc), dev.out(rows * batch * 4)

    def product():
        ctx.mxfp4_matmul(dwc, dev.up(ws), dxc, dev.up(xs), dy, rows, cols, batch)
        ctx.synchronize()
        return dev.down(dy, rows * batch * 4, np.float32, (batch, rows))

    clean = product()
    assert np.isfinite(clean).all()
    nan = _plant(ws, rows)[None, :] | _plant(xs, batch)[:, None]
    y = product()
    assert np.array_equal(np.isnan(y), nan)
    assert np.array_equal(y[~nan], clean[~nan])


# tokens, top_k, experts, hidden, ffn: the K-split kernels (rows of 9 and 2, 2 and 8 blocks),
# the tiles of short rows (15 and 1, 8 and 9, 17 and 5), of 128 x 64, 128 x 128 and 256 x 256
LAYERS = [(7, 2, 5, 288, 64), (7, 2, 5, 64, 256), (400, 3, 5, 480, 32), (260, 1, 3, 256, 288),
          (300, 4, 4, 544, 160), (333, 6, 40, 544, 544), (700, 3, 8, 544, 576),
          (2100, 1, 2, 544, 1056)]


@pytest.mark.parametrize("h_type", [F32, MXFP4])
@pytest.mark.parametrize("tokens,top_k,n,hidden,ffn", LAYERS)
def test_nan_blocks_of_expert_products(ctx, dev, axc, tokens, top_k, n, hidden, ffn, h_type):
    _say(f"NaN blocks, {tokens} of {n} k{top_k} {hidden}/{ffn}, h of type {h_type}")
    gc, gs = MX.gen_weights(1, n, ffn, hidden)
    uc, us = MX.gen_weights(2, n, ffn, hidden)
    wc, ws = MX.gen_weights(3, n, hidden, ffn)
    e = _choices(4, tokens, top_k, n)
    flat, slots = e.reshape(-1), tokens * top_k
    real = np.nonzero(flat >= 0)[0]
    xc, xs = MX.quantize(activations(5, tokens, hidden))
    hc, hs = MX.quantize(activations(6, slots, ffn))
    dp = dev.out(axc.expert_plan_bytes(tokens, top_k, n))
    ctx.expert_plan(dev.up(e), dp, tokens, top_k, n)
    codes = [dev.up(a) for a in (gc, uc, wc, xc, hc)]
    size = slots * ffn // 2 if h_type == MXFP4 else slots * ffn * 4

    def products():
        g, u, w, x, h = codes
        dh, dhs, dy = dev.out(size), dev.out(slots * ffn // 32), dev.out(slots * hidden * 4)
        ctx.mxfp4_expert_gate_up_matmul(g, dev.up(gs), u, dev.up(us), x, dev.up(xs), dp, dh,
                                        dhs if h_type == MXFP4 else None, ffn, hidden, tokens,
                                        top_k, n, h_type)
        ctx.mxfp4_expert_matmul(w, dev.up(ws), h, dev.up(hs), dp, dy, hidden, ffn, tokens, top_k, n)
        ctx.synchronize()
        if h_type == MXFP4:
            out = MX.decode(dev.down(dh, size, np.uint8, (slots, ffn // 2)),
                            dev.down(dhs, slots * ffn // 32, np.uint8, (slots, ffn // 32)))
        else:
            out = dev.down(dh, size, np.float32, (slots, ffn))
        return out[real], dev.down(dy, slots * hidden * 4, np.float32, (slots, hidden))[real]

    clean = products()
    assert all(np.isfinite(a).all() for a in clean)
    of = flat[real]
    token_nan, slot_nan = _plant(xs, tokens), _plant(hs, slots)
    h_nan = (_plant(gs, ffn) | _plant(us, ffn))[of] | token_nan[real // top_k][:, None]
    y_nan = _plant(ws, hidden)[of] | slot_nan[real][:, None]
    if h_type == MXFP4:  # one NaN makes its block of 32 one
        h_nan = np.repeat(h_nan.reshape(len(real), -1, 32).any(axis=2), 32, axis=1)
    for got, before, nan in zip(products(), clean, (h_nan, y_nan)):
        assert np.array_equal(np.isnan(got), nan)
        assert np.array_equal(got[~nan], before[~nan])


@pytest.mark.parametrize("tokens,top_k,n,hidden,ffn", [(1, 2, 3, 96, 64), (3, 2, 5, 1024, 544),
                                                       (2, 3, 4, 2080, 1056)])
def test_nan_blocks_of_expert_layers_for_few_tokens(ctx, dev, tokens, top_k, n, hidden, ffn):
    _say(f"NaN blocks, few tokens, {tokens} of {n} k{top_k} {hidden}/{ffn}")
    gc, gs = MX.gen_weights(1, n, ffn, hidden)
    uc, us = MX.gen_weights(2, n, ffn, hidden)
    wc, ws = MX.gen_weights(3, n, hidden, ffn)
    e = _choices(4, tokens, top_k, n, holes=False)
    slots = tokens * top_k
    h = activations(6, slots, ffn)
    weights = np.random.default_rng(7).random((tokens, top_k)).astype(np.float32)
    codes = [dev.up(a) for a in (gc, uc, wc)]
    dx, de, dw = dev.up(activations(5, tokens, hidden)), dev.up(e), dev.up(weights)

    def products():
        dh, dy = dev.out(slots * ffn * 4), dev.out(tokens * hidden * 4)
        ctx.mxfp4_expert_gate_up(codes[0], dev.up(gs), codes[1], dev.up(us), dx, de, dh, ffn,
                                 hidden, tokens, top_k, n)
        ctx.mxfp4_expert_down(codes[2], dev.up(ws), dev.up(h), de, dw, dy, hidden, ffn, tokens,
                              top_k, n)
        ctx.synchronize()
        return (dev.down(dh, slots * ffn * 4, np.float32, (slots, ffn)),
                dev.down(dy, tokens * hidden * 4, np.float32, (tokens, hidden)))

    clean = products()
    assert all(np.isfinite(a).all() for a in clean)
    h_nan = (_plant(gs, ffn) | _plant(us, ffn))[e.reshape(-1)]
    y_nan = _plant(ws, hidden)[e].any(axis=1)
    for got, before, nan in zip(products(), clean, (h_nan, y_nan)):
        assert np.array_equal(np.isnan(got), nan)
        assert np.array_equal(got[~nan], before[~nan])


# ---- silu ------------------------------------------------------------------------------------
POWERS = list(range(13, -5, -1))  # of two: one block each
GATES = [0.0, 0.0625, 1.0, 5.5, 20.0, 60.25, 86.9375, 87.0, 87.1875, 87.25, 87.375, 87.5, 88.0,
         88.5, 88.6875, 88.75, 89.0, 91.5, 92.0, 100.0, 103.9375, 104.0, 104.0625, 105.0, 128.0,
         149.0, 150.0, 200.5, 1000.0, 8192.0, 10000.0, 16383.9375]
UPS = [1.0, -2.5, 0.0625, 16383.9375]


def _matrix(values, cols, scale=0):
    """A row for each value, a sum of POWERS, times 2^scale: multiplied with ones it is exact."""
    codes = np.zeros((len(values), cols // 2), dtype=np.uint8)
    scales = np.full((len(values), cols // 32), 127, dtype=np.uint8)
    for b, p in enumerate(POWERS):
        scales[:, b] = 127 + p + scale
        for r, v in enumerate(values):
            if int(abs(v) * 16) >> (p + 4) & 1:
                codes[r, 16 * b + b % 16] = 2 | (8 if v < 0 else 0)  # +-1, an even element
    return codes, scales


def _gates():
    g, u = (a.reshape(-1) for a in np.meshgrid([s * v for v in GATES for s in (1, -1)], UPS))
    return g, u  # 256 of each


@pytest.mark.parametrize("up_scale", [0, 60])
@pytest.mark.parametrize("cols", [576, 2080])
@pytest.mark.parametrize("prompt", [0, 40, 600])
def test_gates_over_the_range_of_silu(ctx, dev, axc, prompt, cols, up_scale):
    """Few tokens (0), and prompts on the tiles of 128 x 64 and 128 x 128."""
    _say(f"silu over its range, {prompt or 'few'} tokens, {cols} columns, up times 2^{up_scale}")
    g, u = _gates()
    rows, tokens = len(g), prompt or 2
    gc, gs = _matrix(g, cols)
    uc, us = _matrix(u, cols, up_scale)
    u = u * 2.0 ** up_scale
    assert np.array_equal(MX.decode(gc, gs).sum(1), g)
    assert np.array_equal(MX.decode(uc, us).sum(1), u)
    ones = np.ones((tokens, cols), dtype=np.float32)
    e = np.zeros((tokens, 1), dtype=np.int32)
    dh, de = dev.out(tokens * rows * 4), dev.up(e)
    w = [dev.up(a) for a in (gc, gs, uc, us)]
    if prompt:
        dp = dev.out(axc.expert_plan_bytes(tokens, 1, 1))
        ctx.expert_plan(de, dp, tokens, 1, 1)
        xc, xs = MX.quantize(ones)
        ctx.mxfp4_expert_gate_up_matmul(*w, dev.up(xc), dev.up(xs), dp, dh, None, rows, cols,
                                        tokens, 1, 1, F32)
    else:
        ctx.mxfp4_expert_gate_up(*w, dev.up(ones), de, dh, rows, cols, tokens, 1, 1)
    ctx.synchronize()
    h = dev.down(dh, tokens * rows * 4, np.float32, (tokens, rows)).astype(np.float64)
    want = MX.swiglu(g, u)
    bound = 8 * U23 * np.abs(want) + np.where(g < -87.3, 2e-36, 0) * np.abs(u) + 2.0 ** -148
    assert (np.abs(h - want) <= bound).all()


def test_gates_of_few_tokens_are_exact_to_three_ulp(ctx, dev):
    """f32's exponential (1 ulp), an addition, a quotient and a product (half each), until the
    exponential of -g is beyond f32: below g = -88.72, silu(g) is within 2.7e-37."""
    cols = 576
    g, u = _gates()
    rows = len(g)
    gc, gs = _matrix(g, cols)
    uc, us = _matrix(u, cols, 60)
    u = u * 2.0 ** 60
    dh = dev.out(rows * 4)
    ctx.mxfp4_expert_gate_up(dev.up(gc), dev.up(gs), dev.up(uc), dev.up(us),
                             dev.up(np.ones((1, cols), dtype=np.float32)),
                             dev.up(np.zeros((1, 1), dtype=np.int32)), dh, rows, cols, 1, 1, 1)
    ctx.synchronize()
    h = dev.down(dh, rows * 4, np.float32, rows).astype(np.float64)
    want = MX.swiglu(g, u)
    bound = 3 * U23 * np.abs(want) + np.where(g < -88.72, 2.7e-37, 0) * np.abs(u) + 2.0 ** -148
    assert (np.abs(h - want) <= bound).all()


def test_infinite_gates_for_few_tokens(ctx, dev):
    """g beyond f32 is an infinity: silu(inf) is inf, silu(-inf) the formula's NaN, and neither
    reaches another row."""
    cols, rows = 576, 64
    gc, gs = _matrix([1.0] * rows, cols)
    uc, us = _matrix([2.0] * rows, cols)
    gc[5, :16], gs[5, 0] = 0x66, 254  # 4 * 2^127, thirty-two times
    gc[6, :16], gs[6, 0] = 0xEE, 254
    dh = dev.out(rows * 4)
    ctx.mxfp4_expert_gate_up(dev.up(gc), dev.up(gs), dev.up(uc), dev.up(us),
                             dev.up(np.ones((1, cols), dtype=np.float32)),
                             dev.up(np.zeros((1, 1), dtype=np.int32)), dh, rows, cols, 1, 1, 1)
    ctx.synchronize()
    h = dev.down(dh, rows * 4, np.float32, rows).astype(np.float64)
    assert h[5] == np.inf and np.isnan(h[6])
    rest = np.delete(h, [5, 6])
    want = float(MX.swiglu(np.float64(1), np.float64(2)))
    assert (np.abs(rest - want) <= 8 * U23 * want).all()


# ---- short rows on 128 x 128 tiles in the smallest arrays that they are taken for -------------
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,batch", [(16, 32, 8224), (8224, 32, 16), (16, 480, 8224),
                                             (8208, 256, 17), (4100, 288, 70)])
def test_small_products_of_short_rows(ctx, dev, axc, rows, cols, batch, t):
    assert "_t128x128n_" in axc.mxfp4_matmul_kernel_name(rows, cols, batch, t)
    test_gpu_mx.test_matmul(ctx, dev, axc, rows, cols, batch, t)
    if t == F32:
        test_nan_blocks_of_a_product_stay_in_their_rows(ctx, dev, axc, rows, cols, batch,
                                                        "t128x128n")


def test_launches_of_more_work_items_than_a_dimension_has(ctx, dev, axc):
    """2^32 of them or more are a typed error on the host, before any launch: the buffers here
    are far smaller than such calls' and stay as they were."""
    p = dev.out(1 << 12)
    for call in (lambda: ctx.expert_combine(p, p, p, p, 8, 1 << 24, 1),
                 lambda: ctx.mxfp4_dequant(p, p, p, (1 << 30) - 1),
                 lambda: ctx.mxfp4_unpack_ggml(p, p, p, (1 << 30) - 63),
                 lambda: ctx.expert_route(p, None, p, p, 1 << 26, axc.RouteOptions(4, 1)),
                 lambda: ctx.mxfp4_matmul(p, p, p, p, p, 1 << 31, 32, 1)):
        with pytest.raises(axc.DispatchError) as err:
            call()
        assert err.value.variant == "WorkgroupCountExceedsDeviceLimit"
    ctx.synchronize()
    assert (dev.down(p, 1 << 12, np.uint8, (1 << 12,)) == 0xA5).all()
