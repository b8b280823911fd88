"""Rotary positions, the paged 4-bit cache and attention over it on the GPU (marked `gpu`)
against the 64-bit numpy restatement (oracle/kv_numpy.py).

Tolerances, fixed from the arithmetic before any run:
  * what is written to the cache and read back: equal bit for bit, but for turned keys;
  * a turned element: angles are within 2^-32 turns and 2^-24 of themselves, cosine and
    sine within 2^-22, two products and a sum, all relative to |a| + |b|, magnitude one more
    rounding: 2^-21 (|a| + |b|), and the output's rounding;
  * a turned key in the cache: the MXFP4 value of some number so near to the exact one;
  * attention: oracle.attention_bound, and the output's rounding (2^-11, 2^-8 relative).
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv_numpy as KV
from oracle import mx_numpy as MX
from test_gpu_mx import BF16, F16, F32, ROUND, SIZE, Dev, _say, as_type, read_out

pytestmark = pytest.mark.gpu
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
# Rounding of the softmax's weights: once to bf16 or f16, three terms of bf16 for f32.  The sums
# are those of the rounded weights w (1 + e): y is off by sum w e (v - y) to first order, at
# most e (sum w |v| + |y|), and as |y| <= sum w |v|, by 2 e sum w |v|.
WEIGHTS = {BF16: 2 * 2.0 ** -8, F16: 2 * 2.0 ** -11, F32: 2 * 2.0 ** -24}


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    ctx.synchronize()
    d.close()


def rows_of(seed, *shape):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape).astype(np.float32)
    return x * np.where(rng.random(shape[-1]) < 0.05, 6, 1).astype(np.float32)


def strided(dev, x, t, stride):
    """Device rows (tokens, ...) of type t `stride` elements apart, and their values."""
    raw, val = as_type(x, t)
    n = raw.shape[0]
    flat = raw.reshape(n, -1)
    if stride and n:
        wide = np.zeros((n, stride), dtype=flat.dtype)
        wide[:, :flat.shape[1]] = flat
        flat = wide
    return dev.up(flat), val


# ---- rotary positions ----------------------------------------------------------------
SCALINGS = {
    "none": dict(),
    "linear": dict(scale=0.125, magnitude=0.5),
    "yarn": dict(scale=0.0625, extrapolate=1.0, original=4096, magnitude=1.25),
    "half": dict(scale=0.25, extrapolate=0.5, original=8192, beta_fast=16.0, beta_slow=2.0,
                 base=500000.0),
}


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("scaling", [*SCALINGS, "factors"])
@pytest.mark.parametrize("t,tokens,heads,head_dim,dim,in_place,stride", [
    (BF16, 1, 32, 128, 128, False, 0), (F32, 7, 3, 96, 64, True, 0),
    (F16, 33, 5, 80, 80, False, 480), (F32, 5, 2, 20, 14, False, 0),
    (BF16, 3, 7, 64, 30, True, 449), (F16, 1000, 4, 256, 2, False, 0),
    (F32, 400, 40, 128, 96, True, 5200)])
def test_rope(ctx, dev, axc, layout, scaling, t, tokens, heads, head_dim, dim, in_place, stride):
    _say(f"rope {layout} {scaling} {NAMES[t]} {tokens}x{heads}x{head_dim}/{dim}")
    rng = np.random.default_rng(3)
    pos = rng.integers(-100, 1 << 20, tokens, dtype=np.int32)
    pos[:3] = [0, (1 << 31) - 1, 1][:min(3, tokens)]
    factors = np.exp(rng.random(dim // 2) * 3).astype(np.float32) if scaling == "factors" else None
    opts = {} if scaling == "factors" else SCALINGS[scaling]
    table = axc.RopeTable(ctx, axc.RopeOptions(dim=dim, layout=layout, **opts), factors)
    dx, x = strided(dev, rows_of(4, tokens, heads, head_dim), t, stride)
    row = heads * head_dim
    y_stride = stride if in_place else 0
    size = tokens * (y_stride or row) * SIZE[t]
    dy = dx if in_place else dev.out(size)
    ctx.rope(dx, dy, dev.up(pos), tokens, heads, head_dim, table, t, stride, y_stride)
    ctx.synchronize()
    if in_place:
        raw = np.frombuffer(ctx.download(dy, size), dtype=np.uint8)
        p = dev.out(size)
        ctx.upload(p, raw)
    else:
        p = dy
    y = read_out(dev, p, t, (tokens, y_stride or row))
    if y_stride:
        assert (y[:, row:] == 0).all()  # between the rows
    y = y[:, :row].reshape(x.shape)
    f = KV.frequencies(dim, factors=factors, **{k: v for k, v in opts.items() if k != "magnitude"})
    mag = float(np.float32(opts.get("magnitude", 1.0)))
    exact = KV.rotate(x, pos, f, layout == "halves", mag)
    size_of = KV.rotate(np.abs(x), pos * 0, f, layout == "halves", mag)  # |a| of each element
    pair = np.array(size_of)
    n = dim // 2
    a = slice(0, n) if layout == "halves" else slice(0, dim, 2)
    b = slice(n, dim) if layout == "halves" else slice(1, dim, 2)
    pair[..., a] = pair[..., b] = size_of[..., a] + size_of[..., b]
    pair[..., dim:] = 0
    tol = 2.0 ** -21 * pair + ROUND[t] * np.abs(exact) + (2.0 ** -24 if t == F16 else 0)
    assert (np.abs(y - exact) <= tol).all(), np.max(np.abs(y - exact) - tol)
    assert np.array_equal(y[..., dim:], x[..., dim:].astype(np.float64))
    table.close()


def test_rope_of_far_positions_is_that_of_near_ones(ctx, dev, axc):
    """A frequency of a whole part of a turn repeats exactly: bit-equal rotations."""
    table = axc.RopeTable(ctx, axc.RopeOptions(dim=2))
    raw = np.zeros(1, dtype=np.uint64)
    raw[0] = 1 << 40  # 2^-24 turns a position, in the table's own form
    ctx.upload(table.table, raw)
    pos = np.array([5, 5 + (1 << 24), 5 + 100 * (1 << 24), 5 - (1 << 24)], dtype=np.int32)
    x = np.tile(rows_of(5, 1, 3, 8), (4, 1, 1))
    dy = dev.out(x.nbytes)
    ctx.rope(dev.up(x), dy, dev.up(pos), 4, 3, 8, table)
    ctx.synchronize()
    y = dev.down(dy, x.nbytes, np.float32, x.shape)
    assert (y == y[:1]).all() and not (y == x).all()
    table.close()


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_the_gradient_of_a_rotation(ctx, dev, axc, layout):
    """dL/dx = the rotation of dL/dy by the negated positions: against the formula's transpose,
    and against differences of L = sum g y along a direction (L is linear in x: they are exact
    but for rounding)."""
    _say(f"a rotation's gradient, {layout}")
    tokens, heads, head_dim, dim = 9, 3, 40, 32
    pos = np.array([0, 1, 2, 1000, -7, 65535, 1 << 20, (1 << 31) - 1, 12345], np.int32)
    table = axc.RopeTable(ctx, axc.RopeOptions(dim=dim, layout=layout, scale=0.25, magnitude=1.125))
    x, g, way = (rows_of(s, tokens, heads, head_dim) for s in (50, 51, 52))

    def turned(v, positions):
        out = dev.out(v.nbytes)
        ctx.rope(dev.up(v), out, dev.up(positions), tokens, heads, head_dim, table)
        ctx.synchronize()
        return dev.down(out, v.nbytes, np.float32, v.shape).astype(np.float64)

    dx = turned(g, -pos)
    f = KV.frequencies(dim, scale=0.25)
    # the formula's transpose, column by column: y = R x, so R^T g
    eye = np.eye(head_dim)[None].repeat(tokens, 0)
    r = KV.rotate(eye, pos, f, layout == "halves", 1.125)  # row j: R e_j
    exact = np.einsum("tji,thi->thj", r, g.astype(np.float64))
    size = np.einsum("tji,thi->thj", np.abs(r), np.abs(g).astype(np.float64))
    assert (np.abs(dx - exact) <= 2.0 ** -21 * size + 2.0 ** -24 * np.abs(exact)).all()
    step = 0.5
    up, down = (turned((x + s * way).astype(np.float32), pos) for s in (step, -step))
    change = ((up - down) * g).sum() / (2 * step)
    # x +- way / 2 rounds by 2^-24 of each, a turned element by 2^-21 of its pair, all times g
    most = (np.abs(x) + np.abs(way)).max() * 2 * 1.125
    tol = np.abs(g).sum() * most * (2.0 ** -20) / step
    assert abs(change - (dx * way).sum()) <= tol
    table.close()


# ---- the cache -------------------------------------------------------------------------
class Batch:
    """A batch on the host and on the device: new tokens and lengths of sequences, pages in
    no order, some of them not there, and tokens around them that no sequence has."""

    def __init__(self, dev, axc, seed, new, lengths, page_size, n_pages=None, missing=(),
                 before=0, after=0, max_pages=None, plain=False):
        rng = np.random.default_rng(seed)
        self.new, self.lengths = np.array(new, np.int32), np.array(lengths, np.int32)
        need = [-(-max(0, int(n)) // page_size) for n in self.lengths]
        self.max_pages = max_pages or max(1, max(need, default=1))
        total = sum(min(n, self.max_pages) for n in need)
        self.n_pages = n_pages or total + 2
        order = rng.permutation(self.n_pages)[:total]
        self.table = np.full((len(new), self.max_pages), -1, dtype=np.int32)
        for s, n in enumerate(need):
            n = min(n, self.max_pages)
            self.table[s, :n], order = order[:n], order[n:]
        for s, slot, page in missing:
            self.table[s, slot] = page if page is not None else self.n_pages
        self.starts = (before + np.concatenate([[0], np.cumsum(self.new)])).astype(np.int32)
        self.n_tokens = int(self.starts[-1]) + after
        d = [dev.up(a) for a in (self.lengths, self.table, self.starts)]
        self.d_lengths, self.d_table = d[0], d[1]
        self.c = axc.KvBatch(len(new), self.n_tokens, self.max_pages, d[0], d[1],
                             None if plain else d[2])


def device_cache(dev, axc, cache, copies=1):
    k, v = (np.tile(x, (1, copies, 1)) for x in (cache.k, cache.v))
    return axc.KvCache(dev.up(k), dev.up(v), cache.n_pages, cache.page_size, cache.heads * copies,
                       cache.dim)


def fill(cache, batch, seed, loud=()):
    """All the sequences' rows; `loud`: (sequence, position, head, block, "k" or "v") NaN blocks."""
    for s in range(len(batch.new)):
        n = int(batch.lengths[s])
        if n > 0:
            x = rows_of(seed + s, n, 2, cache.heads, cache.dim)
            for p in range(n):
                cache.write(batch.table, s, p, x[p, 0], x[p, 1])
    for s, p, h, block, what in loud:
        page = cache.there(batch.table, s, p)
        _, scale = cache._bytes(p % cache.page_size, what == "v")
        (cache.k if what == "k" else cache.v)[page, h, scale[block]] = 255


APPEND = [
    # type, new, lengths, page, heads, dim, rotated, layout, strides, around
    (BF16, [1], [1], 16, 1, 32, 0, "pairs", 0, 0),
    (F32, [1, 1, 1], [1, 17, 40], 16, 8, 128, 128, "halves", 0, 0),
    (F16, [5, 0, 33, 1], [5, 3, 50, 100], 16, 3, 96, 48, "pairs", 296, 2),
    (BF16, [70, 3], [130, 2], 64, 2, 256, 100, "halves", 0, 3),  # more tokens than a length
    (F32, [200], [333], 32, 4, 64, 6, "halves", 268, 0),
    (F16, [0, 600, 0, 0, 9], [0, 600, 5, 0, 1000], 128, 5, 160, 160, "halves", 0, 1),
]


@pytest.mark.parametrize("t,new,lengths,page,heads,dim,rotated,layout,stride,around", APPEND)
def test_append_and_read(ctx, dev, axc, t, new, lengths, page, heads, dim, rotated, layout, stride,
                         around):
    _say(f"append {NAMES[t]} {new} of {lengths}, pages of {page}, {heads}x{dim} {rotated} {layout}")
    b = Batch(dev, axc, 7, new, lengths, page, before=around, after=around,
              missing=[(len(new) - 1, 0, -1)] if len(new) > 3 else [])
    cache = KV.Cache(b.n_pages, page, heads, dim)
    dc = device_cache(dev, axc, cache)
    dk, k = strided(dev, rows_of(8, b.n_tokens, heads, dim), t, stride)
    dv, v = strided(dev, rows_of(9, b.n_tokens, heads, dim), t, 0)
    rope, turned = None, k.astype(np.float64)
    at = KV.places(b.starts, b.lengths, b.n_tokens)
    if rotated:
        rope = axc.RopeTable(ctx, axc.RopeOptions(dim=rotated, layout=layout))
        pos = np.array([0 if a is None else a[1] for a in at])
        turned = KV.rotate(k, pos, KV.frequencies(rotated), layout == "halves")
    ctx.kv_append(dk, dv, dc, b.c, rope, t, stride, 0)
    ctx.synchronize()
    written = [np.frombuffer(ctx.download(p, c.nbytes), np.uint8).reshape(c.shape)
               for p, c in ((dc.k, cache.k), (dc.v, cache.v))]
    for a, x, y in zip(at, turned, v):
        if a is not None:
            cache.write(b.table, a[0], a[1], x, y)
    assert np.array_equal(written[1], cache.v)
    if not rotated:
        assert np.array_equal(written[0], cache.k)
    got = KV.Cache(b.n_pages, page, heads, dim)
    got.k, got.v = written
    # rows that nothing wrote are as they were
    untouched = np.ones(cache.k.shape, dtype=bool)
    for a in at:
        if a is not None and cache.there(b.table, *a) is not None:
            code, scale = cache._bytes(a[1] % page, False)
            untouched[cache.there(b.table, *a)][:, np.concatenate([code, scale])] = False
    assert (written[0][untouched] == 0xFF).all()
    for y_type in (F32, F16, BF16):
        size = b.n_tokens * heads * dim * SIZE[y_type]
        ok, ov = dev.out(size), dev.out(size)
        ctx.kv_read(dc, b.c, ok, ov, y_type)
        ctx.synchronize()
        rk = read_out(dev, ok, y_type, (b.n_tokens, heads, dim))
        rv = read_out(dev, ov, y_type, (b.n_tokens, heads, dim))
        blank = read_out(dev, dev.out(size), y_type, (b.n_tokens, heads, dim))
        for i, a in enumerate(at):
            if a is None:
                assert np.array_equal(rk[i], blank[i]) and np.array_equal(rv[i], blank[i])
                continue
            for r, values in ((rk[i], False), (rv[i], True)):
                x = got.row(b.table, a[0], a[1], values)
                x = np.zeros((heads, dim)) if x is None else x
                with np.errstate(over="ignore"):
                    x = x.astype(np.float16).astype(np.float64) if y_type == F16 else x
                assert np.array_equal(r, x)
            if rotated and y_type == F32 and cache.there(b.table, *a) is not None:
                # between the MXFP4 values of both ends of what the turned key may be
                eps = 2.0 ** -21 * (np.abs(turned[i]) + np.abs(k[i]).max())
                near = np.abs(turned[i]) * 2.0 ** -7 + eps
                m = np.abs(turned[i]).reshape(heads, -1, 32).max(2)
                e = np.exp2(np.floor(np.log2(m * (1 + 2.0 ** -18))) - 2)
                step = np.repeat(e, 32, axis=1).reshape(heads, dim)
                exact = MX.decode(*MX.quantize(turned[i]))
                same = rk[i] == exact
                # elsewhere: at most a step of the format away, and no more of them than ties
                assert (np.abs(rk[i] - exact)[~same] <= 2 * step[~same]).all()
                assert (~same).sum() <= 2, (near[~same], exact[~same])
    if rope:
        rope.close()


# ---- attention ---------------------------------------------------------------------------
def run_attention(ctx, dev, axc, t, cache, dc, b, heads, window=0, max_length=0, seed=11, q=None,
                  q_stride=0, y_stride=0, scale=None, copies=1):
    """(output, exact, tolerance) of a call; rows of no sequence are checked to be left.  copies:
    `dc` has the cache's heads so often, one copy after the other, and so has the call; all
    copies are checked to be equal."""
    dim = cache.dim
    scale = float(np.float32(scale or dim ** -0.5))
    x = rows_of(seed, b.n_tokens, heads, dim) if q is None else q
    dq, _ = strided(dev, np.tile(x, (1, copies, 1)), t, q_stride)
    x = as_type(x, t)[1]
    o = axc.AttentionOptions(n_heads=heads * copies, scale=scale, window=window,
                             max_length=max_length)
    row = heads * copies * dim
    size = b.n_tokens * (y_stride or row) * SIZE[t]
    dy = dev.out(size)
    n = axc.kv_attention_bytes(dc, b.c, o, t)
    ws = ctx.alloc(max(16, n) + 64)
    ctx.upload(ws, np.full(max(16, n) + 64, 0xA5, np.uint8))
    ctx.kv_attention(dq, dy, dc, b.c, o, ws, t, q_stride, y_stride)
    ctx.synchronize()
    tail = np.frombuffer(ctx.download(ws.ptr + n, 64), np.uint8)
    assert (tail == 0xA5).all(), "written past the workspace"
    ws.close()
    y = read_out(dev, dy, t, (b.n_tokens, y_stride or row))
    blank = read_out(dev, dev.out(size), t, (b.n_tokens, y_stride or row))
    assert np.array_equal(y[:, row:], blank[:, row:])
    exact, terms = KV.attention(x.astype(np.float64), cache, b.starts, b.lengths, b.table, scale,
                                window)
    at = KV.places(b.starts, b.lengths, b.n_tokens)
    free = [i for i, a in enumerate(at) if a is None]
    assert np.array_equal(y[free], blank[free])
    mine = [i for i, a in enumerate(at) if a is not None]
    y = y[:, :row].reshape(b.n_tokens, copies, heads, dim)[mine]
    assert np.array_equal(y, np.repeat(y[:, :1], copies, 1), equal_nan=True)
    y = y[:, 0]
    exact, terms = exact[mine], terms[:, mine]
    tol = KV.attention_bound(terms, dim, WEIGHTS[t])
    return y, exact, tol + ROUND[t] * (np.abs(exact) + tol) + (2.0 ** -24 if t == F16 else 0)


def check(y, exact, tol):
    assert np.array_equal(np.isnan(y), np.isnan(exact))
    real = ~np.isnan(exact)
    off = np.abs(y - exact)[real] - tol[real]
    assert (off <= 0).all(), off.max()


# new tokens, lengths, page, kv heads, query heads, dim, window
ATTEND = [
    ([1], [1], 16, 1, 1, 32, 0),
    ([1], [333], 64, 2, 8, 128, 0),
    ([1, 1, 1, 1, 1], [0, 15, 16, 17, 129], 16, 1, 3, 64, 0),
    ([1, 1, 1], [31, 32, 33], 16, 2, 2, 96, 5),
    ([1, 1], [700, 255], 128, 1, 17, 160, 100),
    ([1, 1, 1], [128, 511, 1030], 32, 1, 40, 256, 0),
    ([2, 0, 3, 1], [70, 9, 3, 0], 16, 2, 12, 192, 0),
    ([33, 5], [33, 100], 16, 1, 4, 128, 0),
    ([100], [60], 16, 2, 2, 64, 0),          # forty tokens before the sequence's first
    ([64, 1, 70], [200, 300, 70], 32, 1, 5, 224, 33),
    ([130, 31], [131, 500], 256, 1, 1, 128, 1),
    ([300], [300], 64, 1, 2, 32, 64),
]


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("new,lengths,page,kv,heads,dim,window", ATTEND)
def test_attention(ctx, dev, axc, t, new, lengths, page, kv, heads, dim, window):
    _say(f"attention {NAMES[t]} {new} of {lengths}, {heads}/{kv}x{dim}, window {window}")
    b = Batch(dev, axc, 12, new, lengths, page, before=1, after=2)
    cache = KV.Cache(b.n_pages, page, kv, dim)
    fill(cache, b, 13)
    dc = device_cache(dev, axc, cache)
    for max_length in (0, 40):  # keys in one part, or bounded too low: the last part has the rest
        check(*run_attention(ctx, dev, axc, t, cache, dc, b, heads, window, max_length))


@pytest.mark.parametrize("t", [BF16, F16, F32])
def test_attention_of_single_tokens_without_starts(ctx, dev, axc, t):
    _say(f"attention without starts, {NAMES[t]}")
    b = Batch(dev, axc, 14, [1] * 70, [3 * i for i in range(70)], 16, plain=True)
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 15)
    check(*run_attention(ctx, dev, axc, t, cache, device_cache(dev, axc, cache), b, 2))


@pytest.mark.parametrize("new", [[1] * 150, [0] * 70 + [9] + [0] * 60 + [2, 0], [40] + [1] * 66])
def test_attention_of_many_sequences(ctx, dev, axc, new):
    """More sequences than a wave looks at together, most of them with nothing."""
    lengths = [n and n + 7 * i % 90 for i, n in enumerate(new)]
    _say(f"attention of {len(new)} sequences")
    b = Batch(dev, axc, 16, new, lengths, 16, before=3)
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 17)
    check(*run_attention(ctx, dev, axc, F32, cache, device_cache(dev, axc, cache), b, 3))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("new,lengths,window", [([1, 1], [100, 90], 0), ([40, 3], [100, 90], 0),
                                                ([90], [90], 20)])
def test_pages_that_are_not_there(ctx, dev, axc, t, new, lengths, window):
    """Pages of -1, of n_pages and far beyond are left out; a row with no other is 0."""
    last = len(new) - 1
    b = Batch(dev, axc, 18, new, lengths, 16,
              missing=[(0, 0, -1), (0, 3, None), (0, 4, 1 << 30), (last, 2, -(1 << 31))])
    if last:
        b.table[last] = [-1] * b.max_pages
        b.d_table = dev.up(b.table)
        b.c = axc.KvBatch(len(new), b.n_tokens, b.max_pages, b.d_lengths, b.d_table, b.c.starts)
    _say(f"missing pages, {NAMES[t]} {new}")
    cache = KV.Cache(b.n_pages, 16, 2, 96)
    fill(cache, b, 19)
    y, exact, tol = run_attention(ctx, dev, axc, t, cache, device_cache(dev, axc, cache), b, 4,
                                  window)
    check(y, exact, tol)
    if last:
        assert (y[new[0]:] == 0).all()


@pytest.mark.parametrize("t", [BF16, F32])
def test_lengths_beyond_the_table(ctx, dev, axc, t):
    """Rows past max_pages have no page: nothing is read or written there."""
    b = Batch(dev, axc, 20, [1, 40], [200, 90], 16, max_pages=4)
    _say(f"lengths beyond the table, {NAMES[t]}")
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 21)
    dc = device_cache(dev, axc, cache)
    check(*run_attention(ctx, dev, axc, t, cache, dc, b, 2))
    k, v = rows_of(22, 41, 1, 64), rows_of(23, 41, 1, 64)
    ctx.kv_append(dev.up(k), dev.up(v), dc, b.c)
    ctx.synchronize()
    for i, a in enumerate(KV.places(b.starts, b.lengths, 41)):
        cache.write(b.table, a[0], a[1], k[i], v[i])
    for p, c in ((dc.k, cache.k), (dc.v, cache.v)):
        assert np.array_equal(np.frombuffer(ctx.download(p, c.nbytes), np.uint8), c.reshape(-1))


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_blocks_reach_the_rows_that_see_them(ctx, dev, axc, t, dim):
    """NaN blocks of keys and values at positions that some rows of a tile see and others do
    not (causal, window): NaN exactly where the formula has it."""
    _say(f"NaN blocks, {NAMES[t]} {dim}")
    b = Batch(dev, axc, 24, [40, 1], [90, 65], 16)
    last = dim // 32 - 1
    loud = [(0, 70, 0, last, "v"), (0, 3, 1, 0, "v"), (0, 88, 1, 0, "k"), (1, 64, 0, last, "v"),
            (1, 0, 1, 0, "k"), (1, 40, 1, last, "v")]
    cache = KV.Cache(b.n_pages, 16, 2, dim)
    fill(cache, b, 25, loud)
    dc = device_cache(dev, axc, cache)
    for window in (0, 30):
        y, exact, tol = run_attention(ctx, dev, axc, t, cache, dc, b, 6, window)
        assert np.isnan(exact).any() and not np.isnan(exact).all()
        check(y, exact, tol)


def test_scores_of_any_size(ctx, dev, axc):
    """Scores from -1e4 to 1e4, maxima that rise along the keys and ones that fall: the
    largest key's value alone, or the mean of equals."""
    _say("scores of any size")
    b = Batch(dev, axc, 26, [1, 1, 1], [400, 400, 400], 32)
    cache = KV.Cache(b.n_pages, 32, 1, 64)
    v = rows_of(27, 400, 1, 64)
    for s in range(3):
        for p in range(400):
            k = np.zeros((1, 64))
            k[0, 0] = {0: 4.0 * (p // 50), 1: 4.0 * (8 - p // 50), 2: 6.0}[s]
            cache.write(b.table, s, p, k, v[p])
    q = np.zeros((3, 2, 64), np.float32)
    q[:, 0, 0], q[:, 1, 0] = 400.0, -400.0
    y, exact, tol = run_attention(ctx, dev, axc, F32, cache, device_cache(dev, axc, cache), b, 2,
                                  q=q, scale=1.0)
    check(y, exact, tol)


def test_queries_that_are_infinite_or_nan(ctx, dev, axc):
    _say("queries that are not finite")
    b = Batch(dev, axc, 28, [1, 1, 1], [50, 50, 50], 16)
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 29)
    dc = device_cache(dev, axc, cache)
    for t in (BF16, F16, F32):
        q = rows_of(30, 3, 2, 64)
        q[0, 0, 5], q[1, 1, 7] = np.nan, np.inf
        y, exact, tol = run_attention(ctx, dev, axc, t, cache, dc, b, 2, q=q)
        assert np.isnan(y[0, 0]).all() and np.isnan(y[1, 1]).all()
        for i, h in ((0, 1), (1, 0), (2, 0), (2, 1)):
            check(y[i, h], exact[i, h], tol[i, h])


@pytest.mark.parametrize("t", [BF16, F32])
def test_strides(ctx, dev, axc, t):
    """Queries and outputs inside wider rows, as a fused projection leaves them."""
    _say(f"strides, {NAMES[t]}")
    b = Batch(dev, axc, 31, [3, 40], [80, 41], 16)
    cache = KV.Cache(b.n_pages, 16, 2, 64)
    fill(cache, b, 32)
    check(*run_attention(ctx, dev, axc, t, cache, device_cache(dev, axc, cache), b, 4, q_stride=512,
                         y_stride=264))


def test_attention_repeats_bit_for_bit(ctx, dev, axc):
    b = Batch(dev, axc, 33, [1, 1, 1, 1], [1500, 900, 33, 1200], 16)
    cache = KV.Cache(b.n_pages, 16, 2, 128)
    fill(cache, b, 34)
    dc = device_cache(dev, axc, cache)
    _say("attention, twice")
    first = run_attention(ctx, dev, axc, F32, cache, dc, b, 8)
    check(*first)
    assert np.array_equal(first[0], run_attention(ctx, dev, axc, F32, cache, dc, b, 8)[0])


def test_a_cache_beyond_4_gib(ctx, dev, axc):
    """Pages whose bytes start past 2^32, and past 2^31 of a page's index times its size."""
    page, heads, dim = 64, 8, 128
    size = axc.kv_page_bytes(page, heads, dim)
    n = (5 << 30) // size
    _say(f"a cache of {n} pages of {size} bytes")
    big = [ctx.alloc(n * size) for _ in range(2)]
    b = Batch(dev, axc, 35, [1, 3], [100, 130], page)
    small = KV.Cache(b.n_pages, page, heads, dim)
    fill(small, b, 36)
    where = n - 1 - 37 * np.arange(b.n_pages)
    for d, pages in ((big[0], small.k), (big[1], small.v)):
        for p in range(b.n_pages):
            ctx.upload(d.ptr + int(where[p]) * size, pages[p])
    table = np.where(b.table >= 0, where[np.maximum(b.table, 0)], -1).astype(np.int32)
    b.c = axc.KvBatch(2, b.n_tokens, b.max_pages, b.d_lengths, dev.up(table), b.c.starts)
    dc = axc.KvCache(big[0], big[1], n, page, heads, dim)
    check(*run_attention(ctx, dev, axc, BF16, small, dc, b, 32))
    k, v = rows_of(37, 4, heads, dim), rows_of(38, 4, heads, dim)
    ctx.kv_append(dev.up(k), dev.up(v), dc, b.c)
    ok, ov = dev.out(k.nbytes), dev.out(k.nbytes)
    ctx.kv_read(dc, b.c, ok, ov)
    ctx.synchronize()
    for o, x in ((ok, k), (ov, v)):
        got = dev.down(o, x.nbytes, np.float32, x.shape)
        c, s = MX.quantize(x.reshape(-1, dim))
        assert np.array_equal(got.reshape(-1, dim), MX.decode(c, s))
    for d in big:
        d.close()


def test_a_decode_step_in_a_graph(ctx, dev, axc):
    """Rotation, cache and attention of a step, captured once and replayed while the lengths
    grow on the device, with eager work between: every replay equals the eager calls, and the
    formula."""
    _say("a decode step in a graph")
    heads, kv, dim, page, seqs = 8, 2, 64, 16, 3
    b = Batch(dev, axc, 39, [1] * seqs, [120, 40, 80], page, plain=True)
    b.lengths = np.array([100, 15, 64], np.int32)
    cache = KV.Cache(b.n_pages, page, kv, dim)
    fill(cache, b, 40)
    dc, other = device_cache(dev, axc, cache), device_cache(dev, axc, cache)
    rope = axc.RopeTable(ctx, axc.RopeOptions(dim=dim, layout="halves"))
    o = axc.AttentionOptions(n_heads=heads, scale=dim ** -0.5)
    ws = ctx.alloc(max(16, axc.kv_attention_bytes(dc, b.c, o)))
    ws2 = ctx.alloc(ws.nbytes)
    pos = dev.up(b.lengths - 1)
    dq, dk, dv = (dev.up(np.zeros((seqs, n, dim), np.float32)) for n in (heads, kv, kv))
    turned, y, turned2, y2 = (dev.out(seqs * heads * dim * 4) for _ in range(4))

    def step(cache_, turned_, y_, ws_):
        ctx.rope(dq, turned_, pos, seqs, heads, dim, rope)
        ctx.kv_append(dk, dv, cache_, b.c, rope)
        ctx.kv_attention(turned_, y_, cache_, b.c, o, ws_)

    step(dc, turned, y, ws)  # prepares the kernels
    ctx.synchronize()
    graph = ctx.capture(lambda: step(dc, turned, y, ws))
    f = KV.frequencies(dim)
    for i in range(5):
        b.lengths += 1
        q, k, v = (rows_of(41 + 3 * i + j, seqs, n, dim) for j, n in enumerate((heads, kv, kv)))
        for d, x in ((dq, q), (dk, k), (dv, v), (pos, b.lengths - 1), (b.d_lengths, b.lengths)):
            ctx.upload(d, x)
        graph.launch()
        ctx.synchronize()
        step(other, turned2, y2, ws2)
        ctx.synchronize()
        got, eager = (dev.down(p, seqs * heads * dim * 4, np.float32, (seqs, heads, dim))
                      for p in (y, y2))
        x = dev.down(turned, seqs * heads * dim * 4, np.float32, (seqs, heads, dim))
        cache.k = np.frombuffer(ctx.download(dc.k, cache.k.nbytes), np.uint8).reshape(cache.k.shape)
        cache.v = np.frombuffer(ctx.download(dc.v, cache.v.nbytes), np.uint8).reshape(cache.v.shape)
        if i == 0:  # the other cache lacks nothing
            ctx.copy_device(other.k, dc.k, cache.k.nbytes)
            ctx.copy_device(other.v, dc.v, cache.v.nbytes)
        assert np.allclose(x, KV.rotate(q, b.lengths - 1, f, True), rtol=0, atol=1e-5)
        exact, terms = KV.attention(x.astype(np.float64), cache, b.starts, b.lengths, b.table,
                                    float(np.float32(dim ** -0.5)))
        check(got, exact, KV.attention_bound(terms, dim, WEIGHTS[F32]) + 2.0 ** -23 * np.abs(exact))
        assert np.array_equal(got, eager)
    graph.close()
    rope.close()


def test_calls_on_the_default_stream(ctx, dev, axc):
    """Another stream than the context's: the same results, waited for there."""
    _say("the default stream")
    b = Batch(dev, axc, 60, [1, 5], [300, 70], 16)
    cache = KV.Cache(b.n_pages, 16, 2, 64)
    fill(cache, b, 61)
    dc = device_cache(dev, axc, cache)
    y, exact, tol = run_attention(ctx, dev, axc, F32, cache, dc, b, 4)
    check(y, exact, tol)
    o = axc.AttentionOptions(n_heads=4, scale=0.125)
    x = rows_of(11, b.n_tokens, 4, 64)
    dy = dev.out(x.nbytes)
    ws = ctx.alloc(max(16, axc.kv_attention_bytes(dc, b.c, o)))
    ctx.kv_attention(dev.up(x), dy, dc, b.c, o, ws, stream=axc.DEFAULT_STREAM)
    ctx.synchronize(axc.DEFAULT_STREAM)
    assert np.array_equal(dev.down(dy, x.nbytes, np.float32, x.shape), y)


# ---- prompts: heads enough that workgroups have 32 and 128 rows ----------------------------
def copies_for(b, per, kv, rows):
    """Copies of the heads that make as many workgroups of `rows` rows as such calls have, by
    their mean length: 256 of 32, 1024 of 128."""
    seqs = len(b.new)
    mean = -(-b.n_tokens * per // seqs)
    assert mean >= {32: 17, 128: 128}[rows]
    groups = min(seqs * -(-mean // rows), (b.n_tokens * per + seqs * (rows - 1)) // rows)
    return -(-{32: 256, 128: 1024}[rows] // (groups * kv))


def attend_copies(ctx, dev, axc, t, cache, b, heads, rows, **kw):
    n = copies_for(b, heads // cache.heads, cache.heads, rows)
    return run_attention(ctx, dev, axc, t, cache, device_cache(dev, axc, cache, n), b, heads,
                         copies=n, **kw)


# new tokens, lengths, page, kv heads, query heads, dim, window
PROMPTS = [
    ([130, 300], [131, 500], 64, 1, 1, 128, 0),
    ([40], [333], 32, 1, 5, 64, 0),
    ([64, 1, 70], [200, 300, 70], 32, 1, 5, 224, 33),
    ([300], [300], 16, 1, 1, 32, 64),
    ([100, 0, 200], [60, 9, 700], 16, 1, 3, 96, 100),  # forty tokens before a sequence's first
    ([129], [129], 256, 2, 4, 256, 0),
    ([250], [1100], 128, 1, 1, 192, 0),
    ([150, 140], [150, 2], 16, 1, 1, 160, 1),
]


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("new,lengths,page,kv,heads,dim,window", PROMPTS)
@pytest.mark.parametrize("rows", [32, 128])
def test_attention_of_prompts(ctx, dev, axc, rows, t, new, lengths, page, kv, heads, dim, window):
    _say(f"{rows} rows, {NAMES[t]} {new} of {lengths}, {heads}/{kv}x{dim}, window {window}")
    b = Batch(dev, axc, 70, new, lengths, page, before=1, after=2)
    cache = KV.Cache(b.n_pages, page, kv, dim)
    fill(cache, b, 71)
    check(*attend_copies(ctx, dev, axc, t, cache, b, heads, rows, window=window))


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("rows", [32, 128])
def test_nan_blocks_in_prompts(ctx, dev, axc, rows, t, dim):
    """NaN blocks where some rows of a workgroup see them and others do not."""
    _say(f"NaN blocks, {rows} rows, {NAMES[t]} {dim}")
    b = Batch(dev, axc, 72, [90, 70], [190, 75], 16)
    last = dim // 32 - 1
    loud = [(0, 150, 0, last, "v"), (0, 3, 1, 0, "v"), (0, 188, 1, 0, "k"), (1, 64, 0, last, "v"),
            (1, 5, 1, 0, "k"), (1, 40, 1, last, "v")]
    cache = KV.Cache(b.n_pages, 16, 2, dim)
    fill(cache, b, 73, loud)
    for window in (0, 30):
        y, exact, tol = attend_copies(ctx, dev, axc, t, cache, b, 4, rows, window=window)
        assert np.isnan(exact).any() and not np.isnan(exact).all()
        check(y, exact, tol)


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [32, 128])
def test_pages_and_rows_that_are_not_there_in_prompts(ctx, dev, axc, rows, t):
    """Missing pages, a sequence without any, lengths beyond the table, rows of it that see
    nothing, and what a page that is not there has in the cache: NaN."""
    _say(f"missing pages, {rows} rows, {NAMES[t]}")
    b = Batch(dev, axc, 74, [140, 160, 130], [500, 190, 150], 16, max_pages=20,
              missing=[(0, 1, -1), (0, 2, None), (0, 5, 1 << 30), (0, 6, -(1 << 31)),
                       (2, 0, -1), (2, 8, -1)])
    b.table[1] = -1
    b.d_table = dev.up(b.table)
    b.c = axc.KvBatch(3, b.n_tokens, b.max_pages, b.d_lengths, b.d_table, b.c.starts)
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 75)  # (pages that no row of the table names are NaN all over)
    y, exact, tol = attend_copies(ctx, dev, axc, t, cache, b, 1, rows)
    check(y, exact, tol)
    assert (y[140:300] == 0).all() and not np.isnan(exact).any()


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [32, 128])
def test_scores_of_any_size_in_prompts(ctx, dev, axc, rows, t):
    """Maxima that rise along the keys by more than the slack, fall, or stay, differently in
    neighbouring rows; queries that are infinite or NaN beside them."""
    _say(f"scores of any size, {rows} rows, {NAMES[t]}")
    n = 300
    b = Batch(dev, axc, 76, [n], [n], 32)
    cache = KV.Cache(b.n_pages, 32, 1, 64)
    v = rows_of(77, n, 1, 64)
    for p in range(n):
        k = np.zeros((1, 64))
        k[0, 0], k[0, 1] = 1.0 * (p // 50), 1.0 * (6 - p // 50)
        cache.write(b.table, 0, p, k, v[p])
    q = np.zeros((n, 1, 64), np.float32)
    q[0::4, 0, 0], q[1::4, 0, 1], q[2::4, 0, 0], q[3::4, 0, 2] = 400.0, 400.0, -30.0, 1.0
    # Weights e^-400 and less are below what the kernels can hold.  In f32 and bf16 one that
    # falls below 2^-126 may become 0; the sum of weights is at least 1, that of the largest or
    # more, so a key's part of y is off by 2^-126 |v|, and the sum's by as much times |y| <= max
    # |v|.  In f16 a weight is off by at most half of the smallest number, 2^-25, the largest at
    # least 2^7: 2^-32 in the place of 2^-126.
    lost = 2 * n * np.abs(MX.decode(*MX.quantize(v.reshape(-1, 64)))).max()
    lost *= 2.0 ** -32 if t == F16 else 2.0 ** -126
    y, exact, tol = attend_copies(ctx, dev, axc, t, cache, b, 1, rows, q=q, scale=1.0)
    check(y, exact, tol + lost)
    q[17, 0, 5], q[133, 0, 7], q[260, 0, 9] = np.nan, np.inf, -np.inf
    y, exact, tol = attend_copies(ctx, dev, axc, t, cache, b, 1, rows, q=q, scale=1.0)
    loud = [17, 133, 260]
    assert np.isnan(y[loud]).all()
    quiet = np.setdiff1d(np.arange(n), loud)
    check(y[quiet], exact[quiet], tol[quiet] + lost)


@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [32, 128])
def test_strides_of_prompts(ctx, dev, axc, rows, t):
    _say(f"strides, {rows} rows, {NAMES[t]}")
    b = Batch(dev, axc, 78, [131], [140], 16)
    cache = KV.Cache(b.n_pages, 16, 1, 32)
    fill(cache, b, 79)
    row = 2 * 32 * copies_for(b, 2, 1, rows)
    check(*attend_copies(ctx, dev, axc, t, cache, b, 2, rows, q_stride=row + 200,
                         y_stride=row + 8))


@pytest.mark.parametrize("new", [[1], [20], [130]])
def test_windows_and_lengths_up_to_2_to_the_31(ctx, dev, axc, new):
    """Windows of 2^31 and more hide nothing; a window of 2^31 - 1 neither."""
    _say(f"large windows, {new}")
    b = Batch(dev, axc, 80, new, [200], 16)
    cache = KV.Cache(b.n_pages, 16, 2, 64)
    fill(cache, b, 81)
    for rows in ([128] if new[0] > 128 else []) + [16]:
        n = copies_for(b, 1, 2, 128) if rows == 128 else 1
        dc = device_cache(dev, axc, cache, n)
        plain = run_attention(ctx, dev, axc, F32, cache, dc, b, 2, copies=n)
        check(*plain)
        for window in ((1 << 31) - 1, 1 << 31, (1 << 32) - 1):
            y = run_attention(ctx, dev, axc, F32, cache, dc, b, 2, window, copies=n)[0]
            assert np.array_equal(y, plain[0])


@pytest.mark.parametrize("length", [-1, -5, -(1 << 31)])
@pytest.mark.parametrize("t", [BF16, F32])
def test_lengths_below_zero(ctx, dev, axc, t, length):
    """Such a sequence has no cached token: its rows are 0, and none is written or read."""
    _say(f"a length of {length}")
    b = Batch(dev, axc, 82, [3, 2], [length, 40], 16)
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 83)
    b.lengths = np.maximum(b.lengths, 0)  # (as the formula has it)
    y, exact, tol = run_attention(ctx, dev, axc, t, cache, device_cache(dev, axc, cache), b, 2)
    check(y, exact, tol)
    assert (y[:3] == 0).all()


@pytest.mark.parametrize("rows", [16, 32, 128])
@pytest.mark.parametrize("factor", [-5.8e6, -1.0, 5.8e6])
def test_scores_up_to_their_limit(ctx, dev, axc, rows, factor):
    """All keys equal, so that every row is the mean of the values that it sees, whatever the
    score, up to 2^23 in base 2 (5.8e6 log2 e = 8.37e6).  The weights are all the same, 1 but for
    the rounding of the maximum (2^-24 of it, half a unit: a factor that the sum has too), so only
    the weights' terms round, by 2^-24 each, and the sums, by 2^-22 a term, and the division."""
    _say(f"scores of {factor}, {rows} rows")
    n = 150 if rows > 16 else 40
    b = Batch(dev, axc, 84, [n], [n], 16)
    cache = KV.Cache(b.n_pages, 16, 1, 32)
    v = rows_of(85, n, 1, 32)
    k = np.zeros((1, 32))
    k[0, 0] = 1.0
    for p in range(n):
        cache.write(b.table, 0, p, k, v[p])
    q = np.zeros((n, 1, 32), np.float32)
    q[:, 0, 0] = factor
    c = copies_for(b, 1, 1, rows) if rows > 16 else 1
    y = run_attention(ctx, dev, axc, F32, cache, device_cache(dev, axc, cache, c), b, 1, q=q,
                      scale=1.0, copies=c)[0]
    values = MX.decode(*MX.quantize(v[:, 0])).astype(np.float64)
    many = np.arange(1, n + 1)[:, None]
    exact = np.cumsum(values, 0) / many
    # (the sum of up to n terms is n times a mean of them: n 2^-22 of the mean magnitude)
    tol = (2.0 ** -22 * many + 2.0 ** -22) * np.cumsum(np.abs(values), 0) / many
    assert (np.abs(y[:, 0] - exact) <= tol).all(), np.max(np.abs(y[:, 0] - exact) - tol)


@pytest.mark.parametrize("rows", [16, 32, 128])
def test_blocks_that_f16_does_not_hold(ctx, dev, axc, rows):
    """f16 operands: values of 2^16 and more make the rows that see them infinite or NaN, in
    their block, and no other row or element; values below f16's normal range are off by at
    most half of its smallest step."""
    _say(f"values outside of f16, {rows} rows")
    n = 150 if rows > 16 else 40
    b = Batch(dev, axc, 86, [n], [n], 16)
    cache = KV.Cache(b.n_pages, 16, 1, 64)
    fill(cache, b, 87)
    for p, block, byte in ((21, 1, 141), (7, 0, 100), (12, 1, 103)):
        codes, scale = cache._bytes(p % 16, True)
        cache.v[b.table[0, p // 16], 0, scale[block]] = byte
        if byte == 141:
            cache.v[b.table[0, p // 16], 0, codes[16 * block:16 * block + 16]] = 0x77
    c = copies_for(b, 1, 1, rows) if rows > 16 else 1
    y, exact, tol = run_attention(ctx, dev, axc, F16, cache, device_cache(dev, axc, cache, c), b, 1,
                                  copies=c)
    loud = np.zeros(y.shape, bool)
    loud[21:, :, 32:] = True
    assert not np.isfinite(y[loud]).any()
    check(y[~loud], exact[~loud], tol[~loud] + 2.0 ** -25)


def test_calls_at_once(ctx, dev, axc):
    """Two batches over one cache, on two streams at once and in two graphs replayed in turn, each
    with its own workspace: what they give alone, bit for bit."""
    _say("calls at once")
    heads, kv, dim = 16, 4, 128
    batches = [Batch(dev, axc, 90, [1, 1, 1], [2900, 1500, 60], 16),
               Batch(dev, axc, 90, [7, 1, 30], [2900, 1500, 60], 16)]
    cache = KV.Cache(batches[0].n_pages, 16, kv, dim)
    rng = np.random.default_rng(91)
    cache.k[:] = rng.integers(0, 256, cache.k.shape, dtype=np.uint8)
    cache.v[:] = rng.integers(0, 256, cache.v.shape, dtype=np.uint8)
    for pages, values in ((cache.k, False), (cache.v, True)):  # scales near 1
        for p in range(16):
            pages[:, :, cache._bytes(p, values)[1]] = 126
    dc = device_cache(dev, axc, cache)
    o = axc.AttentionOptions(n_heads=heads, scale=dim ** -0.5)
    calls = []
    for i, b in enumerate(batches):
        x = rows_of(92 + i, b.n_tokens, heads, dim)
        n = axc.kv_attention_bytes(dc, b.c, o)
        assert n > 0  # (its keys are split)
        calls.append((dev.up(x), dev.out(x.nbytes), b, ctx.alloc(n), x))

    def run(i, stream=None):
        q, y, b, ws, _ = calls[i]
        ctx.kv_attention(q, y, dc, b.c, o, ws, stream=stream)

    def result(i):
        return dev.down(calls[i][1], calls[i][4].nbytes, np.float32, calls[i][4].shape)

    alone = []
    for i in range(2):
        run(i)
        ctx.synchronize()
        alone.append(result(i))
        assert np.isfinite(alone[i]).all() and np.abs(alone[i]).max() > 0
    for _ in range(20):
        run(0)
        run(1, axc.DEFAULT_STREAM)
    ctx.synchronize()
    ctx.synchronize(axc.DEFAULT_STREAM)
    assert np.array_equal(result(0), alone[0]) and np.array_equal(result(1), alone[1])
    graphs = [ctx.capture(lambda i=i: run(i)) for i in range(2)]
    for _ in range(5):
        for i in range(2):
            ctx.upload(calls[i][1], np.zeros_like(calls[i][4]))
        ctx.synchronize()
        for g in graphs:
            g.launch()
        ctx.synchronize()
        assert np.array_equal(result(0), alone[0]) and np.array_equal(result(1), alone[1])
        run(0)
    ctx.synchronize()
    for g in graphs:
        g.close()
    for c in calls:
        c[3].close()
