"""Rotary positions and the paged 4-bit cache without a GPU: the oracle against itself, sizes,
and every refusal that the host makes before it looks at a device."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import kv_numpy as KV
from oracle import mx_numpy as MX

OK, INVALID = 0, 100
F32, F16, BF16 = 0, 1, 30


@pytest.mark.parametrize("values", [False, True])
@pytest.mark.parametrize("rows,dim", [(16, 32), (32, 96), (64, 256)])
def test_a_page_holds_its_rows(rows, dim, values):
    rng = np.random.default_rng(rows + dim)
    codes = rng.integers(0, 256, (rows, dim // 2), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, dim // 32), dtype=np.uint8)
    page = KV.pack_page(codes, scales, values)
    assert page.size == rows * dim // 32 * 17
    c, s = KV.unpack_page(page, rows, dim, values)
    assert np.array_equal(c, codes) and np.array_equal(s, scales)


def test_a_row_written_is_the_row_read_and_its_place_is_the_pages():
    cache = KV.Cache(3, 16, 2, 64)
    table = np.array([[2, 0]], dtype=np.int32)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((32, 2, 2, 64))
    for pos in range(32):
        cache.write(table, 0, pos, x[pos, 0], x[pos, 1])
    for pos in range(32):
        for i, values in ((0, False), (1, True)):
            c, s = MX.quantize(x[pos, i])
            assert np.array_equal(cache.row(table, 0, pos, values), MX.decode(c, s))
            page = (cache.v if values else cache.k)[table[0, pos // 16]]
            for h in range(2):
                codes, scales = KV.unpack_page(page[h], 16, 64, values)
                assert np.array_equal(codes[pos % 16], c[h])
                assert np.array_equal(scales[pos % 16], s[h])
    assert (cache.k[1] == 0xFF).all() and (cache.v[1] == 0xFF).all()


def test_rotation_keeps_lengths_and_differences():
    """Products of a query and a key depend on the distance of their positions only."""
    f = KV.frequencies(64, scale=0.25, extrapolate=1.0, original=4096)
    rng = np.random.default_rng(2)
    q, k = rng.standard_normal((2, 1, 1, 96))
    for halves in (False, True):
        def turned(x, p):
            return KV.rotate(x, [p], f, halves)[0, 0]
        base = turned(q, 11) @ turned(k, 4)
        assert abs(turned(q, 1000011) @ turned(k, 1000004) - base) < 1e-9
        assert abs(np.linalg.norm(turned(q, 77777)) - np.linalg.norm(q)) < 1e-12
        assert np.array_equal(turned(q, 5)[64:], q[0, 0, 64:])


def test_sizes(axc):
    assert axc.kv_page_bytes(64, 8, 128) == 64 * 8 * 68
    assert axc.kv_page_bytes(16, 1, 32) == 16 * 17
    for sizes in ((0, 8, 128), (8, 8, 128), (24, 8, 128), (8192, 8, 128), (64, 0, 128),
                  (64, 8, 0), (64, 8, 100), (64, 8, 288), (64, 65537, 128)):
        with pytest.raises(ValueError):
            axc.kv_page_bytes(*sizes)
    lib = axc.load_library()
    assert [lib.axh_rope_table_bytes(d) for d in (0, 1, 2, 128, 129, 1024, 1026)] == \
        [0, 0, 16, 520, 0, 4104, 0]


class Calls:
    """Calls on what is no context and no device memory: all of them end on the host."""

    def __init__(self, axc):
        self.axc, self.lib = axc, axc.load_library()
        self.nothing = ctypes.create_string_buffer(64)
        self.ctx = ctypes.addressof(self.nothing)

    def describe(self, cache=None, batch=None, options=None, rope=None):
        c = dict(k=4096, v=8192, n_pages=4, page_size=16, kv_heads=2, head_dim=64)
        b = dict(n_seqs=2, n_tokens=3, max_pages=2, lengths=64, table=128, starts=256)
        o = dict(n_heads=4, scale=0.125)
        c.update(cache or {})
        b.update(batch or {})
        o.update(options or {})
        r = dict(table=512, dim=64, layout=0)
        r.update(rope or {})
        return (ctypes.byref(self.axc.KvCache(**c)._c), ctypes.byref(self.axc.KvBatch(**b)._c),
                ctypes.byref(self.axc.AttentionOptions(**o)._c),
                ctypes.byref(self.axc.axh._Rope(r["table"], r["dim"], r["layout"])))

    def append(self, x_type=F32, k=4096, k_stride=0, v=4096, v_stride=0, **parts):
        c, b, _, r = self.describe(**parts)
        return self.lib.axh_kv_append(self.ctx, x_type, k, k_stride, v, v_stride, c, b, r, None)

    def read(self, y_type=F32, k=4096, k_stride=0, v=4096, v_stride=0, **parts):
        c, b, _, _ = self.describe(**parts)
        return self.lib.axh_kv_read(self.ctx, c, b, y_type, k, k_stride, v, v_stride, None)

    def attend(self, x_type=F32, q=4096, q_stride=0, y=4096, y_stride=0, ws=4096, n=1 << 40,
               **parts):
        c, b, o, _ = self.describe(**parts)
        return self.lib.axh_kv_attention(self.ctx, x_type, q, q_stride, y, y_stride, c, b, o, ws,
                                         n, None)

    def rope(self, x_type=F32, x=4096, x_stride=0, y=8192, y_stride=0, positions=64, tokens=3,
             heads=2, head_dim=64, **parts):
        r = self.describe(**parts)[3]
        return self.lib.axh_rope_apply(self.ctx, x_type, x, x_stride, y, y_stride, positions,
                                       tokens, heads, head_dim, r, None)


@pytest.fixture
def calls(axc):
    return Calls(axc)


BAD_CACHE = [dict(k=0), dict(v=0), dict(k=8), dict(v=4104), dict(n_pages=0),
             dict(n_pages=1 << 31), dict(page_size=8), dict(page_size=48), dict(page_size=8192),
             dict(kv_heads=0), dict(head_dim=48), dict(head_dim=288), dict(head_dim=0)]
BAD_BATCH = [dict(lengths=0), dict(table=0), dict(starts=2), dict(lengths=66), dict(table=129),
             dict(max_pages=0), dict(max_pages=1 << 27), dict(n_tokens=1 << 31),
             dict(n_seqs=1 << 31), dict(starts=None), dict(starts=None, n_tokens=1)]


@pytest.mark.parametrize("call", ["append", "read", "attend"])
def test_caches_and_batches_that_are_refused(calls, call):
    run = getattr(calls, call)
    for cache in BAD_CACHE:
        assert run(cache=cache) == INVALID, cache
    for batch in BAD_BATCH:
        assert run(batch=batch) == INVALID, batch
    for t in (2, 12, 39):
        assert run(t) == INVALID
    assert run(batch=dict(n_tokens=0)) == OK  # launches nothing
    assert run(batch=dict(n_seqs=0)) == OK


@pytest.mark.parametrize("t,row,odd", [(F32, 128, 130), (F16, 128, 132), (BF16, 128, 129)])
def test_rows_that_are_refused(calls, t, row, odd):
    for call in (calls.append, calls.read):
        for bad in (dict(k=0), dict(v=0), dict(k=4104), dict(v=4100), dict(k_stride=row - 8),
                    dict(v_stride=1 << 31), dict(k_stride=odd)):
            assert call(t, **bad) == INVALID, bad
    for bad in (dict(q=0), dict(y=0), dict(q=4104), dict(y=4100), dict(q_stride=2 * row - 8),
                dict(y_stride=1 << 31), dict(q_stride=2 * row + odd - row)):
        assert calls.attend(t, **bad) == INVALID, bad


def test_attention_options_that_are_refused(calls, axc):
    for o in (dict(n_heads=0), dict(n_heads=3), dict(n_heads=65538), dict(scale=0.0),
              dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert calls.attend(options=o) == INVALID, o
        c, b, opts, _ = calls.describe(options=o)
        assert calls.lib.axh_kv_attention_bytes(c, b, opts, F32) == 0
    # a workspace that is too short, not there or not aligned, where one is needed
    batch = dict(n_seqs=1, n_tokens=1, max_pages=64, starts=None)
    c, b, o, _ = calls.describe(batch=batch)
    n = calls.lib.axh_kv_attention_bytes(c, b, o, F32)
    assert n > 0
    for bad in (dict(n=n - 1), dict(ws=0), dict(ws=4104)):
        assert calls.attend(batch=batch, **bad) == INVALID, bad
    assert calls.attend(batch=dict(n_tokens=1 << 30)) == INVALID  # 2^32 rows


def test_rotations_that_are_refused(calls, axc):
    for bad in (dict(dim=0), dict(dim=63), dict(dim=66), dict(layout=2), dict(table=0),
                dict(table=516)):
        assert calls.rope(rope=bad) == INVALID, bad
        assert calls.append(rope=bad) == INVALID, bad
    for bad in (dict(x_type=2), dict(x=0), dict(y=0), dict(positions=0), dict(x=4098),
                dict(positions=66), dict(head_dim=1026), dict(heads=65537), dict(x_stride=100),
                dict(y_stride=1 << 31), dict(y=4096, x_stride=256)):
        assert calls.rope(**bad) == INVALID, bad
    assert calls.rope(tokens=0) == OK and calls.rope(heads=0) == OK

    def table(factors=None, where=64, **o):
        opts = dict(dim=4)
        opts.update(o)
        f = (ctypes.c_float * 2)(*factors) if factors else None
        c = axc.RopeOptions(**opts)._c
        return calls.lib.axh_rope_table(calls.ctx, ctypes.byref(c), f, where)

    nan, inf = float("nan"), float("inf")
    for bad in (dict(dim=0), dict(dim=3), dict(dim=1026), dict(base=1.0), dict(base=inf),
                dict(base=nan), dict(scale=0.0), dict(scale=-1.0), dict(scale=nan),
                dict(extrapolate=-0.1), dict(extrapolate=1.1), dict(extrapolate=nan),
                dict(extrapolate=1.0), dict(extrapolate=1.0, original=4096, beta_fast=0.0),
                dict(extrapolate=1.0, original=4096, beta_slow=inf), dict(magnitude=inf),
                dict(where=68), dict(where=0), dict(factors=[1.0, 0.0]), dict(factors=[nan, 1.0]),
                dict(factors=[1.0, -2.0]), dict(factors=[1.0, inf])):
        assert table(**bad) == INVALID, bad
    with pytest.raises(ValueError):
        axc.RopeOptions(4, layout="thirds")._c


def test_sizes_past_what_the_kernels_count(calls, axc):
    """Pages of 2^31 bytes and more (the kernels count a page's bytes in 32 bits), scales whose
    base-2 form is infinite."""
    lib = calls.lib
    assert lib.axh_kv_page_bytes(4096, 3855, 256) == 4096 * 3855 * 8 * 17  # below 2^31
    assert lib.axh_kv_page_bytes(4096, 3856, 256) == 0
    assert lib.axh_kv_page_bytes(4096, 65536, 256) == 0
    big = dict(page_size=4096, kv_heads=3856, head_dim=256)
    assert calls.attend(cache=big, options=dict(n_heads=3856)) == INVALID
    assert calls.append(cache=big) == INVALID
    assert calls.attend(options=dict(scale=3.0e38)) == INVALID
