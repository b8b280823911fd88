"""Stream arguments: what stands for which stream."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import mx_numpy as MX


def test_stream_handles(axc):
    handle = axc.axh._stream
    assert handle(None) is None and handle(0) == 0 and handle(0x7F00) == 0x7F00
    assert handle(axc.DEFAULT_STREAM) == axc.DEFAULT_STREAM != 0
    for bad in ("0", 1.5, object()):
        with pytest.raises(TypeError):
            handle(bad)


@pytest.mark.gpu
def test_the_default_stream_can_be_named(ctx, axc):
    """Calls on DEFAULT_STREAM are the runtime's default stream's work: it is busy after them and
    the context's own stream is not, and its copies see what they wrote without any wait."""
    axc.load_library()
    hip = ctypes.CDLL("libamdhip64.so.7")  # the one that the library is linked with
    ready, not_ready = 0, 600
    rows = cols = 8192
    codes, scales = MX.gen_weights(1, rows, cols)
    x = np.random.default_rng(2).standard_normal((2048, cols)).astype(np.float32)
    want_c, want_s = MX.quantize(x)
    up = [ctx.alloc(a.nbytes) for a in (codes, scales, x)]
    for b, a in zip(up, (codes, scales, x)):
        ctx.upload(b, a)
    dw, dws, dx = up
    dc, ds, dy = ctx.alloc(want_c.nbytes), ctx.alloc(want_s.nbytes), ctx.alloc(rows * 2048 * 4)
    copy = ctx.alloc(want_c.nbytes)

    def work(times):
        for _ in range(times):
            ctx.mxfp4_quantize(dx, dc, ds, 2048, cols, stream=axc.DEFAULT_STREAM)
            ctx.mxfp4_matmul(dw, dws, dc, ds, dy, rows, cols, 2048, stream=axc.DEFAULT_STREAM)

    work(1)
    ctx.synchronize(axc.DEFAULT_STREAM)
    ctx.synchronize()
    work(40)  # some milliseconds
    busy, own = hip.hipStreamQuery(None), hip.hipStreamQuery(ctypes.c_void_p(ctx.stream))
    assert hip.hipMemcpyAsync(ctypes.c_void_p(copy.ptr), ctypes.c_void_p(dc.ptr),
                              ctypes.c_size_t(want_c.nbytes), 3, None) == 0
    assert hip.hipStreamSynchronize(None) == 0
    assert busy == not_ready and own == ready
    got = np.frombuffer(ctx.download(copy, want_c.nbytes), dtype=np.uint8)
    assert np.array_equal(got.reshape(want_c.shape), want_c)
    ctx.synchronize(axc.DEFAULT_STREAM)
    for b in (*up, dc, ds, dy, copy):
        b.close()
