"""Expert layers of GGUF files on the GPU (marked `gpu`): what a token's result depends on."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import mx_numpy as MX
from test_gpu_mx import F32, MXFP4, U23, Dev, _say, activations  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    ctx.synchronize()
    d.close()


def _file(axc, path, n, hidden, ffn):
    """Writes the layer blk.3, all in MXFP4, and returns its router's matrix in 64 bits."""
    tensors, router = [], None
    for i, (name, rows, cols) in enumerate((("ffn_gate_inp", (n,), hidden),
                                            ("ffn_gate_exps", (n, ffn), hidden),
                                            ("ffn_up_exps", (n, ffn), hidden),
                                            ("ffn_down_exps", (n, hidden), ffn))):
        c, s = MX.gen_weights(60 + i, *rows, cols)
        router = MX.decode(c, s) if router is None else router
        tensors.append((f"blk.3.{name}.weight", MXFP4, (cols,) + rows[::-1],
                        MX.to_ggml(c, s).tobytes()))
    axc.gguf.write_gguf(path, [], tensors)
    return router


@pytest.mark.parametrize("few_tokens", [None, 0, 70])
def test_a_packed_router_in_f32_does_not_depend_on_the_batch(ctx, dev, axc, tmp_path, few_tokens):
    """A token's logits are those of f32 activations, and its experts the same, whether it
    comes alone, with two others or with 69.  Tolerance: a sum of `hidden` products in f32,
    in any order, by truncating additions."""
    n, k, hidden, ffn = 12, 3, 544, 96
    w = _file(axc, tmp_path / "layer.gguf", n, hidden, ffn)
    with axc.gguf.GgufFile(tmp_path / "layer.gguf") as f:
        layer = axc.experts.ExpertLayer(ctx, f, "blk.3", axc.RouteOptions(n_experts=n, top_k=k),
                                        max_tokens=70, few_tokens=few_tokens, router_f32=True)
    x = activations(61, 70, hidden)
    dx, dy = dev.up(x), dev.out(70 * hidden * 4)
    exact = x.astype(np.float64) @ w.T
    bound = (hidden + 1) * U23 * (np.abs(x.astype(np.float64)) @ np.abs(w).T)
    # tokens no two of whose logits are so near that their order is open
    clear = np.diff(np.sort(exact, axis=1), axis=1).min(axis=1) > 2 * bound.max(axis=1)
    assert clear[0] and clear.sum() >= 60
    chosen = np.argsort(-exact, axis=1, kind="stable")[:, :k]
    for tokens in (1, 3, 70):
        _say(f"layer with a router in f32, {tokens} tokens")
        layer.run(dx, dy, tokens)
        ctx.synchronize()
        logits = np.frombuffer(ctx.download(layer.logits, tokens * n * 4), dtype=np.float32)
        assert (np.abs(logits.reshape(tokens, n) - exact[:tokens]) <= bound[:tokens]).all()
        got = np.frombuffer(ctx.download(layer.experts, tokens * k * 4), dtype=np.int32)
        assert np.array_equal(got.reshape(tokens, k)[clear[:tokens]],
                              chosen[:tokens][clear[:tokens]])
    layer.close()
