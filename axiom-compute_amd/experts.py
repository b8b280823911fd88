"""An expert layer (mixture-of-experts feed-forward) in MXFP4 from a GGUF file,
run through the library's own operations: router product, routing, the experts'
gate and up products with SiLU, their down products, and the weighted sum.

    with gguf.GgufFile(path) as f:
        layer = experts.ExpertLayer(ctx, f, "blk.0", RouteOptions(n_experts=64, top_k=8),
                                    max_tokens=4096)
    layer.run(x, y, n_tokens)       # x, y: n_tokens x hidden f32 on the device

Tensors are those of a GGUF layer `prefix`: ffn_gate_exps.weight and
ffn_up_exps.weight (hidden x ffn x experts, ne[0] first), ffn_down_exps.weight (ffn x
hidden x experts), of type MXFP4; the router's ffn_gate_inp.weight (hidden x experts), f32,
f16 or bf16 (its product is in f32 then), or MXFP4; and exp_probs_b.bias (experts, f32)
where the router adds a bias to its choices.  What is computed is y = sum over a token's
choices of weight * (down (silu(gate x) * (up x))): a file whose layer holds more than that
(biases of the experts' or the router's products, shared experts) is refused.

The codes and scales are laid out once, when the layer is made, and so are the
workspaces: run() allocates nothing and can be captured in a graph.  No counterpart
in the reference, which has no expert layers.
"""
from __future__ import annotations

import re
from typing import Iterable, Optional

from . import axh as _axh
from .gguf import GGML_MXFP4, GgufFile

GGML_F32 = 0


def _unused(file: GgufFile, prefix: str, used: Iterable[str]) -> list[str]:
    """Tensors of the router or the experts that are not used: all that are called ffn_* or
    exp_* but norms (of the layer's input) and a dense feed-forward beside the experts."""
    part = re.compile(re.escape(prefix) + r"\.(?!ffn_norm|ffn_post_norm|ffn_(gate|up|down)\.)"
                      r"(ffn_|exp_)")
    return sorted(n for n in file.tensors if part.match(n) and n not in used)


class _Matrix:
    """An MXFP4 tensor as codes and scales on the device."""

    def __init__(self, ctx, file: GgufFile, name: str):
        t = file.tensors[name]
        if t.type != GGML_MXFP4:
            raise ValueError(f"{name} is of type {t.type}, not MXFP4")
        self.cols, self.shape = t.shape[0], t.shape
        blocks = t.nbytes // 17
        self.codes, self.scales = ctx.alloc(blocks * 16), ctx.alloc(blocks)
        raw = file.upload(ctx, name)
        ctx.mxfp4_unpack_ggml(raw, self.codes, self.scales, blocks)
        ctx.synchronize()
        raw.close()

    def close(self) -> None:
        self.codes.close()
        self.scales.close()


class _Router:
    """The router's matrix: f32, f16 or bf16 as it stands in the file, or MXFP4 (in_f32: decoded
    to f32, which holds its values exactly)."""

    def __init__(self, ctx, file: GgufFile, name: str, in_f32: bool):
        t = file.tensors[name]
        self.type, self.packed = t.type, None
        if t.type == GGML_MXFP4:
            self.packed = _Matrix(ctx, file, name)
            if in_f32:
                packed, self.packed, self.type = self.packed, None, GGML_F32
                blocks = t.nbytes // 17
                self.w = ctx.alloc(blocks * 128)
                ctx.mxfp4_dequant(packed.codes, packed.scales, self.w, blocks, GGML_F32)
                ctx.synchronize()
                packed.close()
        elif t.type in (_axh.GGML_F32, _axh.GGML_F16, _axh.GGML_BF16):
            self.w = file.upload(ctx, name)
        else:
            raise ValueError(f"{name} is of type {t.type}, not MXFP4, f32, f16 or bf16")

    def close(self) -> None:
        (self.packed or self.w).close()


class ExpertLayer:
    """Up to few_tokens tokens, run() takes the single-token products, which read the
    weights of each choice and keep the activations in f32; more tokens are
    quantised to MXFP4 and grouped by expert.  The default is three choices for four
    experts, about where the times cross (us): 64 experts, 8 choices, 2048 x 1024, 6
    tokens 36 / 45, 12 tokens 58 / 54; 32, 4, 4096 x 1408, 6 tokens 50 / 51; 8, 2, 4096 x
    14336, 2 tokens 71 / 90, 4 tokens 131 / 109.  So the precision of a token's activations
    depends on how many tokens come with it, unless few_tokens is 0 (all in MXFP4) or
    max_tokens (all in f32; choices of 65535 / top_k tokens at most).  A run in a graph (us): 64
    experts, 8 choices, 2048 x 1024, 1 token 17, 64 tokens 61, 333 70, 4096 335; 32, 4, 2048 x
    1024, 14, 38, 45, 180; 8, 2, 4096 x 14336, 45, 155, 214, 1096.

    A router in MXFP4 multiplies one token's activations in f32 and those of several in MXFP4,
    so that even the choice of a token's experts may depend on the others.  With router_f32 its
    matrix is decoded once and the product is in f32 for any number of tokens, as it is for
    routers in f32, f16 or bf16 without it.

    The workspaces are the layer's: runs of one layer must follow one another, on one stream or
    with a wait between, as two at once overwrite each other's logits, plan and slots.

    The gate's activation is `activation`, of which "silu" is the only one there is.  A tensor
    of the layer that run() does not use is a ValueError, as the layer would be another one
    without it; leave_out names those (without the prefix) that the caller computes itself,
    such as shared experts whose output it adds."""

    def __init__(self, ctx, file: GgufFile, prefix: str, options: "_axh.RouteOptions",
                 max_tokens: int, few_tokens: Optional[int] = None, activation: str = "silu",
                 leave_out: Iterable[str] = (), router_f32: bool = False):
        if max_tokens < 1:
            raise ValueError("max_tokens must be at least 1")
        self.ctx, self.options = ctx, options
        if few_tokens is None:
            few_tokens = max(1, 3 * options.n_experts // (4 * max(1, options.top_k)))
        self.max_tokens, self.few_tokens = max_tokens, min(few_tokens, max_tokens)
        names = {n: f"{prefix}.{n}.weight" for n in ("ffn_gate_inp", "ffn_gate_exps",
                                                     "ffn_up_exps", "ffn_down_exps")}
        for n in names.values():
            if n not in file.tensors:
                raise ValueError(f"the file has no tensor {n}")
        if activation != "silu":
            raise ValueError(f"unknown activation {activation!r}")
        bias = f"{prefix}.exp_probs_b.bias"
        unused = _unused(file, prefix, {*names.values(), bias,
                                        *(f"{prefix}.{n}" for n in leave_out)})
        if unused:
            raise ValueError(f"the layer has tensors that are not computed: {', '.join(unused)}")
        shapes = {n: tuple(file.tensors[t].shape) for n, t in names.items()}
        hidden, n = shapes["ffn_gate_inp"]
        ffn = shapes["ffn_gate_exps"][1]
        if (n != options.n_experts or shapes["ffn_gate_exps"] != (hidden, ffn, n)
                or shapes["ffn_up_exps"] != (hidden, ffn, n)
                or shapes["ffn_down_exps"] != (ffn, hidden, n)):
            raise ValueError(f"the tensors' shapes do not make a layer of {options.n_experts} "
                             f"experts: {shapes}")
        self.hidden, self.ffn = hidden, ffn
        self.router = _Router(ctx, file, names["ffn_gate_inp"], router_f32)
        self.gate, self.up, self.down = (
            _Matrix(ctx, file, names[k]) for k in ("ffn_gate_exps", "ffn_up_exps",
                                                   "ffn_down_exps"))
        self.bias = None
        if bias in file.tensors:
            t = file.tensors[bias]
            if t.type != GGML_F32 or tuple(t.shape) != (n,):
                raise ValueError(f"{bias} must be f32 of {n} elements")
            self.bias = file.upload(ctx, bias)
        k, t, few = options.top_k, max_tokens, max(1, self.few_tokens)
        alloc = ctx.alloc
        self.logits = alloc(4 * t * n)
        self.experts, self.weights = alloc(4 * t * k), alloc(4 * t * k)
        self.x_codes, self.x_scales = alloc(t * hidden // 2), alloc(t * hidden // 32)
        self.plan = alloc(_axh.expert_plan_bytes(t, k, n))
        self.h = alloc(4 * few * k * ffn)  # f32, few tokens
        self.h_codes, self.h_scales = alloc(t * k * ffn // 2), alloc(t * k * ffn // 32)
        self.slots = alloc(4 * t * k * hidden)

    def run(self, x, y, n_tokens: int, stream=None) -> None:
        """y = the layer of x (n_tokens x hidden, f32, 16-byte aligned); asynchronous."""
        if not 0 <= n_tokens <= self.max_tokens:
            raise ValueError(f"n_tokens must be 0 to {self.max_tokens}")
        ctx, n, k = self.ctx, self.options.n_experts, self.options.top_k
        hidden, ffn = self.hidden, self.ffn
        few = n_tokens <= self.few_tokens
        router = self.router.packed
        if not few or (router and n_tokens != 1):
            ctx.mxfp4_quantize(x, self.x_codes, self.x_scales, n_tokens, hidden, GGML_F32,
                               stream=stream)
        if not router:
            ctx.expert_logits(self.router.w, x, self.logits, n, hidden, n_tokens,
                              self.router.type, stream=stream)
        elif n_tokens == 1 and few:
            ctx.mxfp4_matvec(router.codes, router.scales, x, self.logits, n, hidden,
                             stream=stream)
        else:
            ctx.mxfp4_matmul(router.codes, router.scales, self.x_codes, self.x_scales,
                             self.logits, n, hidden, n_tokens, stream=stream)
        ctx.expert_route(self.logits, self.bias, self.experts, self.weights, n_tokens,
                         self.options, stream=stream)
        gate, up, down = self.gate, self.up, self.down
        if few:
            ctx.mxfp4_expert_gate_up(gate.codes, gate.scales, up.codes, up.scales, x, self.experts,
                                     self.h, ffn, hidden, n_tokens, k, n, stream=stream)
            ctx.mxfp4_expert_down(down.codes, down.scales, self.h, self.experts, self.weights, y,
                                  hidden, ffn, n_tokens, k, n, stream=stream)
            return
        ctx.expert_plan(self.experts, self.plan, n_tokens, k, n, stream=stream)
        ctx.mxfp4_expert_gate_up_matmul(gate.codes, gate.scales, up.codes, up.scales, self.x_codes,
                                        self.x_scales, self.plan, self.h_codes, self.h_scales, ffn,
                                        hidden, n_tokens, k, n, stream=stream)
        ctx.mxfp4_expert_matmul(down.codes, down.scales, self.h_codes, self.h_scales, self.plan,
                                self.slots, hidden, ffn, n_tokens, k, n, stream=stream)
        ctx.expert_combine(self.slots, self.experts, self.weights, y, hidden, n_tokens, k,
                           n_experts=n, stream=stream)

    def close(self) -> None:
        """Frees the layer's device memory (not while a run is on its way)."""
        for m in (self.router, self.gate, self.up, self.down):
            m.close()
        for b in (self.bias, self.logits, self.experts, self.weights, self.x_codes, self.x_scales,
                  self.plan, self.h, self.h_codes, self.h_scales, self.slots):
            if b is not None:
                b.close()
