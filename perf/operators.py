"""Performance cases of the microscaled 4-bit operators and of expert layers.

The operators: quantisation to MXFP4 (E2M1 codes, two to a byte with the even
element in the low nibble, and one E8M0 scale byte for 32 elements), products
with MXFP4 weights (a matvec with f32 activations, a matmul with MXFP4
activations), routing of tokens to experts, and the experts' SwiGLU layer for
single tokens and for prompts.

`run` computes them in elementary torch operations, or, where `own` is true,
through the package's entry points.
"""
import math

import torch

own = False

# torch type -> ggml type id, the package's names for element types
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}

# What a drawn case may cost at most: the largest listed ones.
MAX_FLOPS = 2.0 * 14336 * 4096 * 2048
MAX_VALUES = 8192 * 4096
MAX_WEIGHTS = 128256 * 4096

_ctx = None


def _context():
    """The program's one device context."""
    global _ctx
    if _ctx is None:
        from __graft_entry__ import load_package

        _ctx = load_package().HipContext.new()
    return _ctx


def _package():
    from __graft_entry__ import load_package

    return load_package()


# ---- cases -------------------------------------------------------------------
def listed():
    return [
        # One token's activations before a product: the latency of a call.
        {"name": "quantize f32 1x4096", "kind": "quantize", "x": "f32", "rows": 1, "cols": 4096},
        # A prompt's activations (or a weight matrix being converted).
        {"name": "quantize bf16 8192x4096", "kind": "quantize", "x": "bf16", "rows": 8192,
         "cols": 4096},
        # Single-token decode: a small ragged projection, and the down
        # projection of an 8B-class model.
        {"name": "matvec 999x1056", "kind": "matvec", "rows": 999, "cols": 1056},
        {"name": "matvec 4096x14336", "kind": "matvec", "rows": 4096, "cols": 14336},
        # Batched decode: 32 sequences against the up projection.
        {"name": "linear bf16 14336x4096 b32", "kind": "linear", "x": "bf16", "rows": 14336,
         "cols": 4096, "batch": 32},
        # A short prompt, sizes that no tile divides.
        {"name": "linear f16 5001x5408 b77", "kind": "linear", "x": "f16", "rows": 5001,
         "cols": 5408, "batch": 77},
        # Prefill of 2048 tokens.
        {"name": "linear bf16 14336x4096 b2048", "kind": "linear", "x": "bf16", "rows": 14336,
         "cols": 4096, "batch": 2048},
        # Routing of one token, softmax scores.
        {"name": "route softmax 1x32 k4", "kind": "route", "score": "softmax", "tokens": 1,
         "experts": 32, "top_k": 4, "bias": False, "groups": 1, "groups_kept": 1,
         "group_best": 1},
        # Routing of a prompt: sigmoid scores, a bias for balance, half of the groups.
        {"name": "route sigmoid 4096x256 k8", "kind": "route", "score": "sigmoid",
         "tokens": 4096, "experts": 256, "top_k": 8, "bias": True, "groups": 8,
         "groups_kept": 4, "group_best": 2},
        # An expert layer for one token.
        {"name": "experts 1 of 64 k8", "kind": "decode", "tokens": 1, "experts": 64, "top_k": 8,
         "hidden": 2048, "ffn": 1024},
        # A short ragged prompt through an expert layer: few tokens an expert.
        {"name": "experts 333 of 40 k6", "kind": "prefill", "tokens": 333, "experts": 40,
         "top_k": 6, "hidden": 1312, "ffn": 736},
        # A prompt of 4096 tokens through an expert layer.
        {"name": "experts 4096 of 32 k4", "kind": "prefill", "tokens": 4096, "experts": 32,
         "top_k": 4, "hidden": 2048, "ffn": 1024},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    lo, hi = int(lo), max(int(lo), int(hi))
    v = int(round(lo * (hi / lo) ** rng.random()))
    return min(hi, max(lo, v))


def draw(rng):
    kind = rng.choices(["quantize", "matvec", "linear", "route", "decode", "prefill"],
                       [2, 2, 4, 2, 2, 3])[0]
    if kind == "quantize":
        cols = 32 * _log(rng, 1, 448)
        return {"kind": kind, "x": rng.choice(list(TYPES)), "cols": cols,
                "rows": _log(rng, 1, min(8192, MAX_VALUES // cols))}
    if kind == "matvec":
        cols = 32 * _log(rng, 8, 896)
        return {"kind": kind, "cols": cols, "rows": _log(rng, 64, MAX_WEIGHTS // 4 // cols)}
    if kind == "linear":
        cols, rows = 32 * _log(rng, 8, 448), _log(rng, 64, 28672)
        return {"kind": kind, "x": rng.choice(list(TYPES)), "rows": rows, "cols": cols,
                "batch": _log(rng, 1, min(4096, MAX_FLOPS / (2.0 * rows * cols)))}
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        per = _log(rng, 8, 384 // groups)
        best = rng.choice([1, 2])
        score = rng.choice(["softmax", "sigmoid"])
        kept = groups if groups == 1 else rng.randint(groups // 4, groups // 2)
        return {"kind": kind, "score": score, "tokens": _log(rng, 1, 4096),
                "experts": groups * per, "top_k": rng.randint(1, 8),
                # a bias of softmax scores would compare rounded sums of exponentials
                "bias": score == "sigmoid" and rng.random() < 0.5, "groups": groups,
                "groups_kept": kept, "group_best": best if score == "sigmoid" else 1}
    experts = _log(rng, 8, 128)
    hidden, ffn = 32 * _log(rng, 16, 128), 32 * _log(rng, 8, 64)
    experts = max(8, min(experts, MAX_WEIGHTS // (3 * hidden * ffn)))
    top_k = rng.randint(1, 8)
    tokens = _log(rng, 1, 8) if kind == "decode" else _log(
        rng, 16, min(4096, MAX_FLOPS / (6.0 * hidden * ffn * top_k)))
    return {"kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k,
            "hidden": hidden, "ffn": ffn}


# ---- inputs ------------------------------------------------------------------
def _weights(g, cols, *rows):
    """A random MXFP4 matrix whose products with unit activations are near 1."""
    codes = torch.randint(0, 256, (*rows, cols // 2), dtype=torch.uint8, generator=g,
                          device="cuda")
    mid = 127 - int(math.log2(3.0 * math.sqrt(cols)))
    scales = torch.randint(mid - 1, mid + 2, (*rows, cols // 32), dtype=torch.uint8, generator=g,
                           device="cuda")
    return codes, scales


def _activations(g, rows, cols):
    """Unit normal values, a few channels of them much larger, as after a norm."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return torch.where(loud, 12 * x, x)


def _choices(g, case):
    """Experts that a router chose: some are in more demand than others."""
    want = torch.randn(case["experts"], generator=g, device="cuda") * 0.5
    logits = want + torch.randn(case["tokens"], case["experts"], generator=g, device="cuda")
    top = torch.topk(logits, case["top_k"], dim=1)
    return top.indices.int().contiguous(), torch.softmax(top.values, 1)


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind = case["kind"]
    if kind == "quantize":
        return {"x": _activations(g, case["rows"], case["cols"]).to(TYPES[case["x"]])}
    if kind == "matvec":
        w, s = _weights(g, case["cols"], case["rows"])
        return {"w": w, "ws": s, "x": _activations(g, 1, case["cols"]).reshape(-1)}
    if kind == "linear":
        w, s = _weights(g, case["cols"], case["rows"])
        x = _activations(g, case["batch"], case["cols"]).to(TYPES[case["x"]])
        return {"w": w, "ws": s, "x": x}
    if kind == "route":
        d = {"logits": torch.randn(case["tokens"], case["experts"], generator=g,
                                   device="cuda") * 1.5}
        if case["bias"]:
            d["bias"] = (torch.rand(case["experts"], generator=g, device="cuda") - 0.5) * 0.2
        return d
    d = {}
    for name, rows, cols in (("gate", case["ffn"], case["hidden"]),
                             ("up", case["ffn"], case["hidden"]),
                             ("down", case["hidden"], case["ffn"])):
        d[name], d[name + "_s"] = _weights(g, cols, case["experts"], rows)
    d["chosen"], d["weights"] = _choices(g, case)
    x = _activations(g, case["tokens"], case["hidden"])
    d["x"] = x if kind == "decode" else x.bfloat16()
    return d


def prepare(case, seed):
    """The inputs, and the outputs and workspaces that a program keeps."""
    t = _inputs(case, seed)
    kind = case["kind"]

    def empty(*shape, type=torch.float32):
        return torch.empty(*shape, dtype=type, device="cuda")

    def packed(rows, cols):
        return (empty(rows, cols // 2, type=torch.uint8),
                empty(rows, cols // 32, type=torch.uint8))

    b = {}
    if kind == "quantize":
        b["xq"], b["xs"] = packed(case["rows"], case["cols"])
        b["y"] = empty(case["rows"], case["cols"], type=torch.bfloat16)
    elif kind == "matvec":
        b["y"] = empty(case["rows"])
    elif kind == "linear":
        b["xq"], b["xs"] = packed(case["batch"], case["cols"])
        b["y"] = empty(case["batch"], case["rows"])
    elif kind == "route":
        b["experts"] = empty(case["tokens"], case["top_k"], type=torch.int32)
        b["weights"] = empty(case["tokens"], case["top_k"])
    else:
        slots = case["tokens"] * case["top_k"]
        if kind == "decode":
            b["h"] = empty(slots, case["ffn"])
            b["y"] = empty(case["tokens"], case["hidden"])
        else:
            b["xq"], b["xs"] = packed(case["tokens"], case["hidden"])
            b["hq"], b["hs"] = packed(slots, case["ffn"])
            b["slots"] = empty(slots, case["hidden"], type=torch.bfloat16)
            b["y"] = empty(case["tokens"], case["hidden"], type=torch.bfloat16)
    counts = torch.bincount(t["chosen"].reshape(-1).long(), minlength=case["experts"]) \
        if kind == "prefill" else None
    return {"case": case, "t": t, "b": b,
            "most": int(counts.max()) if counts is not None else 0}


# ---- one pass, elementary torch ----------------------------------------------
def _power(e):
    """2^(e - 127) of scale bytes."""
    return (e.int() << 23).view(torch.float32)


def _decode(codes, scales):
    """The f32 values of MXFP4 rows: (..., cols / 2) and (..., cols / 32) bytes."""
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6],
                       device=codes.device)
    v = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], -1)
    v = v.reshape(*scales.shape, 32) * _power(scales).unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def _quantize(x):
    """The f32 values that MXFP4 holds of x."""
    b = x.float().reshape(-1, 32)
    _, e = torch.frexp(b.abs().amax(1, keepdim=True))  # max = m * 2^e, m in [1/2, 1)
    e = (e + 124).clamp(1, 254)
    v = b * _power(254 - e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.copysign(q, v) * _power(e)).reshape(x.shape)


def _swiglu(g, u):
    return g / (1 + torch.exp(-g)) * u


def _route(case, t):
    logits = t["logits"]
    if case["score"] == "softmax":
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    # the order of single scores is the logits' own
    single = case["groups"] == 1 or case["group_best"] == 1
    key = logits if single and not case["bias"] else score
    if case["bias"]:
        key = key + t["bias"]
    if case["groups"] > 1:
        grouped = key.reshape(len(key), case["groups"], -1)
        best = torch.sort(grouped, dim=2, descending=True).values[:, :, :case["group_best"]].sum(2)
        order = torch.sort(best, dim=1, descending=True, stable=True).indices
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(
            1, order[:, :case["groups_kept"]], True)
        key = torch.where(kept.unsqueeze(2), grouped, float("-inf")).reshape(key.shape)
    chosen = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    w = score.gather(1, chosen)
    return {"experts": chosen.int(), "weights": w / w.sum(1, keepdim=True)}


def _experts_decode(case, t):
    slots = t["chosen"].reshape(-1).long()
    x = t["x"].repeat_interleave(case["top_k"], 0).unsqueeze(2)
    gate = torch.bmm(_decode(t["gate"][slots], t["gate_s"][slots]), x)
    up = torch.bmm(_decode(t["up"][slots], t["up_s"][slots]), x)
    h = _swiglu(gate, up)
    y = torch.bmm(_decode(t["down"][slots], t["down_s"][slots]), h).squeeze(2)
    y = y * t["weights"].reshape(-1, 1)
    return {"h": h.squeeze(2), "y": y.reshape(case["tokens"], case["top_k"], -1).sum(1)}


def _experts_prefill(case, t, most):
    """Every expert's slots, padded to the most that one has."""
    slots = t["chosen"].reshape(-1).long()
    order = torch.argsort(slots, stable=True)
    count = torch.bincount(slots, minlength=case["experts"])
    first = torch.cumsum(count, 0) - count
    at = torch.empty_like(order)
    at[order] = torch.arange(len(order), device=order.device)
    place = slots * most + at - first[slots]
    x = _quantize(t["x"])
    xs = x.new_zeros(case["experts"] * most, case["hidden"])
    xs[place] = x.repeat_interleave(case["top_k"], 0)
    xs = xs.reshape(case["experts"], most, -1)
    gate = torch.bmm(xs, _decode(t["gate"], t["gate_s"]).transpose(1, 2))
    up = torch.bmm(xs, _decode(t["up"], t["up_s"]).transpose(1, 2))
    h = _quantize(_swiglu(gate, up))
    y = torch.bmm(h, _decode(t["down"], t["down_s"]).transpose(1, 2))
    y = y.reshape(case["experts"] * most, -1)[place] * t["weights"].reshape(-1, 1)
    return y.reshape(case["tokens"], case["top_k"], -1).sum(1).bfloat16()


def _run_plain(state):
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if kind == "quantize":
        return _quantize(t["x"]).bfloat16()
    if kind == "matvec":
        return torch.mv(_decode(t["w"], t["ws"]), t["x"])
    if kind == "linear":
        return torch.mm(_quantize(t["x"]), _decode(t["w"], t["ws"]).t())
    if kind == "route":
        return _route(case, t)
    if kind == "decode":
        return _experts_decode(case, t)
    return _experts_prefill(case, t, state["most"])


# ---- one pass, the package's operators -----------------------------------------
def _run_own(state):
    ctx, case, t, b = _context(), state["case"], state["t"], state["b"]
    kind = case["kind"]
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        ctx.mxfp4_quantize(t["x"], b["xq"], b["xs"], rows, cols, GGML[case["x"]])
        ctx.mxfp4_dequant(b["xq"], b["xs"], b["y"], rows * cols // 32, GGML["bf16"])
        return b["y"]
    if kind == "matvec":
        ctx.mxfp4_matvec(t["w"], t["ws"], t["x"], b["y"], case["rows"], case["cols"])
        return b["y"]
    if kind == "linear":
        rows, cols, batch = case["rows"], case["cols"], case["batch"]
        ctx.mxfp4_quantize(t["x"], b["xq"], b["xs"], batch, cols, GGML[case["x"]])
        ctx.mxfp4_matmul(t["w"], t["ws"], b["xq"], b["xs"], b["y"], rows, cols, batch)
        return b["y"]
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    if kind == "route":
        if "options" not in state:
            state["options"] = _package().RouteOptions(
                n_experts=experts, top_k=top_k, score=case["score"], n_groups=case["groups"],
                groups_kept=case["groups_kept"], group_best=case["group_best"])
        ctx.expert_route(t["logits"], t.get("bias"), b["experts"], b["weights"], tokens,
                         state["options"])
        return {"experts": b["experts"], "weights": b["weights"]}
    hidden, ffn = case["hidden"], case["ffn"]
    if kind == "decode":
        ctx.mxfp4_expert_gate_up(t["gate"], t["gate_s"], t["up"], t["up_s"], t["x"], t["chosen"],
                                 b["h"], ffn, hidden, tokens, top_k, experts)
        ctx.mxfp4_expert_down(t["down"], t["down_s"], b["h"], t["chosen"], t["weights"], b["y"],
                              hidden, ffn, tokens, top_k, experts)
        return {"h": b["h"], "y": b["y"]}
    if "plan" not in state:
        state["plan"] = ctx.alloc(_package().expert_plan_bytes(tokens, top_k, experts))
    plan = state["plan"]
    ctx.mxfp4_quantize(t["x"], b["xq"], b["xs"], tokens, hidden, GGML["bf16"])
    ctx.expert_plan(t["chosen"], plan, tokens, top_k, experts)
    ctx.mxfp4_expert_gate_up_matmul(t["gate"], t["gate_s"], t["up"], t["up_s"], b["xq"], b["xs"],
                                    plan, b["hq"], b["hs"], ffn, hidden, tokens, top_k, experts)
    ctx.mxfp4_expert_matmul(t["down"], t["down_s"], b["hq"], b["hs"], plan, b["slots"], hidden,
                            ffn, tokens, top_k, experts, y_type=GGML["bf16"])
    ctx.expert_combine(b["slots"], t["chosen"], t["weights"], b["y"], hidden, tokens, top_k,
                       y_type=GGML["bf16"])
    return b["y"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """Bytes of the inputs and outputs, each once, and the products' operations."""
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        # the values in, the packed form out and in again, the values that it holds out
        return {"bytes": n * (size[case["x"]] + 2 * 17 / 32 + 2), "flops": 2 * n}
    if kind == "matvec":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": rows * cols * 17 / 32 + 4 * (rows + cols), "flops": 2 * rows * cols}
    if kind == "linear":
        rows, cols, batch = case["rows"], case["cols"], case["batch"]
        return {"bytes": rows * cols * 17 / 32 + batch * cols * size[case["x"]]
                + 4 * batch * rows, "flops": 2 * rows * cols * batch}
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    if kind == "route":
        return {"bytes": 4 * tokens * experts + 8 * tokens * top_k,
                "flops": 8 * tokens * experts}
    matrix = case["hidden"] * case["ffn"]
    # the experts that random choices touch
    touched = experts * (1 - (1 - top_k / experts) ** tokens)
    values = tokens * case["hidden"]
    n = {"bytes": touched * 3 * matrix * 17 / 32 + 8 * tokens * top_k,
         "flops": 6 * matrix * tokens * top_k}
    if kind == "decode":
        n["bytes"] += 8 * values + 4 * tokens * top_k * case["ffn"]
    else:
        n["bytes"] += 4 * values
    return n


# ---- 64-bit results ------------------------------------------------------------
def _exact_values(codes, scales):
    """MXFP4 rows in 64 bits: sign, two exponent bits, one mantissa bit."""
    n = torch.empty(*codes.shape, 2, dtype=torch.float64, device=codes.device)
    for half, c in enumerate((codes & 15, codes >> 4)):
        exponent, mantissa = ((c >> 1) & 3).double(), (c & 1).double()
        v = torch.where(exponent == 0, mantissa / 2,
                        (1 + mantissa / 2) * torch.pow(2.0, exponent - 1))
        n[..., half] = torch.where(c >= 8, -v, v)
    two = torch.full((), 2.0, dtype=torch.float64, device=codes.device)
    n = n.reshape(*scales.shape, 32) * torch.pow(two, scales.double() - 127).unsqueeze(-1)
    return n.reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def _exact_quantized(x):
    """What MXFP4 holds of x, from the places between two values of the format."""
    b = x.double().reshape(-1, 32)
    most = b.abs().amax(1, keepdim=True)
    e = torch.where(most > 0, torch.floor(torch.log2(most)) - 2, -127.0).clamp(-127, 127)
    scale = torch.pow(torch.full_like(e, 2.0), e)
    a = b.abs() / scale
    code = torch.zeros_like(a, dtype=torch.int32)
    # a tie goes to the code whose mantissa bit is 0
    for k, place in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a >= place) if k % 2 else (a > place)
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (torch.sign(b) * values[code] * scale).reshape(x.shape)


def _exact_experts(case, t):
    """One expert after another, over the slots that chose it."""
    slots = t["chosen"].reshape(-1).long()
    packed = case["kind"] == "prefill"
    x = _exact_quantized(t["x"]) if packed else t["x"].double()
    hidden = torch.zeros(len(slots), case["ffn"], dtype=torch.float64, device=x.device)
    y = torch.zeros(len(slots), case["hidden"], dtype=torch.float64, device=x.device)
    for e in torch.unique(slots).tolist():
        mine = torch.nonzero(slots == e).reshape(-1)
        rows = x[mine // case["top_k"]].t().contiguous()
        gate = torch.mm(_exact_values(t["gate"][e], t["gate_s"][e]), rows)
        up = torch.mm(_exact_values(t["up"][e], t["up_s"][e]), rows)
        h = (gate * torch.sigmoid(gate) * up).t().contiguous()
        hidden[mine] = _exact_quantized(h) if packed else h
        y[mine] = torch.mm(hidden[mine], _exact_values(t["down"][e], t["down_s"][e]).t()
                           .contiguous())
    y = (y * t["weights"].double().reshape(-1, 1)).reshape(case["tokens"], case["top_k"], -1)
    return y.sum(1) if packed else {"h": hidden, "y": y.sum(1)}


def _exact_routing(case, t):
    """The weights; the choice is made of whole numbers and has no 64-bit form."""
    logits = t["logits"].double()
    score = torch.softmax(logits, 1) if case["score"] == "softmax" else torch.sigmoid(logits)
    key = score + t["bias"].double() if case["bias"] else score
    if case["groups"] > 1:
        grouped = key.reshape(len(key), case["groups"], -1)
        best = torch.topk(grouped, case["group_best"], dim=2).values.sum(2)
        kept = torch.topk(best, case["groups_kept"], dim=1).indices
        mask = torch.full_like(best, float("-inf")).scatter_(1, kept, 0.0)
        key = (grouped + mask.unsqueeze(2)).reshape(key.shape)
    w = score.gather(1, torch.topk(key, case["top_k"], dim=1).indices)
    return {"experts": None, "weights": w / w.sum(1, keepdim=True)}


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _exact_quantized(t["x"])
    if kind == "route":
        return _exact_routing(case, t)
    if kind in ("decode", "prefill"):
        return _exact_experts(case, t)
    x = t["x"].double().reshape(1, -1) if kind == "matvec" else _exact_quantized(t["x"])
    step = max(1, (1 << 26) // case["cols"])
    y = torch.cat([torch.mm(x, _exact_values(t["w"][r:r + step], t["ws"][r:r + step]).t()
                            .contiguous()) for r in range(0, case["rows"], step)], 1)
    return y.reshape(-1) if kind == "matvec" else y
