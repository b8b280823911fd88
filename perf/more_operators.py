"""Performance cases of rotary positions and of attention over a paged 4-bit cache.

The operators: rotation of heads by their position; writing a token's key and
value rows into a paged cache in MXFP4 (the keys rotated on the way) and reading
rows back; attention of query rows over the cached rows of their sequence, for
single tokens, a few at once, and prompts.

A page of the cache holds, for each key/value head, `page` rows of `dim` elements:
  keys:    the rows' codes (dim / 2 bytes each), then their scales (dim / 32 bytes each);
  values:  for each four rows, 4 bytes of codes (8 elements) of every one of them,
           then the next 8 elements; then for each four rows the scales, block by block.

`run` computes the operators in elementary torch operations, or, where `own` is
true, through the package's entry points.
"""
import math
import random

import torch

own = False

# torch type -> ggml type id, the package's names for element types
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# What a drawn case may cost at most: the largest listed ones.
MAX_ROPE = 4096 * 40 * 128
MAX_ROWS = 40000 * 8 * 128
MAX_CACHE = 32 * 8192 * 8 * 128
MAX_SCORES = 4096 * 4096 * 32

_ctx = None


def _package():
    from __graft_entry__ import load_package

    return load_package()


def _context():
    """The program's one device context."""
    global _ctx
    if _ctx is None:
        _ctx = _package().HipContext.new()
    return _ctx


# ---- cases -------------------------------------------------------------------
def listed():
    return [
        # The queries of one new token: the latency of a call.
        {"name": "rope bf16 1x32x128", "kind": "rope", "x": "bf16", "tokens": 1, "heads": 32,
         "dim": 128, "rotated": 128, "layout": "halves", "scaling": "none", "reach": 8192},
        # A prompt's queries and keys, far out in a context that is longer than the trained one.
        {"name": "rope bf16 4096x40x128 yarn", "kind": "rope", "x": "bf16", "tokens": 4096,
         "heads": 40, "dim": 128, "rotated": 128, "layout": "pairs", "scaling": "yarn",
         "reach": 131072},
        # A decode step of 16 sequences: their new rows into the cache.
        {"name": "append bf16 16x8x128", "kind": "append", "x": "bf16", "seqs": 16, "tokens": 16,
         "before": 4000, "kv_heads": 8, "dim": 128, "page": 64, "rotated": 128,
         "layout": "halves", "scaling": "factors"},
        # Five prompts of odd lengths, a head of which half is rotated.
        {"name": "append f16 9001x4x96", "kind": "append", "x": "f16", "seqs": 5, "tokens": 9001,
         "before": 700, "kv_heads": 4, "dim": 96, "page": 16, "rotated": 48, "layout": "pairs",
         "scaling": "linear"},
        # A shared prefix read back, for a kernel that takes plain rows.
        {"name": "read bf16 40000x8x128", "kind": "read", "x": "bf16", "seqs": 4,
         "tokens": 40000, "kv_heads": 8, "dim": 128, "page": 64},
        # One token of a short conversation: the latency of a call.
        {"name": "attend bf16 1 to 333", "kind": "attend", "x": "bf16", "seqs": 1, "queries": 1,
         "length": 333, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0},
        # Batched decode of an 8B-class model: 32 sequences of many lengths.
        {"name": "attend bf16 32 to 8192", "kind": "attend", "x": "bf16", "seqs": 32,
         "queries": 32, "length": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0},
        # One token of a very long context, f32 activations as the matvecs have, a head of its
        # own for each query head.
        {"name": "attend f32 1 to 131072", "kind": "attend", "x": "f32", "seqs": 1, "queries": 1,
         "length": 131072, "heads": 16, "kv_heads": 16, "dim": 64, "page": 256, "window": 0},
        # A sliding window, six query heads to a key/value head of 96 elements.
        {"name": "attend f16 7 to 5003 window", "kind": "attend", "x": "f16", "seqs": 7,
         "queries": 7, "length": 5003, "heads": 24, "kv_heads": 4, "dim": 96, "page": 16,
         "window": 1024},
        # Drafted tokens being verified: a few of each sequence at once, wide heads.
        {"name": "attend bf16 8x4 to 6000", "kind": "attend", "x": "bf16", "seqs": 8,
         "queries": 32, "length": 6000, "heads": 32, "kv_heads": 4, "dim": 256, "page": 32,
         "window": 0},
        # A prompt of 4096 tokens.
        {"name": "attend bf16 4096 to 4096", "kind": "attend", "x": "bf16", "seqs": 1,
         "queries": 4096, "length": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0},
        # The next chunks of three prompts of odd lengths, behind what is cached of them.
        {"name": "attend f16 1501 to 6007", "kind": "attend", "x": "f16", "seqs": 3,
         "queries": 1501, "length": 6007, "heads": 28, "kv_heads": 4, "dim": 128, "page": 64,
         "window": 0},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    lo, hi = int(lo), max(int(lo), int(hi))
    v = int(round(lo * (hi / lo) ** rng.random()))
    return min(hi, max(lo, v))


def draw(rng):
    kind = rng.choices(["rope", "append", "read", "attend"], [2, 2, 1, 7])[0]
    x, dim = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([64, 96, 128, 128, 192, 256])
    if kind == "rope":
        heads = _log(rng, 1, 64)
        return {"kind": kind, "x": x, "heads": heads, "dim": dim,
                "tokens": _log(rng, 1, min(8192, MAX_ROPE // (2 * heads * dim))),
                "rotated": rng.choice([dim, dim, dim // 2, 2 * rng.randint(8, dim // 2)]),
                "layout": rng.choice(["halves", "pairs"]),
                "scaling": rng.choice(["none", "linear", "yarn", "factors"]),
                "reach": _log(rng, 10000, 1 << 20)}
    kv_heads, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        tokens = _log(rng, 1, min(16384, MAX_ROWS // (3 * kv_heads * dim)))
        return {"kind": kind, "x": x, "seqs": _log(rng, 1, min(64, tokens)), "tokens": tokens,
                "before": _log(rng, 1, 4000), "kv_heads": kv_heads, "dim": dim, "page": page,
                "rotated": rng.choice([0, dim, dim, dim // 2]),
                "layout": rng.choice(["halves", "pairs"]),
                "scaling": rng.choice(["none", "linear", "yarn", "factors"])}
    if kind == "read":
        return {"kind": kind, "x": x, "seqs": _log(rng, 1, 16), "kv_heads": kv_heads, "dim": dim,
                "page": page,
                "tokens": _log(rng, 64, min(65536, MAX_ROWS // (2 * kv_heads * dim)))}
    heads = kv_heads * rng.randint(1, min(12, 64 // kv_heads))
    window = rng.choice([0, 0, _log(rng, 64, 4096)])
    if rng.random() < 0.55:  # a token of each sequence, or a few
        seqs = _log(rng, 1, 64)
        few = rng.choice([1, 1, 1, rng.randint(2, 8)])
        most = min(131072, MAX_CACHE // (2 * seqs * kv_heads * dim),
                   MAX_SCORES // (8 * seqs * heads * few))
        queries, length = few * seqs, _log(rng, 64, most)
    else:
        seqs = _log(rng, 1, 4)
        length = _log(rng, 64, min(16384, MAX_CACHE // (2 * seqs * kv_heads * dim)))
        # (f16 and f32 rows take two and three times the matrix instructions of bf16 ones)
        most = MAX_SCORES // 2 // (heads * length * max(128, dim) // 128)
        if x != "bf16":
            most //= 3
        queries = seqs + _log(rng, 8, min(4096, seqs * (length - 1), max(16, most)))
    return {"kind": kind, "x": x, "seqs": seqs, "queries": queries, "length": length,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "window": window}


# ---- inputs ------------------------------------------------------------------
def _shares(rng, total, parts):
    """`total` as a sum of `parts` uneven numbers, each at least 1."""
    w = [0.5 + rng.random() for _ in range(parts)]
    n = [1 + int((total - parts) * v / sum(w)) for v in w]
    n[-1] += total - sum(n)
    return n


def _rows(g, n, *shape):
    """Unit normal rows, a few channels of them larger, as projections make them."""
    x = torch.randn(n, *shape, generator=g, device="cuda")
    return x * (1 + 3 * (torch.rand(shape, generator=g, device="cuda") < 0.03).float())


def _lengths(case, rng):
    """Tokens of the batch and rows in the cache, of each sequence."""
    seqs = case["seqs"]
    if case["kind"] == "append":
        new = _shares(rng, case["tokens"], seqs) if case["tokens"] > seqs else [1] * seqs
        return new, [n + rng.randint(0, case["before"]) for n in new]
    if case["kind"] == "read":
        new = _shares(rng, case["tokens"], seqs)
        return new, new
    longest = case["length"]
    rows = [longest] + [rng.randint(max(1, longest // 4), longest) for _ in range(seqs - 1)]
    new = _shares(rng, case["queries"], seqs) if case["queries"] % seqs else \
        [case["queries"] // seqs] * seqs
    return new, [max(n, r) for n, r in zip(new, rows)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _places(case, rng, t):
    """The sequences' places in the batch and in the cache, whose pages are in no order."""
    new, rows = _lengths(case, rng)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    page = case["page"]
    pages = [-(-r // page) for r in rows]
    order = list(range(sum(pages) + 3))
    rng.shuffle(order)
    table = []
    for n in pages:
        table += order[:n] + [-1] * (max(pages) - n)
        order = order[n:]
    t["n_pages"], t["max_pages"] = sum(pages) + 3, max(pages)
    t["new"], t["rows"] = new, rows
    t["starts"], t["lengths"] = _ints(starts), _ints(rows)
    t["table"] = _ints(table).reshape(len(rows), -1)


def _factors(case, seed):
    """Divisors of the frequencies, as files of models with long contexts hold them."""
    rng = random.Random(seed + 7)
    return [math.exp(rng.random() * 3 * i / max(1, case["rotated"] // 2))
            for i in range(case["rotated"] // 2)]


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    rng = random.Random(int(seed))
    kind, dim, type_ = case["kind"], case["dim"], TYPES[case["x"]]
    t = {}
    if kind == "rope":
        t["x"] = _rows(g, case["tokens"], case["heads"], dim).to(type_)
        far = max(0, case["reach"] - case["tokens"])
        t["positions"] = (torch.arange(case["tokens"], device="cuda")
                          + rng.randint(far // 2, far)).int()
    else:
        _places(case, rng, t)
        if kind == "append":
            t["k"] = _rows(g, case["tokens"], case["kv_heads"], dim).to(type_)
            t["v"] = _rows(g, case["tokens"], case["kv_heads"], dim).to(type_)
        else:
            shape = (t["n_pages"], case["kv_heads"], case["page"], dim)
            t["cache_k"] = _pack(*_quantize(_rows(g, *shape)), values=False)
            t["cache_v"] = _pack(*_quantize(_rows(g, *shape)), values=True)
        if kind == "attend":
            t["q"] = _rows(g, case["queries"], case["heads"], dim).to(type_)
    if case.get("scaling") == "factors":
        t["factors"] = [float(torch.tensor(f)) for f in _factors(case, int(seed))]  # f32 values
    return t


def prepare(case, seed):
    """The inputs, and the cache and outputs that a program keeps."""
    t = _inputs(case, seed)
    kind, dim = case["kind"], case["dim"]

    def empty(*shape, type=TYPES[case["x"]]):
        return torch.empty(*shape, dtype=type, device="cuda")

    b = {}
    if kind == "rope":
        b["y"] = torch.empty_like(t["x"])
    elif kind == "attend":
        b["y"] = torch.empty_like(t["q"])
    else:
        n = sum(t["new"])
        held = TYPES["bf16"] if kind == "append" else TYPES[case["x"]]  # bf16 holds MXFP4 exactly
        b["k"] = empty(n, case["kv_heads"], dim, type=held)
        b["v"] = empty(n, case["kv_heads"], dim, type=held)
        if kind == "append":
            size = t["n_pages"] * case["kv_heads"] * case["page"] * dim // 32 * 17
            t["cache_k"] = empty(size, type=torch.uint8)
            t["cache_v"] = empty(size, type=torch.uint8)
    return {"case": case, "t": t, "b": b}


# ---- one pass, elementary torch ----------------------------------------------
def _power(e):
    """2^(e - 127) of scale bytes."""
    return (e.int() << 23).view(torch.float32)


def _quantize(x):
    """MXFP4 codes, one to a byte, and scale bytes of rows of f32."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # max = m * 2^e, m in [1/2, 1)
    e = (e + 124).clamp(1, 254)
    v = b * _power(254 - e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4))
    code = code.to(torch.uint8) + torch.where(v < 0, 8, 0).to(torch.uint8)
    return code.reshape(x.shape), e.squeeze(-1).to(torch.uint8)


def _values(codes, scales):
    """The f32 values of codes, one to a byte, and scale bytes."""
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6],
                       device=codes.device)
    v = lut[codes.int()].reshape(*scales.shape, 32) * _power(scales).unsqueeze(-1)
    return v.reshape(codes.shape)


def _pack(codes, scales, values):
    """Pages as the cache holds them, of codes (pages, heads, rows, dim) and their scales."""
    pages, heads, rows, dim = codes.shape
    pairs = codes.reshape(pages, heads, rows, dim // 2, 2)
    c = pairs[..., 0] + 16 * pairs[..., 1]
    if values:
        c = c.reshape(pages, heads, rows // 4, 4, dim // 8, 4).transpose(3, 4)
        scales = scales.reshape(pages, heads, rows // 4, 4, dim // 32).transpose(3, 4)
    return torch.cat([c.reshape(pages, heads, -1), scales.reshape(pages, heads, -1)],
                     2).contiguous()


def _unpack(cache, case, values):
    """Codes, one to a byte, and scales of pages (..., heads, bytes), by row."""
    lead, rows, dim = cache.shape[:-1], case["page"], case["dim"]
    c = cache[..., :rows * dim // 2]
    s = cache[..., rows * dim // 2:]
    if values:
        c = c.reshape(*lead, rows // 4, dim // 8, 4, 4).transpose(-3, -2)
        s = s.reshape(*lead, rows // 4, dim // 32, 4).transpose(-2, -1)
    c, s = c.reshape(*lead, rows, dim // 2), s.reshape(*lead, rows, dim // 32)
    return torch.stack([c & 15, c >> 4], -1).reshape(*lead, rows, dim), s


def _cached(cache, t, case, values):
    """The cached rows (sequences, heads, rows, dim) in f32."""
    pages = cache[t["table"].clamp(min=0).long()]  # sequences, pages, heads, bytes
    v = _values(*_unpack(pages, case, values)).transpose(1, 2)
    return v.reshape(v.shape[0], v.shape[1], -1, v.shape[-1])


def _speeds(case, t):
    """Radians a position, in 64 bits, and the factor of the rotated elements."""
    dim = case["rotated"]
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(i * (-2 * math.log(10000.0) / dim))
    if case["scaling"] == "linear":
        return f * 0.25, 1.0
    if case["scaling"] == "factors":
        return f / torch.tensor(t["factors"], dtype=torch.float64, device="cuda"), 1.0
    if case["scaling"] == "yarn":
        turns = [dim * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(10000.0))
                 for b in (32.0, 1.0)]
        low, high = max(0, math.floor(turns[0])), min(dim - 1, math.ceil(turns[1]))
        ramp = ((i - low) / max(0.001, high - low)).clamp(0, 1)
        return f * (1 - ramp + 0.0625 * ramp), 0.1 * math.log(16.0) + 1
    return f, 1.0


def _rotate(x, positions, case, t):
    """The rotated heads (tokens, heads, dim), in f32."""
    dim = case["rotated"]
    if dim == 0:
        return x.float()
    f, factor = _speeds(case, t)
    angle = positions.double().unsqueeze(1) * f
    cos = (torch.cos(angle) * factor).float().unsqueeze(1)
    sin = (torch.sin(angle) * factor).float().unsqueeze(1)
    y = x.float().clone()
    if case["layout"] == "pairs":
        a, b = y[..., 0:dim:2].clone(), y[..., 1:dim:2].clone()
        y[..., 0:dim:2], y[..., 1:dim:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = y[..., :dim // 2].clone(), y[..., dim // 2:dim].clone()
        y[..., :dim // 2], y[..., dim // 2:dim] = a * cos - b * sin, a * sin + b * cos
    return y


def _token_places(t):
    """Sequence and position of each token of the batch."""
    n = t["starts"].long().diff()
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n,
                                  output_size=sum(t["new"]))
    at = torch.arange(len(seq), device=n.device) - t["starts"].long()[seq]
    return seq, at, (t["lengths"].long() - n)[seq] + at


def _run_plain(state):
    case, t = state["case"], state["t"]
    kind, type_ = case["kind"], TYPES[case["x"]]
    if kind == "rope":
        return _rotate(t["x"], t["positions"], case, t).to(type_)
    seq, at, pos = _token_places(t)
    if kind == "append":
        k = _rotate(t["k"], pos, case, t)
        return {"k": _values(*_quantize(k)).bfloat16(),
                "v": _values(*_quantize(t["v"].float())).bfloat16()}
    if kind == "read":
        return {n: _cached(t["cache_" + n], t, case, n == "v")[seq, :, pos].to(type_)
                for n in ("k", "v")}
    seqs, kv, dim, most = case["seqs"], case["kv_heads"], case["dim"], max(t["new"])
    per = case["heads"] // kv
    k, v = (_cached(t["cache_" + n], t, case, n == "v").reshape(seqs * kv, -1, dim)
            for n in ("k", "v"))
    q = torch.zeros(seqs, most, kv, per, dim, device="cuda")
    q[seq, at] = t["q"].float().reshape(-1, kv, per, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs * kv, most * per, dim)
    s = torch.bmm(q, k.transpose(1, 2)) * dim ** -0.5
    n = t["starts"].diff()
    row = (t["lengths"] - n).unsqueeze(1) + torch.arange(most, device="cuda")  # positions
    key = torch.arange(k.shape[1], device="cuda")
    seen = (key <= row.unsqueeze(2)) & (key < t["lengths"].reshape(-1, 1, 1))
    if case["window"]:
        seen &= key > row.unsqueeze(2) - case["window"]
    s = s.reshape(seqs, kv, most, per, -1).masked_fill_(~seen.reshape(seqs, 1, most, 1, -1),
                                                        float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    y = torch.bmm(p.reshape(seqs * kv, most * per, -1), v).reshape(seqs, kv, most, per, dim)
    y = (y / total).permute(0, 2, 1, 3, 4)[seq, at]
    return y.reshape(-1, case["heads"], dim).to(type_)


# ---- one pass, the package's operators -----------------------------------------
def _keep(state):
    """What a program makes once: the rotation's table, the cache's and the batch's description,
    the workspace."""
    axc, ctx, case, t = _package(), _context(), state["case"], state["t"]
    kind, kept = case["kind"], {}
    if case.get("rotated"):
        scaled = {"none": {}, "factors": {}, "linear": {"scale": 0.25},
                  "yarn": {"scale": 0.0625, "extrapolate": 1.0, "original": 8192,
                           "magnitude": 0.1 * math.log(16.0) + 1}}[case["scaling"]]
        kept["rope"] = axc.RopeTable(ctx, axc.RopeOptions(dim=case["rotated"],
                                                          layout=case["layout"], **scaled),
                                     factors=t.get("factors"))
    if kind != "rope":
        kept["cache"] = axc.KvCache(t["cache_k"], t["cache_v"], t["n_pages"], case["page"],
                                    case["kv_heads"], case["dim"])
        kept["batch"] = axc.KvBatch(case["seqs"], sum(t["new"]), t["max_pages"], t["lengths"],
                                    t["table"], None if max(t["new"]) == 1 else t["starts"])
    if kind == "attend":
        kept["options"] = axc.AttentionOptions(n_heads=case["heads"], scale=case["dim"] ** -0.5,
                                               window=case["window"], max_length=max(t["rows"]))
        kept["workspace"] = ctx.alloc(max(16, axc.kv_attention_bytes(
            kept["cache"], kept["batch"], kept["options"], GGML[case["x"]])))
    return kept


def _run_own(state):
    ctx, case, t, b = _context(), state["case"], state["t"], state["b"]
    if "kept" not in state:
        state["kept"] = _keep(state)
    kept, kind, type_ = state["kept"], case["kind"], GGML[case["x"]]
    if kind == "rope":
        ctx.rope(t["x"], b["y"], t["positions"], case["tokens"], case["heads"], case["dim"],
                 kept["rope"], type_)
        return b["y"]
    if kind == "attend":
        ctx.kv_attention(t["q"], b["y"], kept["cache"], kept["batch"], kept["options"],
                         kept["workspace"], type_)
        return b["y"]
    if kind == "append":
        ctx.kv_append(t["k"], t["v"], kept["cache"], kept["batch"], kept.get("rope"), type_)
        ctx.kv_read(kept["cache"], kept["batch"], b["k"], b["v"], GGML["bf16"])
    else:
        ctx.kv_read(kept["cache"], kept["batch"], b["k"], b["v"], type_)
    return {"k": b["k"], "v": b["v"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """Bytes of the inputs and outputs, each once, and the products' operations."""
    kind, dim, size = case["kind"], case["dim"], SIZE[case["x"]]
    if kind == "rope":
        n = case["tokens"] * case["heads"] * dim
        return {"bytes": 2 * n * size, "flops": 3 * n}
    if kind == "append":
        n = 2 * case["tokens"] * case["kv_heads"] * dim
        # the rows in, their 4-bit form out and in again, the values that it holds out
        return {"bytes": n * (size + 2 * 17 / 32 + 2), "flops": 3 * n}
    seqs, kv = case["seqs"], case["kv_heads"]
    if kind == "read":
        n = 2 * case["tokens"] * kv * dim
        return {"bytes": n * (size + 17 / 32), "flops": n}
    mean = case["length"] if seqs == 1 else case["length"] * (1 + 0.625 * (seqs - 1)) / seqs
    new = case["queries"] / seqs
    reach, keys = mean, mean - (new - 1) / 2
    if case["window"]:
        reach = min(mean, case["window"] + new)
        keys = min(keys, case["window"])
    return {"bytes": 2 * seqs * reach * kv * dim * 17 / 32
            + 2 * case["queries"] * case["heads"] * dim * size,
            "flops": 4 * case["queries"] * case["heads"] * dim * keys}


# ---- 64-bit results ------------------------------------------------------------
def _exact_angles(case, t, positions):
    """Cosines and sines of one row a token, as a complex number."""
    dim = case["rotated"]
    f = torch.tensor([10000.0 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    factor = 1.0
    if case["scaling"] == "linear":
        f /= 4
    elif case["scaling"] == "factors":
        f /= torch.tensor(t["factors"], dtype=torch.float64)
    elif case["scaling"] == "yarn":
        factor = 1 + math.log(16.0) / 10

        def at(rotations):  # the pair that turns so often in the trained context
            return dim / 2 * math.log(8192 / (2 * math.pi * rotations), 10000.0)

        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), dim - 1)
        for i in range(dim // 2):
            part = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f[i] = f[i] * (1 - part) + f[i] / 16 * part
    a = torch.outer(positions.double().cpu(), f).cuda()
    return torch.polar(torch.full_like(a, factor), a).unsqueeze(1)


def _exact_rotated(x, positions, case, t):
    x, dim = x.double(), case["rotated"]
    if dim == 0:
        return x
    turn = _exact_angles(case, t, positions)
    if case["layout"] == "pairs":
        z = torch.view_as_complex(x[..., :dim].reshape(*x.shape[:-1], dim // 2, 2).contiguous())
        y = torch.view_as_real(z * turn).reshape(*x.shape[:-1], dim)
    else:
        z = torch.complex(x[..., :dim // 2].contiguous(), x[..., dim // 2:dim].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., dim:]], -1)


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


def _exact_rows(cache, t, case, seq, values):
    """One sequence's cached rows (rows, heads, dim) in 64 bits, byte by byte."""
    page, dim, n = case["page"], case["dim"], t["rows"][seq]
    row = torch.arange(n, device="cuda")
    held = cache[t["table"][seq].long()[row // page]]  # rows, heads, bytes
    r = (row % page).reshape(-1, 1)
    d = torch.arange(dim, device="cuda").reshape(1, -1)
    if values:
        byte = (r // 4) * 2 * dim + d // 8 * 16 + r % 4 * 4 + d % 8 // 2
        scale = page * dim // 2 + (r // 4) * (dim // 8) + d // 32 * 4 + r % 4
    else:
        byte = r * (dim // 2) + d // 2
        scale = page * dim // 2 + r * (dim // 32) + d // 32
    heads = held.shape[1]
    c = held.gather(2, byte.unsqueeze(1).expand(-1, heads, -1))
    c = torch.where(d % 2 == 1, c >> 4, c & 15)
    e = held.gather(2, scale.unsqueeze(1).expand(-1, heads, -1)).double()
    high, low = ((c >> 1) & 3).double(), (c & 1).double()
    v = torch.where(high == 0, low / 2, (1 + low / 2) * torch.exp2(high - 1))
    return torch.where(c >= 8, -v, v) * torch.exp2(e - 127)


def _exact_attention(case, t):
    """One sequence and one head after another."""
    per, out = case["heads"] // case["kv_heads"], torch.zeros(t["q"].shape, dtype=torch.float64,
                                                              device="cuda")
    first = 0
    for seq, (new, rows) in enumerate(zip(t["new"], t["rows"])):
        k, v = (_exact_rows(t["cache_" + n], t, case, seq, n == "v") for n in ("k", "v"))
        pos = torch.arange(rows - new, rows, device="cuda").reshape(-1, 1)
        key = torch.arange(rows, device="cuda").reshape(1, -1)
        hidden = key > pos
        if case["window"]:
            hidden |= key + case["window"] <= pos
        for h in range(case["heads"]):
            q = t["q"][first:first + new, h].double()
            s = torch.mm(q, k[:, h // per].t().contiguous()) / math.sqrt(case["dim"])
            p = torch.softmax(s.masked_fill(hidden, float("-inf")), 1)
            out[first:first + new, h] = torch.mm(p, v[:, h // per].contiguous())
        first += new
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rotated(t["x"], t["positions"], case, t)
    if kind == "attend":
        return _exact_attention(case, t)
    if kind == "append":
        pos = torch.cat([torch.arange(r - n, r) for n, r in zip(t["new"], t["rows"])])
        return {"k": _exact_quantized(_exact_rotated(t["k"], pos, case, t)),
                "v": _exact_quantized(t["v"])}
    return {n: torch.cat([_exact_rows(t["cache_" + n], t, case, s, n == "v")
                          for s in range(case["seqs"])]) for n in ("k", "v")}
