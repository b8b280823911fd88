"""MXFP4 and expert operations without a GPU: the numpy restatement that the GPU
tests compare with (oracle/mx_numpy.py) against independent statements of the
formats, the entry points' host-side functions, ggml's type 39 in GGUF files,
and the performance cases' plain forms against their 64-bit results."""
from __future__ import annotations

import ctypes
import importlib.util
import random
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

from oracle import mx_numpy as MX

ROOT = Path(__file__).resolve().parents[1]


def _e2m1(code: int) -> Fraction:
    """Sign, two exponent bits (bias 1), one mantissa bit."""
    e, m = (code >> 1) & 3, code & 1
    v = Fraction(m, 2) if e == 0 else (1 + Fraction(m, 2)) * Fraction(2) ** (e - 1)
    return -v if code & 8 else v


def test_code_values():
    assert [Fraction(float(v)) for v in MX.VALUES] == [_e2m1(c) for c in range(16)]
    assert np.signbit(MX.VALUES[8])


def test_quantize_is_the_nearest_value_of_the_block():
    """By search over all codes, in fractions; ties to the even code."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((6, 64)) * 10.0 ** rng.integers(-30, 30, (6, 1))).astype(np.float32)
    x[0, :8] = np.float32(2.0) ** np.arange(8)
    x[1, 32:] = np.arange(32) / 4
    codes, scales = MX.quantize(x)
    for r in range(6):
        for b in range(2):
            block = [Fraction(float(v)) for v in x[r, 32 * b:32 * b + 32]]
            top, e = max(abs(v) for v in block), -127
            while Fraction(2) ** (e + 3) <= top:
                e += 1
            assert scales[r, b] == e + 127
            for i, v in enumerate(block):
                code = (codes[r, 16 * b + i // 2] >> (4 * (i % 2))) & 15
                a = abs(v) / Fraction(2) ** e
                best = min(range(8), key=lambda c: (abs(_e2m1(c) - a), c & 1))
                assert code & 7 == best and bool(code & 8) == bool(np.signbit(x[r, 32 * b + i]))


def test_quantize_special_blocks():
    x = np.zeros((5, 32), dtype=np.float32)
    x[1, 3] = np.inf
    x[2, 4] = np.nan
    x[3, 0] = np.float32(2.0) ** -149
    x[4, 0] = np.finfo(np.float32).max
    codes, scales = MX.quantize(x)
    assert scales.ravel().tolist() == [0, 255, 255, 0, 252]
    assert not codes[:4].any() and codes[4, 0] == 7
    assert np.isnan(MX.decode(codes, scales)[1:3]).all()


def test_decode_and_ggml_blocks_agree():
    codes, scales = MX.gen_weights(3, 5, 96)
    v = MX.decode(codes, scales).reshape(-1, 32)
    q = MX.to_ggml(codes, scales)
    for n in range(len(q)):
        for i in range(16):  # ggml: low nibbles are elements 0..15, high ones 16..31
            s = Fraction(2) ** (int(q[n, 0]) - 127)
            assert Fraction(v[n, i]) == _e2m1(int(q[n, 1 + i]) & 15) * s
            assert Fraction(v[n, 16 + i]) == _e2m1(int(q[n, 1 + i]) >> 4) * s


def test_a_planted_mistake_is_seen():
    """Rounding ties up, a scale one step off and swapped nibbles all differ."""
    x = np.array([[0.25, 1.25, 2.5, 5.0, 4.0] + [0.75] * 27], dtype=np.float32)
    codes, scales = MX.quantize(x)
    v = MX.decode(codes, scales)[0]
    assert v[:5].tolist() == [0, 1, 2, 4, 4] and (v[5:] == 1).all()
    up = (np.abs(x[..., None]) >= np.array(MX.PLACES)).sum(-1)
    assert (up[0, :4] != [0, 2, 4, 6]).all()
    assert not np.array_equal(MX.decode(codes >> 4 | codes << 4, scales)[0], v)
    assert not np.array_equal(MX.decode(codes, scales + 1)[0], v)


def test_route_oracle_by_hand():
    logits = np.log(np.array([[1.0, 2, 4, 1]]))
    e, w = MX.route(logits, 2)
    assert e.tolist() == [[2, 1]] and np.allclose(w, [[4 / 6, 2 / 6]])
    e, w = MX.route(logits, 2, normalize=False, scale=2.0)
    assert np.allclose(w, [[1.0, 0.5]])
    # groups {0, 1} and {2, 3}: bests 2 and 4, sums of two 3 and 5
    e, _ = MX.route(logits, 1, n_groups=2, groups_kept=1)
    assert e.tolist() == [[2]]
    e, w = MX.route(np.zeros((1, 4)), 2, "sigmoid", bias=[0, 0, 0, 1])
    assert e.tolist() == [[3, 0]] and np.allclose(w, 0.5)
    e, w = MX.route(np.full((1, 3), -np.inf), 2)
    assert e.tolist() == [[-1, -1]] and not w.any()


def test_plan_oracle_by_hand():
    offsets, order = MX.plan(np.array([[2, 0], [0, -1], [5, 2]]), 3)
    assert offsets.tolist() == [0, 2, 2, 4] and order.tolist() == [1, 2, 0, 5]


def test_ggml_type_39(axc):
    assert axc.axh.ggml_type_size(axc.axh.GGML_MXFP4) == (32, 17)


def test_mxfp4_tensor_of_a_gguf_file(axc, tmp_path):
    codes, scales = MX.gen_weights(5, 3, 64)
    q = MX.to_ggml(codes, scales)
    path = tmp_path / "m.gguf"
    axc.gguf.write_gguf(path, [], [("w", axc.gguf.GGML_MXFP4, (64, 3), q.tobytes())])
    with axc.gguf.GgufFile(path) as f:
        t = f.tensors["w"]
        assert (t.type, t.n_rows, t.n_cols, t.nbytes) == (39, 3, 64, 6 * 17)
        assert f.tensor_bytes("w") == q.tobytes()


def test_plan_bytes(axc):
    assert axc.expert_plan_bytes(1, 1, 1) == 4 * (16 + 1)
    assert axc.expert_plan_bytes(10, 8, 15) == 4 * (16 + 80)
    assert axc.expert_plan_bytes(10, 8, 16) == 4 * (32 + 80)
    assert axc.expert_plan_bytes(1 << 31, 64, 1024) == 4 * (1040 + (1 << 37))


def test_matmul_kernel_names(axc):
    name = axc.mxfp4_matmul_kernel_name
    lib = axc.load_library()
    begin, end = (ctypes.addressof(ctypes.c_char.in_dll(lib, f"axh_mx_matmul_co_{n}"))
                  for n in ("begin", "end"))
    co = ctypes.string_at(begin, end - begin)
    for batch in (1, 32, 33, 64, 65, 4096):
        for rows in (1, 100, 5000, 100000):
            for t, suffix in ((0, "_f32"), (1, "_f16"), (30, "_bf16")):
                n = name(rows, 4096, batch, t)
                assert n.endswith(suffix) and n.encode() + b"\0" in co
    for bad in ((1, 0, 1, 0), (1, 48, 1, 0), (1, 1 << 23, 1, 0), (1, 32, 1, 39), (1, 32, 1, 2)):
        with pytest.raises(axc.DispatchError):
            name(*bad)


def test_calls_without_a_context_are_refused(axc):
    lib = axc.load_library()
    z = None
    for status in (lib.axh_mxfp4_quantize(z, 0, z, 0, z, z, 1, 32, z),
                   lib.axh_mxfp4_dequant(z, z, z, 0, z, 1, z),
                   lib.axh_mxfp4_unpack_ggml(z, z, z, z, 1, z),
                   lib.axh_mxfp4_matvec(z, z, z, z, z, 1, 32, z),
                   lib.axh_mxfp4_matmul(z, z, z, z, z, 0, z, 1, 32, 1, z),
                   lib.axh_expert_route(z, 0, z, z, z, z, 1, z, z),
                   lib.axh_mxfp4_expert_gate_up(z, z, z, z, z, z, z, z, 1, 32, 1, 1, 1, z),
                   lib.axh_mxfp4_expert_down(z, z, z, z, z, z, z, 1, 32, 1, 1, 1, z),
                   lib.axh_expert_plan(z, z, z, 1, 1, 1, z),
                   lib.axh_mxfp4_expert_gate_up_matmul(z, z, z, z, z, z, z, z, 0, z, z, 1, 32, 1,
                                                       1, 1, z),
                   lib.axh_mxfp4_expert_matmul(z, z, z, z, z, z, 0, z, 1, 32, 1, 1, 1, z),
                   lib.axh_expert_combine(z, 0, z, z, z, z, 1, 1, 1, 1, z)):
        assert status == 100


def test_router_product_without_a_context_is_refused(axc):
    lib = axc.load_library()
    assert lib.axh_expert_logits(None, 0, None, None, None, 4, 32, 1, None) != 0


def test_unknown_score_is_refused(axc):
    with pytest.raises(ValueError):
        axc.RouteOptions(n_experts=4, top_k=1, score="max")._c()


@pytest.fixture(scope="module")
def cases():
    """perf/operators.py with its tensors on the CPU."""
    torch = pytest.importorskip("torch")
    source = (ROOT / "perf" / "operators.py").read_text().replace('"cuda"', '"cpu"')
    spec = importlib.util.spec_from_loader("operators_on_cpu", loader=None)
    m = importlib.util.module_from_spec(spec)
    exec(compile(source, "operators.py", "exec"), m.__dict__)
    torch.manual_seed(0)
    return m


SMALL = [
    {"kind": "quantize", "x": "bf16", "rows": 5, "cols": 96},
    {"kind": "matvec", "rows": 33, "cols": 352},
    {"kind": "linear", "x": "f16", "rows": 65, "cols": 256, "batch": 7},
    {"kind": "route", "score": "sigmoid", "tokens": 50, "experts": 32, "top_k": 8, "bias": True,
     "groups": 4, "groups_kept": 2, "group_best": 2},
    {"kind": "route", "score": "softmax", "tokens": 50, "experts": 32, "top_k": 4, "bias": False,
     "groups": 1, "groups_kept": 1, "group_best": 1},
    {"kind": "decode", "tokens": 3, "experts": 8, "top_k": 3, "hidden": 128, "ffn": 64},
    {"kind": "prefill", "tokens": 40, "experts": 8, "top_k": 3, "hidden": 128, "ffn": 64},
]


@pytest.mark.parametrize("case", SMALL, ids=lambda c: c["kind"])
def test_plain_forms_of_the_performance_cases(cases, case):
    """f32 sums: 1e-6 relative by norm is far above their rounding at these
    sizes; bf16 outputs 2^-8."""
    got, want = cases.run(cases.prepare(case, 3)), cases.exact(case, 3)
    pairs = [(got[k], want[k]) for k in got] if isinstance(got, dict) else [(got, want)]
    for g, w in pairs:
        if w is None:
            continue
        assert g.shape == w.shape
        bar = 2.0 ** -8 if case["kind"] == "prefill" else 2e-6
        assert (g.double() - w).norm() <= bar * w.norm()


def test_plain_forms_agree_with_the_oracle(cases):
    t = cases._inputs(SMALL[2], 5)
    codes, scales = MX.quantize(t["x"].double().numpy())
    assert np.array_equal(cases._quantize(t["x"]).numpy(), MX.decode(codes, scales))
    assert np.array_equal(cases._decode(t["w"], t["ws"]).numpy(),
                          MX.decode(t["w"].numpy(), t["ws"].numpy()))
    case = SMALL[3]
    t = cases._inputs(case, 6)
    e, w = MX.route(t["logits"].numpy(), 8, "sigmoid", t["bias"].numpy(), 4, 2, 2)
    got = cases.run({"case": case, "t": t, "b": {}})
    assert np.array_equal(got["experts"].numpy(), e)
    assert np.allclose(got["weights"].numpy(), w, rtol=1e-5)


def test_drawn_cases_are_within_the_operators_limits(cases):
    rng = random.Random(4)
    for _ in range(400):
        c = cases.draw(rng)
        w = cases.work(c)
        assert w["bytes"] > 0 and w["flops"] <= 1.01 * cases.MAX_FLOPS
        if c["kind"] == "route":
            assert c["experts"] % c["groups"] == 0 and c["experts"] <= 1024
            assert c["top_k"] <= c["groups_kept"] * (c["experts"] // c["groups"])
        for k in ("cols", "hidden", "ffn"):
            assert c.get(k, 32) % 32 == 0


def _layer_file(axc, path, *more):
    """The layer blk.3 in the smallest sizes, of zeros, and f32 tensors called `more`."""
    n, hidden, ffn = 4, 64, 32
    shapes = [("ffn_gate_inp.weight", (hidden, n)), ("ffn_gate_exps.weight", (hidden, ffn, n)),
              ("ffn_up_exps.weight", (hidden, ffn, n)), ("ffn_down_exps.weight", (ffn, hidden, n))]
    tensors = [(f"blk.3.{name}", axc.gguf.GGML_MXFP4, s, bytes(int(np.prod(s)) // 32 * 17))
               for name, s in shapes]
    axc.gguf.write_gguf(path, [], tensors + [(name, axc.gguf.GGML_F32, (n,), bytes(4 * n))
                                             for name in more])


@pytest.mark.parametrize("name", ["ffn_gate_inp.bias", "ffn_gate_exps.bias", "ffn_up_exps.bias",
                                  "ffn_down_exps.bias", "ffn_up_exps.scale",
                                  "ffn_gate_inp_shexp.weight", "ffn_gate_shexp.weight",
                                  "ffn_up_shexp.weight", "ffn_down_shexp.weight",
                                  "ffn_gate_chexps.weight", "exp_probs_b.weight"])
def test_expert_layer_refuses_tensors_that_it_does_not_compute(axc, tmp_path, name):
    """Before anything is put on the device (there is none here)."""
    options = axc.RouteOptions(n_experts=4, top_k=1)
    _layer_file(axc, tmp_path / "layer.gguf", f"blk.3.{name}")
    with axc.gguf.GgufFile(tmp_path / "layer.gguf") as f:
        with pytest.raises(ValueError, match=f"not computed: blk.3.{name}"):
            axc.experts.ExpertLayer(None, f, "blk.3", options, max_tokens=8)
        # another name does not stand for it, its own does: then the device is asked for
        with pytest.raises(ValueError, match="not computed"):
            axc.experts.ExpertLayer(None, f, "blk.3", options, max_tokens=8,
                                    leave_out=["ffn_gate_inp"])
        with pytest.raises(AttributeError):
            axc.experts.ExpertLayer(None, f, "blk.3", options, max_tokens=8, leave_out=[name])


def test_expert_layer_takes_what_stands_beside_it(axc, tmp_path):
    """Norms, a dense feed-forward, attention and other layers' tensors are no part of it."""
    options = axc.RouteOptions(n_experts=4, top_k=1)
    _layer_file(axc, tmp_path / "layer.gguf", "blk.3.ffn_norm.weight",
                "blk.3.ffn_norm_exps.weight", "blk.3.ffn_post_norm.weight",
                "blk.3.ffn_gate.weight", "blk.3.ffn_up.weight", "blk.3.ffn_down.bias",
                "blk.3.attn_q.bias", "blk.4.ffn_up_exps.bias", "blk.31.ffn_gate_inp.bias",
                "blk.3.exp_probs_b.bias")
    with axc.gguf.GgufFile(tmp_path / "layer.gguf") as f:
        with pytest.raises(AttributeError):  # the device, which is None
            axc.experts.ExpertLayer(None, f, "blk.3", options, max_tokens=8)


def test_expert_layer_refuses_another_activation(axc, tmp_path):
    _layer_file(axc, tmp_path / "layer.gguf")
    with axc.gguf.GgufFile(tmp_path / "layer.gguf") as f:
        with pytest.raises(ValueError, match="activation"):
            axc.experts.ExpertLayer(None, f, "blk.3", axc.RouteOptions(n_experts=4, top_k=1),
                                    max_tokens=8, activation="gelu")
