"""MXFP4 and expert layers restated in numpy, 64 bits: the oracle of the
MXFP4 operations (the reference has no counterpart).

Formats: OCP Microscaling Formats v1.0 (E2M1 elements, E8M0 scale for 32);
ggml's 17-byte blocks of the same values.
"""
from __future__ import annotations

import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
# places between two magnitudes; a tie goes to the code with mantissa bit 0
PLACES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scales) bytes of rows x cols values: scale 2^(floor(log2 max) - 2),
    at least 2^-127; 255 and codes 0 where a block holds an infinity or a NaN."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    b = x.reshape(rows, cols // 32, 32)
    m = np.abs(b).max(axis=2)
    bad = ~np.isfinite(b).all(axis=2)
    safe = np.where(bad | (m == 0), 1.0, m)
    e = np.clip(np.frexp(safe)[1] - 1 - 2, -127, 127)
    e = np.where(m == 0, -127, e)
    with np.errstate(invalid="ignore"):
        a = np.abs(np.where(bad[..., None], 0.0, b)) * np.exp2(-e)[..., None]
    code = np.zeros(b.shape, dtype=np.uint8)
    for k, place in enumerate(PLACES):
        code += ((a >= place) if k % 2 else (a > place)).astype(np.uint8)
    code |= np.where(np.signbit(b), 8, 0).astype(np.uint8)
    code[bad] = 0
    code = code.reshape(rows, cols)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """The values (64 bits) of (..., cols / 2) codes and (..., cols / 32) scales."""
    v = np.stack([VALUES[codes & 15], VALUES[codes >> 4]], axis=-1)
    v = v.reshape(*scales.shape, 32) * np.exp2(scales.astype(np.float64) - 127)[..., None]
    v = np.where((scales == 255)[..., None], np.nan, v)
    return v.reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def to_ggml(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """17-byte ggml blocks of the same values (n x 17 bytes)."""
    n = scales.size
    c = codes.reshape(n, 16)
    code = np.stack([c & 15, c >> 4], axis=-1).reshape(n, 32)
    out = np.zeros((n, 17), dtype=np.uint8)
    out[:, 0] = scales.reshape(-1)
    out[:, 1:] = code[:, :16] | (code[:, 16:] << 4)
    return out


def swiglu(g: np.ndarray, u: np.ndarray) -> np.ndarray:
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


def route(logits: np.ndarray, top_k: int, score: str = "softmax", bias=None, n_groups: int = 1,
          groups_kept: int = 1, group_best: int = 1, normalize: bool = True, scale: float = 1.0):
    """(experts, weights) of tokens x experts logits, one token at a time."""
    logits = np.asarray(logits, dtype=np.float64)
    tokens, n = logits.shape
    chosen = np.full((tokens, top_k), -1, dtype=np.int32)
    weights = np.zeros((tokens, top_k))
    for t in range(tokens):
        l = np.where(np.isnan(logits[t]), -np.inf, logits[t])
        open_ = l > -np.inf
        s = np.zeros(n)
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                s[open_] = 1 / (1 + np.exp(-l[open_]))
        elif open_.any():
            m = l[open_].max()
            with np.errstate(invalid="ignore"):
                e = np.where(l[open_] == m, 1.0, np.exp(l[open_] - m))
            s[open_] = e / e.sum()
        s = s.astype(np.float32).astype(np.float64)  # scores are f32: 0 below its range
        key = l.copy() if bias is None and (n_groups == 1 or group_best == 1) else s.copy()
        if bias is not None:
            key = key + np.asarray(bias, dtype=np.float64)
        key[~open_ | np.isnan(key)] = -np.inf
        if n_groups > 1:
            per = n // n_groups
            best = np.sort(key.reshape(n_groups, per), axis=1)[:, ::-1]
            if group_best == 2 and per == 1:
                gk = np.full(n_groups, -np.inf)
            else:
                gk = best[:, :group_best].sum(axis=1)
            kept = np.argsort(-gk, kind="stable")[:groups_kept]
            mask = np.ones(n_groups, dtype=bool)
            mask[kept] = False
            key[np.repeat(mask, per)] = -np.inf
        order = np.argsort(-key, kind="stable")[:top_k]
        order = order[key[order] > -np.inf]
        chosen[t, :len(order)] = order
        w = s[order]
        if normalize and w.sum() > 0:
            w = w / w.sum()
        weights[t, :len(order)] = w * scale
    return chosen, weights


def plan(experts: np.ndarray, n_experts: int) -> tuple[np.ndarray, np.ndarray]:
    """(offsets, slots by expert) of tokens x top_k choices."""
    flat = np.asarray(experts).reshape(-1)
    lists = [np.nonzero(flat == e)[0] for e in range(n_experts)]
    offsets = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    return offsets.astype(np.uint32), np.concatenate(lists).astype(np.uint32)


def gen_weights(seed: int, *shape: int) -> tuple[np.ndarray, np.ndarray]:
    """Random codes and scales of (..., cols) weights; products with unit
    activations are near 1."""
    rng = np.random.default_rng(seed)
    *rows, cols = shape
    mid = 127 - int(np.log2(3 * np.sqrt(cols)))
    codes = rng.integers(0, 256, (*rows, cols // 2), dtype=np.uint8)
    return codes, rng.integers(mid - 1, mid + 2, (*rows, cols // 32), dtype=np.uint8)
