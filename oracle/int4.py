"""CPU restatement of the 4-bit row cache: rows quantised per group of channels, their values, page
bounds, attention and page selection, in NumPy (values and sums in float64)."""
from __future__ import annotations

import numpy as np

from oracle.layout import F32


def quantise(x: np.ndarray, group: int):
    """Codes (uint8), scale and minimum (float16) of float32 rows ``x [..., D]``: every step in float32."""
    g = x.astype(F32).reshape(*x.shape[:-1], x.shape[-1] // group, group)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    scale = np.clip((hi - lo) / F32(15), F32(1e-5), F32(1e5)).astype(F32)
    codes = np.clip(np.rint((g - lo) / scale), 0, 15).astype(np.uint8)
    return codes.reshape(x.shape), scale[..., 0].astype(np.float16), lo[..., 0].astype(np.float16)


def values(x: np.ndarray, group: int) -> np.ndarray:
    """Float64 of what the cache holds of rows ``x`` (exact: an 11- by 4-bit product and a sum)."""
    codes, scale, lo = quantise(x, group)
    c = codes.reshape(*x.shape[:-1], x.shape[-1] // group, group).astype(np.float64)
    v = c * scale.astype(np.float64)[..., None] + lo.astype(np.float64)[..., None]
    return v.reshape(x.shape)


def to_bf16_up(x: np.ndarray) -> np.ndarray:
    """float32 rounded up to bfloat16 (as float32)."""
    u = np.ascontiguousarray(x, dtype=F32).view(np.uint32).astype(np.int64)
    up = np.where(u >> 31, u, u + 0xFFFF) >> 16 << 16
    return up.astype(np.uint32).view(F32)


def bounds(vals: np.ndarray, page: int) -> np.ndarray:
    """Float32 ``[n_kv, pages, 2, D]``: every full page's bounds of ``vals [n_kv, T, D]``, bfloat16 outward."""
    H, T, D = vals.shape
    v = vals[:, : T // page * page].astype(F32).reshape(H, T // page, page, D)
    return np.stack([-to_bf16_up(-v.min(2)), to_bf16_up(v.max(2))], 2)


def select(q: np.ndarray, bnd: np.ndarray, own: int, top: int) -> np.ndarray:
    """Pages of one (query token, kv head): ``q [g, D]``, ``bnd [pages, 2, D]``; -1 behind the last one."""
    out = np.full(top, -1, dtype=np.int32)
    if own > 0:
        lo, hi = (bnd[None, :own, i].astype(np.float64) for i in (0, 1))
        wide = q.astype(np.float64)[:, None]
        score = np.maximum(wide * lo, wide * hi).sum(-1).max(0)
        picked = np.sort(np.argsort(-score, kind="stable")[:top])
        out[: len(picked)] = picked
    return out


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scaling: float, seen: np.ndarray) -> np.ndarray:
    """Float64 softmax attention of ``q [rows, D]`` over ``k, v [T, D]`` where ``seen [rows, T]``; a row that
    sees nothing is zeros."""
    if k.shape[0] == 0:
        return np.zeros(q.shape)
    s = np.where(seen, scaling * (q.astype(np.float64) @ k.T), -np.inf)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isinf(top), 0, top))
    total = p.sum(-1, keepdims=True)
    return np.where(total > 0, (p @ v) / np.where(total > 0, total, 1), 0.0)
