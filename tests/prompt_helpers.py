"""Inputs, float64 results and error bounds of the prompt attention's tests."""
from __future__ import annotations

import numpy as np
import torch

from tests.helpers import f32

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def inputs(shape_q, shape_k, dtype: str, seed: int):
    """Query, Key, Value rows: a scale per channel of the Keys with outliers."""
    g = torch.Generator().manual_seed(seed)
    D = shape_q[-1]
    sigma = torch.exp(0.7 * torch.randn(D, generator=g))
    sigma[:: D // 4] *= 8
    q = torch.randn(shape_q, generator=g) * D ** -0.5
    k = torch.randn(shape_k, generator=g) * sigma
    v = torch.randn(shape_k, generator=g)
    return tuple(t.to(TYPES[dtype]) for t in (q, k, v))


def attend(q, k, v, scaling: float, seen, dtype: str):
    """Float64 softmax attention of rows ``q [n, D]`` with the mask ``seen [n, T]``, and the largest admitted error.

    * the output's rounding, HALF_STEP of it;
    * a weight is rounded to the rows' type (not in fp32): HALF_STEP of the weighted mean of |v|; fp16 weights are
      formed as 2^7 or more where the row's largest is, so that one below fp16's least step is off by 2^-25 / 2^7;
    * a score is a sum of D products in float32, in any order: off by D 2^-24 of sum |q k|; times the scale, less the
      reference point and its exponential: 4 2^-24 of the largest score's size and 2^-20; a score off by d moves the
      weights by e^d above and below the quotient, 2 d of the largest |v|;
    * float32 sums of T weights and weighted Values, the parts' merges: (T + 40) 2^-24 of the weighted mean of |v|."""
    n, T = seen.shape
    out, tol = np.zeros((n, v.shape[1])), np.zeros((n, v.shape[1]))
    rows = seen.any(1)
    if not rows.any():
        return out, tol
    q, seen = q[rows].astype(np.float64), seen[rows]
    s = np.where(seen, (q @ k.T) * scaling, -np.inf)
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    mean = w @ np.abs(v)
    size = abs(scaling) * np.where(seen, np.abs(q) @ np.abs(k).T, 0).max(1, keepdims=True)
    d = q.shape[1] * 2.0 ** -24 * size + 4 * 2.0 ** -24 * size + 2.0 ** -20
    reach = np.where(seen[:, :, None], np.abs(v)[None], 0).max(1) if T * v.size * n < 1 << 26 else np.abs(v).max(0, keepdims=True)
    out[rows] = w @ v
    bound = HALF_STEP[dtype] * np.abs(out[rows]) + 2 * d * reach + (T + 40) * 2.0 ** -24 * mean
    if dtype != "fp32":
        bound += HALF_STEP[dtype] * mean * (1 + HALF_STEP[dtype])
    if dtype == "fp16":
        bound += T * 2.0 ** -32 * reach + 2.0 ** -25
    tol[rows] = bound
    return out, tol


def expected(q, k, v, lengths, key_lengths, scaling: float, dtype: str, packed_q: bool, packed_k: bool):
    """``(out, tolerance) [B, n_q, T, D]`` in float64; rows that no sequence has: zeros, exactly."""
    qn, kn, vn = (f32(t).astype(np.float64) for t in (q, k, v))
    out, tol = np.zeros(qn.shape), np.zeros(qn.shape)
    g = qn.shape[1] // kn.shape[1]
    qa = ka = 0
    for b, (n, m) in enumerate(zip(lengths, key_lengths)):
        (qb, q0), (kb, k0) = (0, qa) if packed_q else (b, 0), (0, ka) if packed_k else (b, 0)
        seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + m - n
        for h in range(qn.shape[1]):
            r = attend(qn[qb, h, q0 : q0 + n], kn[kb, h // g, k0 : k0 + m], vn[kb, h // g, k0 : k0 + m], scaling, seen, dtype)
            out[qb, h, q0 : q0 + n], tol[qb, h, q0 : q0 + n] = r
        qa, ka = qa + n, ka + m
    return out, tol


def assert_within(ours: torch.Tensor, ref: np.ndarray, tol: np.ndarray, what=""):
    diff = np.abs(ours.detach().double().cpu().numpy() - ref)
    assert np.isfinite(diff).all(), f"{what}: {int((~np.isfinite(diff)).sum())} values are not finite"
    bad = diff > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} outside, worst {(diff / np.maximum(tol, 1e-30)).max():.3g} x the bound"
