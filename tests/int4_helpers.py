"""Inputs, the float64 results and the error bounds of the 4-bit row cache's tests."""
from __future__ import annotations

import numpy as np
import torch

from oracle import int4 as o4
from tests.helpers import f32

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
# P' = p * scale is kept in one, two and two fp16 parts, each rounded
WEIGHT_STEP = {"bf16": 2.0 ** -11, "fp16": 2.0 ** -22, "fp32": 2.0 ** -22}


def rows(shape, dtype: str, seed: int):
    """Key, Value rows: a scale per channel with outliers, normal Values."""
    g = torch.Generator().manual_seed(seed)
    sigma = torch.exp(torch.randn(shape[-1], generator=g))
    sigma[:: shape[-1] // 4] *= 10
    key = torch.randn(shape, generator=g) * sigma
    value = torch.randn(shape, generator=g)
    return key.to(TYPES[dtype]), value.to(TYPES[dtype])


def query(shape, dtype: str, seed: int):
    g = torch.Generator().manual_seed(seed + 77)
    return (torch.randn(shape, generator=g) * shape[-1] ** -0.5).to(TYPES[dtype])


def _size(x, group: int) -> np.ndarray:
    """|value| + 32 scale of every element: codes enter the products counted from -16."""
    scale = np.repeat(o4.quantise(x, group)[1].astype(np.float64), group, axis=-1)
    return np.abs(o4.values(x, group)) + 32 * scale


def many_rows_bound(q, k, v, scaling):
    """What the many-row kernel's fp16 steps add: a Key off by 2^-11 of itself (2^-25 at least) and a query by 2^-24
    of its row's largest element move a score by d; a weight off by 2^-11 and a Value off by 2^-11 (2^-25)."""
    if k.shape[0] == 0:
        return 0.0
    a, qa = np.abs(k), np.abs(q).astype(np.float64)
    d = abs(scaling) * ((qa @ (a * 2.0 ** -11 + 2.0 ** -25).T).max(-1, keepdims=True)
                        + 2.0 ** -24 * qa.max(-1, keepdims=True) * a.sum(-1).max())
    return (2 * d + 3 * 2.0 ** -11) * np.abs(v).max() + 2.0 ** -25


def attention_bound(q, k_size, v_size, scaling, ref, dtype: str, smax: float, top: float):
    """Largest admitted |out - ref| per element of ``ref [rows, D]``.

    * the output's rounding;
    * a rounding of P' = p * scale moves the output by at most that step times scale * |code - 7.5|, and by
      2^-25 times 7.5 over the sum of the weights where P' is subnormal: the weights' largest is at least
      2^7 over the largest scale of a record, ``top`` where rows of it were taken back;
    * float32: a score's term passes 5 sums inside a product of 32, one per product and part, two per
      group, each off by 2^-24 of sum |q| (|k| + 32 scale); the exponential is off by 2^-20; a score off by
      d moves the weights by a factor e^d above and below the quotient; the Value sums pass T / 32
      records and the merges, each off by 2^-23 of |v| + 32 scale.
    """
    T, D = k_size.shape
    if T == 0:
        return np.zeros(ref.shape)
    parts = {"bf16": 1, "fp16": 2, "fp32": 3}[dtype]
    steps = 10 + (D // 32) * (parts + 2)
    size = (np.abs(q).astype(np.float64) @ k_size.T).max(-1, keepdims=True)
    d = abs(scaling) * steps * 2.0 ** -24 * size + 2.0 ** -20
    reach = v_size.max()
    return (HALF_STEP[dtype] * np.abs(ref) + 7.5 * (WEIGHT_STEP[dtype] * smax + T * 2.0 ** -32 * top) + 2 * d * reach
            + (T / 32 + 40) * 2.0 ** -23 * reach)


def expected(q, key, value, lengths, group: int, scaling: float, dtype: str, *, page=0, pages=None, q_lens=None, top=0.0):
    """Float64 output and its bound, ``[B, n_q, n, D]``: ``key/value [B, H, T, D]`` are the rows written, sequence b
    holding the first ``lengths[b]`` (``top``: the largest Value scale of rows taken back); with ``pages`` [B, H, n, K] the attended pages."""
    qn, kn, vn = f32(q), f32(key), f32(value)
    B, n_q, n, D = qn.shape
    H = kn.shape[1]
    g = n_q // H
    out, tol = np.zeros(qn.shape), np.zeros(qn.shape)
    for b, total in enumerate(lengths):
        m = n if q_lens is None else q_lens[b]
        for h in range(H):
            k, v = o4.values(kn[b, h, :total], group), o4.values(vn[b, h, :total], group)
            k_size, v_size = _size(kn[b, h, :total], group), _size(vn[b, h, :total], group)
            smax = float(o4.quantise(vn[b, h, :total], group)[1].max(initial=0))
            for j in range(m):
                at = total - m + j
                seen = np.arange(total) <= at
                if pages is not None and at >= 0:
                    own = at // page
                    attended = {own}
                    last = -1
                    for p in pages[b, h, j]:
                        if 0 <= p < own and p > last:
                            attended.add(int(p))
                        last = p
                    seen &= np.isin(np.arange(total) // page, list(attended))
                head = slice(h * g, (h + 1) * g)
                r = o4.attend(qn[b, head, j], k, v, scaling, np.broadcast_to(seen, (g, total)))
                out[b, head, j] = r
                tol[b, head, j] = attention_bound(qn[b, head, j], k_size[seen], v_size[seen], scaling, r, dtype, smax,
                                                   max(smax, top))
                if pages is None and g * n >= 64 and k.shape[-1] <= 128 and dtype != "fp32":
                    tol[b, head, j] += many_rows_bound(qn[b, head, j], k[seen], v[seen], scaling)
    return out, tol


def assert_within(ours: torch.Tensor, ref: np.ndarray, tol: np.ndarray, what=""):
    diff = np.abs(ours.detach().double().cpu().numpy() - ref)
    assert np.isfinite(diff).all(), f"{what}: {int((~np.isfinite(diff)).sum())} values are not finite"
    bad = diff > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} outside, worst {(diff / np.maximum(tol, 1e-30)).max():.3g} x the bound"
