"""Float64 attention over the 4-bit row cache with bounds that follow the softmax's own weights: a row lost, seen too
early or twice stands out where a bound by the largest Value would cover it.

Per element, with w the weights, e a weight's relative error and o the output:

* a relative error e_t of weight t moves the output by sum_t w_t e_t (v_t - o), at most sum w e |v| + |o| sum w e;
* scores: a term passes 5 sums inside a product of 32, one per product and part, two per group, each off by 2^-24 of
  sum |q| (|k| + 32 scale); the exponential is off by 2^-20 of itself;
* general kernel: P' = p scale in one (bf16) or two fp16 parts, each rounded, on code - 7.5; where P' is subnormal
  it is off by 2^-25, and a row's largest P' is at least 2^6 over the largest scale of its records;
* many-row kernel: a weight and a Value in fp16 (half a step 2^-11), a weight below 2^-14 off by 2^-25 where the largest
  is at least 2^7, a Value by 2^-25 where the split's largest is at least 2^14 (or all times 2^15), a query off by
  2^-25 of its row's largest element; its sum over a group in two fp16 parts (2^-22);
* sums: 5 steps inside a product of 32, one per record and the merges', 2^-23 each of sum w (|v| + 32 scale), in float32,
  whose codes count from their middle, of sum w (|v| + 8 scale);
* the output's own rounding, half a step."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from logitfill_amd.packed import int4
from oracle import int4 as o4
from tests.helpers import f32
from tests.int4_helpers import HALF_STEP, TYPES, WEIGHT_STEP, rows

PARTS = {"bf16": 1, "fp16": 2, "fp32": 3}


class Rows:
    """The rows of one (sequence, kv head): values, scales per element, and the codes' distance from their middle."""

    def __init__(self, x: np.ndarray, group: int):
        codes, scale, _ = o4.quantise(x, group)
        self.x = o4.values(x, group)
        self.scale = np.repeat(scale.astype(np.float64), group, axis=-1)
        self.codes = codes.astype(np.float64)
        self.size = np.abs(self.x) + 32 * self.scale
        self.spread = self.scale * np.abs(self.codes - 7.5)


def weights(q, k, scaling, seen):
    """Softmax weights ``[rows, T]``; a row that sees nothing has none."""
    s = np.where(seen, scaling * (q @ k.T), -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isinf(top), 0, top))
    total = p.sum(-1, keepdims=True)
    return p / np.where(total > 0, total, 1), p.max(-1, keepdims=True, initial=0) / np.where(total > 0, total, 1)


def row_bound(q, k: Rows, v: Rows, scaling, w, peak, out, dtype: str, many: bool, top=None):
    """Largest admitted error of ``out [rows, D]``; ``peak``: every row's largest weight; ``top``: the largest Value scale per
    element of rows taken back, too."""
    T, D = k.x.shape
    if T == 0:
        return np.zeros(out.shape)
    qa, av = np.abs(q), np.abs(v.x)
    steps = 10 + (D // 32) * (PARTS[dtype] + 2)
    e = abs(scaling) * steps * 2.0 ** -24 * (qa @ k.size.T) + 2.0 ** -20
    most = v.scale.max(0) if top is None else np.maximum(v.scale.max(0), top)
    if many:
        most_q = qa.max(-1, keepdims=True)
        e = e + 2.0 ** -11 + abs(scaling) * (2.0 ** -25 * most_q * (k.scale * k.codes).sum(-1)
                                             + 2.0 ** -22 * (qa @ k.size.T))
    e = w * (e * 1.05)  # (the second order)
    bound = e @ av + np.abs(out) * e.sum(-1, keepdims=True)
    bound += WEIGHT_STEP[dtype] * (w @ v.spread) + T * 2.0 ** -31 * 7.5 * peak * most
    if many:
        small = T * 2.0 ** -32 * peak
        floor = 2.0 ** -25 * max(av.max() * 2.0 ** -13, 2.0 ** -15)
        bound += 2.0 ** -11 * (w @ av) + small * (av.max(0) + np.abs(out)) + 16 * floor
    bound += (T / 32 + 20) * 2.0 ** -23 * (w @ (av + (8 if dtype == "fp32" else 32) * v.scale) + np.abs(out))
    return bound + HALF_STEP[dtype] * (np.abs(out) + bound) + 1e-37


def exact(q, key, value, lengths, group: int, scaling: float, dtype: str, *, q_lens=None, many=False, top=None,
          change=None):
    """Output and bound ``[B, n_q, n, D]``; ``change(seen, b)`` edits what the rows ``(j)`` of sequence b see, for oracles
    that are wrong on purpose (the bound stays the right one's)."""
    qn, kn, vn = (f32(t).astype(np.float64) if i == 0 else f32(t) for i, t in enumerate((q, key, value)))
    B, n_q, n, D = qn.shape
    H = kn.shape[1]
    g = n_q // H
    out, tol = np.zeros(qn.shape), np.zeros(qn.shape)
    for b, total in enumerate(lengths):
        m = n if q_lens is None else q_lens[b]
        if m == 0 or total == 0:
            continue
        at = total - m + np.arange(m)
        seen = np.arange(total)[None] <= at[:, None]
        wrong = seen if change is None else change(seen.astype(np.float64), b)
        for h in range(H):
            k, v = Rows(kn[b, h, :total], group), Rows(vn[b, h, :total], group)
            for i in range(h * g, (h + 1) * g):
                w, peak = weights(qn[b, i, :m], k.x, scaling, seen)
                right = w @ v.x
                tol[b, i, :m] = row_bound(qn[b, i, :m], k, v, scaling, w, peak, right, dtype, many, top)
                if change is not None:  # (rows counted more than once: weights of a sum that is not theirs)
                    s = scaling * (qn[b, i, :m] @ k.x.T)
                    p = np.exp(s - s.max(-1, keepdims=True)) * wrong
                    total_p = p.sum(-1, keepdims=True)
                    right = np.where(total_p > 0, p @ v.x / np.where(total_p > 0, total_p, 1), 0)
                out[b, i, :m] = right
    return out, tol


def seam_rows(shape, dtype, seed: int, q_len: int):
    """``rows``, with Values of +-128 where a mask can go wrong: at the last ``q_len`` + 1 tokens of every sequence and at the
    first and last rows of the records around them and where the many-row kernel's part ends."""
    key, value = rows(shape, dtype, seed)
    T = shape[2]
    marks = set(range(max(0, T - q_len - 1), T))
    for t in (T - q_len, T - q_len - 32, T - q_len // 2, 0, 32):
        marks |= {t // 32 * 32 + d for d in (-1, 0, 31, 32)}
    marks = sorted(t for t in marks if 0 <= t < T)
    # (in four channels of its own each: in all of them their sum would cover one that is missing)
    g = torch.Generator().manual_seed(seed + 5)
    for t in marks:
        at = torch.randperm(shape[3], generator=g)[:4]
        value[:, :, t] = 0
        value[:, :, t, at] = torch.tensor([128.0, 128.0, -128.0, -128.0]).to(TYPES[dtype])
    return key, value


@pytest.fixture
def prefixes(monkeypatch):
    """Every attention call's splits of the many-row kernel."""
    args, blocks = int4._args, []

    def record(*a, **k):
        blocks.append(args(*a, **k))
        return blocks[-1]
    monkeypatch.setattr(int4, "_args", record)
    return lambda: [a.prefix_splits for a in blocks]
