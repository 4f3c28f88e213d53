"""Rotary positions for the queries and Keys that the caches' attention takes.

``Rotary`` holds a model's frequencies; ``rotate`` turns query and Key rows by their tokens' positions in
one launch.  Angles are formed in float64: a position of 2^20 loses none of its bits.  No reference
counterpart (there the model's own code rotates, ``src/logitfill/models/qwen2_attention.py:76-146``).
Nothing here runs on the CPU.
"""
from __future__ import annotations

import math
import operator
from typing import Optional

import torch

from logitfill_amd import _native
from logitfill_amd.packed.cache import _check_device

LAYOUTS = ("half", "interleaved")
MAX_START = 1 << 53  # what float64 counts exactly


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None) -> tuple[list[float], float]:
    """Every pair's angle per position, and the factor on the rotated channels.

    Pair i turns by ``base^(-2 i / rotary_dim)`` a position.  ``scaling`` stretches that for contexts
    ``factor`` times as long as the model was trained on:

    * ``{"type": "linear", "factor": s}`` -- every frequency over s (positions are interpolated).
    * ``{"type": "ntk", "factor": s}`` -- base times s^(rotary_dim / (rotary_dim - 2)): the slowest pair
      is stretched by s, the fastest not at all.
    * ``{"type": "yarn", "factor": s, "original_positions": n}`` -- pairs that turn at most
      ``beta_slow`` (1) times over n positions are over s, those that turn at least ``beta_fast`` (32)
      times stay, those between are mixed in proportion to their index; rotated channels are multiplied
      by ``attention_factor`` (0.1 ln s + 1)."""
    if not (math.isfinite(base) and base > 1):
        raise ValueError(f"base must be a finite number above 1, got {base}")
    kind, s = None, 1.0
    if scaling is not None:
        left = dict(scaling)
        kind, s = left.pop("type", None), float(left.pop("factor", 1.0))
        if kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"scaling type must be linear, ntk or yarn, got {kind!r}")
        if not (math.isfinite(s) and s >= 1):
            raise ValueError(f"scaling factor must be a finite number of at least 1, got {s}")
        original = left.pop("original_positions", None)
        fast, slow = float(left.pop("beta_fast", 32.0)), float(left.pop("beta_slow", 1.0))
        attention = left.pop("attention_factor", None)
        if left:
            raise ValueError(f"scaling has no {', '.join(map(repr, left))}")
        if kind == "ntk":
            if rotary_dim < 4:
                raise ValueError("ntk scaling takes a rotary_dim of at least 4")
            base = base * s ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == "linear":
        return [f / s for f in freq], 1.0
    if kind != "yarn":
        return freq, 1.0
    if original is None or not original > 0 or not fast > slow > 0:
        raise ValueError("yarn scaling takes original_positions above 0 and beta_fast above beta_slow above 0")

    def pair_of(turns):
        return rotary_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

    first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
    width = max(last - first, 0.001)
    mixed = [min(max((i - first) / width, 0.0), 1.0) for i in range(rotary_dim // 2)]
    factor = 0.1 * math.log(s) + 1 if attention is None else float(attention)
    return [f / s * m + f * (1 - m) for f, m in zip(freq, mixed)], factor


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new tensor of ``t``'s memory order (contiguous where that does not end with the channels)."""
    out = torch.empty_like(t)
    return out if out.stride(3) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


class Rotary:
    """The rotation of a model's rows of ``head_dim`` channels (even, up to 512).

    ``rotary_dim``: the front channels that are rotated (even; default all).  ``layout``: pairs are channel
    j of both halves of those (``"half"``) or neighbours (``"interleaved"``).  ``scaling``: see
    ``frequencies``.  ``inv_freq``: the pairs' angles per position in place of ``base`` and ``scaling``
    (a model's own), with ``attention_factor`` on the rotated channels.  A captured graph reads the frequencies: keep the
    object as long as it."""

    def __init__(self, head_dim: int, base: float = 10000.0, *, rotary_dim: Optional[int] = None, layout: str = "half",
                 scaling: Optional[dict] = None, inv_freq=None, attention_factor: Optional[float] = None, device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 2 <= self.head_dim <= 512 or self.head_dim % 2:
            raise ValueError(f"head_dim must be even, 2 .. 512, got {head_dim}")
        if not 2 <= self.rotary_dim <= self.head_dim or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even, 2 .. {self.head_dim}, got {rotary_dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
        self.layout = layout
        if inv_freq is None:
            freq, factor = frequencies(self.rotary_dim, float(base), scaling)
        else:
            if scaling is not None:
                raise ValueError("inv_freq takes the place of scaling")
            freq, factor = [float(f) for f in inv_freq], 1.0
            if len(freq) != self.rotary_dim // 2 or not all(map(math.isfinite, freq)):
                raise ValueError(f"inv_freq must hold {self.rotary_dim // 2} finite numbers")
        self.inv_freq = freq
        self.attention_factor = factor if attention_factor is None else float(attention_factor)
        if not math.isfinite(self.attention_factor):
            raise ValueError(f"attention_factor must be finite, got {attention_factor}")
        self.device = _check_device(device)
        # (a copy from pageable memory has ended when it returns: any stream may read it)
        with torch.inference_mode(False):
            self._turns = torch.tensor([f / (2 * math.pi) for f in freq], dtype=torch.float64).to(self.device)
        self._stream = _native.current_stream_ptr(self.device)
        self._args: dict = {}  # argument blocks by the tensors' forms

    def _check_rows(self, t: torch.Tensor, name: str) -> torch.Tensor:
        if t.device != self.device:
            if not t.is_cuda:
                raise RuntimeError(f"{name} is on {t.device}; logitfill_amd runs on ROCm devices only")
            raise ValueError(f"{name} is on {t.device}, the frequencies on {self.device}")
        if t.dim() != 4 or t.shape[3] != self.head_dim:
            raise ValueError(f"{name} must be [batch, heads, tokens, {self.head_dim}], got {tuple(t.shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient, which rotate does not give: call it under torch.no_grad()")
        return t if t.stride(3) == 1 else t.contiguous()

    def rotate(self, query: torch.Tensor, key: Optional[torch.Tensor], positions):
        """``(query, key)`` rotated: ``query [B, n_q, T, D]`` and ``key [B, n_kv, T, D]`` (or None) of one type (bf16,
        fp16 or fp32), any strides; new tensors of the inputs' memory order.  ``positions``: every token's, an int32 or
        int64 tensor ``[T]``, ``[1, T]`` or ``[B, T]`` on the device, or the first token's as an int (the others
        follow it).  Enqueued on the current stream."""
        tensor = isinstance(positions, torch.Tensor)
        form = (query.shape, query.stride(), query.dtype,
                None if key is None else (key.shape, key.stride(), key.dtype),
                (positions.shape, positions.stride(), positions.dtype) if tensor else None)
        kept = self._args.get(form)
        if kept is None or query.device != self.device or (key is not None and key.device != self.device) or (
                tensor and positions.device != self.device) or (
                torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))):
            query, key = self._check(query, key, positions)
            form = (query.shape, query.stride(), query.dtype, None if key is None else (key.shape, key.stride(), key.dtype), form[4])
            kept = self._args.get(form)
        q_out, k_out = _like(query), None if key is None else _like(key)
        if query.numel() == 0 and (key is None or key.numel() == 0):
            return q_out, k_out
        if kept is None:
            if len(self._args) >= 64:
                self._args.clear()
            kept = self._args[form] = self._describe(query, key, q_out, k_out, form[4])
        a = _native.RotaryArgs.from_buffer_copy(kept)
        a.query, a.query_out = query.data_ptr(), q_out.data_ptr()
        if key is not None:
            a.key, a.key_out = key.data_ptr(), k_out.data_ptr()
        if tensor:
            a.positions = positions.data_ptr()
        else:
            a.start = operator.index(positions)
            if a.start != positions or not -MAX_START <= a.start <= MAX_START:
                raise ValueError(f"the first position must lie in -2^53 .. 2^53, got {positions}")
        if torch.cuda.current_device() == self.device.index:
            self._launch(a)
        else:
            with torch.cuda.device(self.device):
                self._launch(a)
        return q_out, k_out

    def _check(self, query, key, positions):
        """Query and Key as the kernel reads them; errors for what it does not."""
        query = self._check_rows(query, "query")
        B, n_q, T, D = query.shape
        if key is not None:
            key = self._check_rows(key, "key")
            if key.shape[0] != B or key.shape[2] != T:
                raise ValueError(f"key must be [{B}, n_kv, {T}, {D}], got {tuple(key.shape)}")
            if key.dtype != query.dtype:
                raise TypeError("query and key must share a dtype")
        if B * T >= 1 << 27 or n_q + (0 if key is None else key.shape[1]) > 4096:
            raise ValueError("at most 2^27 - 1 tokens and 4096 heads a call")
        _native.dtype_code(query.dtype)
        if isinstance(positions, torch.Tensor):
            if positions.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
            if positions.device != self.device:
                raise ValueError(f"positions are on {positions.device}, the frequencies on {self.device}")
            shape = positions.shape
            if shape != (T,) and shape != (1, T) and shape != (B, T):
                raise ValueError(f"positions must be [{T}], [1, {T}] or [{B}, {T}], got {tuple(shape)}")
        return query, key

    def _describe(self, query, key, q_out, k_out, where):
        """The argument block of calls of this form, without their addresses."""
        a = _native.RotaryArgs()
        a.dtype = _native.dtype_code(query.dtype)
        a.batch, a.n_q, a.tokens, a.head_dim = query.shape
        a.n_kv = 0 if key is None else key.shape[1]
        a.rotary_dim, a.interleaved = self.rotary_dim, self.layout == "interleaved"
        a.turns, a.factor = self._turns.data_ptr(), self.attention_factor
        a.q_strides[:], a.qo_strides[:] = _native.steps(query), _native.steps(q_out)
        if key is not None:
            a.k_strides[:], a.ko_strides[:] = _native.steps(key), _native.steps(k_out)
        if where is not None:
            shape, stride, dtype = where
            a.wide = dtype == torch.int64
            a.position_strides[0] = stride[0] if len(shape) == 2 and shape[0] > 1 else 0
            a.position_strides[1] = stride[-1]
        return a

    def _launch(self, a) -> None:
        stream = _native.current_stream_ptr(self.device)
        if stream != self._stream and not torch.cuda.is_current_stream_capturing():
            self._turns.record_stream(torch.cuda.current_stream(self.device))
        _native.check(_native.load().lf_rotary(a, stream), "lf_rotary")
