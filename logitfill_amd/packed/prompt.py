"""Causal attention of whole prompts: sequences of unlike lengths, packed one behind another or padded to a batch.

* ``PromptPlan``       -- the lengths of a batch of prompts and the work they make; kept for all layers.
* ``prompt_attention`` -- attention of every sequence's tokens to its Keys up to their own.

It is a prompt's first pass, whose rows are not in a cache yet (the caches' own attention serves what follows);
with more Keys than queries the queries are the last tokens: a prompt fed in pieces, single tokens.  No reference
counterpart (its prefill runs the model's dense attention, ``src/logitfill/models/qwen2_attention.py:76-146``).
Nothing here runs on the CPU.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import numpy as np
import torch

from logitfill_amd import _native
from logitfill_amd.packed.cache import _check_device
from logitfill_amd.packed.reference import _cu_count

MAX_TOKENS = 1 << 24  # of a sequence (LF_PROMPT_TOKENS)


def key_tile(head_dim: int, dtype) -> int:
    """``LF_PROMPT_KEYS``."""
    return 32 if head_dim == 256 or dtype == torch.float32 else 64


def tile_rows(lengths, group: int) -> int:
    """Query rows of a workgroup: one wave's 32 where no sequence has more, else four waves' 128."""
    return 32 if max(lengths) * group <= 32 else 128


def split_size(batch: _native.PromptBatch) -> tuple[int, int]:
    """``(Key tiles that a workgroup takes at most, its groups)``: ``lf_prompt_split``."""
    split = (ctypes.c_int32 * 2)()
    _native.check(_native.load().lf_prompt_split(batch, split), "lf_prompt_split")
    return split[0], split[1]


class _Form(NamedTuple):
    """A plan's work for one form of call, on the device."""

    items: torch.Tensor
    n_items: int
    n_merges: int
    n_slots: int
    rows: int
    groups: int
    stream: int
    event: torch.cuda.Event


def work_items(lengths, key_lengths, packed_q: bool, packed_k: bool, group: int, rows: int, head_dim: int, dtype, n_kv: int, cus: int,
               tokens: int = 0):
    """The ``lf_prompt_item`` rows of a call (int32 ``[n, 12]``) and, behind them, of its merges; ``(n_items, n_merges, n_slots)`` and
    the groups of a workgroup.  What lies behind the sequences in rows of ``tokens`` is queries that see no Key, whose output is
    zeros."""
    n, m = np.asarray(lengths, dtype=np.int32), np.asarray(key_lengths, dtype=np.int32)
    batch = _native.PromptBatch(n.ctypes.data, m.ctypes.data, len(n), packed_q, packed_k, tokens, group, n_kv, head_dim,
                                _native.dtype_code(dtype), rows, cus)
    size, groups = split_size(batch)
    counts = (ctypes.c_int32 * 3)()
    lib = _native.load()
    cap = 0
    while True:  # (asks for the counts first)
        items = np.zeros((cap, 12), dtype=np.int32)
        status = lib.lf_prompt_items(batch, size, items.ctypes.data, cap, counts)
        if status != _native.LF_E_WORKSPACE or cap:
            break
        cap = counts[0] + counts[1]
    _native.check(status, "lf_prompt_items")
    return items, tuple(counts), groups


class PromptPlan:
    """The sequences of a batch of prompts: ``lengths[b]`` query tokens, the last of ``key_lengths[b]`` (default: as many)
    Keys.  Holds the work of every form of call made with it (head counts, types), on the device: keep it for a
    model's layers, and as long as a captured graph that used it."""

    def __init__(self, lengths, key_lengths=None, *, device="cuda"):
        self.lengths = [int(n) for n in lengths]
        self.key_lengths = list(self.lengths) if key_lengths is None else [int(n) for n in key_lengths]
        if not self.lengths or len(self.key_lengths) != len(self.lengths):
            raise ValueError("a plan takes the lengths of at least one sequence, and as many key_lengths")
        if min(self.lengths + self.key_lengths) < 0 or max(self.lengths + self.key_lengths) > MAX_TOKENS:
            raise ValueError(f"lengths must lie in 0 .. {MAX_TOKENS}")
        self.device = _check_device(device)
        self._longest = max(self.lengths), max(self.key_lengths)
        self._total = sum(self.lengths), sum(self.key_lengths)
        self._forms: dict = {}
        self._args: dict = {}  # argument blocks by the tensors' forms

    @property
    def batch(self) -> int:
        return len(self.lengths)

    def _rows(self, shape, of: int, name: str) -> bool:
        """Whether the sequences' queries (``of`` 0) or Keys (1) lie packed in ``[B, heads, T, D]``; ``ValueError`` where they do
        not fit."""
        B, T = shape[0], shape[2]
        if B == len(self.lengths) and self._longest[of] <= T:
            return False  # (one sequence: both forms are the same)
        if B == 1 and self._total[of] <= T:
            if self._total[of] >= 1 << 31:
                raise ValueError(f"{name}: at most 2^31 - 1 packed tokens")
            return True
        lengths = (self.lengths, self.key_lengths)[of]
        raise ValueError(f"{name} {tuple(shape)} does not hold sequences of {lengths[:8]}{'...' if self.batch > 8 else ''} tokens")

    def _form(self, packed_q: bool, packed_k: bool, group: int, n_kv: int, head_dim: int, dtype, tokens: int) -> _Form:
        key = (packed_q, packed_k, group, n_kv, head_dim, dtype, tokens)
        form = self._forms.get(key)
        if form is None:
            stream = _native.current_stream_ptr(self.device)
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a plan's first call uploads its work: run the step once before the capture")
            rows = tile_rows(self.lengths, group)
            items, counts, groups = work_items(self.lengths, self.key_lengths, packed_q, packed_k, group, rows, head_dim, dtype, n_kv,
                                                      _cu_count(self.device), tokens)
            with torch.inference_mode(False):
                device = _native.upload(items.reshape(-1), torch.int32, self.device)
            event = torch.cuda.Event()
            event.record(torch.cuda.current_stream(self.device))
            form = self._forms[key] = _Form(device, *counts, rows, groups, stream, event)
        return form

    def _order(self, form: _Form, stream: int) -> None:
        """The current stream, ``stream``, behind the upload of a form's work (a capture follows a run)."""
        if stream != form.stream and not torch.cuda.is_current_stream_capturing():
            here = torch.cuda.current_stream(self.device)
            here.wait_event(form.event)
            form.items.record_stream(here)


def _check_rows(t: torch.Tensor, name: str, query: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernel reads it: unit channel stride, rows on 16 bytes."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}; logitfill_amd runs on ROCm devices only")
    if t.device != query.device:
        raise ValueError(f"{name} is on {t.device}, the query on {query.device}")
    if t.dim() != 4:
        raise ValueError(f"{name} must be [batch, heads, tokens, head_dim], got {tuple(t.shape)}")
    if t.dtype != query.dtype:
        raise TypeError("query, key and value must share a dtype")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, which prompt_attention does not give: call it under torch.no_grad()")
    size = t.element_size()
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(s * size % 16 for s in _native.steps(t)):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: float,
                     plan: Optional[PromptPlan] = None) -> torch.Tensor:
    """Causal attention: ``query [B, n_q, T, D]``, ``key / value [B, n_kv, S, D]`` -> ``[B, n_q, T, D]`` (tokens
    outermost in memory, as an output projection takes it); bf16, fp16 or fp32, any strides, head_dim 64, 128 or 256.

    ``plan``: the sequences.  B of them, each from the start of its own row (padded), or, in a batch of one row, all
    behind one another (packed); queries and Keys each in one of the two ways.  None: every row is a sequence of
    all its tokens (not in a capture).  A sequence's queries are the last of its Keys, and each sees the Keys up to its own.  Rows of
    the output behind a sequence's last token, and rows of queries that see no Key, are zeros.  What a row does not see need
    not be finite; a Value that it sees and that is not counts whatever its weight.  Finite ones in bf16 and fp32 may overflow
    the sums past 2^119 over the tokens.

    Everything is enqueued on the current stream."""
    scaling = float(scaling)
    if plan is None and query.is_cuda and query.dim() == key.dim() == 4 and query.shape[0] == key.shape[0] > 0:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured call takes a plan, which the graph's replays read: make one before the capture")
        plan = _whole(query.shape[0], query.shape[2], key.shape[2], query.device)
    if plan is not None:  # (tensors of a form that has been checked)
        kept = plan._args.get(_form_of(query, key, value, scaling))
        if kept is not None:
            q, k, v = query.data_ptr(), key.data_ptr(), value.data_ptr()
            if not (q | k | v) & 15 and query.device == key.device == value.device == plan.device and not (
                    torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad)):
                if torch.cuda.current_device() == plan.device.index:
                    return _launch(query, key, value, plan, *kept)
                with torch.cuda.device(plan.device):
                    return _launch(query, key, value, plan, *kept)
    if not math.isfinite(scaling):
        raise ValueError(f"scaling must be finite, got {scaling}")
    query, key, value = (_check_rows(t, name, query) for t, name in ((query, "query"), (key, "key"), (value, "value")))
    B, n_q, T, D = query.shape
    n_kv = key.shape[1]
    if key.shape != value.shape or key.shape[3] != D:
        raise ValueError(f"key and value must be of one shape [B, n_kv, S, {D}], got {tuple(key.shape)} and {tuple(value.shape)}")
    if n_kv <= 0 or n_q <= 0 or n_q % n_kv:
        raise ValueError("query heads must divide into KV heads")
    if D not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {D}")
    code = _native.dtype_code(query.dtype)
    if plan is None:
        if key.shape[0] != B:
            raise ValueError(f"query has {B} rows, key {key.shape[0]}")
        return torch.empty(B, T, n_q, D, dtype=query.dtype, device=query.device).transpose(1, 2)
    if plan.device != query.device:
        raise ValueError(f"query is on {query.device}, the plan on {plan.device}")
    packed_q, packed_k = plan._rows(query.shape, 0, "query"), plan._rows(key.shape, 1, "key")
    if T * (n_q // n_kv) > 1 << 30:
        raise ValueError("too many query tokens for one call: feed them in chunks")
    with torch.cuda.device(query.device):
        if not plan._longest[0] or not plan._longest[1]:
            return torch.zeros(B, T, n_q, D, dtype=query.dtype, device=query.device).transpose(1, 2)
        form = plan._form(packed_q, packed_k, n_q // n_kv, n_kv, D, query.dtype, T)
        if len(plan._args) >= 64:
            plan._args.clear()
        kept = plan._args[_form_of(query, key, value, scaling)] = (_describe(query, key, value, code, scaling, form), form)
        return _launch(query, key, value, plan, *kept)


def _form_of(query, key, value, scaling: float):
    """What a call's argument block hangs on, but for the tensors' addresses."""
    return (query.shape, query.stride(), query.dtype, key.shape, key.stride(), key.dtype, value.shape, value.stride(), value.dtype,
            scaling)


@functools.lru_cache(maxsize=64)
def _whole(B: int, T: int, S: int, device) -> PromptPlan:
    return PromptPlan([T] * B, [S] * B, device=device)


def _describe(query, key, value, code: int, scaling: float, form: _Form):
    """The argument block of calls of one form, without their tensors' addresses."""
    a = _native.PromptArgs()
    B, n_q, T, D = query.shape
    a.dtype, a.n_q, a.n_kv, a.head_dim = code, n_q, key.shape[1], D
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = _native.steps(query), _native.steps(key), _native.steps(value)
    a.out_strides[:] = T * n_q * D, D, n_q * D
    a.scaling, a.tile_rows, a.groups = scaling, form.rows, form.groups
    a.items, a.n_items = form.items.data_ptr(), form.n_items
    if form.n_merges:
        a.merges, a.n_merges, a.n_slots = a.items + 48 * form.n_items, form.n_merges, form.n_slots
        a.workspace_bytes = 4 * form.n_slots * a.n_kv * form.rows * (D + 2)  # lf_prompt_workspace_bytes
    return a


def _launch(query, key, value, plan: PromptPlan, kept, form: _Form) -> torch.Tensor:
    """``prompt_attention`` of checked tensors on the current device."""
    B, n_q, T, D = query.shape
    stream = _native.current_stream_ptr(plan.device)
    if stream != form.stream:
        plan._order(form, stream)
    out = torch.empty((B, T, n_q, D), dtype=query.dtype, device=plan.device)
    a = _native.PromptArgs.from_buffer_copy(kept)
    a.query, a.key, a.value, a.out = query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr()
    if form.n_merges:
        ws = torch.empty(kept.workspace_bytes, dtype=torch.uint8, device=plan.device)
        a.workspace = ws.data_ptr()
    _native.check(_native.load().lf_prompt_attention(a, stream), "lf_prompt_attention")
    return out.transpose(1, 2)
