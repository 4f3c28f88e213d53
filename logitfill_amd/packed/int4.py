"""A KV cache held in 4 bits, quantised as it is written, and the attention that reads it.

It stands beside ``PackedKVManager`` for the cases that need no tier table: every token's Key and
Value row is kept as 4-bit codes with a float16 scale and minimum per ``group_size`` channels (the
rule of ``layout.asymmetric_codes`` at 4 bits), written the moment it is committed.  There is no
residual page and nothing to flush, the cache can be truncated (rejected draft tokens), and every
write position lives on the device, so a step that commits and attends can be captured in a HIP
graph and replayed until the capacity is reached.

* ``Int4KVManager``  -- the cache of a model's layers (``commit``, ``truncate``, ``reset``; a layer's
  ``read`` / ``dequantize``).
* ``int4_attention`` -- commits the new tokens, then attends over the cached rows; with ``pages``
  over those pages and the query's own one only; of a manager with a ``prefix``, behind the rows of another
  manager that several of its sequences share.
* ``select_pages``   -- the pages whose Keys' bounds admit the largest ``q . k``, per query token and
  kv head.

No reference counterpart: the reference's packed backend keeps Values at 2 bits in its kernel and
falls back to the dense path for other widths (``src/logitfill/packed/reference.py:62-68``).
Nothing here runs on the CPU.
"""
from __future__ import annotations

import ctypes
import functools
import math
import threading
from typing import Optional

import torch

from logitfill_amd import _native
from logitfill_amd.packed.cache import _check_device
from logitfill_amd.packed.reference import _cu_count

BLOCK = 32  # tokens of a storage record
MAX_SPLITS = 1024
MAX_PAGES = 1024


def _block_bytes(head_dim: int, group: int) -> int:
    """``LF_INT4_BLOCK_BYTES``."""
    return BLOCK * (head_dim + 8 * (head_dim // group))


def check_layout(head_dim: int, page_size: int, group_size: int) -> None:
    """The layouts the kernels serve; ``ValueError`` for any other."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if group_size not in (32, 64, 128) or group_size > head_dim:
        raise ValueError(f"group_size must be 32, 64 or 128 and at most head_dim {head_dim}, got {group_size}")
    if page_size <= 0 or page_size % BLOCK or page_size > 1024:
        raise ValueError(f"page_size must be a multiple of {BLOCK} up to 1024, got {page_size}")


def _here(fn):
    """``fn(owner, ...)`` with the owner's device current (the default stream names no device)."""
    @functools.wraps(fn)
    def call(owner, *args, **kwargs):
        if torch.cuda.current_device() == owner.device.index:
            return fn(owner, *args, **kwargs)
        with torch.cuda.device(owner.device):
            return fn(owner, *args, **kwargs)
    return call


def _check_rows(t: torch.Tensor, device: torch.device, name: str) -> torch.Tensor:
    """``t`` as the kernels read it: on this device, a row type they take, unit channel stride."""
    if t.device != device:
        if not t.is_cuda:
            raise RuntimeError(f"{name} is on {t.device}; logitfill_amd runs on ROCm devices only")
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    _native.dtype_code(t.dtype)
    if t.requires_grad:
        t = t.detach()
    return t if t.stride(-1) == 1 else t.contiguous()


@functools.lru_cache(maxsize=256)
def _stride_array(strides: tuple):
    return (ctypes.c_int64 * 3)(*strides[:3])


def _strides(t: torch.Tensor):
    return _stride_array(t.stride())


def _ints(values):
    return (ctypes.c_int32 * len(values))(*values)


class _Lengths:
    """The device's lengths of a cache's layers, int32 ``[layers, batch]``, and their order among streams.

    Appends move them on the stream of their call.  What the host sets (``truncate``, ``reset``) belongs to the stream that
    was current there: the next call on it brings a layer's lengths along (an append in its arguments, any other
    call by a launch), and the first call on any other stream sets there what is still to be set and waits for that
    stream.  Where graphs name the arrays, whose replays ask nobody, the lengths are set at once."""

    def __init__(self, layers: int, batch: int, device: torch.device):
        self.device = device
        with torch.inference_mode(False):
            self.rows = torch.zeros(layers, batch, dtype=torch.int32, device=device)
        self.layers: list = []
        self.lock = threading.RLock()  # over a layer's host lengths and the launch that takes them to the device
        self._at = None     # the handle of the stream of the host's last change
        self._event = None  # there, once another stream has asked

    def changed(self) -> None:
        """The host has changed lengths (of layers now ``_dirty``) at this place of the current stream."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("lengths that the host sets are a step of their own: set them before the capture")
        self._at, self._event = _native.current_stream_ptr(self.device), None

    def order(self, at: int) -> None:
        """The current stream, ``at``, behind the host's last change."""
        if self._at is None or at == self._at:
            return
        with self.lock:
            if self._event is None:
                there = torch.cuda.ExternalStream(self._at, self.device) if self._at else torch.cuda.default_stream(self.device)
                with torch.cuda.stream(there):
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("the stream on which the cache was truncated is being captured: "
                                           "call manager.sync_lengths() before the capture")
                    self.send()
                    event = torch.cuda.Event()
                    event.record()
                self._event = event
            event = self._event
        torch.cuda.current_stream(self.device).wait_event(event)

    def send(self, every: bool = False) -> None:
        """The host's lengths to the device, of the layers that wait for it (or all), on the current stream; under the lock."""
        todo = [layer for layer in self.layers if (layer._dirty or every) and layer.capacity]
        if not todo:
            return
        if len(todo) < len(self.layers):
            for layer in todo:
                layer.send_lengths()
            return
        s = _native.Int4Layer.from_buffer_copy(max(todo, key=lambda layer: layer.capacity).describe())
        batch = self.rows.shape[1]
        some = max(1, 65535 // batch)  # layers in one call: to it they are more sequences
        for i in range(0, len(todo), some):
            part = [n for layer in todo[i : i + some] for n in layer.lengths]
            s.lens, s.batch = self.rows[i].data_ptr(), len(part)
            _native.check(_native.load().lf_int4_set_lens(s, _ints(part), _native.current_stream_ptr(self.device)),
                          "lf_int4_set_lens")
        for layer in todo:
            layer._dirty = False


class _Int4Store:
    """One layer's 4-bit rows for ``batch`` sequences; ``lens``: its row of ``order``."""

    def __init__(self, n_kv: int, head_dim: int, page_size: int, group_size: int, order: _Lengths, lens: torch.Tensor, *,
                 device="cuda", batch: int = 1, capacity_tokens: int = 0):
        self.device = _check_device(device)
        self.n_kv, self.head_dim = int(n_kv), int(head_dim)
        self.page_size, self.group_size = int(page_size), int(group_size)
        check_layout(self.head_dim, self.page_size, self.group_size)
        if self.n_kv <= 0 or int(batch) <= 0:
            raise ValueError("n_kv and batch must be positive")
        self.batch = int(batch)
        self.lengths = [0] * self.batch
        self._cap = 0
        self._blocks: Optional[torch.Tensor] = None
        self._bounds: Optional[torch.Tensor] = None
        self._struct: Optional[_native.Int4Layer] = None
        self._order, self._lens = order, lens
        self._dirty = False  # the device's lengths are behind the host's
        self._tops: Optional[torch.Tensor] = None
        self._captured = False  # a graph names the arrays, and its replays move the device's lengths
        self._kept: list = []   # arrays that a captured graph may still name
        if capacity_tokens:
            self.reserve(capacity_tokens)

    @property
    def length(self) -> int:
        """Tokens of sequence 0."""
        return self.lengths[0]

    @property
    def capacity(self) -> int:
        return self._cap

    # ---- storage -------------------------------------------------------------
    def reserve(self, tokens: int) -> None:
        """Grow the capacity to at least ``tokens`` per sequence (doubling, page aligned).  The new arrays have
        other addresses: a captured graph keeps the old ones (which live as long as the cache), so reserve before the
        capture."""
        P = self.page_size
        need = -(-int(tokens) // P) * P
        if need <= self._cap:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"the cache holds {self._cap} tokens and the captured step needs {tokens}: "
                               "reserve the capacity before the capture")
        cap = max(need, 2 * self._cap)
        if cap > 1 << 30:
            cap = need
        if cap > 1 << 30:
            raise ValueError(f"{tokens} tokens per sequence (at most {1 << 30})")
        B, H, D = self.batch, self.n_kv, self.head_dim
        with torch.inference_mode(False), torch.no_grad():
            blocks = torch.zeros(B, H, cap // BLOCK, _block_bytes(D, self.group_size), dtype=torch.uint8,
                                 device=self.device)
            bounds = torch.zeros(B, H, cap // P, 2, D, dtype=torch.bfloat16, device=self.device)
            tops = torch.zeros(B, H, cap // BLOCK, dtype=torch.float16, device=self.device)
            if self._cap:
                tops[:, :, : self._cap // BLOCK].copy_(self._tops)
                blocks[:, :, : self._cap // BLOCK].copy_(self._blocks)
                bounds[:, :, : self._cap // P].copy_(self._bounds)
            # the copies run on this stream, which need not be the arrays' own; a captured graph may still name them
            old = (self._blocks, self._bounds, self._tops)
            for t in old if self._cap else ():
                t.record_stream(torch.cuda.current_stream(self.device))
            if self._captured:
                self._kept.append(old)
        self._blocks, self._bounds, self._tops = blocks, bounds, tops
        self._cap, self._struct = cap, None

    def describe(self) -> _native.Int4Layer:
        """The ``lf_int4_layer`` describing this store."""
        if self._cap == 0:
            self.reserve(self.page_size)
        if self._struct is None:
            s = _native.Int4Layer()
            s.blocks, s.bounds, s.lens = self._blocks.data_ptr(), self._bounds.data_ptr(), self._lens.data_ptr()
            s.tops = self._tops.data_ptr()
            s.batch, s.n_kv, s.head_dim = self.batch, self.n_kv, self.head_dim
            s.cap_tokens, s.page_size, s.group = self._cap, self.page_size, self.group_size
            self._struct = s
        return self._struct

    def send_lengths(self) -> None:
        """The host's lengths to the device, on the current stream."""
        _native.check(_native.load().lf_int4_set_lens(self.describe(), _ints(self.lengths),
                                                      _native.current_stream_ptr(self.device)), "lf_int4_set_lens")
        self._dirty = False

    def layer_struct(self, lengths: bool = True) -> _native.Int4Layer:
        """``describe()`` for a call on the current stream, in its place behind what the host set; ``lengths``: the device's
        up to date there."""
        s = self.describe()
        if torch.cuda.is_current_stream_capturing():
            if lengths and self._dirty:
                raise RuntimeError("the cache was truncated or reset since its last launch: "
                                   "call manager.sync_lengths() before the capture")
            self._captured = True
            return s
        self._order.order(_native.current_stream_ptr(self.device))
        if lengths and self._dirty:
            with self._order.lock:
                self.send_lengths()
        return s

    def page_bounds(self) -> torch.Tensor:
        """bf16 ``[batch, n_kv, capacity / page_size, 2, head_dim]``: every full page's smallest and largest Key per
        channel (the values read back, rounded outward); what stands behind a sequence's full pages has no meaning."""
        if self._cap == 0:
            self.reserve(self.page_size)
        return self._bounds

    # ---- rows ------------------------------------------------------------------
    def check_append(self, key: torch.Tensor, value: torch.Tensor, lengths):
        """Checked ``(key, value, per-sequence counts or None)`` of an append."""
        shape = key.shape
        if len(shape) != 4 or shape != value.shape:
            raise ValueError(f"Key and Value rows must be of one shape [batch, n_kv, T, head_dim], got "
                             f"{tuple(shape)} and {tuple(value.shape)}")
        B, H, T, D = shape
        if B != self.batch or H != self.n_kv or D != self.head_dim:
            raise ValueError(f"expected [{self.batch}, {self.n_kv}, T, {self.head_dim}], got {tuple(shape)}")
        if key.dtype != value.dtype:
            raise TypeError("key and value must share a dtype")
        key, value = _check_rows(key, self.device, "key"), _check_rows(value, self.device, "value")
        if lengths is not None:
            lengths = [int(n) for n in lengths]
            if len(lengths) != B or min(lengths) < 0 or max(lengths) > T:
                raise ValueError("lengths must give 0 <= length <= T for every sequence")
            if min(lengths) == T:
                lengths = None
        return key, value, lengths

    def append_batch(self, key: torch.Tensor, value: torch.Tensor, lengths=None) -> None:
        """Append ``key/value [batch, n_kv, T, head_dim]`` (sequence b its first ``lengths[b]`` tokens)."""
        self._append(*self.check_append(key, value, lengths))

    @_here
    def _append(self, key: torch.Tensor, value: torch.Tensor, lengths) -> None:
        T = key.shape[2]
        if T == 0 or (lengths is not None and max(lengths) == 0):
            return
        old = self.lengths
        new = [n + T for n in old] if lengths is None else [n + t for n, t in zip(old, lengths)]
        if max(new) > self._cap:
            self.reserve(max(new))
        # the rows go where the host's lengths end and the device's follow; a captured commit moves the device's own, when
        # it is replayed, and advance() the host's
        captured = torch.cuda.is_current_stream_capturing()
        s = self.layer_struct(captured)
        with self._order.lock:
            st = _native.load().lf_int4_append(
                s, key.data_ptr(), value.data_ptr(), _native.dtype_code(key.dtype), _strides(key), _strides(value),
                None if captured else _ints(old), None if lengths is None else _ints(lengths), T,
                _native.current_stream_ptr(self.device))
            _native.check(st, "lf_int4_append")
            if not captured:
                self.lengths, self._dirty = new, False

    @_here
    def read(self, starts, tokens: int, dtype=torch.float32):
        """``tokens`` rows of every sequence read back: ``(K, V) [batch, n_kv, tokens, head_dim]``, row t of sequence b
        the cache's row ``starts[b] + t`` (an int for all; rows outside the sequence are zeros)."""
        starts = [int(starts)] * self.batch if isinstance(starts, int) else [int(x) for x in starts]
        tokens = int(tokens)
        if len(starts) != self.batch or min(starts) < 0 or max(starts) > 1 << 30 or not 0 <= tokens <= 1 << 30:
            raise ValueError("read takes one start per sequence and a number of tokens, none negative")
        code = _native.dtype_code(dtype)
        k = torch.empty(self.batch, self.n_kv, tokens, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if tokens:
            st = _native.load().lf_int4_read(self.layer_struct(), _ints(starts), tokens, k.data_ptr(), v.data_ptr(),
                                             code, _native.current_stream_ptr(self.device))
            _native.check(st, "lf_int4_read")
        return k, v

    def dequantize(self, b: int = 0):
        """Dense float32 ``(K, V) [n_kv, length, head_dim]`` of sequence ``b`` (as ``_LayerStore.dequantize``)."""
        if not 0 <= b < self.batch:
            raise IndexError(f"sequence {b} of a batch of {self.batch}")
        k, v = self.read(0, self.lengths[b])
        return k[b], v[b]


class Int4KVManager:
    """The 4-bit cache of ``n_layers`` layers for ``batch_size`` sequences.

    ``head_dim`` 64, 128 or 256; ``group_size`` 32, 64 or 128 channels per scale and minimum;
    ``page_size`` (a multiple of 32 up to 1024) is the unit of ``select_pages``.  ``top_pages``: the
    model integration attends that many selected pages per query and kv head (0: every row).
    ``prefix``: another manager whose sequences stand in front of this one's (the attribute, too).
    """

    commits_new_tokens = True  # the attention writes the new tokens before it reads

    def __init__(self, n_layers: int, n_q: int, n_kv: int, head_dim: int, page_size: int = 128, group_size: int = 64,
                 device="cuda", *, batch_size: int = 1, capacity_tokens: int = 0, top_pages: int = 0,
                 prefix: Optional["Int4KVManager"] = None):
        self.n_q, self.n_kv, self.head_dim = int(n_q), int(n_kv), int(head_dim)
        self.page_size, self.group_size = int(page_size), int(group_size)
        self.batch_size, self.top_pages = int(batch_size), int(top_pages)
        if self.n_kv <= 0 or self.n_q <= 0 or self.n_q % self.n_kv:
            raise ValueError("query heads must divide into KV heads")
        if self.batch_size <= 0 or int(n_layers) < 0:
            raise ValueError("batch_size must be positive and n_layers not negative")
        if not 0 <= self.top_pages <= MAX_PAGES:
            raise ValueError(f"top_pages must lie in 0 .. {MAX_PAGES}, got {top_pages}")
        check_layout(self.head_dim, self.page_size, self.group_size)
        self.device = _check_device(device)
        self.seq_len = 0
        self._lens = _Lengths(int(n_layers), self.batch_size, self.device)
        self.layers = [_Int4Store(self.n_kv, self.head_dim, self.page_size, self.group_size, self._lens, row,
                                  device=self.device, batch=self.batch_size, capacity_tokens=capacity_tokens)
                       for row in self._lens.rows]
        self._lens.layers = self.layers
        self._args: dict = {}
        self._prefix: Optional[Int4KVManager] = None
        self.prefix = prefix

    @property
    def prefix(self) -> Optional["Int4KVManager"]:
        """The manager of a prefix that this one's sequences share, or None: of ``prefix.batch_size`` prefixes, each in
        front of ``batch_size / prefix.batch_size`` sequences in turn (all the samples of a prompt, the chats behind a system
        prompt).  ``int4_attention`` then attends a prefix's rows, read once for all its sequences, and the sequence's own
        behind them; commits, ``truncate`` and ``reset`` are of the own rows, and the prefix may be written between calls
        as any cache.  A captured call reads the prefix's arrays and device lengths in its replays, by the split plan of the
        captured ones: keep it as long as the graph."""
        return self._prefix

    @prefix.setter
    def prefix(self, prefix: Optional["Int4KVManager"]) -> None:
        if prefix is not None:
            if not isinstance(prefix, Int4KVManager):
                raise TypeError(f"prefix must be an Int4KVManager, got {type(prefix).__name__}")
            mine = (self.n_q, self.n_kv, self.head_dim, self.group_size, len(self.layers), self.device)
            its = (prefix.n_q, prefix.n_kv, prefix.head_dim, prefix.group_size, len(prefix.layers), prefix.device)
            if mine != its:
                raise ValueError(f"the prefix has (n_q, n_kv, head_dim, group_size, layers, device) {its}, the manager {mine}")
            if self.batch_size % prefix.batch_size:
                raise ValueError(f"{prefix.batch_size} prefixes do not divide {self.batch_size} sequences")
            if prefix is self or prefix.prefix is not None:
                raise ValueError("a prefix stands in front of every row: it has no prefix of its own")
            if self.top_pages:
                raise ValueError("a manager of top_pages takes no prefix: pages are selected among its own rows")
        self._prefix = prefix

    def prefix_lengths(self, layer_idx: int) -> list:
        """Tokens in front of every sequence's own (zeros without a prefix)."""
        if self._prefix is None:
            return [0] * self.batch_size
        lengths = self._prefix.layers[layer_idx].lengths
        return [n for n in lengths for _ in range(self.batch_size // len(lengths))]

    def commit(self, layer_idx: int, key: torch.Tensor, value: torch.Tensor, lengths=None) -> None:
        """Append ``key/value [batch, n_kv, T, head_dim]`` to layer ``layer_idx``, quantised as they are written.
        ``lengths``: per-sequence token counts for ragged batches."""
        if key.shape[0] != self.batch_size:
            raise NotImplementedError(
                f"this manager holds {self.batch_size} sequence(s); got a batch of {key.shape[0]}")
        self.layers[layer_idx].append_batch(key, value, lengths)
        self._note(layer_idx)

    def _note(self, layer_idx: int) -> None:
        if self.layers[layer_idx] is self.layers[-1]:
            self.seq_len = self.layers[-1].length

    def layer_length(self, layer_idx: int) -> int:
        return self.layers[layer_idx].length

    def truncate(self, lengths) -> None:
        """Forget every layer's tokens past ``lengths[b]`` (an int for all; rejected draft tokens, a prompt's common
        start).  A write on the current stream: it follows the calls and replays that stand there, and later calls on
        other streams wait for that stream (a replay does not by itself).  Before a capture, call ``sync_lengths``."""
        lengths = [int(lengths)] * self.batch_size if isinstance(lengths, int) else [int(n) for n in lengths]
        if len(lengths) != self.batch_size:
            raise ValueError("truncate takes one length per sequence")
        for layer in self.layers:
            if any(n < 0 or n > have for n, have in zip(lengths, layer.lengths)):
                raise ValueError(f"truncate to {lengths}: the cache holds {layer.lengths}")
        self._set_lengths(lengths)

    @_here
    def _set_lengths(self, lengths: list) -> None:
        captured = any(layer._captured for layer in self.layers)
        if captured or any(layer.lengths != lengths for layer in self.layers):
            with self._lens.lock:
                self._lens.changed()
                for layer in self.layers:
                    layer.lengths, layer._dirty = list(lengths), True
                if captured:
                    self._lens.send()
        self.seq_len = self.layers[-1].length if self.layers else 0

    def advance(self, tokens) -> None:
        """Tell the host of tokens that replays of a captured step committed on the device (per sequence, or an int for
        all): graph replays move the device's lengths only."""
        tokens = [int(tokens)] * self.batch_size if isinstance(tokens, int) else [int(n) for n in tokens]
        if len(tokens) != self.batch_size or min(tokens) < 0:
            raise ValueError("advance takes one count of tokens per sequence, none negative")
        for layer in self.layers:
            if any(n + t > layer.capacity for n, t in zip(layer.lengths, tokens)):
                raise ValueError("more tokens than the cache's capacity")
        for layer in self.layers:
            layer.lengths = [n + t for n, t in zip(layer.lengths, tokens)]
        self.seq_len = self.layers[-1].length if self.layers else 0

    @_here
    def sync_lengths(self) -> None:
        """Set the device's lengths to the host's on the current stream (before a capture; after replays that ``advance`` is
        not told of)."""
        for layer in self.layers:
            layer.describe()
        self._lens.order(_native.current_stream_ptr(self.device))
        with self._lens.lock:
            self._lens.changed()
            self._lens.send(every=True)

    def reset(self) -> None:
        """Forget every token (storage is kept for reuse); a write on the current stream, as ``truncate``."""
        self._set_lengths([0] * self.batch_size)


def _check_query(manager, query: torch.Tensor, paged: bool) -> torch.Tensor:
    shape = query.shape
    if len(shape) != 4 or shape[0] != manager.batch_size or shape[1] != manager.n_q or shape[3] != manager.head_dim:
        raise ValueError(f"query must be [{manager.batch_size}, {manager.n_q}, q_len, {manager.head_dim}], "
                         f"got {tuple(shape)}")
    n, group = shape[2], manager.n_q // manager.n_kv
    if n < 1:
        raise ValueError("query holds no token")
    # (the kernels' grids)
    tiles = -(-group // 16) * n if paged else -(-group * n // 16)
    if n * manager.n_q > 1 << 20 or shape[0] * n * manager.n_q >= 1 << 24 or manager.n_kv * tiles > 65535:
        raise ValueError(f"{n} query tokens are too many for one call: feed them in chunks")
    return _check_rows(query, manager.device, "query")


def _query_lengths(manager, q_len: int, lengths):
    """Per-sequence query tokens as a device tensor, or None when every sequence has ``q_len``."""
    if lengths is None:
        return None
    lengths = [int(n) for n in lengths]
    if len(lengths) != manager.batch_size or min(lengths) < 0 or max(lengths) > q_len:
        raise ValueError("lengths must give 0 <= length <= q_len for every sequence")
    if min(lengths) == q_len:
        return None
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a call of ragged lengths uploads them and cannot be captured")
    return _native.upload(lengths, torch.int32, manager.device)


def _workspace(manager, nbytes: int) -> torch.Tensor:
    """Scratch of one call, of the current stream's memory (in a capture the graph's own): calls on other streams or
    from other threads, and other graphs, have another."""
    return torch.empty(nbytes, dtype=torch.uint8, device=manager.device)


def _args(manager, query: torch.Tensor, counts, scaling: float) -> _native.Int4Args:
    """The call's argument block: a copy of the one kept for the query's form, with this call's tensors."""
    key = (query.shape[2], query.dtype, query.stride(), scaling)
    kept = manager._args.get(key)
    if kept is None:
        if len(manager._args) >= 64:
            manager._args.clear()
        kept = a = _native.Int4Args()
        a.dtype = _native.dtype_code(query.dtype)
        a.n_q, a.q_len = manager.n_q, int(query.shape[2])
        a.q_strides = _strides(query)
        a.scaling = float(scaling)
        manager._args[key] = kept
    a = _native.Int4Args.from_buffer_copy(kept)
    a.query = query.data_ptr()
    if counts is not None:
        a.q_lens = counts.data_ptr()
    return a


# Tokens a split is a multiple of (a record for each of a workgroup's four waves).
SPLIT_UNIT = 128
# A workgroup's fixed cost (its queries, the first records' way, the waves' merge, its share of the splits') in
# units of its work: some 5 us against 2 us a unit.  A many-row workgroup writes eight times the sums.
SPLIT_OVERHEAD = 3.0
MANY_ROWS_OVERHEAD = 4.0


def workgroups_per_cu(head_dim: int, group: int) -> int:
    """Attention workgroups that a plan counts per CU: the 4, 3 and 2 of the kernels' launch bounds at head_dim 64, 128
    and 256 (the registers of bf16 groups of 128 at head_dim 128, 123, admit 4, those of groups of 64 at head_dim 64,
    78, admit 6), and by the record rings' LDS 1 at head_dim 256 with groups of 32."""
    return {64: 4, 128: 3, 256: 2 if group > 32 else 1}[head_dim]


def many_rows_per_cu(head_dim: int, group: int) -> int:
    """Many-row workgroups that a CU holds, by registers."""
    return 2 if head_dim == 128 and group < 128 else 3


@functools.lru_cache(maxsize=512)
def _plan(units: tuple, rows: int, slots: int, overhead: float, most: int) -> int:
    """Units a split takes, of sequences of ``units`` (their work, ``rows`` workgroups a split): the size of least
    estimated time -- all work and every split's fixed cost over the slots, and part of a split's for the last round,
    or one split's where all are there at once.  No sequence is in more than ``most``."""
    total, longest = sum(units) * rows, max(units)
    least = -(-longest // most)

    def items(size):
        return rows * sum(-(-u // size) for u in units)

    share = max(1, least, -(-total // slots))
    sizes = {max(least, total // (slots * k), 1) for k in (2, 3, 4, 6, 8, 12, 16)} | {share, longest}
    # the first size past the even share that makes one round of sequences it does not divide
    once = next((size for size in range(share, min(longest, 2 * share) + 1) if items(size) <= slots), None)
    if once:
        sizes.add(once)

    # (one round of unlike items leaves the compute units unlike loads: 32 contexts of 4K-64K tokens in 6 splits, all
    # there at once, 322 us, in 10 290, in 24 297; 16 equal ones in 12 56, in 24 62)
    uneven = 1.0 if min(units) == longest else 1.15

    def cost(size):
        n = items(size)
        return uneven * (size + overhead) if n <= slots else (total + overhead * n) / slots + 0.3 * size

    return min((min(size, longest) for size in sorted(sizes, reverse=True)), key=cost)


def plan_splits(tokens, rows: int, cus: int, per_cu: int = 3, overhead: float = SPLIT_OVERHEAD,
                most: int = MAX_SPLITS) -> tuple[int, int]:
    """``(splits, tokens of each)`` for sequences of ``tokens`` rows (an int, or one per sequence), ``rows``
    workgroups per sequence and split; at most ``most`` splits."""
    tokens = (tokens,) if isinstance(tokens, int) else tokens
    size = _plan(tuple([(n + SPLIT_UNIT - 1) // SPLIT_UNIT or 1 for n in tokens]), rows, per_cu * cus,
                 overhead, most) * SPLIT_UNIT
    return -(-max(max(tokens), 1) // size), size


# From this many query rows per kv head up, this many tokens in front of the queries, and this many products of a
# row's channel and a token's in front of them (per 32 channels of a group: the general kernel takes a term per group), the
# many-row kernel takes what every query sees (bf16: it holds weights and Values in fp16).  It unpacks a record once for 128
# rows, and costs two launches, 128-row partial sums and their merge, which is work per row: past MANY_ROWS_FULL rows in all
# the products have to grow with them.  28 / 4 heads of 128, general against many-row, us, groups of 128, 64 and 32 (32 / 8
# heads): one sequence of 16K tokens, 64 queries 45 / 58, 51 / 53, 67 / 54 (28 / 4), 128 73 / 74, 86 / 75, 118 / 81, 512 225 /
# 192, 266 / 203, 359 / 241; four of 4K, 512 queries 210 / 236, 254 / 237, 390 / 284; of 2K 108 / 154, 131 / 153, 201 / 181;
# of 16K 827 / 624, 993 / 741, 1 556 / 896.  14 / 2 heads of 64, one sequence of 16K, 512 queries, groups of 64 and 32: 95 / 76
# and 119 / 79; four of 2K 42 / 63 and 53 / 65.
MANY_ROWS = 64
MANY_ROWS_HISTORY = 256
MANY_ROWS_WORK = 3e9
MANY_ROWS_FULL = 12000


def _many_rows(group: int, q_len: int, n_kv: int, head_dim: int, group_size: int, dtype, tokens) -> bool:
    """Whether the many-row kernel takes part in the attention of sequences of ``tokens``."""
    rows = group * q_len
    if rows < MANY_ROWS or head_dim > 128 or dtype != torch.bfloat16 or max(tokens) < q_len + MANY_ROWS_HISTORY:
        return False
    work = sum(n - q_len for n in tokens if n > q_len) * rows * n_kv * head_dim
    return work >= MANY_ROWS_WORK * {32: 1, 64: 2, 128: 3}[group_size] * max(1.0, rows * n_kv * len(tokens) / MANY_ROWS_FULL)


def int4_attention(manager: Int4KVManager, layer_idx: int, query: torch.Tensor, key_new: Optional[torch.Tensor],
                   value_new: Optional[torch.Tensor], scaling: float, *, lengths=None,
                   pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Commit the new tokens, then attend: ``query [B, n_q, q_len, D]`` -> ``[B, n_q, q_len, D]``.

    ``key_new / value_new [B, n_kv, q_len, D]`` (None: they are in the cache already) are appended to
    the layer as ``manager.commit`` does; the queries are the sequence's last ``q_len`` tokens, each
    of which sees the cached rows up to its own.  ``lengths``: per-sequence token counts of a ragged
    batch; rows of the output behind them, and rows of queries that see no token, are zeros.

    ``pages`` (int32 ``[B, n_kv, q_len, n]``, from ``select_pages``): each query token attends its own
    page up to itself and the listed pages before it.  Entries ascend; a negative one, one that is
    not before the own page or not above its predecessor is not attended.  Without it a manager of
    ``top_pages`` selects that many itself.

    Of a manager with a ``prefix``, whose rows stand in front of the sequences' own, each prefix is read once for all
    its sequences (no ``pages``).

    Everything is enqueued on the current stream.
    """
    scaling = float(scaling)
    if not math.isfinite(scaling):
        raise ValueError(f"scaling must be finite, got {scaling}")
    layer = manager.layers[layer_idx]
    query = _check_query(manager, query, pages is not None or manager.top_pages > 0)
    q_len = query.shape[2]
    B = manager.batch_size
    if manager._prefix is not None:
        if pages is not None or manager.top_pages:  # (the attribute may be set behind the prefix)
            raise ValueError("pages are of a sequence's own rows: a manager with a prefix attends them all")
        if manager.prefix.prefix is not None:
            raise ValueError("the manager's prefix has a prefix of its own")
    new = None
    if (key_new is None) != (value_new is None):
        raise ValueError("key_new and value_new come together")
    if key_new is not None:
        new = layer.check_append(key_new, value_new, lengths)
        if key_new.shape[2] != q_len:
            raise ValueError(f"{key_new.shape[2]} new tokens and {q_len} query tokens")
    if pages is not None:
        if pages.dim() != 4 or tuple(pages.shape[:3]) != (B, manager.n_kv, q_len) or not 1 <= pages.shape[3] <= MAX_PAGES:
            raise ValueError(f"pages must be [{B}, {manager.n_kv}, {q_len}, 1 .. {MAX_PAGES}], got {tuple(pages.shape)}")
        if pages.dtype != torch.int32:
            raise TypeError(f"pages must be int32, got {pages.dtype}")
        if pages.device != manager.device:
            raise ValueError(f"pages are on {pages.device}, the cache on {manager.device}")
        pages = pages.contiguous()
    return _attend(manager, layer_idx, layer, query, new, scaling, lengths, pages)


@_here
def _attend(manager, layer_idx: int, layer, query: torch.Tensor, new, scaling: float, lengths, pages) -> torch.Tensor:
    """``int4_attention`` of checked arguments; ``new``: those of the append."""
    B, n_q, q_len, D = query.shape
    counts = _query_lengths(manager, q_len, lengths)
    if new is not None:
        layer._append(*new)
        manager._note(layer_idx)
    if pages is None and manager.top_pages:
        pages = _select(manager, layer, query, manager.top_pages, counts)
    out = torch.empty(B, n_q, q_len, D, dtype=query.dtype, device=manager.device)
    a = _args(manager, query, counts, scaling)
    a.out = out.data_ptr()
    group, cus = n_q // manager.n_kv, _cu_count(manager.device)
    tokens, tiles = layer.lengths, -(-group * q_len // 16)
    if pages is not None:
        a.pages, a.n_pages = pages.data_ptr(), pages.shape[3]
        # (the list is cut as a whole: a sequence of fewer pages leaves the later splits idle)
        tokens, tiles = ((a.n_pages + 1) * layer.page_size,), -(-group // 16) * q_len * B
    shared = None if manager._prefix is None else _shared_plan(manager, layer_idx, q_len, query.dtype, lengths, cus)
    if pages is None and _many_rows(group, q_len, manager.n_kv, D, manager.group_size, query.dtype, tokens):
        a.prefix_splits, _ = plan_splits(tokens, manager.n_kv * -(-group * q_len // 128), cus,
                                         many_rows_per_cu(D, manager.group_size), MANY_ROWS_OVERHEAD)
        a.splits = 1
        if shared:
            a.prefix_splits = min(a.prefix_splits, MAX_SPLITS // 2)
    elif shared:
        a.splits, a.split_tokens = shared[1]
    else:
        a.splits, a.split_tokens = plan_splits(tokens, manager.n_kv * tiles, cus,
                                               workgroups_per_cu(D, manager.group_size))
    parts = a.splits + a.prefix_splits + (shared[0][0] if shared else 0)
    if parts > 1:
        nbytes = 4 * B * n_q * q_len * parts * (D + 2)  # lf_int4_workspace_bytes
        ws = _workspace(manager, nbytes)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    stream = _native.current_stream_ptr(manager.device)
    if shared:
        prefix = manager.prefix.layers[layer_idx].layer_struct()
        st = _native.load().lf_int4_shared_attention(layer.layer_struct(), prefix, a, *shared[0], stream)
        _native.check(st, "lf_int4_shared_attention")
        return out
    st = _native.load().lf_int4_attention(layer.layer_struct(), a, stream)
    _native.check(st, "lf_int4_attention")
    return out


# From this much work on (products of a row's channel and a token's, over all prefixes) the many-row kernel takes shared
# prefixes, per group size (bf16, head_dim up to 128, 64 rows): below, the general kernel's launch, which holds the sequences' own
# rows too, is faster although it unpacks a record for every 16 rows.  us a call with 200 own tokens, general / many-row: 28 /
# 4 heads of 128, a prefix of 32K, groups of 64, 224 rows 53 / 59, 448 86 / 81, 896 155 / 121; groups of 128, 896 rows 134 /
# 141, 1 792 243 / 233; 32 / 8 heads, groups of 32, 64 rows 44 / 54, 128 73 / 60, 512 216 / 155; 14 / 2 heads of 64, 896 rows,
# groups of 64 and 32, 49 / 55 and 58 / 55, 1 792, groups of 64, 104 / 84; prefixes of 4K and 8K, 896 rows, groups of 64, 33 / 52 and
# 53 / 63.
SHARED_MANY_ROWS = {32: 3e9, 64: 6e9, 128: 3e10}
SHARED_LEAST_ROWS = 64


# What an item of a shared prefix's launch costs beside its units, in units of a compute unit's time, and how long a unit takes
# an item that has its compute unit to itself (two of them fill it).  Fitted to 16 sequences behind 32 768 tokens (28 / 4 heads
# of 128) in items of 768 to 4 096 tokens, 30 to 41 us a call: 11 us, and half a microsecond of these.  (Over 21 calls of 16 to
# 224 rows and head_dim 64 to 256 its choice is 2 % off the best size's time; the longest split that fills every place was 9 % off.)
SHARED_ITEM, SHARED_ALONE = 4.0, 1.75


@functools.lru_cache(maxsize=512)
def _shared_split(prefixes: tuple, rows: int, batch: int, longest: int, own: int, own_rows: int, cus: int, per_cu: int,
                  item: float) -> int:
    """Units that a split takes of shared prefixes (their units, ``rows`` workgroups a split) and of the rows of the ``batch``
    sequences behind them (``own`` units in all, ``own_rows`` workgroups a split), which run side by side, ``per_cu`` to a
    compute unit, ``item`` units an item: the size of least estimated time."""
    total, longest = sum(prefixes) * rows + own * own_rows, max(max(prefixes), longest)
    least = -(-longest // (MAX_SPLITS // 2))

    def cost(size):
        n = rows * sum(-(-u // size) for u in prefixes) + own_rows * (batch + own // size)
        whole = rows * sum(u // size for u in prefixes) + own_rows * batch * (own // batch // size)
        # turns of a compute unit; the last splits, which are shorter, find a place between (the dispatch is not even enough for
        # a whole number of turns)
        turns = (whole + 1) / cus
        load = (math.ceil(turns) if turns <= per_cu else turns + 0.5) * size + (total - whole * size) / cus
        return max(load, SHARED_ALONE * min(size, longest)) + item * n / cus

    sizes = {longest}
    for k in (1, 2, 3, 4, 6, 8, 12):
        share = -(-total // (cus * k))
        sizes |= {min(max(size, least, 1), longest) for size in range(share - 1, share + 3)}
    return min(sorted(sizes, reverse=True), key=cost)


def _shared_plan(manager, layer_idx: int, q_len: int, dtype, lengths, cus: int):
    """``((splits, split_tokens, many_rows)`` of the manager's prefix, ``(splits, split_tokens)`` of the own rows), or None
    where there is no prefix."""
    prefix = manager.prefix
    tokens = prefix.layers[layer_idx].lengths
    if not max(tokens) and not torch.cuda.is_current_stream_capturing():
        return None
    D, group, n_kv = manager.head_dim, manager.group_size, manager.n_kv
    each = manager.n_q // n_kv * q_len
    rows = each * (manager.batch_size // prefix.batch_size)
    own = manager.layers[layer_idx].lengths
    # every query sees all of its prefix
    behind = min(own) >= q_len or lengths is not None and all(n >= m for n, m in zip(own, lengths))
    if (rows >= SHARED_LEAST_ROWS and dtype == torch.bfloat16 and D <= 128 and behind
            and sum(tokens) * rows * n_kv * D >= SHARED_MANY_ROWS[group]):
        splits, size = plan_splits(tokens, n_kv * -(-rows // 128), cus, many_rows_per_cu(D, group), MANY_ROWS_OVERHEAD)
        splits = min(splits, MAX_SPLITS // 2)
        # (a row's parts are at most MAX_SPLITS + 1; one long sequence among short ones asks for many)
        return (splits, size, 1), plan_splits(own, n_kv * -(-each // 16), cus, workgroups_per_cu(D, group), most=MAX_SPLITS + 1 - splits)
    size = _shared_split(tuple([(n + SPLIT_UNIT - 1) // SPLIT_UNIT or 1 for n in tokens]), n_kv * -(-rows // 16),
                         len(own), max(own) // SPLIT_UNIT + 1, sum(own) // SPLIT_UNIT, n_kv * -(-each // 16),
                         cus, workgroups_per_cu(D, group), SHARED_ITEM * max(D, 128) / 128) * SPLIT_UNIT
    return (-(-max(max(tokens), 1) // size), size, 0), (-(-max(max(own), 1) // size), size)


@_here
def _select(manager, layer, query: torch.Tensor, top_pages: int, counts) -> torch.Tensor:
    q_len = int(query.shape[2])
    lib = _native.load()
    struct = layer.layer_struct()
    pages = torch.empty(manager.batch_size, manager.n_kv, q_len, top_pages, dtype=torch.int32, device=manager.device)
    a = _args(manager, query, counts, 1.0)
    a.pages, a.n_pages = pages.data_ptr(), top_pages
    a.workspace_bytes = lib.lf_int4_select_workspace_bytes(struct, q_len)
    ws = _workspace(manager, a.workspace_bytes)
    a.workspace = ws.data_ptr()
    st = lib.lf_int4_select(struct, a, _native.current_stream_ptr(manager.device))
    _native.check(st, "lf_int4_select")
    return pages


def select_pages(manager: Int4KVManager, layer_idx: int, query: torch.Tensor, top_pages: int, *,
                 lengths=None) -> torch.Tensor:
    """The pages that each query token's kv head attends: int32 ``[B, n_kv, q_len, top_pages]``, ascending, -1
    behind the last one.

    ``query [B, n_q, q_len, D]``: the sequence's last ``q_len`` tokens, already committed.  Candidates
    are the pages before the query's own one (which ``int4_attention`` attends by itself); a page's
    score is the largest, over the kv head's query heads, of ``sum_c max(q_c lo_c, q_c hi_c)`` with the
    page's ``page_bounds``, formed in float64 (exact but for elements that span very much: ``lf_int4_select``).  Equal
    scores: the lower page first, NaN ones last.
    """
    query = _check_query(manager, query, True)
    top_pages = int(top_pages)
    if not 1 <= top_pages <= MAX_PAGES:
        raise ValueError(f"top_pages must lie in 1 .. {MAX_PAGES}, got {top_pages}")
    counts = _query_lengths(manager, query.shape[2], lengths)
    return _select(manager, manager.layers[layer_idx], query, top_pages, counts)
