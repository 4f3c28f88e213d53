"""Qwen2 decoder on the packed backend: the model-integration caller of the decode path.

The reference patches every ``Qwen2Attention.forward`` so that, with the ``packed`` backend,
a layer with history runs ``packed_attention`` over the packed cache and every layer then
commits its new Key/Value states (attention first, then commit: completed pages are
compressed after the attention that produced them), while a layer with no history (the
prefill) runs the model's own dense attention (``src/logitfill/models/qwen2_attention.py:
76-146,223-256``; adapter ``models/deepseek_qwen.py:123-146``).

``attach_packed(model, manager)`` does the same for the installed transformers (5.x
``Qwen2Attention.forward(hidden_states, position_embeddings, attention_mask,
past_key_values=None, **kwargs)``), with two differences: the packed output
``[B, n_q, q_len, D]`` is transposed to the ``[B, q_len, n_q, D]`` the projection expects (the
reference reshapes it directly, which is right only for ``q_len == 1``), and the model runs
without a transformers cache -- the packed cache holds the history, so callers pass explicit
``position_ids`` (``PackedDecoder`` does).  ``detach_packed`` restores the original forwards.

With an ``Int4KVManager`` the layers run ``int4_attention`` instead, which caches the new tokens
before it reads (of a manager with ``top_pages``, over the pages it selects; of a manager with a
``prefix``, behind its shared rows).

``prompt_kernels=True`` takes the prompt's own pass to this package, too: positions are turned into
queries and Keys by ``Rotary``, and a layer without history runs ``prompt_attention`` in place of the
model's dense attention -- of several prompts at once, packed one behind another
(``PackedDecoder.prefill`` of a list).
"""
from __future__ import annotations

import torch

from logitfill_amd import _native
from logitfill_amd.packed.int4 import Int4KVManager, int4_attention
from logitfill_amd.packed.prompt import PromptPlan, prompt_attention
from logitfill_amd.packed.reference import packed_attention, reference_attention
from logitfill_amd.packed.rotary import Rotary


def _dense_attention(attn, query, key, value, attention_mask, kwargs):
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    from transformers.models.qwen2.modeling_qwen2 import eager_attention_forward

    impl = ALL_ATTENTION_FUNCTIONS.get_interface(attn.config._attn_implementation, eager_attention_forward)
    out, _ = impl(attn, query, key, value, attention_mask, dropout=0.0, scaling=attn.scaling,
                  sliding_window=getattr(attn, "sliding_window", None), **kwargs)
    return out  # [B, q_len, n_q, D]


def _is_causal(mask, tokens: int) -> bool:
    """Whether an attention mask (additive, or truth values) is the causal one of ``tokens``, for every sequence (a host
    synchronisation; not in a capture)."""
    if not isinstance(mask, torch.Tensor) or mask.dim() != 4 or tuple(mask.shape[2:]) != (tokens, tokens):
        return False
    if mask.is_cuda and torch.cuda.is_current_stream_capturing():
        return False
    if mask.dtype == torch.bool:
        seen, hidden = mask, ~mask
    elif mask.is_floating_point():
        seen, hidden = mask == 0, mask <= torch.finfo(mask.dtype).min
    else:
        return False
    return bool(torch.where(torch.ones(tokens, tokens, dtype=torch.bool, device=mask.device).tril(), seen, hidden).all())


class _PromptKernels:
    """What the layers of a model with ``prompt_kernels`` share: its rotation, what is known of the masks of the pass that is
    under way, and, while packed prompts pass through, their plan and the places of their tokens in a padded batch."""

    def __init__(self, model, device):
        rope = model.model.rotary_emb
        kind = str(getattr(rope, "rope_type", "default"))
        if "dynamic" in kind or kind == "longrope":
            raise ValueError(f"prompt_kernels takes frequencies that hang on no length; the model's are {kind!r}")
        head_dim = model.model.layers[0].self_attn.head_dim
        if head_dim not in (64, 128, 256):
            raise ValueError(f"prompt_kernels takes heads of 64, 128 or 256 channels, the model has {head_dim}")
        freq = rope.inv_freq.tolist()
        self.rotary = Rotary(head_dim, rotary_dim=2 * len(freq), inv_freq=freq,
                             attention_factor=float(getattr(rope, "attention_scaling", 1.0)), device=device)
        self.windows = any(getattr(layer.self_attn, "sliding_window", None) for layer in model.model.layers)
        self.plan: PromptPlan | None = None
        self.places: torch.Tensor | None = None
        self.masks: list | None = None  # of the pass under way: (mask, whether it is the causal one)

    def watch(self, model) -> None:
        """Learn of the model's passes, until ``_drop_kernels``."""
        # (functions, not methods: a copy of the model does not copy what is behind them)
        hooks = (model.model.register_forward_pre_hook(lambda *args: self._begin(*args)),
                 model.model.register_forward_hook(lambda *args: self._end(*args), always_call=True))
        model._lf_drop_kernels = lambda: [hook.remove() for hook in hooks]

    def _begin(self, module, args) -> None:
        self.masks = []

    def _end(self, module, args, output) -> None:
        self.masks = None

    def pack(self, lengths) -> None:
        """Prompts of ``lengths`` pass through next, packed."""
        if self.windows:
            raise ValueError("packed prompts take a model without sliding windows")
        self.plan = PromptPlan(lengths, device=self.rotary.device)
        longest, at, rows = max(lengths), 0, []
        for n in lengths:
            rows += [min(at + t, at + n - 1) for t in range(longest)]  # (what stands behind its last token is not read)
            at += n
        self.places = _native.upload(rows, torch.int64, self.rotary.device)

    def serves(self, attn, attention_mask, tokens: int, is_causal=None) -> bool:
        """Whether a layer without history is ``prompt_attention``'s: where the model's own attention of ``tokens`` would be
        causal over every whole sequence.  Packed prompts are (they come without a mask); so is sdpa without a mask (it gets
        one for padding and for sequences in one row), and an eager model, which gets one for every call, where that is the causal
        one.  Other implementations tell padding and packed rows in ways of their own."""
        if getattr(attn, "sliding_window", None):
            return False
        if self.plan is not None:
            return True
        if is_causal is False or not getattr(attn, "is_causal", True) or not getattr(attn.config, "is_causal", True):
            return False
        kind = getattr(attn.config, "_attn_implementation", None)
        if kind == "sdpa":
            return attention_mask is None
        return kind == "eager" and self._is_causal(attention_mask, tokens)

    def _is_causal(self, mask, tokens: int) -> bool:
        """``_is_causal``, looked up once a pass (its layers get one mask)."""
        for seen, answer in self.masks or ():
            if seen is mask:
                return answer
        answer = _is_causal(mask, tokens)
        if self.masks is not None:
            self.masks.append((mask, answer))
        return answer

    def unpack(self) -> None:
        self.plan = self.places = None

    def rotate(self, query, key, position_ids):
        return self.rotary.rotate(query, key, position_ids)

    def commit(self, manager, layer_idx: int, key, value) -> None:
        """The prompts' rows into the cache, each sequence's its own."""
        if self.plan is None:
            manager.commit(layer_idx, key, value)
            return
        shape = (key.shape[1], self.plan.batch, -1, key.shape[3])
        key, value = (t[0].index_select(1, self.places).view(shape).transpose(0, 1) for t in (key, value))
        manager.commit(layer_idx, key, value, self.plan.lengths)


def _history(manager, layer_idx: int) -> int:
    """Tokens in front of a call's own: of the longest sequence, its prefix's among them."""
    lengths = getattr(manager.layers[layer_idx], "lengths", None)
    if lengths is None:  # (a cache of one sequence)
        return manager.layer_length(layer_idx)
    own = max(lengths() if callable(lengths) else lengths)
    return own if getattr(manager, "prefix", None) is None else own + max(manager.prefix_lengths(layer_idx))


def _make_forward(attn, manager, attention_fn, kernels=None):
    from transformers.models.qwen2.modeling_qwen2 import apply_rotary_pos_emb

    layer_idx = attn.layer_idx

    def forward(hidden_states, position_embeddings, attention_mask=None, past_key_values=None, **kwargs):
        input_shape = hidden_states.shape[:-1]
        hidden_shape = (*input_shape, -1, attn.head_dim)
        query = attn.q_proj(hidden_states).view(hidden_shape).transpose(1, 2)
        key = attn.k_proj(hidden_states).view(hidden_shape).transpose(1, 2)
        value = attn.v_proj(hidden_states).view(hidden_shape).transpose(1, 2)
        if kernels is not None and kwargs.get("position_ids") is not None:
            query, key = kernels.rotate(query, key, kwargs["position_ids"])
        else:
            cos, sin = position_embeddings
            query, key = apply_rotary_pos_emb(query, key, cos, sin)
        past = _history(manager, layer_idx)
        if past == 0 and kernels is not None and kernels.serves(attn, attention_mask, query.shape[2], kwargs.get("is_causal")):
            out = prompt_attention(query, key, value, attn.scaling, kernels.plan).transpose(1, 2)
            kernels.commit(manager, layer_idx, key, value)
        elif past == 0:
            out = _dense_attention(attn, query, key, value, attention_mask, kwargs)
            manager.commit(layer_idx, key, value)
        elif getattr(manager, "commits_new_tokens", False):
            out = attention_fn(manager, layer_idx, query, key, value, attn.scaling).transpose(1, 2)
        elif attention_fn is packed_attention:
            # attention then commit, the commit folded into the decode launch where it can be
            out = packed_attention(manager, layer_idx, query, key, value, attn.scaling, commit=True).transpose(1, 2)
        else:
            out = attention_fn(manager, layer_idx, query, key, value, attn.scaling).transpose(1, 2)
            manager.commit(layer_idx, key, value)
        if past_key_values is not None and hasattr(past_key_values, "note_layer"):
            past_key_values.note_layer(layer_idx, manager.seq_len)  # LogitFillCache (qwen2_attention.py:254-255)
        out = out.reshape(*input_shape, -1).contiguous()
        return attn.o_proj(out), None

    return forward


def attach_packed(model, manager, attention_fn=packed_attention, *, prompt_kernels: bool = False):
    """Route every decoder layer's attention through ``manager`` (a ``PackedKVManager`` whose
    layers match the model's).  ``attention_fn`` is ``packed_attention`` (the HIP path) or
    ``reference_attention`` (dense dequantise-then-attend), same signature.  An ``Int4KVManager``
    takes ``int4_attention`` in place of the default; any other function given for it commits the new
    tokens itself (``reference_attention``, which reads packed pages, does not: ``ValueError``).

    ``prompt_kernels``: queries and Keys are rotated by ``Rotary`` with the model's own frequencies (in float64 angles), and
    layers without history run ``prompt_attention`` where the model's own attention (eager or sdpa) would be causal over every
    whole sequence: those of a sliding window keep the model's, and so do calls whose mask hides more (padding, sequences in one
    row, a mask of the caller's; an eager model's mask is looked at once a pass, which waits for the device).  These give no
    gradients: call the model under ``torch.no_grad()``."""
    if isinstance(manager, Int4KVManager):
        if attention_fn is reference_attention:
            raise ValueError("reference_attention reads packed pages; an Int4KVManager takes int4_attention")
        if attention_fn is packed_attention:
            attention_fn = int4_attention
    cfg = model.config
    n_kv = int(cfg.num_key_value_heads)
    layers = model.model.layers
    if len(manager.layers) != len(layers):
        raise ValueError(f"manager has {len(manager.layers)} layers, the model {len(layers)}")
    for layer in layers:
        if manager.n_kv != n_kv or manager.head_dim != layer.self_attn.head_dim:
            raise ValueError("manager shape does not match the model's attention")
    kernels = _PromptKernels(model, manager.device) if prompt_kernels else None
    _drop_kernels(model)
    if kernels is not None:
        kernels.watch(model)
    for layer in layers:
        attn = layer.self_attn
        if not hasattr(attn, "_lf_original_forward"):
            attn._lf_original_forward = attn.forward
        attn.forward = _make_forward(attn, manager, attention_fn, kernels)
    return kernels


def _drop_kernels(model) -> None:
    model.__dict__.pop("_lf_drop_kernels", lambda: None)()


def detach_packed(model) -> None:
    _drop_kernels(model)
    for layer in model.model.layers:
        attn = layer.self_attn
        if hasattr(attn, "_lf_original_forward"):
            attn.forward = attn._lf_original_forward
            del attn._lf_original_forward


class PackedDecoder:
    """Prefill + token-by-token decode of a ``Qwen2ForCausalLM`` over a packed cache (batch 1, as
    the reference, or as many sequences as the manager holds).  ``step`` returns the logits of the
    last position.

    ``hf_cache=True`` passes a ``LogitFillCache`` as ``past_key_values`` (the reference adapter's
    ``make_cache``, ``deepseek_qwen.py:141-146``), so the model derives positions and mask sizes
    from the packed length; otherwise the decoder passes the positions itself.

    ``defer_flush``: None (default) keeps the manager's own setting; True or False sets it on
    the manager.  A deferring manager leaves every layer's completed page for one
    ``flush_pending`` launch after each forward pass (``step`` calls it) instead of one launch
    per layer; results are the same either way.

    ``prompt_kernels``: see ``attach_packed``; ``prefill`` then takes a list of prompts, too, one for each of the
    manager's sequences.  A manager with a ``prefix`` continues it: positions start behind the prefix's tokens."""

    def __init__(self, model, manager, attention_fn=packed_attention, *, hf_cache: bool = False,
                 defer_flush: bool | None = None, prompt_kernels: bool = False):
        self.model, self.manager = model, manager
        if defer_flush is not None and hasattr(manager, "defer_flush"):
            manager.defer_flush = bool(defer_flush)
        self.kernels = attach_packed(model, manager, attention_fn, prompt_kernels=prompt_kernels)
        self.cache = None
        if hf_cache:
            from logitfill_amd.packed.cache import LogitFillCache

            self.cache = LogitFillCache(manager)
        self.pos = 0

    def _flush(self) -> None:
        flush = getattr(self.manager, "flush_pending", None)  # managers without deferral have none
        if flush is not None:
            flush()

    def _prefix_lengths(self) -> list:
        """Tokens of a shared prefix in front of every sequence."""
        if getattr(self.manager, "prefix", None) is not None:
            return self.manager.prefix_lengths(0)
        return [0] * getattr(self.manager, "batch_size", 1)

    def _lengths(self) -> list:
        """Every sequence's tokens, those of a shared prefix among them."""
        own = self.manager.layers[0].lengths
        return [p + n for p, n in zip(self._prefix_lengths(), own() if callable(own) else own)]

    def _forward(self, ids: torch.Tensor, start) -> torch.Tensor:
        """``start``: the position of the first token, or of every sequence's."""
        if isinstance(start, list):
            if len(set(start)) == 1:
                start = start[0]
            else:
                first = _native.upload(start, torch.int64, ids.device)
                pos = first[:, None] + torch.arange(ids.shape[-1], device=ids.device)
        if not isinstance(start, list):
            pos = torch.arange(start, start + ids.shape[-1], device=ids.device)[None]
        if self.cache is not None:
            # (the cache's length is sequence 0's: positions of unlike ones are passed, too)
            more = {"position_ids": pos} if isinstance(start, list) else {}
            out = self.model(input_ids=ids, past_key_values=self.cache, use_cache=True, **more)
        else:
            out = self.model(input_ids=ids, position_ids=pos, use_cache=False)
        self._flush()
        return out.logits[:, -1]

    def _prefill_packed(self, prompts) -> torch.Tensor:
        lengths = [int(p.shape[-1]) for p in prompts]
        if self.kernels is None:
            raise ValueError("a list of prompts takes prompt_kernels=True")
        if any(p.dim() != 1 for p in prompts) or min(lengths, default=0) < 1:
            raise ValueError("prompts are one-dimensional, of at least one token")
        if len(prompts) != self.manager.batch_size:
            raise ValueError(f"{len(prompts)} prompts for a manager of {self.manager.batch_size} sequences")
        if max(self._prefix_lengths()):
            raise ValueError("prompts behind a shared prefix are fed as one tensor [batch, tokens]")
        device = prompts[0].device
        last = torch.cumsum(torch.tensor(lengths), 0) - 1
        pos = torch.cat([torch.arange(n, device=device) for n in lengths])[None]
        self.kernels.pack(lengths)
        try:
            # (no mask is made of the packed positions: every layer attends by the plan)
            out = self.model(input_ids=torch.cat(list(prompts))[None], position_ids=pos, use_cache=False,
                             attention_mask={"full_attention": None}, logits_to_keep=last.to(device))
        finally:
            self.kernels.unpack()
        self._flush()
        self.pos = lengths[0]
        return out.logits[0]

    @torch.no_grad()
    def prefill(self, input_ids) -> torch.Tensor:
        """Logits of the last position ``[batch, vocab]`` of prompts ``[batch, T]``, or of a list of one-dimensional ones."""
        self.manager.reset()
        if isinstance(input_ids, (list, tuple)):
            return self._prefill_packed(input_ids)
        start = self._prefix_lengths()
        logits = self._forward(input_ids, start)
        self.pos = start[0] + int(input_ids.shape[-1])
        return logits

    @torch.no_grad()
    def step(self, token: torch.Tensor) -> torch.Tensor:
        """``token``: the next one, or one for each sequence of the manager."""
        batch = getattr(self.manager, "batch_size", 1)
        # (one sequence behind a prefix may begin with a step; a cache that tells no lengths counts here)
        own = batch == 1 and getattr(self.manager, "prefix", None) is None
        logits = self._forward(token.view(batch, 1), self.pos if own else self._lengths())
        self.pos += 1
        return logits
