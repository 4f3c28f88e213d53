"""Which calls of a model's layers the prompt attention takes, by the masks that the installed transformers makes (no GPU)."""
from types import SimpleNamespace

import pytest
import torch

from logitfill_amd.qwen2 import _PromptKernels, _is_causal

T = 6


def mask_of(kind, positions=None, padding=None, batch=2, dtype=torch.float32):
    from transformers import Qwen2Config
    from transformers.masking_utils import create_causal_mask

    cfg = Qwen2Config(vocab_size=8, hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=1,
                      num_key_value_heads=1, attn_implementation=kind)
    positions = torch.arange(T)[None].expand(batch, T) if positions is None else positions
    return create_causal_mask(config=cfg, inputs_embeds=torch.zeros(batch, T, 64, dtype=dtype), attention_mask=padding,
                              past_key_values=None, position_ids=positions)


def kernels():
    k = _PromptKernels.__new__(_PromptKernels)
    k.plan, k.masks = None, None
    return k


def attention(kind, **changes):
    config = SimpleNamespace(_attn_implementation=kind, is_causal=changes.pop("config_causal", True))
    return SimpleNamespace(config=config, **{"is_causal": True, "sliding_window": None, **changes})


def padded(*hidden):
    mask = torch.ones(2, T, dtype=torch.long)
    for b, t in hidden:
        mask[b, t] = 0
    return mask


@pytest.mark.parametrize("kind", ["eager", "sdpa"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("call,serves", [
    ({}, True), ({"padding": padded()}, True), ({"padding": padded((0, 0), (0, 1))}, False), ({"padding": padded((1, 5))}, False),
    ({"positions": torch.tensor([[0, 1, 2, 0, 1, 2]] * 2)}, False),
    ({"positions": torch.tensor([[0, 1, 2, 3, 4, 5], [0, 1, 0, 1, 2, 3]])}, False),
    ({"positions": torch.tensor([[7, 8, 9, 10, 11, 12]] * 2)}, True), ({"batch": 1}, True),
])
def test_masks_that_the_model_makes(kind, dtype, call, serves):
    mask = mask_of(kind, dtype=dtype, **call)
    assert kernels().serves(attention(kind), mask, T) is serves


@pytest.mark.parametrize("kind,changes", [
    ("sdpa", {"sliding_window": 4}), ("eager", {"sliding_window": 4}), ("sdpa", {"is_causal": False}), ("eager", {"is_causal": False}),
    ("sdpa", {"config_causal": False}), ("flash_attention_2", {}), ("flex_attention", {}), (None, {}),
])
def test_layers_that_keep_their_own_attention(kind, changes):
    mask = mask_of("eager") if kind == "eager" else None
    assert not kernels().serves(attention(kind, **changes), mask, T)


def test_calls_that_say_they_are_not_causal():
    assert not kernels().serves(attention("sdpa"), None, T, is_causal=False)
    assert kernels().serves(attention("sdpa"), None, T, is_causal=True)


def test_packed_prompts_come_without_a_mask():
    k = kernels()
    assert not k.serves(attention("eager"), None, T)  # (an eager layer without a mask sees everything)
    k.plan = object()
    assert k.serves(attention("eager"), None, T) and k.serves(attention("flash_attention_2"), None, T)


def test_masks_of_the_caller_s():
    seen = torch.ones(T, T, dtype=torch.bool).tril()
    causal = torch.where(seen, 0.0, -torch.inf)[None, None]
    assert _is_causal(causal, T) and _is_causal(seen[None, None], T) and _is_causal(causal.expand(3, 2, T, T), T)
    least = torch.finfo(torch.float32).min
    assert _is_causal(causal.clamp(min=least), T)
    slopes = causal - torch.arange(T)[None, None, :, None] * 0.1
    soft = torch.where(seen, 0.0, -1e4)[None, None]
    some = causal.expand(3, 1, T, T).clone()
    some[2, 0, 4, 1] = least
    for other in (slopes, soft, some, torch.zeros(1, 1, T, T), causal[..., :-1], causal[:, :, 1:], causal[0], causal.long(), None,
                  torch.where(seen, 0.0, torch.nan)[None, None], torch.full((1, 1, T, T), -torch.inf)):
        assert not _is_causal(other, T)


def test_a_pass_looks_at_a_mask_once(monkeypatch):
    from logitfill_amd import qwen2

    looked = []
    monkeypatch.setattr(qwen2, "_is_causal", lambda mask, tokens: looked.append(mask) or bool(mask.any()))
    k, layer = kernels(), attention("eager")
    yes, no = torch.ones(1, 1, T, T), torch.zeros(1, 1, T, T)
    k._begin(None, ())
    assert [k.serves(layer, m, T) for m in (yes, yes, no, yes, no)] == [True, True, False, True, False] and len(looked) == 2
    k._end(None, (), None)
    yes.zero_()  # (nothing is known of it outside the pass)
    k._begin(None, ())
    assert not k.serves(layer, yes, T) and len(looked) == 3
    k._end(None, (), None)
    assert not k.serves(layer, yes, T) and not k.serves(layer, yes, T) and len(looked) == 5
