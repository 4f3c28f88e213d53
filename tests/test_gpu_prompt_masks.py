"""Calls of a model with ``prompt_kernels`` whose masks hide more than later tokens: the model's own result, whichever way its
attention is made; calls without such a mask run the prompt attention."""
import copy

import pytest
import torch

from logitfill_amd import qwen2
from logitfill_amd.packed import Int4KVManager
from logitfill_amd.qwen2 import PackedDecoder, attach_packed, detach_packed
from tests.test_gpu_qwen2 import _model

pytestmark = pytest.mark.gpu


@pytest.fixture
def calls(monkeypatch):
    made = []
    attend = qwen2.prompt_attention
    monkeypatch.setattr(qwen2, "prompt_attention", lambda *args: made.append(args[0].shape) or attend(*args))
    return made


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _logits(gpu, model, kernels, batch, **call):
    attach_packed(model, Int4KVManager(2, 4, 2, 128, 64, 32, gpu, batch_size=batch), prompt_kernels=kernels)
    with torch.no_grad():
        out = model(use_cache=False, **call).logits
    detach_packed(model)
    return out


def _batch(gpu, left):
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(6)).to(gpu)
    mask = torch.ones(2, 20, dtype=torch.long, device=gpu)
    mask[1, slice(0, 7) if left else slice(13, 20)] = 0
    return ids, mask, (mask.cumsum(1) - 1).clamp(min=0)


@pytest.mark.parametrize("kind", ["eager", "sdpa"])
@pytest.mark.parametrize("left", [True, False])
def test_a_padded_batch(gpu, calls, kind, left):
    model = _model(gpu)
    model.config._attn_implementation = kind
    ids, mask, pos = _batch(gpu, left)
    call = dict(input_ids=ids, attention_mask=mask, position_ids=pos)
    want, got = (_logits(gpu, model, kernels, 2, **call) for kernels in (False, True))
    real = mask.bool()
    # float32 all through: the rotation's angles, 2^-24 of up to 20
    assert _rel(got[real], want[real]) < 1e-4 and not calls


@pytest.mark.parametrize("kind", ["eager", "sdpa"])
def test_sequences_in_one_row(gpu, calls, kind):
    """Told apart by their positions alone: neither sees the other."""
    model = _model(gpu)
    model.config._attn_implementation = kind
    ids, _, _ = _batch(gpu, True)
    pos = torch.cat([torch.arange(12), torch.arange(8)])[None].to(gpu)
    want, got = (_logits(gpu, model, kernels, 1, input_ids=ids[:1], position_ids=pos) for kernels in (False, True))
    assert _rel(got, want) < 1e-4 and not calls
    alone = _logits(gpu, model, True, 1, input_ids=ids[:1, 12:], position_ids=pos[:, 12:])
    assert _rel(got[:, 12:], alone) < 1e-4 and len(calls) == 2


@pytest.mark.parametrize("kind", ["eager", "sdpa"])
@pytest.mark.parametrize("ones", [False, True])
def test_calls_without_padding(gpu, calls, kind, ones):
    model = _model(gpu)
    model.config._attn_implementation = kind
    ids, mask, _ = _batch(gpu, True)
    more = {"attention_mask": torch.ones_like(mask)} if ones else {}
    want, got = (_logits(gpu, model, kernels, 2, input_ids=ids, **more) for kernels in (False, True))
    assert _rel(got, want) < 1e-4 and len(calls) == 2


@pytest.mark.parametrize("kind", ["eager", "sdpa"])
@pytest.mark.parametrize("hf_cache", [False, True])
def test_a_decoder_s_prompt(gpu, calls, kind, hf_cache):
    model = _model(gpu)
    model.config._attn_implementation = kind
    dec = PackedDecoder(model, Int4KVManager(2, 4, 2, 128, 64, 32, gpu), hf_cache=hf_cache, prompt_kernels=True)
    dec.prefill(torch.arange(30, device=gpu)[None])
    assert len(calls) == 2
    dec.step(torch.tensor([3], device=gpu))
    assert len(calls) == 2
    detach_packed(model)
    assert not model.model._forward_pre_hooks and not model.model._forward_hooks


def test_attaching_anew_and_passes_that_fail(gpu, calls):
    """One pair of hooks however often the model is attached; a pass that raised leaves nothing known."""
    model = _model(gpu)
    mgr = Int4KVManager(2, 4, 2, 128, 64, 32, gpu)
    for _ in range(2):
        kernels = attach_packed(model, mgr, prompt_kernels=True)
    assert len(model.model._forward_pre_hooks) == len(model.model._forward_hooks) == 1
    with pytest.raises(NotImplementedError), torch.no_grad():
        model(input_ids=torch.arange(6, device=gpu).view(2, 3), use_cache=False)
    assert kernels.masks is None
    attach_packed(model, mgr)
    assert not model.model._forward_pre_hooks and not model.model._forward_hooks
    detach_packed(model)


def test_a_model_with_the_kernels_can_be_copied(gpu):
    model = _model(gpu)
    ids = torch.arange(9, device=gpu)[None]
    want = PackedDecoder(model, Int4KVManager(2, 4, 2, 128, 64, 32, gpu), prompt_kernels=True).prefill(ids)
    other = copy.deepcopy(model)
    detach_packed(model)
    got = PackedDecoder(other, Int4KVManager(2, 4, 2, 128, 64, 32, gpu), prompt_kernels=True).prefill(ids)
    assert torch.equal(got, want)
