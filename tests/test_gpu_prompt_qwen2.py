"""A prompt's way through a small Qwen2 model: rotated and attended by this package, packed prompts, and samples of one prompt
that share it as a prefix, against the model's own attention and against sequences on their own."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager
from logitfill_amd.qwen2 import PackedDecoder, attach_packed, detach_packed
from tests.test_gpu_qwen2 import _manager, _model

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _ids(n, seed, gpu):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).to(gpu)


def _int4(gpu, batch=1, **kw):
    return Int4KVManager(2, 4, 2, 128, 64, 32, gpu, batch_size=batch, **kw)


@pytest.mark.parametrize("packed_pages", [False, True])
@pytest.mark.parametrize("hf_cache", [False, True])
def test_prefill_and_steps_match_the_model_s_own_attention(gpu, hf_cache, packed_pages):
    model = _model(gpu)
    prompt, forced = _ids(300, 1, gpu)[None], _ids(6, 2, gpu)
    runs = []
    for kernels in (False, True):
        dec = PackedDecoder(model, _manager(gpu) if packed_pages else _int4(gpu), hf_cache=hf_cache, prompt_kernels=kernels)
        runs.append(torch.cat([dec.prefill(prompt)] + [dec.step(t) for t in forced]))
        detach_packed(model)
    # float32 all through; positions up to 306 times 2^-24 of an angle, which the model forms in float32
    assert _rel(runs[1][0], runs[0][0]) < 1e-4
    # (a code decided at the border of two moves a row's value by a step of 15, or of 3)
    assert _rel(runs[1], runs[0]) < 2e-2


def test_packed_prompts_are_each_one_s_own(gpu):
    """Prompts of unlike lengths in one pass, then a step for all: logits and cached rows as each by itself."""
    model = _model(gpu)
    prompts, tokens = [_ids(n, n, gpu) for n in (37, 300, 1, 64)], _ids(4, 9, gpu)
    mgr = _int4(gpu, 4)
    dec = PackedDecoder(model, mgr, prompt_kernels=True)
    out = [dec.prefill(prompts), dec.step(tokens), dec.step(tokens + 1)]
    detach_packed(model)
    assert mgr.layers[0].lengths == mgr.layers[1].lengths == [39, 302, 3, 66]
    for b, prompt in enumerate(prompts):
        one = _int4(gpu)
        alone = PackedDecoder(model, one, prompt_kernels=True)
        want = [alone.prefill(prompt[None]), alone.step(tokens[b]), alone.step(tokens[b] + 1)]
        detach_packed(model)
        assert _rel(out[0][b], want[0][0]) < 1e-4, b
        assert all(_rel(out[i][b], want[i][0]) < 2e-2 for i in (1, 2)), b
        k, v = mgr.layers[0].read(0, len(prompt))
        k1, v1 = one.layers[0].read(0, len(prompt))
        # (the first layer's rows are projections of the embeddings: a few codes lie at a border)
        assert float((k[b] - k1[0]).abs().gt(1e-5).float().mean()) < 1e-2 and _rel(v[b], v1[0]) < 2e-2


def test_packed_prompts_into_packed_pages(gpu):
    from logitfill_amd import synth
    from logitfill_amd.packed import PackedKVManager

    model = _model(gpu)
    prompts, tokens = [_ids(n, n, gpu) for n in (150, 20)], _ids(2, 9, gpu)
    levels = [synth.sample_tier_levels(2, 128, 2.5, seed=s) for s in range(2)]
    mgr = PackedKVManager(levels, 4, 2, 128, 128, 128, 128, 2, gpu, batch_size=2)
    dec = PackedDecoder(model, mgr, prompt_kernels=True)
    out = [dec.prefill(prompts), dec.step(tokens)]
    detach_packed(model)
    assert mgr.layers[1].lengths() == [151, 21]
    for b, prompt in enumerate(prompts):
        alone = PackedDecoder(model, _manager(gpu), prompt_kernels=True)
        want = [alone.prefill(prompt[None]), alone.step(tokens[b])]
        detach_packed(model)
        assert _rel(out[0][b], want[0][0]) < 1e-4 and _rel(out[1][b], want[1][0]) < 2e-2


@pytest.mark.parametrize("kernels", [False, True])
def test_samples_of_one_prompt_share_it(gpu, kernels):
    """A prompt is prefilled once; its samples' steps are those of sequences that hold it by themselves."""
    model = _model(gpu)
    prompt, tokens = _ids(200, 3, gpu), _ids(15, 4, gpu).view(5, 3)
    prefix = _int4(gpu)
    first = PackedDecoder(model, prefix, prompt_kernels=kernels)
    start = first.prefill(prompt[None])
    detach_packed(model)
    mgr = _int4(gpu, 3, prefix=prefix)
    dec = PackedDecoder(model, mgr, prompt_kernels=kernels)
    got = [dec.step(t) for t in tokens[:2]]
    more = dec.prefill(tokens[:2].T.contiguous())  # the same again, two tokens at once
    got += [dec.step(t) for t in tokens[2:]]
    detach_packed(model)
    assert mgr.layers[0].lengths == [5] * 3 and prefix.layers[0].lengths == [200]
    for b in range(3):
        alone = PackedDecoder(model, _int4(gpu), prompt_kernels=kernels)
        assert _rel(alone.prefill(prompt[None]), start) < 1e-5
        want = [alone.step(t) for t in tokens[:, b]]
        detach_packed(model)
        for i in range(5):
            assert _rel(got[i][b], want[i][0]) < 2e-2, (b, i)
        assert _rel(more[b], want[1][0]) < 2e-2


def test_a_prefix_that_only_some_sequences_have(gpu):
    """The first pass behind prefixes of which the first is empty attends the others, too."""
    model = _model(gpu)
    prompt, tokens = _ids(50, 3, gpu), _ids(6, 4, gpu).view(2, 3)
    one, got = _int4(gpu), []
    first = PackedDecoder(model, one, prompt_kernels=True)
    first.prefill(prompt[None])
    want = [first.step(t) for t in tokens[1]]
    detach_packed(model)
    rows = [[t[:, :, :50].repeat(2, 1, 1, 1) for t in one.layers[i].read(0, 50)] for i in range(2)]
    for lengths in ([0, 50], [50, 0]):
        prefix = _int4(gpu, 2)
        for i in range(2):
            prefix.commit(i, *rows[i], lengths)
        dec = PackedDecoder(model, _int4(gpu, 2, prefix=prefix), prompt_kernels=True)
        got.append(dec.prefill(tokens if lengths[1] else tokens.flip(0)))
        detach_packed(model)
    # (rows quantised once more on their way into the prefix; the one without a prefix attends what its cache reads back, too)
    assert _rel(got[0][1], want[-1][0]) < 2e-2 and _rel(got[1].flip(0), got[0]) < 1e-4


def test_a_padded_batch_s_mask_is_the_model_s_own(gpu):
    """Of a model whose attention makes masks for padding only, a masked batch keeps its result."""
    model = _model(gpu)
    model.config._attn_implementation = "sdpa"
    ids = _ids(40, 6, gpu).view(2, 20)
    mask = torch.ones(2, 20, dtype=torch.long, device=gpu)
    mask[1, :7] = 0
    pos = (mask.cumsum(1) - 1).clamp(min=0)
    runs = []
    for kernels in (False, True):
        attach_packed(model, _int4(gpu, 2), prompt_kernels=kernels)
        with torch.no_grad():
            runs.append(model(input_ids=ids, attention_mask=mask, position_ids=pos, use_cache=False).logits[:, -1])
        detach_packed(model)
    assert _rel(runs[1], runs[0]) < 1e-4


def test_bfloat16_prompts(gpu):
    """The matrix-core kernels of 16-bit rows under the model: close to its own attention in the same type."""
    model = _model(gpu).bfloat16()
    prompt = _ids(500, 5, gpu)[None]
    runs = []
    for kernels in (False, True):
        dec = PackedDecoder(model, _int4(gpu), prompt_kernels=kernels)
        runs.append(dec.prefill(prompt))
        detach_packed(model)
    # two layers of a dozen roundings of 2^-9 each on either side
    assert _rel(runs[1], runs[0]) < 24 * 2 * 2.0 ** -9


def test_refused(gpu):
    model = _model(gpu)
    dec = PackedDecoder(model, _int4(gpu, 2))
    prompts = [_ids(5, 1, gpu), _ids(7, 2, gpu)]
    with pytest.raises(ValueError, match="prompt_kernels"):
        dec.prefill(prompts)
    dec = PackedDecoder(model, _int4(gpu, 2), prompt_kernels=True)
    for bad in (prompts[:1], [p[None] for p in prompts], [prompts[0], prompts[1][:0]]):
        with pytest.raises(ValueError):
            dec.prefill(bad)
    assert dec.kernels.plan is None
    dec.prefill(prompts)
    with pytest.raises(RuntimeError, match="gradient"):
        model(input_ids=prompts[0][None].expand(2, 5), position_ids=torch.arange(5, device=gpu)[None], use_cache=False)
    prefix = _int4(gpu)
    PackedDecoder(model, prefix, prompt_kernels=True).prefill(prompts[0][None])
    with pytest.raises(ValueError, match="shared prefix"):
        PackedDecoder(model, _int4(gpu, 2, prefix=prefix), prompt_kernels=True).prefill(prompts)
    detach_packed(model)
    model.model.rotary_emb.rope_type = "dynamic"
    with pytest.raises(ValueError, match="dynamic"):
        attach_packed(model, _int4(gpu), prompt_kernels=True)
    assert not hasattr(model.model.layers[0].self_attn, "_lf_original_forward")
