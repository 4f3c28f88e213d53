"""Steps of a decoder whose sequences are not where its own last call left them: behind a prefix, or cut back one by one."""
import pytest
import torch

from logitfill_amd import qwen2, synth
from logitfill_amd.packed import Int4KVManager, PackedKVManager
from logitfill_amd.qwen2 import PackedDecoder, detach_packed
from tests.test_gpu_qwen2 import _model

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _ids(n, seed, gpu):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).to(gpu)


def _int4(gpu, batch=1, **kw):
    return Int4KVManager(2, 4, 2, 128, 64, 32, gpu, batch_size=batch, **kw)


@pytest.mark.parametrize("hf_cache", [False, True])
@pytest.mark.parametrize("kernels", [False, True])
def test_one_sequence_behind_a_prefix_begins_with_a_step(gpu, kernels, hf_cache):
    """Its positions are those behind the prefix's tokens; after the prefix was cut back, too."""
    model = _model(gpu)
    prompt, tokens = _ids(150, 3, gpu), _ids(4, 4, gpu)
    prefix = _int4(gpu)
    PackedDecoder(model, prefix, prompt_kernels=kernels).prefill(prompt[None])
    mgr = _int4(gpu, prefix=prefix)
    dec = PackedDecoder(model, mgr, hf_cache=hf_cache, prompt_kernels=kernels)
    got = [dec.step(t) for t in tokens]
    prefix.truncate(100)
    mgr.reset()
    short = [dec.step(t) for t in tokens]
    detach_packed(model)
    for n, out in ((150, got), (100, short)):
        alone = PackedDecoder(model, _int4(gpu), prompt_kernels=kernels)
        alone.prefill(prompt[None, :n])
        # (a code decided at the border of two moves a row's value by a step of 15)
        for i, t in enumerate(tokens):
            assert _rel(out[i], alone.step(t)) < 2e-2, (n, i)
        detach_packed(model)


def _pages(gpu, batch=1):
    levels = [synth.sample_tier_levels(2, 128, 2.5, seed=s) for s in range(2)]
    return PackedKVManager(levels, 4, 2, 128, 128, 128, 128, 2, gpu, batch_size=batch)


@pytest.mark.parametrize("kernels", [False, True])
def test_a_sequence_that_was_cut_to_nothing(gpu, kernels, monkeypatch):
    """The first sequence begins anew, the others go on behind their rows.  All attend what the cache reads back (a row of 4 bits
    is off by up to a fifteenth of its range), so the first one's counterpart does from its first token on."""
    model = _model(gpu)
    prompts, tokens = _ids(90, 3, gpu).view(3, 30), _ids(6, 4, gpu).view(2, 3)
    mgr = _int4(gpu, 3)
    dec = PackedDecoder(model, mgr, prompt_kernels=kernels)
    dec.prefill(prompts)
    mgr.truncate([0, 30, 17])
    got = [dec.step(t) for t in tokens]
    detach_packed(model)
    assert mgr.layers[0].lengths == mgr.layers[1].lengths == [2, 32, 19]
    for b, n in enumerate((0, 30, 17)):
        with monkeypatch.context() as patch:
            alone = PackedDecoder(model, _int4(gpu), prompt_kernels=kernels)
            if n:
                alone.prefill(prompts[b : b + 1, :n])
            else:
                patch.setattr(qwen2, "_history", lambda *args: 1)
            for i in range(2):
                assert _rel(got[i][b], alone.step(tokens[i, b])[0]) < 2e-2, (b, i)
        detach_packed(model)


@pytest.mark.parametrize("kernels", [False, True])
def test_rows_of_some_sequences_only(gpu, kernels):
    """Packed pages that were filled for one sequence of two."""
    model = _model(gpu)
    prompt, tokens = _ids(150, 3, gpu), _ids(4, 4, gpu).view(2, 2)
    first = _int4(gpu)
    PackedDecoder(model, first, prompt_kernels=kernels).prefill(prompt[None])
    rows = [[t[:, :, :150] for t in first.layers[i].read(0, 150)] for i in range(2)]
    mgr, one = _pages(gpu, 2), _pages(gpu)
    for i, (k, v) in enumerate(rows):
        mgr.commit(i, k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1), [0, 150])
        one.commit(i, k, v)
    dec = PackedDecoder(model, mgr, prompt_kernels=kernels)
    got = [dec.step(t) for t in tokens]
    detach_packed(model)
    assert mgr.layers[1].lengths() == [2, 152]
    for b, cache in enumerate((_pages(gpu), one)):
        alone = PackedDecoder(model, cache, prompt_kernels=kernels)
        alone.pos = 150 * b
        for i in range(2):
            assert _rel(got[i][b], alone.step(tokens[i, b])[0]) < 2e-2, (b, i)
        detach_packed(model)


@pytest.mark.parametrize("kind", ["eager", "sdpa"])
@pytest.mark.parametrize("hf_cache", [False, True])
def test_prefixes_of_unlike_lengths(gpu, kind, hf_cache):
    """Two sequences behind each of two prefixes: a pass of three tokens, then steps, as sequences on their own."""
    model = _model(gpu)
    model.config._attn_implementation = kind
    prompts, tokens = [_ids(n, n, gpu) for n in (60, 35)], _ids(20, 4, gpu).view(4, 5)
    prefix = _int4(gpu, 2)
    PackedDecoder(model, prefix, prompt_kernels=True).prefill(prompts)
    mgr = _int4(gpu, 4, prefix=prefix)
    dec = PackedDecoder(model, mgr, hf_cache=hf_cache, prompt_kernels=True)
    got = [dec.prefill(tokens[:, :3])] + [dec.step(tokens[:, i]) for i in (3, 4)]
    detach_packed(model)
    assert mgr.prefix_lengths(1) == [60, 60, 35, 35] and mgr.layers[1].lengths == [5] * 4
    for b in range(4):
        alone = PackedDecoder(model, _int4(gpu), prompt_kernels=True)
        alone.prefill(prompts[b // 2][None])
        want = [alone.step(t) for t in tokens[b]][2:]
        detach_packed(model)
        assert all(_rel(x[b], w[0]) < 2e-2 for x, w in zip(got, want)), b
