"""Steps of a decoder whose sequences are not where its own last call left them: behind a prefix, or cut back one by one."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager
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
