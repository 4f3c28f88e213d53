"""The 4-bit row cache in the model integration: a small Qwen2 model decodes through PackedDecoder, its logits against
the same model with dense float32 attention over the rows that its cache reads back; selected pages; cropping."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, LogitFillCache, select_pages
from logitfill_amd.qwen2 import PackedDecoder, detach_packed
from tests.test_gpu_qwen2 import _model

pytestmark = pytest.mark.gpu


def _dense(manager, layer_idx, query, key_new, value_new, scaling):
    """Commits, then attends what the cache reads back, in float32."""
    manager.commit(layer_idx, key_new, value_new)
    layer = manager.layers[layer_idx]
    k, v = (t.repeat_interleave(manager.n_q // manager.n_kv, 1) for t in layer.read(0, layer.length))
    n, total = query.shape[2], layer.length
    s = torch.matmul(query.float(), k.transpose(-1, -2).contiguous()) * scaling
    hidden = torch.arange(total, device=s.device)[None, :] > torch.arange(n, device=s.device)[:, None] + total - n
    return torch.matmul(torch.softmax(s.masked_fill(hidden, float("-inf")), -1), v).to(query.dtype)


def _run(model, mgr, prompt, forced, *args, **kwargs):
    dec = PackedDecoder(model, mgr, *args, **kwargs)
    out = [dec.prefill(prompt)] + [dec.step(tok) for tok in forced]
    detach_packed(model)
    return torch.cat(out).float()


def _inputs(gpu, n=300, steps=40):
    g = torch.Generator().manual_seed(3)
    return torch.randint(0, 512, (1, n), generator=g).to(gpu), torch.randint(0, 512, (steps,), generator=g).to(gpu)


def test_decoder_matches_dense_attention_over_its_rows(gpu):
    model = _model(gpu)
    prompt, forced = _inputs(gpu)
    managers = [Int4KVManager(2, 4, 2, 128, 64, 32, gpu) for _ in range(2)]
    ours = _run(model, managers[0], prompt, forced)
    ref = _run(model, managers[1], prompt, forced, _dense)
    assert managers[0].seq_len == 340 and managers[0].layers[0].length == 340
    # float32 all through; a code decided at the border of two moves a row's value by a step of 15
    for s in range(ours.shape[0]):
        rel = float((ours[s] - ref[s]).norm() / ref[s].norm())
        assert rel < 2e-2, f"step {s}: rel-L2 {rel:.3g}"
    assert float((ours[:2] - ref[:2]).norm() / ref[:2].norm()) < 1e-4
    with torch.no_grad():
        dense = model(input_ids=torch.cat([prompt[0], forced]).view(1, -1), use_cache=False).logits[0, 299:].float()
    cos = torch.nn.functional.cosine_similarity(ours, dense, dim=-1)
    assert float(cos.min()) > 0.98, cos


def test_decoder_over_selected_pages(gpu):
    """Every page selected is every row; fewer pages are what select_pages says."""
    model = _model(gpu)
    prompt, forced = _inputs(gpu, steps=6)
    every = _run(model, Int4KVManager(2, 4, 2, 128, 32, 32, gpu), prompt, forced)
    mgr = Int4KVManager(2, 4, 2, 128, 32, 32, gpu, top_pages=16)
    assert float((_run(model, mgr, prompt, forced) - every).norm() / every.norm()) < 2e-2
    few = Int4KVManager(2, 4, 2, 128, 32, 32, gpu, top_pages=3)
    out = _run(model, few, prompt, forced)
    assert torch.isfinite(out).all() and not torch.equal(out[1:], every[1:])
    pages = select_pages(few, 0, torch.ones(1, 4, 1, 128, device=gpu), 3)
    assert (pages >= 0).all() and (pages < 305 // 32).all()


def test_transformers_cache_positions_and_cropping(gpu):
    """hf_cache drives positions from the cache's length; a cropped cache continues as if the rest had not been."""
    model = _model(gpu)
    prompt, forced = _inputs(gpu, n=90, steps=5)
    mgr = Int4KVManager(2, 4, 2, 128, 32, 64, gpu)
    want = _run(model, mgr, prompt, forced, hf_cache=True)
    assert float((want - _run(model, Int4KVManager(2, 4, 2, 128, 32, 64, gpu), prompt, forced)).norm()) < 1e-3
    dec = PackedDecoder(model, mgr, hf_cache=True)
    dec.prefill(prompt)
    for tok in forced[:3]:
        dec.step(tok)
    for tok in (7, 8, 9):  # drafts that are turned down
        dec.step(torch.tensor(tok, device=gpu))
    cache = LogitFillCache(mgr)
    cache.crop(-3)
    assert mgr.seq_len == 93 and cache.get_seq_length() == 93
    dec.pos = 93
    got = dec.step(forced[3])
    detach_packed(model)
    assert float((got[0] - want[4]).norm() / want[4].norm()) < 1e-5
    cache.crop(200)
    assert mgr.seq_len == 94
    cache.crop(10)
    assert mgr.seq_len == 10 and mgr.layers[0].lengths == [10]
