"""Attention over the 4-bit row cache where groups of sequences share a prefix, against float64 over the prefix's rows and the
sequence's own one behind the other."""
import numpy as np
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, LogitFillCache, int4, int4_attention, select_pages
from oracle import int4 as o4
from tests.helpers import f32
from tests.int4_helpers import assert_within, attention_bound, many_rows_bound, query, rows, _size

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["rule", "many"])
def kernel(request, monkeypatch):
    """By the rule, which takes these sizes to the general kernel, and by the many-row kernel wherever it serves."""
    if request.param == "many":
        monkeypatch.setattr(int4, "SHARED_MANY_ROWS", dict.fromkeys((32, 64, 128), 0))
        monkeypatch.setattr(int4, "SHARED_LEAST_ROWS", 1)
    return request.param


def pair(gpu, D, group, heads, prefixes, batch, layers=1, **kw):
    n_q, n_kv = heads
    prefix = Int4KVManager(layers, n_q, n_kv, D, 64, group, gpu, batch_size=prefixes)
    return prefix, Int4KVManager(layers, n_q, n_kv, D, 64, group, gpu, batch_size=batch, prefix=prefix, **kw)


def want(q, before, behind, common, own, group, scaling, dtype, q_lens=None, top=0.0):
    """Float64 output and its bound (the bounds of the cache's own attention, of all rows)."""
    qn = f32(q)
    (pk, pv), (ok, ov) = (tuple(f32(t) for t in p) for p in (before, behind))
    B, n_q, n, D = qn.shape
    H, each = pk.shape[1], B // pk.shape[0]
    g = n_q // H
    out, tol = np.zeros(qn.shape), np.zeros(qn.shape)
    for b in range(B):
        p, m = b // each, n if q_lens is None else q_lens[b]
        total = common[p] + own[b]
        for h in range(H):
            k = np.concatenate([pk[p, h, : common[p]], ok[b, h, : own[b]]])
            v = np.concatenate([pv[p, h, : common[p]], ov[b, h, : own[b]]])
            kd, vd = o4.values(k, group), o4.values(v, group)
            smax = float(o4.quantise(v, group)[1].max(initial=0))
            for j in range(m):
                seen = np.arange(total) <= total - m + j
                head = slice(h * g, (h + 1) * g)
                out[b, head, j] = r = o4.attend(qn[b, head, j], kd, vd, scaling, np.broadcast_to(seen, (g, total)))
                tol[b, head, j] = attention_bound(qn[b, head, j], _size(k, group)[seen], _size(v, group)[seen], scaling, r, dtype,
                                                  smax, max(smax, top))
                if dtype == "bf16" and D <= 128:
                    tol[b, head, j] += many_rows_bound(qn[b, head, j], kd[seen], vd[seen], scaling)
    return out, tol


def check(gpu, D, group, heads, dtype, common, own, q_len=1, seed=0, lengths=None, scaling=None):
    n_q, n_kv = heads
    before = rows((len(common), n_kv, max(common + [1]), D), dtype, seed)
    behind = rows((len(own), n_kv, max(own + [1]), D), dtype, seed + 1)
    q = query((len(own), n_q, q_len, D), dtype, seed)
    prefix, mgr = pair(gpu, D, group, heads, len(common), len(own))
    prefix.commit(0, *(t.to(gpu) for t in before), common)
    mgr.commit(0, *(t.to(gpu) for t in behind), own)
    scaling = D ** -0.5 if scaling is None else scaling
    out = int4_attention(mgr, 0, q.to(gpu), None, None, scaling, lengths=lengths)
    assert_within(out, *want(q, before, behind, common, own, group, scaling, dtype, lengths), f"{common} {own}")
    return before, behind, q, prefix, mgr, out


LAYOUTS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("D,group", LAYOUTS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_layouts(gpu, D, group, dtype):
    """Few rows a prefix and many, prefixes of unlike lengths, own rows from one on."""
    check(gpu, D, group, (4, 2), dtype, [333, 70], [1, 40, 65, 7], seed=D + group)
    check(gpu, D, group, (14, 2), dtype, [200], [5, 1, 33, 64, 3, 2, 90], seed=D + group + 1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 63, 64, 129, 1000])
def test_prefix_lengths(gpu, length, dtype):
    check(gpu, 128, 64, (7, 1), dtype, [length], [3, 5, 70, 1, 2, 33], seed=length)


@pytest.mark.parametrize("rows_", [32, 33, 64, 127, 128, 129, 300])
def test_row_tile_borders(gpu, rows_):
    check(gpu, 64, 32, (1, 1), "bf16", [100], [2] * rows_, seed=rows_)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_drafts_and_ragged_queries(gpu, dtype):
    """Several tokens a sequence, fewer in some; rows behind a sequence's last query are zeros."""
    *_, out = check(gpu, 128, 64, (6, 2), dtype, [300, 64], [9, 4, 30, 6], q_len=4, seed=5, lengths=[4, 0, 2, 3])
    assert not out[1].any() and not out[2, :, 2:].any() and not out[3, :, 3:].any()
    check(gpu, 64, 64, (8, 2), dtype, [90], [5, 80, 6], q_len=5, seed=6)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_queries_inside_the_prefix(gpu, dtype):
    """A sequence of fewer rows than queries: its first queries stand in the prefix, or in front of it."""
    check(gpu, 128, 128, (4, 2), dtype, [50], [0, 1, 3, 2], q_len=3, seed=7)
    *_, out = check(gpu, 64, 32, (28, 2), dtype, [2], [0, 1, 5, 0], q_len=5, seed=8)
    assert not out[0, :, :3].any() and not out[1, :, :2].any() and out[0, :, 3:].any()


def test_no_prefix_rows_and_no_own_rows(gpu):
    check(gpu, 64, 64, (4, 2), "bf16", [0, 40], [3, 4, 5, 6], seed=9)
    check(gpu, 64, 64, (4, 2), "bf16", [0], [3, 4], seed=10)
    check(gpu, 64, 64, (40, 2), "bf16", [77], [0, 0], seed=11)


@pytest.mark.parametrize("scaling", [0.0, -0.2, 2.0])
def test_scalings(gpu, scaling):
    check(gpu, 128, 64, (14, 2), "bf16", [150], [20, 7, 33], seed=12, scaling=scaling)


def test_without_the_prefix_it_is_the_cache_s_own(gpu):
    before, behind, q, prefix, mgr, out = check(gpu, 128, 64, (4, 2), "bf16", [100], [30, 40], seed=13)
    alone = Int4KVManager(1, 4, 2, 128, 64, 64, gpu, batch_size=2)
    alone.commit(0, *(t.to(gpu) for t in behind), [30, 40])
    mgr.prefix = None
    a = int4_attention(mgr, 0, q.to(gpu), None, None, 0.1)
    assert torch.equal(a, int4_attention(alone, 0, q.to(gpu), None, None, 0.1))
    mgr.prefix = prefix
    assert torch.equal(int4_attention(mgr, 0, q.to(gpu), None, None, 128 ** -0.5), out)
    prefix.reset()
    assert torch.equal(int4_attention(mgr, 0, q.to(gpu), None, None, 0.1), a)


@pytest.mark.parametrize("heads", [(4, 2), (28, 2)])
def test_rows_taken_back_need_not_be_finite(gpu, heads, kernel):
    """What stands behind a prefix's last row: infinities and NaN of rows that were truncated."""
    D, group, common, own = 128, 64, [75], [4, 9, 2]
    before, behind, q, prefix, mgr, out = check(gpu, D, group, heads, "bf16", common, own, seed=14)
    bad = torch.full((1, heads[1], 40, D), float("inf"), dtype=torch.bfloat16, device=gpu)
    bad[..., ::3] = float("nan")
    prefix.commit(0, bad, bad)
    prefix.truncate(75)
    again = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5)
    assert_within(again, *want(q, before, behind, common, own, group, D ** -0.5, "bf16", top=65504.0))
    if kernel == "many":  # (it takes its ranges from the rows that are there)
        assert torch.equal(again, out)


def test_commits_steps_and_layers(gpu):
    """Samples of one prompt continue by themselves: tokens are appended to the own rows, layer by layer."""
    D, B, H, n_q = 64, 6, 2, 8
    prefix, mgr = pair(gpu, D, 32, (n_q, H), 2, B, layers=2)
    before = [rows((2, H, 90, D), "bf16", 20 + i) for i in range(2)]
    for i in range(2):
        prefix.commit(i, *(t.to(gpu) for t in before[i]), [90, 41])
    behind = [[torch.zeros(B, H, 0, D, dtype=torch.bfloat16)] * 2 for _ in range(2)]
    for step in range(4):
        for i in range(2):
            k, v = rows((B, H, 1, D), "bf16", 100 + 2 * step + i)
            q = query((B, n_q, 1, D), "bf16", 50 + step)
            behind[i] = [torch.cat(pair_, 2) for pair_ in zip(behind[i], (k, v))]
            out = int4_attention(mgr, i, q.to(gpu), k.to(gpu), v.to(gpu), 0.2)
            assert_within(out, *want(q, before[i], behind[i], [90, 41], [step + 1] * B, 32, 0.2, "bf16"))
    assert prefix.layers[0].lengths == [90, 41] and mgr.layers[1].lengths == [4] * B and mgr.seq_len == 4
    assert mgr.prefix_lengths(0) == [90] * 3 + [41] * 3
    cache = LogitFillCache(mgr)
    assert cache.get_seq_length() == 94 and cache.get_mask_sizes(1) == (95, 0)
    cache.crop(-1)
    assert mgr.layers[0].lengths == [3] * B
    with pytest.raises(ValueError, match="shared prefix"):
        cache.crop(40)


def test_streams_and_captured_steps(gpu):
    """A captured step appends and attends; replays follow the device's lengths; a truncation of the prefix on another
    stream is waited for."""
    D, B = 128, 5
    before, behind, q, prefix, mgr, _ = check(gpu, D, 64, (28, 4), "bf16", [500], [20] * B, seed=15)
    mgr.layers[0].reserve(200)
    k, v = (t.to(gpu) for t in rows((B, 4, 1, D), "bf16", 30))
    qd = q.to(gpu)
    int4_attention(mgr, 0, qd, k, v, 0.1)
    mgr.truncate(20)
    mgr.sync_lengths()
    prefix.sync_lengths()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_attention(mgr, 0, qd, k, v, 0.1)
    eager = []
    for step in range(3):
        k += 0.25
        graph.replay()
        mgr.advance(1)
        again = int4_attention(mgr, 0, qd, None, None, 0.1)
        torch.cuda.synchronize()
        # (the splits follow the lengths: equal within the output's rounding)
        assert float((out.float() - again.float()).norm() / again.float().norm()) < 2.0 ** -7
        eager.append(out.clone())
    assert not torch.equal(eager[0], eager[2])
    side = torch.cuda.Stream()
    prefix.truncate(64)
    short = int4_attention(mgr, 0, qd, None, None, 0.1)
    with torch.cuda.stream(side):
        again = int4_attention(mgr, 0, qd, None, None, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(short, again) and not torch.equal(short, out)


def test_a_captured_prefix_fills_later(gpu):
    """What is captured of an empty prefix attends what its device lengths say in a replay."""
    D = 64
    prefix, mgr = pair(gpu, D, 32, (4, 2), 1, 2)
    for m in (prefix, mgr):
        m.layers[0].reserve(128)
    before, behind = rows((1, 2, 70, D), "bf16", 1), rows((2, 2, 9, D), "bf16", 2)
    q = query((2, 4, 1, D), "bf16", 3)
    qd = q.to(gpu)
    mgr.commit(0, *(t.to(gpu) for t in behind))
    int4_attention(mgr, 0, qd, None, None, 0.1)
    prefix.sync_lengths()
    mgr.sync_lengths()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_attention(mgr, 0, qd, None, None, 0.1)
    for common in ([0], [70]):
        if common[0]:
            prefix.commit(0, *(t.to(gpu) for t in before))
        graph.replay()
        torch.cuda.synchronize()
        assert_within(out, *want(q, before, behind, common, [9, 9], 32, 0.1, "bf16"))


def test_queries_of_any_strides(gpu):
    before, behind, q, prefix, mgr, out = check(gpu, 128, 64, (28, 4), "bf16", [120], [3, 9, 20], q_len=2, seed=16)
    turned = q.transpose(1, 2).contiguous().to(gpu).transpose(1, 2)
    assert torch.equal(int4_attention(mgr, 0, turned, None, None, 128 ** -0.5), out)
    wide = torch.zeros(3, 28, 2, 131, dtype=q.dtype, device=gpu)[..., 3:]
    wide.copy_(q)
    assert torch.equal(int4_attention(mgr, 0, wide, None, None, 128 ** -0.5), out)


def test_refused_prefixes(gpu):
    def manager(heads=(4, 2), D=64, group=32, layers=1, batch=1, **kw):
        return Int4KVManager(layers, *heads, D, 64, group, gpu, batch_size=batch, **kw)

    base = manager(batch=2)
    for other in (manager((2, 2)), manager((4, 1)), manager(D=128), manager(group=64), manager(layers=2)):
        with pytest.raises(ValueError, match="the prefix has"):
            manager(prefix=other)
    with pytest.raises(ValueError, match="do not divide"):
        manager(batch=3, prefix=base)
    with pytest.raises(ValueError, match="top_pages"):
        manager(batch=2, prefix=base, top_pages=3)
    with pytest.raises(TypeError):
        manager(prefix="base")
    with pytest.raises(ValueError, match="no prefix of its own"):
        base.prefix = base
    behind = manager(batch=4, prefix=base)
    with pytest.raises(ValueError, match="no prefix of its own"):
        manager(batch=4, prefix=behind)
    q, rows_ = torch.zeros(4, 4, 1, 64, device=gpu), torch.zeros(4, 2, 70, 64, device=gpu)
    behind.commit(0, rows_, rows_)
    pages = select_pages(behind, 0, q, 2)
    with pytest.raises(ValueError, match="pages"):
        int4_attention(behind, 0, q, None, None, 0.1, pages=pages)
    base.prefix = manager()
    with pytest.raises(ValueError, match="prefix of its own"):
        int4_attention(behind, 0, q, None, None, 0.1)
