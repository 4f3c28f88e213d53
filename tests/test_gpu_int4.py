"""The 4-bit row cache on the device against its float64 oracle: rows written and read back bit for bit,
attention within the rounding's bounds, page selection equal, for lengths, layouts, strides and masks where
each can go wrong."""
import threading

import numpy as np
import pytest
import torch

from logitfill_amd import _native
from logitfill_amd.packed import Int4KVManager, int4, int4_attention, layout, select_pages
from oracle import int4 as o4
from tests.helpers import f32
from tests.int4_helpers import TYPES, assert_within, expected, query, rows

pytestmark = pytest.mark.gpu

LAYOUTS = [(64, 32, 32), (64, 64, 64), (128, 32, 128), (128, 64, 64), (128, 128, 32), (256, 32, 64), (256, 64, 128),
           (256, 128, 256)]  # head_dim, group, page


def manager(gpu, D, group, page, n_q, n_kv, batch=1, layers=1, **kw):
    return Int4KVManager(layers, n_q, n_kv, D, page, group, gpu, batch_size=batch, **kw)


def check_rows(mgr, key, value, lengths, group, page):
    """The cache's rows and bounds against the oracle's, bit for bit."""
    T = max(lengths)
    k, v = mgr.layers[0].read(0, T + 3)
    bounds = mgr.layers[0].page_bounds()
    for b, n in enumerate(lengths):
        for ours, x in ((k, key), (v, value)):
            want = o4.values(f32(x[b, :, :n]), group).astype(np.float32)
            assert np.array_equal(f32(ours[b, :, :n]), want), b
            assert not ours[b, :, n:].any()
        want = o4.bounds(o4.values(f32(key[b, :, :n]), group), page)
        assert np.array_equal(f32(bounds[b, :, : n // page]), want), b


@pytest.mark.parametrize("D,group,page", LAYOUTS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_rows_written_in_pieces(gpu, D, group, page, dtype):
    """Single tokens, a few, and runs that start and end inside records and pages, ragged."""
    B, H, T = 3, 2, 2 * page + 70
    key, value = rows((B, H, T, D), dtype, D + group)
    mgr = manager(gpu, D, group, page, 2 * H, H, B)
    at = [0] * B
    for step, sizes in enumerate([(1, 1, 1), (7, 0, 3), (1, 1, 1), (40, 33, page), (2, 9, 1), (page, page + 5, 31), (1, 1, 1)]):
        n = max(sizes)
        k, v = torch.zeros(B, H, n, D, dtype=key.dtype), torch.zeros(B, H, n, D, dtype=key.dtype)
        for b, m in enumerate(sizes):
            k[b, :, :m], v[b, :, :m] = key[b, :, at[b]:at[b] + m], value[b, :, at[b]:at[b] + m]
        ragged = None if len(set(sizes)) == 1 else list(sizes)
        mgr.commit(0, k.to(gpu), v.to(gpu), ragged)
        at = [a + m for a, m in zip(at, sizes)]
        assert mgr.layers[0].lengths == at
    check_rows(mgr, key, value, at, group, page)


def test_a_token_at_a_time_is_the_prompt_at_once(gpu):
    D, group, page, T = 128, 64, 64, 130
    key, value = (t.to(gpu) for t in rows((1, 2, T, D), "bf16", 3))
    a, b = (manager(gpu, D, group, page, 2, 2) for _ in range(2))
    a.commit(0, key, value)
    for t in range(T):
        b.commit(0, key[:, :, t:t + 1], value[:, :, t:t + 1])
    for x, y in zip(a.layers[0].read(0, T), b.layers[0].read(0, T)):
        assert torch.equal(x, y)
    assert torch.equal(a.layers[0].page_bounds()[:, :, :2], b.layers[0].page_bounds()[:, :, :2])


def test_codes_are_the_layout_modules(gpu):
    """The same codes, scales and minima as a page of int4 Values in the packed layout."""
    D, group = 128, 32
    key, value = (t.to(gpu) for t in rows((1, 2, 128, D), "bf16", 5))
    mgr = manager(gpu, D, group, 128, 2, 2)
    mgr.commit(0, key, value)
    got = mgr.layers[0].read(0, 128)
    for ours, x in zip(got, (key, value)):
        code, scale, lo = layout.asymmetric_codes(x[0].float().reshape(2, 128, D // group, group).contiguous(), 4)[:3]
        want = code.double() * scale.half().double().reshape(2, 128, -1, 1) + lo.half().double().reshape(2, 128, -1, 1)
        assert torch.equal(ours[0], want.reshape(2, 128, D).float())


def test_sources_of_other_strides_and_alignment(gpu):
    """[B, T, H, D] transposed, an offset of one element, unlike Key and Value strides."""
    B, H, T, D, group, page = 2, 3, 75, 64, 32, 32
    key, value = rows((B, H, T, D), "fp16", 9)
    wide = torch.zeros(B, T, H, D + 1, dtype=key.dtype)
    wide[..., 1:] = key.transpose(1, 2)
    k = wide.to(gpu)[..., 1:].transpose(1, 2)
    v = value.transpose(1, 2).contiguous().to(gpu).transpose(1, 2)
    assert k.stride() != v.stride()
    mgr = manager(gpu, D, group, page, 3, H, B)
    mgr.commit(0, k, v)
    check_rows(mgr, key, value, [T] * B, group, page)
    strided = torch.zeros(B, H, T, 2 * D, dtype=key.dtype)  # channel stride 2
    strided[..., ::2] = key
    mgr.reset()
    mgr.commit(0, strided.to(gpu)[..., ::2], v)
    check_rows(mgr, key, value, [T] * B, group, page)


def test_edge_rows(gpu):
    """Constant rows, tiny and large ranges, borders between two codes, zeros of both signs."""
    D, group = 64, 32
    x = torch.zeros(1, 1, 40, D)
    x[0, 0, 1] = 3.0
    x[0, 0, 2] = torch.linspace(0, 15, D)
    x[0, 0, 3] = torch.arange(D) % 31 / 2                   # halves: ties go to the even code
    x[0, 0, 4] = torch.linspace(-1e-6, 1e-6, D)
    x[0, 0, 5] = torch.linspace(-60000, 60000, D)
    x[0, 0, 6] = -torch.arange(D) * 0.25
    x[0, 0, 7, ::2] = -0.0
    x[0, 0, 8:] = torch.randn(32, D, generator=torch.Generator().manual_seed(1)).round(decimals=1)
    for dtype in TYPES:
        rounded = x.to(TYPES[dtype])
        mgr = manager(gpu, D, group, 32, 1, 1)
        mgr.commit(0, rounded.to(gpu), -rounded.to(gpu))
        check_rows(mgr, rounded, -rounded, [40], group, 32)


def test_read_ranges_and_types(gpu):
    B, H, T, D, group, page = 2, 2, 100, 128, 64, 64
    key, value = rows((B, H, T, D), "bf16", 12)
    mgr = manager(gpu, D, group, page, 2, H, B)
    mgr.commit(0, key.to(gpu), value.to(gpu), [100, 41])
    full = mgr.layers[0].read(0, T)
    for dtype in TYPES.values():
        got = mgr.layers[0].read([37, 5], 50, dtype)
        for ours, ref in zip(got, full):
            assert ours.dtype == dtype
            assert torch.equal(ours[0], ref[0, :, 37:87].to(dtype))
            assert torch.equal(ours[1, :, :36], ref[1, :, 5:41].to(dtype)) and not ours[1, :, 36:].any()
    k, v = mgr.layers[0].dequantize(1)
    assert k.shape == (H, 41, D) and torch.equal(k, full[0][1, :, :41]) and torch.equal(v, full[1][1, :, :41])
    assert mgr.layers[0].read(0, 0)[0].shape == (B, H, 0, D)
    far = mgr.layers[0].read([1 << 30, 90], 20)[0]
    assert not far[0].any() and not far[1].any()


def test_capacity_grows_and_truncation_rewrites(gpu):
    """Growth keeps rows and bounds; rows, nibbles and bounds behind a truncation are written anew."""
    D, group, page = 64, 64, 32
    key, value = rows((1, 2, 200, D), "bf16", 20)
    mgr = manager(gpu, D, group, page, 2, 2)
    dk, dv = key.to(gpu), value.to(gpu)
    mgr.commit(0, dk[:, :, :50], dv[:, :, :50])
    first = mgr.layers[0].capacity
    mgr.commit(0, dk[:, :, 50:150], dv[:, :, 50:150])
    assert mgr.layers[0].capacity > first
    check_rows(mgr, key, value, [150], group, page)
    other_k, other_v = rows((1, 2, 210, D), "bf16", 21)
    for keep in (133, 64, 45, 0):
        for step in (1, 70):
            mgr.truncate(keep)
            mgr.commit(0, other_k[:, :, keep:keep + step].to(gpu), other_v[:, :, keep:keep + step].to(gpu))
            k = torch.cat([key[:, :, :keep], other_k[:, :, keep:keep + step]], 2)
            v = torch.cat([value[:, :, :keep], other_v[:, :, keep:keep + step]], 2)
            check_rows(mgr, k, v, [keep + step], group, page)
        mgr.truncate(keep)
    assert mgr.seq_len == 0


CASES = [
    # D, group, page, n_q, n_kv, lengths, q_len, dtype
    (128, 64, 128, 28, 4, [1061], 1, "bf16"),
    (128, 128, 128, 12, 2, [1, 2, 33, 640], 1, "bf16"),
    (128, 32, 64, 10, 2, [300, 0, 31], 1, "fp16"),
    (64, 32, 64, 14, 2, [700, 129], 1, "fp16"),
    (64, 64, 32, 8, 8, [65], 3, "bf16"),
    (256, 128, 128, 8, 2, [257, 40], 1, "bf16"),
    (256, 32, 256, 6, 1, [511], 2, "fp32"),
    (256, 64, 32, 4, 4, [90], 1, "fp16"),
    (128, 64, 128, 32, 1, [200, 77], 1, "bf16"),
    (128, 64, 128, 40, 1, [150], 5, "fp32"),
    (128, 32, 128, 14, 2, [530, 4, 2], 4, "bf16"),      # queries in front of the first token
    (128, 128, 32, 28, 4, [400], 61, "bf16"),
    (64, 32, 128, 7, 1, [333, 150], 97, "fp16"),
    (128, 64, 128, 4, 4, [4099], 1, "fp32"),
    (64, 64, 64, 2, 1, [3], 3, "fp32"),
    (128, 64, 64, 56, 2, [2100], 130, "bf16"),
]


@pytest.mark.parametrize("D,group,page,n_q,n_kv,lengths,q_len,dtype", CASES)
def test_attention(gpu, D, group, page, n_q, n_kv, lengths, q_len, dtype):
    B = len(lengths)
    key, value = rows((B, n_kv, max(max(lengths), 1), D), dtype, sum(lengths))
    q = query((B, n_q, q_len, D), dtype, D + q_len)
    mgr = manager(gpu, D, group, page, n_q, n_kv, B)
    mgr.commit(0, key.to(gpu), value.to(gpu), lengths)
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5)
    assert out.dtype == q.dtype and out.shape == q.shape
    ref, tol = expected(q, key, value, lengths, group, D ** -0.5, dtype)
    assert_within(out, ref, tol)
    assert torch.equal(out, int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5))


MANY = [
    # rows of several 128-row tiles, tiles of one head and of several, ragged histories, a history of whole records
    (128, 128, 128, 28, 4, [1500], 61, "bf16"),
    (128, 64, 64, 8, 2, [900, 400, 290], 40, "bf16"),
    (128, 32, 32, 12, 2, [1024, 77], 130, "bf16"),
    (64, 64, 64, 4, 2, [2000], 300, "bf16"),
    (64, 32, 32, 16, 1, [640, 0, 5], 9, "bf16"),
    (128, 64, 128, 64, 1, [1333], 1, "bf16"),
    (64, 32, 32, 16, 1, [640], 90, "fp16"),  # (the general kernel)
]


@pytest.mark.parametrize("D,group,page,n_q,n_kv,lengths,q_len,dtype", MANY)
def test_many_query_rows(gpu, monkeypatch, D, group, page, n_q, n_kv, lengths, q_len, dtype):
    """The many-row kernel in front of the general one; the whole output close in the mean, too: independent roundings
    of weights, Keys and Values (fp16) and of the output."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)  # (the rule wants longer calls)
    B = len(lengths)
    key, value = rows((B, n_kv, max(lengths), D), dtype, sum(lengths) + 1)
    q = query((B, n_q, q_len, D), dtype, D + q_len)
    mgr = manager(gpu, D, group, page, n_q, n_kv, B)
    mgr.commit(0, key.to(gpu), value.to(gpu), lengths)
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5)
    ref, tol = expected(q, key, value, lengths, group, D ** -0.5, dtype)
    assert_within(out, ref, tol)
    rel = np.linalg.norm(f32(out) - ref) / np.linalg.norm(ref)
    assert rel <= {"bf16": 2.0 ** -8, "fp16": 2.0 ** -10}[dtype], rel
    assert torch.equal(out, int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5))
    # queries of unlike counts: zeros behind them, and NaN rows of the cache no query of theirs sees
    counts = [max(1, min(n, q_len - 7 * b)) if n else 0 for b, n in enumerate(lengths)]
    out = int4_attention(mgr, 0, q.to(gpu), None, None, -D ** -0.5, lengths=counts)
    ref, tol = expected(q, key, value, lengths, group, -D ** -0.5, dtype, q_lens=counts)
    assert_within(out, ref, tol)


def test_many_query_rows_of_any_size(gpu, monkeypatch):
    """Rows of 2^-60 to 2^60 (float16's range is passed through the rows' factor), of zeros, and one of NaN."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)
    D, T, n = 128, 700, 70
    key, value = rows((1, 1, T, D), "bf16", 8)
    q = query((1, 1, n, D), "bf16", 8).float()
    size = torch.exp2(torch.linspace(-60, 0, n))
    q = (q * size[:, None]).to(torch.bfloat16)
    q[0, 0, 11] = 0
    mgr = manager(gpu, D, 64, 64, 1, 1)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = expected(q, key, value, [T], 64, D ** -0.5, "bf16")
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)
    big = (q.float() * 2.0 ** 60).to(torch.bfloat16)
    ref, tol = expected(big, key, value, [T], 64, 2.0 ** -60, "bf16")
    assert_within(int4_attention(mgr, 0, big.to(gpu), None, None, 2.0 ** -60), ref, tol)
    q[0, 0, 30] = float("nan")
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5)[0, 0]
    assert out[30].isnan().all() and torch.isfinite(out[:30]).all() and torch.isfinite(out[31:]).all()


@pytest.mark.parametrize("n", [1, 64])
def test_a_nan_key_reaches_every_query_that_sees_it(gpu, monkeypatch, n):
    """In a split of its own, too, far below the others' scores."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)
    D, T = 64, 5000
    key, value = rows((1, 1, T, D), "bf16", 9)
    key[0, 0, 3] = float("nan")
    q = query((1, 2, n, D), "bf16", 9).to(gpu)
    mgr = manager(gpu, D, 32, 32, 2, 1)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    assert int4_attention(mgr, 0, q, None, None, 1.0).isnan().all()


@pytest.mark.parametrize("scaling", [3.0, -0.4, 0.0])
def test_attention_sharp_and_flat(gpu, scaling):
    """Scores of hundreds (one token takes all), of the other sign, and all equal."""
    D, group, page, T = 128, 64, 64, 321
    key, value = rows((1, 2, T, D), "bf16", 4)
    q = query((1, 6, 2, D), "bf16", 4) * 3
    mgr = manager(gpu, D, group, page, 6, 2)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = expected(q, key, value, [T], group, scaling, "bf16")
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, scaling), ref, tol)


@pytest.mark.parametrize("dtype,n", [("bf16", 1), ("fp16", 2), ("bf16", 40)])
def test_values_of_any_size(gpu, monkeypatch, dtype, n):
    """Value rows of 2^-14 to 2^14, zeros among them, and rows as large that were taken back."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)
    D, group, T = 128, 64, 600
    key, value = rows((1, 2, T, D), "fp32", 13)
    size = torch.exp2(torch.randint(-14, 12, (T,), generator=torch.Generator().manual_seed(2)).float())
    value = value * size[:, None]
    value[:, :, ::7] = 0
    key, value = key.to(TYPES[dtype]), value.to(TYPES[dtype])
    q = query((1, 6, n, D), dtype, 13)
    mgr = manager(gpu, D, group, 64, 6, 2)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = expected(q, key, value, [T], group, D ** -0.5, dtype)
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)
    top = float(o4.quantise(f32(value), group)[1].max())
    small = value * (2.0 ** -10 / size[:, None].clamp(min=2.0 ** -10)).to(value.dtype)
    for keep, s_top in ((1, top), (0, 0.0)):  # a row is left, and none
        mgr.truncate(keep)
        mgr.commit(0, key[:, :, keep:].to(gpu), small[:, :, keep:].to(gpu))
        v = torch.cat([value[:, :, :keep], small[:, :, keep:]], 2)
        ref, tol = expected(q, key, v, [T], group, D ** -0.5, dtype, top=s_top)
        assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)


def test_float32_queries_of_any_size(gpu):
    """Rows of 2^-90 to 2^90, of zeros, and one of NaN: the factor that fits a row into float16 parts is its own."""
    D, T, n = 128, 700, 40
    key, value = rows((1, 1, T, D), "fp32", 31)
    size = torch.exp2(torch.linspace(-90, 0, n))[:, None]
    q = query((1, 1, n, D), "fp32", 31) * size
    q[0, 0, 11] = 0
    mgr = manager(gpu, D, 64, 64, 1, 1)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = expected(q, key, value, [T], 64, D ** -0.5, "fp32")
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)
    big = q * 2.0 ** 90
    ref, tol = expected(big, key, value, [T], 64, 2.0 ** -91, "fp32")
    assert_within(int4_attention(mgr, 0, big.to(gpu), None, None, 2.0 ** -91), ref, tol)
    q[0, 0, 30] = float("nan")
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5)[0, 0]
    assert out[30].isnan().all() and torch.isfinite(out[:30]).all() and torch.isfinite(out[31:]).all()


def test_more_sequences_than_a_launch_takes(gpu):
    """70 ragged sequences: written by pages, then a few tokens each, read from starts of their own, attended."""
    B, H, D, group, page = 70, 2, 64, 32, 32
    g = torch.Generator().manual_seed(6)
    first = torch.randint(0, 80, (B,), generator=g).tolist()
    more = torch.randint(0, 4, (B,), generator=g).tolist()
    lengths = [a + c for a, c in zip(first, more)]
    key, value = rows((B, H, max(lengths), D), "bf16", 33)
    mgr = manager(gpu, D, group, page, 4, H, B)
    mgr.commit(0, key[:, :, :max(first)].to(gpu), value[:, :, :max(first)].to(gpu), first)
    new = [torch.stack([torch.nn.functional.pad(x[b], (0, 0, 0, 3))[:, first[b]:first[b] + 3] for b in range(B)]) for x in (key, value)]
    mgr.commit(0, new[0].to(gpu), new[1].to(gpu), more)
    check_rows(mgr, key, value, lengths, group, page)
    q = query((B, 4, 1, D), "bf16", 33)
    ref, tol = expected(q, key, value, lengths, group, D ** -0.5, "bf16")
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)


def test_broadcast_rows_and_queries(gpu):
    """Inputs whose batch, heads or tokens stand on one another (strides of zero)."""
    B, H, T, D, group, page = 2, 2, 70, 128, 64, 64
    key, value = rows((1, 1, T, D), "bf16", 34)
    q = query((1, 1, 1, D), "bf16", 34)
    mgr = manager(gpu, D, group, page, 4, H, B)
    mgr.commit(0, key.to(gpu).expand(B, H, T, D), value.to(gpu)[:, :, :1].expand(B, H, T, D))
    k, v = key.expand(B, H, T, D), value[:, :, :1].expand(B, H, T, D)
    check_rows(mgr, k, v, [T] * B, group, page)
    out = int4_attention(mgr, 0, q.to(gpu).expand(B, 4, 3, D), None, None, D ** -0.5)
    ref, tol = expected(q.expand(B, 4, 3, D), k, v, [T] * B, group, D ** -0.5, "bf16")
    assert_within(out, ref, tol)


def test_growing_scores_move_the_reference_point(gpu):
    """Every record's scores pass the last one's by more than the step that moves the reference point."""
    D, T = 64, 700
    key, value = rows((1, 1, T, D), "bf16", 6)
    key = (torch.arange(T)[:, None] * 0.5 * torch.ones(D) + 0.01 * key[0, 0].float()).to(torch.bfloat16)[None, None]
    q = torch.ones(1, 2, 1, D, dtype=torch.bfloat16)
    q[0, 1] = -1
    mgr = manager(gpu, D, 32, 32, 2, 1)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = expected(q, key, value, [T], 32, D ** -0.5, "bf16")
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)


def test_commit_and_attend_in_one_call(gpu):
    """New tokens are cached, then seen causally; ragged counts leave zeros behind."""
    B, H, n_q, D, group, page = 3, 2, 6, 128, 32, 32
    lengths, q_len, counts = [90, 31, 0], 5, [5, 2, 0]
    key, value = rows((B, H, 100, D), "bf16", 30)
    q = query((B, n_q, q_len, D), "bf16", 31)
    mgr = manager(gpu, D, group, page, n_q, H, B)
    mgr.commit(0, key.to(gpu), value.to(gpu), lengths)
    new_k, new_v = rows((B, H, q_len, D), "bf16", 32)
    out = int4_attention(mgr, 0, q.to(gpu), new_k.to(gpu), new_v.to(gpu), D ** -0.5, lengths=counts)
    ends = [n + c for n, c in zip(lengths, counts)]
    assert mgr.layers[0].lengths == ends
    for b, (n, c) in enumerate(zip(lengths, counts)):
        key[b, :, n:n + c], value[b, :, n:n + c] = new_k[b, :, :c], new_v[b, :, :c]
    ref, tol = expected(q, key, value, ends, group, D ** -0.5, "bf16", q_lens=counts)
    assert_within(out, ref, tol)
    assert not out[1, :, 2:].any() and not out[2].any()
    check_rows(mgr, key, value, ends, group, page)


def test_what_stands_behind_a_sequence_is_not_seen(gpu):
    """Rows of NaN and infinities behind the length, in the same record, change nothing."""
    D, group, page, T = 128, 64, 64, 70
    key, value = rows((2, 2, 200, D), "bf16", 40)
    bad = torch.full_like(key, float("nan"))
    bad[:, :, ::3] = float("inf")
    bad[:, :, 1::3] = -float("inf")
    q = query((2, 8, 3, D), "bf16", 41).to(gpu)
    clean, dirty = (manager(gpu, D, group, page, 8, 2, 2, capacity_tokens=256) for _ in range(2))
    dirty.commit(0, bad.to(gpu), bad.to(gpu))
    dirty.truncate(0)
    for mgr in (clean, dirty):
        mgr.commit(0, key[:, :, :T].to(gpu), value[:, :, :T].to(gpu), [T, 33])
    a, b = (int4_attention(m, 0, q, None, None, D ** -0.5) for m in (clean, dirty))
    assert torch.isfinite(b).all() and torch.equal(a, b)
    pages = select_pages(dirty, 0, q, 1)
    a, b = (int4_attention(m, 0, q, None, None, D ** -0.5, pages=pages) for m in (clean, dirty))
    assert torch.isfinite(b).all() and torch.equal(a, b)
    # a row of NaN reaches the queries that see it, and no other sequence, head or earlier query
    poison = torch.cat([key[:, :, :2], bad[:, :, :1]], 2)
    poison[1] = key[1, :, :3]
    mgr = manager(gpu, D, group, page, 8, 2, 2)
    mgr.commit(0, poison.to(gpu), value[:, :, :3].to(gpu))
    out = int4_attention(mgr, 0, q, None, None, D ** -0.5)
    assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :, :2]).all()


def test_queries_of_other_strides(gpu):
    B, H, n_q, q_len, D, T = 2, 2, 6, 4, 64, 150
    key, value = rows((B, H, T, D), "fp16", 50)
    q = query((B, n_q, q_len, D), "fp16", 50).to(gpu)
    mgr = manager(gpu, D, 32, 32, n_q, H, B)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    want = int4_attention(mgr, 0, q, None, None, 0.125)
    pages = select_pages(mgr, 0, q, 2)
    for view in (q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([q, q], -1)[..., 1:D + 1],
                 q.repeat_interleave(2, -1)[..., ::2]):
        same = torch.equal(view, q)
        other = view if same else view.contiguous()
        assert torch.equal(int4_attention(mgr, 0, view, None, None, 0.125),
                           want if same else int4_attention(mgr, 0, other, None, None, 0.125))
        assert torch.equal(select_pages(mgr, 0, view, 2), pages if same else select_pages(mgr, 0, other, 2))


SPARSE = [
    # D, group, page, n_q, n_kv, lengths, q_len, top, dtype
    (128, 64, 32, 14, 2, [700, 45, 20, 0], 1, 4, "bf16"),
    (64, 32, 32, 4, 2, [1000], 3, 7, "fp16"),
    (256, 128, 64, 6, 2, [641, 64], 1, 3, "bf16"),
    (128, 32, 32, 20, 1, [500], 2, 40, "fp32"),      # more than there are
    (128, 128, 128, 34, 2, [1300, 5], 5, 2, "bf16"),
    (64, 64, 32, 8, 8, [9000], 1, 100, "bf16"),
    (64, 32, 32, 2, 1, [33, 32, 1], 1, 1, "bf16"),
]


@pytest.mark.parametrize("D,group,page,n_q,n_kv,lengths,q_len,top,dtype", SPARSE)
def test_selected_pages(gpu, D, group, page, n_q, n_kv, lengths, q_len, top, dtype):
    B = len(lengths)
    key, value = rows((B, n_kv, max(lengths), D), dtype, top)
    q = query((B, n_q, q_len, D), dtype, top)
    mgr = manager(gpu, D, group, page, n_q, n_kv, B)
    mgr.commit(0, key.to(gpu), value.to(gpu), lengths)
    pages = select_pages(mgr, 0, q.to(gpu), top)
    assert pages.shape == (B, n_kv, q_len, top) and pages.dtype == torch.int32
    want = np.full((B, n_kv, q_len, top), -1, dtype=np.int32)
    qn, g = f32(q), n_q // n_kv
    for b, n in enumerate(lengths):
        bnd = o4.bounds(o4.values(f32(key[b, :, :n]), group), page)
        for j in range(q_len):
            at = n - q_len + j
            if at >= 0:
                for h in range(n_kv):
                    want[b, h, j] = o4.select(qn[b, h * g:(h + 1) * g, j], bnd[h], at // page, top)
    assert np.array_equal(pages.cpu().numpy(), want)
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5, pages=pages)
    ref, tol = expected(q, key, value, lengths, group, D ** -0.5, dtype, page=page, pages=want)
    assert_within(out, ref, tol)


@pytest.mark.parametrize("splits", [2, 5, 50, 64])
def test_pages_in_any_number_of_splits(gpu, monkeypatch, splits):
    """Splits that end inside a page, pass the list's end, and belong to a sequence without a token."""
    D, group, page, n = 64, 32, 256, 5
    lengths = [3000, 0, 700, 1]
    key, value = rows((4, 2, 3000, D), "bf16", 36)
    q = query((4, 4, 1, D), "bf16", 36)
    mgr = manager(gpu, D, group, page, 4, 2, 4)
    mgr.commit(0, key.to(gpu), value.to(gpu), lengths)
    pages = select_pages(mgr, 0, q.to(gpu), n)
    monkeypatch.setattr(int4, "plan_splits", lambda *a, **k: (splits, 128))
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5, pages=pages)
    ref, tol = expected(q, key, value, lengths, group, D ** -0.5, "bf16", page=page, pages=pages.cpu().numpy())
    assert_within(out, ref, tol)


def test_more_pages_than_registers_hold(gpu):
    """17 000 pages: the choice reads its scores from memory."""
    D, group, page, T, top = 64, 64, 32, 17000 * 32 + 5, 300
    g = torch.Generator().manual_seed(35)
    key = torch.randn(1, 1, T, D, generator=g).to(torch.bfloat16)
    q = query((1, 2, 1, D), "bf16", 35)
    mgr = manager(gpu, D, group, page, 2, 1)
    mgr.commit(0, key.to(gpu), key.to(gpu))
    bnd = f32(mgr.layers[0].page_bounds())[0, 0]
    want = o4.select(f32(q)[0, :, 0], bnd, T // page, top)
    assert np.array_equal(select_pages(mgr, 0, q.to(gpu), top)[0, 0, 0].cpu().numpy(), want)


def test_equal_scores_take_the_lower_pages(gpu):
    """Pages of the same rows, and a few better ones: ties in order, also across the 256-page rounds."""
    D, page, n = 64, 32, 700
    one_k, one_v = rows((1, 1, page, D), "bf16", 60)
    key = one_k.repeat(1, 1, n, 1).to(gpu)
    value = one_v.repeat(1, 1, n, 1).to(gpu)
    mgr = manager(gpu, D, 32, page, 2, 1)
    mgr.commit(0, key, value)
    mgr.commit(0, key[:, :, :5], value[:, :, :5])
    q = torch.ones(1, 2, 1, D, dtype=torch.bfloat16, device=gpu)
    assert select_pages(mgr, 0, q, 300)[0, 0, 0].tolist() == list(range(300))
    mgr.reset()
    key[:, :, 650 * page:651 * page] *= 8
    key[:, :, 3 * page:4 * page] *= 8
    mgr.commit(0, key, value)
    mgr.commit(0, key[:, :, :5], value[:, :, :5])
    assert select_pages(mgr, 0, q, 5)[0, 0, 0].tolist() == [0, 1, 2, 3, 650]
    assert select_pages(mgr, 0, q * 0, 4)[0, 0, 0].tolist() == [0, 1, 2, 3]


def test_entries_that_are_no_page_in_front(gpu):
    """Negative entries, the own page, pages past the end, repeats and descending ones are not attended."""
    D, group, page, T = 64, 32, 32, 200
    key, value = rows((1, 2, T, D), "bf16", 70)
    q = query((1, 4, 1, D), "bf16", 70)
    mgr = manager(gpu, D, group, page, 4, 2)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    lists = np.array([[[[1, 1, 4, 2, 5, 6]], [[-1, -7, 0, 3, 1 << 30, 2147483647]]]], dtype=np.int32)
    out = int4_attention(mgr, 0, q.to(gpu), None, None, 0.125, pages=torch.from_numpy(lists).to(gpu))
    ref, tol = expected(q, key, value, [T], group, 0.125, "bf16", page=page, pages=lists)
    assert_within(out, ref, tol)


def test_all_pages_selected_is_the_whole_cache(gpu):
    D, group, page, T = 128, 64, 32, 300
    key, value = rows((2, 2, T, D), "bf16", 80)
    q = query((2, 4, 3, D), "bf16", 80).to(gpu)
    mgr = manager(gpu, D, group, page, 4, 2, 2, top_pages=16)
    mgr.commit(0, key.to(gpu), value.to(gpu), [T, 77])
    by_manager = int4_attention(mgr, 0, q, None, None, D ** -0.5)
    mgr.top_pages = 0
    ref, tol = expected(q.cpu(), key, value, [T, 77], group, D ** -0.5, "bf16")
    assert_within(by_manager, ref, tol)
    assert_within(int4_attention(mgr, 0, q, None, None, D ** -0.5), ref, tol)


@pytest.mark.parametrize("top", [0, 2])
def test_a_captured_step_replays_as_the_cache_grows(gpu, top):
    """Commit and attention of two layers in one graph, replayed over page ends with the new token's tensors
    refilled, eager work of the same manager's twin in between; two graphs of one manager do not meet."""
    D, group, page, n_q, H, T = 128, 64, 32, 8, 2, 60
    key, value = (t.to(gpu) for t in rows((2, H, 130, D), "bf16", 90))
    q = query((2, n_q, 130, D), "bf16", 90).to(gpu)
    graphed, eager = (manager(gpu, D, group, page, n_q, H, 2, 2, capacity_tokens=160, top_pages=top) for _ in range(2))
    for mgr in (graphed, eager):
        for layer in range(2):
            mgr.commit(layer, key[:, :, :T], value[:, :, :T], [T, 29])
    step_q, step_k, step_v = (torch.empty(2, n, 1, D, dtype=torch.bfloat16, device=gpu) for n in (n_q, H, H))

    def step(mgr):
        return [int4_attention(mgr, layer, step_q, step_k, step_v, D ** -0.5) for layer in range(2)]

    def load(t):
        step_q.copy_(q[:, :, t:t + 1])
        step_k.copy_(key[:, :, t:t + 1])
        step_v.copy_(value[:, :, t:t + 1])

    load(T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)
    torch.cuda.current_stream().wait_stream(side)
    graphed.truncate([T, 29])
    graphed.sync_lengths()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(graphed)
        graphs.append((graph, outs))
    assert [layer.lengths for layer in graphed.layers] == [[T, 29]] * 2  # a capture commits nothing
    for t in range(T, T + 50):
        load(t)
        want = step(eager)
        torch.cuda.synchronize()
        graph, outs = graphs[t % 2]
        graph.replay()
        noise = torch.randn(1 << 16, device=gpu).sum()  # eager work between replays
        torch.cuda.synchronize()
        assert torch.isfinite(noise)
        graphed.advance(1)
        for ours, ref in zip(outs, want):
            # (the split of the tokens is the capture's: sums in another order)
            assert (ours.float() - ref.float()).abs().max() <= 2 ** -6
    assert graphed.layers[0].lengths == eager.layers[0].lengths
    for a, b in zip(graphed.layers[1].read(0, 110), eager.layers[1].read(0, 110)):
        assert torch.equal(a, b)
    assert torch.equal(graphed.layers[0].page_bounds()[0, :, :3], eager.layers[0].page_bounds()[0, :, :3])


def test_replays_past_the_capacity_write_nothing(gpu):
    D, page = 64, 32
    key, value = (t.to(gpu) for t in rows((1, 1, 64, D), "bf16", 91))
    mgr = manager(gpu, D, 32, page, 1, 1, capacity_tokens=32)
    mgr.commit(0, key[:, :, :30], value[:, :, :30])
    before = mgr.layers[0]._blocks.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mgr.commit(0, key[:, :, 30:31], value[:, :, 30:31])
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
    assert mgr.layers[0]._lens.tolist() == [32]
    mgr.advance(2)
    assert not torch.equal(mgr.layers[0]._blocks, before)
    got = mgr.layers[0].read(0, 32)[0]
    assert torch.equal(got[:, :, 30], got[:, :, 31])


def test_commits_around_a_capture(gpu):
    """A capture commits nothing; replays are told of with advance() or taken back with truncate(), to the host's own
    lengths too, and eager commits go behind what is left."""
    D, page, T = 64, 32, 90
    key, value = rows((1, 2, T, D), "bf16", 92)
    k, v = key.to(gpu), value.to(gpu)
    mgr = manager(gpu, D, 32, page, 2, 2, capacity_tokens=128)
    mgr.commit(0, k[:, :, :30], v[:, :, :30])
    step_k, step_v = k[:, :, 30:31].clone(), v[:, :, 30:31].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mgr.commit(0, step_k, step_v)
    assert mgr.seq_len == 30
    mgr.commit(0, k[:, :, 30:33], v[:, :, 30:33])
    check_rows(mgr, key, value, [33], 32, page)
    step_k.copy_(k[:, :, 33:34])
    step_v.copy_(v[:, :, 33:34])
    graph.replay()
    mgr.advance(1)
    mgr.commit(0, k[:, :, 34:60], v[:, :, 34:60])
    check_rows(mgr, key, value, [60], 32, page)
    for _ in range(3):
        graph.replay()
    mgr.truncate(60)
    check_rows(mgr, key, value, [60], 32, page)
    mgr.commit(0, k[:, :, 60:], v[:, :, 60:])
    check_rows(mgr, key, value, [T], 32, page)
    # the cache grows away from the graph, whose replays reach arrays that are still theirs
    mgr.layers[0].reserve(1000)
    others = [torch.zeros(1 << 16, dtype=torch.uint8, device=gpu) for _ in range(8)]
    graph.replay()
    torch.cuda.synchronize()
    assert not any(bool(t.any()) for t in others)
    mgr.truncate(T)
    check_rows(mgr, key, value, [T], 32, page)


def test_on_another_stream(gpu):
    D, T = 128, 3000
    key, value = (t.to(gpu) for t in rows((1, 2, T, D), "bf16", 95))
    q = query((1, 4, 1, D), "bf16", 95).to(gpu)
    mgr = manager(gpu, D, 64, 64, 4, 2, capacity_tokens=T)
    mgr.commit(0, key, value)
    want = int4_attention(mgr, 0, q, None, None, 0.1)
    torch.cuda.synchronize()
    mgr.reset()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mgr.commit(0, key, value)
        got = int4_attention(mgr, 0, q, None, None, 0.1)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_streams_attend_one_cache_at_once(gpu):
    D, T = 128, 4000
    key, value = (t.to(gpu) for t in rows((2, 2, T, D), "bf16", 96))
    qs = [query((2, 8, 1, D), "bf16", 96 + i).to(gpu) for i in range(2)]
    mgr = manager(gpu, D, 64, 64, 8, 2, 2)
    mgr.commit(0, key, value)
    want = [int4_attention(mgr, 0, q, None, None, 0.1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(int4_attention(mgr, 0, qs[i], None, None, 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_two_threads_attend_one_cache_at_once(gpu):
    """Each on a stream of its own, with queries of unlike forms."""
    D, T = 128, 2000
    key, value = (t.to(gpu) for t in rows((2, 2, T, D), "bf16", 97))
    mgr = manager(gpu, D, 64, 64, 8, 2, 2)
    mgr.commit(0, key, value)
    qs = [query((2, 8, n, D), "bf16", 97 + n).to(gpu) for n in (1, 3)]

    def call(q):
        return int4_attention(mgr, 0, q, None, None, D ** -0.5, pages=select_pages(mgr, 0, q, 5))

    want = [call(q) for q in qs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i].append(call(qs[i]))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(x, want[i]) for x in got[i])


def test_refusals(gpu):
    mgr = manager(gpu, 128, 64, 64, 8, 2, 2)
    key = torch.zeros(2, 2, 4, 128, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros(2, 8, 4, 128, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(NotImplementedError):
        mgr.commit(0, key[:1], key[:1])
    for bad in (key[:, :1], key[..., :64], key[:, :, :2]):
        with pytest.raises(ValueError):
            mgr.commit(0, key, bad)
    with pytest.raises(TypeError):
        mgr.commit(0, key, key.half())
    with pytest.raises(TypeError):
        mgr.commit(0, key.double(), key.double())
    with pytest.raises(RuntimeError):
        mgr.commit(0, key.cpu(), key.cpu())
    for lengths in ([1], [5, 1], [-1, 2]):
        with pytest.raises(ValueError):
            mgr.commit(0, key, key, lengths)
    assert mgr.layers[0].lengths == [0, 0]
    mgr.commit(0, key, key)
    for bad in (q[:, :4], q[:1], q[..., :64], q[:, :, :0], q[0]):
        with pytest.raises(ValueError):
            int4_attention(mgr, 0, bad, None, None, 1.0)
        with pytest.raises(ValueError):
            select_pages(mgr, 0, bad, 1)
    with pytest.raises(ValueError):
        int4_attention(mgr, 0, q, key, None, 1.0)
    with pytest.raises(ValueError):
        int4_attention(mgr, 0, q, key[:, :, :3], key[:, :, :3], 1.0)
    with pytest.raises(TypeError):
        int4_attention(mgr, 0, q.double(), None, None, 1.0)
    for top in (0, 1025):
        with pytest.raises(ValueError):
            select_pages(mgr, 0, q, top)
    pages = torch.zeros(2, 2, 4, 1, dtype=torch.int32, device=gpu)
    with pytest.raises(TypeError):
        int4_attention(mgr, 0, q, None, None, 1.0, pages=pages.long())
    with pytest.raises(ValueError):
        int4_attention(mgr, 0, q, None, None, 1.0, pages=pages[:, :, :3])
    with pytest.raises(ValueError):
        mgr.truncate([5, 0])
    with pytest.raises(ValueError):
        mgr.advance(10 ** 6)
    with pytest.raises(ValueError):
        mgr.layers[0].read(-1, 4)
    assert mgr.layers[0].lengths == [4, 4] and mgr.seq_len == 4
