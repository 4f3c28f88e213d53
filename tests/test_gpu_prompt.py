"""Causal attention of whole prompts on the device against float64: lengths from none to long, packed and padded, grouped
heads, types, strides, masked places that are not finite, streams and captured graphs."""
import numpy as np
import pytest
import torch

from logitfill_amd.packed import PromptPlan, prompt_attention
from tests.helpers import f32
from tests.prompt_helpers import assert_within, attend, expected, inputs

pytestmark = pytest.mark.gpu


def run(gpu, lengths, key_lengths, heads, D, dtype, *, packed_q=True, packed_k=True, seed=0, scaling=None, spare=0):
    n_q, n_kv = heads
    m = lengths if key_lengths is None else key_lengths
    T = sum(lengths) + spare if packed_q else max(lengths) + spare
    S = sum(m) + spare if packed_k else max(m) + spare
    q, k, v = inputs((1 if packed_q else len(lengths), n_q, T, D), (1 if packed_k else len(m), n_kv, S, D), dtype, seed)
    scaling = D ** -0.5 if scaling is None else scaling
    plan = PromptPlan(lengths, key_lengths, device=gpu)
    out = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), scaling, plan)
    assert out.shape == q.shape and out.dtype == q.dtype
    assert_within(out, *expected(q, k, v, lengths, m, scaling, dtype, packed_q, packed_k), f"{lengths} {m}")
    return q, k, v, plan, out


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (7, 1), (3, 3)])
def test_packed_prompts(gpu, D, heads, dtype):
    run(gpu, [1, 0, 37, 130, 300, 65, 64], None, heads, D, dtype, seed=D + heads[0])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_padded_prompts(gpu, D, dtype):
    """Rows behind a sequence's last token are zeros."""
    run(gpu, [200, 1, 129, 0], None, (6, 2), D, dtype, packed_q=False, packed_k=False, seed=D, spare=3)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("packed_q,packed_k", [(True, True), (False, False), (True, False), (False, True)])
def test_queries_behind_a_history(gpu, packed_q, packed_k, dtype):
    run(gpu, [3, 70, 1, 128], [300, 75, 64, 1000], (4, 2), 128, dtype, packed_q=packed_q, packed_k=packed_k, seed=3, spare=2)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_single_tokens(gpu, D, dtype):
    """Few rows over long Keys: one wave a workgroup, the Keys divided among many."""
    run(gpu, [1, 1, 1, 1, 1], [1, 63, 65, 2000, 5003], (7, 1), D, dtype, seed=D)
    run(gpu, [4, 2], [4100, 33], (8, 2), D, dtype, packed_q=False, packed_k=False, seed=D + 1)


@pytest.mark.parametrize("rows", [31, 32, 33, 127, 128, 129, 256, 257])
def test_row_tile_borders(gpu, rows):
    run(gpu, [rows], [rows + 40], (1, 1), 128, "bf16", seed=rows)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_more_queries_than_keys(gpu, dtype):
    """The first queries see nothing: zeros."""
    *_, out = run(gpu, [10, 200, 5], [3, 1, 0], (4, 2), 64, dtype, seed=9)
    assert not out[:, :, :7].any() and not out[:, :, 10:209].any() and not out[:, :, 210:].any()


def test_divided_row_tiles_agree_with_whole_ones(gpu, monkeypatch):
    from logitfill_amd.packed import prompt

    q, k, v, _, out = run(gpu, [150, 40], [1500, 700], (4, 2), 128, "bf16", seed=2)
    for size, groups in ((1, 1), (2, 1), (5, 1), (1000, 1), (1, 2), (2, 2), (7, 2), (1000, 2)):
        monkeypatch.setattr(prompt, "split_size", lambda *args: (size, groups))
        plan = PromptPlan([150, 40], [1500, 700], device=gpu)
        again = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), 128 ** -0.5, plan)
        assert_within(again, *expected(q, k, v, [150, 40], [1500, 700], 128 ** -0.5, "bf16", True, True), f"split {size}")
        form, = plan._forms.values()
        assert (form.n_merges > 0) == (size < 24) and form.groups == groups


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scaling", [0.0, -0.1, 3.0, 1e-30])
def test_scalings(gpu, scaling, dtype):
    """Zero weighs every Key alike, a negative one turns the order; sharp weights move the reference point often."""
    run(gpu, [140, 50], None, (4, 2), 64, dtype, seed=4, scaling=scaling)


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("fp16", 128)])
def test_two_groups_of_a_workgroup(gpu, monkeypatch, dtype, D):
    """One, an even and an odd number of Key tiles; rows that see nothing; what is masked need not be finite."""
    from logitfill_amd.packed import prompt

    monkeypatch.setattr(prompt, "split_size", lambda *args: (1000, 2))
    run(gpu, [1, 0, 37, 130, 300, 65, 64], None, (7, 1), D, dtype, seed=D)
    run(gpu, [50, 130, 5], [700, 128, 3], (4, 2), D, dtype, packed_q=False, packed_k=False, seed=D + 1, spare=2)
    test_what_is_masked_need_not_be_finite(gpu, D, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_masked_need_not_be_finite(gpu, D, dtype):
    """Keys and Values of later tokens, of other sequences and of the padding; what a row does see counts."""
    lengths = [100, 90, 7]
    q, k, v = inputs((3, 4, 110, D), (3, 2, 110, D), dtype, D)
    want = expected(q, k, v, lengths, lengths, D ** -0.5, dtype, False, False)
    late = (70, 71, 95)
    for b, n in enumerate(lengths):
        k[b, :, n:], v[b, :, n:], q[b, :, n:] = float("nan"), float("inf"), float("nan")
    k[0, 0, late[0], 5], v[0, 0, late[1], 3], v[0, 1, late[2], 6] = float("nan"), float("inf"), float("nan")
    out = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), D ** -0.5, PromptPlan(lengths, device=gpu)).cpu()
    clean = torch.ones_like(out, dtype=torch.bool)
    clean[0, :2, late[0] : 100] = False       # a NaN score: every channel
    clean[0, 2:, late[2] : 100, 6] = False    # a NaN Value: its channel
    assert_within(torch.where(clean, out, 0), np.where(clean, want[0], 0), want[1])
    assert not torch.isfinite(out[~clean]).any()
    v[0, 0, late[1], 3] = float("inf")
    k[0, 0, late[0], 5] = 0
    out = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), D ** -0.5, PromptPlan(lengths, device=gpu)).cpu()
    assert torch.isinf(out[0, :2, late[1] : 100, 3]).all() and torch.isfinite(out[0, :2, : late[1]]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("late", [False, True])
def test_float32_s_ends(gpu, D, late):
    """Keys whose scores are -inf (of rows that see them in whole tiles or in masked ones), Values of a quarter of the largest
    number and of 2^-100: as float64 has them."""
    T, at = 300, 290 if late else 40
    q, k, v = inputs((1, 2, T, D), (1, 2, T, D), "fp32", 12)
    q[..., 3] = q[..., 3].abs() + 0.5
    v[0, 1, 41, 7] = torch.finfo(torch.float32).max / 4
    v[0, 0, :, 9] = 2.0 ** -100
    hidden = k.clone()
    k[0, 0, at, 3] = -float("inf")
    hidden[0, 0, at] = 0
    out = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), D ** -0.5).cpu()
    want, tol = expected(q, hidden, v, [T], [T], D ** -0.5, "fp32", True, True)
    # rows that see it: without it
    qn, kn, vn = (f32(t).astype(np.float64) for t in (q, hidden, v))
    seen = np.tril(np.ones((T, T), dtype=bool))
    seen[:, at] = False
    want[0, 0], tol[0, 0] = attend(qn[0, 0], kn[0, 0], vn[0, 0], D ** -0.5, seen, "fp32")
    assert_within(out, want, tol)
    assert float(out[0, 0, :, 9].min()) > 0.9 * 2.0 ** -100 and torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_strides_and_alignment(gpu, dtype):
    """Views of one fused projection, rows off 16 bytes, broadcast kv heads, channels not innermost."""
    T, D = 77, 64
    q, k, v = inputs((1, 4, T, D), (1, 2, T, D), dtype, 8)
    want = expected(q, k, v, [T], [T], 0.125, dtype, True, True)
    fused = torch.cat([t.transpose(1, 2).flatten(2) for t in (q, k, v)], -1)
    for off in (0, 1):
        wide = torch.zeros(1, T, 8 * D + off, dtype=q.dtype)
        wide[..., off:] = fused
        wide = wide.to(gpu)[..., off:]
        parts = [t.unflatten(-1, (-1, D)).transpose(1, 2) for t in wide.split([4 * D, 2 * D, 2 * D], -1)]
        assert_within(prompt_attention(*parts, 0.125), *want, f"offset {off}")
    one = k[:, :1].to(gpu)
    ref = expected(q, k[:, :1].expand(1, 2, T, D), v[:, :1].expand(1, 2, T, D), [T], [T], 0.125, dtype, True, True)
    assert_within(prompt_attention(q.to(gpu), one.expand(1, 2, T, D), v[:, :1].to(gpu).expand(1, 2, T, D), 0.125), *ref)
    turned = [t.to(gpu).transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    out = prompt_attention(*turned, 0.125)
    assert_within(out, *want)
    assert out.transpose(1, 2).is_contiguous()


def test_axes_of_one_have_any_stride(gpu):
    """What is never stepped over may be off 16 bytes: a batch of one, a head, a token."""
    D = 64
    for T, n_q, n_kv in ((9, 1, 1), (1, 2, 1), (1, 1, 1)):
        q, k, v = inputs((1, n_q, T, D), (1, n_kv, T, D), "bf16", 11)
        odd = [t.to(gpu).as_strided(t.shape, [s if n > 1 else 8 * T * D + 3 for s, n in zip(t.stride()[:3], t.shape)] + [1]) for t in (q, k, v)]
        out = prompt_attention(*odd, 0.125)
        assert_within(out, *expected(q, k, v, [T], [T], 0.125, "bf16", True, True))


def test_offsets_past_32_bits(gpu):
    """Rows 2^26 elements apart: the last ones lie past 2^32 elements."""
    T, D, step = 70, 64, 1 << 26
    q, k, v = inputs((1, 2, T, D), (1, 1, T, D), "bf16", 1)
    far = torch.empty((T - 1) * step + 2 * D, dtype=torch.bfloat16, device=gpu)
    kf = far.as_strided((1, 1, T, D), (step, D, step, 1))
    vf = far[D:].as_strided((1, 1, T, D), (step, D, step, 1))
    kf.copy_(k.to(gpu))
    vf.copy_(v.to(gpu))
    assert_within(prompt_attention(q.to(gpu), kf, vf, 0.125), *expected(q, k, v, [T], [T], 0.125, "bf16", True, True))


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("fp32", 128)])
def test_a_long_prompt_s_pieces(gpu, dtype, D):
    """Rows of a long prompt, as a whole and fed in pieces, against float64 at some of its rows."""
    T, piece = 3001, 1024
    q, k, v = inputs((1, 2, T, D), (1, 1, T, D), dtype, 6)
    whole = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), D ** -0.5)
    qd, kd, vd = (t.to(gpu) for t in (q, k, v))
    parts = [prompt_attention(qd[:, :, a : a + piece], kd[:, :, : min(T, a + piece)], vd[:, :, : min(T, a + piece)], D ** -0.5)
             for a in range(0, T, piece)]
    rows = [0, 1, 63, 64, 1023, 1024, 2047, 2048, 2999, 3000]
    kn, vn = f32(k)[0, 0].astype(np.float64), f32(v)[0, 0].astype(np.float64)
    for out in (whole, torch.cat(parts, 2)):
        for h in range(2):
            seen = np.arange(T)[None, :] <= np.array(rows)[:, None]
            ref, tol = attend(f32(q)[0, h, rows], kn, vn, D ** -0.5, seen, dtype)
            assert_within(out[0, h, rows], ref, tol)


def test_streams_threads_and_graphs(gpu):
    """One plan on several streams; a captured call replayed with new inputs; the same bits each time."""
    lengths, totals = [40, 3, 1], [900, 3, 2500]
    q, k, v = (t.to(gpu) for t in inputs((1, 4, 44, 128), (1, 2, 3403, 128), "bf16", 5))
    plan = PromptPlan(lengths, totals, device=gpu)
    want = prompt_attention(q, k, v, 0.1, plan)
    assert plan._forms and next(iter(plan._forms.values())).n_merges
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs = [prompt_attention(q, k, v, 0.1, plan) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = prompt_attention(q, k, v, 0.1, plan)
        graphs.append((graph, captured))
    for step in range(3):
        v += 1
        for graph, captured in graphs:
            graph.replay()
        again = prompt_attention(q, k, v, 0.1, plan)
        torch.cuda.synchronize()
        assert all(torch.equal(captured, again) for _, captured in graphs)


def test_a_plan_s_first_call_in_a_capture_is_refused(gpu):
    q, k, v = (t.to(gpu) for t in inputs((1, 2, 9, 64), (1, 1, 9, 64), "bf16", 5))
    plan = PromptPlan([4, 5], device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.add(1)
        with pytest.raises(RuntimeError, match="before the capture"):
            prompt_attention(q, k, v, 0.1, plan)
        with pytest.raises(RuntimeError, match="takes a plan"):
            prompt_attention(q, k, v, 0.1)
    prompt_attention(q, k, v, 0.1, plan)


def test_refused_calls(gpu):
    q, k, v = (t.to(gpu) for t in inputs((1, 4, 9, 64), (1, 2, 9, 64), "bf16", 5))
    plan = PromptPlan([4, 5], device=gpu)
    for bad, error in ((lambda: prompt_attention(q.cpu(), k, v, 0.1), RuntimeError), (lambda: prompt_attention(q, k.cpu(), v, 0.1), RuntimeError),
                       (lambda: prompt_attention(q, k.float(), v, 0.1), TypeError), (lambda: prompt_attention(q.double(), k.double(), v.double(), 0.1), TypeError),
                       (lambda: prompt_attention(q[0], k, v, 0.1), ValueError), (lambda: prompt_attention(q, k, v[:, :, :8], 0.1), ValueError),
                       (lambda: prompt_attention(q[:, :3], k, v, 0.1), ValueError), (lambda: prompt_attention(q, k[:, :0], v[:, :0], 0.1), ValueError),
                       (lambda: prompt_attention(q[..., :32], k[..., :32], v[..., :32], 0.1), ValueError),
                       (lambda: prompt_attention(q, k, v, float("nan")), ValueError), (lambda: prompt_attention(q, k, v, float("inf"), plan), ValueError),
                       (lambda: prompt_attention(q[:, :, :8], k, v, 0.1, plan), ValueError), (lambda: prompt_attention(q, k[:, :, :8], v[:, :, :8], 0.1, plan), ValueError),
                       (lambda: prompt_attention(q.expand(3, 4, 9, 64), k, v, 0.1, plan), ValueError), (lambda: prompt_attention(q.expand(2, 4, 9, 64), k, v, 0.1), ValueError),
                       (lambda: prompt_attention(q.clone().requires_grad_(), k, v, 0.1), RuntimeError)):
        with pytest.raises(error):
            bad()
    with torch.no_grad():
        prompt_attention(q.clone().requires_grad_(), k, v, 0.1, plan)


def test_nothing_to_do(gpu):
    q, k = torch.ones(2, 4, 0, 64, device=gpu), torch.ones(2, 2, 0, 64, device=gpu)
    assert prompt_attention(q, k, k, 0.1).shape == (2, 4, 0, 64)
    q = torch.ones(2, 4, 3, 64, device=gpu)
    assert not prompt_attention(q, k, k, 0.1).any()
    assert not prompt_attention(q, torch.ones(2, 2, 5, 64, device=gpu), torch.ones(2, 2, 5, 64, device=gpu), 0.1, PromptPlan([0, 0], [5, 5], device=gpu)).any()
    assert prompt_attention(q[:0], k[:0], k[:0], 0.1).shape == (0, 4, 3, 64)
