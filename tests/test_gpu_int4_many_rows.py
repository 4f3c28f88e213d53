"""The many-row kernel where float16 does not hold what it is given."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, int4, int4_attention
from tests.int4_exact import exact, prefixes  # noqa: F401  (a fixture)
from tests.int4_helpers import assert_within, query, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
def test_keys_beside_a_constant(gpu, monkeypatch, prefixes, D, group):  # noqa: F811
    """Channels that are large in every token (Keys with a bias): scores within float32's error, and no step in the results
    where the rule passes from one kernel to the other."""
    T, n, n_q, H = 1500, 61, 8, 2
    g = torch.Generator().manual_seed(D + group)
    key = torch.randn(1, H, T, D, generator=g) * 3
    key[..., 5] += 400
    key[..., D // 2 + 3] -= 300
    key, value = key.bfloat16(), torch.randn(1, H, T, D, generator=g).bfloat16()
    q = torch.randn(1, n_q, n, D, generator=g) * 12 / D ** 0.5
    q[..., [5, D // 2 + 3]] = 12
    q = q.bfloat16()
    mgr = Int4KVManager(1, n_q, H, D, 64, group, gpu)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = exact(q, key, value, [T], group, D ** -0.5, "bf16", many=True)
    for work in (0, 1e30):
        monkeypatch.setattr(int4, "MANY_ROWS_WORK", work)
        assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol, f"work {work}")
    assert [p > 0 for p in prefixes()] == [True, False]
    assert [p > 0 for p in prefixes()] == [True, False]


def test_very_many_tokens_of_small_weight(gpu, monkeypatch, prefixes):  # noqa: F811
    """131 071 tokens of 2^-26 of the first one's weight each, in one split: 2^-9 of the whole together."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)
    monkeypatch.setattr(int4, "plan_splits", lambda *a, **k: (1, 128))
    D, T, n = 64, 1 << 17, 64
    key = torch.zeros(1, 1, T, D, dtype=torch.bfloat16)
    key[:, :, 0] = 18  # (rows of one number are kept as they are)
    value = torch.full((1, 1, T, D), 512.0, dtype=torch.bfloat16)
    value[:, :, 0] = 0
    q = torch.zeros(1, 1, n, D, dtype=torch.bfloat16)
    q[..., 7] = 1
    mgr = Int4KVManager(1, 1, 1, D, 32, 64, gpu, capacity_tokens=T)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = exact(q[:, :, -1:], key, value, [T], 64, 1.0, "bf16", many=True)
    out = int4_attention(mgr, 0, q.to(gpu), None, None, 1.0)
    assert_within(out[:, :, -1:], ref, tol)
    assert prefixes() == [1] and 0.9 < float(ref.min()) < 1.1


@pytest.mark.parametrize("D,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
def test_rows_past_fp16(gpu, monkeypatch, prefixes, D, group):  # noqa: F811
    """Values read back of up to 9e5 in one group, of 1e-4 in the next sequence, and Keys as large beside small queries; in
    rows of float32, for minima and scales are float16."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)
    T, n, n_q, H = 900, 40, 8, 2
    key, value = rows((3, H, T, D), "fp32", D + group)
    key[0, :, :, :group] = key[0, :, :, :group] / key[0, :, :, :group].abs().amax() * 4e5 + 3.4e5
    value[0, :, ::3, :group] = value[0, :, ::3, :group] / value[0, :, :, :group].abs().amax() * 4.5e5 + 4.2e5
    key[0, :, :, 0] = -6e4  # (every row's minimum within fp16)
    value[0, :, ::3, 0] = -3e4
    value[1] *= 1e-4
    value[2, :, ::50] *= 2.0 ** 12
    q = query((3, n_q, n, D), "bf16", D)
    q[0, :, :, :group] *= 2.0 ** -16
    mgr = Int4KVManager(1, n_q, H, D, 32, group, gpu, batch_size=3)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    assert float(mgr.layers[0].read(0, T)[1][0].max()) > 7e5
    out = int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5)
    ref, tol = exact(q, key, value, [T] * 3, group, D ** -0.5, "bf16", many=True)
    assert_within(out, ref, tol)
    assert all(p > 0 for p in prefixes())


def test_chunks_of_a_prompt_are_committed_and_attended(gpu, monkeypatch, prefixes):  # noqa: F811
    """Ragged chunks through the call the model makes, then a captured one replayed over page ends: both kernels over the
    device's lengths, the plan the capture's."""
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0)
    D, group, page, n_q, H, n = 128, 64, 64, 8, 2, 45
    key, value = rows((2, H, 900, D), "bf16", 41)
    q = query((2, n_q, 900, D), "bf16", 41)
    k, v, dq = key.to(gpu), value.to(gpu), q.to(gpu)
    mgr = Int4KVManager(1, n_q, H, D, page, group, gpu, batch_size=2, capacity_tokens=960)
    starts = [400, 333]
    mgr.commit(0, k[:, :, :400], v[:, :, :400], starts)

    def chunk(x, counts):
        out = torch.zeros(2, x.shape[1], n, D, dtype=x.dtype, device=x.device)
        for b, (t, c) in enumerate(zip(starts, counts)):
            out[b, :, :c] = x[b, :, t:t + c]
        return out

    def check(out, at, counts):
        ends = [t + c for t, c in zip(starts, counts)]
        ref, tol = exact(at, key, value, ends, group, D ** -0.5, "bf16", q_lens=counts, many=True)
        assert_within(out, ref, tol)
        starts[:] = ends

    for counts in ([n, n], [n, 20], [7, n], [n, 0]):
        out = int4_attention(mgr, 0, chunk(dq, counts), chunk(k, counts), chunk(v, counts), D ** -0.5, lengths=counts)
        check(out, chunk(q, counts), counts)
    assert mgr.layers[0].lengths == starts and prefixes()[0] > 0
    step = [chunk(x, [n, n]) for x in (dq, k, v)]
    int4_attention(mgr, 0, *step, D ** -0.5)
    mgr.truncate(starts)
    mgr.sync_lengths()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int4_attention(mgr, 0, *step, D ** -0.5)
    assert prefixes()[-1] > 0
    for _ in range(5):
        for held, x in zip(step, (dq, k, v)):
            held.copy_(chunk(x, [n, n]))
        graph.replay()
        noise = torch.randn(1 << 16, device=gpu).sum()
        torch.cuda.synchronize()
        assert torch.isfinite(noise)
        mgr.advance(n)
        check(out, chunk(q, [n, n]), [n, n])
    assert mgr.layers[0].lengths == starts
