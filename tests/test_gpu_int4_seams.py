"""Attention over the 4-bit row cache at the seams of its masks, within bounds that a token lost, seen too early or a record
counted twice leaves (``test_int4_bounds_host.py`` shows it): the general kernel, and the many-row kernel with it."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, int4, int4_attention
from tests.int4_exact import exact, prefixes, seam_rows  # noqa: F401  (a fixture)
from tests.int4_helpers import assert_within, query

pytestmark = pytest.mark.gpu

# D, group, page, n_q, n_kv, lengths, q_len, dtype, many-row kernel
CASES = [
    (128, 64, 64, 56, 2, [2100], 130, "bf16", False), (64, 32, 128, 7, 1, [333, 150], 97, "fp16", False),
    (128, 64, 128, 4, 4, [4099], 1, "fp32", False), (256, 128, 32, 4, 2, [900, 33], 3, "bf16", False),
    (64, 32, 32, 4, 2, [1500, 64, 0], 5, "fp32", False), (128, 128, 32, 28, 4, [400], 61, "bf16", False),
    (64, 64, 64, 4, 2, [2000], 300, "bf16", True), (128, 128, 128, 28, 4, [1500], 61, "bf16", True),
    (128, 64, 64, 56, 2, [2100], 130, "bf16", True), (128, 32, 32, 12, 2, [1024, 77], 130, "bf16", True),
    (64, 32, 32, 16, 1, [700, 0, 5], 9, "bf16", True), (128, 64, 128, 64, 1, [1333], 1, "bf16", True),
]


@pytest.mark.parametrize("D,group,page,n_q,n_kv,lengths,q_len,dtype,many", CASES)
def test_seams(gpu, monkeypatch, prefixes, D, group, page, n_q, n_kv, lengths, q_len, dtype, many):  # noqa: F811
    monkeypatch.setattr(int4, "MANY_ROWS_WORK", 0 if many else 1e30)
    B = len(lengths)
    key, value = seam_rows((B, n_kv, max(lengths), D), dtype, sum(lengths), q_len)
    q = query((B, n_q, q_len, D), dtype, D + q_len)
    mgr = Int4KVManager(1, n_q, n_kv, D, page, group, gpu, batch_size=B)
    mgr.commit(0, key.to(gpu), value.to(gpu), lengths)
    counts = [max(1, min(n, q_len - 7 * b - 2)) if n else 0 for b, n in enumerate(lengths)]
    for scaling, given in ((D ** -0.5, None), (-D ** -0.5, counts)):
        out = int4_attention(mgr, 0, q.to(gpu), None, None, scaling, lengths=given)
        ref, tol = exact(q, key, value, lengths, group, scaling, dtype, q_lens=given, many=many)
        assert_within(out, ref, tol)
    assert len(prefixes()) == 2 and all((n > 0) == many for n in prefixes())
