"""Shared prefixes whose plans reach the most splits that a call takes, against float64."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, int4, int4_attention
from tests.int4_helpers import assert_within, query, rows
from tests.test_gpu_shared import want

pytestmark = pytest.mark.gpu


def test_one_long_sequence_among_short_ones_behind_a_long_prefix(gpu, monkeypatch):
    """The many-row kernel's prefix in 512 splits, and own rows that would ask for 516."""
    monkeypatch.setattr(int4, "SHARED_MANY_ROWS", dict.fromkeys((32, 64, 128), 0))
    D, group, heads, common, own = 64, 32, (8, 1), [70000], [66000, 9, 40, 1, 3, 65, 2, 7]
    before = rows((1, 1, common[0], D), "bf16", 1)
    behind = rows((len(own), 1, 66, D), "bf16", 2)
    long = rows((1, 1, own[0], D), "bf16", 3)
    q = query((len(own), heads[0], 1, D), "bf16", 4)
    prefix = Int4KVManager(1, *heads, D, 64, group, gpu)
    mgr = Int4KVManager(1, *heads, D, 64, group, gpu, batch_size=len(own), prefix=prefix, capacity_tokens=66048)
    prefix.commit(0, *(t.to(gpu) for t in before))
    new = [t[:, :, :1].clone() for t in behind]
    for i, n in enumerate(own):  # (all but each one's last token)
        k, v = ((long, behind)[i > 0][s][0 if i == 0 else i : 1 if i == 0 else i + 1, :, : n - 1] for s in (0, 1))
        wide = [torch.zeros(len(own), 1, n - 1, D, dtype=k.dtype, device=gpu) for _ in (0, 1)]
        for t, x in zip(wide, (k, v)):
            t[i] = x[0].to(gpu)
        mgr.commit(0, *wide, [n - 1 if j == i else 0 for j in range(len(own))])
        for t, x in zip(new, (long if i == 0 else behind)):
            t[i] = x[0 if i == 0 else i, :, n - 1 : n]
    out = int4_attention(mgr, 0, q.to(gpu), *(t.to(gpu) for t in new), D ** -0.5)
    assert mgr.layers[0].lengths == own
    ref = want(q[:1], before, long, common, own[:1], group, D ** -0.5, "bf16")
    assert_within(out[:1], *ref, "the long one")
    some = want(q[1:], before, tuple(t[1:] for t in behind), common, own[1:], group, D ** -0.5, "bf16")
    assert_within(out[1:], *some, "the short ones")


def test_top_pages_set_behind_a_prefix(gpu):
    """Refused before the new tokens are committed."""
    prefix = Int4KVManager(1, 4, 2, 64, 64, 32, gpu)
    mgr = Int4KVManager(1, 4, 2, 64, 64, 32, gpu, batch_size=2, prefix=prefix)
    k = torch.ones(2, 2, 200, 64, device=gpu)
    prefix.commit(0, k[:1], k[:1])
    mgr.commit(0, k, k)
    q = torch.ones(2, 4, 1, 64, device=gpu)
    mgr.top_pages = 2
    with pytest.raises(ValueError, match="pages"):
        int4_attention(mgr, 0, q, k[:, :, :1], k[:, :, :1], 0.1)
    assert mgr.layers[0].lengths == [200, 200]
    mgr.top_pages = 0
    assert torch.isfinite(int4_attention(mgr, 0, q, k[:, :, :1], k[:, :, :1], 0.1)).all()
