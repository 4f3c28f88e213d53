"""The bounds of the 4-bit row cache's attention tests against oracles that are wrong on purpose (no GPU): a query that
misses its own token or sees one too early, and a record lost or counted twice, leave them."""
import numpy as np
import pytest

from tests.int4_exact import exact, seam_rows
from tests.int4_helpers import query

# D, group, n_q, n_kv, tokens, q_len, dtype, many-row kernel
CASES = [
    (128, 32, 4, 2, 2000, 200, "bf16", True), (128, 128, 28, 4, 1500, 61, "bf16", True),
    (128, 64, 56, 2, 2100, 130, "bf16", False), (64, 32, 7, 1, 333, 97, "fp16", False), (128, 64, 4, 4, 4099, 1, "fp32", False),
    (256, 128, 4, 2, 900, 3, "bf16", False),
]


def own(seen, b):
    n, T = seen.shape
    seen[np.arange(n), np.arange(T - n, T)] = 0
    return seen


def early(seen, b):
    n, T = seen.shape
    seen[np.arange(n - 1), np.arange(T - n + 1, T)] = 1
    return seen


def record(first, times):
    def change(seen, b):
        at = first if first >= 0 else (seen.shape[1] - seen.shape[0]) // 32 * 32 + 32 * (first + 1)
        seen[:, at:at + 32] *= times
        return seen
    return change


@pytest.mark.parametrize("D,group,n_q,n_kv,T,n,dtype,many", CASES)
def test_wrong_masks_leave_the_bound(D, group, n_q, n_kv, T, n, dtype, many):
    key, value = seam_rows((1, n_kv, T, D), dtype, T, n)
    q = query((1, n_q, n, D), dtype, D + n)
    ref, tol = exact(q, key, value, [T], group, D ** -0.5, dtype, many=many)
    assert np.isfinite(ref).all() and (tol > 0).all()
    changes = {"own": own, "early": early} if n > 1 else {"own": own}
    for times in (0, 2):
        for first in (0, 32, T // 2 // 32 * 32, -1, -2):
            changes[f"record {first} x {times}"] = record(first, times)
    for name, change in changes.items():
        bad, _ = exact(q, key, value, [T], group, D ** -0.5, dtype, many=many, change=change)
        outside = (np.abs(bad - ref) > 2 * tol).any(-1)  # of every query, with the kernel's own error beside
        if name == "early":
            outside = outside[:, :, :-1]  # (the last query has no next token)
        # (a query whose weight of the row is small may hide it)
        assert outside.mean() >= 0.9, f"{name}: {int((~outside).sum())} of {outside.size} queries within the bound"
