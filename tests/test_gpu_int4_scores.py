"""Page scores that are not numbers, and scores whose products span more than float64 sums exactly."""
import numpy as np
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, select_pages
from oracle import int4 as o4
from tests.helpers import f32
from tests.int4_helpers import query, rows

pytestmark = pytest.mark.gpu


def _manager(gpu, key, value, n_q, group, page):
    B, H, _, D = key.shape
    mgr = Int4KVManager(1, n_q, H, D, page, group, gpu, batch_size=B)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    return mgr


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("g", [1, 4, 13])
@pytest.mark.parametrize("T", [700, 40000])
def test_a_nan_query_takes_the_lowest_pages(gpu, dtype, g, T):
    """NaN in one head of a kv head's group makes its every score NaN; the other kv heads, tokens and sequences keep
    their own."""
    D, group, page, H, n, top = 64, 32, 32, 2, 2, 5
    key, value = rows((2, H, T, D), dtype, g)
    mgr = _manager(gpu, key, value, g * H, group, page)
    q = query((2, g * H, n, D), dtype, g)
    want = select_pages(mgr, 0, q.to(gpu), top).cpu().numpy()
    bounds = f32(mgr.layers[0].page_bounds())
    for b in range(2):
        for h in range(H):
            for j in range(n):
                own = (T - n + j) // page
                assert np.array_equal(want[b, h, j], o4.select(f32(q)[b, h * g:(h + 1) * g, j], bounds[b, h], own, top))
    q[1, g * H - 1, 0, 17] = float("nan")
    want[1, 1, 0] = np.arange(top)
    assert np.array_equal(select_pages(mgr, 0, q.to(gpu), top).cpu().numpy(), want)
    q[:] = float("nan")
    want[:] = np.arange(top)
    assert np.array_equal(select_pages(mgr, 0, q.to(gpu), top).cpu().numpy(), want)


def test_infinities_in_a_query(gpu):
    """A page whose bounds make an infinite score comes first, one of infinities of both signs counts as NaN and last."""
    D, page = 64, 32
    key = torch.zeros(1, 1, 8 * page + 1, D)
    key += 1
    key[0, 0, 3 * page:4 * page, 0] = -1
    key[0, 0, 5 * page:6 * page, 0] = -1
    key[0, 0, 5 * page:6 * page, 1] = -1
    mgr = _manager(gpu, key, key, 1, 64, page)
    q = torch.ones(1, 1, 1, D)
    q[..., 0] = -float("inf")  # scores: -inf, at pages 3 and 5 +inf
    assert select_pages(mgr, 0, q.to(gpu), 2)[0, 0, 0].tolist() == [3, 5]
    q[..., 1] = float("inf")   # NaN: all but page 3, +inf (page 5: +inf - inf)
    assert select_pages(mgr, 0, q.to(gpu), 3)[0, 0, 0].tolist() == [0, 1, 3]


def test_float32_queries_of_a_wide_span(gpu):
    """Queries over 2^17 and bounds over 2^8: sums that float64 rounds.  Pages whose scores lie further apart than that
    rounding, 64 sums of 2^-53 of sum |q bound|, are chosen as by the exact scores."""
    D, group, page, T, top = 128, 64, 32, 6000, 20
    g = torch.Generator().manual_seed(7)
    key, value = rows((1, 1, T, D), "fp32", 7)
    q = torch.randn(1, 2, 1, D, generator=g) * torch.exp2(torch.randint(-17, 0, (D,), generator=g).float())
    mgr = _manager(gpu, key, value, 2, group, page)
    bounds = f32(mgr.layers[0].page_bounds())[0, 0]
    own = (T - 1) // page
    from fractions import Fraction

    def score(head, p):
        return sum(max(Fraction(float(a)) * Fraction(float(lo)), Fraction(float(a)) * Fraction(float(hi)))
                   for a, lo, hi in zip(f32(q)[0, head, 0], *bounds[p]))
    scores = [max(score(i, p) for i in range(2)) for p in range(own)]
    order = sorted(range(own), key=lambda p: (-scores[p], p))
    gap = scores[order[top - 1]] - scores[order[top]]
    size = max(float((np.abs(f32(q)[0, :, 0]).astype(np.float64) @ np.abs(bounds[p]).max(0).astype(np.float64)).max()) for p in range(own))
    assert float(gap) > 2 * D * 2.0 ** -53 * size
    assert select_pages(mgr, 0, q.to(gpu), top)[0, 0, 0].tolist() == sorted(order[:top])
