"""Channel groups whose Values differ by powers of two: every group's output as exact as if it stood alone."""
import pytest
import torch

from logitfill_amd.packed import Int4KVManager, int4_attention, select_pages
from tests.int4_exact import exact
from tests.int4_helpers import TYPES, assert_within, query, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,group", [(64, 32), (128, 32), (128, 64), (256, 32), (256, 128)])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("ratio", [10, 20])
def test_groups_of_unlike_size(gpu, D, group, dtype, ratio):
    T, n, n_q, H, page = 500, 2, 4, 2, 32
    key, value = rows((1, H, T, D), "fp32", D + group + ratio)
    large = 2.0 ** (ratio * 0.6)
    for g in range(D // group):  # the largest group is another one in each kv head
        for h in range(H):
            value[0, h, :, g * group:(g + 1) * group] *= large if g == (h + 1) % (D // group) else large * 2.0 ** -ratio
    key, value = key.to(TYPES[dtype]), value.to(TYPES[dtype])
    q = query((1, n_q, n, D), dtype, D)
    mgr = Int4KVManager(1, n_q, H, D, page, group, gpu)
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = exact(q, key, value, [T], group, D ** -0.5, dtype)
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)
    pages = select_pages(mgr, 0, q.to(gpu), T // page)  # every page
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5, pages=pages), ref, tol)
    # a longer context, in many splits
    key, value = (torch.cat([t] * 9, 2) for t in (key, value))
    mgr.reset()
    mgr.commit(0, key.to(gpu), value.to(gpu))
    ref, tol = exact(q, key, value, [9 * T], group, D ** -0.5, dtype)
    assert_within(int4_attention(mgr, 0, q.to(gpu), None, None, D ** -0.5), ref, tol)
