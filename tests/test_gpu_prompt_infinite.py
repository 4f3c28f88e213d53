"""A Value that is not finite in a row's sight counts whatever its weight: zero times infinity is NaN wherever the Key falls, in a
tile that a wave sees whole, in a masked one, or in a part of divided Keys."""
import numpy as np
import pytest
import torch

from logitfill_amd.packed import PromptPlan, prompt, prompt_attention
from tests.helpers import f32
from tests.prompt_helpers import assert_within, attend, inputs

pytestmark = pytest.mark.gpu

SPLITS = [None, (1, 1), (3, 1), (1000, 2), (2, 2)]


def check(gpu, monkeypatch, split, D, dtype, T, hidden, value):
    """``hidden``: Keys whose weight is zero; the last one's Value is not finite in channel 3."""
    if split is not None:
        monkeypatch.setattr(prompt, "split_size", lambda *args: split if D <= 128 and dtype != "fp32" else (split[0], 1))
    q, k, v = inputs((1, 2, T, D), (1, 1, T, D), dtype, 21)
    q[..., 3] = q[..., 3].abs() + 0.5
    k[0, 0, hidden] = 0
    # scores of -60 000 / 2 / 16 at most (exp(-1 875) is zero in float64, too), or of minus infinity
    k[0, 0, hidden, 3] = value
    kn, vn = (f32(t)[0, 0].astype(np.float64) for t in (k, v))
    kn[hidden] = 0
    at = hidden[-1]
    v[0, 0, at, 3] = float("inf")
    out = prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), D ** -0.5, PromptPlan([T], device=gpu)).cpu()
    seen = np.tril(np.ones((T, T), dtype=bool))
    seen[:, hidden] = False
    for h in range(2):
        ref, tol = attend(f32(q)[0, h].astype(np.float64), kn, vn, D ** -0.5, seen, dtype)
        mine = out[0, h].clone()
        assert not torch.isfinite(mine[at:, 3]).any(), f"rows {torch.nonzero(torch.isfinite(mine[at:, 3])).flatten()[:8] + at}"
        mine[at:, 3] = 0
        ref[at:, 3] = 0
        assert_within(mine, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("split", SPLITS)
def test_weights_that_underflow(gpu, monkeypatch, split, D, dtype):
    """Seen whole by the last rows' waves, masked for its neighbours'; beside another row's Value that makes a masked tile odd."""
    check(gpu, monkeypatch, split, D, dtype, 300, [40], -60000.0)
    check(gpu, monkeypatch, split, D, dtype, 300, [290], -60000.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("split", SPLITS)
def test_parts_without_a_weight(gpu, monkeypatch, split, D, dtype):
    """A tile all of whose scores are minus infinity: a part of its own where the Keys are divided so."""
    check(gpu, monkeypatch, split, D, dtype, 300, list(range(64, 128)), -float("inf"))
