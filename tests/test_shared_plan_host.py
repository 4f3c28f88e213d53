"""The split plans of shared prefixes (host logic, no GPU): a row's parts, of the prefix and of the sequence's own rows, stay
within what the entry point takes."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from logitfill_amd.packed import int4


def parts(heads, D, group, common, own, q_len=1, dtype=torch.bfloat16):
    """``(prefix's splits, own splits, many-row prefix, tokens covered)`` of a call, as ``int4_attention`` plans it."""
    n_q, n_kv = heads
    layer = [SimpleNamespace(lengths=list(n)) for n in (common, own)]
    prefix = SimpleNamespace(layers=layer[:1], batch_size=len(common))
    manager = SimpleNamespace(n_q=n_q, n_kv=n_kv, head_dim=D, group_size=group, batch_size=len(own), layers=layer[1:], prefix=prefix)
    (splits, size, many), (mine, tokens) = int4._shared_plan(manager, 0, q_len, dtype, None, 256)
    if int4._many_rows(n_q // n_kv, q_len, n_kv, D, group, dtype, own):
        mine, tokens = 1, max(own)  # (its own rows in even shares, whose number is cut to half of the most)
        splits += int4.MAX_SPLITS // 2
    assert size % int4.BLOCK == 0 and tokens * mine >= max(own)
    return splits, mine, many


@pytest.fixture(autouse=True)
def no_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


@pytest.mark.parametrize("heads,D,group,common,own", [
    ((8, 1), 128, 32, [262144], [98304] + [100] * 15),
    ((16, 1), 128, 32, [96769], [108643] + [900] * 15),
    ((16, 1), 64, 32, [131072], [200000] + [5] * 63),
])
def test_one_long_sequence_among_short_ones(heads, D, group, common, own):
    splits, mine, many = parts(heads, D, group, common, own)
    assert many and splits + mine <= int4.MAX_SPLITS + 1


@pytest.mark.parametrize("seed", range(200))
def test_ragged_lengths(seed):
    rng = np.random.default_rng(seed)
    D = int(rng.choice([64, 128]))
    group = int(rng.choice([g for g in (32, 64, 128) if g <= D]))
    n_kv = int(rng.choice([1, 2, 4, 8]))
    heads = n_kv * int(rng.integers(1, 17)), n_kv
    prefixes, each = int(rng.integers(1, 5)), int(rng.integers(1, 65))
    draw = lambda n, top: [int(x) for x in np.exp(rng.uniform(0, np.log(top), n))]
    common, own = draw(prefixes, 1 << 20), draw(prefixes * each, 1 << int(rng.integers(1, 20)))
    own[int(rng.integers(len(own)))] = draw(1, 1 << 20)[0]
    for dtype in (torch.bfloat16, torch.float16):
        for q_len in (1, int(rng.integers(1, 9))):
            splits, mine, _ = parts(heads, D, group, common, own, q_len, dtype)
            assert 1 <= splits and 1 <= mine and splits + mine <= int4.MAX_SPLITS + 1, (heads, common, own, q_len)


@pytest.mark.parametrize("most", [1, 3, 513, 1024])
@pytest.mark.parametrize("tokens", [(1,), (65536, 1), (131073,) * 3, (1 << 30, 5)])
def test_a_plan_s_most_splits(tokens, most):
    splits, size = int4.plan_splits(tokens, 4, 256, most=most)
    assert 1 <= splits <= most and (splits - 1) * size < max(tokens) <= splits * size
