"""The prompt attention's work list and its refusals on the host (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from logitfill_amd import _native
from logitfill_amd.packed import LogitFillCache, PromptPlan, prompt_attention
from logitfill_amd.packed.prompt import key_tile, tile_rows, work_items


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("rows,D,dtype", [(32, 64, torch.bfloat16), (128, 128, torch.float16), (128, 64, torch.float32)])
def test_every_row_tile_s_keys_are_covered_once(seed, rows, D, dtype):
    keys = key_tile(D, dtype)
    rng = np.random.default_rng(seed)
    B, g, n_kv = int(rng.integers(1, 7)), int(rng.integers(1, 9)), int(rng.integers(1, 9))
    n = rng.integers(0, 700, B)
    m = np.maximum(0, n + rng.integers(-20, 4000, B))
    packed = bool(seed % 2)
    items, (n_items, n_merges, slots), groups = work_items(n, m, packed, not packed, g, rows, D, dtype, n_kv, 256)
    items, merges = items[:n_items], items[n_items:]
    assert len(merges) == n_merges and groups in (1, 2)
    assert (np.diff(items[:, 8] - items[:, 7]) <= 0).all()  # the longest first
    assert sorted(items[items[:, 9] >= 0, 9]) == list(range(slots))
    by_tile = {}
    for x in items:
        b = int(x[3])  # (packed queries: Keys are padded, and the other way about)
        if not packed:
            b = int(x[0])
        assert (x[2], x[5]) == (n[b], m[b])
        assert (x[0], x[1]) == ((0, n[:b].sum()) if packed else (b, 0))
        assert (x[3], x[4]) == ((b, 0) if packed else (0, m[:b].sum()))
        by_tile.setdefault((b, int(x[6])), []).append(x)
    assert len(by_tile) == sum(-(-int(k) * g // rows) for k in n)
    divided = {(int(x[0] if not packed else x[3]), int(x[6])): x for x in merges}
    for (b, t), parts in by_tile.items():
        parts.sort(key=lambda x: x[7])
        seen = max(0, m[b] - n[b] + min((t * rows + rows - 1) // g, n[b] - 1) + 1)
        assert parts[0][7] == 0 and parts[-1][8] == -(-seen // keys)
        assert all(x[8] == y[7] for x, y in zip(parts, parts[1:]))
        if len(parts) == 1:
            assert parts[0][9] == -1 and (b, t) not in divided
        else:
            assert [x[9] for x in parts] == list(range(parts[0][9], parts[0][9] + len(parts)))
            assert all(x[8] > x[7] for x in parts)
            assert (divided[b, t][9], divided[b, t][10]) == (parts[0][9], len(parts))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths,tokens", [([3, 0, 40], 50), ([7], 7), ([0, 0], 3), ([300, 299], 1000)])
def test_rows_behind_the_sequences_are_zeros_of_their_own(packed, lengths, tokens):
    g, rows = 3, 32
    items, (n_items, _, _), _ = work_items(lengths, [n + 5 for n in lengths], packed, False, g, rows, 64, torch.bfloat16, 2, 256, tokens)
    items = items[:n_items]
    written = np.zeros((1 if packed else len(lengths), tokens), dtype=int)
    for q_row, start, n, k_row, k_start, m, tile, begin, end, slot, parts, _ in items:
        if begin:
            continue
        for r in range(tile * rows, min((tile + 1) * rows, n * g)):
            if r % g == 0:
                written[q_row, start + r // g] += 1
                inside = start < sum(lengths) if packed else start < lengths[q_row]
                assert inside == (m > 0) and (inside or (begin, end, slot) == (0, 0, -1))
    assert (written == 1).all()


def test_long_keys_of_few_rows_are_divided():
    items, counts, groups = work_items([1], [32768], True, True, 4, 32, 128, torch.bfloat16, 4, 256)
    assert max(items[:, 8] - items[:, 7]) < 64 and counts == (len(items) - 1, 1, len(items) - 1) and groups == 1
    items, counts, groups = work_items([4096] * 64, [16384] * 64, True, True, 8, 128, 128, torch.bfloat16, 8, 256)
    assert counts == (64 * 256, 0, 0) and groups == 1  # enough row tiles
    assert tile_rows([1, 4], 8) == 32 and tile_rows([5], 8) == 128


@pytest.mark.parametrize("lengths,keys", [([], None), ([3, -1], None), ([3], [3, 4]), ([1 << 25], None), ([1], [1 << 25])])
def test_refused_plans(lengths, keys):
    with pytest.raises(ValueError):
        PromptPlan(lengths, keys)


def test_the_cpu():
    with pytest.raises(RuntimeError, match="ROCm device"):
        PromptPlan([3], device="cpu")
    t = torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        prompt_attention(t, t, t, 0.1)
    with pytest.raises(ValueError, match="finite"):
        prompt_attention(t, t, t, float("nan"))


def _args(**changes):
    a = _native.PromptArgs()
    a.dtype, a.n_q, a.n_kv, a.head_dim, a.scaling, a.tile_rows, a.groups, a.n_items = 0, 4, 2, 64, 0.1, 128, 1, 1
    for name in ("query", "key", "value", "out", "items"):
        setattr(a, name, 4096)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 3}, _native.LF_E_DTYPE), ({"head_dim": 96}, _native.LF_E_UNSUPPORTED), ({"n_q": 3}, _native.LF_E_SHAPE),
    ({"n_kv": 0}, _native.LF_E_SHAPE), ({"n_items": -1}, _native.LF_E_SHAPE), ({"tile_rows": 64}, _native.LF_E_SHAPE),
    ({"groups": 0}, _native.LF_E_SHAPE), ({"groups": 2, "tile_rows": 32}, _native.LF_E_SHAPE), ({"groups": 2, "dtype": 2}, _native.LF_E_SHAPE),
    ({"groups": 2, "head_dim": 256}, _native.LF_E_SHAPE),
    ({"n_items": 1 << 30, "n_kv": 2}, _native.LF_E_SHAPE), ({"n_items": 1 << 23}, _native.LF_E_SHAPE),
    ({"n_merges": 1 << 23, "merges": 4096, "n_slots": 1 << 24}, _native.LF_E_SHAPE), ({"n_items": 1 << 25, "tile_rows": 32}, _native.LF_E_SHAPE),
    ({"n_items": 1 << 22, "groups": 2}, _native.LF_E_SHAPE), ({"scaling": float("nan")}, _native.LF_E_SHAPE),
    ({"scaling": float("inf")}, _native.LF_E_SHAPE), ({"n_items": 0}, _native.LF_OK), ({"query": None}, _native.LF_E_NULL),
    ({"out": None}, _native.LF_E_NULL), ({"items": None}, _native.LF_E_NULL), ({"n_merges": 1}, _native.LF_E_NULL),
    ({"n_merges": 1, "merges": 4096}, _native.LF_E_SHAPE), ({"n_merges": 2, "merges": 4096, "n_slots": 3}, _native.LF_E_SHAPE),
    ({"key": 4098}, _native.LF_E_SHAPE), ({"n_slots": 2}, _native.LF_E_NULL),
    ({"n_slots": 2, "workspace": 4100}, _native.LF_E_SHAPE), ({"n_slots": 2, "workspace": 4096, "workspace_bytes": 2 * 2 * 128 * 66 * 4 - 1}, _native.LF_E_WORKSPACE),
])
def test_the_c_entry_refuses(changes, status):
    assert _native.load().lf_prompt_attention(ctypes.byref(_args(**changes)), None) == status


def test_strides_off_16_bytes_and_null_arguments():
    lib = _native.load()
    a = _args()
    a.v_strides[2] = 68
    assert lib.lf_prompt_attention(ctypes.byref(a), None) == _native.LF_E_SHAPE
    assert lib.lf_prompt_attention(None, None) == _native.LF_E_NULL
    assert lib.lf_prompt_workspace_bytes(2, 64, 128, 2) == 2 * 2 * 128 * 66 * 4
    assert lib.lf_prompt_workspace_bytes(0, 64, 128, 2) == _native.LF_E_SHAPE


class _Layer:
    def __init__(self, lengths):
        self.lengths = list(lengths)


class _Shared:
    """What the transformers view sees of an ``Int4KVManager`` behind a prefix."""

    def __init__(self, before, lengths):
        self.layers, self.before = [_Layer(lengths)], before
        self.prefix = type("_Prefix", (), {"seq_len": before[0]})()

    seq_len = property(lambda self: self.layers[0].lengths[0])

    def prefix_lengths(self, layer_idx):
        return list(self.before)

    def truncate(self, lengths):
        self.layers[0].lengths = list(lengths)


@pytest.mark.parametrize("before,lengths,crop,want", [
    ([0, 5], [4, 4], 7, [4, 2]), ([5, 0], [4, 4], 7, [2, 4]), ([0, 5], [4, 4], -4, [0, 0]), ([0, 0], [4, 3], 2, [2, 2]), ([0, 5], [4, 4], 3, None),
    ([6, 6], [1, 4], -2, None), ([6, 6], [1, 4], 6, [0, 0]),
])
def test_crops_behind_prefixes_of_unlike_lengths(before, lengths, crop, want):
    mgr = _Shared(before, lengths)
    cache = LogitFillCache(mgr)
    assert cache.get_seq_length() == before[0] + lengths[0]
    if want is None:
        with pytest.raises(ValueError, match="shared prefix"):
            cache.crop(crop)
    else:
        cache.crop(crop)
    assert mgr.layers[0].lengths == (lengths if want is None else want)


def _batch(lengths=(5, 7), key_lengths=(9, 7), **changes):
    n, m = np.array(lengths, dtype=np.int32), np.array(key_lengths, dtype=np.int32)
    b = _native.PromptBatch(n.ctypes.data, m.ctypes.data, len(n), 1, 1, 0, 4, 2, 64, 0, 128, 256)
    for name, value in changes.items():
        setattr(b, name, value)
    return b, (n, m)


@pytest.mark.parametrize("changes,status", [
    ({"lengths": None}, _native.LF_E_NULL), ({"key_lengths": None}, _native.LF_E_NULL), ({"dtype": 3}, _native.LF_E_DTYPE),
    ({"head_dim": 96}, _native.LF_E_UNSUPPORTED), ({"batch": 0}, _native.LF_E_SHAPE), ({"tokens": -1}, _native.LF_E_SHAPE),
    ({"group": 0}, _native.LF_E_SHAPE), ({"n_kv": 0}, _native.LF_E_SHAPE), ({"compute_units": 0}, _native.LF_E_SHAPE),
    ({"tile_rows": 64}, _native.LF_E_SHAPE), ({"group": 1 << 29}, _native.LF_E_SHAPE), ({"tokens": 1 << 30}, _native.LF_E_SHAPE),
])
def test_the_planner_refuses(changes, status):
    b, kept = _batch(**{k: v for k, v in changes.items() if v is not None})
    for name in (k for k, v in changes.items() if v is None):
        setattr(b, name, None)
    lib, split, counts = _native.load(), (ctypes.c_int32 * 2)(), (ctypes.c_int32 * 3)()
    assert lib.lf_prompt_split(b, split) == status and lib.lf_prompt_items(b, 4, None, 0, counts) == status
    for lengths in ((-1, 4), ((1 << 24) + 1, 4)):
        b, kept = _batch(lengths)
        assert lib.lf_prompt_split(b, split) == _native.LF_E_SHAPE
    b, kept = _batch()
    assert lib.lf_prompt_split(b, None) == lib.lf_prompt_items(b, 4, None, 9, counts) == _native.LF_E_NULL
    assert lib.lf_prompt_split(None, split) == lib.lf_prompt_items(b, 4, None, 0, None) == _native.LF_E_NULL
    assert lib.lf_prompt_items(b, 0, None, 0, counts) == _native.LF_E_SHAPE


def test_the_planner_writes_what_fits_only():
    b, kept = _batch((300, 7), (900, 7))
    lib, counts = _native.load(), (ctypes.c_int32 * 3)()
    assert lib.lf_prompt_items(b, 4, None, 0, counts) == _native.LF_E_WORKSPACE
    n = counts[0] + counts[1]
    assert counts[1] > 0 and counts[2] >= 2 * counts[1]
    items = np.full((n + 1, 12), -7, dtype=np.int32)
    assert lib.lf_prompt_items(b, 4, items.ctypes.data, n - 1, counts) == _native.LF_E_WORKSPACE and (items == -7).all()
    assert lib.lf_prompt_items(b, 4, items.ctypes.data, n, counts) == _native.LF_OK
    assert (items[n] == -7).all() and (items[:n, 2] > 0).all()
