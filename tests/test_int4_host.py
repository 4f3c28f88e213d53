"""Host side of the 4-bit row cache (no GPU): struct layouts against the C compiler, argument checks of the entry
points (nothing is enqueued), the layouts Python refuses, the split plan, and the oracle's own known answers."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from logitfill_amd import _native
from logitfill_amd.packed import int4
from oracle import int4 as o4

HEADER = Path(__file__).resolve().parents[1] / "include" / "logitfill_amd.h"
AT = 1 << 20  # an address (nothing reads it)


def test_struct_layouts_match_c(tmp_path):
    structs = {"lf_int4_layer": _native.Int4Layer, "lf_int4_args": _native.Int4Args}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines += ['printf("block %d\\n", LF_INT4_BLOCK_BYTES(128, 32));', "return 0;}"]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(src)], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    got = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f
    assert int(got["block"]) == int4._block_bytes(128, 32) == 32 * (128 + 32)


def _layer(**kw):
    L = _native.Int4Layer()
    L.blocks, L.bounds, L.lens, L.tops = AT, AT, AT, AT
    L.batch, L.n_kv, L.head_dim, L.cap_tokens, L.page_size, L.group = 2, 4, 128, 1024, 128, 64
    for k, v in kw.items():
        setattr(L, k, v)
    return L


def _args(**kw):
    a = _native.Int4Args()
    a.query, a.dtype, a.n_q, a.q_len, a.out = AT, _native.LF_BF16, 28, 1, AT
    a.q_strides = (ctypes.c_int64 * 3)(28 * 128, 128, 128)
    a.splits, a.split_tokens, a.workspace, a.workspace_bytes = 2, 512, AT, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


NULL, SHAPE, UNSUPPORTED, WORKSPACE, DTYPE = (_native.LF_E_NULL, _native.LF_E_SHAPE, _native.LF_E_UNSUPPORTED,
                                              _native.LF_E_WORKSPACE, _native.LF_E_DTYPE)
BAD_LAYERS = [
    ({"blocks": 0}, NULL), ({"bounds": 0}, NULL), ({"lens": 0}, NULL), ({"tops": 0}, NULL), ({"batch": 0}, SHAPE), ({"n_kv": 0}, SHAPE),
    ({"batch": 65536}, SHAPE), ({"head_dim": 96}, UNSUPPORTED), ({"head_dim": 512}, UNSUPPORTED),
    ({"group": 16}, UNSUPPORTED), ({"group": 128, "head_dim": 64}, UNSUPPORTED), ({"page_size": 48}, SHAPE),
    ({"page_size": 2048, "cap_tokens": 4096}, SHAPE), ({"page_size": 0}, SHAPE), ({"cap_tokens": 1000}, SHAPE),
    ({"cap_tokens": 0}, SHAPE), ({"blocks": AT + 8}, SHAPE), ({"bounds": AT + 2}, SHAPE),
]


@pytest.mark.parametrize("change,want", BAD_LAYERS)
def test_every_entry_point_checks_the_layer(change, want):
    lib, L = _native.load(), _layer(**change)
    s = (ctypes.c_int64 * 3)(0, 0, 0)
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, None, None, 4, None) == want
    assert lib.lf_int4_read(L, None, 4, AT, AT, 0, None) == want
    assert lib.lf_int4_attention(L, _args(), None) == want
    assert lib.lf_int4_select(L, _args(n_pages=4, pages=AT), None) == want


def test_append_and_read_refusals():
    lib, L = _native.load(), _layer()
    s = (ctypes.c_int64 * 3)(0, 0, 0)
    assert lib.lf_int4_append(None, AT, AT, 0, s, s, None, None, 4, None) == NULL
    assert lib.lf_int4_append(L, 0, AT, 0, s, s, None, None, 4, None) == NULL
    assert lib.lf_int4_append(L, AT, AT, 0, None, s, None, None, 4, None) == NULL
    assert lib.lf_int4_append(L, AT, AT, 3, s, s, None, None, 4, None) == DTYPE
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, None, None, -1, None) == SHAPE
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, None, None, 0, None) == 0
    bad = [(ctypes.c_int32 * 2)(*x) for x in ((-1, 0), (0, 5), (0, 1025))]
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, None, bad[0], 4, None) == SHAPE
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, None, bad[1], 4, None) == SHAPE
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, bad[0], None, 4, None) == SHAPE
    assert lib.lf_int4_append(L, AT, AT, 0, s, s, bad[2], None, 4, None) == SHAPE
    assert lib.lf_int4_set_lens(L, None, None) == NULL
    assert lib.lf_int4_set_lens(L, bad[0], None) == SHAPE
    assert lib.lf_int4_set_lens(L, bad[2], None) == SHAPE
    assert lib.lf_int4_read(L, bad[0], 4, AT, AT, 0, None) == SHAPE
    assert lib.lf_int4_read(L, None, 4, AT + 8, AT, 0, None) == SHAPE
    assert lib.lf_int4_read(L, None, 4, 0, 0, 0, None) == NULL
    assert lib.lf_int4_read(L, None, 4, AT, 0, -1, None) == DTYPE
    assert lib.lf_int4_read(L, None, -4, AT, 0, 0, None) == SHAPE
    assert lib.lf_int4_read(L, None, 0, AT, AT, 0, None) == 0


@pytest.mark.parametrize("change,want", [
    ({"query": 0}, NULL), ({"out": 0}, NULL), ({"out": AT + 8}, SHAPE), ({"dtype": 7}, DTYPE), ({"n_q": 27}, SHAPE), ({"n_q": 0}, SHAPE),
    ({"q_len": 0}, SHAPE), ({"q_len": 1 << 20}, SHAPE), ({"splits": 0}, SHAPE), ({"splits": 1025}, SHAPE),
    ({"split_tokens": 100}, SHAPE), ({"split_tokens": 0}, SHAPE), ({"workspace": 0}, NULL),
    ({"workspace": AT + 4}, SHAPE), ({"workspace_bytes": 100}, WORKSPACE), ({"n_pages": 4}, NULL),
    ({"n_pages": 1025, "pages": AT}, SHAPE), ({"n_pages": -1}, SHAPE),
    ({"n_pages": 4, "pages": AT, "q_len": 20000}, SHAPE),
    ({"prefix_splits": -1}, SHAPE), ({"prefix_splits": 1025}, SHAPE), ({"prefix_splits": 4}, SHAPE),
    ({"prefix_splits": 4, "splits": 1, "dtype": 1}, UNSUPPORTED), ({"prefix_splits": 4, "splits": 1, "dtype": 2}, UNSUPPORTED),
    ({"prefix_splits": 4, "splits": 1, "n_pages": 2, "pages": AT}, UNSUPPORTED),
    ({"prefix_splits": 4, "splits": 1, "workspace_bytes": 5 * 2 * 28 * 130 * 4 - 1}, WORKSPACE),
])
def test_attention_refusals(change, want):
    assert _native.load().lf_int4_attention(_layer(), _args(**change), None) == want


def test_more_rows_than_a_grid_holds():
    layer, args = _layer(batch=1 << 13), _args(q_len=64, splits=1)
    layer.n_kv, args.n_q = 32, 32
    assert _native.load().lf_int4_attention(layer, args, None) == SHAPE

    class Manager:
        batch_size, n_q, n_kv, head_dim, device = 2, 28, 4, 128, torch.device("cpu")
    for n, paged in ((40000, False), (16384, True), (0, False)):
        with pytest.raises(ValueError):
            int4._check_query(Manager, torch.empty(2, 28, n, 1, dtype=torch.bfloat16).expand(2, 28, n, 128), paged)
    Manager.batch_size = 9000
    with pytest.raises(ValueError, match="too many"):
        int4._check_query(Manager, torch.empty(1, 28, 70, 1, dtype=torch.bfloat16).expand(9000, 28, 70, 128), False)


@pytest.mark.parametrize("change,want", [
    ({"n_pages": 0}, SHAPE), ({"pages": 0}, NULL), ({"n_pages": 1025}, SHAPE), ({"workspace": 0}, NULL),
    ({"workspace_bytes": 2 * 4 * 8 * 8 - 1}, WORKSPACE), ({"q_len": 20000}, SHAPE), ({"dtype": 3}, DTYPE),
])
def test_select_refusals(change, want):
    args = _args(**{"n_pages": 4, "pages": AT, **change})
    assert _native.load().lf_int4_select(_layer(), args, None) == want


def test_workspace_sizes():
    lib = _native.load()
    assert lib.lf_int4_workspace_bytes(_layer(), 28, 1, 1) == 0
    assert lib.lf_int4_workspace_bytes(_layer(), 28, 3, 5) == 2 * 28 * 3 * 5 * 130 * 4
    assert lib.lf_int4_workspace_bytes(_layer(), 28, 3, 0) == SHAPE
    assert lib.lf_int4_workspace_bytes(None, 28, 3, 1) == SHAPE
    assert lib.lf_int4_select_workspace_bytes(_layer(), 3) == 2 * 4 * 3 * 8 * 8
    assert lib.lf_int4_select_workspace_bytes(_layer(), 0) == SHAPE


@pytest.mark.parametrize("head_dim,page,group", [(96, 128, 32), (32, 128, 32), (64, 128, 128), (128, 48, 32),
                                                 (128, 2048, 32), (128, 0, 32), (128, 128, 16)])
def test_layouts_python_refuses(head_dim, page, group):
    with pytest.raises(ValueError):
        int4.Int4KVManager(1, 4, 2, head_dim, page, group, "cuda:0")


def test_the_cache_needs_a_device():
    with pytest.raises(RuntimeError):
        int4.Int4KVManager(1, 4, 2, 128, 128, 64, "cpu")
    with pytest.raises(ValueError):
        int4.Int4KVManager(1, 5, 2, 128, 128, 64, "cuda:0")
    with pytest.raises(ValueError):
        int4.Int4KVManager(1, 4, 2, 128, 128, 64, "cuda:0", top_pages=1025)


@pytest.mark.parametrize("tokens", [1, 31, 128, 129, 1061, 8229, 65536, 262207, 1 << 24, 1 << 30])
@pytest.mark.parametrize("rows", [1, 4, 64, 1000, 100000])
def test_split_plan_covers_the_tokens(tokens, rows):
    splits, size = int4.plan_splits(tokens, rows, 256)
    assert 1 <= splits <= int4.MAX_SPLITS and size % int4.BLOCK == 0
    assert (splits - 1) * size < tokens <= splits * size


def test_oracle_known_answers():
    x = np.array([[0, 1, 2, 15] * 8, [4.0] * 32], dtype=np.float32)
    codes, scale, lo = o4.quantise(x, 32)
    assert codes[0, :4].tolist() == [0, 1, 2, 15] and scale[0, 0] == 1 and lo[0, 0] == 0
    assert not codes[1].any() and lo[1, 0] == 4
    assert np.array_equal(o4.values(x, 32)[0], x[0])
    up = o4.to_bf16_up(np.array([1.0, 1.001, -1.001, 0.0], dtype=np.float32))
    assert up.tolist() == [1.0, 1.0078125, -1.0, 0.0]
    b = np.zeros((4, 2, 2), dtype=np.float32)
    b[:, 1, 0] = [1, 3, 3, 9]
    q = np.array([[1.0, 0.0]])
    assert o4.select(q, b, 4, 2).tolist() == [1, 3] and o4.select(q, b, 3, 2).tolist() == [1, 2]
    assert o4.select(q, b, 1, 2).tolist() == [0, -1] and o4.select(q, b, 0, 2).tolist() == [-1, -1]
    v = np.eye(3)
    out = o4.attend(np.zeros((2, 3)), v, v, 1.0, np.array([[True, True, False], [False] * 3]))
    assert np.allclose(out, [[0.5, 0.5, 0], [0, 0, 0]])


def test_many_row_rule():
    """Long calls of many rows in bf16, twice as soon with groups of 32; never at head_dim 256."""
    bf16, fp16 = torch.bfloat16, torch.float16
    for args, want in (((7, 512, 4, 128, 128, bf16, [16896]), True), ((7, 32, 4, 128, 128, bf16, [16384]), False),
                       ((7, 64, 4, 128, 32, bf16, [16384]), True), ((7, 64, 4, 128, 64, bf16, [16384]), False),
                       ((7, 512, 4, 128, 32, fp16, [16896]), False), ((7, 512, 4, 128, 32, torch.float32, [16896]), False),
                       ((7, 512, 4, 256, 64, bf16, [16896]), False), ((7, 512, 4, 128, 128, bf16, [700]), False),
                       ((1, 63, 4, 128, 32, bf16, [1 << 24]), False), ((7, 512, 4, 128, 32, bf16, [0, 3]), False)):
        assert int4._many_rows(*args) is want, args
