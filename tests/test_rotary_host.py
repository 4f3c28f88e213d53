"""Rotary positions on the host: the frequencies of each stretching, and what is refused before anything runs (no GPU)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from logitfill_amd import _native
from logitfill_amd.packed import Rotary
from logitfill_amd.packed.rotary import frequencies


def test_plain_and_linear_frequencies():
    freq, factor = frequencies(128, 10000.0)
    assert factor == 1.0 and np.allclose(freq, 10000.0 ** (-np.arange(64) / 64), rtol=1e-15)
    slow, factor = frequencies(128, 10000.0, {"type": "linear", "factor": 4.0})
    assert factor == 1.0 and np.allclose(np.array(freq) / 4, slow, rtol=1e-15)


def test_ntk_stretches_the_slowest_pair_only():
    freq, _ = frequencies(64, 10000.0)
    ntk, _ = frequencies(64, 10000.0, {"type": "ntk", "factor": 8.0})
    assert ntk[0] == freq[0] == 1.0 and math.isclose(ntk[-1] * 8.0, freq[-1], rel_tol=1e-12)


def test_yarn_keeps_the_fast_pairs_and_stretches_the_slow_ones():
    freq, _ = frequencies(128, 1e6)
    yarn, factor = frequencies(128, 1e6, {"type": "yarn", "factor": 4.0, "original_positions": 32768})
    ratio = np.array(freq) / np.array(yarn)
    turns = np.array(freq) * 32768 / (2 * math.pi)
    assert math.isclose(factor, 0.1 * math.log(4.0) + 1)
    assert (ratio[turns > 40] == 1).all() and np.allclose(ratio[turns < 0.8], 4) and (np.diff(ratio) >= 0).all()
    assert frequencies(128, 1e6, {"type": "yarn", "factor": 4.0, "original_positions": 32768, "attention_factor": 1.0})[1] == 1.0


@pytest.mark.parametrize("args,kwargs,what", [
    ((7,), {}, "head_dim"), ((0,), {}, "head_dim"), ((514,), {}, "head_dim"),
    ((64,), {"rotary_dim": 66}, "rotary_dim"), ((64,), {"rotary_dim": 15}, "rotary_dim"), ((64,), {"rotary_dim": 0}, "rotary_dim"),
    ((64,), {"layout": "quarters"}, "layout"), ((64, 1.0), {}, "base"), ((64, float("nan")), {}, "base"),
    ((64,), {"scaling": {"type": "dynamic", "factor": 2.0}}, "type"),
    ((64,), {"scaling": {"type": "linear", "factor": 0.5}}, "factor"),
    ((64,), {"scaling": {"type": "linear", "factor": 2.0, "alpha": 1}}, "alpha"),
    ((64,), {"scaling": {"type": "yarn", "factor": 2.0}}, "original_positions"),
    ((64,), {"scaling": {"type": "ntk", "factor": 2.0}, "rotary_dim": 2}, "ntk"),
    ((64,), {"inv_freq": [1.0] * 31}, "inv_freq"), ((64,), {"inv_freq": [float("inf")] * 32}, "inv_freq"),
    ((64,), {"inv_freq": [1.0] * 32, "scaling": {"type": "linear", "factor": 2.0}}, "inv_freq"),
    ((64,), {"attention_factor": float("nan")}, "attention_factor"),
])
def test_refused_rotations(args, kwargs, what):
    with pytest.raises(ValueError, match=what):
        Rotary(*args, **kwargs)


def test_a_cpu_device():
    with pytest.raises(RuntimeError, match="ROCm device"):
        Rotary(64, device="cpu")


def _rotary(**kwargs):
    r = Rotary.__new__(Rotary)
    r.head_dim, r.rotary_dim, r.device, r._args = 64, 64, torch.device("cuda", 0), {}
    return r


def test_rows_on_the_cpu():
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        _rotary().rotate(torch.zeros(1, 2, 3, 64), None, 0)


def _args(**changes):
    a = _native.RotaryArgs()
    a.dtype, a.batch, a.tokens, a.n_q, a.n_kv, a.head_dim, a.rotary_dim, a.factor = 0, 1, 1, 1, 1, 64, 64, 1.0
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,status", [
    ({}, _native.LF_E_NULL), ({"dtype": 3}, _native.LF_E_DTYPE), ({"head_dim": 63}, _native.LF_E_SHAPE),
    ({"head_dim": 514}, _native.LF_E_SHAPE), ({"rotary_dim": 66}, _native.LF_E_SHAPE), ({"rotary_dim": 0}, _native.LF_E_SHAPE),
    ({"batch": -1}, _native.LF_E_SHAPE), ({"batch": 1 << 16, "tokens": 1 << 15}, _native.LF_E_SHAPE), ({"batch": 1 << 13, "tokens": 1 << 14}, _native.LF_E_SHAPE),
    ({"n_q": 4096}, _native.LF_E_SHAPE), ({"factor": float("inf")}, _native.LF_E_SHAPE), ({"tokens": 0}, _native.LF_OK),
    ({"start": (1 << 53) + 1}, _native.LF_E_SHAPE), ({"start": -(1 << 53) - 1}, _native.LF_E_SHAPE),
])
def test_the_c_entry_refuses(changes, status):
    assert _native.load().lf_rotary(ctypes.byref(_args(**changes)), None) == status


def test_the_c_entry_takes_no_null_arguments():
    assert _native.load().lf_rotary(None, None) == _native.LF_E_NULL
