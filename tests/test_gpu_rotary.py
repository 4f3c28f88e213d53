"""Rotary positions on the device against float64: layouts, parts of a head, types, strides, odd sizes, far positions,
streams and captured graphs."""
import math

import numpy as np
import pytest
import torch

from logitfill_amd.packed import Rotary
from tests.helpers import f32

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def expected(x, positions, rot):
    """Float64 rows and their bound: the output's rounding; sine, cosine and factor rounded to float32, two products
    and a sum, 2^-24 each of |x| + |y|; the angle's float64 steps; fp16's least step."""
    x = f32(x).astype(np.float64)
    R = rot.rotary_dim
    angle = np.asarray(positions, dtype=np.float64)[:, None, :, None] * np.array(rot.inv_freq)
    cos, sin = np.cos(angle) * rot.attention_factor, np.sin(angle) * rot.attention_factor
    one, two = (slice(0, R // 2), slice(R // 2, R)) if rot.layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    out, tol = x.copy(), np.zeros(x.shape)
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * cos - b * sin, b * cos + a * sin
    size = (np.abs(a) + np.abs(b)) * abs(rot.attention_factor)
    tol[..., one] = tol[..., two] = size * (4 * 2.0 ** -24 + 4 * np.abs(angle) * 2.0 ** -53)
    return out, tol


def check(ours, x, positions, rot, dtype):
    want, tol = expected(x, positions, rot)
    rotated = np.abs(f32(ours).astype(np.float64) - want)
    tol = tol + HALF_STEP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "fp16" else 0)
    assert (rotated <= tol).all(), f"worst {(rotated / np.maximum(tol, 1e-300)).max():.3g} x the bound"
    R = rot.rotary_dim
    assert torch.equal(ours[..., R:].cpu(), x[..., R:].cpu())  # the rest passes through


def rows(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (128, 32), (64, 16), (256, 192), (80, 80), (96, 20), (2, 2), (512, 512), (10, 6)])
def test_layouts(gpu, D, R, layout, dtype):
    rot = Rotary(D, 10000.0, rotary_dim=R, layout=layout, device=gpu)
    q, k = rows((2, 5, 37, D), dtype, D + R), rows((2, 3, 37, D), dtype, D + R + 1)
    positions = torch.arange(37) + torch.tensor([[0], [1000]])
    oq, ok = rot.rotate(q.to(gpu), k.to(gpu), positions.to(gpu))
    check(oq, q, positions, rot, dtype)
    check(ok, k, positions, rot, dtype)
    # a projection's order: tokens outermost; the outputs keep it
    qt, kt = (t.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for t in (q, k))
    tq, tk = rot.rotate(qt, kt, positions.int().to(gpu))
    assert torch.equal(tq, oq) and torch.equal(tk, ok) and tq.stride() == qt.stride()


@pytest.mark.parametrize("B,T,n_q,n_kv", [(1, 1, 1, 1), (8, 1, 12, 2), (1, 3, 1, 0), (3, 1025, 2, 1), (1, 4099, 7, 1), (5, 0, 2, 2)])
def test_sizes(gpu, B, T, n_q, n_kv):
    rot = Rotary(128, 1e6, scaling={"type": "yarn", "factor": 4.0, "original_positions": 4096}, device=gpu)
    q, k = rows((B, n_q, T, 128), "bf16", T), rows((B, n_kv, T, 128), "bf16", T + 1)
    oq, ok = rot.rotate(q.to(gpu), k.to(gpu) if n_kv else None, 17)
    positions = np.broadcast_to(17 + np.arange(T), (B, T))
    check(oq, q, positions, rot, "bf16")
    if n_kv:
        check(ok, k, positions, rot, "bf16")
    else:
        assert ok is None


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_far_and_unordered_positions(gpu, dtype):
    """2^31 and beyond lose nothing: angles are formed in float64."""
    rot = Rotary(64, 5e5, device=gpu)
    positions = torch.tensor([[0, 1, 2 ** 20 + 1, 2 ** 31 + 5, 3, 3, -7, 10 ** 9]])
    q = rows((1, 4, 8, 64), dtype, 3)
    oq, _ = rot.rotate(q.to(gpu), None, positions.to(gpu))
    check(oq, q, positions, rot, dtype)
    every = rot.rotate(q.to(gpu), None, positions[0].to(gpu))[0]
    assert torch.equal(every, oq)
    near = positions.clamp(max=2 ** 30).int()
    check(rot.rotate(q.to(gpu), None, near.to(gpu))[0], q, near, rot, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_strides_and_alignment(gpu, dtype):
    """Views of one fused projection, rows that start off 16 bytes, broadcast heads, another channel order."""
    rot = Rotary(64, device=gpu)
    positions = torch.arange(19)[None]
    for off in (0, 1, 3):
        fused = rows((1, 19, (4 + 2 + 2) * 64 + off), dtype, 5 + off).to(gpu)[..., off:]
        q = fused[..., : 4 * 64].unflatten(-1, (4, 64)).transpose(1, 2)
        k = fused[..., 4 * 64 : 6 * 64].unflatten(-1, (2, 64)).transpose(1, 2)
        oq, ok = rot.rotate(q, k, positions.to(gpu))
        check(oq, q.cpu(), positions, rot, dtype)
        check(ok, k.cpu(), positions, rot, dtype)
    one = rows((1, 1, 19, 64), dtype, 9).to(gpu)
    oq, _ = rot.rotate(one.expand(1, 5, 19, 64), None, positions.to(gpu))
    check(oq, one.expand(1, 5, 19, 64).cpu(), positions, rot, dtype)
    odd = rows((1, 64, 19, 3), dtype, 10).to(gpu).transpose(1, 3)  # channels outermost
    check(rot.rotate(odd, None, 0)[0], odd.cpu(), positions, rot, dtype)
    every_other = rows((1, 2, 38, 64), dtype, 11).to(gpu)[:, :, ::2]
    check(rot.rotate(every_other, None, positions[0].repeat_interleave(2).to(gpu)[::2])[0], every_other.cpu(), positions, rot, dtype)


def test_a_model_s_own_frequencies_and_infinities(gpu):
    inv = [0.5 ** i for i in range(32)]
    rot = Rotary(64, inv_freq=torch.tensor(inv), attention_factor=1.25, device=gpu)
    q = rows((1, 2, 9, 64), "fp32", 1)
    check(rot.rotate(q.to(gpu), None, 100)[0], q, 100 + np.arange(9)[None], rot, "fp32")
    q[0, 0, 3, 5] = math.inf
    q[0, 1, 4, 6] = math.nan
    out = rot.rotate(q.to(gpu), None, 0)[0].cpu()
    bad = ~torch.isfinite(out)
    assert bad.sum() == 4 and bad[0, 0, 3, [5, 37]].all() and bad[0, 1, 4, [6, 38]].all()


def test_another_stream_and_a_captured_graph(gpu):
    rot = Rotary(128, device=gpu)
    q, k = rows((2, 4, 50, 128), "bf16", 1).to(gpu), rows((2, 2, 50, 128), "bf16", 2).to(gpu)
    positions = torch.arange(50, device=gpu)
    want = rot.rotate(q, k, positions)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rot.rotate(q, k, positions)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rot.rotate(q, k, positions)
    for step in range(3):
        positions += 7
        graph.replay()
        again = rot.rotate(q, k, positions)
        torch.cuda.synchronize()
        assert torch.equal(captured[0], again[0]) and torch.equal(captured[1], again[1])


def test_more_tokens_than_one_token_workgroups(gpu):
    """2^24 tokens and more of wide rows: a grid holds 2^32 threads."""
    T, D = (1 << 24) + 5, 258
    rot = Rotary(D, device=gpu)
    x = torch.ones(1, 1, T, D, dtype=torch.bfloat16, device=gpu)
    out, _ = rot.rotate(x, None, 7)
    for at in (0, T // 2, T - 3):
        check(out[:, :, at : at + 3], x[:, :, at : at + 3].cpu(), torch.arange(at + 7, at + 10)[None], rot, "bf16")


def test_refused_calls(gpu):
    rot = Rotary(64, device=gpu)
    q, k = torch.zeros(2, 4, 5, 64, device=gpu), torch.zeros(2, 2, 5, 64, device=gpu)
    for bad, error in ((lambda: rot.rotate(q[..., :32], None, 0), ValueError), (lambda: rot.rotate(q, k[:1], 0), ValueError),
                       (lambda: rot.rotate(q, k[:, :, :4], 0), ValueError), (lambda: rot.rotate(q, k.half(), 0), TypeError),
                       (lambda: rot.rotate(q[0], None, 0), ValueError), (lambda: rot.rotate(q.double(), None, 0), TypeError),
                       (lambda: rot.rotate(q, k, torch.arange(5.0, device=gpu)), TypeError),
                       (lambda: rot.rotate(q, k, torch.arange(4, device=gpu)), ValueError),
                       (lambda: rot.rotate(q, k, torch.zeros(3, 5, dtype=torch.int32, device=gpu)), ValueError),
                       (lambda: rot.rotate(q, k, torch.arange(5)), ValueError),
                       (lambda: rot.rotate(q, k, 1.5), TypeError), (lambda: rot.rotate(q, k, 1 << 70), ValueError),
                       (lambda: rot.rotate(q, k, -(1 << 53) - 1), ValueError),
                       (lambda: rot.rotate(q.clone().requires_grad_(), k, 0), RuntimeError)):
        with pytest.raises(error):
            bad()
    with torch.no_grad():
        rot.rotate(q.clone().requires_grad_(), k, 0)
