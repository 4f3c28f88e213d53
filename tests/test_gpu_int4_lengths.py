"""Lengths that the host sets (truncate, reset) reach the device in their place: before replays on the same stream, and
before calls on any other."""
import threading

import pytest
import torch

from logitfill_amd.packed import Int4KVManager, int4_attention
from tests.int4_exact import exact
from tests.int4_helpers import assert_within, query, rows

pytestmark = pytest.mark.gpu
D, GROUP, PAGE, N_Q, H = 128, 64, 32, 4, 2


def _busy(gpu):
    """Some 20 ms of work on the current stream."""
    a = torch.ones(8192, 8192, dtype=torch.bfloat16, device=gpu)
    for _ in range(16):
        a = torch.matmul(a, a)


@pytest.mark.parametrize("how", ["truncate", "reset"])
def test_the_second_stream_after_a_truncation(gpu, how):
    """The stream of the truncation is busy; a call there, then one on another stream: both over the rows that are left."""
    key, value = rows((2, H, 500, D), "bf16", 21)
    q = query((2, N_Q, 1, D), "bf16", 21)
    dq = q.to(gpu)
    mgr = Int4KVManager(2, N_Q, H, D, PAGE, GROUP, gpu, batch_size=2, capacity_tokens=512)
    for layer in range(2):
        mgr.commit(layer, key.to(gpu), value.to(gpu), [500, 411])
    left = [77, 300] if how == "truncate" else [0, 0]
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        _busy(gpu)
        mgr.truncate(left) if how == "truncate" else mgr.reset()
        outs = [int4_attention(mgr, 0, dq, None, None, D ** -0.5)]
    with torch.cuda.stream(second):
        outs += [int4_attention(mgr, layer, dq, None, None, D ** -0.5) for layer in range(2)]
        k, v = mgr.layers[1].read(0, 500)
    torch.cuda.synchronize()
    ref, tol = exact(q, key, value, left, GROUP, D ** -0.5, "bf16")
    for out in outs:
        assert_within(out, ref, tol)
    assert not k[0, :, left[0]:].any() and not v[1, :, left[1]:].any()
    assert mgr.layers[0]._lens.tolist() == mgr.layers[1]._lens.tolist() == left


def test_streams_that_take_turns(gpu):
    """Truncations on one busy stream and calls on another, append and attention, a layer each, again and again."""
    T = 300
    key, value = rows((1, H, 400, D), "bf16", 24)
    k, v = key.to(gpu), value.to(gpu)
    q = query((1, N_Q, 1, D), "bf16", 24)
    dq = q.to(gpu)
    mgr = Int4KVManager(3, N_Q, H, D, PAGE, GROUP, gpu, capacity_tokens=512)
    for layer in range(3):
        mgr.commit(layer, k[:, :, :T], v[:, :, :T])
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for left in (200, 100, 37):
        with torch.cuda.stream(first):
            first.wait_stream(second)
            _busy(gpu)
            mgr.truncate(left)
            mgr.commit(0, k[:, :, 350:352], v[:, :, 350:352])
        with torch.cuda.stream(second):
            outs = [int4_attention(mgr, layer, dq, None, None, D ** -0.5) for layer in (1, 0)]
            mgr.commit(2, k[:, :, 360:361], v[:, :, 360:361])
            outs.append(int4_attention(mgr, 2, dq, None, None, D ** -0.5))
        torch.cuda.synchronize()
        assert [layer.lengths for layer in mgr.layers] == [[left + 2], [left], [left + 1]]
        assert mgr._lens.rows.tolist() == [[left + 2], [left], [left + 1]]
        for out, more in zip(outs, ([], [350, 351], [360])):
            at = list(range(left)) + more
            ref, tol = exact(q, key[:, :, at], value[:, :, at], [len(at)], GROUP, D ** -0.5, "bf16")
            assert_within(out, ref, tol)
        mgr.truncate(left)


def test_threads_with_a_layer_and_a_stream_each(gpu):
    """After a truncation one thread appends to its layer while others read theirs; the streams have waited for it."""
    T, L = 120, 4
    key, value = rows((1, H, 200, D), "bf16", 25)
    k, v = key.to(gpu), value.to(gpu)
    q = query((1, N_Q, 1, D), "bf16", 25)
    dq = q.to(gpu)
    mgr = Int4KVManager(L, N_Q, H, D, PAGE, GROUP, gpu, capacity_tokens=256)
    for layer in range(L):
        mgr.commit(layer, k[:, :, :T], v[:, :, :T])
    streams = [torch.cuda.Stream() for _ in range(L)]
    torch.cuda.synchronize()
    for left in range(100, 60, -2):
        with torch.cuda.stream(streams[0]):
            mgr.truncate(left)
        outs, failed = [None] * L, []
        start = threading.Barrier(L)

        def work(i):
            try:
                with torch.cuda.stream(streams[i]):
                    start.wait(30)
                    if i % 2 == 0:
                        mgr.commit(i, k[:, :, 150:153], v[:, :, 150:153])
                    outs[i] = int4_attention(mgr, i, dq, None, None, D ** -0.5)
                streams[i].synchronize()
            except Exception as e:  # (a thread's error is not the test's by itself)
                failed.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(L)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert not failed, failed
        torch.cuda.synchronize()
        want = [[left + 3 if i % 2 == 0 else left] for i in range(L)]
        assert [layer.lengths for layer in mgr.layers] == want and mgr._lens.rows.tolist() == want
        for i in range(L):
            at = list(range(left)) + ([150, 151, 152] if i % 2 == 0 else [])
            ref, tol = exact(q, key[:, :, at], value[:, :, at], [len(at)], GROUP, D ** -0.5, "bf16")
            assert_within(outs[i], ref, tol)


def test_a_replay_after_a_truncation(gpu):
    """Rejected tokens are taken back between replays of one captured step, with no other call."""
    T = 60
    key, value = rows((1, H, 100, D), "bf16", 22)
    k, v = key.to(gpu), value.to(gpu)
    mgr = Int4KVManager(2, N_Q, H, D, PAGE, GROUP, gpu, capacity_tokens=128)
    q = query((1, N_Q, 1, D), "bf16", 22)
    dq, step_k, step_v = q.to(gpu), k[:, :, :1].clone(), v[:, :, :1].clone()
    for layer in range(2):
        mgr.commit(layer, k[:, :, :T], v[:, :, :T])
    graph = torch.cuda.CUDAGraph()
    mgr.truncate(T - 1)
    with pytest.raises(RuntimeError, match="sync_lengths"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        int4_attention(mgr, 0, dq, None, None, D ** -0.5)
    mgr.sync_lengths()
    for layer in range(2):
        mgr.commit(layer, k[:, :, T - 1:T], v[:, :, T - 1:T])
    with torch.cuda.graph(graph):
        outs = [int4_attention(mgr, layer, dq, step_k, step_v, D ** -0.5) for layer in range(2)]
        with pytest.raises(RuntimeError):
            mgr.truncate(5)
        with pytest.raises(RuntimeError):
            mgr.sync_lengths()
    for n in (T, 41, 33):  # (41, 33: of the prompt, too)
        for _ in range(3):  # drafts
            graph.replay()
        mgr.truncate(n)
        step_k.copy_(k[:, :, 70:71])
        step_v.copy_(v[:, :, 70:71])
        graph.replay()
        noise = torch.randn(1 << 16, device=gpu).sum()
        torch.cuda.synchronize()
        assert torch.isfinite(noise) and mgr.layers[1]._lens.tolist() == [n + 1]
        kk, vv = (torch.cat([t[:, :, :n], t[:, :, 70:71]], 2) for t in (key, value))
        ref, tol = exact(q, kk, vv, [n + 1], GROUP, D ** -0.5, "bf16")
        for out in outs:
            assert_within(out, ref, tol)
        mgr.truncate(n)
    mgr.advance(0)
    for _ in range(2):
        graph.replay()
    mgr.sync_lengths()  # replays that the host is not told of
    torch.cuda.synchronize()
    assert [layer._lens.tolist() for layer in mgr.layers] == [[33], [33]]


def test_more_lengths_than_a_launch_takes(gpu):
    """600 sequences in two layers: every length in its place."""
    B = 600
    key, value = (t.to(gpu) for t in rows((B, 1, 3, 64), "bf16", 23))
    mgr = Int4KVManager(2, 1, 1, 64, 32, 32, gpu, batch_size=B)
    counts = [(3, 1, 2)[b % 3] for b in range(B)]
    mgr.commit(0, key, value)
    mgr.commit(1, key, value)
    mgr.truncate(counts)
    mgr.sync_lengths()
    assert [layer._lens.tolist() for layer in mgr.layers] == [counts] * 2
    mgr.reset()
    mgr.sync_lengths()
    assert not mgr._lens.rows.any()


def test_an_empty_cache_takes_lengths(gpu):
    mgr = Int4KVManager(2, N_Q, H, D, PAGE, GROUP, gpu)
    mgr.reset()
    mgr.truncate(0)
    mgr.sync_lengths()
    assert mgr.seq_len == 0 and not mgr._lens.rows.any()
    with pytest.raises(ValueError):
        Int4KVManager(1, N_Q, H, D, PAGE, GROUP, gpu, batch_size=0)
