"""The calls around a stream's cache of 8 bits beside other work: derivatives, numbers of any kind, another stream, two threads, another current device."""
import threading

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import sana_amd
from sana_amd import ops
from test_gpu_heads import filled, freqs_of, i32, make

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def state(seed=0, B=2, H=4, G=2, d=64, R=300):
    q, k, v, qw, kw = (t.cuda() for t in make(B, 1, H, G, d, BF16, seed=seed))
    ck, cv, sc = (t.cuda() for t in filled(B, G, R, d, seed + 1))
    return q, k, v, qw, kw, (ck, cv, sc / 64), i32([40, 5000]), freqs_of(d).cuda(), H


def turn(s, sinks=4, scale=None):
    q, k, v, qw, kw, cache, pos, f, H = s
    q, _ = ops.qk_norm_rope_append_q8_(q, k, v, cache, pos, H, qw, kw, 1e-6, f, sinks=sinks)
    return q, ops.window_attention_q8(q, cache, pos, H, sinks, scale), *ops.window_cache_read(cache, pos, sinks, 20)


@gpu
def test_derivatives_are_refused(cuda):
    q, k, v, qw, kw, cache, pos, f, H = state()
    before = [t.clone() for t in cache]
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = lambda w: [lambda: ops.qk_norm_rope(w(q), k, H, qw, kw), lambda: ops.qk_norm_rope(q, k, H, qw, w(kw)), lambda: ops.qk_norm_rope(q, k, H, freqs=w(f)),  # noqa: E731
                       lambda: ops.window_cache_append_q8_(cache, k, w(v), pos), lambda: ops.qk_norm_rope_append_q8_(q, w(k), v, cache, pos, H),
                       lambda: ops.window_attention_q8(w(q), cache, pos, H), lambda: ops.window_attention_q8(q, (*cache[:2], w(cache[2])), pos, H),
                       lambda: ops.window_cache_read((*cache[:2], w(cache[2])), pos)]
    for i, call in enumerate(calls(grad)):
        with pytest.raises(sana_amd.SanaHipError):
            call()
            pytest.fail(f"case {i} was taken")
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for i, call in enumerate(calls(dual)):
            with pytest.raises(sana_amd.SanaHipError):
                call()
                pytest.fail(f"case {i} was taken")
    with torch.no_grad():
        ops.qk_norm_rope(grad(q), k, H, qw, kw)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


@gpu
def test_numbers_of_any_kind(cuda):
    q, k, v, qw, kw, cache, pos, f, H = state()
    want = ops.qk_norm_rope(q, k, H, qw, kw, 0.5, f, magnitude=1.5)
    att = ops.window_attention_q8(q, cache, pos, H, 4, 0.5)
    for kind in (np.float32, np.float64, torch.tensor, lambda x: torch.tensor(x, device="cuda")):
        got = ops.qk_norm_rope(q, k, H, qw, kw, kind(0.5), f, magnitude=kind(1.5))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(ops.window_attention_q8(q, cache, pos, H, 4, kind(0.5)), att)


@gpu
def test_another_stream_and_lists_of_tensors(cuda):
    want = turn(state(3))
    s = state(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = turn((*s[:5], list(s[5]), *s[6:]))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_two_threads_on_one_stream(cuda):
    """Parts of long caches lie in scratch memory of each thread's own."""
    states = [state(i, B=2, R=4000) for i in range(2)]
    want = [turn(s)[1].clone() for s in states]
    assert not torch.equal(want[0], want[1])
    wrong = []

    def loop(i):
        for _ in range(60):
            if not torch.equal(turn(states[i])[1], want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@gpu
def test_the_same_call_again_is_the_same(cuda):
    """Nothing depends on what a cache held in the rows that a call writes, on the call before, or on an order of sums."""
    s = state(5, B=2, R=9000)
    first = [t.clone() for t in turn(s)]
    held = [t.clone() for t in s[5]]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(turn(s), first)) and all(torch.equal(a, b) for a, b in zip(s[5], held))


@gpu
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_a_chunk_behind_the_rows_of_its_cache(cuda, dtype):
    """The past read into the front of a buffer, the chunk's keys normed and rotated into its end and into the cache in one pass: the attention over the
    buffer is what it is over the same rows put together by single calls."""
    B, N, H, G, d, window, sinks = 2, 150, 4, 2, 72, 200, 5
    cache, f = ops.window_cache_q8(B, sinks + window, G, d), ops.rotary_frequencies(d)
    positions, past = torch.zeros(B, dtype=torch.int32, device="cuda"), 0
    for chunk in range(4):
        q, k, v, qw, kw = (t.cuda() for t in make(B, N, H, G, d, dtype, seed=chunk))
        past = min(past, sinks + window - 1)
        rows = torch.full((2, B, past + N, G * d), float("nan"), dtype=dtype, device="cuda")
        if past:
            ops.window_cache_read(cache, positions, sinks, past - sinks, d, dtype, out=rows[:, :, :past].unbind(0))
            front = ops.window_cache_read(cache, positions, sinks, past - sinks, d, dtype)
            assert torch.equal(front[0], rows[0, :, :past]) and torch.equal(front[1], rows[1, :, :past])
        rows[1, :, past:] = v
        alone = ops.qk_norm_rope(q, k, H, qw, kw, 1e-6, f, positions=positions)
        want = ops.window_attention(alone[0], torch.cat([rows[0, :, :past], alone[1]], 1), rows[1].clone(), H, window, sinks)
        q, back = ops.qk_norm_rope_append_q8_(q, k, v, cache, positions, H, qw, kw, 1e-6, f, sinks=sinks, k_out=rows[0, :, past:])
        assert torch.equal(back, alone[1]) and torch.equal(q, alone[0]) and not torch.isnan(rows).any()
        assert torch.equal(ops.window_attention(q, rows[0], rows[1], H, window, sinks), want)
        positions += N
        past += N


def test_no_cpu_tensors():
    q, k, v, qw, kw = make(1, 1, 2, 1, 32, BF16)
    cache, pos = ops.window_cache_q8(1, 9, 1, 32, device="cpu"), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.window_attention_q8(q, cache, pos, 2), lambda: ops.window_cache_read(cache, pos), lambda: ops.window_cache_read((k, k), pos)):
        with pytest.raises(sana_amd.SanaHipError):
            call()
