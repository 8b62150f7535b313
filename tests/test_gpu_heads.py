"""Norms and rotation of a stream's heads, and their keys and values in 8 bits, against the formulas in 64 bits."""
import ctypes
import math
import os
import re

import pytest
import torch

import sana_amd
from sana_amd import _lib, ops
from test_gpu_window_attention import row_of, to_gpu

gpu = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
U = 2.0 ** -24


def i32(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def definition(x, heads, weight, eps, freqs, interleaved, magnitude, positions):
    """(the heads [B, N, heads, d] in 64 bits, and how far 32 bits may be off before the last rounding).

    The sum of squares takes 8 products and sums in a lane and 4 sums between lanes, its mean, eps and the reciprocal root (1 step of 2^-23) two
    more each, half of which reach the root; x * root * weight rounds twice: 12 U.  A cosine is off by the angle's rounding to 32 bits of a turn
    (2 pi 2^-26 and, in 64 bits before, 2 steps of the turns), by 2 steps of 2^-23 itself, by its product with the magnitude, each
    product and the sum by U: (1.6 + 4 + 4) U and 2 pi 2^-52 a turn, of |a| + |b| each."""
    B, N, C = x.shape
    d = C // heads
    x = x.double().reshape(B, N, heads, d)
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    off = (12 * U if weight is not None else 0) * x.abs()
    if freqs is not None:
        r = 2 * freqs.numel()
        at = torch.tensor([0] * B if positions is None else positions, dtype=torch.float64)[:, None] + torch.arange(N, dtype=torch.float64)
        angle = at[:, :, None] * freqs.double()
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
        c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
        pair = [magnitude * (a * c - b * s), magnitude * (a * s + b * c)]
        far = (22 * U + 2 * math.pi * 2.0 ** -52 * (angle.abs() / (2 * math.pi))[:, :, None]) * abs(magnitude) * (a.abs() + b.abs())
        join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat([p, q], -1))
        x = torch.cat([join(*pair), x[..., r:]], -1)
        off = torch.cat([join(far, far), off[..., r:]], -1)
    return x, off


def near(got, want, off):
    """Rounded once to got's dtype: half a step of the value, at least half of the smallest number of f16."""
    half = torch.finfo(got.dtype).eps / 2
    tol = off + half * (want.abs() + off) + (2.0 ** -25 if got.dtype == F16 else 0)
    err = (got.double().cpu().reshape(want.shape) - want).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def make(B, N, H, G, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, N, (H + 2 * G) * d, generator=g).to(dtype)
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)]
    return *x.split([H * d, G * d, G * d], dim=2), *w


def freqs_of(rotary, base=10000.0):
    return ops.rotary_frequencies(rotary, base, device="cpu") if rotary else None


def compare(B, N, H, G, d, rotary, dtype, *, norm=True, interleaved=True, magnitude=1.0, positions=None, lengths=None, eps=1e-6, seed=0):
    q, k, _, qw, kw = make(B, N, H, G, d, dtype, seed)
    f = freqs_of(rotary)
    qw, kw = (qw, kw) if norm else (None, None)
    gq, gk = ops.qk_norm_rope(*to_gpu(q, k), H, None if qw is None else qw.cuda(), None if kw is None else kw.cuda(), eps, None if f is None else f.cuda(),
                              interleaved, magnitude, i32(positions), i32(lengths))
    assert gq.shape == q.shape and gk.shape == k.shape and gq.dtype == dtype
    for got, x, n, w in ((gq, q, H, qw), (gk, k, G, kw)):
        want, off = definition(x, n, w, eps, f, interleaved, magnitude, positions)
        for b in range(B):
            live = N if lengths is None else min(max(lengths[b], 0), N)
            live = 0 if positions is not None and positions[b] < 0 else live
            want[b, live:], off[b, live:] = 0, 0
            assert not got[b, live:].any()
        near(got, want, off)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d", [8, 16, 32, 40, 64, 72, 80, 96, 104, 112, 128])
def test_head_dims(cuda, d, interleaved, dtype):
    compare(2, 5, 6, 3, d, d, dtype, interleaved=interleaved, positions=[3, 100], seed=d)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,rotary", [(64, 8), (64, 32), (72, 16), (72, 64), (112, 56), (128, 96), (128, 0), (32, 0)])
def test_part_of_the_head(cuda, d, rotary, interleaved, dtype):
    compare(1, 7, 5, 2, d, rotary, dtype, interleaved=interleaved, magnitude=1.25, positions=[77])
    compare(1, 7, 5, 2, d, rotary, dtype, interleaved=interleaved, norm=False, positions=[77])


@gpu
@pytest.mark.parametrize("B,N,H,G", [(1, 1, 1, 1), (1, 1, 33, 1), (3, 1, 16, 16), (1, 257, 20, 20), (70, 2, 4, 4), (2, 1500, 3, 1), (5000, 1, 2, 1), (1, 4, 70, 70)])
@pytest.mark.parametrize("d,interleaved", [(32, True), (112, False)])
def test_sizes(cuda, B, N, H, G, d, interleaved):
    compare(B, N, H, G, d, d, BF16, interleaved=interleaved, positions=list(range(B)), seed=N)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_far_positions(cuda, interleaved, dtype):
    """What 32 bits of an angle would lose: at position 2^31 - 1 its step is 128 radians."""
    compare(4, 3, 2, 2, 64, 64, dtype, interleaved=interleaved, positions=[1 << 17, 12345678, 2 ** 31 - 5, 2 ** 31 - 1])


@gpu
def test_scaled_frequencies(cuda):
    """All divided; or few turns divided, many kept, a blend between."""
    r, base, trained = 64, 10000.0, 4096
    f = ops.rotary_frequencies(r, base)
    i = torch.arange(r // 2, dtype=torch.float64)
    assert f.dtype == torch.float64 and f.is_cuda and torch.allclose(f.cpu(), torch.exp(-2 * i / r * math.log(base)), rtol=1e-14, atol=0)
    assert torch.equal(ops.rotary_frequencies(r, base, factor=8.0), f / 8)
    g = ops.rotary_frequencies(r, base, factor=8.0, trained=trained, slow=1.0, fast=32.0)
    turns = trained * f / (2 * math.pi)
    assert torch.equal(g[turns > 32], f[turns > 32]) and torch.allclose(g[turns < 1], f[turns < 1] / 8, rtol=1e-15, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((g < f) & (g > f / 8))[between].all()
    for bad in (lambda: ops.rotary_frequencies(7), lambda: ops.rotary_frequencies(0), lambda: ops.rotary_frequencies(8, 0.0),
                lambda: ops.rotary_frequencies(8, factor=-1.0), lambda: ops.rotary_frequencies(8, trained=0),
                lambda: ops.rotary_frequencies(8, trained=9, slow=3.0, fast=3.0)):
        with pytest.raises(sana_amd.SanaHipError):
            bad()


@gpu
@pytest.mark.parametrize("power", [-64, -60, 0, 55])
def test_rows_of_any_size_without_eps(cuda, power):
    """bf16 rows whose squares are far from 1, down to the subnormal numbers of fp32: there a square is off by 2^-150, and so is the mean, of some 2^-128."""
    H, d = 4, 64
    q, k, _, qw, kw = make(2, 5, H, 2, d, BF16)
    q, k = (t.contiguous() * 2.0 ** power for t in (q, k))
    got = ops.qk_norm_rope(q.cuda(), k.cuda(), H, qw.cuda(), kw.cuda(), 0.0)
    for g, x, n, w in ((got[0], q, H, qw), (got[1], k, 2, kw)):
        want, off = definition(x, n, w, 0.0, None, True, 1.0, None)
        mean = x.double().reshape(2, 5, n, d).square().mean(-1, keepdim=True)
        near(g, want, off + want.abs() * (2.0 ** -150 + 2.0 ** -150) / mean)


@gpu
@pytest.mark.parametrize("d", [8, 64, 128])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e38])
@pytest.mark.parametrize("power", [60, 64, 90, 124])
def test_rows_whose_squares_leave_32_bits(cuda, power, eps, d):
    """bf16 heads of up to the largest numbers beside ordinary ones, of one token and of others: each by its own mean."""
    H, G, N = 5, 3, 7
    q, k, _, qw, kw = make(2, N, H, G, d, BF16, seed=power)
    big = (torch.arange(N)[:, None] + torch.arange(H)) % 3 == 0
    f = freqs_of(d)
    q, k = (torch.where(big[:, :n, None], t.reshape(2, N, n, d).float() * 2.0 ** power, t.reshape(2, N, n, d).float()).clamp(-3.3e38, 3.3e38).flatten(2).to(BF16)
            for t, n in ((q, H), (k, G)))
    got = ops.qk_norm_rope(q.cuda(), k.cuda(), H, qw.cuda(), kw.cuda(), eps, f.cuda(), positions=i32([3, 70]))
    for g, x, n, w in ((got[0], q, H, qw), (got[1], k, G, kw)):
        want, off = definition(x, n, w, float(torch.tensor(eps)), f, True, 1.0, [3, 70])
        assert torch.isfinite(g).all()
        near(g, want, off)


@gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_lengths_and_idle_streams(cuda, interleaved):
    """Rows without a token: zeros in new outputs, left as they were in given ones, NaN of the inputs there not looked at."""
    positions, lengths = [5, -1, 0, 9, 2 ** 31 - 1, -7], [4, 9, 0, 12, 1, -3]
    compare(6, 9, 4, 2, 72, 72, BF16, interleaved=interleaved, positions=positions, lengths=lengths)
    q, k, _, qw, kw = (t.cuda() for t in make(6, 9, 4, 2, 72, BF16))
    f = freqs_of(72).cuda()
    want = ops.qk_norm_rope(q, k, 4, qw, kw, 1e-6, f, interleaved, positions=i32(positions), lengths=i32(lengths))
    live = torch.tensor([[p >= 0 and t < n for t in range(9)] for p, n in zip(positions, lengths)], device="cuda")[..., None]
    q, k = torch.where(live, q, math.nan), torch.where(live, k, math.inf)
    outs = torch.full_like(q, 7.0), torch.full_like(k, 8.0)
    got = ops.qk_norm_rope(q, k, 4, qw, kw, 1e-6, f, interleaved, positions=i32(positions), lengths=i32(lengths), q_out=outs[0], k_out=outs[1])
    assert got[0] is outs[0] and got[1] is outs[1]
    assert torch.equal(got[0], torch.where(live, want[0], 7.0)) and torch.equal(got[1], torch.where(live, want[1], 8.0))


@gpu
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d", [40, 112])
def test_views_and_in_place(cuda, d, interleaved):
    B, N, H, G = 3, 11, 6, 2
    q, k, _, qw, kw = make(B, N, H, G, d, F16)
    f, w, pos = freqs_of(d - 8).cuda(), (qw.cuda(), kw.cuda()), i32([4, 0, 30])
    want = ops.qk_norm_rope(q.contiguous().cuda(), k.contiguous().cuda(), H, *w, 1e-6, f, interleaved, positions=pos)
    wide = torch.full((B, N + 3, 4, H * d + 8), float("nan"), dtype=F16, device="cuda")
    views = [wide[:, 1:1 + N, 0, 8:], wide[:, 1:1 + N, 1, :G * d], wide[:, 1:1 + N, 2, 8:], wide[:, 1:1 + N, 3, :G * d]]
    views[0].copy_(q), views[1].copy_(k)
    ops.qk_norm_rope(views[0], views[1], H, *w, 1e-6, f, interleaved, positions=pos, q_out=views[2], k_out=views[3])
    assert torch.equal(views[2], want[0]) and torch.equal(views[3], want[1])
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1).cuda() for t in (q, k)]
    got = ops.qk_norm_rope(*swapped, H, *w, 1e-6, f, interleaved, positions=pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ops.qk_norm_rope(views[0], views[1], H, *w, 1e-6, f, interleaved, positions=pos, q_out=views[0], k_out=views[1])
    assert torch.equal(views[0], want[0]) and torch.equal(views[1], want[1])
    assert torch.isnan(wide[:, :1]).all() and torch.isnan(wide[:, 1 + N:]).all() and torch.isnan(wide[:, :, 0, :8]).all()
    assert torch.isnan(wide[:, :, 3, G * d:]).all()


@gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_values_that_are_not_finite_stay_in_their_head(cuda, interleaved):
    """With a norm: in their head.  Without: in their channel, or the pair that turns with it."""
    B, N, H, G, d, r = 1, 6, 5, 2, 64, 32
    q, k, _, qw, kw = (t.cuda() for t in make(B, N, H, G, d, BF16))
    f = freqs_of(r).cuda()
    for norm in (True, False):
        args = (H, qw if norm else None, kw if norm else None, 1e-6, f, interleaved)
        want = ops.qk_norm_rope(q, k, *args)
        bad_q, bad_k = q.clone(), k.clone()
        bad_q[0, 2, 1 * d + 3], bad_q[0, 3, 2 * d + 40], bad_k[0, 5, d + 1] = math.nan, math.inf, -math.inf
        got = ops.qk_norm_rope(bad_q, bad_k, *args)
        partner = (lambda c: c ^ 1) if interleaved else (lambda c: (c + r // 2) % r)
        for x, y, t, h, c in ((got[0], want[0], 2, 1, 3), (got[0], want[0], 3, 2, 40), (got[1], want[1], 5, 1, 1)):
            assert not torch.isfinite(x[0, t, h * d + c])
            touched = range(h * d, (h + 1) * d) if norm else [h * d + c] + ([h * d + partner(c)] if c < r else [])
            x[0, t, list(touched)] = y[0, t, list(touched)]
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# --------------------------------------------------------------------------- 8 bits

def coded(x):
    """x [..., d] of 16-bit values -> (codes, scales): the nearest whole numbers to 127 x / max|x|, ties to even, in 64 bits."""
    most = x.double().abs().amax(-1, keepdim=True)
    codes = torch.round(torch.where(most > 0, 127 * x.double() / most, 0.0))
    return codes.to(torch.int8), (most[..., 0].float() / 127)


def filled(B, G, R, d, seed=1):
    """A cache that holds something in every place, those behind d among them."""
    g = torch.Generator().manual_seed(seed)
    wide = -(-d // 16) * 16
    return (*(torch.randint(-127, 128, (B, G, R, wide), generator=g, dtype=torch.int8) for _ in range(2)), torch.rand(B, G, R, 2, generator=g))


def appended(cache, parts, positions, sinks, lengths, d):
    """The cache after the tokens' (codes, scales) [B, N, G, ...] of keys and of values went in one by one."""
    cache = [t.clone() for t in cache]
    R, N = cache[0].shape[2], parts[0][0].shape[1]
    for b, pos in enumerate(positions):
        for t in range((N if lengths is None else min(max(lengths[b], 0), N)) if pos >= 0 else 0):
            row = row_of(pos + t, sinks, R - sinks)
            for i, (codes, scales) in enumerate(parts):
                cache[i][b, :, row, :d], cache[2][b, :, row, i] = codes[b, t], scales[b, t]
    return cache


def same(got, want, d):
    for g, w in zip(got[:2], want[:2]):
        assert torch.equal(g.cpu()[..., :d], w[..., :d])
    assert torch.equal(got[2].cpu().view(torch.int32), want[2].view(torch.int32))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 112, 128])
@pytest.mark.parametrize("window,sinks,N", [(1, 0, 3), (64, 4, 1), (64, 4, 50), (37, 100, 200)])
def test_append(cuda, window, sinks, N, d, dtype):
    B, G = 6, 3
    _, k, v, _, _ = make(B, N, 1, G, d, dtype, seed=N)
    cache = filled(B, G, sinks + window, d)
    parts = [coded(t.reshape(B, N, G, d)) for t in (k, v)]
    positions = [0, 3, sinks, -1, sinks + window, 2 ** 31 - 1 - N]
    for lengths in (None, [N, 0, N // 2, N, N + 5, -3]):
        dev = [t.cuda() for t in cache]
        ops.window_cache_append_q8_(dev, *to_gpu(k, v), i32(positions), sinks, i32(lengths))
        same(dev, appended(cache, parts, positions, sinks, lengths, d), d)
        pad = [t.cpu()[..., d:].eq(c[..., d:]).all() for t, c in zip(dev[:2], cache[:2])]
        assert all(pad)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_codes_of_every_quotient(cuda, dtype):
    """Every magnitude of a binade and its like below the largest, as the largest and next to it: among them all ties, which go to the even number."""
    bits = 7 if dtype == BF16 else 10
    most = 1 + torch.arange(1 << bits) / (1 << bits)
    rows = []
    for e in range(0, 9):
        for shift in range(0, 1 << bits, 61):
            x = most.roll(shift) * 2.0 ** -e
            rows.append(torch.stack([most, torch.minimum(x, most), -torch.minimum(x.flip(0), most)], -1))
    x = torch.cat([torch.cat(rows).to(dtype), torch.zeros(len(rows) << bits, 5, dtype=dtype)], -1)[None]     # [1, N, 8]
    x = torch.cat([x, x[:, :, :3] / 2, torch.zeros_like(x)[:, :, :5]], -1)          # a second head
    N = x.shape[1]
    cache = filled(1, 2, N, 8)
    dev = [t.cuda() for t in cache]
    ops.window_cache_append_q8_(dev, x.cuda(), x.flip(1).cuda(), i32([0]))
    parts = [coded(t.reshape(1, N, 2, 8)) for t in (x, x.flip(1))]
    half = (127 * x.double().reshape(1, N, 2, 8) / x.double().reshape(1, N, 2, 8).abs().amax(-1, keepdim=True)) % 1 == 0.5
    assert half.sum() > 100
    same(dev, appended(cache, parts, [0], 0, None, 8), 8)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_of_every_size(cuda, dtype):
    """Zeros, the smallest and the largest numbers, inf and NaN: the scale of a row that is not finite is NaN, its neighbours are what they are."""
    tiny, huge = (2.0 ** -133, 3.0e38) if dtype == BF16 else (2.0 ** -24, 65504.0)
    d, G = 16, 2
    x = torch.randn(1, 12, G * d, generator=torch.Generator().manual_seed(0))
    for t, f in enumerate((0.0, tiny * 3, huge / 8, 1e-30, 1e30)):
        x[0, t, :d] *= f
    x = x.to(dtype).clamp(-huge, huge)
    x[0, 0, :d] = 0
    x[0, 5, 3], x[0, 6, 4], x[0, 7, 5] = math.inf, -math.inf, math.nan
    bad = torch.zeros(12, G, dtype=torch.bool)
    bad[5:8, 0] = True
    dev = [t.cuda() for t in filled(1, G, 12, d)]
    ops.window_cache_append_q8_(dev, x.cuda(), x.cuda(), i32([0]))
    codes, scales = coded(torch.where(bad[None, :, :, None], 0.0, x.reshape(1, 12, G, d).double()).to(dtype))
    for i in (0, 1):
        got = dev[2][0, :, :, i].T.cpu()
        assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], scales[0][~bad])
        assert torch.equal(dev[i][0, :, :, :d].transpose(0, 1).cpu()[~bad], codes[0][~bad])
    k, v = ops.window_cache_read(dev, i32([12]), dtype=dtype)
    k = k.cpu().reshape(12, G, d)
    assert torch.isnan(k[bad]).all() and torch.isfinite(k[~bad]).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,N,H,G,d,rotary,window,sinks", [(3, 5, 6, 2, 72, 72, 20, 2), (2, 1, 8, 8, 64, 32, 9, 0), (1, 70, 4, 4, 112, 112, 33, 5),
                                                           (2, 33, 3, 3, 32, 24, 64, 0), (40, 1, 2, 1, 128, 128, 7, 1)])
def test_all_in_one_pass(cuda, B, N, H, G, d, rotary, window, sinks, interleaved, dtype):
    """Queries, and keys if asked for, bit for bit as without a cache; values' codes as if appended alone; keys' codes from the unrounded key."""
    q, k, v, qw, kw = make(B, N, H, G, d, dtype, seed=d)
    positions, lengths = [(7 * b) % 50 for b in range(B)], [N - b % 2 for b in range(B)]
    f = freqs_of(rotary)
    args = (qw.cuda(), kw.cuda(), 1e-6, f.cuda(), interleaved, 1.1)
    dev_q, dev_k, dev_v = to_gpu(q, k, v)
    cache = filled(B, G, window + sinks, d)
    for keep in (False, True):
        dev = [t.cuda() for t in cache]
        k_out = torch.zeros_like(dev_k) if keep else None
        got_q, got_k = ops.qk_norm_rope_append_q8_(dev_q, dev_k, dev_v, dev, i32(positions), H, *args, sinks, i32(lengths), k_out=k_out)
        want = ops.qk_norm_rope(dev_q, dev_k, H, *args, i32(positions), i32(lengths))
        assert torch.equal(got_q, want[0]) and got_k is k_out and (k_out is None or torch.equal(k_out, want[1]))
        y, off = definition(k, G, kw, 1e-6, f, interleaved, 1.1, positions)
        value = coded(v.reshape(B, N, G, d))
        ref = appended(cache, [(torch.zeros_like(value[0]), torch.zeros_like(value[1])), value], positions, sinks, lengths, d)
        assert torch.equal(dev[1].cpu()[..., :d], ref[1][..., :d]) and torch.equal(dev[2][..., 1].cpu(), ref[2][..., 1])
        for b in range(B):
            for t in range(lengths[b]):
                p = positions[b] + t
                if p >= sinks and t < lengths[b] - window:
                    continue
                row = row_of(p, sinks, window)
                s = dev[2][b, :, row, 0].double().cpu()
                most, far = y[b, t].abs().amax(-1), off[b, t].amax(-1)
                assert ((s - most / 127).abs() <= far / 127 + U * most / 127).all()
                # half a step, the quotient's rounding (127 times U), the key's own error, and the scale's
                err = (dev[0][b, :, row, :d].double().cpu() * s[:, None] - y[b, t]).abs()
                assert (err <= s[:, None] * (0.5 + 2.0 ** -16) + 3 * far[:, None] + 2.0 ** -22 * most[:, None]).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,N,H,G,d,rotary", [(1, 8229, 3, 1, 72, 72), (3, 2999, 2, 2, 32, 16), (2, 4100, 5, 5, 112, 112), (90, 97, 4, 2, 128, 64), (1, 9000, 1, 3, 8, 8), (2, 5000, 3, 2, 64, 0), (2, 4100, 15, 13, 72, 40)])
def test_many_tokens_are_what_they_are_in_pieces(cuda, B, N, H, G, d, rotary, interleaved, dtype):
    """Runs of tokens a wave and heads of one token a wave: the same numbers, one call or many, with and without a cache."""
    q, k, v, qw, kw = (t.cuda() for t in make(B, N, H, G, d, dtype, seed=N))
    f = freqs_of(rotary)
    args = (qw, kw, 1e-6, None if f is None else f.cuda(), interleaved, 0.9)
    positions = torch.arange(B) * 1000003 + 5
    positions[B // 2] = -1 if B > 2 else 17
    lengths = N - torch.arange(B) * (N // (B + 3))
    window, sinks, pieces = 600, 130, 1000
    whole, parts = ([t.cuda() for t in filled(B, G, window + sinks, d)] for _ in range(2))
    got = ops.qk_norm_rope_append_q8_(q, k, v, whole, i32(positions.tolist()), H, *args, sinks, i32(lengths.tolist()), k_out=torch.zeros_like(k))
    alone = ops.qk_norm_rope(q, k, H, *args, i32(positions.tolist()), i32(lengths.tolist()))
    want = torch.zeros_like(q), torch.zeros_like(k)
    for at in range(0, N, pieces):
        now = slice(at, min(at + pieces, N))
        pos = torch.where(positions < 0, positions, positions + at)
        for b in range(B):     # (piece by piece and stream by stream)
            one = slice(b, b + 1)
            n = max(0, min(int(lengths[b]) - at, pieces))
            outs = ops.qk_norm_rope_append_q8_(q[one, now], k[one, now], v[one, now], [t[one] for t in parts], i32([int(pos[b])]), H, *args, sinks, i32([n]),
                                               k_out=torch.zeros_like(k[one, now]))
            want[0][one, now], want[1][one, now] = outs
    for g, a, w in zip(got, alone, want):
        assert torch.equal(g, w) and torch.equal(a, w)
    assert all(torch.equal(a.view(torch.int8 if a.dtype == torch.int8 else torch.int32), b.view(torch.int8 if b.dtype == torch.int8 else torch.int32)) for a, b in zip(whole, parts))


@gpu
@pytest.mark.parametrize("window,sinks,N", [(500, 70, 9000), (5, 0, 8192), (8000, 3, 8300), (9000, 100, 9001), (64, 9500, 9000), (1, 1, 20000)])
def test_long_appends_leave_out_what_does_not_stay(cuda, window, sinks, N):
    """All tokens of a call without lengths: those between the sinks and the last window are not even looked at (they are NaN here)."""
    B, G, d = 3, 2, 40
    _, k, v, _, _ = (t.cuda() for t in make(B, N, 1, G, d, BF16, seed=window))
    positions = [0, 50, 1000000]
    whole, parts = ([t.cuda() for t in filled(B, G, window + sinks, d)] for _ in range(2))
    for at in range(0, N, 1000):
        n = min(1000, N - at)
        ops.window_cache_append_q8_(parts, k[:, at:at + n], v[:, at:at + n], i32([p + at for p in positions]), sinks)
    for b, p in enumerate(positions):
        gone = torch.arange(N, device="cuda")
        gone = (gone + p >= sinks) & (gone < N - window)
        k[b, gone], v[b, gone] = math.nan, math.nan
    ops.window_cache_append_q8_(whole, k, v, i32(positions), sinks)
    # a row of NaN has the scale NaN: none is there, and all are those of the pieces
    assert all(torch.equal(a, b) for a, b in zip(whole, parts))


@gpu
@pytest.mark.parametrize("cached", [False, True])
def test_more_tokens_than_a_layer_of_the_grid(cuda, cached):
    """Heads of one token a wave, 2^17 tokens of a stream a layer: bit for bit the two calls that the second layer's tokens divide it into."""
    B, N, at, H, G, d, W, S = 2, (1 << 17) + 203, 1 << 17, (8 if cached else 16), (8 if cached else 16), 72, 700, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(B, N, n * d, generator=g, device="cuda", dtype=BF16) for n in (H, G, G))
    w = [(1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(BF16) for _ in range(2)]
    args, positions = (*w, 1e-6, freqs_of(72).cuda()), [3, 1 << 20]
    whole, parts = ([t.cuda() for t in filled(B, G, W + S, d)] for _ in range(2))

    def call(now, positions, lengths, cache, outs):
        if not cached:
            return ops.qk_norm_rope(q[:, now], k[:, now], H, *args, positions=i32(positions), lengths=i32(lengths), q_out=outs[0][:, now], k_out=outs[1][:, now])
        return ops.qk_norm_rope_append_q8_(q[:, now], k[:, now], v[:, now], cache, i32(positions), H, *args, sinks=S, lengths=i32(lengths), q_out=outs[0][:, now],
                                           k_out=outs[1][:, now])

    for lengths in ([N, at + 100], [at - 1, N], [N, at + 1]):
        got, want = ([torch.full_like(t, 7.0) for t in (q, k)] for _ in range(2))
        call(slice(0, N), positions, lengths, whole, got)
        call(slice(0, at), positions, [min(n, at) for n in lengths], parts, want)
        call(slice(at, N), [p + at for p in positions], [max(n - at, 0) for n in lengths], parts, want)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(whole, parts))
        assert (got[0][0, lengths[0]:] == 7).all() and (got[1][1, lengths[1]:] == 7).all()


@gpu
@pytest.mark.parametrize("lengths", [None, [640003, 524289]])
def test_more_runs_of_tokens_than_a_layer_of_the_grid(cuda, lengths):
    """Runs of tokens a wave, 2^19 tokens of a stream a layer, into the cache alone; without lengths those between the sinks and the last window are left out
    (NaN here), and two layers of tiles are left."""
    B, N, G, d, W, S = 2, 640003, 1, 80, 540001, 1000
    k, v = (torch.randn(B, N, G * d, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda", dtype=BF16) for i in (0, 1))
    positions = [0, 77777]
    whole, parts = ([t.cuda() for t in filled(B, G, W + S, d)] for _ in range(2))
    for at in range(0, N, 100000):
        n = min(100000, N - at)
        ops.window_cache_append_q8_(parts, k[:, at:at + n], v[:, at:at + n], i32([p + at for p in positions]), S, i32([max(0, min(n, x - at)) for x in lengths or [N] * B]))
    if lengths is None:
        for b, p in enumerate(positions):
            gone = torch.arange(N, device="cuda")
            gone = (gone + p >= S) & (gone < N - W)
            assert gone.sum() > 90000
            k[b, gone], v[b, gone] = math.nan, math.nan
    ops.window_cache_append_q8_(whole, k, v, i32(positions), S, i32(lengths))
    # a row of NaN has the scale NaN: none is there, and all are those of the pieces
    assert all(torch.equal(a, b) for a, b in zip(whole, parts))


# --------------------------------------------------------------------------- refusals

def test_calls_that_are_refused_before_any_launch():
    """Host checks of the C entry (the pointers are never followed)."""
    lib, P, bf16 = _lib.load(), 0x10000, _lib.DT_BF16
    names = ("q k v q_out k_out q_weight k_weight freqs positions lengths codes_k codes_v scales q_b q_n k_b k_n v_b v_n qo_b qo_n ko_b ko_n ck_b cv_b sc_b "
             "B N H Hkv d rotary interleaved window sinks zero_rest io_dtype eps magnitude").split()
    good = dict(q=P, k=2 * P, v=3 * P, q_out=4 * P, k_out=5 * P, q_weight=P, k_weight=P, freqs=P, positions=P, lengths=P, codes_k=6 * P, codes_v=7 * P, scales=8 * P,
                q_b=8 * 256, q_n=256, k_b=8 * 128, k_n=128, v_b=8 * 128, v_n=128, qo_b=8 * 256, qo_n=256, ko_b=8 * 128, ko_n=128, ck_b=2 * 20 * 64,
                cv_b=2 * 20 * 64, sc_b=2 * 20 * 2, B=2, N=8, H=4, Hkv=2, d=64, rotary=64, interleaved=1, window=16, sinks=4, zero_rest=0, io_dtype=bf16,
                eps=1e-6, magnitude=1.0)

    def call(**change):
        return lib.sana_hip_heads(_lib.HEADS_ARGS.pack(*[{**good, **change}[n] for n in names]), None)

    ARG, SHAPE, ALIGN, DTYPE = -1, -2, -3, -6
    assert lib.sana_hip_heads(None, None) == ARG
    for n in ("k", "q", "q_out", "v", "codes_k", "codes_v", "scales", "positions", "q_weight", "k_weight", "freqs", "B", "N", "H", "Hkv", "d", "window", "rotary"):
        assert call(**{n: 0}) == ARG, n
    assert call(codes_k=0, codes_v=0, scales=0, k_out=0) == ARG
    for change in (dict(sinks=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(magnitude=float("inf")), dict(magnitude=float("nan")),
                   dict(q_n=248), dict(k_n=120), dict(v_n=120), dict(qo_n=248), dict(ko_n=120), dict(qo_b=248), dict(ko_b=120), dict(q_b=-8), dict(ck_b=2 * 20 * 64 - 16),
                   dict(cv_b=0), dict(sc_b=2 * 20 * 2 - 2), dict(q_out=P, qo_n=264), dict(k_out=2 * P, ko_b=9 * 128), dict(rotary=-8), dict(H=-1)):
        assert call(**change) == ARG, change
    for change in (dict(d=60, rotary=56), dict(d=136), dict(rotary=60), dict(rotary=72), dict(N=(1 << 30) + 1), dict(window=(1 << 30), ck_b=1 << 40, cv_b=1 << 40, sc_b=1 << 40),
                   dict(B=2 ** 31 - 1, N=1 << 30)):
        assert call(**change) == SHAPE, change
    for change in (dict(q=P + 8), dict(k=P + 2), dict(v=P + 8), dict(q_out=P + 8), dict(k_out=P + 4), dict(q_n=260), dict(v_b=1026), dict(codes_k=P + 8), dict(scales=P + 4),
                   dict(ck_b=2 * 20 * 64 + 8), dict(sc_b=2 * 20 * 2 + 1), dict(positions=P + 2), dict(lengths=P + 1), dict(freqs=P + 4), dict(q_weight=P + 1)):
        assert call(**change) == ALIGN, change
    assert call(io_dtype=0) == DTYPE and call(io_dtype=7) == DTYPE


def test_rows_of_an_output_that_is_not_there_cannot_be_zeroed():
    """``zero_rest`` names q_out and k_out: what it names has to be there (the pointers are never followed)."""
    lib, P = _lib.load(), 0x10000

    def call(q, k_out, zero_rest):
        pointers = dict(q=P if q else 0, k=2 * P, v=3 * P, q_out=4 * P if q else 0, k_out=5 * P if k_out else 0, q_weight=0, k_weight=0, freqs=0, positions=P, lengths=P,
                        codes_k=6 * P, codes_v=7 * P, scales=8 * P)
        strides = [8 * 256, 256, 8 * 128, 128, 8 * 128, 128, 8 * 256, 256, 8 * 128, 128, 2 * 20 * 64, 2 * 20 * 64, 2 * 20 * 2]
        return lib.sana_hip_heads(_lib.HEADS_ARGS.pack(*pointers.values(), *strides, 2, 8, 4 if q else 0, 2, 64, 0, 1, 16, 4, zero_rest, _lib.DT_BF16, 1e-6, 1.0), None)

    for zero_rest in (2, 3):
        assert call(True, False, zero_rest) == -1 and call(False, False, zero_rest) == -1
    for zero_rest in (1, 3):
        assert call(False, True, zero_rest) == -1
    for zero_rest in (-1, 4, 7):
        assert call(True, True, zero_rest) == -1


@gpu
@pytest.mark.parametrize("N", [1, 6, 8192])
@pytest.mark.parametrize("zero_rest", [0, 1])
def test_one_pass_with_idle_streams_and_no_key_output(cuda, zero_rest, N):
    """The C entry, keys into the cache alone: queries' rows without a token are zeros or as they were, and nothing else of the call depends on ``zero_rest``."""
    B, H, G, d, W, S = 4, 4, 2, 64, 20, 2
    q, k, v, _, _ = (t.contiguous().cuda() for t in make(B, N, H, G, d, BF16, seed=N))
    pos, lens = i32([3, -1, 0, 40]), i32([N, N, 0, max(N - 2, 0)])
    cache, ref = ([t.cuda() for t in filled(B, G, W + S, d)] for _ in range(2))
    out = torch.full_like(q, 7.0)
    rows_q, rows_k, codes = [N * H * d, H * d], [N * G * d, G * d], G * (W + S) * d
    args = _lib.HEADS_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, 0, 0, 0, pos.data_ptr(), lens.data_ptr(), *(t.data_ptr() for t in cache),
                                *rows_q, *rows_k, *rows_k, *rows_q, 0, 0, codes, codes, 2 * G * (W + S), B, N, H, G, d, 0, 1, W, S, zero_rest, _lib.DT_BF16, 1e-6, 1.0)
    assert _lib.load().sana_hip_heads(args, torch.cuda.current_stream().cuda_stream) == 0
    want, _ = ops.qk_norm_rope_append_q8_(q, k, v, ref, pos, H, sinks=S, lengths=lens)
    live = torch.tensor([[p >= 0 and t < n for t in range(N)] for p, n in zip(pos.tolist(), lens.tolist())], device="cuda")[..., None]
    assert torch.equal(out, torch.where(live, want, 0.0 if zero_rest else 7.0))
    assert all(torch.equal(a, b) for a, b in zip(cache, ref))


def header_fields(name):
    """The (type, field) pairs of a structure of include/sana_hip.h, in order."""
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "sana_hip.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1), flags=re.S)
    fields = []
    for line in filter(None, (x.strip().replace("* ", " *") for x in body.split(";"))):
        kind, names = re.match(r"((?:const )?\w+)\s+(.*)", line, re.S).groups()
        for n in names.split(","):
            n = n.strip()
            fields.append((ctypes.c_void_p, n[1:].strip()) if n.startswith("*") else
                          ({"size_t": ctypes.c_size_t, "int64_t": ctypes.c_int64, "int": ctypes.c_int, "float": ctypes.c_float}[kind], n))
    return fields


@pytest.mark.parametrize("name,layout", [("sana_heads_args", "HEADS_ARGS"), ("sana_window_q8_args", "WINDOW_Q8_ARGS"), ("sana_cache_read_args", "CACHE_READ_ARGS")])
def test_packed_arguments_lie_as_in_the_header(name, layout):
    """Each field in turn holds something, the others nothing: the packed bytes are those of the C structure."""
    fields, layout = header_fields(name), getattr(_lib, layout)
    args = type(name, (ctypes.Structure,), {"_fields_": [(n, t) for t, n in fields]})
    assert layout.size == ctypes.sizeof(args)
    for i, (kind, n) in enumerate(fields):
        held = args()
        value = 1.5 if kind is ctypes.c_float else 0x01020304
        setattr(held, n, value)
        assert layout.pack(*[value if j == i else 0.0 if t is ctypes.c_float else 0 for j, (t, _) in enumerate(fields)]) == bytes(held), n


def test_no_cpu_tensors():
    q, k, v, qw, kw = make(1, 2, 2, 1, 32, BF16)
    cache = ops.window_cache_q8(1, 8, 1, 32, device="cpu")
    pos = torch.zeros(1, dtype=torch.int32)
    for bad in (lambda: ops.qk_norm_rope(q, k, 2, qw, kw), lambda: ops.window_cache_append_q8_(cache, k, v, pos),
                lambda: ops.qk_norm_rope_append_q8_(q, k, v, cache, pos, 2, qw, kw)):
        with pytest.raises(sana_amd.SanaHipError):
            bad()


@gpu
def test_refusals(cuda):
    q, k, v, qw, kw = (t.cuda() for t in make(2, 4, 4, 2, 64, BF16))
    f, pos, cache = freqs_of(64).cuda(), i32([0, 0]), [t.cuda() for t in filled(2, 2, 20, 64)]
    norm = lambda **c: ops.qk_norm_rope(**{**dict(q=q, k=k, num_heads=4, q_weight=qw, k_weight=kw, freqs=f, positions=pos), **c})  # noqa: E731
    put = lambda **c: ops.window_cache_append_q8_(**{**dict(cache=cache, k=k, v=v, positions=pos, sinks=4), **c})  # noqa: E731
    both = lambda **c: ops.qk_norm_rope_append_q8_(**{**dict(q=q, k=k, v=v, cache=cache, positions=pos, num_heads=4, q_weight=qw, k_weight=kw, freqs=f, sinks=4), **c})  # noqa: E731
    norm(), put(), both()
    ck, cv, sc = cache
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    bad = [lambda: norm(q=q.float()), lambda: norm(k=k.half()), lambda: norm(num_heads=3), lambda: norm(num_heads=0), lambda: norm(k_weight=None),
           lambda: norm(q_weight=qw.float()), lambda: norm(q_weight=qw[:32]), lambda: norm(freqs=f.float()), lambda: norm(freqs=f[:2]), lambda: norm(freqs=torch.cat([f, f])),
           lambda: norm(positions=pos.long()), lambda: norm(lengths=pos[:1]), lambda: norm(q=q[:, :3]), lambda: norm(q_out=q[:, :3]), lambda: norm(k_out=k.half()),
           lambda: norm(q=q[:1].expand(2, 4, 256), q_out=q[:1].expand(2, 4, 256)), lambda: norm(eps=-1.0), lambda: norm(magnitude=float("inf")), lambda: norm(q=grad(q)),
           lambda: norm(q_weight=grad(qw)), lambda: norm(q=q.transpose(1, 2)), lambda: norm(q=q.cpu()), lambda: norm(positions=pos.cpu()),
           lambda: put(cache=cache[:2]), lambda: put(cache=(ck, cv, sc[:, :, :19])), lambda: put(cache=(ck.float(), cv, sc)), lambda: put(cache=(ck, cv[:1], sc)),
           lambda: put(cache=(ck, cv, sc.double())), lambda: put(cache=(ck[:, :, ::2], cv[:, :, ::2], sc[:, :, ::2])), lambda: put(sinks=20), lambda: put(sinks=-1), lambda: put(v=v[:, :3]),
           lambda: put(k=k[..., :64], v=v[..., :64]), lambda: put(k=grad(k)), lambda: put(cache=(ck[:1].expand(2, -1, -1, -1), cv, sc)),
           lambda: put(cache=(ck, cv, sc[:1].expand(2, -1, -1, -1))), lambda: put(positions=pos[:1]),
           lambda: both(v=v.half()), lambda: both(k=q, v=q), lambda: both(cache=tuple(t[:, :1] for t in cache)), lambda: both(k_out=q), lambda: both(q_out=k)]
    before = [t.clone() for t in cache]
    for i, call in enumerate(bad):
        with pytest.raises(sana_amd.SanaHipError):
            call()
            pytest.fail(f"case {i} was taken")
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    empty = ops.qk_norm_rope(q[:, :0], k[:, :0], 4, qw, kw, freqs=f, positions=pos)
    assert empty[0].shape == (2, 0, 256) and empty[1].shape == (2, 0, 128)
    put(k=k[:, :0], v=v[:, :0])
    none = ops.qk_norm_rope(q[:0], k[:0], 4, qw, kw, freqs=f, positions=pos[:0])
    assert none[0].shape == (0, 4, 256)
