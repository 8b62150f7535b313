"""Attention over a sliding window and sinks, its ring cache and its single tokens against the definition in 64 bits."""
import math

import pytest
import torch

import sana_amd
from sana_amd import _lib, ops

gpu = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def definition(q, k, v, H, window, sinks, scale, lengths=None):
    """(out, the average of |v|, the largest sum of absolute products in a score), 64 bits, every query against every key."""
    B, N, C = q.shape
    Nk, d = k.shape[1], C // H
    G = k.shape[2] // d
    q, k, v = (t.double().reshape(B, t.shape[1], -1, d).transpose(1, 2) for t in (q, k, v))
    i, j = torch.arange(Nk - N, Nk)[:, None], torch.arange(Nk)[None, :]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    out, out_abs, size = torch.zeros(B, H, N, d, dtype=torch.float64), torch.zeros(B, H, N, d, dtype=torch.float64), 0.0
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        for h in range(H):
            kh, vh, m = k[b, h * G // H, :Nk - N + n], v[b, h * G // H, :Nk - N + n], seen[:n, :Nk - N + n]
            p = (q[b, h, :n] @ kh.T * scale).masked_fill(~m, -math.inf).softmax(1)
            out[b, h, :n], out_abs[b, h, :n] = p @ vh, p @ vh.abs()
            if n:
                size = max(size, scale * (q[b, h, :n].abs() @ kh.abs().T).max().item())
    rows = lambda t: t.transpose(1, 2).reshape(B, N, C)  # noqa: E731
    return rows(out), rows(out_abs), size


def check(got, want, keys, dtype):
    """A probability is off by half a step as it enters the product, the result by half a step of itself (or of the smallest
    f16).  In 32 bits: a score by the roundings of its chain of products (at most 16) and of its scale, its maximum and its
    power, each 2^-24 of the sum of its absolute terms, in p and in the sum of p; the sums by the roundings of their chains (a quarter of
    the keys a lane, the parts).  f16 probabilities, times 2^6, are off by 2^-25 where they are subnormal."""
    ref, ref_abs, size = want
    half = torch.finfo(dtype).eps / 2
    tol = half * (ref.abs() + ref_abs) + 2.0 ** -24 * (keys / 2 + 100 + 2 * 24 * 1.45 * size) * ref_abs
    if dtype == F16:
        tol = tol + 2.0 ** -25 + 2.0 ** -31 * keys * 6
    off = (got.double().cpu() - ref).abs()
    assert (off <= tol).all(), (off / tol).max().item()


def make(B, N, Nk, H, G, d, dtype, seed=0, packed=True, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(B, Nk, (H + 2 * G) * d, generator=g)).clamp(-6, 6).to(dtype)
    q, k, v = x.split([H * d, G * d, G * d], dim=2)
    q = q[:, Nk - N:]
    return (q, k, v) if packed else tuple(t.contiguous() for t in (q, k, v))


def to_gpu(*ts):
    if ts[0]._base is not None:
        base = ts[0]._base.cuda()
        return [base.as_strided(t.size(), t.stride(), t.storage_offset()) for t in ts]
    return [t.cuda() for t in ts]


def compare(q, k, v, H, window, sinks, scale=None, lengths=None):
    d = q.shape[2] // H
    want = definition(q, k, v, H, window, sinks, scale or d ** -0.5, lengths)
    got = ops.window_attention(*to_gpu(q, k, v), H, window, sinks, scale,
                               None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert got.dtype == q.dtype
    check(got, want, k.shape[1], q.dtype)
    return got


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 80, 96, 104, 112, 128])
def test_head_dims(cuda, d, dtype):
    compare(*make(2, 150, 200, 4, 2, d, dtype, seed=d), 4, 60, 3)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 64), (65, 4), (100, 130), (300, 1), (5000, 0), (5000, 5000)])
@pytest.mark.parametrize("N,past", [(1, 0), (2, 0), (64, 0), (127, 0), (129, 1), (300, 333), (3, 1000)])
def test_windows_and_sinks(cuda, N, past, window, sinks, dtype):
    compare(*make(1, N, past + N, 2, 1, 64, dtype, seed=N), 2, window, sinks)


@gpu
@pytest.mark.parametrize("H,G", [(1, 1), (6, 6), (6, 2), (8, 1), (20, 5)])
def test_shared_key_heads(cuda, H, G):
    compare(*make(2, 140, 170, H, G, 72, BF16), H, 50, 2)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,past", [(1, 4000), (5, 3333), (130, 2000), (64, 1985)])
def test_few_queries_of_many_keys_are_split_over_the_keys(cuda, N, past, dtype):
    assert _lib.load().sana_hip_window_attention_workspace_bytes(2, N, past + N, 2, 112, 1900, 70) > 0
    q, k, v = make(2, N, past + N, 2, 2, 112, dtype, packed=False)
    compare(q, k, v, 2, 1900, 70)
    compare(q, k, v, 2, 1900, 0)
    compare(q, k, v, 2, 9000, 70, lengths=[N, N // 2])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_of_every_size(cuda, dtype):
    """Rows that one key takes whole, a maximum that rises from tile to tile, and scores of thousands."""
    q, k, v = make(1, 200, 200, 2, 2, 64, dtype, packed=False)
    compare(q, k, v, 2, 150, 4, scale=30.0)
    ramp = torch.linspace(0.05, 6, 200)[None, :, None]
    compare((q.abs() * ramp).to(dtype), (k.abs() * ramp).to(dtype), v, 2, 150, 4, scale=1.0)
    compare((q.abs() * ramp.flip(1)).to(dtype), (k.abs() * ramp.flip(1)).to(dtype), v, 2, 150, 4, scale=1.0)
    compare(-q.abs() * 6, k.abs() * 6, v, 2, 150, 4, scale=4.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,past,window,sinks,d", [(300, 0, 70, 5, 112), (300, 20, 400, 0, 64), (5, 3333, 3000, 2, 112), (2500, 0, 100, 3, 128), (90, 7, 64, 0, 8)])
def test_values_that_are_not_finite_reach_who_sees_them(cuda, N, past, window, sinks, d, dtype):
    """A value of inf or NaN in front of a query's window, or behind the query: its output is what it is without; a query that sees it has
    the definition's inf or NaN in that channel.  A key of NaN makes the outputs of its head NaN for who sees it."""
    H, G, Nk = 20 if N > 1000 else 4, 2, N + past
    q, k, v = make(1, N, Nk, H, G, d, dtype, seed=N, packed=False)
    bad = [(1, 0, 3, math.inf), (Nk - N // 2, 0, 5, -math.inf), (Nk - N // 2 - 1, 1, 3, math.nan), (Nk - N // 2, 0, 6, math.inf),
           (Nk - N // 2 + 1, 0, 6, -math.inf), (Nk - 1, 1, 7, math.inf), (Nk - 2, 0, 3, math.inf)]
    i = torch.arange(Nk - N, Nk)
    sees = lambda j: (j <= i) & ((i - j < window) | (j < sinks))  # noqa: E731
    extra = torch.zeros(1, N, H, d, dtype=torch.float64)
    clean = v.clone()
    for j, g, c, x in bad:
        v[0, j, g * d + c], clean[0, j, g * d + c] = x, 0
        extra[0, sees(j), g * H // G:(g + 1) * H // G, c] += x
    want = definition(q, k, clean, H, window, sinks, d ** -0.5)
    extra = extra.reshape(1, N, H * d)

    def hold(got, extra):
        got = got.double().cpu()
        odd = extra != 0
        assert torch.equal(torch.nan_to_num(got[odd], nan=7.0, posinf=8.0, neginf=9.0), torch.nan_to_num(extra[odd], nan=7.0, posinf=8.0, neginf=9.0))
        check(torch.where(odd, want[0], got), want, Nk, dtype)

    hold(ops.window_attention(q.cuda(), k.cuda(), v.cuda(), H, window, sinks), extra)
    j = Nk - N // 2 - 1
    k[0, j, 2] = math.nan
    extra = extra.reshape(1, N, H, d)
    extra[0, sees(j), :H // G] = math.nan
    hold(ops.window_attention(q.cuda(), k.cuda(), v.cuda(), H, window, sinks), extra.reshape(1, N, H * d))


@gpu
@pytest.mark.parametrize("past", [0, 40, 2500])
def test_lengths_leave_rows_alone(cuda, past):
    N, H = 130, 2
    q, k, v = make(5, N, past + N, H, 1, 64, BF16, packed=False)
    lengths = [0, N, 67, N + 9, -4]
    for b, n in enumerate(lengths):
        q[b, max(n, 0):] = float("nan")
        k[b, past + max(n, 0):] = float("nan")
        v[b, past + max(n, 0):] = float("inf")
    clean = [torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (q, k, v)]
    want = definition(*clean, H, 90, 4, 0.125, lengths)
    out = torch.full_like(q, 7.0).cuda()
    dev = [t.cuda() for t in (q, k, v)]
    lengths_dev = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert ops.window_attention(*dev, H, 90, 4, None, lengths_dev, out) is out
    for b, n in enumerate(lengths):
        assert (out[b, max(n, 0):] == 7.0).all()
        out[b, max(n, 0):] = 0
    check(out, want, past + N, BF16)
    assert torch.equal(ops.window_attention(*dev, H, 90, 4, None, lengths_dev), out)


@gpu
def test_a_past_that_was_cut_short(cuda):
    """Of a long past only the sinks and the window in front of the queries: the same queries see the same keys."""
    N, past, W, S = 40, 700, 100, 3
    q, k, v = make(1, N, past + N, 2, 2, 64, BF16, packed=False)
    want = definition(q, k, v, 2, W, S, 0.125)
    kept = torch.cat([torch.arange(S), torch.arange(past - (W - 1), past + N)])
    got = ops.window_attention(q.cuda(), k[:, kept].cuda(), v[:, kept].cuda(), 2, W, S)
    check(got, want, past + N, BF16)


@gpu
def test_views_of_every_kind(cuda):
    B, N, H, d = 2, 150, 3, 40
    q, k, v = make(B, N, N, H, H, d, BF16, packed=False)
    want = ops.window_attention(*[t.cuda() for t in (q, k, v)], H, 70, 2)
    wide = torch.full((B, N + 9, 5, H * d + 8), float("nan"), dtype=BF16, device="cuda")
    views = [wide[:, 4:4 + N, i, 8:] for i in range(3)]
    for view, t in zip(views, (q, k, v)):
        view.copy_(t)
    assert torch.equal(ops.window_attention(*views, H, 70, 2, out=wide[:, 4:4 + N, 3, 4:-4]), want)
    assert torch.isnan(wide[:, :4]).all() and torch.isnan(wide[:, 4 + N:]).all() and torch.isnan(wide[:, :, 4]).all()
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1).cuda() for t in (q, k, v)]
    assert torch.equal(ops.window_attention(*swapped, H, 70, 2), want)


# --------------------------------------------------------------------------- the cache

def row_of(p, sinks, window):
    return p if p < sinks else sinks + (p - sinks) % window


def appended(cache, new, positions, sinks, lengths=None):
    """The cache after the tokens went in one by one."""
    cache = cache.clone()
    for b, pos in enumerate(positions):
        n = new.shape[1] if lengths is None else min(max(lengths[b], 0), new.shape[1])
        for t in range(n if pos >= 0 else 0):
            cache[b, row_of(pos + t, sinks, cache.shape[1] - sinks)] = new[b, t]
    return cache


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N", [1, 3, 50, 200])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 4), (37, 100)])
def test_append(cuda, window, sinks, N, dtype):
    g = torch.Generator().manual_seed(N)
    ck, cv = torch.randn(2, 6, sinks + window, 72, generator=g).to(dtype).unbind(0)
    k, v = torch.randn(6, N, 2 * 72, generator=g).to(dtype).split(72, dim=2)
    positions = [0, 3, sinks, -1, sinks + window, 2 ** 31 - 1 - N]
    for lengths in (None, [N, 0, N // 2, N, N + 5, -3]):
        a, b = ck.cuda(), cv.cuda()
        ops.window_cache_append_(a, b, *to_gpu(k, v), torch.tensor(positions, dtype=torch.int32, device="cuda"), sinks,
                                 None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        assert torch.equal(a.cpu(), appended(ck, k, positions, sinks, lengths))
        assert torch.equal(b.cpu(), appended(cv, v, positions, sinks, lengths))


def step_definition(q, k, v, ck, cv, positions, H, sinks, scale):
    """(caches after, out, averages of |v|, largest sum of absolute products)."""
    ck, cv = appended(ck, k, positions, sinks), appended(cv, v, positions, sinks)
    B, _, C = q.shape
    d = C // H
    G = k.shape[2] // d
    out, out_abs, size = torch.zeros(B, 1, C, dtype=torch.float64), torch.zeros(B, 1, C, dtype=torch.float64), 0.0
    for b, p in enumerate(positions):
        if p < 0:
            continue
        n = min(p + 1, ck.shape[1])
        for h in range(H):
            at, kv = slice(h * d, (h + 1) * d), slice(h * G // H * d, (h * G // H + 1) * d)
            kh, vh, qh = ck[b, :n, kv].double(), cv[b, :n, kv].double(), q[b, 0, at].double()
            w = torch.softmax(kh @ qh * scale, 0)
            out[b, 0, at], out_abs[b, 0, at] = w @ vh, w @ vh.abs()
            size = max(size, scale * (kh.abs() @ qh.abs()).max().item())
    return ck, cv, (out, out_abs, size)


def step_compare(B, H, G, d, window, sinks, positions, dtype, seed=0, scale=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, 1, (H + 2 * G) * d, generator=g).clamp(-6, 6).to(dtype)
    q, k, v = x.split([H * d, G * d, G * d], dim=2)
    ck, cv = torch.randn(2, B, sinks + window, G * d, generator=g).clamp(-6, 6).to(dtype).unbind(0)
    for b, p in enumerate(positions):   # rows that hold no token yet
        ck[b, max(p, 0):] = ck[b, max(p, 0):] if p >= sinks + window else float("nan")
        cv[b, max(p, 0):] = cv[b, max(p, 0):] if p >= sinks + window else float("inf")
    want_k, want_v, want = step_definition(q, k, v, ck, cv, positions, H, sinks, scale or d ** -0.5)
    a, b = ck.cuda(), cv.cuda()
    out = torch.full((B, 1, H * d), float("nan"), dtype=dtype, device="cuda")
    got = ops.window_attention_step_(*to_gpu(q, k, v), a, b, torch.tensor(positions, dtype=torch.int32, device="cuda"), H, sinks,
                                     scale, out)
    assert got is out
    assert torch.equal(a.cpu().view(torch.int16), want_k.view(torch.int16)) and torch.equal(b.cpu().view(torch.int16), want_v.view(torch.int16))
    check(got, want, sinks + window, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 80, 96, 112, 128])
def test_step_head_dims(cuda, d, dtype):
    step_compare(3, 6, 2, d, 70, 4, [5, 74, 300], dtype, seed=d)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (31, 1), (32, 0), (250, 6), (3000, 40)])
def test_step_positions(cuda, window, sinks, dtype):
    """Empty, young, just full, wrapped and idle streams; rows that hold nothing yet are full of NaN and inf."""
    rows = window + sinks
    step_compare(9, 2, 1, 64, window, sinks, [0, 1, -1, max(sinks - 1, 0), sinks, rows - 1, rows, 3 * rows + 5, 2 ** 31 - 1], dtype)


@gpu
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (16, 1), (17, 1), (40, 2), (20, 5)])
def test_step_shared_key_heads(cuda, H, G):
    step_compare(2, H, G, 112, 600, 4, [90, 5000], BF16)
    step_compare(70, H, G, 32, 90, 4, [9 * i for i in range(70)], F16)


@gpu
def test_step_scores_of_thousands(cuda):
    step_compare(2, 2, 1, 64, 500, 4, [400, 800], BF16, scale=20.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [5, 33, 700, 4000])
def test_step_values_that_are_not_finite(cuda, rows, dtype):
    """The newest token's value of inf, a row that the last tile of rows holds alone or with others that are not there yet: inf, not NaN."""
    g = torch.Generator().manual_seed(rows)
    q, k, v = (torch.randn(1, 1, 128, generator=g).to(dtype) for _ in range(3))
    ck, cv = torch.randn(2, 1, rows + 90, 128, generator=g).to(dtype).unbind(0)
    v[0, 0, 3], v[0, 0, 70] = math.inf, -math.inf
    want_k, want_v, want = step_definition(q, k, v, ck, cv, [rows - 1], 2, 4, 0.125)
    got = ops.window_attention_step_(q.cuda(), k.cuda(), v.cuda(), ck.cuda(), cv.cuda(), torch.tensor([rows - 1], dtype=torch.int32, device="cuda"), 2, 4)
    assert got[0, 0, 3] == math.inf and got[0, 0, 70] == -math.inf
    fine = torch.isfinite(want[0])
    assert fine.sum() == 126
    zero = torch.zeros(1, dtype=torch.float64)
    check(torch.where(fine, got.double().cpu(), zero), (torch.where(fine, want[0], zero), torch.where(fine, want[1], zero), want[2]), rows, dtype)


@gpu
def test_a_cache_of_more_than_32_bits_of_bytes(cuda):
    """Streams whose rows lie further into a cache than 2^31 elements and 2^32 bytes."""
    B, rows, C = 3, 9000, 1 << 17
    base = torch.zeros(B, rows, C, dtype=BF16, device="cuda")   # 7 GB
    H, G, d = 2, 1, 64
    ck, cv = base[:, :, :64], base[:, :, 64:128]
    g = torch.Generator().manual_seed(1)
    new = torch.randn(2, B, 500, 64, generator=g).to(BF16)
    positions = torch.tensor([8800, 8600, 9100], dtype=torch.int32, device="cuda")
    ops.window_cache_append_(ck, cv, new[0].cuda(), new[1].cuda(), positions, 0)
    want_k = appended(torch.zeros(B, rows, 64, dtype=BF16), new[0], positions.tolist(), 0)
    want_v = appended(torch.zeros(B, rows, 64, dtype=BF16), new[1], positions.tolist(), 0)
    assert torch.equal(ck.cpu(), want_k) and torch.equal(cv.cpu(), want_v)
    x = torch.randn(B, 1, 4 * 64, generator=g).to(BF16)
    q, k, v = x.split([128, 64, 64], dim=2)
    positions += 500
    want = step_definition(q, k, v, want_k, want_v, positions.tolist(), H, 0, 0.125)
    got = ops.window_attention_step_(*to_gpu(q, k, v), ck, cv, positions, H)
    check(got, want[2], rows, BF16)
    assert torch.equal(ck.cpu(), want[0]) and torch.equal(cv.cpu(), want[1]) and not base[:, :, 128:].any()


# --------------------------------------------------------------------------- refusals

@gpu
def test_refusals(cuda):
    q, k, v = (t.contiguous().cuda() for t in make(2, 8, 8, 4, 2, 32, BF16, packed=False))
    ck, cv = torch.zeros(2, 2, 20, 64, dtype=BF16, device="cuda").unbind(0)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    w, s, a = ops.window_attention, ops.window_attention_step_, ops.window_cache_append_
    q1, k1, v1 = q[:, :1], k[:, :1], v[:, :1]
    odd = torch.zeros(2 * 8 * 128 + 1, dtype=BF16, device="cuda")[1:].view(2, 8, 128)
    bad = [lambda: w(q.float(), k.float(), v.float(), 4, 5), lambda: w(q, k.half(), v, 4, 5), lambda: w(q, k, v, 3, 5),
           lambda: w(q, k, v, 4, 0), lambda: w(q, k, v, 4, 5, -1), lambda: w(q, k, v, 4, 5, scale=0.0), lambda: w(q, k, v, 4, 5, scale=-1.0),
           lambda: w(q, k, v, 4, 5, scale=float("nan")), lambda: w(q, k, v, 4, 1 << 31),
           lambda: w(q, k[:, :4], v[:, :4], 4, 5), lambda: w(q, k, v[:, :, :32], 4, 5), lambda: w(q[..., :96], k, v, 3, 5),
           lambda: w(q[..., :112], k[..., :56], v[..., :56], 4, 5), lambda: w(odd, k, v, 4, 5), lambda: w(q, k, v, 4, 5, out=q[:, :4]),
           lambda: w(q, k, v, 4, 5, lengths=pos.long()), lambda: w(q, k, v, 4, 5, lengths=pos[:1]), lambda: w(q, k, v, 4, 5, lengths=pos.cpu()),
           lambda: w(q.clone().requires_grad_(), k, v, 4, 5), lambda: w(q, k[:1].expand(2, 8, 64)[:, :1].expand(2, 8, 64), v, 4, 5),
           lambda: w(q, k, v, 4, 5, scale=float("inf")), lambda: w(q, k, v, 4, 5, out=torch.empty_like(q[:1]).expand(2, 8, 128)),
           lambda: s(q1, k1, v1, ck[:1].expand(2, 20, 64), cv, pos, 4), lambda: a(ck, cv[:1].expand(2, 20, 64), k, v, pos),
           lambda: s(q, k, v, ck, cv, pos, 4), lambda: s(q1, k1, v1, ck[:1], cv[:1], pos, 4), lambda: s(q1, k1, v1, ck, cv[:, :9], pos, 4),
           lambda: s(q1, k1, v1, ck.half(), cv.half(), pos, 4), lambda: s(q1, k1, v1, ck, cv, pos, 4, 20), lambda: s(q1, k1, v1, ck, cv, pos, 4, -1),
           lambda: s(q1, k1, v1, ck, cv, pos.long(), 4), lambda: s(q1, k1, v1, ck, cv, None, 4), lambda: s(q1, k1, v1, ck, cv, pos, 5),
           lambda: a(ck, cv, k.half(), v.half(), pos), lambda: a(ck, cv, k, v[:, :3], pos), lambda: a(ck, cv, k, v, pos, 20),
           lambda: a(ck, cv[:, :19], k, v, pos), lambda: a(ck, cv, k, v, pos[:1]), lambda: a(ck, cv, k, v, pos, lengths=pos.long()),
           lambda: a(ck[..., :36], cv[..., :36], k[..., :36], v[..., :36], pos), lambda: a(ck.cpu(), cv, k, v, pos)]
    for i, f in enumerate(bad):
        with pytest.raises(sana_amd.SanaHipError):
            f()
            pytest.fail(f"case {i} was taken")
    assert w(q[:, :0], k, v, 4, 5).shape == (2, 0, 128) and w(q[:0], k[:0], v[:0], 4, 5).shape == (0, 8, 128)
    assert s(q1[:0], k1[:0], v1[:0], ck[:0], cv[:0], pos[:0], 4).shape == (0, 1, 128)
    a(ck, cv, k[:, :0], v[:, :0], pos)
    assert not ck.any() and not cv.any()


def test_c_entries_refuse_before_any_launch():
    """Host checks: the pointers below are never followed."""
    lib, P, bf16 = _lib.load(), 0x10000, _lib.DT_BF16
    #       q  k  v out len  ws   B  N  Nk  H  G  d  W  S   strides
    good = [P, P, P, P, None, None, 0, 1, 200, 200, 64, 32, 64, 50, 4] + [200 * 4096, 4096, 200 * 2048, 2048, 200 * 2048, 2048, 200 * 4096, 4096, 0.1, bf16]
    call = lambda *change: lib.sana_hip_window_attention(*[dict(change).get(i, x) for i, x in enumerate(good)], None)  # noqa: E731
    for i in range(4):
        assert call((i, None)) == -1
    for i in (7, 8, 9, 10, 11, 12, 13):
        assert call((i, 0)) == -1
    assert call((9, 199)) == -1 and call((14, -1)) == -1 and call((11, 7)) == -1 and call((23, 0.0)) == -1 and call((23, float("nan"))) == -1
    assert call((24, _lib.DT_F32)) == -6
    assert call((12, 60)) == -2 and call((12, 136)) == -2 and call((13, 1 << 31 - 1)) != 0
    for i in (16, 18, 20, 22):
        assert call((i, 1024)) == -1
        assert call((i - 1, -8)) == -1
    assert call((18, 1 << 23)) == -2 and call((16, 4100)) == -3 and call((0, P + 8)) == -3 and call((3, P + 4)) == -3 and call((4, P + 2)) == -3
    few = ((8, 2), (9, 8000), (10, 2), (11, 1), (13, 6000))
    need = lib.sana_hip_window_attention_workspace_bytes(1, 2, 8000, 2, 64, 6000, 4)
    assert need > 0 and call(*few) == -4 and call(*few, (5, P), (6, need - 1)) == -4 and call(*few, (5, P + 8), (6, need)) == -3
    #       q  k  v ck cv pos out ws      B  H  G  d   W   S
    good = [P, P, P, P, P, P, P, None, 0, 64, 64, 32, 64, 100, 4] + [4096, 2048, 2048, 104 * 2048, 2048, 104 * 2048, 2048, 4096, 0.1, bf16]
    step = lambda *change: lib.sana_hip_window_step(*[dict(change).get(i, x) for i, x in enumerate(good)], None)  # noqa: E731
    for i in range(7):
        assert step((i, None)) == -1
    for i in (9, 10, 11, 12, 13):
        assert step((i, 0)) == -1
    many = ((9, 2),)
    assert step(*many, (18, 0)) == -1 and step(*many, (20, 0)) == -1 and step(*many, (22, 0)) == -1 and step((13, 1 << 30)) == -2
    assert step((23, float("inf"))) == -1
    assert step((14, -1)) == -1 and step((11, 7)) == -1 and step((23, -1.0)) == -1 and step((24, 0)) == -6 and step((12, 132)) == -2
    assert step((19, 1024)) == -1 and step((21, 1024)) == -1 and step((18, -8)) == -1 and step((15, 4100)) == -3 and step((5, P + 2)) == -3
    need = lib.sana_hip_window_step_workspace_bytes(1, 4, 2, 64, 4000, 4)
    few = ((9, 1), (10, 4), (11, 2), (13, 4000))
    assert need > 0 and step(*few) == -4 and step(*few, (7, P), (8, need - 1)) == -4 and step(*few, (7, P + 8), (8, need)) == -3
    #       ck cv k  v pos len  B  N   C    W   S
    good = [P, P, P, P, P, None, 2, 10, 256, 50, 4] + [54 * 256, 256] * 2 + [2560, 256] * 2 + [bf16]
    put = lambda *change: lib.sana_hip_window_cache_append(*[dict(change).get(i, x) for i, x in enumerate(good)], None)  # noqa: E731
    for i in range(5):
        assert put((i, None)) == -1
    for i in (6, 7, 8, 9):
        assert put((i, 0)) == -1
    assert put((11, 0)) == -1 and put((13, 0)) == -1 and put((9, 1 << 30)) == -2
    assert put((10, -1)) == -1 and put((8, 252)) == -2 and put((6, 70000)) == -2 and put((19, 0)) == -6 and put((12, 128)) == -1
    assert put((0, P + 2)) == -3 and put((15, 2564)) == -3 and put((17, -8)) == -1


def test_c_entries_refuse_launches_of_too_many_threads():
    """Host checks of sizes whose grids no launch takes (2^32 threads an axis), and of a scale that overflows in powers of two."""
    lib, P, bf16 = _lib.load(), 0x10000, _lib.DT_BF16
    rows = [200 * 4096, 4096, 200 * 2048, 2048, 200 * 2048, 2048, 200 * 4096, 4096]
    prompt = lambda B, scale: lib.sana_hip_window_attention(P, P, P, P, None, None, 0, B, 200, 200, 64, 32, 64, 50, 4, *rows, scale, bf16, None)  # noqa: E731
    assert prompt(1 << 16, 0.1) == -2 and prompt(1, 3e38) == -1
    step = lambda B, scale: lib.sana_hip_window_step(P, P, P, P, P, P, P, None, 0, B, 64, 32, 64, 100, 4, 4096, 2048, 2048, 104 * 2048,  # noqa: E731
                                                     2048, 104 * 2048, 2048, 4096, scale, bf16, None)
    assert step(1 << 19, 0.1) == -2 and step(1, 3e38) == -1
    assert lib.sana_hip_window_cache_append(P, P, P, P, P, None, 2, 1 << 27, 256, 50, 4, 54 * 256, 256, 54 * 256, 256, 2560, 256, 2560, 256, bf16, None) == -2


def test_cpu_tensors_are_refused():
    q, k, v = make(1, 4, 4, 2, 2, 32, BF16, packed=False)
    with pytest.raises(sana_amd.SanaHipError):
        ops.window_attention(q, k, v, 2, 3)
    with pytest.raises(sana_amd.SanaHipError):
        ops.window_attention_step_(q[:, :1], k[:, :1], v[:, :1], k, v, torch.zeros(1, dtype=torch.int32), 2)
    with pytest.raises(sana_amd.SanaHipError):
        ops.window_cache_append_(k, v, k, v, torch.zeros(1, dtype=torch.int32))
