"""Single tokens over a cache of 8 bits, a cache's rows in order, and a stream's whole turn."""
import math

import pytest
import torch

import sana_amd
from sana_amd import _lib, ops
from test_gpu_heads import U, filled, freqs_of, i32, make
from test_gpu_window_attention import definition as window_definition
from test_gpu_window_attention import row_of

gpu = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def realistic(B, G, R, d, seed=1):
    ck, cv, sc = filled(B, G, R, d, seed)
    return ck, cv, (0.5 + sc) * 2.5 / 127


def definition(q, cache, positions, H, sinks, scale):
    """(out, averages of |v|, the largest sum of absolute products in a score), 64 bits."""
    ck, cv, sc = cache
    B, G, R, _ = ck.shape
    d = q.shape[2] // H
    out, out_abs, size = torch.zeros(B, 1, H, d, dtype=torch.float64), torch.zeros(B, 1, H, d, dtype=torch.float64), 0.0
    for b, p in enumerate(positions):
        n = min(p + 1, R)
        for h in range(H if p >= 0 else 0):
            g = h * G // H
            k = ck[b, g, :n, :d].double() * sc[b, g, :n, :1].double()
            v = cv[b, g, :n, :d].double() * sc[b, g, :n, 1:].double()
            x = q[b, 0, h * d:(h + 1) * d].double()
            w = torch.softmax(k @ x * scale, 0)
            out[b, 0, h], out_abs[b, 0, h] = w @ v, w @ v.abs()
            size = max(size, scale * (k.abs() @ x.abs()).max().item())
    return out.flatten(2), out_abs.flatten(2), size


def check(got, want, keys):
    """The result by half a step of itself (or of the smallest f16).  In front of it: a probability with its value's scale as two bf16 numbers, half
    a step of half a step, 2^-16; in 32 bits a score by the roundings of its chain of products (at most 16), of the scales' product and of that with them,
    its maximum and its power, each U of the sum of its absolute terms, in p and in the sum of p; the sums by the roundings of their chains (a
    quarter of the keys a lane, the parts)."""
    ref, ref_abs, size = want
    half = torch.finfo(got.dtype).eps / 2
    tol = half * ref.abs() + (2.0 ** -16 + U * (keys / 2 + 100 + 2 * 26 * 1.45 * size)) * ref_abs + (2.0 ** -25 if got.dtype == F16 else 0)
    off = (got.double().cpu() - ref).abs()
    assert (off <= tol).all(), (off / tol).max().item()


def compare(B, H, G, d, window, sinks, positions, dtype, seed=0, scale=None, spoil=True):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, 1, H * d, generator=g).clamp(-6, 6).to(dtype)
    cache = realistic(B, G, sinks + window, d, seed)
    want = definition(q, cache, positions, H, sinks, scale or d ** -0.5)
    if spoil:
        for b, p in enumerate(positions):   # rows that hold no token yet
            cache[2][b, :, max(p + 1, 0):] = math.nan
    out = torch.full((B, 1, H * d), math.nan, dtype=dtype, device="cuda")
    dev = [t.cuda() for t in cache]
    got = ops.window_attention_q8(q.cuda(), dev, i32(positions), H, sinks, scale, out)
    assert got is out
    check(got, want, sinks + window)
    assert all(torch.equal(a.cpu().view(torch.int8 if a.dtype == torch.int8 else torch.int32), b.view(torch.int8 if b.dtype == torch.int8 else torch.int32))
               for a, b in zip(dev, cache))
    return got


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", list(range(8, 129, 8)))
def test_head_dims(cuda, d, dtype):
    compare(3, 6, 2, d, 70, 4, [5, 74, 300], dtype, seed=d)
    compare(2, 2, 1, d, 4000, 4, [3000, 74000], dtype, seed=d)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (31, 1), (32, 0), (64, 1), (250, 6), (6000, 40)])
def test_positions(cuda, window, sinks, dtype):
    """Young, just full, wrapped and idle streams; the scales of rows that hold nothing yet are NaN."""
    rows = window + sinks
    compare(9, 2, 1, 64, window, sinks, [0, 1, -1, max(sinks - 1, 0), sinks, rows - 1, rows, 3 * rows + 5, 2 ** 31 - 1], dtype)


@gpu
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (16, 1), (17, 1), (40, 2), (20, 5)])
def test_shared_key_heads(cuda, H, G):
    compare(2, H, G, 112, 600, 4, [90, 5000], BF16)
    compare(70, H, G, 32, 90, 4, [9 * i for i in range(70)], F16)
    compare(3, H, G, 72, 2500, 0, [2000, 5000, 17], F16)


@gpu
@pytest.mark.parametrize("B,H,G,d,rows", [(1, 1, 1, 128, 40000), (1, 32, 8, 128, 9000), (130, 4, 4, 112, 1500), (260, 2, 1, 64, 700)])
def test_parts_and_whole(cuda, B, H, G, d, rows):
    compare(B, H, G, d, rows - 3, 3, [(rows // 2 + 37 * i) % (2 * rows) for i in range(B)], BF16)


@gpu
@pytest.mark.parametrize("d", [16, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("B,H,G,rows", [(40, 4, 2, 60), (33, 3, 3, 100), (100, 2, 2, 37), (1, 3, 1, 9000), (2, 2, 1, 7000)])
def test_values_over_several_workgroups(cuda, B, H, G, rows, d):
    """64, 80, 99 and 200 workgroups of whole caches, few of long ones in parts: a workgroup takes 32 channels of the values, half of them, or all; idle streams' zeros too."""
    compare(B, H, G, d, rows - 2, 2, [-1 if i % 7 == 3 else (rows // 2 + 11 * i) % (3 * rows) for i in range(B)], BF16, seed=d)


@gpu
def test_scores_of_thousands(cuda):
    compare(2, 2, 1, 64, 500, 4, [400, 800], BF16, scale=20.0)
    compare(2, 2, 1, 64, 5000, 4, [400, 8000], F16, scale=20.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [5, 33, 700, 9000])
def test_a_row_that_is_not_finite_reaches_its_head(cuda, rows, dtype):
    """The scale NaN of a key or a value, the newest or another that is seen: NaN in the outputs of the heads that share it, in no others."""
    H, G, d = 4, 2, 64
    g = torch.Generator().manual_seed(rows)
    q = torch.randn(1, 1, H * d, generator=g).to(dtype)
    cache = realistic(1, G, rows + 90, d)
    clean = ops.window_attention_q8(q.cuda(), [t.cuda() for t in cache], i32([rows - 1]), H, 4)
    for at, i in ((rows - 1, 0), (rows - 1, 1), (rows // 2, 1), (0, 0)):
        odd = cache[2].clone()
        odd[0, 1, at, i] = math.nan
        got = ops.window_attention_q8(q.cuda(), (cache[0].cuda(), cache[1].cuda(), odd.cuda()), i32([rows - 1]), H, 4)
        assert torch.isnan(got[..., 2 * d:]).all() and torch.equal(got[..., :2 * d], clean[..., :2 * d])


@gpu
@pytest.mark.parametrize("scale", [None, 3.0])
@pytest.mark.parametrize("B,H,G,d,rows", [(2, 4, 2, 64, 40), (1, 4, 4, 72, 700), (2, 20, 1, 128, 700), (2, 4, 2, 64, 9000), (130, 2, 2, 40, 100)])
@pytest.mark.parametrize("kind", ["huge", "tiny", "zeros", "any", "huge last", "huge first", "tiny first"])
def test_values_of_any_size(cuda, kind, B, H, G, d, rows, scale):
    """Values next to the largest number of their type, next to the smallest, of all sizes side by side: averages of them, which are finite.

    Where some rows are huge, they are zero in every other channel, whose outputs are those of the other rows.  A score's distance from its reference is
    up to 56 + 8 larger than without (the lift and the lazy maximum), which is rounded: 64 ln 2 U of a probability, in it and in the sums.  An output that is
    no normal number is off by half of the smallest bf16 number, and what it is rounded from by half of the smallest fp32 number."""
    g = torch.Generator().manual_seed(rows)
    q = torch.randn(B, 1, H * d, generator=g).clamp(-6, 6).to(BF16)
    k, v = (torch.randn(B, rows, G * d, generator=g).clamp(-1, 1) for _ in range(2))
    at, huge, tiny = torch.arange(rows), 3.3e38, 2.0 ** -122
    size = {"huge": torch.full((rows,), huge), "tiny": torch.full((rows,), tiny), "zeros": torch.zeros(rows),
            "any": 2.0 ** (torch.rand(rows, generator=g) * 187 - 60), "huge last": torch.where(at >= rows - rows // 4, huge, 1.0),
            "huge first": torch.where(at < rows // 4, huge, 1.0), "tiny first": torch.where(at < rows // 4, tiny, 1.0)}[kind]
    v = v * size[:, None]
    if kind.startswith("huge "):
        v[..., ::2] *= (size[:, None] <= 1)
    v = v.clamp(-huge, huge).to(BF16)
    cache = [t.cuda() for t in filled(B, G, rows, d)]
    ops.window_cache_append_q8_(cache, k.to(BF16).cuda(), v.cuda(), i32([0] * B))
    positions = [rows - 1 - i % 3 for i in range(B)]
    got = ops.window_attention_q8(q.cuda(), cache, i32(positions), H, 0, scale)
    assert torch.isfinite(got).all()
    ref, ref_abs, most = definition(q, [t.cpu() for t in cache], positions, H, 0, scale or d ** -0.5)
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -16 + U * (rows / 2 + 100 + 2 * 26 * 1.45 * most + 2 * 64 * math.log(2))) * ref_abs + 2.0 ** -134 + 2.0 ** -150
    off = (got.double().cpu() - ref).abs()
    assert (off <= tol).all(), (off / tol).max().item()


@gpu
def test_streams_of_a_pool(cuda):
    """Every other stream of a larger cache, outputs and queries among other rows."""
    B, H, G, d, R = 3, 4, 2, 40, 200
    q = torch.randn(B, 1, H * d, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    pool = [t.cuda() for t in realistic(2 * B, G, R, d)]
    part = [t[::2] for t in pool]
    pos = i32([50, 199, 1000])
    want = ops.window_attention_q8(q, [t.contiguous() for t in part], pos, H, 3)
    wide = torch.full((B, 1, H * d + 16), math.nan, dtype=BF16, device="cuda")
    ops.window_attention_q8(q, part, pos, H, 3, out=wide[..., 8:-8])
    assert torch.equal(wide[..., 8:-8], want) and torch.isnan(wide[..., :8]).all() and torch.isnan(wide[..., -8:]).all()
    k, v = (torch.randn(B, 5, G * d, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in (1, 2))
    before = [t.clone() for t in pool]
    dense = [t.contiguous() for t in part]
    ops.window_cache_append_q8_(part, k, v, pos, 3), ops.window_cache_append_q8_(dense, k, v, pos, 3)
    assert all(torch.equal(a, b) for a, b in zip(part, dense)) and all(torch.equal(a[1::2], b[1::2]) for a, b in zip(pool, before))
    for got, ref in zip(ops.window_cache_read(part, pos, 3, dim=d), ops.window_cache_read(dense, pos, 3, dim=d)):
        assert torch.equal(got, ref)


# --------------------------------------------------------------------------- rows in order

def in_order(cache, positions, sinks, last, fill, rows_of):
    """rows_of(b, row) of each token in order -> [B, sinks + last, C], `fill` behind the last one."""
    B = cache[0].shape[0]
    R = cache[0].shape[2] if len(cache) == 3 else cache[0].shape[1]
    out = fill.clone()
    for b, n in enumerate(positions):
        n = max(n, 0)
        tokens = range(n) if n <= sinks + last else [*range(sinks), *range(n - last, n)]
        for i, t in enumerate(tokens):
            out[b, i] = rows_of(b, row_of(t, sinks, R - sinks))
    return out


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("G,d,window,sinks,last", [(2, 72, 37, 5, None), (3, 32, 64, 0, 63), (1, 128, 1, 3, 0), (5, 112, 200, 1, 40), (2, 8, 16, 16, 16), (7, 40, 100, 0, 1), (1, 8, 300, 7, 299), (2, 128, 90, 0, 90), (1, 104, 500, 3, 411), (3, 88, 64, 1, 60)])
def test_rows_in_order(cuda, G, d, window, sinks, last, bits, dtype):
    R = window + sinks
    cache = realistic(9, G, R, d)
    if bits == 16:
        cache = [torch.randn(9, R, G * d, generator=torch.Generator().manual_seed(i)).to(dtype) for i in (0, 1)]
    M = sinks + (window if last is None else last)
    positions = [0, 1, -3, sinks, M, M + 1, R, 3 * R + 2, 2 ** 31 - 1]
    dev = [t.cuda() for t in cache]
    for given in (False, True):
        fill = torch.full((9, M, G * d), 7.0 if given else 0.0, dtype=dtype)
        out = [fill.clone().cuda() for _ in range(2)] if given else None
        half = torch.finfo(dtype).eps / 2
        got = ops.window_cache_read(dev, i32(positions), sinks, last, d if bits == 8 else None, dtype, out)
        for i in (0, 1):
            if bits == 16:
                assert torch.equal(got[i].cpu(), in_order(cache, positions, sinks, last if last is not None else window, fill, lambda b, r: cache[i][b, r]))
            else:
                # A product of 7 and 24 bits, exact in 64.  It may be rounded to 32 bits (U of itself) before it is to 16 (half a step of what that left) or
                # not: the two differ where 32 bits put it on a tie, so no order of them is asked for bit by bit.
                want = in_order(cache, positions, sinks, last if last is not None else window, fill.double(),
                                lambda b, r: (cache[i][b, :, r, :d].double() * cache[2][b, :, r, i, None].double()).flatten())
                tol = (half * (1 + U) + U) * want.abs() + (2.0 ** -25 if dtype == F16 else 0)
                assert ((got[i].cpu().double() - want).abs() <= tol).all()
                assert torch.equal(got[i].cpu() == fill, want == fill.double())
            assert not given or got[i] is out[i]


@gpu
@pytest.mark.parametrize("bits", [8, 16])
def test_rows_into_the_front_of_a_buffer(cuda, bits):
    """Views: every other stream of a cache, the front rows of wide buffers, keys and values side by side."""
    B, G, d, R, sinks = 3, 2, 64, 50, 4
    cache = [t.cuda() for t in realistic(2 * B, G, R, d)]
    if bits == 16:
        cache = [torch.randn(2 * B, R, G * d + 8, device="cuda").to(BF16)[..., 8:] for _ in range(2)]
    part, pos = [t[1::2] for t in cache], i32([60, 50, 777])
    want = ops.window_cache_read([t.contiguous() for t in part], pos, sinks, 45)
    buf = torch.full((B, 49 + 10, 2 * G * d), 9.0, dtype=BF16, device="cuda")
    ops.window_cache_read(part, pos, sinks, 45, out=(buf[:, :49, :G * d], buf[:, :49, G * d:]))
    assert torch.equal(buf[:, :49], torch.cat(want, -1)) and (buf[:, 49:] == 9).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits", [8, 16])
def test_a_stream_from_its_prompt_to_its_tokens(cuda, bits, dtype):
    """Three chunks and five tokens of two streams, each chunk behind the rows that the cache gives back; against the attention, in 64 bits, over what
    each query's cache held (its codes times their scales), so that what 8 bits take from the keys is no part of the difference."""
    B, H, G, d, W, S, r = 2, 4, 2, 64, 96, 3, 32
    R, chunk, f = W + S, 70, freqs_of(32).cuda()
    cache = ops.window_cache_q8(B, R, G, d) if bits == 8 else tuple(torch.zeros(B, R, G * d, dtype=dtype, device="cuda") for _ in range(2))
    seen, pos = 0, torch.zeros(B, dtype=torch.int32, device="cuda")
    for turn in range(3):
        q, k, v, qw, kw = (t.cuda() for t in make(B, chunk, H, G, d, dtype, seed=turn))
        args = (H, qw, kw, 1e-6, f)
        held = min(seen, S + W - 1)
        rows = torch.empty(2, B, held + chunk, G * d, dtype=dtype, device="cuda")
        if held:
            last = held - S
            ops.window_cache_read(cache, pos, S, last, d if bits == 8 else None, dtype, out=rows[:, :, :held].unbind(0))
        q, k = ops.qk_norm_rope(q, k, *args, positions=pos)
        rows[0, :, held:], rows[1, :, held:] = k, v
        got = ops.window_attention(q, rows[0], rows[1], H, W, S)
        ref, ref_abs, size = window_definition(q.cpu(), rows[0].cpu(), rows[1].cpu(), H, W, S, d ** -0.5)
        half = torch.finfo(dtype).eps / 2     # the probabilities' rounding and the result's
        tol = half * (ref.abs() + ref_abs) + U * (held + chunk + 100 + 80 * size) * ref_abs + (2.0 ** -24 if dtype == F16 else 0)
        assert ((got.double().cpu() - ref).abs() <= tol).all()
        if bits == 8:
            ops.window_cache_append_q8_(cache, k, v, pos, S)
        else:
            ops.window_cache_append_(*cache, k, v, pos, S)
        seen += chunk
        pos += chunk
        # what the cache holds is what the chunk put there, in order
        back = ops.window_cache_read(cache, pos, S, min(seen, R) - S, d if bits == 8 else None, dtype)
        n = min(chunk, W)
        step = 1 / 254 if bits == 8 else 0     # of a head's largest value
        for x, y in zip(back, (k, v)):
            x, y = (t[:, -n:].float().unflatten(2, (G, d)) for t in (x, y))
            most = y.abs().amax(-1, keepdim=True)
            assert ((x - y).abs() <= (step * 1.001 + half) * most).all()
    for turn in range(5 if bits == 8 else 0):
        q, k, v, qw, kw = (t.cuda() for t in make(B, 1, H, G, d, dtype, seed=9 + turn))
        q, _ = ops.qk_norm_rope_append_q8_(q, k, v, cache, pos, H, qw, kw, 1e-6, f, sinks=S)
        got = ops.window_attention_q8(q, cache, pos, H, S)
        check(got, definition(q.cpu(), [t.cpu() for t in cache], pos.tolist(), H, S, d ** -0.5), R)
        pos += 1


@gpu
def test_replayed_turns(cuda):
    """A token's turn, captured once: each replay is what the eager calls give, with eager work and other sizes in between; two graphs side by side."""
    B, H, G, d, W, S = 3, 8, 2, 64, 3000, 4
    f = freqs_of(64).cuda()

    def state(seed):
        q, k, v, qw, kw = (t.cuda() for t in make(B, 1, H, G, d, BF16, seed=seed))
        return dict(q=q.contiguous(), k=k.contiguous(), v=v.contiguous(), w=(qw, kw), cache=[t.cuda() for t in realistic(B, G, W + S, d, seed)], pos=i32([9, 2000, 7000]))

    def turn(s):
        q, _ = ops.qk_norm_rope_append_q8_(s["q"], s["k"], s["v"], s["cache"], s["pos"], H, *s["w"], 1e-6, f, sinks=S)
        rows = ops.window_cache_read(s["cache"], s["pos"], S, 10)
        return ops.window_attention_q8(q, s["cache"], s["pos"], H, S), *rows

    states = [state(i) for i in range(2)]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for s in states:
            turn(s)
    torch.cuda.current_stream().wait_stream(stream)
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(turn(s))
        graphs.append(g)
    sides = [torch.cuda.Stream() for _ in graphs]
    for round_ in range(4):
        for s in states:
            for n in "qkv":
                s[n].copy_(torch.randn(s[n].shape, generator=torch.Generator().manual_seed(50 + round_)).to(BF16))
            s["pos"] += 1
        eager = []
        for s in states:
            twin = {**s, "cache": [t.clone() for t in s["cache"]]}
            eager.append((turn(twin), twin["cache"]))
        compare(2, 3, 1, 32, 2000, 0, [5, 9000], F16)
        torch.cuda.synchronize()
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                g.replay()
        torch.cuda.synchronize()
        for s, out, (want, cache) in zip(states, outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(s["cache"], cache))


@gpu
def test_a_cache_of_more_than_32_bits_of_bytes(cuda):
    """Streams and rows that lie further than 2^32 bytes into a cache."""
    G, d, R, S = 17, 128, 1 << 20, 2     # 2.3 GB of keys a stream, two streams, and as much of values
    ck, cv = (torch.zeros(2, G, R, d, dtype=torch.int8, device="cuda") for _ in range(2))
    sc = torch.zeros(2, G, R, 2, device="cuda")
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(2, 300, G * d, generator=g).to(BF16).cuda() for _ in range(2))
    pos = i32([R - 200, 3 * R + 11])
    ops.window_cache_append_q8_((ck, cv, sc), k, v, pos, S)
    small = ops.window_cache_q8(2, 302, G, d)
    ops.window_cache_append_q8_(small, k, v, i32([2, 2]), S)
    after = pos + 300
    got = ops.window_cache_read((ck, cv, sc), after, S, 300)
    want = ops.window_cache_read(small, i32([302, 302]), S, 300)
    for x, y in zip(got, want):
        assert torch.equal(x[:, S:], y[:, S:])
    # nothing else was written, and the attention sees these rows: all others are zeros with a score of 0
    assert int(ck.count_nonzero()) == int(small[0].count_nonzero()) and int(sc.count_nonzero()) == int(small[2].count_nonzero())
    q = torch.randn(2, 1, G * d, generator=g).to(BF16).cuda()
    out = ops.window_attention_q8(q, (ck, cv, sc), after - 1, G, S, scale=1.0)
    for b in range(2):
        held = min(int(after[b]), R)
        rows = [row_of(int(pos[b]) + t, S, R - S) for t in range(300)]
        for h in (0, G - 1):
            kh, vh = (c[b, h, rows].double() * sc[b, h, rows, i, None].double() for i, c in enumerate((ck, cv)))
            s = kh @ q[b, 0, h * d:(h + 1) * d].double()
            top = max(float(s.max()), 0.0)
            w = torch.exp(s - top)
            den = w.sum() + (held - 300) * math.exp(-top)
            ref, ref_abs = w @ vh / den, w @ vh.abs() / den
            size = float((kh.abs() @ q[b, 0, h * d:(h + 1) * d].double().abs()).max())
            # (the sums of a lane's quarter of the keys of a wave: R / 4 of equal size at most)
            tol = 2.0 ** -8 * ref.abs() + (2.0 ** -16 + U * (R / 2 + 52 * 1.45 * size)) * ref_abs
            assert ((out[b, 0, h * d:(h + 1) * d].double() - ref).abs() <= tol).all()


@gpu
def test_the_longest_cache(cuda):
    """2^30 rows of two heads, 80 GiB: a head's scales are 2^31 numbers, its codes 2^34 bytes.  What is written is what a short cache holds of the same tokens, in
    both heads; the first rows, then the last ones and those that the ring goes on with."""
    G, d, S, R, n = 2, 8, 4, 1 << 30, 7
    cache = (*(torch.empty(1, G, R, 16, dtype=torch.int8, device="cuda") for _ in range(2)), torch.empty(1, G, R, 2, device="cuda"))
    g = torch.Generator().manual_seed(5)
    k, v, q = (torch.randn(1, n, G * d, generator=g).to(BF16).cuda() for _ in range(3))
    small = ops.window_cache_q8(1, 2 * n, G, d)
    ops.window_cache_append_q8_(small, k, v, i32([0]), S)

    def rows_are(at):
        for a, b, width in zip(cache, small, (d, d, 2)):
            for head in range(G):
                assert torch.equal(torch.stack([a[0, head, r, :width] for r in at]), b[0, head, :n, :width])

    ops.window_cache_append_q8_(cache, k, v, i32([0]), S)
    rows_are(list(range(n)))
    got, want = (ops.window_attention_q8(q[:, -1:], c, i32([n - 1]), G, S) for c in (cache, small))
    check(got, definition(q[:, -1:].cpu(), [t.cpu() for t in small], [n - 1], G, S, d ** -0.5), n)
    check(want, definition(q[:, -1:].cpu(), [t.cpu() for t in small], [n - 1], G, S, d ** -0.5), n)
    first = R - 3
    ops.window_cache_append_q8_(cache, k, v, i32([first]), S)
    rows_are([row_of(first + t, S, R - S) for t in range(n)])
    for a, b in zip(ops.window_cache_read(cache, i32([first + n]), S, n, d), ops.window_cache_read(small, i32([n]), 0, n, d)):
        assert torch.equal(a[:, S:], b)
    del cache, got, want
    torch.cuda.empty_cache()


# --------------------------------------------------------------------------- refusals

def test_calls_that_are_refused_before_any_launch():
    lib, P, bf16 = _lib.load(), 0x10000, _lib.DT_BF16
    ARG, SHAPE, ALIGN, WORK, DTYPE = -1, -2, -3, -4, -6
    base = dict(q=P, ck=P, cv=P, sc=P, pos=P, out=P, ws=0, bytes=0, q_b=256, o_b=256, ck_b=2 * 20 * 64, cv_b=2 * 20 * 64, sc_b=80, B=2, H=4, G=2, d=64, window=20, sinks=0,
                dt=bf16, scale=0.1)
    step = lambda **c: lib.sana_hip_window_q8(_lib.WINDOW_Q8_ARGS.pack(*{**base, **c}.values()), None)  # noqa: E731
    assert lib.sana_hip_window_q8(None, None) == ARG and lib.sana_hip_window_cache_read(None, None) == ARG
    for n in ("q", "ck", "cv", "sc", "pos", "out"):
        assert step(**{n: 0}) == ARG
        assert step(**{n: P + 2}) == ALIGN
    for c in (dict(B=0), dict(H=3), dict(G=0), dict(d=0), dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(o_b=248),
              dict(ck_b=-16), dict(q_b=-8)):
        assert step(**c) == ARG, c
    for c in (dict(d=60), dict(d=136), dict(window=1 << 30, sinks=1), dict(B=1 << 24)):
        assert step(**c) == SHAPE, c
    for c in (dict(q_b=260), dict(ck_b=24), dict(sc_b=81), dict(o_b=258)):
        assert step(**c) == ALIGN, c
    assert step(dt=0) == DTYPE
    need = lib.sana_hip_window_q8_workspace_bytes(2, 4, 2, 64, 9000, 0)
    assert need > 0 and lib.sana_hip_window_q8_workspace_bytes(2, 4, 2, 64, 20, 0) == 0
    assert step(window=9000) == WORK and step(window=9000, ws=P, bytes=need - 1) == WORK and step(window=9000, ws=P + 8, bytes=need) == ALIGN
    M = 2 ** 31 - 1
    assert lib.sana_hip_window_q8_workspace_bytes(M, M, M, M, M, M) == 0 and lib.sana_hip_window_q8_workspace_bytes(M, M, 1, 128, 1 << 29, 1 << 29) == 0
    base2 = dict(ck=P, cv=P, sc=P, pos=P, ok=P, ov=P, ck_b=4 << 10, ck_n=128, cv_b=4 << 10, cv_n=128, sc_b=96, ok_b=24 * 128, ok_n=128, ov_b=24 * 128, ov_n=128,
                 B=2, G=2, d=64, window=20, sinks=4, last=20, zero=0, dt=bf16)
    read = lambda **c: lib.sana_hip_window_cache_read(_lib.CACHE_READ_ARGS.pack(*{**base2, **c}.values()), None)  # noqa: E731
    for n in ("ck", "cv", "pos", "ok", "ov"):
        assert read(**{n: 0}) == ARG
    for c in (dict(last=21), dict(last=-1), dict(last=0, sinks=0), dict(ok_n=120), dict(ov_b=120), dict(B=0), dict(sc=0, ck_n=120), dict(ck_b=-16), dict(d=0), dict(d=0, sc=0)):
        assert read(**c) == ARG, c
    for c in (dict(d=60), dict(d=60, sc=0), dict(d=136), dict(window=1 << 30, last=1 << 30, sinks=4), dict(B=1 << 26), dict(B=1 << 26, sc=0, G=1),
              dict(d=1 << 22, sc=0, ck_n=1 << 23, cv_n=1 << 23, ok_n=1 << 23, ov_n=1 << 23, ok_b=1 << 30, ov_b=1 << 30)):
        assert read(**c) == SHAPE, c
    for c in (dict(ck=P + 8), dict(ok=P + 2), dict(pos=P + 2), dict(sc=P + 4), dict(ck_b=24), dict(sc_b=97), dict(ok_n=132), dict(sc=0, ck_n=132)):
        assert read(**c) == ALIGN, c
    assert read(dt=0) == DTYPE


def test_sizes_that_no_launch_takes_are_refused():
    """An axis of a launch has fewer than 2^32 threads: 2^23 workgroups of 512 (a token), 2^24 of 256 (rows in order) are one too many.  (The pointers are never followed.)"""
    lib, P, bf16, SHAPE = _lib.load(), 0x10000, _lib.DT_BF16, -2
    codes = 20 * 16
    for B, H, G in ((1 << 23, 1, 1), (1 << 22, 2, 2), (1 << 20, 68, 4), (1 << 4, 1 << 19, 1 << 19)):
        args = _lib.WINDOW_Q8_ARGS.pack(P, P, P, P, P, P, 0, 0, H * 8, H * 8, G * codes, G * codes, G * 40, B, H, G, 8, 20, 0, bf16, 0.1)
        assert lib.sana_hip_window_q8(args, None) == SHAPE, (B, H, G)
        assert lib.sana_hip_window_q8_workspace_bytes(B, H, G, 8, 20, 0) == 0

    def read(B, G, d, last, bits):
        width, held = G * d, last + 1
        row = width if bits == 16 else 0
        return lib.sana_hip_window_cache_read(_lib.CACHE_READ_ARGS.pack(P, P, 0 if bits == 16 else P, P, P, P, row * held, row, row * held, row, 0, width * held, width,
                                                                        width * held, width, B, G, d, last, 1, last, 0, bf16), None)

    for bits, B, G, d, held in ((16, 1, 1, 512, (1 << 25) - 1), (16, 1, 1, 512, 1 << 25), (16, 3, 1, 512, 11184811), (16, 1, 1, 64, 1 << 25), (8, 1, 1, 128, (1 << 29) - 16),
                                (8, 1, (1 << 15) - 1, 128, 16 * ((1 << 10) + 1)), (8, 3, 1, 128, 16 * 11184811)):
        assert read(B, G, d, held - 1, bits) == SHAPE, (bits, B, G, d, held)


@gpu
def test_refusals(cuda):
    B, H, G, d, R = 2, 4, 2, 40, 30
    cache, pos = [t.cuda() for t in realistic(B, G, R, d)], i32([3, 50])
    q = torch.randn(B, 1, H * d, device="cuda").to(BF16)
    ck, cv, sc = cache
    step = lambda **c: ops.window_attention_q8(**{**dict(q=q, cache=cache, positions=pos, num_heads=H, sinks=4), **c})  # noqa: E731
    read = lambda **c: ops.window_cache_read(**{**dict(cache=cache, positions=pos, sinks=4, dim=d), **c})  # noqa: E731
    pair = [torch.zeros(B, R, G * d, dtype=BF16, device="cuda") for _ in range(2)]
    step(), read(), read(cache=pair, dim=None), read(out=pair)
    bad = [lambda: step(q=q.float()), lambda: step(q=q.expand(B, 2, H * d)), lambda: step(num_heads=3), lambda: step(num_heads=0), lambda: step(cache=cache[:2]),
           lambda: step(cache=(ck, cv, sc[..., :1])), lambda: step(sinks=R), lambda: step(sinks=-1), lambda: step(scale=0.0), lambda: step(scale=float("inf")), lambda: step(positions=pos.long()),
           lambda: step(out=q.half()), lambda: step(q=q.clone().requires_grad_()), lambda: step(q=q.cpu()), lambda: step(q=q[..., :2 * d], num_heads=1), lambda: step(q=q[:1]),
           lambda: step(q=q[..., :3 * d], num_heads=3), lambda: step(cache=(ck.transpose(1, 2).contiguous().transpose(1, 2), cv, sc)),
           lambda: read(dim=64), lambda: read(dim=44), lambda: read(dtype=torch.float32), lambda: read(last=27), lambda: read(last=-1), lambda: read(sinks=0, last=0), lambda: read(sinks=R),
           lambda: read(out=(pair[0][:, 1:], pair[1][:, 1:])), lambda: read(out=(pair[0],)), lambda: read(out=(pair[0].half(), pair[1].half())), lambda: read(cache=(ck,)),
           lambda: read(cache=pair, dtype=F16), lambda: read(cache=(pair[0], pair[1][:, 1:])), lambda: read(cache=[t.float() for t in pair]), lambda: read(positions=pos[:1]),
           lambda: read(cache=[t[..., 4:] for t in pair], dim=None), lambda: read(out=[t[:1].expand(B, R, G * d) for t in pair])]
    for i, call in enumerate(bad):
        with pytest.raises(sana_amd.SanaHipError):
            call()
            pytest.fail(f"case {i} was taken")
    none = i32([])
    assert step(q=q[:0], cache=[t[:0] for t in cache], positions=none).shape == (0, 1, H * d)
    assert read(cache=[t[:0] for t in cache], positions=none)[0].shape == (0, R, G * d)
    for bad in (lambda: ops.window_cache_q8(1, 0, 1, 64), lambda: ops.window_cache_q8(1, 5, 1, 60), lambda: ops.window_cache_q8(1, 5, 1, 136), lambda: ops.window_cache_q8(1, 5, 0, 64)):
        with pytest.raises(sana_amd.SanaHipError):
            bad()


@gpu
def test_refusals_of_what_no_call_holds(cuda):
    """No positions, numbers beyond 32 bits, a cache without heads: the library's own error, and nothing is written."""
    B, H, G, d, R = 2, 4, 2, 40, 30
    cache, pos, far = [t.cuda() for t in realistic(B, G, R, d)], i32([3, 50]), 1e39
    q, k, v, _, _ = (t.cuda() for t in make(B, 1, H, G, d, BF16))
    w = torch.ones(d, dtype=BF16, device="cuda")
    f = freqs_of(40).cuda()
    before = [t.clone() for t in cache]
    none = [t[:, :0] for t in cache]
    for call in (lambda: ops.window_attention_q8(q, cache, None, H), lambda: ops.window_attention_q8(q, cache, pos, H, scale=far), lambda: ops.window_attention_q8(q, none, pos, H),
                 lambda: ops.window_cache_read(cache, None, dim=d), lambda: ops.window_cache_read(cache, None, dim=d, out=[torch.zeros(B, R, G * d, dtype=BF16, device="cuda")] * 2),
                 lambda: ops.window_cache_read(none, pos, dim=d), lambda: ops.window_cache_read([t[..., :16].flatten(2).to(BF16) for t in cache[:2]], None),
                 lambda: ops.window_cache_append_q8_(cache, k, v, None), lambda: ops.window_cache_append_q8_(none, k, v, pos), lambda: ops.qk_norm_rope(q, k, H, w, w, eps=far),
                 lambda: ops.qk_norm_rope(q, k, H, freqs=f, magnitude=far), lambda: ops.qk_norm_rope(q, k, H, freqs=f, magnitude=-far),
                 lambda: ops.qk_norm_rope_append_q8_(q, k, v, cache, None, H), lambda: ops.qk_norm_rope_append_q8_(q, k, v, cache, pos, H, w, w, far),
                 lambda: ops.qk_norm_rope_append_q8_(q, k, v, none, pos, H)):
        with pytest.raises(sana_amd.SanaHipError):
            call()
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
