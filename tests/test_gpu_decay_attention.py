"""Linear attention with a decay for each head against its definition in 64 bits, and what the call refuses."""
import ctypes

import pytest
import torch

import sana_amd
from sana_amd import _lib, ops

gpu = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def definition(q, k, v, log_decay, scale, state, lengths):
    """(out, state, and for each the sum of the absolute values of its terms), 64 bits, head by head, every pair of tokens."""
    B, N, C = q.shape
    H = log_decay.numel()
    d = C // H
    q, k, v = (t.double().reshape(B, N, H, d).transpose(1, 2) for t in (q, k, v))
    g = log_decay.double()
    out, out_abs = torch.zeros(2, B, H, N, d, dtype=torch.float64)
    fin, fin_abs = torch.zeros(2, B, H, d, d, dtype=torch.float64)
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        i = torch.arange(n, dtype=torch.float64)
        for h in range(H):
            apart = i[:, None] - i[None, :]
            power = lambda e: torch.where(e == 0, 1.0, torch.exp(g[h] * e.clamp(min=0)))  # noqa: E731   (-inf * 0)
            w = torch.where(apart >= 0, power(apart), 0.0)
            s0 = state[b, h].double() if state is not None else torch.zeros(d, d, dtype=torch.float64)
            for o, s, f in ((out, fin, lambda x: x), (out_abs, fin_abs, torch.abs)):
                qh, kh, vh = (f(t[b, h, :n]) for t in (q, k, v))
                o[b, h, :n] = abs(scale) * ((w * (qh @ kh.T)) @ vh + power(i + 1)[:, None] * (qh @ f(s0).T))
                s[b, h] = vh.T @ (kh * power(n - 1 - i)[:, None]) + power(torch.tensor(float(n), dtype=torch.float64)) * f(s0)
            if scale < 0:
                out[b, h] = -out[b, h]
    rows = lambda t: t.transpose(1, 2).reshape(B, N, C)  # noqa: E731
    return rows(out), fin, rows(out_abs), fin_abs


def chained(N):
    """Roundings of 2^-24 in a row that an fp32 sum over N tokens can have: two a chunk of 64 (decay, products), those of
    the 16-term products within a chunk, and of the powers, whose exponents g n are rounded (n g a^n stays below 1/e)."""
    return 2 * (N // 64) + 64


def check(got, want, q, N):
    half = torch.finfo(q.dtype).eps / 2
    out, state = got[0].double().cpu(), got[1].double().cpu()
    ref, fin, ref_abs, fin_abs = want
    # a score's rounding is half a step of its term, the result's half a step of itself (or of the smallest f16)
    tol = half * (ref.abs() + ref_abs) + chained(N) * 2.0 ** -24 * ref_abs + (2.0 ** -25 if q.dtype == F16 else 0)
    assert ((out - ref).abs() <= tol).all(), ((out - ref).abs() / tol).max().item()
    # a weighted value is the sum of two 16-bit values: half a step of half a step
    tol = half * half * fin_abs + chained(N) * 2.0 ** -24 * fin_abs
    assert ((state - fin).abs() <= tol + 1e-300).all(), ((state - fin).abs() / tol).max().item()


def make(B, N, H, d, dtype, seed=0, carried=False, packed=True, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    C = H * d
    qkv = (spread * torch.randn(B, N, 3 * C, generator=g)).to(dtype)
    q, k, v = qkv.split(C, dim=2) if packed else (t.contiguous() for t in qkv.split(C, dim=2))
    log_decay = torch.log1p(-torch.exp2(-torch.linspace(1.0, 10.0, H)))
    state = torch.randn(B, H, d, d, generator=g) if carried else None
    return q, k, v, log_decay, state


def to_gpu(q, k, v):
    """The same views on the GPU: of one packed tensor where they are of one here."""
    if q._base is not None and q._base is k._base:
        base = q._base.cuda()
        return [base.as_strided(t.size(), t.stride(), t.storage_offset()) for t in (q, k, v)]
    return [t.cuda() for t in (q, k, v)]


def compare(q, k, v, log_decay, state=None, lengths=None, scale=0.3):
    want = definition(q, k, v, log_decay, scale, state, lengths)
    got = ops.decay_linear_attention(*to_gpu(q, k, v), log_decay.cuda(), scale, None if state is None else state.cuda(),
                                     None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert got[0].dtype == q.dtype and got[1].dtype == torch.float32
    check(got, want, q, q.shape[1])
    return got


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 104, 112, 128])
@pytest.mark.parametrize("N", [1, 2, 64, 130])
def test_head_dims_and_lengths(cuda, N, d, dtype):
    compare(*make(2, N, 3, d, dtype, seed=N + d, carried=True))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N", [1, 3, 16, 17, 33, 63, 65, 127, 128, 129, 300, 1000])
def test_token_counts(cuda, N, dtype):
    compare(*make(1, N, 5, 32, dtype, seed=N))
    compare(*make(1, N, 2, 112, dtype, seed=N, packed=False))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 96, 112])
@pytest.mark.parametrize("N,lengths", [(1500, [1500, 1499, 64, 0]), (2048, [2048, 1024, 1, 1087])])
def test_long_streams_in_segments(cuda, N, lengths, d, dtype):
    """Few heads and many tokens: segments side by side, joined by their states; lengths that end in front of, on and in a segment."""
    assert _lib.load().sana_hip_decay_attention_workspace_bytes(4, N, 2, d) > 0
    q, k, v, log_decay, state = make(4, N, 2, d, dtype, seed=d, carried=True)
    compare(q, k, v, log_decay, state, lengths)
    compare(q, k, v, log_decay)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N", [1, 100, 1300])
def test_lengths_leave_rows_and_states_alone(cuda, N, dtype):
    """Rows behind a stream's end are neither read (NaN there reaches nothing) nor written; lengths are clamped to the rows there are."""
    q, k, v, log_decay, state = make(5, N, 2, 64, dtype, seed=3, carried=True, packed=False)
    lengths = [0, N, min(N, 67), N + 9, -4]
    for t in (q, k, v):
        for b, n in enumerate(lengths):
            t[b, max(n, 0):] = float("nan")
    clean = [torch.where(torch.isnan(t), torch.zeros_like(t), t) for t in (q, k, v)]
    want = definition(*clean, log_decay, 0.5, state, lengths)
    out = torch.full_like(q, 7.0).cuda()
    args = [t.cuda() for t in (q, k, v, log_decay)]
    lengths_dev = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = ops.decay_linear_attention(*args, 0.5, state.cuda(), lengths_dev, out=out)
    assert got[0] is out
    for b, n in enumerate(lengths):
        assert (out[b, max(n, 0):] == 7.0).all()
        out[b, max(n, 0):] = 0
    check(got, want, q, N)
    assert torch.equal(got[1][0].cpu(), state[0]) and torch.equal(got[1][4].cpu(), state[4])
    new, _ = ops.decay_linear_attention(*args, 0.5, state.cuda(), lengths_dev)
    assert torch.equal(new, out)


@gpu
@pytest.mark.parametrize("N", [1, 200, 1300])
def test_states_in_place_and_aside_are_the_same_bits(cuda, N):
    q, k, v, log_decay, state = make(2, N, 3, 72, BF16, carried=True)
    args = [*to_gpu(q, k, v), log_decay.cuda()]
    mine, kept = state.cuda(), state.cuda()
    out, new = ops.decay_linear_attention(*args, state=kept)
    assert torch.equal(kept.cpu(), state)
    out2, same = ops.decay_linear_attention(*args, state=mine, state_out=mine)
    assert same is mine and torch.equal(same, new) and torch.equal(out, out2)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decays_of_every_size(cuda, dtype):
    """No decay, no memory (-inf), and decays whose powers leave fp32 within a chunk."""
    for N in (1, 150):
        q, k, v, _, state = make(1, N, 6, 32, dtype, carried=True)
        compare(q, k, v, torch.tensor([0.0, -float("inf"), -1e30, -50.0, -3.0, -1e-7]), state, scale=-1.5)


@gpu
@pytest.mark.parametrize("N", [1, 190])
def test_half_precision_where_states_and_scores_leave_its_range(cuda, N):
    """fp16 ends at 65504: scores of 1e6 and states of 1e7 with outputs of ordinary size, and values whose second parts are subnormal."""
    q, k, v, log_decay, state = make(1, N, 3, 64, F16, carried=True)
    compare(q * 60, k * 200, v * 1e-3, log_decay, state * 30, scale=1e-3)
    compare(q * 1e-3, k * 0 + 1, v * 300, log_decay * 0, state * 1e7, scale=1e-4)
    compare(q, k * 1e-3, v * 1e-3, log_decay, None, scale=1.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,H,d", [(1, 3, 32), (100, 3, 32), (150, 3, 112), (90, 3, 96), (1300, 2, 64), (1500, 2, 112)])
def test_what_is_not_finite_reaches_nothing_in_front_of_it(cuda, N, H, d, dtype):
    """Values of inf and NaN: the outputs in front of them, the other channels' and the other heads' are what they are without; from the
    token on their channel is not finite, nor are its rows of the state.  A key of NaN: the same for all channels of its head."""
    q, k, v, log_decay, state = make(2, N, H, d, dtype, seed=N, carried=True, packed=False)
    clean_k, clean_v = k.clone(), v.clone()
    odd, odd_state = torch.zeros(2, N, H, d, dtype=torch.bool), torch.zeros(2, H, d, d, dtype=torch.bool)
    for b, j, h, c, x in [(0, N // 2, 0, 3, float("inf")), (0, N // 2, 1, 7, -float("inf")), (1, N // 3, 1, 7, float("nan")), (1, N - 1, 0, 1, float("inf"))]:
        v[b, j, h * d + c], clean_v[b, j, h * d + c] = x, 0
        odd[b, j:, h, c], odd_state[b, h, c] = True, True
    for b, j, h, c in [(1, 2 * N // 3, H - 1, 2)]:
        k[b, j, h * d + c], clean_k[b, j, h * d + c] = float("nan"), 0
        odd[b, j:, h], odd_state[b, h, :, c] = True, True
    want = definition(q, clean_k, clean_v, log_decay, 0.3, state, None)
    got, last = ops.decay_linear_attention(q.cuda(), k.cuda(), v.cuda(), log_decay.cuda(), 0.3, state.cuda())
    odd = odd.reshape(2, N, H * d)
    got, last = got.double().cpu(), last.double().cpu()
    assert not torch.isfinite(got[odd]).any() and not torch.isfinite(last[odd_state]).any()
    check((torch.where(odd, want[0], got), torch.where(odd_state, want[1], last)), want, q, N)


@gpu
def test_views_of_every_kind(cuda):
    """Rows further apart than their channels, batches in front of tokens, a stream cut out of a longer one, an out of other strides."""
    B, N, H, d = 2, 150, 3, 40
    q, k, v, log_decay, _ = make(B, N, H, d, BF16, packed=False)
    want = ops.decay_linear_attention(*[t.cuda() for t in (q, k, v)], log_decay.cuda())
    wide = torch.full((B, N + 9, 5, H * d + 8), float("nan"), dtype=BF16, device="cuda")
    views = [wide[:, 4:4 + N, i, 8:] for i in range(3)]
    for view, t in zip(views, (q, k, v)):
        view.copy_(t)
    got = ops.decay_linear_attention(*views, log_decay.cuda(), out=wide[:, 4:4 + N, 3, 4:-4])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.isnan(wide[:, :4]).all() and torch.isnan(wide[:, 4 + N:]).all() and torch.isnan(wide[:, :, 4]).all()
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1).cuda() for t in (q, k, v)]
    got = ops.decay_linear_attention(*swapped, log_decay.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_then_tokens_is_the_whole_stream(cuda, dtype):
    """A prompt and then token after token, the state in place, against one call over all of them."""
    B, N, H, d, prompt = 3, 90, 4, 112, 70
    q, k, v, log_decay, _ = make(B, N, H, d, dtype)
    want = definition(q, k, v, log_decay, 0.2, None, None)
    q, k, v = to_gpu(q, k, v)
    g = log_decay.cuda()
    outs, state = ops.decay_linear_attention(q[:, :prompt], k[:, :prompt], v[:, :prompt], g, 0.2)
    outs = [outs]
    for t in range(prompt, N):
        outs.append(ops.decay_linear_attention(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], g, 0.2, state, state_out=state)[0])
    check((torch.cat(outs, 1), state), want, q, N)


@gpu
@pytest.mark.parametrize("N", [1, 80, 1300])
def test_replays_are_the_eager_result(cuda, N):
    """Two graphs of one stream replayed side by side, eager calls between: the segments' states are each graph's own."""
    sets = []
    for seed in (1, 2):
        q, k, v, log_decay, state = make(1, N, 4, 112, BF16, seed=seed, carried=True)
        args = [t.contiguous().cuda() for t in (q, k, v, log_decay, state)]
        call = lambda q, k, v, g, s: torch.cat([t.flatten().float() for t in ops.decay_linear_attention(q, k, v, g, 0.4, s)])  # noqa: E731
        want = call(*args).clone()
        sets.append((sana_amd.GraphedCall(call, args), args, want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        torch.cuda.synchronize()
        got = []
        for (graph, args, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(graph(*args).clone())
        torch.cuda.synchronize()
        for g, (_, args, want) in zip(got, sets):
            assert torch.equal(g, want)
            assert torch.equal(call(*args), want)


@gpu
def test_empty_calls(cuda):
    q, k, v, log_decay, state = make(2, 4, 3, 32, BF16, carried=True)
    q, k, v = (t.cuda() for t in (q, k, v))
    g, s = log_decay.cuda(), state.cuda()
    out, new = ops.decay_linear_attention(q[:, :0], k[:, :0], v[:, :0], g, state=s)
    assert out.shape == (2, 0, 96) and torch.equal(new, s) and new is not s
    out, new = ops.decay_linear_attention(q[:, :0], k[:, :0], v[:, :0], g)
    assert (new == 0).all() and new.shape == (2, 3, 32, 32)
    out, new = ops.decay_linear_attention(q[:0], k[:0], v[:0], g)
    assert out.shape == (0, 4, 96) and new.shape == (0, 3, 32, 32)


@gpu
def test_refusals(cuda):
    q, k, v, log_decay, state = make(2, 8, 3, 32, BF16, carried=True)
    q, k, v, g, s = (t.contiguous().cuda() for t in (q, k, v, log_decay, state))
    call = ops.decay_linear_attention
    bad = [lambda: call(q.float(), k.float(), v.float(), g), lambda: call(q, k.half(), v, g), lambda: call(q, k[:, :4], v, g),
           lambda: call(q, k, v, g.double()), lambda: call(q, k, v, g[:2].repeat(4)[:5]), lambda: call(q, k, v, g[None]),
           lambda: call(q, k, v, g.cpu()), lambda: call(q, k, v, g, state=s.half()), lambda: call(q, k, v, g, state=s[:1]),
           lambda: call(q, k, v, g, state=s.transpose(2, 3)), lambda: call(q, k, v, g, state_out=s.transpose(2, 3)),
           lambda: call(q, k, v, g, lengths=torch.tensor([1, 2], device="cuda")),
           lambda: call(q, k, v, g, lengths=torch.tensor([1], dtype=torch.int32, device="cuda")),
           lambda: call(q, k, v, g, out=q.float()), lambda: call(q[0], k[0], v[0], g),
           lambda: call(q[..., :84], k[..., :84], v[..., :84], g), lambda: call(*[t[:, :, ::2] for t in (q, k, v)], g),
           lambda: call(*[t[:1].expand(2, 8, 96)[:, :1].expand(2, 8, 96) for t in (q, k, v)], g),
           lambda: call(*[torch.zeros(2 * 8 * 96 + 1, dtype=BF16, device="cuda")[1:].view(2, 8, 96)] * 3, g),
           lambda: call(q, k, v, g, out=torch.empty_like(q[:1]).expand(2, 8, 96)),
           lambda: call(q, k, v.clone().requires_grad_(), g)]
    for i, f in enumerate(bad):
        with pytest.raises(sana_amd.SanaHipError):
            f()
            pytest.fail(f"case {i} was taken")
    with torch.no_grad():
        call(q, k, v.clone().requires_grad_(), g)   # (leaves that want gradients are fine where none are recorded)


def test_c_entry_refuses_before_any_launch():
    """Host checks: the pointers below are never followed."""
    lib, P = _lib.load(), 0x10000
    good = [P, P, P, P, None, P, P, None, None, 0, 2, 8, 3, 32] + [8 * 96, 96] * 4 + [1.0, _lib.DT_BF16]
    call = lambda *change: lib.sana_hip_decay_attention(*[dict(change).get(i, x) for i, x in enumerate(good)], None)  # noqa: E731
    for i in (0, 1, 2, 3, 5, 6):
        assert call((i, None)) == -1
    for i in (10, 11, 12, 13):
        assert call((i, 0)) == -1
    assert call((23, _lib.DT_F32)) == -6 and call((23, 9)) == -6
    assert call((13, 36)) == -2 and call((13, 136)) == -2 and call((12, 1 << 24)) == -2
    for i in (15, 17, 19, 21):
        assert call((i, 88)) == -1 and call((i, 1 << 23)) == -2
        assert call((i, 98)) == -3 and call((i - 1, -8)) == -1
    assert call((20, 0)) == -1 and call((20, 0), (10, 0)) == -1   # two entries of one output
    for i in (0, 1, 2, 4, 5):
        assert call((i, P + 8)) == -3
    assert call((6, P + 4)) == -3 and call((3, P + 2)) == -3 and call((7, P + 2)) == -3
    # a long stream of few heads needs its workspace, aligned and whole
    need = lib.sana_hip_decay_attention_workspace_bytes(1, 32760, 3, 32)
    assert need > 0 and need % (3 * 32 * 32 * 4) == 0
    long = ((10, 1), (11, 32760))
    assert call(*long) == -4 and call(*long, (8, P), (9, need - 1)) == -4 and call(*long, (8, P + 8), (9, need)) == -3
    assert lib.sana_hip_decay_attention_workspace_bytes(1, 1, 3, 32) == 0
    assert lib.sana_hip_decay_attention_workspace_bytes(0, 8, 3, 32) == 0
    assert lib.sana_hip_decay_attention_workspace_bytes(64, 32760, 64, 32) == 0


def test_c_entry_refuses_launches_of_too_many_threads():
    """Host checks of sizes whose grids no launch takes (2^32 threads)."""
    lib, P = _lib.load(), 0x10000
    call = lambda B, N, H: lib.sana_hip_decay_attention(P, P, P, P, None, P, P, None, None, 0, B, N, H, 32, *[8 * 96, 96] * 4, 1.0, _lib.DT_BF16, None)  # noqa: E731
    assert call(1 << 22, 8, 3) == -2 and call(1 << 24, 1, 1) == -2


def test_cpu_tensors_are_refused():
    q, k, v, log_decay, _ = make(1, 4, 2, 32, BF16)
    with pytest.raises(sana_amd.SanaHipError):
        ops.decay_linear_attention(q, k, v, log_decay)
