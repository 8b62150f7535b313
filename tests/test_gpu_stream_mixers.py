"""The decayed linear attention and the window attention as a stream uses them together: a padded batch of prompts, then tokens, eagerly
and from a graph, each token checked against the definitions over its whole stream."""
import pytest
import torch

import sana_amd
from sana_amd import ops
from test_gpu_decay_attention import check as check_decay, definition as decay_definition
from test_gpu_window_attention import check as check_window, definition as window_definition

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype,H,G,d", [(BF16, 4, 2, 112), (F16, 6, 1, 32)])
def test_prompts_then_tokens(cuda, dtype, H, G, d, graph):
    B, prompt, steps, window, sinks = 3, 90, 12, 40, 3
    C, gen = H * d, torch.Generator().manual_seed(d)
    lengths = [90, 17, 64]
    total = prompt + steps
    x = torch.randn(B, total, 3 * C + (H + 2 * G) * d, generator=gen).clamp(-6, 6).to(dtype)   # both mixers' projections
    log_decay = torch.log1p(-torch.exp2(-torch.linspace(1.0, 8.0, H)))
    split = [C, C, C, C, G * d, G * d]

    # every stream as one, from the definitions: its prompt, then its tokens (which lie behind the padding here)
    streams = [torch.cat([x[b, :lengths[b]], x[b, prompt:]])[None] for b in range(B)]
    dev, g = x.cuda(), log_decay.cuda()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q1, k1, v1, q2, k2, v2 = dev[:, :prompt].split(split, dim=2)
    out1, state = ops.decay_linear_attention(q1, k1, v1, g, 0.2, lengths=n)
    out2 = ops.window_attention(q2, k2, v2, H, window, sinks, lengths=n)
    ck, cv = torch.full((2, B, sinks + window, G * d), float("nan"), dtype=dtype, device="cuda").unbind(0)
    positions = torch.zeros(B, dtype=torch.int32, device="cuda")
    ops.window_cache_append_(ck, cv, k2, v2, positions, sinks, n)
    positions += n

    def token(t):
        q1, k1, v1, q2, k2, v2 = t.split(split, dim=2)
        a, _ = ops.decay_linear_attention(q1, k1, v1, g, 0.2, state, state_out=state)
        b = ops.window_attention_step_(q2, k2, v2, ck, cv, positions, H, sinks)
        positions.add_(1)
        return torch.cat([a, b], 2)

    if graph:
        kept = [t.clone() for t in (state, ck, cv, positions)]
        token = sana_amd.GraphedCall(token, [dev[:, prompt:prompt + 1].contiguous()])
        torch.cuda.synchronize()
        for t, was in zip((state, ck, cv, positions), kept):   # (the warm-up tokens are forgotten)
            t.copy_(was)
    got = [token(dev[:, prompt + i:prompt + i + 1].contiguous()).clone() for i in range(steps)]
    got = torch.cat(got, 1)
    for b in range(B):
        q1, k1, v1, q2, k2, v2 = streams[b].split(split, dim=2)
        N = lengths[b] + steps
        rows = torch.cat([out1[b, :lengths[b]], got[b, :, :C]])[None], state[b:b + 1]
        check_decay(rows, decay_definition(q1, k1, v1, log_decay, 0.2, None, None), q1, N)
        rows = torch.cat([out2[b, :lengths[b]], got[b, :, C:]])[None]
        check_window(rows, window_definition(q2, k2, v2, H, window, sinks, d ** -0.5), N, dtype)
    assert positions.tolist() == [a + steps for a in lengths]


@pytest.mark.gpu
def test_a_stream_of_its_own_and_two_calls_at_once(cuda):
    """The calls run on the current stream, each stream with scratch of its own."""
    gen = torch.Generator().manual_seed(5)
    sets = []
    for _ in range(2):
        x = torch.randn(1, 2000, 3 * 2 * 112, generator=gen).to(BF16).cuda()
        q, k, v = x.split(224, dim=2)
        cache = [t.contiguous().clone() for t in (k, v)]
        pos = torch.tensor([1999], dtype=torch.int32, device="cuda")
        g = torch.tensor([-0.1, -0.001], device="cuda")
        sets.append((q, k, v, g, cache, pos))

    def calls(q, k, v, g, cache, pos):
        a = ops.decay_linear_attention(q, k, v, g)
        return [*a, ops.window_attention(q[:, -3:], k, v, 2, 1500, 4),
                ops.window_attention_step_(q[:, -1:], k[:, -1:], v[:, -1:], *cache, pos, 2, 4)]

    want = [[t.clone() for t in calls(*s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(calls(*s))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i % 2]))
