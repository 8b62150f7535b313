"""The streams' calls at every head width, and the decayed attention against its recurrence, token by token."""
import pytest
import torch

import test_gpu_window_attention as window
from sana_amd import _lib, ops
from test_gpu_decay_attention import BF16, F16, check, compare, definition, make

gpu = pytest.mark.gpu
WIDTHS = list(range(8, 129, 8))


def recurrence(q, k, v, log_decay, scale, state):
    """S_t = exp(g) S_{t-1} + v_t k_t^T, o_t = scale S_t q_t in 64 bits, as it is written; for each the same of absolute values."""
    B, N, C = q.shape
    H = log_decay.numel()
    d = C // H
    q, k, v = (t.double().reshape(B, N, H, d) for t in (q, k, v))
    a = torch.exp(log_decay.double())[None, :, None, None]
    got = []
    for f in (lambda x: x, torch.abs):
        s = f(state.double()) if state is not None else torch.zeros(B, H, d, d, dtype=torch.float64)
        outs = []
        for t in range(N):
            s = a * s + f(v[:, t])[..., :, None] * f(k[:, t])[..., None, :]
            outs.append(f(torch.tensor(scale, dtype=torch.float64)) * (s @ f(q[:, t])[..., None])[..., 0])
        got.append((torch.stack(outs, 1).reshape(B, N, C), s))
    return got[0][0], got[0][1], got[1][0], got[1][1]


def test_the_pairwise_definition_is_the_recurrence():
    q, k, v, log_decay, state = make(2, 70, 3, 16, BF16, carried=True)
    for s in (None, state):
        for a, b in zip(recurrence(q, k, v, log_decay, -0.7, s), definition(q, k, v, log_decay, -0.7, s, None)):
            assert torch.allclose(a, b, rtol=1e-12, atol=1e-13)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,d", [(1, 64), (2, 8), (63, 40), (130, 112), (200, 128)])
def test_against_the_recurrence(cuda, N, d, dtype):
    q, k, v, log_decay, state = make(2, N, 3, d, dtype, seed=N, carried=True, packed=False)
    got = ops.decay_linear_attention(q.cuda(), k.cuda(), v.cuda(), log_decay.cuda(), 0.3, state.cuda())
    check(got, recurrence(q, k, v, log_decay, 0.3, state), q, N)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", WIDTHS)
def test_decay_at_every_width(cuda, d, dtype):
    for N in (1, 97):
        compare(*make(2, N, 5, d, dtype, seed=d, carried=True))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", WIDTHS)
def test_decay_in_segments_at_every_width(cuda, d, dtype):
    assert _lib.load().sana_hip_decay_attention_workspace_bytes(2, 1100, 2, d) > 0
    q, k, v, log_decay, state = make(2, 1100, 2, d, dtype, seed=d, carried=True)
    compare(q, k, v, log_decay, state, [1100, 555])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", WIDTHS)
def test_window_at_every_width(cuda, d, dtype):
    window.compare(*window.make(2, 150, 200, 4, 2, d, dtype, seed=d), 4, 60, 3)
    window.compare(*window.make(1, 3, 2000, 2, 1, d, dtype, seed=d), 2, 1500, 70)          # in parts
    window.step_compare(3, 6, 2, d, 70, 4, [5, 74, 300], dtype, seed=d)
    window.step_compare(1, 2, 1, d, 9000, 4, [9100], dtype, seed=d)
