"""What the streams' calls refuse, and what they take in the place of a number."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import sana_amd
from sana_amd import _lib, ops
from test_gpu_decay_attention import check, definition, make

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def stream(cuda):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 8, 64, generator=g).to(BF16).to(cuda) for _ in range(3))
    cache = [torch.zeros(1, 20, 64, dtype=BF16, device=cuda) for _ in range(2)]
    return q, k, v, torch.tensor([-0.1, -0.2], device=cuda), cache, torch.zeros(1, dtype=torch.int32, device=cuda)


@gpu
def test_forward_mode_derivatives_are_refused(cuda):
    """A dual tensor wants no gradient, so only its tangent tells it: an output without one would be a wrong derivative of zero."""
    q, k, v, g, (ck, cv), pos = stream(cuda)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        one = slice(0, 1)
        bad = [lambda: ops.decay_linear_attention(dual(q), k, v, g), lambda: ops.decay_linear_attention(q, k, v, dual(g)),
               lambda: ops.decay_linear_attention(q, k, v, g, state=dual(torch.zeros(1, 2, 32, 32, device=cuda))),
               lambda: ops.window_attention(q, dual(k), v, 2, 5), lambda: ops.window_cache_append_(ck, cv, k, dual(v), pos),
               lambda: ops.window_attention_step_(q[:, one], k[:, one], dual(v[:, one]), ck, cv, pos, 2),
               lambda: ops.window_attention_step_(q[:, one], k[:, one], v[:, one], dual(ck), cv, pos, 2)]
        for i, f in enumerate(bad):
            with pytest.raises(sana_amd.SanaHipError):
                f()
                pytest.fail(f"case {i} was taken")
        want = ops.window_attention(q, k, v, 2, 5)   # primals are fine within a level
        assert torch.equal(ops.window_attention(forward_ad.unpack_dual(dual(q)).primal, k, v, 2, 5), want)
    assert not ck.any() and not cv.any()


@gpu
@pytest.mark.parametrize("tokens", [1, 8])
def test_a_scale_is_any_number(cuda, tokens):
    q, k, v, g, (ck, cv), pos = stream(cuda)
    q, k, v = (t[:, :tokens] for t in (q, k, v))
    want = ops.decay_linear_attention(q, k, v, g, 0.5)[0]
    wide = ops.window_attention(q, k, v, 2, 5, scale=0.5)
    for scale in (np.float32(0.5), np.float64(0.5), torch.tensor(0.5), torch.tensor(0.5, device=cuda)):
        assert torch.equal(ops.decay_linear_attention(q, k, v, g, scale)[0], want)
        assert torch.equal(ops.window_attention(q, k, v, 2, 5, scale=scale), wide)
    assert torch.equal(ops.decay_linear_attention(q, k, v, g, 2)[0], ops.decay_linear_attention(q, k, v, g, 2.0)[0])


def test_entries_whose_rows_overlap_are_refused_before_any_launch():
    """Host checks (the pointers are never followed): two batch entries of an output or of a cache that are less than a row apart."""
    lib, P, bf16 = _lib.load(), 0x10000, _lib.DT_BF16
    ARG = -1
    decay = lambda o_b, B=2: lib.sana_hip_decay_attention(P, P, P, P, None, P, P + 4, None, None, 0, B, 8, 3, 32, *[8 * 96, 96] * 3, o_b, 96,  # noqa: E731
                                                         1.0, bf16, None)
    assert decay(88) == ARG and decay(96) == -3 and decay(0, 1) == -3   # (-3: an output of 4-byte alignment, found behind this)
    window = lambda o_b: lib.sana_hip_window_attention(P, P, P, P, None, None, 0, 2, 8, 8, 4, 2, 32, 5, 0, *[8 * 128, 128] * 3, o_b, 128, 0.1,  # noqa: E731
                                                       bf16, None)
    assert window(120) == ARG and window(0) == ARG
    step = lambda ck=20 * 64, cv=20 * 64, o=128: lib.sana_hip_window_step(P, P, P, P, P, P, P, None, 0, 2, 4, 2, 32, 20, 0, 128, 64, 64, ck, 64, cv, 64,  # noqa: E731
                                                                          o, 0.1, bf16, None)
    assert step(o=120) == ARG and step(ck=56) == ARG and step(cv=56) == ARG
    put = lambda ck, cv: lib.sana_hip_window_cache_append(P, P, P, P, P, None, 2, 8, 64, 20, 0, ck, 64, cv, 64, 512, 64, 512, 64, bf16, None)  # noqa: E731
    assert put(56, 20 * 64) == ARG and put(20 * 64, 56) == ARG


HUGE = """
import sys
sys.path.insert(0, sys.argv[1])
from sana_amd import _lib
lib, P, bf16 = _lib.load(), 0x10000, _lib.DT_BF16
M = 2 ** 31 - 1
# batches x heads x blocks of queries that pass 2^63, to the multiples of 2^64 that a product in 64 bits calls 0
assert lib.sana_hip_window_attention_workspace_bytes(1 << 30, 1024, 2048, 1 << 30, 8, 4000, 0) == 0
assert lib.sana_hip_window_attention_workspace_bytes(1 << 30, 1 << 22, 1 << 22, 1 << 18, 8, 4000, 0) == 0
assert lib.sana_hip_window_attention_query_tiles(1 << 30, 1024, 1 << 30, 8) == 0
assert lib.sana_hip_window_attention(P, P, P, P, None, None, 0, 1 << 30, 1 << 22, 1 << 22, 1 << 18, 1 << 18, 8, 4000, 0, *[1 << 43, 1 << 21] * 4, 0.1, bf16, None) == -2
# counts next to the type's end
for f, n in ((lib.sana_hip_window_attention_workspace_bytes, 7), (lib.sana_hip_window_step_workspace_bytes, 6),
             (lib.sana_hip_decay_attention_workspace_bytes, 4)):
    assert f(*[M] * n) == 0
assert lib.sana_hip_window_attention_query_tiles(1, M, 1, 8) == 0 and lib.sana_hip_window_attention_workspace_bytes(1, M, M, 1, 8, M, 0) == 0
assert lib.sana_hip_decay_attention_workspace_bytes(1, M, 1, 8) == 0
assert lib.sana_hip_window_step_workspace_bytes(M, M, M, M, 1 << 29, 1 << 29) == 0
print("whole")
"""


def test_sizes_beyond_all_memory_end_no_process():
    """(In a process of its own: a division by a wrapped product of 0 ends it.)"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", HUGE, root], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and run.stdout.strip().endswith("whole"), (run.returncode, run.stderr[-400:])


@gpu
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
@pytest.mark.parametrize("N,H,d", [(1, 3, 64), (100, 3, 32), (150, 3, 64), (90, 3, 112), (1500, 2, 112)])
@pytest.mark.parametrize("size", [1e7, 1e-4])
def test_a_carried_inf_stays_in_its_channel(cuda, N, H, d, dtype, size):
    """An inf of the state in front: its channel is not finite, all others are what they are without it, f16 states beyond and far below the type's
    range among them (the power of two that takes a wave's states there must not come from the inf)."""
    q, k, v, log_decay, state = make(1, N, H, d, dtype, carried=True)
    q, v, state, scale = q * 1e-3, (v * 3e-5 * size).to(dtype), state * size, 1e3 / size
    state[0, 0, 5, 7], state[0, H - 1, d - 2, 0] = float("inf"), -float("inf")
    clean = torch.where(torch.isfinite(state), state, torch.zeros_like(state))
    odd, odd_state = torch.zeros(1, N, H, d, dtype=torch.bool), torch.zeros(1, H, d, d, dtype=torch.bool)
    for h, c in ((0, 5), (H - 1, d - 2)):
        odd[0, :, h, c], odd_state[0, h, c] = True, True
    want = definition(q, k, v, log_decay, scale, clean, None)
    out, last = ops.decay_linear_attention(q.cuda(), k.cuda(), v.cuda(), log_decay.cuda(), scale, state.cuda())
    out, last = out.double().cpu(), last.double().cpu()
    odd = odd.reshape(1, N, H * d)
    assert not torch.isfinite(out[0, 0][odd[0, 0]]).any()
    # A state whose terms sum to less than fp32's smallest normal number, 2^-126, has no half step relative to itself: 0.5^150 * 1e-4 of the first head
    # is 7e-50 where fp32 ends at 1.4e-45, so it is off by itself; by 2^-126 at most.
    small = want[3] < 2.0 ** -126
    assert ((last - want[1]).abs() <= 2.0 ** -126)[small & ~odd_state].all()
    check((torch.where(odd, want[0], out), torch.where(odd_state | small, want[1], last)), want, q, N)
