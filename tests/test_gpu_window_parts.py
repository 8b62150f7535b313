"""Window attention whose keys are split into parts: what is not finite in a part that weighs nothing."""
import math

import pytest
import torch

from sana_amd import _lib, ops
from test_gpu_window_attention import BF16, F16, check, definition, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("loud", [3000, 200])
def test_values_that_are_not_finite_in_parts_without_weight(cuda, loud, dtype):
    """The scores of one stretch of keys are 2^300 above all others, whose parts have a weight of 0 in 32 bits.  They are seen all the same:
    their inf and NaN reach the output, as they do where the keys are not split."""
    N, Nk, H, d = 2, 4000, 2, 64
    assert _lib.load().sana_hip_window_attention_workspace_bytes(1, N, Nk, H, d, 5000, 4) > 0
    q, k, v = make(1, N, Nk, H, H, d, dtype, packed=False)
    q, k = torch.ones_like(q), k.abs() * -0.5
    k[0, loud:loud + 40] = 4.0
    clean = v.clone()
    extra = torch.zeros(1, N, H * d, dtype=torch.float64)
    for j, c, x in [(5, 3, math.inf), (1500, 70, -math.inf), (2200, 9, math.nan), (2900, 100, math.inf), (2901, 100, -math.inf), (3999, 40, math.inf)]:
        v[0, j, c], clean[0, j, c] = x, 0
        extra[0, 1 if j == Nk - 1 else 0:, c] += x   # (only the last query sees the last key)
    want = definition(q, k, clean, H, 5000, 4, 1.0)
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), H, 5000, 4, 1.0).double().cpu()
    odd = extra != 0
    same = lambda t: torch.nan_to_num(t[odd], nan=7.0, posinf=8.0, neginf=9.0)  # noqa: E731
    assert torch.equal(same(got), same(extra)), (got[odd], extra[odd])
    check(torch.where(odd, want[0], got), want, Nk, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_token_sees_what_is_not_finite_in_parts_without_weight(cuda, dtype):
    rows, H, d = 6000, 2, 64
    assert _lib.load().sana_hip_window_step_workspace_bytes(1, H, H, d, rows - 4, 4) > 0
    q, k, v = make(1, rows, rows, H, H, d, dtype, packed=False)
    q, k = torch.ones_like(q), k.abs() * -0.5
    k[0, 3000:3040] = 4.0
    v[0, 10, 3], v[0, 5500, 70], v[0, 4000, 9] = math.inf, -math.inf, math.nan
    clean = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    want = definition(q[:, -1:], k, clean, H, rows, 4, 1.0)
    pos = torch.tensor([rows - 1], dtype=torch.int32, device=cuda)
    got = ops.window_attention_step_(q[:, -1:].cuda(), k[:, -1:].cuda(), v[:, -1:].cuda(), k.cuda(), v.cuda(), pos, H, 4, 1.0).double().cpu()
    odd = torch.zeros(1, 1, H * d, dtype=torch.bool)
    odd[..., [3, 70, 9]] = True
    assert not torch.isfinite(got[odd]).any()
    check(torch.where(odd, want[0], got), want, rows, dtype)
