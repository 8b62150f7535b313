"""Window attention by the kernel whose waves take two tiles of 16 queries: wide heads and many blocks."""
import pytest
import torch

from sana_amd import _lib
from test_gpu_window_attention import BF16, F16, compare, make, test_values_that_are_not_finite_reach_who_sees_them as not_finite

gpu = pytest.mark.gpu


def tiles(B, N, H, d):
    return _lib.load().sana_hip_window_attention_query_tiles(B, N, H, d)


def test_which_calls_take_two_query_tiles():
    for d in (104, 112, 128):
        assert tiles(1, 2560, 20, d) == 1 and tiles(1, 2561, 20, d) == 2   # 400 and 420 blocks of 128 queries
        assert tiles(4, 385, 40, d) == 2 and tiles(1, 1, 400, d) == 1 and tiles(1, 1, 401, d) == 2
    assert tiles(4, 385, 40, 96) == 1 and tiles(0, 1, 1, 112) == 0 and tiles(1, 1, 1, 136) == 0


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [104, 112, 128])
@pytest.mark.parametrize("N,past,window,sinks", [(385, 0, 100, 3), (385, 200, 130, 70), (400, 77, 5000, 0), (511, 0, 1, 0), (385, 64, 64, 64)])
def test_blocks_of_128_queries(cuda, N, past, window, sinks, d, dtype):
    assert tiles(4, N, 40, d) == 2
    compare(*make(4, N, past + N, 40, 8, d, dtype, seed=N + d), 40, window, sinks)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths", [[385, 129, 128, 1], [0, 16, 17, 300]])
def test_streams_of_unlike_length(cuda, lengths, dtype):
    assert tiles(4, 385, 40, 112) == 2
    compare(*make(4, 385, 450, 40, 4, 112, dtype, packed=False), 40, 90, 66, lengths=lengths)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_of_every_size(cuda, dtype):
    """Rows that one key takes whole, a maximum that rises or falls from tile to tile, and scores of thousands."""
    assert tiles(3, 300, 50, 112) == 2
    q, k, v = make(3, 300, 300, 50, 2, 112, dtype, packed=False)
    compare(q, k, v, 50, 150, 4, scale=20.0)
    ramp = torch.linspace(0.05, 6, 300)[None, :, None]
    compare((q.abs() * ramp).to(dtype), (k.abs() * ramp).to(dtype), v, 50, 150, 4, scale=0.5)
    compare((q.abs() * ramp.flip(1)).to(dtype), (k.abs() * ramp.flip(1)).to(dtype), v, 50, 150, 4, scale=0.5)
    compare(-q.abs() * 6, k.abs() * 6, v, 50, 150, 4, scale=2.0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,past,window,sinks,d", [(2600, 0, 100, 3, 128), (2570, 90, 300, 70, 112)])
def test_values_that_are_not_finite(cuda, N, past, window, sinks, d, dtype):
    assert tiles(1, N, 20, d) == 2
    not_finite(cuda, N, past, window, sinks, d, dtype)
