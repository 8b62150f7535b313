"""Host threads that call at the same time on one stream: a call of several launches keeps its scratch from the other's."""
import threading

import pytest
import torch

from sana_amd import _lib, ops

BF16 = torch.bfloat16


def in_thread(f):
    got = []
    t = threading.Thread(target=lambda: got.append(f()))
    t.start()
    t.join()
    return got[0]


def test_threads_have_scratch_of_their_own(monkeypatch):
    """ctypes releases the interpreter's lock between the launches of a call, so the launches of two threads' calls may lie between each
    other's on the one stream that both use."""
    monkeypatch.setattr(ops, "_workspaces", {})
    handle, cpu = 0x5eed, torch.device("cpu")
    mine = ops._workspace(cpu, 1000, handle)
    other = in_thread(lambda: ops._workspace(cpu, 1000, handle))
    assert mine.data_ptr() != other.data_ptr()
    assert ops._workspace(cpu, 1000, handle) is mine          # one thread's calls on a stream share it
    assert ops._workspace(cpu, 1000, handle + 1) is not mine


@pytest.mark.gpu
def test_two_threads_on_one_stream_get_the_serial_results(cuda):
    lib = _lib.load()
    assert lib.sana_hip_decay_attention_workspace_bytes(1, 2000, 2, 64) > 0
    assert lib.sana_hip_window_attention_workspace_bytes(1, 3, 2000, 2, 64, 1500, 4) > 0
    assert lib.sana_hip_window_step_workspace_bytes(1, 2, 2, 64, 3996, 4) > 0
    sets = []
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        x = torch.randn(1, 4000, 3 * 128, generator=gen).to(BF16).cuda()
        q, k, v = x.split(128, dim=2)
        g = torch.tensor([-0.1, -0.001], device=cuda)
        cache = [t.contiguous().clone() for t in (k, v)]
        pos = torch.tensor([3999], dtype=torch.int32, device=cuda)
        sets.append((q, k, v, g, cache, pos))

    def calls(q, k, v, g, cache, pos):
        h = slice(0, 2000)
        return [*ops.decay_linear_attention(q[:, h], k[:, h], v[:, h], g), ops.window_attention(q[:, 1997:2000], k[:, h], v[:, h], 2, 1500, 4),
                ops.window_attention_step_(q[:, -1:], k[:, -1:], v[:, -1:], *cache, pos, 2, 4),
                ops.relu_linear_attention(q, k, v, 1e-8)]

    want = [calls(*s) for s in sets]
    torch.cuda.synchronize()
    got, start = [[], []], threading.Barrier(2)

    def loop(i):
        start.wait()
        for _ in range(40):
            got[i].append(calls(*sets[i]))

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 40
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
