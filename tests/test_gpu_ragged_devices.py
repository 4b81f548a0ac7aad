"""GPU (two of them): the ragged-batch operators of one device's context while another device is the current one."""
import numpy as np
import pytest
import torch

from chunkcases import ChunkCase, check

pytestmark = pytest.mark.gpu


@pytest.fixture
def two():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    yield
    torch.cuda.set_device(0)


def test_the_current_device_is_put_back(mfk, two):
    """Plan, append, attention and moves on device 0 while device 1 is current: done there, and 1 is current after each."""
    torch.cuda.set_device(0)
    f = mfk.Foundry(0, torch.cuda.current_stream(0).cuda_stream)
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[2, 40], kv_lens=[100, 300])
    cache, out = case.cache(mfk), torch.zeros_like(case.q)
    new = torch.randn((case.tokens, 2 * 128), device="cuda:0").half()
    ones, zeros = torch.ones((1, 64), device="cuda:0").half(), torch.zeros((1, 64), device="cuda:0").half()
    pos = torch.zeros((1, case.tokens), dtype=torch.int32, device="cuda:0")
    begin = torch.tensor([0, 2, 42], dtype=torch.int32, device="cuda:0")
    free = sorted(set(range(case.n_pages)) - set(case.table.flatten().tolist()))[:1]
    torch.cuda.synchronize()
    torch.cuda.set_device(1)
    plan = case.plan(f)
    assert torch.cuda.current_device() == 1
    f.paged_chunk_attention(plan, cache, case.q, out)
    assert torch.cuda.current_device() == 1
    f.synchronize()
    check(out, case)
    f.paged_mrope_append(cache, None, new, new, None, ones, zeros, pos, begin, bytes(64), n_heads=8)
    assert torch.cuda.current_device() == 1
    f.paged_move_pages(mfk.kv_layers([cache]), case.table[0, :1].cpu().numpy(), np.array(free))
    assert torch.cuda.current_device() == 1
    f.synchronize()
    assert torch.equal(case.k[free[0]].view(torch.int16), case.k[int(case.table[0, 0])].view(torch.int16))
    t = 0
    for b, n in enumerate(case.q_lens):
        for r in range(n):
            row = case.kv_lens[b] - n + r
            at = case.k[int(case.table[b, row // 16]), :, row % 16]
            assert torch.equal(at, new[t + r].view(2, 128))
        t += n
    plan.close()
    assert torch.cuda.current_device() == 1
    f.close()


def test_a_plan_of_another_device_is_refused(mfk, two):
    a, b = (mfk.Foundry(i, torch.cuda.current_stream(i).cuda_stream) for i in range(2))
    torch.cuda.set_device(0)
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[2], kv_lens=[100])
    plan = case.plan(a)
    q, kv = np.array([2], np.uint32), np.array([100], np.uint32)
    assert mfk.lib.mf_chunk_plan_update(b._h, plan._h, q.ctypes.data, kv.ctypes.data) == 3  # InvalidOperation
    assert mfk.lib.mf_chunk_plan_update(a._h, plan._h, q.ctypes.data, kv.ctypes.data) == 0
    plan.close()
    a.close()
    b.close()

