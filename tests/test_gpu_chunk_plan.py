"""GPU: plans of ragged batches, stream capture and memory: what cannot be is refused and leaves everything as it was."""
import pytest
import torch

from chunkcases import ChunkCase, check

pytestmark = pytest.mark.gpu


def test_no_plan_is_made_during_a_capture(mfk):
    stream = torch.cuda.Stream()
    f = mfk.Foundry(0, stream.cuda_stream)
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[3, 1], kv_lens=[100, 50])
    plan, out = case.plan(f), torch.zeros_like(case.q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        f.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
        with pytest.raises(mfk.MetalError) as e:
            case.plan(f)
        assert e.value.kind == "InvalidOperation" and "captured" in str(e.value)
    with torch.cuda.stream(stream):
        graph.replay()
    f.synchronize()
    check(out, case)
    del graph
    plan.close()
    f.close()


def test_a_captured_call_has_room_for_later_updates(mfk):
    """The plan may grow to max_tokens before a replay: q and out that do not hold as many are refused in a capture."""
    stream = torch.cuda.Stream()
    f = mfk.Foundry(0, stream.cuda_stream)
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[3, 1], kv_lens=[100, 50])
    plan, cache = case.plan(f, max_tokens=40), case.cache(mfk)
    q, out = torch.zeros((40, 1024), dtype=torch.float16, device="cuda"), torch.zeros((40, 1024), dtype=torch.float16, device="cuda")
    q[:4] = case.q
    torch.cuda.synchronize()
    f.paged_chunk_attention(plan, cache, q[:4], out[:4])  # not captured: the step's own tokens are enough
    f.synchronize()
    check(out[:4], case)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for a, b in ((q[:39], out), (q, out[:39]), (q[:4], out[:4])):
            with pytest.raises(mfk.MetalError) as e:
                f.paged_chunk_attention(plan, cache, a, b)
            assert e.value.kind == "InvalidShape" and "40" in str(e.value)
        f.paged_chunk_attention(plan, cache, q, out)
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    f.synchronize()
    check(out[:4], case)
    assert not bool(out[4:].any())
    del graph
    plan.close()
    f.close()


def test_a_plan_that_does_not_fit_leaves_nothing_behind(mfk, foundry):
    """More work items than the GPU's memory holds (some 258 GB): refused, and the next call is not blamed for it."""
    with pytest.raises(mfk.MetalError) as e:
        foundry.chunk_plan([1], [1], n_heads=960, n_kv_heads=960, head_dim=64, page_size=16, max_tokens=1 << 30)
    assert e.value.kind == "OutOfMemory"
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[3, 1], kv_lens=[100, 50])
    plan, out = case.plan(foundry), torch.zeros_like(case.q)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    foundry.synchronize()
    check(out, case)
    plan.close()


def test_more_items_than_can_be_numbered(mfk, foundry):
    with pytest.raises(mfk.MetalError) as e:
        foundry.chunk_plan([1], [1], n_heads=4096, n_kv_heads=4096, head_dim=64, page_size=16, max_tokens=1 << 30)
    assert e.value.kind == "InvalidShape"
