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


def test_a_plan_on_another_stream_than_its_updates(mfk):
    """A launch of another context waits for the update in front of it, and the next update waits for the launch, however late
    either stream is."""
    late = [torch.cuda.Stream() for _ in range(2)]
    a, b = (mfk.Foundry(0, s.cuda_stream) for s in late)
    kw = dict(hq=8, hkv=2, d=128, page=16)
    cases = [ChunkCase(**kw, q_lens=q, kv_lens=kv, seed=i) for i, (q, kv) in
             enumerate((([1, 1], [3000, 2000]), ([200, 3], [900, 3]), ([2, 190], [5, 700])))]
    caches = [c.cache(mfk) for c in cases]
    outs = [torch.zeros((256, 1024), dtype=torch.float16, device="cuda") for _ in cases]
    qs = [torch.zeros((256, 1024), dtype=torch.float16, device="cuda") for _ in cases]
    for q, c in zip(qs, cases):
        q[:c.tokens] = c.q
    plan = cases[0].plan(a, max_tokens=256)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(late[0]):
            torch.cuda._sleep(3_000_000)
        plan.update(cases[1].q_lens, cases[1].kv_lens)      # late, on a's stream
        b.paged_chunk_attention(plan, caches[1], qs[1], outs[1])
        with torch.cuda.stream(late[1]):
            torch.cuda._sleep(3_000_000)
        b.paged_chunk_attention(plan, caches[1], qs[1], outs[1])
        plan.update(cases[2].q_lens, cases[2].kv_lens)      # not before b's launches are over
        a.paged_chunk_attention(plan, caches[2], qs[2], outs[2])
        a.synchronize()
        b.synchronize()
        for out, case in list(zip(outs, cases))[1:]:
            check(out[:case.tokens], case)
            assert not bool(out[case.tokens:].any())
            out.zero_()
        torch.cuda.synchronize()
    plan.close()
    a.close()
    b.close()
