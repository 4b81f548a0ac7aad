"""GPU: plans of ragged batches and stream capture: what a capture cannot hold is refused and leaves the capture as it was."""
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
