"""GPU: attention of ragged batches of new tokens over a paged cache (causal, window, sinks) against the definition in 64
bits, at the sizes and masks where it can go wrong; strides, streams, captured launches, refusals."""
import ctypes as C

import numpy as np
import pytest
import torch

from chunkcases import BAD_PAGE, ChunkCase, check

pytestmark = pytest.mark.gpu

# hq, hkv, d, page, q_lens, kv_lens, window, sinks
CASES = {
    "one_token": (16, 2, 128, 16, [1], [1], 0, 0),
    "one_token_d64": (14, 2, 64, 16, [1], [513], 0, 0),
    "decode_ragged": (16, 2, 128, 16, [1] * 9, [1, 2, 15, 16, 17, 127, 128, 129, 1000], 0, 0),
    "decode_pages64": (8, 8, 128, 64, [1, 1, 1], [63, 64, 700], 0, 0),
    "decode_long": (8, 1, 128, 32, [1, 1], [20000, 3], 0, 0),
    "verify": (16, 2, 128, 16, [5, 3, 8, 1], [700, 3, 8, 4097], 0, 0),
    "empty_sequences": (16, 2, 128, 16, [0, 4, 0, 1, 0], [300, 40, 0, 7, 9], 0, 0),
    "rows_before_the_start": (8, 2, 128, 16, [6, 5, 130], [4, 0, 100], 0, 0),
    "prompt": (16, 2, 128, 16, [333], [833], 0, 0),
    "prompt_from_nothing": (8, 8, 128, 32, [257], [257], 0, 0),
    "prompt_d64_group7": (14, 2, 64, 16, [200, 131], [500, 131], 0, 0),
    "prompt_pages8": (8, 2, 128, 8, [129], [259], 0, 0),
    "prompt_pages128": (16, 2, 128, 128, [148], [1148], 0, 0),
    "mixed": (16, 2, 128, 16, [1, 300, 1, 17, 64, 1], [900, 1500, 1, 17, 64, 2049], 0, 0),
    "group1": (4, 4, 128, 16, [140, 1], [300, 77], 0, 0),
    "group3": (6, 2, 128, 16, [90, 1, 2], [300, 77, 5], 0, 0),
    "group5": (5, 1, 64, 64, [55, 1], [300, 777], 0, 0),
    "group16": (32, 2, 128, 16, [20, 1], [300, 77], 0, 0),
    "group64": (64, 1, 128, 16, [5, 1], [300, 77], 0, 0),
    "group48_d64": (48, 1, 64, 32, [7, 1], [300, 77], 0, 0),
    "window_decode": (16, 2, 128, 16, [1] * 6, [1, 100, 128, 129, 5000, 4096], 128, 0),
    "window_decode_sinks": (16, 2, 128, 16, [1] * 6, [1, 3, 130, 1025, 5000, 4096], 1024, 4),
    "window_one": (16, 2, 128, 16, [1, 40, 200], [50, 50, 1000], 1, 0),
    "window_one_sinks": (16, 2, 64, 16, [1, 40, 200], [50, 50, 1000], 1, 19),
    "window_prompt": (14, 2, 64, 32, [700, 1], [2000, 999], 100, 0),
    "window_prompt_sinks": (16, 2, 128, 16, [300, 5], [2000, 999], 200, 4),
    "window_many_sinks": (8, 2, 128, 16, [100, 1, 1], [900, 400, 90], 33, 150),
    "window_wider_than_all": (8, 2, 128, 64, [100, 1], [300, 77], 100000, 3),
    "window_rows_before_the_start": (8, 2, 128, 16, [20, 9], [4, 9], 3, 2),
    "window_sinks_inside_page": (8, 2, 128, 64, [1, 33], [1000, 1000], 65, 70),
    "window_pages128": (8, 2, 128, 128, [1, 50], [1000, 1100], 129, 1),
    "window_4096": (16, 2, 128, 16, [1] * 5, [512, 4095, 4097, 9001, 16000], 4096, 4),
}


@pytest.mark.parametrize("name", CASES)
def test_against_definition(mfk, foundry, name):
    hq, hkv, d, page, ql, kl, window, sinks = CASES[name]
    case = ChunkCase(hq=hq, hkv=hkv, d=d, page=page, q_lens=ql, kv_lens=kl, window=window, sinks=sinks)
    plan = case.plan(foundry)
    out = torch.full((case.tokens + 2, hq * d), 7.0, dtype=torch.float16, device="cuda")
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    foundry.synchronize()
    check(out[:case.tokens], case)
    assert bool((out[case.tokens:] == 7.0).all()), "rows behind the last sequence were written"
    again = torch.empty_like(out)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, again)
    foundry.synchronize()
    assert torch.equal(out[:case.tokens], again[:case.tokens]), "two calls on the same inputs differ"
    plan.close()


@pytest.mark.parametrize("page", [8, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
@pytest.mark.parametrize("q_len", [1, 20])
def test_last_half_tiles(mfk, foundry, page, window, sinks, q_len):
    """Lengths around the halves of a tile (64 keys): a last half that no row sees is left out, whatever it holds."""
    lens = [x + y for x in (0, 128, 256) for y in (1, 20, 63, 64, 65, 83, 84, 127, 128)]
    lens = [n for n in lens if n >= q_len]
    case = ChunkCase(hq=8, hkv=1, d=128 if page == 64 else 64, page=page, q_lens=[q_len] * len(lens), kv_lens=lens, window=window, sinks=sinks)
    plan, out = case.plan(foundry), torch.empty_like(case.q)
    for _ in range(2):
        out.fill_(float("nan"))
        foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
        foundry.synchronize()
        check(out, case)


def test_scores_far_apart(mfk, foundry):
    """Scores of several hundred (weights that underflow, maxima that keep moving) and a scale of the caller's."""
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[130, 1], kv_lens=[700, 1500], spread=30.0)
    plan, out = case.plan(foundry), torch.empty_like(case.q)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out, scale=0.01)
    foundry.synchronize()
    check(out, case, scale=0.01)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out, scale=0.0)  # every visible key counts alike
    foundry.synchronize()
    check(out, case, scale=0.0)
    # |s| reaches 300 here: f32 scores are off by up to 128 * 2^-24 * 300 = 2^-8.7 relative to the weights
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    foundry.synchronize()
    want, tol = case.expected()
    mean = (tol - 2.0 ** -25) / (2.0 ** -11 + 2.0 ** -12)
    assert bool(((out.double().view_as(want) - want).abs() <= tol + 2.0 ** -8 * mean + 2.0 ** -9).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_hidden_from_some_rows(mfk, foundry, value):
    """A key or value row that is not finite shows in the rows that see it and in no other row of the same chunk."""
    for hq, hkv, q_len, kv_len, window, sinks, at in ((8, 2, 40, 300, 0, 0, 290), (8, 2, 300, 500, 64, 2, 350),
                                                      (8, 1, 4, 2000, 0, 0, 1998)):
        case = ChunkCase(hq=hq, hkv=hkv, d=128, page=16, q_lens=[q_len], kv_lens=[kv_len], window=window, sinks=sinks)
        want, tol = case.expected()
        rows = ~case.visible(0)[:, at]
        assert bool(rows.any()) and not bool(rows.all())
        for pool in (case.k, case.v):
            page = int(case.table[0, at // 16])
            keep = pool[page, :, at % 16].clone()
            pool[page, :, at % 16] = value
            plan, out = case.plan(foundry), torch.empty_like(case.q)
            foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
            foundry.synchronize()
            off = (out.double().view_as(want) - want).abs()[rows]
            assert bool((off <= tol[rows]).all()), "a hidden row's value reached a row that does not see it"
            if pool is case.v and value != value:
                assert bool(torch.isnan(out.view(q_len, hq, 128)[~rows]).all())
            pool[page, :, at % 16] = keep
            plan.close()


def test_strides(mfk, foundry):
    """q as a slice of a fused projection's rows, out head-major, both wider than they need to be."""
    case = ChunkCase(hq=16, hkv=2, d=128, page=16, q_lens=[70, 1, 9], kv_lens=[200, 300, 9])
    wide = torch.randn((case.tokens, 20 * 128 + 8), device="cuda").half()
    wide[:, 8:8 + 2048] = case.q
    out = torch.full((16, case.tokens + 3, 136), 7.0, dtype=torch.float16, device="cuda")
    plan = case.plan(foundry)
    view = out[:, :case.tokens, :128].transpose(0, 1)
    foundry.paged_chunk_attention(plan, case.cache(mfk), wide[:, 8:8 + 2048], view)
    foundry.synchronize()
    check(view.reshape(case.tokens, -1), case)
    assert bool((out[:, case.tokens:] == 7.0).all()) and bool((out[..., 128:] == 7.0).all())


def test_plan_updates_and_max_tokens(mfk, foundry):
    first = ChunkCase(hq=16, hkv=2, d=128, page=16, q_lens=[3, 200], kv_lens=[30, 2000])
    plan = first.plan(foundry, max_tokens=900)
    for ql, kl in (([3, 200], [30, 2000]), ([1, 1], [31, 2001]), ([0, 0], [31, 2001]), ([700, 200], [700, 2100]), ([1, 0], [5000, 0])):
        case = ChunkCase(hq=16, hkv=2, d=128, page=16, q_lens=ql, kv_lens=kl)
        plan.update(ql, kl)
        out = torch.empty_like(case.q)
        foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
        foundry.synchronize()
        check(out[:case.tokens], case)
    with pytest.raises(mfk.MetalError, match="made for 900"):
        plan.update([901, 0], [901, 0])
    out = torch.empty_like(case.q)  # a refused update leaves the plan as it was
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    foundry.synchronize()
    check(out, case)


def test_captured_launch_follows_the_plan(mfk):
    """A captured launch replays the plan as it stands at the replay; an update is refused during capture."""
    stream = torch.cuda.Stream()
    f = mfk.Foundry(0, stream.cuda_stream)
    small = ChunkCase(hq=16, hkv=2, d=128, page=16, q_lens=[1, 1], kv_lens=[3000, 4000], window=256, sinks=4)
    plan = small.plan(f, max_tokens=400)
    q, out = torch.zeros((400, 2048), dtype=torch.float16, device="cuda"), torch.zeros((400, 2048), dtype=torch.float16, device="cuda")
    pools = [torch.zeros((400, 2, 16, 128), dtype=torch.float16, device="cuda") for _ in range(2)]
    table, lens = torch.zeros((2, 260), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = mfk.paged_kv(pools[0], pools[1], table, lens, n_kv_heads=2, page_size=16, head_dim=128)

    def fill(case):
        assert case.n_pages <= 400
        for p, x in zip(pools, (case.k, case.v)):
            p[:case.n_pages] = x
        table.fill_(BAD_PAGE)
        table[:, :case.table.shape[1]] = case.table
        q[:case.tokens] = case.q

    cases = [ChunkCase(hq=16, hkv=2, d=128, page=16, q_lens=ql, kv_lens=kl, window=256, sinks=4)
             for ql, kl in (([1, 1], [1500, 2000]), ([150, 1], [900, 3000]), ([1, 0], [700, 0]), ([200, 200], [200, 777]))]
    torch.cuda.synchronize()
    fill(cases[0])
    plan.update(cases[0].q_lens, cases[0].kv_lens)
    f.paged_chunk_attention(plan, cache, q, out)
    f.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        f.paged_chunk_attention(plan, cache, q, out)
        with pytest.raises(mfk.MetalError, match="captured"):
            plan.update([1, 1], [2, 2])
    for case in cases:
        torch.cuda.synchronize()
        fill(case)
        out.zero_()
        torch.cuda.synchronize()
        plan.update(case.q_lens, case.kv_lens)
        with torch.cuda.stream(stream):
            graph.replay()
            graph.replay()
        f.synchronize()
        check(out[:case.tokens], case)
        assert not bool(out[case.tokens:].any())
    del graph
    plan.close()
    f.close()


def test_two_plans_on_two_streams(mfk):
    """Independent contexts and plans at the same time."""
    runs = []
    for i in range(2):
        s = torch.cuda.Stream()
        f = mfk.Foundry(0, s.cuda_stream)
        case = ChunkCase(hq=16, hkv=2, d=128, page=16, q_lens=[1] * 8 + [90 + i], kv_lens=[1500 + 100 * i] * 8 + [900], seed=i)
        runs.append((f, case, case.plan(f), torch.empty_like(case.q)))
    torch.cuda.synchronize()
    for _ in range(5):
        for f, case, plan, out in runs:
            f.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    for f, case, plan, out in runs:
        f.synchronize()
        check(out, case)
        plan.close()
        f.close()


def test_bad_page_is_reported(mfk, foundry):
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[1, 1], kv_lens=[100, 200])
    plan, out = case.plan(foundry), torch.zeros_like(case.q)
    case.table[0, 3] = BAD_PAGE
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    with pytest.raises(mfk.MetalError) as e:
        foundry.synchronize()
    assert e.value.kind == "InvalidOperation"
    want, tol = case.expected()  # the other sequence is untouched by it
    assert bool(((out.double().view_as(want) - want).abs() <= tol)[1].all())
    foundry.synchronize()


def test_refusals(mfk, foundry):
    f = foundry

    def plan(kind, **kw):
        a = dict(q_lens=[1], kv_lens=[10], n_heads=8, n_kv_heads=2, head_dim=128, page_size=16) | kw
        with pytest.raises(mfk.MetalError) as e:
            f.chunk_plan(a.pop("q_lens"), a.pop("kv_lens"), **a)
        assert e.value.kind == kind, e.value

    plan("OperationNotSupported", head_dim=96)
    plan("OperationNotSupported", page_size=24)
    plan("OperationNotSupported", page_size=4)
    plan("OperationNotSupported", n_heads=130, n_kv_heads=2)
    plan("InvalidShape", n_heads=7)
    plan("InvalidShape", n_heads=0)
    plan("InvalidShape", q_lens=[], kv_lens=[])
    plan("InvalidShape", q_lens=[1, 2], kv_lens=[1])
    plan("InvalidShape", q_lens=[1 << 31])
    plan("InvalidShape", kv_lens=[1 << 31])
    plan("InvalidShape", q_lens=[2], max_tokens=1)
    plan("InvalidOperation", sinks=4)

    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[2, 1], kv_lens=[100, 50])
    p, out = case.plan(f), torch.zeros_like(case.q)
    good = case.cache(mfk)

    def call(kind, cache=good, q=case.q, o=out, **kw):
        with pytest.raises(mfk.MetalError) as e:
            f.paged_chunk_attention(p, cache, q, o, **kw)
        assert e.value.kind == kind, e.value

    def other(**kw):
        c = case.cache(mfk)  # a descriptor with other fields
        for k, x in kw.items():
            setattr(c, k, x)
        return c

    call("InvalidOperation", scale=-1.0)
    call("InvalidOperation", scale=float("nan"))
    call("InvalidOperation", scale=float("inf"))
    call("InvalidOperation", scale=3e38)  # finite, but not in the exponent of two
    call("InvalidOperation", cache=other(page_table_stride=6))
    call("InvalidShape", cache=other(batch=3))
    call("InvalidShape", cache=other(page_size=32))
    call("InvalidShape", cache=other(n_kv_heads=1))
    call("InvalidShape", cache=other(n_pages=0))
    call("InvalidShape", cache=other(n_pages=1 << 30))
    call("InvalidShape", cache=other(k_pool=good.k_pool + 8))
    call("InputNotFound", cache=other(v_pool=None))
    call("InputNotFound", cache=other(page_table=None))
    call("InvalidShape", q=case.q[:2])
    call("InvalidShape", q=torch.zeros((3, 1024 + 4), dtype=torch.float16, device="cuda")[:, 4:])
    call("InvalidShape", o=torch.zeros((3, 1024 + 4), dtype=torch.float16, device="cuda")[:, :1024])
    assert not bool(out.any())
    assert mfk.lib.mf_paged_chunk_attention(None, p._h, C.byref(good), None) == 4
    assert np.all(case.table[:, :1].cpu().numpy() >= 0)


def test_another_current_device_is_put_back(mfk, foundry):
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[2], kv_lens=[100])
    p, out = case.plan(foundry), torch.zeros_like(case.q)
    foundry.paged_chunk_attention(p, case.cache(mfk), case.q, out)
    assert torch.cuda.current_device() == 0
    foundry.synchronize()
    check(out, case)


def test_other_types_and_memories_are_refused(mfk, foundry):
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[2, 1], kv_lens=[100, 50])
    plan, cache, out = case.plan(foundry), case.cache(mfk), torch.zeros_like(case.q)
    for q, o in ((case.q.bfloat16(), out), (case.q, out.bfloat16()), (case.q.cpu(), out), (case.q, out.cpu()),
                 (case.q.view(torch.int16), out), (case.q.flatten(), out)):
        with pytest.raises(mfk.MetalError) as e:
            foundry.paged_chunk_attention(plan, cache, q, o)
        assert e.value.kind == "InvalidShape"
    foundry.synchronize()
    assert not bool(out.any())


def test_sequences_without_keys_among_many(mfk, foundry):
    """Rows that see nothing come out as zeros wherever their units fall in the CTAs' spans."""
    kv_lens = [0 if i % 3 == 1 else 40 + 37 * (i % 11) for i in range(60)]
    q_lens = [i % 4 if kv else 3 for i, kv in enumerate(kv_lens)]
    case = ChunkCase(hq=56, hkv=8, d=128, page=128, q_lens=q_lens, kv_lens=kv_lens)
    plan, out = case.plan(foundry), torch.full_like(case.q, float("nan"))
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    foundry.synchronize()
    check(out, case)
