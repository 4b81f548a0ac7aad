"""GPU: page moves and the multi-axis append directly in front of a fused decode on the pages that they write, with launches that
overlap: the decode waits for them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, P = 16, 2, 128, 16


@pytest.mark.parametrize("overlap", [0, 1, 2])
def test_decode_behind_moves_and_appends(mfk, overlap):
    f = mfk.Foundry(0, torch.cuda.Stream().cuda_stream)
    g = torch.Generator(device="cuda").manual_seed(3)
    batch, kv = 4, 1600
    per = kv // P
    n = batch * per
    base = [torch.randn((2 * n, HKV, P, D), generator=g, device="cuda").half() for _ in range(2)]
    for x in base:
        x[n:] = 0
    order = torch.randperm(n, generator=g, device="cuda").cpu().numpy().astype(np.uint32)
    table = torch.from_numpy((order + n).astype(np.int32)).view(batch, per).cuda()
    lens = torch.full((batch,), kv, dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn((batch, h * D), generator=g, device="cuda").half() for h in (HQ, HKV, HKV))
    cos, sin = (torch.from_numpy(x.view(np.float16).copy()).cuda() for x in mfk.rope_tables(1e4, D, 2048))
    kw = dict(n_kv_heads=HKV, page_size=P, head_dim=D)
    pools = [x.clone() for x in base]
    cache = mfk.paged_kv(*pools, table, lens, **kw)
    layers = mfk.kv_layers([cache])
    plan = f.decode_plan([kv] * batch, n_heads=HQ, **kw)
    news = [torch.randn((batch * 200, HKV * D), generator=g, device="cuda").half() for _ in range(2)]
    begin = torch.arange(0, batch * 200 + 1, 200, dtype=torch.int32, device="cuda")
    pos = torch.arange(kv - 200, kv, dtype=torch.int32, device="cuda").repeat(batch)[None].contiguous()
    out = [torch.empty((batch, HQ * D), dtype=torch.float16, device="cuda") for _ in range(3)]
    args = dict(n_heads=HQ, k=k, v=v, cos=cos, sin=sin, rope=True, append=True)
    f.set_option(mfk.OPTION_OVERLAP_LAUNCHES, overlap)
    results = []
    for _ in range(4):
        for p, x in zip(pools, base):
            p.copy_(x)
        torch.cuda.synchronize()
        f.paged_decode(plan, cache, q, out[0], **args)
        f.paged_move_pages(layers, order, order + n)     # every page that the next launch reads
        f.paged_decode(plan, cache, q, out[1], **args)
        f.paged_mrope_append(cache, None, news[0], news[1], None, cos, sin, pos, begin, bytes(D // 2), n_heads=HQ)
        f.paged_decode(plan, cache, q, out[2], **args)
        f.synchronize()
        results.append([x.clone() for x in out + pools])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
    f.set_option(mfk.OPTION_OVERLAP_LAUNCHES, 0)
    for p, x in zip(pools, base):
        p.copy_(x)
    torch.cuda.synchronize()
    for step in range(3):
        if step == 1:
            f.paged_move_pages(layers, order, order + n)
        elif step == 2:
            f.paged_mrope_append(cache, None, news[0], news[1], None, cos, sin, pos, begin, bytes(D // 2), n_heads=HQ)
        f.synchronize()
        f.paged_decode(plan, cache, q, out[step], **args)
        f.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results[0], out + pools))
    assert not torch.equal(out[0], out[1]) and not torch.equal(out[1], out[2])
    plan.close()
    f.close()
