"""GPU: the ragged-batch operators together, as a serving loop uses them: a prompt in chunks (append with positions on
three axes, windowed attention), a fork, single tokens, freeing behind the window, compaction - against a model in 64
bits that keeps every sequence's rows in plain arrays."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, P, W, SINKS, LAYERS, POOL = 8, 2, 128, 16, 96, 4, 2, 64


class Sequence:
    def __init__(self):
        self.pages = np.zeros(0, np.uint32)
        self.length = 0
        self.rows = [[torch.zeros((HKV, 0, D), dtype=torch.float64, device="cuda") for _ in range(2)] for _ in range(LAYERS)]

    def child(self):
        c = Sequence()
        c.length, c.rows = self.length, [[x.clone() for x in r] for r in self.rows]
        return c


def test_serving_loop(mfk, foundry):
    g = torch.Generator(device="cuda").manual_seed(2)
    pool = mfk.PagePool(POOL)
    k, v = (torch.full((LAYERS, POOL, HKV, P, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    cos, sin = (torch.from_numpy(x.view(np.float16).copy()).cuda() for x in mfk.rope_tables(1e4, D, 4096))
    axes = mfk.mrope_axes([16, 24, 24])
    axis = torch.tensor(list(axes), device="cuda").long()
    table = torch.full((3, 64), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    caches = [mfk.paged_kv(k[i], v[i], table, lens, n_kv_heads=HKV, page_size=P, head_dim=D) for i in range(LAYERS)]
    layers = mfk.kv_layers(caches)
    seqs = [Sequence(), Sequence()]
    plans = {}

    def step(q_lens):
        tokens = int(sum(q_lens))
        table.fill_(-1)
        for b, (s, n) in enumerate(zip(seqs, q_lens)):
            need = -(-(s.length + n) // P) - s.pages.size
            s.pages = np.concatenate([s.pages, pool.alloc(need)]) if need > 0 else s.pages
            s.length += n
            table[b, :s.pages.size] = torch.from_numpy(s.pages.view(np.int32)).cuda()
        q_lens = list(q_lens) + [0] * (3 - len(q_lens))
        kv = [s.length for s in seqs] + [0] * (3 - len(seqs))
        begin = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
        lens.copy_(torch.tensor(kv, dtype=torch.int32))
        if not plans:
            plans["w"] = foundry.chunk_plan(q_lens, kv, n_heads=HQ, n_kv_heads=HKV, head_dim=D, page_size=P, window=W, sinks=SINKS,
                                            max_tokens=512)
        plans["w"].update(q_lens, kv)
        pos = torch.randint(0, 4096, (3, tokens), generator=g, device="cuda", dtype=torch.int32)
        for i in range(LAYERS):
            qkv = torch.randn((tokens, (HQ + 2 * HKV) * D), generator=g, device="cuda").half()
            q, kn, vn = qkv.split([HQ * D, HKV * D, HKV * D], 1)
            rot, out = torch.empty((tokens, HQ * D), dtype=torch.float16, device="cuda"), torch.empty((tokens, HQ * D), dtype=torch.float16, device="cuda")
            foundry.paged_mrope_append(caches[i], q, kn, vn, rot, cos, sin, pos, begin, axes, n_heads=HQ)
            foundry.paged_chunk_attention(plans["w"], caches[i], rot, out)
            foundry.synchronize()
            row = pos.long()[axis].t()
            c, s_ = (t[row, torch.arange(D // 2, device="cuda")].double()[:, None] for t in (cos, sin))

            def turned(x, heads):
                a, b = x.reshape(tokens, heads, 2, D // 2).double().unbind(2)
                return torch.cat([a * c - b * s_, b * c + a * s_], -1).half().double()

            tq, tk, tv = turned(q, HQ), turned(kn, HKV), vn.reshape(tokens, HKV, D).double()
            t = 0
            for b, (s, n) in enumerate(zip(seqs, q_lens)):
                if n == 0:
                    continue
                s.rows[i] = [torch.cat([old, new[t:t + n].transpose(0, 1)], 1) for old, new in zip(s.rows[i], (tk, tv))]
                kk, vv = (x.repeat_interleave(HQ // HKV, 0) for x in s.rows[i])
                key, at = torch.arange(s.length, device="cuda"), torch.arange(s.length - n, s.length, device="cuda")[:, None]
                see = (key <= at) & ((at - key < W) | (key < SINKS))
                w = torch.softmax((tq[t:t + n].transpose(0, 1) @ kk.transpose(1, 2) * D ** -0.5).masked_fill(~see, -float("inf")), -1)
                want, mean = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
                got = out[t:t + n].view(n, HQ, D).double()
                # a weight and the output are each rounded to f16, f32 sums take the rest (see chunkcases.py)
                assert bool(((got - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mean + 2.0 ** -16).all())
                t += n

    def free_hidden():
        for s in seqs:
            s.pages, _ = pool.release_hidden(s.pages, s.length, P, W, SINKS)
        for i in range(POOL):
            if pool.refcount(i) == 0:
                k[:, i], v[:, i] = float("nan"), float("nan")

    step([150, 1])
    step([100, 40])
    free_hidden()
    assert pool.free_count > POOL - 26
    child = seqs[0].child()
    child.pages, copies = pool.fork(seqs[0].pages, seqs[0].length, P)
    assert len(copies) == 1
    foundry.paged_move_pages(layers, *np.array(copies, np.uint32).T)
    seqs.append(child)
    for n in range(5):
        step([1, 1, 1])
    free_hidden()
    src, dst = pool.compact()
    assert src.size > 0
    foundry.paged_move_pages(layers, src, dst)
    for s in seqs:
        s.pages = mfk.remap_page_ids(s.pages, src, dst)
    foundry.synchronize()
    live = POOL - pool.free_count
    k[:, live:], v[:, live:] = float("nan"), float("nan")
    step([1, 5, 1])
    step([33, 1, 64])
    for s in seqs:
        pool.release(s.pages[s.pages != mfk.FREED_PAGE])
    assert pool.free_count == POOL
    plans["w"].close()
    pool.close()


def test_agrees_with_the_batched_decode(mfk):
    """One new token per sequence: mf_paged_decode (append and rotation inside, launches overlapping) and the append with
    equal positions on all axes + chunk attention leave the same rows in the pools and the same attention, up to the two
    kernels' roundings of the weights (each within 2^-11 + 2^-12 of the weighted mean of |v|, see chunkcases.py)."""
    f = mfk.Foundry(0, torch.cuda.Stream().cuda_stream)
    g = torch.Generator(device="cuda").manual_seed(8)
    kv = [1, 40, 700, 800]
    pages = torch.randperm(200, generator=g, device="cuda").int()
    table = pages.view(4, 50).contiguous()
    lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    base = [torch.randn((200, HKV, P, D), generator=g, device="cuda").half() for _ in range(2)]
    q, k, v = (torch.randn((4, h * D), generator=g, device="cuda").half() for h in (HQ, HKV, HKV))
    cos, sin = (torch.from_numpy(x.view(np.float16).copy()).cuda() for x in mfk.rope_tables(1e4, D, 1024))
    a, b = [x.clone() for x in base], [x.clone() for x in base]
    kw = dict(n_kv_heads=HKV, page_size=P, head_dim=D)
    plan = f.decode_plan(kv, n_heads=HQ, **kw)
    chunk = f.chunk_plan([1] * 4, kv, n_heads=HQ, **kw)
    out_a, out_b, rot = (torch.empty((4, HQ * D), dtype=torch.float16, device="cuda") for _ in range(3))
    begin = torch.arange(5, dtype=torch.int32, device="cuda")
    pos = (lens - 1).repeat(3, 1).contiguous()
    torch.cuda.synchronize()
    f.set_option(mfk.OPTION_OVERLAP_LAUNCHES, 1)
    for _ in range(3):  # again and again on the same pools: the same rows are written
        f.paged_decode(plan, mfk.paged_kv(*a, table, lens, **kw), q, out_a, n_heads=HQ, k=k, v=v, cos=cos, sin=sin, rope=True, append=True)
        f.paged_mrope_append(mfk.paged_kv(*b, table, lens, **kw), q, k, v, rot, cos, sin, pos, begin, mfk.mrope_axes([16, 24, 24]), n_heads=HQ)
        f.paged_chunk_attention(chunk, mfk.paged_kv(*b, table, lens, **kw), rot, out_b)
    f.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    mean = 4.0  # |v| of normal rows: its weighted mean stays below
    assert float((out_a.double() - out_b.double()).abs().max()) <= 2 * (2.0 ** -11 + 2.0 ** -12) * mean + 2.0 ** -10 * 4.0
    plan.close()
    chunk.close()
    f.close()


def test_pools_beyond_four_gigabytes(mfk, foundry):
    """Pages whose byte offsets pass 32 bits: append, attention and moves at the far end of 5 GB pools."""
    n_pages, page = 20500, 128
    pools = [torch.empty((n_pages, 8, page, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    far = list(range(n_pages - 9, n_pages))
    table = torch.tensor([[far[3], far[0], far[5]]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    cache = mfk.paged_kv(*pools, table, lens, n_kv_heads=8, page_size=page, head_dim=D)
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn((300, h * D), generator=g, device="cuda").half() for h in (16, 8, 8))
    cos, sin = torch.ones((1, D // 2), dtype=torch.float16, device="cuda"), torch.zeros((1, D // 2), dtype=torch.float16, device="cuda")
    begin = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    foundry.paged_mrope_append(cache, None, k, v, None, cos, sin, torch.zeros((1, 300), dtype=torch.int32, device="cuda"), begin, bytes(64), n_heads=16)
    for pool, rows in zip(pools, (k, v)):
        for t0, pg in ((0, far[3]), (128, far[0]), (256, far[5])):
            n = min(128, 300 - t0)
            foundry.synchronize()
            assert torch.equal(pool[pg, :, :n], rows.view(300, 8, D)[t0:t0 + n].transpose(0, 1))
    src, dst = np.array([far[3], far[0], far[5]], np.uint32), np.array([far[8], 1, far[7]], np.uint32)
    foundry.paged_move_pages(mfk.kv_layers([cache]), src, dst)
    table.copy_(torch.from_numpy(dst.astype(np.int32))[None])
    torch.cuda.synchronize()
    plan = foundry.chunk_plan([300], [300], n_heads=16, n_kv_heads=8, head_dim=D, page_size=page)
    out = torch.empty_like(q)
    foundry.paged_chunk_attention(plan, cache, q, out)
    foundry.synchronize()
    kk, vv = (x.view(300, 8, D).transpose(0, 1).repeat_interleave(2, 0).double() for x in (k, v))
    see = torch.ones((300, 300), dtype=torch.bool, device="cuda").tril()
    w = torch.softmax((q.view(300, 16, D).transpose(0, 1).double() @ kk.transpose(1, 2) * D ** -0.5).masked_fill(~see, -float("inf")), -1)
    want, mean = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
    got = out.view(300, 16, D).double()
    assert bool(((got - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mean + 2.0 ** -16).all())
    plan.close()
