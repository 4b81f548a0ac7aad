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
