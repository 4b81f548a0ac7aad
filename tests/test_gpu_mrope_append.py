"""GPU: append of ragged batches with rotary positions on several axes, f16 and 8-bit caches.  Every result is one
rounding of an f32 expression of f16 operands whose products are exact, so it is compared bit for bit with the
same expression in numpy, and equal axes must give what the one-axis append gives."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, mfk, *, hq, hkv, d, page, q_lens, kv_lens, bits=16, mode=0, axes=None, n_axes=3, seed=3, extra=0):
        self.hq, self.hkv, self.d, self.page, self.q_lens, self.kv_lens, self.bits, self.mode = hq, hkv, d, page, q_lens, kv_lens, bits, mode
        g = torch.Generator().manual_seed(seed)
        t = sum(q_lens)
        self.tokens = t
        rnd = lambda *s: torch.randn(s, generator=g).half()  # noqa: E731
        self.q, self.k, self.v = rnd(t, hq * d + extra), rnd(t, hkv * d + extra), rnd(t, hkv * d + extra)
        need = [-(-n // page) for n in kv_lens]
        self.n_pages = sum(need) + 2
        order = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(kv_lens), max(need + [1])), 0x7FFFFFF0, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.rows = 600
        self.pos = torch.randint(0, self.rows, (n_axes, max(t, 1)), generator=g, dtype=torch.int32)[:, :t]
        cos, sin = mfk.rope_tables(1e4, d, self.rows)
        self.cos, self.sin = (torch.from_numpy(x.view(np.float16).copy()) for x in (cos, sin))
        self.begin = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32)
        self.axes = axes if axes is not None else bytes(np.random.default_rng(seed).integers(0, n_axes, d // 2, np.uint8))
        shape = (self.n_pages, hkv, page, d)
        if bits == 16:
            self.pools = [rnd(*shape), rnd(*shape)]
        else:
            self.pools = [torch.randint(0, 120, shape, generator=g, dtype=torch.uint8) for _ in range(2)] + \
                         [torch.rand(shape[:3], generator=g) for _ in range(2)]

    def turned(self, x, heads):
        x = x[:, :heads * self.d].float().numpy().reshape(-1, heads, self.d)
        half = self.d // 2
        rows = self.pos.numpy()[np.frombuffer(self.axes, np.uint8)].T  # [tokens, half]
        c, s = (tab.numpy()[rows, np.arange(half)].astype(np.float32)[:, None] for tab in (self.cos, self.sin))
        a, b = (x[..., :half], x[..., half:]) if self.mode == 0 else (x[..., 0::2], x[..., 1::2])
        y = np.empty_like(x)
        first, second = a * c - b * s, b * c + a * s
        if self.mode == 0:
            y[..., :half], y[..., half:] = first, second
        else:
            y[..., 0::2], y[..., 1::2] = first, second
        return y.astype(np.float16)

    def expected(self):
        q, k = self.turned(self.q, self.hq), self.turned(self.k, self.hkv)
        v = self.v[:, :self.hkv * self.d].numpy().reshape(-1, self.hkv, self.d)
        pools = [p.numpy().copy() for p in self.pools]
        t = 0
        for b, n in enumerate(self.q_lens):
            for i in range(n):
                row = self.kv_lens[b] - n + i
                page, at = int(self.table[b, row // self.page]), row % self.page
                if self.bits == 16:
                    pools[0][page, :, at], pools[1][page, :, at] = k[t], v[t]
                else:
                    for x, which in ((k[t], 0), (v[t], 1)):
                        x = x.astype(np.float32)
                        top = np.abs(x).max(-1)
                        scale = np.where(top > 0, top / np.float32(448), np.float32(1)).astype(np.float32)
                        by = torch.from_numpy(x / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
                        pools[2 + which][page, :, at] = scale
                        if which == 0:
                            pools[0][page, :, at] = by
                        else:
                            pools[1].reshape(-1, self.hkv, self.page // 16, self.d, 16)[page, :, at // 16, :, at % 16] = by
                t += 1
        return q.reshape(self.tokens, -1), pools

    def run(self, mfk, f, rotate_q=True, into=None):
        dev = [p.cuda() for p in self.pools] if into is None else into
        table, lens = self.table.cuda(), torch.tensor(self.kv_lens, dtype=torch.int32).cuda()
        if self.bits == 16:
            cache = mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=self.hkv, page_size=self.page, head_dim=self.d)
        else:
            cache = mfk.paged_kv8(*dev, table, lens, n_kv_heads=self.hkv, page_size=self.page)
        w = self.hq * self.d
        out = torch.full((self.tokens, w + 8), 7.0, dtype=torch.float16, device="cuda") if rotate_q else None
        q, k, v = (x.cuda() for x in (self.q, self.k, self.v))
        f.paged_mrope_append(cache, q[:, :w] if rotate_q else None, k[:, :self.hkv * self.d], v[:, :self.hkv * self.d],
                             out[:, :w] if rotate_q else None, self.cos.cuda(), self.sin.cuda(), self.pos.cuda(), self.begin.cuda(),
                             self.axes, n_heads=self.hq, rope_mode=self.mode)
        f.synchronize()
        if rotate_q:
            assert bool((out[:, w:] == 7.0).all())
            out = out[:, :w].cpu().numpy()
        return out, [p.cpu().numpy() for p in dev]


CASES = [
    dict(hq=16, hkv=2, d=128, page=16, q_lens=[1], kv_lens=[1]),
    dict(hq=16, hkv=2, d=128, page=16, q_lens=[1] * 33, kv_lens=list(range(1, 34))),
    dict(hq=16, hkv=2, d=128, page=16, q_lens=[3, 0, 70, 1], kv_lens=[17, 9, 70, 400]),
    dict(hq=14, hkv=2, d=64, page=32, q_lens=[3, 0, 70, 1], kv_lens=[17, 9, 70, 400]),
    dict(hq=4, hkv=4, d=64, page=64, q_lens=[129, 64], kv_lens=[129, 65], mode=1),
    dict(hq=8, hkv=2, d=128, page=64, q_lens=[129, 64], kv_lens=[129, 65], mode=1, extra=24),
    dict(hq=7, hkv=1, d=128, page=8, q_lens=[5, 20], kv_lens=[9, 20], extra=8),
    dict(hq=16, hkv=2, d=128, page=16, q_lens=[3, 0, 70, 1], kv_lens=[17, 9, 70, 400], bits=8),
    dict(hq=8, hkv=8, d=128, page=64, q_lens=[1, 1, 131], kv_lens=[64, 65, 300], bits=8, mode=1, extra=16),
    dict(hq=5, hkv=1, d=128, page=32, q_lens=[40], kv_lens=[40], bits=8, n_axes=4),
    dict(hq=8, hkv=2, d=128, page=16, q_lens=[33], kv_lens=[50], n_axes=1),
]


@pytest.mark.parametrize("kw", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_bits(mfk, foundry, kw):
    case = Case(mfk, **kw)
    q, pools = case.expected()
    got, dev = case.run(mfk, foundry)
    assert np.array_equal(got.view(np.uint16), q.view(np.uint16))
    for a, b in zip(dev, pools):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    none, dev = case.run(mfk, foundry, rotate_q=False)
    assert none is None
    for a, b in zip(dev, pools):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("bits", [16, 8])
def test_equal_axes_are_the_one_axis_append(mfk, foundry, bits):
    case = Case(mfk, hq=16, hkv=2, d=128, page=16, q_lens=[37], kv_lens=[90], bits=bits, mode=1)
    case.pos[:] = torch.arange(53, 90, dtype=torch.int32)
    got, dev = case.run(mfk, foundry)
    want = [p.cuda() for p in case.pools]
    table, lens = case.table.cuda(), torch.tensor([90], dtype=torch.int32).cuda()
    q_rot = torch.empty((16, 37, 128), dtype=torch.float16, device="cuda")
    args = [x.cuda() for x in (case.q, case.k, case.v)] + [q_rot, case.cos.cuda(), case.sin.cuda()]
    kw = dict(n_heads=16, rope_mode=1, seq=0, position_offset=53, seq_len=37)
    if bits == 16:
        foundry.paged_kv_append(mfk.paged_kv(*want, table, lens, n_kv_heads=2, page_size=16, head_dim=128), *args, **kw)
    else:
        foundry.paged_kv8_append(mfk.paged_kv8(*want, table, lens, n_kv_heads=2, page_size=16), *args, **kw)
    foundry.synchronize()
    assert np.array_equal(got.view(np.uint16), q_rot.transpose(0, 1).reshape(37, -1).cpu().numpy().view(np.uint16))
    for a, b in zip(dev, want):
        assert np.array_equal(a.view(np.uint8), b.cpu().numpy().view(np.uint8))


def test_axes_helper(mfk):
    assert mfk.mrope_axes([2, 3, 3]) == bytes([0, 0, 1, 1, 1, 2, 2, 2])
    assert mfk.mrope_axes([4, 2, 2], interleaved=True) == bytes([0, 1, 2, 0, 1, 2, 0, 0])
    for sections in ([16, 24, 24], [8, 12, 12], [5, 6, 5]):
        axes = mfk.mrope_axes(sections)
        assert [axes.count(a) for a in range(3)] == sections
        with pytest.raises(mfk.MetalError):  # the first axis takes what the others leave: it cannot have less
            mfk.mrope_axes(sections, interleaved=True)
    for sections in ([24, 20, 20], [12, 10, 10], [22, 21, 21]):
        axes = mfk.mrope_axes(sections, interleaved=True)
        assert [axes.count(a) for a in range(3)] == sections


@pytest.mark.parametrize("bits", [16, 8])
def test_bad_tables_skip_their_rows(mfk, foundry, bits):
    """A page id outside the pool, a sequence shorter than its new tokens, a position outside the tables: reported, and
    nothing but those rows is missing."""
    def report(case, change):
        change(case)
        with pytest.raises(mfk.MetalError) as e:
            case.run(mfk, foundry)
        assert e.value.kind == "InvalidOperation"

    kw = dict(hq=8, hkv=2, d=128, page=16, q_lens=[20, 3], kv_lens=[40, 30], bits=bits)
    case = Case(mfk, **kw)
    dev = [p.cuda() for p in case.pools]
    want = case.expected()[1]
    gone = int(case.table[0, 1])
    keep = case.pools[0][gone].clone()
    report(case, lambda c: c.table.__setitem__((0, 1), c.n_pages))
    with pytest.raises(mfk.MetalError):
        case.run(mfk, foundry, into=dev)
    assert np.array_equal(dev[0][gone].cpu().numpy().view(np.uint8), keep.numpy().view(np.uint8))
    other = int(case.table[1, 1])
    assert np.array_equal(dev[0][other].cpu().numpy().view(np.uint8), want[0][other].view(np.uint8))
    short = Case(mfk, **(kw | dict(kv_lens=[40, 30])))
    short.kv_lens = [19, 30]
    report(short, lambda c: None)
    report(Case(mfk, **kw), lambda c: c.pos.__setitem__((1, 5), c.rows))
    foundry.synchronize()


def test_refusals(mfk, foundry):
    case = Case(mfk, hq=8, hkv=2, d=128, page=16, q_lens=[4], kv_lens=[40])
    dev = [p.cuda() for p in case.pools]
    table, lens = case.table.cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    good = dict(q=case.q.cuda(), k=case.k.cuda(), v=case.v.cuda(), q_rot=torch.zeros((4, 1024), dtype=torch.float16, device="cuda"),
                cos=case.cos.cuda(), sin=case.sin.cuda(), positions=case.pos.cuda(), q_begin=case.begin.cuda(), axes=case.axes)

    def call(kind, n_heads=8, rope_mode=0, cache=None, **kw):
        cache = cache or mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=2, page_size=16, head_dim=128)
        with pytest.raises(mfk.MetalError) as e:
            foundry.paged_mrope_append(cache, *(good | kw).values(), n_heads=n_heads, rope_mode=rope_mode)
        assert e.value.kind == kind, e.value

    call("InvalidOperation", rope_mode=2)
    call("InvalidOperation", axes=bytes([3] * 64))
    call("InvalidShape", axes=bytes(63))
    call("InvalidShape", n_heads=7)
    call("InvalidShape", positions=case.pos.cuda()[:, :3])
    call("InvalidShape", q_begin=case.begin.cuda()[:1])
    call("InvalidShape", cos=case.cos.cuda()[:, :32])
    call("InvalidShape", k=case.k.cuda()[:, 1:])
    call("InputNotFound", q=None)
    odd = torch.zeros((4, 1024 + 4), dtype=torch.float16, device="cuda")
    call("InvalidShape", q=odd[:, :1024])
    call("InvalidShape", q=torch.zeros(4 * 1024 + 4, dtype=torch.float16, device="cuda")[4:].view(4, 1024))
    five = torch.zeros((5, 4), dtype=torch.int32, device="cuda")
    call("InvalidOperation", positions=five, axes=bytes([4] * 64))
    cache = mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=2, page_size=16, head_dim=128)
    cache.k_pool = None
    call("InputNotFound", cache=cache)
    k8 = Case(mfk, hq=8, hkv=2, d=128, page=16, q_lens=[4], kv_lens=[40], bits=8)
    cache = mfk.paged_kv8(*[p.cuda() for p in k8.pools], table, lens, n_kv_heads=2, page_size=16)
    cache.page_size = 8
    call("OperationNotSupported", cache=cache)
    cache.page_size, cache.k_scales = 16, None
    call("InputNotFound", cache=cache)
    assert not bool(good["q_rot"].any())
    empty = {k: (x[:0] if k in ("q", "k", "v", "q_rot") else x[:, :0] if k == "positions" else x) for k, x in good.items()}
    empty["q_begin"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    before = dev[0].clone()
    foundry.paged_mrope_append(mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=2, page_size=16, head_dim=128), *empty.values(), n_heads=8)
    foundry.synchronize()
    assert torch.equal(before, dev[0])


def test_other_types_and_memories_are_refused(mfk, foundry):
    case = Case(mfk, hq=8, hkv=2, d=128, page=16, q_lens=[4], kv_lens=[40])
    dev = [p.cuda() for p in case.pools]
    before = dev[0].clone()
    table, lens = case.table.cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    cache = mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=2, page_size=16, head_dim=128)
    good = dict(q=case.q.cuda(), k=case.k.cuda(), v=case.v.cuda(), q_rot=torch.zeros((4, 1024), dtype=torch.float16, device="cuda"),
                cos=case.cos.cuda(), sin=case.sin.cuda(), positions=case.pos.cuda(), q_begin=case.begin.cuda())
    for name, x in good.items():
        for bad in (x.cpu(), x.bfloat16() if x.dtype == torch.float16 else x.float()):
            with pytest.raises(mfk.MetalError) as e:
                foundry.paged_mrope_append(cache, *(good | {name: bad}).values(), case.axes, n_heads=8)
            assert e.value.kind == "InvalidShape", name
    foundry.synchronize()
    assert torch.equal(before, dev[0]) and not bool(good["q_rot"].any())


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_in_place_on_another_stream(mfk, bits):
    """q may be turned where it is; a captured call reads lengths and positions anew at each replay."""
    stream = torch.cuda.Stream()
    f = mfk.Foundry(0, stream.cuda_stream)
    case = Case(mfk, hq=8, hkv=2, d=128, page=16, q_lens=[20, 3], kv_lens=[40, 30], bits=bits)
    dev, table = [p.cuda() for p in case.pools], case.table.cuda()
    lens, pos, q = torch.tensor(case.kv_lens, dtype=torch.int32).cuda(), case.pos.cuda(), case.q.cuda()
    k, v, cos, sin, begin = case.k.cuda(), case.v.cuda(), case.cos.cuda(), case.sin.cuda(), case.begin.cuda()
    if bits == 16:
        cache = mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=2, page_size=16, head_dim=128)
    else:
        cache = mfk.paged_kv8(*dev, table, lens, n_kv_heads=2, page_size=16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        f.paged_mrope_append(cache, q, k, v, q, cos, sin, pos, begin, case.axes, n_heads=8)
    for kv_lens, shift in (([40, 30], 0), ([33, 17], 5)):
        case.kv_lens, case.pos = kv_lens, case.pos.add(shift) % case.rows
        case.pools = [p.cpu().clone() for p in dev]
        want_q, want = case.expected()
        lens.copy_(torch.tensor(kv_lens, dtype=torch.int32))
        pos.copy_(case.pos)
        q.copy_(case.q)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        f.synchronize()
        assert np.array_equal(q.cpu().numpy().view(np.uint16), want_q.view(np.uint16))
        for a, b in zip(dev, want):
            assert np.array_equal(a.cpu().numpy().view(np.uint8), b.view(np.uint8))
    del graph
    f.close()


def test_rows_that_are_not_finite_in_the_8_bit_cache(mfk, foundry):
    """Infinities and NaN are quantised as the one-axis append does it, and stay in their row."""
    case = Case(mfk, hq=4, hkv=2, d=128, page=16, q_lens=[37], kv_lens=[90], bits=8, mode=1)
    case.pos[:] = torch.arange(53, 90, dtype=torch.int32)
    for t, (x, value) in enumerate(((case.k, float("inf")), (case.k, float("nan")), (case.v, -float("inf")), (case.v, float("nan")))):
        x[5 * t + 1, 7] = value
    _, dev = case.run(mfk, foundry)
    want = [p.cuda() for p in case.pools]
    table, lens = case.table.cuda(), torch.tensor([90], dtype=torch.int32).cuda()
    args = [x.cuda() for x in (case.q, case.k, case.v)] + [torch.empty((4, 37, 128), dtype=torch.float16, device="cuda"),
                                                         case.cos.cuda(), case.sin.cuda()]
    foundry.paged_kv8_append(mfk.paged_kv8(*want, table, lens, n_kv_heads=2, page_size=16), *args, n_heads=4, rope_mode=1, seq=0,
                             position_offset=53, seq_len=37)
    foundry.synchronize()
    for a, b in zip(dev, want):
        assert np.array_equal(a.view(np.uint8), b.cpu().numpy().view(np.uint8))
