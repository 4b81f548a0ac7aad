"""GPU: pages moved in all layers at once, f16 and 8-bit caches, bit for bit against indexing."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(mfk, *, layers, pool, hkv, page, d=128, bits=16, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (layers, pool, hkv, page, d)
    if bits == 16:
        pools = [torch.randn(shape, generator=g, device="cuda").half() for _ in range(2)]
    else:
        pools = [torch.randint(0, 255, shape, generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)] + \
                [torch.rand(shape[:4], generator=g, device="cuda") for _ in range(2)]
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    if bits == 16:
        caches = [mfk.paged_kv(pools[0][i], pools[1][i], table, table, n_kv_heads=hkv, page_size=page, head_dim=d) for i in range(layers)]
    else:
        caches = [mfk.paged_kv8(*[p[i] for p in pools], table, table, n_kv_heads=hkv, page_size=page) for i in range(layers)]
    return pools, mfk.kv_layers(caches)


@pytest.mark.parametrize("kw,n,fork", [
    (dict(layers=1, pool=4, hkv=1, page=16, d=64), 1, False),
    (dict(layers=3, pool=50, hkv=2, page=16), 20, False),
    (dict(layers=3, pool=50, hkv=2, page=16), 20, True),
    (dict(layers=36, pool=20, hkv=2, page=16), 8, True),
    (dict(layers=70, pool=12, hkv=1, page=8, d=64), 5, False),
    (dict(layers=2, pool=9001, hkv=1, page=8, d=64), 4500, False),
    (dict(layers=2, pool=30, hkv=8, page=128), 11, False),
    (dict(layers=1, pool=4, hkv=1, page=16, bits=8), 1, False),
    (dict(layers=5, pool=60, hkv=2, page=32, bits=8), 25, True),
    (dict(layers=40, pool=700, hkv=1, page=16, bits=8), 301, False),
], ids=lambda x: None)
def test_bits(mfk, foundry, kw, n, fork):
    pools, layers = make(mfk, **kw)
    order = np.random.default_rng(n).permutation(kw["pool"]).astype(np.uint32)
    src, dst = order[:n], order[n:2 * n]
    if fork:
        src = src[np.arange(n) // 3 * 3]
    want = [p.clone() for p in pools]
    s, d = torch.from_numpy(src.astype(np.int64)).cuda(), torch.from_numpy(dst.astype(np.int64)).cuda()
    for p in want:
        p[:, d] = p[:, s]
    foundry.paged_move_pages(layers, src, dst)
    foundry.synchronize()
    for a, b in zip(pools, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    foundry.paged_move_pages(layers, src[:0], dst[:0])
    foundry.synchronize()


def test_captured_launch_keeps_its_pairs(mfk):
    stream = torch.cuda.Stream()
    f = mfk.Foundry(0, stream.cuda_stream)
    pools, layers = make(mfk, layers=2, pool=40, hkv=2, page=16)
    src, dst = np.array([3, 5, 7], np.uint32), np.array([30, 31, 32], np.uint32)
    torch.cuda.synchronize()
    f.paged_move_pages(layers, src, dst)
    f.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        f.paged_move_pages(layers, src, dst)
    src[:], dst[:] = 0, 39  # the host arrays are the caller's again
    for p in pools:
        p[:, 30:33] = 0
    want = [p.clone() for p in pools]
    for p in want:
        p[:, 30:33] = p[:, [3, 5, 7]]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    f.synchronize()
    for a, b in zip(pools, want):
        assert torch.equal(a, b)
    del graph
    f.close()


def test_refusals(mfk, foundry):
    pools, layers = make(mfk, layers=2, pool=10, hkv=2, page=16)
    keep = [p.clone() for p in pools]

    def call(kind, src, dst, arr=layers):
        with pytest.raises(mfk.MetalError) as e:
            foundry.paged_move_pages(arr, np.array(src, np.uint32), np.array(dst, np.uint32))
        assert e.value.kind == kind, e.value

    call("InvalidOperation", [0, 1], [5, 5])       # written twice
    call("InvalidOperation", [0, 5], [5, 6])       # read and written
    call("InvalidOperation", [3], [3])
    call("InvalidOperation", [10], [1])
    call("InvalidOperation", [0, 1], [2, 0xFFFFFFFF])
    call("InvalidShape", [0, 1], [2])
    odd = mfk.kv_layers([layers[0], layers[1]])
    odd[1].n_pages = 9
    call("InvalidShape", [0], [1], odd)
    odd[1].n_pages, odd[1].k_pool = 10, None
    call("InputNotFound", [0], [1], odd)
    odd[1].k_pool = layers[1].k_pool + 8
    call("InvalidShape", [0], [1], odd)
    foundry.synchronize()
    for a, b in zip(pools, keep):
        assert torch.equal(a, b)
