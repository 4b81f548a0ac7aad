"""Forking, freeing behind a window and compacting pages on the host: random traces against a plain model."""
import ctypes as C

import numpy as np
import pytest

FREED = 0xFFFFFFFF


def test_fork_shares_full_pages_and_copies_the_last(mfk):
    pool = mfk.PagePool(10)
    ids = pool.alloc(3)
    child, copies = pool.fork(ids, 40, 16)  # 2 full pages and one of 8 rows
    assert list(child[:2]) == list(ids[:2]) and child[2] not in ids
    assert copies == [(int(ids[2]), int(child[2]))]
    assert [pool.refcount(int(i)) for i in ids] == [2, 2, 1] and pool.refcount(int(child[2])) == 1
    whole, copies = pool.fork(ids, 32, 16)
    assert list(whole) == list(ids[:2]) and copies == []
    assert [pool.refcount(int(i)) for i in ids] == [3, 3, 1]
    none, copies = pool.fork(ids, 0, 16)
    assert none.size == 0 and copies == []
    pool.close()


def test_fork_refusals_change_nothing(mfk):
    pool = mfk.PagePool(3)
    ids = pool.alloc(3)
    with pytest.raises(mfk.MetalError) as e:
        pool.fork(ids, 40, 16)
    assert e.value.kind == "OutOfMemory"
    pool.release(ids[2:])
    with pytest.raises(mfk.MetalError) as e:
        pool.fork(ids, 40, 16)  # the last page is not live
    assert e.value.kind == "InvalidOperation"
    assert [pool.refcount(int(i)) for i in ids] == [1, 1, 0]
    with pytest.raises(mfk.MetalError):
        pool.fork(ids[:1], 40, 16)
    with pytest.raises(mfk.MetalError):
        pool.fork(np.array([7], np.uint32), 16, 16)
    src, dst = C.c_uint32(1), C.c_uint32(1)
    assert mfk.lib.mf_page_pool_fork(pool._h, ids.ctypes.data, 16, 0, ids.ctypes.data, C.byref(src), C.byref(dst)) == 3
    assert mfk.lib.mf_page_pool_fork(None, None, 0, 16, None, C.byref(src), C.byref(dst)) == 4
    pool.close()


@pytest.mark.parametrize("page,window,sinks", [(16, 1, 0), (16, 40, 0), (16, 40, 4), (16, 40, 16), (8, 100, 17), (64, 64, 1), (64, 65, 200)])
def test_release_hidden_gives_back_what_no_later_row_sees(mfk, page, window, sinks):
    for kv_len in (0, 1, window, window + 1, window + page, 500, 513):
        n = -(-kv_len // page) + 1  # one page allocated ahead
        pool = mfk.PagePool(n + 4)
        ids = pool.alloc(n)
        left, count = pool.release_hidden(ids, kv_len, page, window, sinks)
        # the next token stands at kv_len; later ones see no older key than it does
        for i in range(n):
            seen = any(k >= kv_len or k > kv_len - window or k < sinks for k in range(i * page, (i + 1) * page))
            assert (left[i] == ids[i]) == seen and (left[i] == FREED) == (not seen), (kv_len, i)
        assert count == int((left == FREED).sum()) and pool.free_count == 4 + count
        again, more = pool.release_hidden(left, kv_len, page, window, sinks)
        assert more == 0 and np.array_equal(again, left)
        child, _ = pool.fork(left, (kv_len // page) * page, page)  # given-back entries stay so in a child
        assert np.array_equal(child, left[:kv_len // page])
        pool.close()
    pool = mfk.PagePool(2)
    ids = pool.alloc(2)
    assert pool.release_hidden(ids, 1000, 16, 0)[1] == 0
    with pytest.raises(mfk.MetalError):
        pool.release_hidden(np.array([1, 9], np.uint32), 1000, 16, 1)
    assert pool.free_count == 0
    pool.close()


def test_compact_random_traces(mfk):
    rng = np.random.default_rng(11)
    for trial in range(30):
        size = int(rng.integers(1, 60))
        pool = mfk.PagePool(size)
        cache = mfk.PrefixCache(pool, 4)
        seqs, data = [], {}
        for _ in range(40):
            op = rng.integers(0, 4)
            if op == 0 and pool.free_count:
                ids = pool.alloc(int(rng.integers(1, pool.free_count + 1)))
                for i in ids:
                    data[int(i)] = int(rng.integers(1 << 30))
                seqs.append(ids)
            elif op == 1 and seqs:
                pool.release(seqs.pop(int(rng.integers(len(seqs)))))
            elif op == 2 and seqs:
                ids = seqs[int(rng.integers(len(seqs)))]
                seqs.append(pool.fork(ids, 4 * len(ids), 4)[0])
            elif op == 3 and seqs:
                ids = seqs[int(rng.integers(len(seqs)))]
                cache.store(rng.integers(0, 3, 4 * len(ids)), ids)
        refs = {i: pool.refcount(i) for i in range(size)}
        content = [[data[int(i)] for i in s] for s in seqs]
        free = pool.free_count
        src, dst = pool.compact()
        live = size - free
        assert len(set(src)) == len(src) == len(set(dst)) and not set(src) & set(dst)
        assert all(s >= live for s in src) and all(d < live for d in dst)
        for s, d in zip(src, dst):
            assert refs[int(s)] > 0 and refs[int(d)] == 0
            data[int(d)] = data[int(s)]
            assert pool.refcount(int(d)) == refs[int(s)] and pool.refcount(int(s)) == 0
        assert pool.free_count == free and all(pool.refcount(i) > 0 for i in range(live))
        seqs = [mfk.remap_page_ids(s, src, dst) for s in seqs]
        cache.remap(src, dst)
        assert [[data[int(i)] for i in s] for s in seqs] == content
        assert pool.compact()[0].size == 0
        for s in seqs:
            pool.release(s)
        cache.close()  # releases what its entries hold under the new ids
        assert pool.free_count == size
        assert sorted(int(i) for i in pool.alloc(size)) == list(range(size))
        pool.close()


def test_compact_refusal_changes_nothing(mfk):
    pool = mfk.PagePool(6)
    ids = pool.alloc(6)
    pool.release(ids[[0, 1, 2]])
    n = C.c_uint32(0)
    two = np.zeros(2, np.uint32)
    assert mfk.lib.mf_page_pool_compact(pool._h, two.ctypes.data, two.ctypes.data, 2, C.byref(n)) == 6 and n.value == 3
    assert [pool.refcount(i) for i in range(6)] == [0, 0, 0, 1, 1, 1]
    assert mfk.lib.mf_page_pool_compact(None, None, None, 0, C.byref(n)) == 4
    src, dst = pool.compact()
    assert sorted(map(int, src)) == [3, 4, 5] and sorted(map(int, dst)) == [0, 1, 2]
    assert np.array_equal(mfk.remap_page_ids([3, FREED, 0, 5], src, dst)[[1, 2]], [FREED, 0])
    pool.close()


def test_null_contexts_are_refused(mfk):
    out = C.c_void_p()
    one = np.ones(1, np.uint32)
    p = one.ctypes.data
    assert mfk.lib.mf_chunk_plan_create(None, p, p, 1, 1, 1, 64, 16, 0, 0, 0, C.byref(out)) == 4
    assert mfk.lib.mf_chunk_plan_update(None, None, p, p) == 4
    assert mfk.lib.mf_chunk_plan_tokens(None) == 0
    mfk.lib.mf_chunk_plan_destroy(None, None)
    assert mfk.lib.mf_paged_chunk_attention(None, None, None, None) == 4
    assert mfk.lib.mf_paged_mrope_append(None, None, None) == 4
    assert mfk.lib.mf_paged_kv8_mrope_append(None, None, None) == 4
    assert mfk.lib.mf_paged_move_pages(None, None, 0, None, None, 0) == 4
    assert mfk.lib.mf_paged_kv8_move_pages(None, None, 0, None, None, 0) == 4
    assert mfk.lib.mf_remap_page_ids(None, 1, p, p, 1) == 4
    assert mfk.lib.mf_prefix_cache_remap(None, p, p, 1) == 4
