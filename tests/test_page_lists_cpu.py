"""Page lists that cannot be right, on the host: refused, and nothing is given back or shared."""
import ctypes as C

import numpy as np
import pytest


def test_a_page_listed_twice_is_not_given_back_twice(mfk):
    """Two hidden entries that name one page with one owner: releasing it for the first leaves nothing for the second."""
    pool = mfk.PagePool(4)
    a, b, c = (int(i) for i in pool.alloc(3))
    for ids in ([a, a, c], [a, b, a, c], [b, b, b, a]):
        with pytest.raises(mfk.MetalError) as e:
            pool.release_hidden(np.array(ids, np.uint32), 16 * len(ids), 16, 8)
        assert e.value.kind == "InvalidOperation"
        assert [pool.refcount(i) for i in (a, b, c)] == [1, 1, 1] and pool.free_count == 1
    pool.retain(np.array([a], np.uint32))  # a second owner: both entries can go
    left, n = pool.release_hidden(np.array([a, a, c], np.uint32), 48, 16, 8)
    assert n == 2 and list(left) == [mfk.FREED_PAGE, mfk.FREED_PAGE, c] and pool.refcount(a) == 0 and pool.free_count == 2
    pool.close()


@pytest.mark.parametrize("seed", range(5))
def test_random_lists(mfk, seed):
    rng = np.random.default_rng(seed)
    for _ in range(100):
        size = int(rng.integers(1, 12))
        pool = mfk.PagePool(size)
        live = pool.alloc(int(rng.integers(1, size + 1)))
        for i in live:
            for _ in range(int(rng.integers(0, 3))):
                pool.retain(np.array([i], np.uint32))
        refs = [pool.refcount(i) for i in range(size)]
        ids = rng.choice(np.concatenate([live, [mfk.FREED_PAGE]]), int(rng.integers(1, 10))).astype(np.uint32)
        hidden = [int(x) for x in ids[:-1] if x != mfk.FREED_PAGE]
        want = [r - hidden.count(i) for i, r in enumerate(refs)]
        free = pool.free_count
        if min(want) < 0:
            with pytest.raises(mfk.MetalError):
                pool.release_hidden(ids, 8 * len(ids) - 1, 8, 8)
            assert [pool.refcount(i) for i in range(size)] == refs and pool.free_count == free
        else:
            left, n = pool.release_hidden(ids, 8 * len(ids) - 1, 8, 8)
            assert n == len(hidden) and [pool.refcount(i) for i in range(size)] == want
            assert (left[:-1] == mfk.FREED_PAGE).all() and left[-1] == ids[-1]
        pool.close()
