"""Sizes past what a plan of a ragged batch can number: refused by the planner before it builds anything."""
import numpy as np
import pytest


@pytest.mark.parametrize("batch,q_len,hq,hkv,n_ctas", [
    (1, 1, 8, 2, 0xFFFFFFFF),          # one more entry than 32 bits count
    (1, 1, 8, 2, (1 << 16) + 1),
    (4, 1 << 30, 64, 1, 4),            # each sequence within the limit, the step not
    (5, 1 << 30, 64, 1, 4),            # (their sum passes 32 bits)
    (1, 1 << 30, 4096, 4096, 4),       # more items than 32 bits number
])
def test_refused(mfk, batch, q_len, hq, hkv, n_ctas):
    q, begin = np.full(batch, q_len, np.uint32), np.zeros(8, np.uint32)
    n = mfk.lib.mf_chunk_plan_build_host(q.ctypes.data, q.ctypes.data, batch, hq, hkv, 16, 0, 0, n_ctas, None, 0, begin.ctypes.data)
    assert n == 0 and not begin.any()


def test_most_ctas(mfk):
    items, begin = mfk.build_chunk_plan_host([40, 1], [300, 7000], n_heads=8, n_kv_heads=2, page_size=16, n_ctas=1 << 16)
    assert len(items) and begin[-1] == len(items)


def test_no_context_is_not_being_captured(mfk):
    assert mfk.lib.mf_is_capturing(None) == 0
