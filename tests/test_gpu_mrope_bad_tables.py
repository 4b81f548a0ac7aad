"""GPU: the multi-axis append with tables that cannot be right: what the documentation says of it, bit for bit: the call is
reported, the rows (or the pairs) that have no place are left out, and everything else is as without them."""
import numpy as np
import pytest
import torch

from test_gpu_mrope_append import Case

pytestmark = pytest.mark.gpu

KW = dict(hq=8, hkv=2, d=128, page=16, q_lens=[20, 3, 0, 1], kv_lens=[40, 30, 5, 17])


def run(mfk, f, case, table=None, lens=None, pos=None):
    """(q_rot, pools) of a call that is reported as InvalidOperation."""
    dev = [p.cuda() for p in case.pools]
    table = (case.table if table is None else table).cuda()
    lens = torch.tensor(case.kv_lens if lens is None else lens, dtype=torch.int32).cuda()
    pos = (case.pos if pos is None else pos).cuda()
    if case.bits == 16:
        cache = mfk.paged_kv(dev[0], dev[1], table, lens, n_kv_heads=case.hkv, page_size=case.page, head_dim=case.d)
    else:
        cache = mfk.paged_kv8(*dev, table, lens, n_kv_heads=case.hkv, page_size=case.page)
    out = torch.full((case.tokens, case.hq * case.d), 7.0, dtype=torch.float16, device="cuda")
    f.paged_mrope_append(cache, case.q.cuda(), case.k.cuda(), case.v.cuda(), out, case.cos.cuda(), case.sin.cuda(), pos,
                         case.begin.cuda(), case.axes, n_heads=case.hq, rope_mode=case.mode)
    with pytest.raises(mfk.MetalError) as e:
        f.synchronize()
    assert e.value.kind == "InvalidOperation"
    f.synchronize()  # reported once
    return out.cpu().numpy(), [p.cpu().numpy() for p in dev]


def same(got, want):
    q, pools = got
    want_q, want_pools = want
    assert np.array_equal(q.view(np.uint16), want_q.view(np.uint16)), "q"
    for i, (a, b) in enumerate(zip(pools, want_pools)):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), f"pool {i}"


def left_out(case, want, pages):
    """The expected result with these pages as they were."""
    q, pools = want
    for got, old in zip(pools, case.pools):
        for page in pages:
            got[page] = old[page].numpy()
    return q, pools


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("bits", [16, 8])
class TestBadTables:
    def test_a_page_outside_the_pool(self, mfk, foundry, bits, mode):
        case = Case(mfk, **KW, bits=bits, mode=mode)
        for bad in (case.n_pages, 0x7FFFFFFF, -1):
            table = case.table.clone()
            gone = int(table[0, 1])
            table[0, 1] = bad
            same(run(mfk, foundry, case, table=table), left_out(case, case.expected(), [gone]))

    def test_a_row_behind_the_table(self, mfk, foundry, bits, mode):
        case = Case(mfk, **KW, bits=bits, mode=mode)
        gone = [int(x) for x in case.table[0, 2:3]]  # rows 32 to 39 of sequence 0 have no entry in a table of two
        same(run(mfk, foundry, case, table=case.table[:, :2].contiguous()), left_out(case, case.expected(), gone))

    def test_a_sequence_shorter_than_its_tokens(self, mfk, foundry, bits, mode):
        case = Case(mfk, **KW, bits=bits, mode=mode)
        for short in (19, 0):
            gone = [int(x) for x in case.table[0] if 0 <= int(x) < case.n_pages]
            same(run(mfk, foundry, case, lens=[short, 30, 5, 17]), left_out(case, case.expected(), gone))

    def test_a_position_outside_the_tables(self, mfk, foundry, bits, mode):
        case = Case(mfk, **KW, bits=bits, mode=mode)
        good = Case(mfk, **KW, bits=bits, mode=mode)
        # a last table row that does not turn stands for the positions that have none
        good.cos, good.sin = torch.cat([good.cos, torch.ones_like(good.cos[:1])]), torch.cat([good.sin, torch.zeros_like(good.sin[:1])])
        for bad in (case.rows, 0x7FFFFFFF, -1):
            pos = case.pos.clone()
            for axis, token in ((1, 5), (0, 21), (2, 23)):
                pos[axis, token] = bad
                good.pos[axis, token] = good.rows
            same(run(mfk, foundry, case, pos=pos), good.expected())
