"""GPU: values and keys that are not finite in the attention of ragged batches: they show in the rows that see them, in their
dims, and nowhere else, and a call with them takes about as long as one without."""
import pytest
import torch

from chunkcases import ChunkCase

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def put(case, b, key, dims, value, pool):
    """value into dims of row `key` of sequence b, all kv heads, where the row is in the cache at all."""
    page = int(case.table[b, key // case.page])
    if 0 <= page < case.n_pages:
        pool[page, :, key % case.page, dims] = value


def shown(case, poison):
    """[tokens, 1, d]: the sum of the values that are not finite over the keys that each row sees (a visible key has a
    positive weight, so this is what the row's output is in these dims), 0 elsewhere."""
    add = torch.zeros((case.tokens, 1, case.d), dtype=torch.float64, device="cuda")
    starts = [sum(case.q_lens[:b]) for b in range(len(case.q_lens))]
    for b, key, dims, value in poison:
        if case.q_lens[b]:
            rows = starts[b] + torch.nonzero(case.visible(b)[:, key])[:, 0]
            for d in dims:
                add[rows, 0, d] += value
    return add


def run(mfk, f, case, plan=None):
    plan = plan or case.plan(f)
    out = torch.empty_like(case.q)
    f.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    f.synchronize()
    return out[:case.tokens].view(case.tokens, case.hq, case.d).double()


def check(got, case, poison):
    """poison: (sequence, key, dims, value); the same rows of the definition's values count as 0 for its finite part."""
    for b, key, dims, _ in poison:
        case.vc[b][:, key, dims] = 0
    want, tol = case.expected()
    add = shown(case, poison).expand_as(want)
    plain = torch.isfinite(add)
    assert bool(((got - want).abs() <= tol)[plain].all()), "a value reached an output that it does not belong to"
    assert bool((torch.isnan(got) == torch.isnan(add)).all()), "NaN"
    assert bool((got[~plain].nan_to_num(0, 1, -1) == add[~plain].nan_to_num(0, 1, -1)).all()), "infinities"


CASES = {
    "prompt": (8, 2, 128, 16, [300], [900], 0, 0),
    "prompt_from_nothing": (8, 8, 128, 32, [257], [257], 0, 0),
    "prompt_d64_group7": (14, 2, 64, 16, [200, 131], [500, 131], 0, 0),
    "verify": (16, 2, 128, 16, [5, 3, 8, 1], [700, 3, 8, 4097], 0, 0),
    "group1": (4, 4, 128, 16, [270, 1], [500, 77], 0, 0),
    "group64": (64, 1, 128, 16, [5, 1], [300, 77], 0, 0),
    "before_the_start": (8, 2, 128, 16, [6, 130, 40], [4, 100, 20], 0, 0),
    "window_prompt": (14, 2, 64, 32, [700, 1], [2000, 999], 100, 0),
    "window_prompt_sinks": (16, 2, 128, 16, [300, 5], [2000, 999], 200, 4),
    "window_small": (8, 2, 128, 64, [100, 9], [400, 90], 3, 0),
    "window_many_sinks": (8, 2, 128, 16, [100, 1, 9], [900, 400, 190], 33, 150),
    "window_sinks_inside_page": (8, 2, 128, 64, [1, 33], [1000, 1000], 65, 70),
    "many_items": (16, 2, 128, 16, [40] * 120, [300 + 5 * i for i in range(120)], 0, 0),
    "long_cut_units": (8, 1, 128, 16, [20, 3], [9000, 5000], 0, 0),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_values_show_where_they_are_seen(mfk, foundry, name, seed):
    hq, hkv, d, page, ql, kl, window, sinks = CASES[name]
    case = ChunkCase(hq=hq, hkv=hkv, d=d, page=page, q_lens=ql, kv_lens=kl, window=window, sinks=sinks, seed=seed + 5)
    g = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    poison = []
    for b in range(min(len(ql), 10)):
        n, m = kl[b], ql[b]
        # among the new tokens, at the window's edge, anywhere
        spots = [max(0, n - 1 - pick(0, max(m, 1))) for _ in range(3)] + [pick(0, n)]
        if window:
            spots += [max(0, n - window - pick(0, max(m, 1))) for _ in range(2)] + ([pick(0, min(sinks, n))] if sinks else [])
        for key in set(spots):
            if m and bool(case.visible(b)[:, key].any()):
                dims = sorted({pick(0, d) for _ in range(pick(1, 5))}) if pick(0, 4) else list(range(d))
                poison.append((b, key, dims, [NAN, INF, -INF][pick(0, 3)]))
    for b, key, dims, value in poison:
        put(case, b, key, dims, value, case.v)
    plan = case.plan(foundry)
    got = run(mfk, foundry, case, plan)
    again = run(mfk, foundry, case, plan)
    assert torch.equal(got.nan_to_num(7, 8, 9), again.nan_to_num(7, 8, 9)), "two calls on the same inputs differ"
    check(got, case, poison)
    plan.close()


def timed(f, stream, call):
    best = INF
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(stream)
        call()
        b.record(stream)
        f.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,key", [
    ([2048, 2048], [16384, 16000], 16, 2, 0),          # the first key of a long prompt: every row sees it
    ([2048, 2048], [16384, 16000], 16, 2, 15000),      # a key of the chunk
    ([5] * 4, [131072] * 4, 16, 2, 0),                 # drafted tokens behind 131 072 keys
    ([5] * 4, [131072] * 4, 16, 2, 131069),            # ... the value of one of them: two rows see it, three do not
    ([5] * 40, [8000] * 40, 64, 8, 7997),
    ([1] * 8, [131072] * 8, 8, 1, 5),
])
def test_a_value_that_is_not_finite_costs_no_time(mfk, foundry, value, q_lens, kv_lens, hq, hkv, key):
    """Long contexts, several items per CTA: the call ends without a status and takes no more than twice the time."""
    case = ChunkCase(hq=hq, hkv=hkv, d=128, page=64, q_lens=q_lens, kv_lens=kv_lens)
    plan, cache, out = case.plan(foundry), case.cache(mfk), torch.empty_like(case.q)
    stream = torch.cuda.current_stream()
    call = lambda: foundry.paged_chunk_attention(plan, cache, case.q, out)  # noqa: E731
    call()
    clean = timed(foundry, stream, call)
    want = out.clone().view(case.tokens, hq, 128)
    for b in range(len(q_lens)):
        put(case, b, key, [3], value, case.v)
    bad = timed(foundry, stream, call)
    got = out.view(case.tokens, hq, 128)
    rows = torch.cat([case.visible(b)[:, key] for b in range(len(q_lens))])
    assert bool((torch.isnan(got) if value != value else got == value)[rows][:, :, 3].all())
    keep = torch.ones(128, dtype=torch.bool, device="cuda")
    keep[3] = False
    assert torch.equal(got[:, :, keep], want[:, :, keep])
    if not bool(rows.all()):
        # the rows that do not see it: as without it, but for a value of the key's own dim that counts as 0 for them anyway
        assert torch.equal(got[~rows], want[~rows])
    assert bad <= 2 * clean + 0.05, f"{bad:.3f} ms with it, {clean:.3f} ms without"
    plan.close()


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,d,window,sinks", [
    ([1], [1], 8, 2, 128, 0, 0),
    ([1, 1, 1], [1, 700, 5000], 8, 1, 64, 1, 0),
    ([40, 7], [40, 300], 16, 2, 128, 0, 0),
    ([200, 3], [900, 3], 14, 2, 64, 40, 2),
    ([9], [4], 8, 2, 128, 0, 0),
    ([1, 5], [20000, 30000], 8, 1, 128, 0, 0),
])
def test_keys_show_as_the_formula_has_them(mfk, foundry, value, q_lens, kv_lens, hq, hkv, d, window, sinks):
    """A key that is not finite makes its score +inf, -inf or NaN: a NaN in the rows that see it, but for a score of -inf beside
    finite ones, whose weight is 0; a row that sees nothing but -inf is not a number either."""
    case = ChunkCase(hq=hq, hkv=hkv, d=d, page=16, q_lens=q_lens, kv_lens=kv_lens, window=window, sinks=sinks)
    for b, n in enumerate(kv_lens):
        for key in {n - 1, n // 2, 0}:
            case.kc[b][:, key, 1] = value
            put(case, b, key, [1], value, case.k)
    got = run(mfk, foundry, case)
    t = 0
    for b, nq in enumerate(q_lens):
        see = case.visible(b)
        for h in range(hq):
            k, v = case.kc[b][h // (hq // hkv)].double(), case.vc[b][h // (hq // hkv)].double()
            s = (case.q[t:t + nq, h * d:(h + 1) * d].double() @ k.T * d ** -0.5).masked_fill(~see, -INF)
            w = torch.softmax(s, -1)
            w[~see.any(1)] = 0
            want, mean = w @ v, w @ v.abs()
            few = see.sum(1, keepdim=True) * 2.0 ** -32 * float(v.abs().max())
            tol = 2.0 ** -25 + 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mean + few
            off = (got[t:t + nq, h] - want).abs()
            assert bool((torch.isnan(got[t:t + nq, h]) == torch.isnan(want)).all()), (b, h)
            assert bool(((off <= tol) | torch.isnan(want)).all()), (b, h)
        t += nq


def test_large_scales(mfk, foundry):
    """With large scales the key of the largest score has all the weight; a scale whose scores would leave the range is refused."""
    case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=[1, 40], kv_lens=[50, 300])
    plan, out = case.plan(foundry), torch.empty_like(case.q)
    t = 0
    best = torch.zeros((case.tokens, 8, 128), dtype=torch.float16, device="cuda")
    clear = torch.zeros((case.tokens, 8, 1), dtype=torch.bool, device="cuda")
    for b, nq in enumerate(case.q_lens):
        for h in range(8):
            s = (case.q[t:t + nq, h * 128:(h + 1) * 128].double() @ case.kc[b][h // 4].double().T).masked_fill(~case.visible(b), -INF)
            top = s.topk(2, 1).values
            clear[t:t + nq, h, 0] = top[:, 0] - top[:, 1] > 2.0 ** -10  # (f32 products of up to 50: off by less than 2^-14)
            best[t:t + nq, h] = case.vc[b][h // 4][s.argmax(1)]
        t += nq
    assert float(clear.float().mean()) > 0.95
    for scale in (1e6, 1e12, 1e18):
        foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out, scale=scale)
        foundry.synchronize()
        got = out.view_as(best)
        assert torch.equal(got[clear.expand_as(got)], best[clear.expand_as(got)])
    out.fill_(7.0)
    for scale in (2e18, 1e30, 2e38):
        with pytest.raises(mfk.MetalError) as e:
            foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out, scale=scale)
        assert e.value.kind == "InvalidOperation"
    foundry.synchronize()
    assert bool((out == 7.0).all())
    plan.close()


@pytest.mark.parametrize("size", [1.0, 250.0, 4000.0, 65504.0])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [4000]), ([60, 1], [300, 90])])
def test_large_scores(mfk, foundry, size, q_lens, kv_lens):
    """Equal scores up to those of f16's largest values, of either sign: every visible key has the same weight."""
    for sign in (1.0, -1.0):
        case = ChunkCase(hq=8, hkv=2, d=128, page=16, q_lens=q_lens, kv_lens=kv_lens)
        case.q.fill_(size)
        case.k[torch.isfinite(case.k)] = sign * size
        got = run(mfk, foundry, case)
        t = 0
        for b, nq in enumerate(q_lens):
            see = case.visible(b).double()
            for h in range(8):
                v = case.vc[b][h // 4].double()
                want, mean = see @ v / see.sum(1, keepdim=True), see @ v.abs() / see.sum(1, keepdim=True)
                tol = 2.0 ** -25 + 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mean
                assert bool(((got[t:t + nq, h] - want).abs() <= tol).all())
            t += nq


@pytest.mark.parametrize("value", [65504.0, -65504.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len,n,page", [(1, 201, 16), (1, 6001, 64), (30, 230, 16), (30, 6001, 128)])
def test_means_stay_in_the_range(mfk, foundry, value, d, q_len, n, page):
    """Weights that all round up (0.6 of a step of f16 above one half) carry a mean of f16's largest values past it."""
    case = ChunkCase(hq=8, hkv=1, d=d, page=page, q_lens=[q_len], kv_lens=[n])
    case.q.zero_()
    case.q.view(-1, 8, d)[..., :2] = 1.0
    score = float(torch.log(torch.tensor(0.5 * (1 + 0.6 * 2.0 ** -10), dtype=torch.float64)))
    first = float(torch.tensor(score).half())
    for page_id in case.table[0].tolist():
        case.k[page_id].zero_()
        case.k[page_id, :, :, 0], case.k[page_id, :, :, 1] = first, score - first
        case.v[page_id] = value
    case.k[int(case.table[0, 0]), :, 0, :2] = 0  # the one with weight 1
    out = torch.empty_like(case.q)
    plan = case.plan(foundry)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out, scale=1.0)
    foundry.synchronize()
    # the weights are off by 2^-11 of each, f32 sums by 2^-12
    assert bool(torch.isfinite(out).all()) and bool(((out.double() - value).abs() <= 2.0 ** -10 * 65504).all())
    plan.close()
