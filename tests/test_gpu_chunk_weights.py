"""GPU: the weights of the attention of ragged batches are held in f16 with headroom: many small ones count, and long contexts
are as exact as short ones."""
import pytest
import torch

from chunkcases import ChunkCase

pytestmark = pytest.mark.gpu

# A weight is rounded to f16 (2^-11 of it); the row's reference maximum is held at 2^7, so that subnormal weights are off by
# at most 2^-25 * 2^-7 of it.  The sum of all weights is at least the largest, which is at least the reference maximum.
FLOOR = 2.0 ** -32


@pytest.mark.parametrize("q_len", [1, 5, 200])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("power", [20, 24, 26])
def test_many_small_weights(mfk, foundry, q_len, d, power):
    """Every 64th key has the whole weight but for 2^-power a key, and a value of 0: the output is what the small ones add."""
    n, hq = 4096, 8
    case = ChunkCase(hq=hq, hkv=1, d=d, page=64, q_lens=[q_len], kv_lens=[n])
    case.q.zero_()
    case.q.view(-1, hq, d)[..., 0] = 8.0
    big = power * 0.6931472 / 8.0
    value = 2.0 ** (power - 16)  # (the output is about 63 * 2^-16)
    for b, page in enumerate(case.table[0].tolist()):
        case.k[page].zero_()
        case.k[page, :, 0, 0] = big
        case.v[page] = value
        case.v[page, :, 0] = 0
    plan, out = case.plan(foundry), torch.empty_like(case.q)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out, scale=1.0)
    foundry.synchronize()
    big = float(torch.tensor(big).half())
    pos = torch.arange(n - q_len, n, dtype=torch.float64, device="cuda")
    large = torch.floor(pos / 64) + 1
    small = pos + 1 - large
    w = torch.exp(torch.tensor(-8.0 * big, dtype=torch.float64))
    want = (small * w * value / (large + small * w))[:, None]
    # 2^-11 of the output for the weights' rounding, 2^-11 for its own, 2^-12 for f32 sums; the floor for each small weight
    tol = (2 * 2.0 ** -11 + 2.0 ** -12) * want + (small / large)[:, None] * FLOOR * value + 2.0 ** -25
    off = (out.double().view(q_len, -1) - want).abs()
    assert bool((off <= tol).all()), (float(off.max()), float(tol.min()), float(want.min()))
    plan.close()


@pytest.mark.parametrize("hq,hkv,d,page,q_lens,kv_lens,window,sinks", [
    (8, 1, 128, 16, [1], [131072], 0, 0),
    (16, 2, 128, 64, [5, 1], [131072, 100001], 0, 0),
    (8, 1, 64, 32, [1, 3], [131071, 65537], 0, 0),
    (4, 1, 128, 128, [130], [131072], 0, 0),
    (8, 1, 128, 16, [1, 40], [131072, 131072], 40000, 4),
])
def test_long_contexts(mfk, foundry, hq, hkv, d, page, q_lens, kv_lens, window, sinks):
    case = ChunkCase(hq=hq, hkv=hkv, d=d, page=page, q_lens=q_lens, kv_lens=kv_lens, window=window, sinks=sinks)
    plan, out = case.plan(foundry), torch.empty_like(case.q)
    foundry.paged_chunk_attention(plan, case.cache(mfk), case.q, out)
    foundry.synchronize()
    assert bool(torch.isfinite(out).all())
    t = 0
    for b, nq in enumerate(q_lens):
        see = case.visible(b)
        for h in range(hq):
            k, v = case.kc[b][h // (hq // hkv)].double(), case.vc[b][h // (hq // hkv)].double()
            s = (case.q[t:t + nq, h * d:(h + 1) * d].double() @ k.T * d ** -0.5).masked_fill(~see, -float("inf"))
            w = torch.softmax(s, -1)
            want, mean = w @ v, w @ v.abs()
            # The reference maximum may be up to 2^8 below the largest weight: larger weights, a lower floor.  f32 sums of
            # n / 16 terms and scores of |s| < 30: 2^-12 of the mean covers 2^-24 * sqrt(n) and 128 * 2^-24 * 30 / 4.
            tol = 2.0 ** -25 + 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * mean + \
                see.sum(1, keepdim=True) * w.max(1, keepdim=True).values * FLOOR * float(v.abs().max())
            off = (out[t:t + nq, h * d:(h + 1) * d].double() - want).abs()
            assert bool((off <= tol).all()), (b, h, float(off.max()), float((off - tol).max()))
        t += nq
    plan.close()
