"""The planner of a ragged batch's attention: every key that some row sees is walked exactly once, by items whose pages
are the visible ones, and the work is spread over the CTAs."""
import numpy as np
import pytest

TILE = 128


def keys_of(item, page):
    """The keys an item's tiles hold."""
    x = np.arange(int(item["tile_begin"]) * TILE, min(int(item["tile_end"]) * TILE, int(item["n_pages"]) * page))
    v = x // page
    return np.where(v < item["n_sink_pages"], v, v - item["n_sink_pages"] + item["first_page"]) * page + x % page


NAMES = ["seq", "kvh", "tok0", "n_tok", "pos0", "n_sink_pages", "first_page", "n_pages", "tile_begin", "tile_end", "slot", "first_slot",
         "n_parts", "counter"]


def decode(row):
    d = {n: int(x) for n, x in zip(NAMES, row)}
    d["pos0"] = int(np.int32(np.uint32(d["pos0"])))
    return d


def check(mfk, q_lens, kv_lens, hq, hkv, page, window, sinks, n_ctas):
    items, begin = mfk.build_chunk_plan_host(q_lens, kv_lens, n_heads=hq, n_kv_heads=hkv, page_size=page, n_ctas=n_ctas, window=window,
                                             sinks=sinks)
    assert begin[0] == 0 and begin[-1] == len(items) and np.all(np.diff(begin.astype(np.int64)) >= 0)
    per_unit = 2 * (TILE // (hq // hkv))
    starts = np.concatenate([[0], np.cumsum(q_lens)])
    cover = {}
    slots, tickets = [], {}
    for it in map(decode, items):
        b = it["seq"]
        assert 1 <= it["n_tok"] <= per_unit and starts[b] <= it["tok0"] and it["tok0"] + it["n_tok"] <= starts[b + 1]
        assert it["pos0"] == int(kv_lens[b]) - int(q_lens[b]) + it["tok0"] - starts[b]
        unit = (it["kvh"], it["tok0"])
        cover.setdefault(unit, []).append(it)
        if it["n_parts"] > 1:
            assert it["tile_end"] > it["tile_begin"] and it["first_slot"] <= it["slot"] < it["first_slot"] + it["n_parts"]
            slots.append(it["slot"])
            tickets.setdefault(it["counter"], set()).add(unit)
    assert len(set(slots)) == len(slots) and all(s < 2 * n_ctas for s in slots)
    assert all(len(u) == 1 and c < n_ctas for c, u in tickets.items())
    tokens = {h: np.zeros(starts[-1], int) for h in range(hkv)}
    for (h, t0), parts in cover.items():
        tokens[h][t0:t0 + parts[0]["n_tok"]] += 1
        assert len(parts) == parts[0]["n_parts"]
        parts.sort(key=lambda i: i["tile_begin"])
        assert parts[0]["tile_begin"] == 0 and all(a["tile_end"] == b["tile_begin"] for a, b in zip(parts, parts[1:]))
        assert parts[-1]["tile_end"] == -(-parts[0]["n_pages"] * page // TILE)
        keys = np.concatenate([keys_of(p, page) for p in parts])
        assert len(set(keys)) == len(keys)
        seen = set()
        for r in range(parts[0]["n_tok"]):
            p = parts[0]["pos0"] + r
            if p < 0:
                continue
            lo = max(0, p - window + 1) if window else 0
            seen |= set(range(min(sinks, lo))) | set(range(lo, p + 1))
        assert seen <= set(keys.tolist())
        assert {k // page for k in seen} == {int(k) // page for k in keys}, "a page that no row sees"
    for h in range(hkv):
        assert np.all(tokens[h] == 1)
    return [decode(r) for r in items], begin


@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,page,window,sinks", [
    ([1], [1], 8, 2, 16, 0, 0),
    ([1] * 5, [1, 17, 128, 129, 3000], 16, 2, 16, 0, 0),
    ([0, 4, 0, 1], [10, 4, 0, 9], 16, 2, 16, 0, 0),
    ([6, 40], [4, 0], 8, 2, 16, 0, 0),
    ([300, 1, 17], [900, 2000, 17], 14, 2, 32, 0, 0),
    ([300, 1, 17], [900, 2000, 17], 64, 1, 64, 0, 0),
    ([1] * 6, [1, 3, 130, 1025, 5000, 4096], 16, 2, 16, 1024, 4),
    ([300, 5], [2000, 999], 16, 2, 16, 200, 4),
    ([100, 1, 1], [900, 400, 90], 8, 2, 16, 33, 150),
    ([20, 9], [4, 9], 8, 2, 8, 3, 2),
    ([1, 33], [1000, 1000], 8, 2, 64, 65, 70),
    ([1, 50], [1000, 1100], 8, 2, 128, 129, 1),
    ([1, 50], [1000, 1100], 8, 2, 16, 1, 0),
])
@pytest.mark.parametrize("n_ctas", [1, 7, 148])
def test_every_seen_key_once(mfk, q_lens, kv_lens, hq, hkv, page, window, sinks, n_ctas):
    check(mfk, q_lens, kv_lens, hq, hkv, page, window, sinks, n_ctas)


def test_random_batches(mfk):
    rng = np.random.default_rng(4)
    for _ in range(60):
        n = int(rng.integers(1, 8))
        kv = rng.integers(0, 1500, n)
        q = np.minimum(rng.integers(0, 90, n), kv + rng.integers(0, 3, n))
        group = int(rng.choice([1, 2, 3, 5, 7, 8, 16]))
        hkv = int(rng.integers(1, 3))
        window = int(rng.choice([0, 1, 50, 400]))
        check(mfk, q, kv, group * hkv, hkv, int(rng.choice([8, 16, 64, 128])), window, int(rng.integers(0, 60)) if window else 0,
              int(rng.choice([3, 20, 148])))


def test_work_is_spread(mfk):
    """No CTA has much more than its share: single long sequences, unequal decode batches, long prompts."""
    rng = np.random.default_rng(6)
    for q, kv, hq, hkv, window in (([1], [131072], 8, 8, 0), ([1] * 64, rng.integers(512, 16384, 64), 16, 2, 0),
                                   ([1] * 64, rng.integers(512, 16384, 64), 16, 2, 4096), ([4096], [8192], 16, 2, 0),
                                   ([512, 384] + [1] * 46, rng.integers(600, 8192, 48), 32, 8, 0)):
        items, begin = mfk.build_chunk_plan_host(q, kv, n_heads=hq, n_kv_heads=hkv, page_size=16, n_ctas=148, window=window)
        # the planner's units: 9 for a tile of a unit with more than 128 rows, 5 for another, 16 for an item
        rows = items[:, 3].astype(int) > TILE // (hq // hkv)
        cost = (items[:, 9] - items[:, 8]).astype(int) * np.where(rows, 9, 5) + 16
        load = np.array([cost[a:b].sum() for a, b in zip(begin, begin[1:])])
        assert load.max() <= 1.15 * load.mean() + 16, (load.max(), load.mean())


def test_arguments_without_a_meaning(mfk):
    one, begin = np.ones(1, np.uint32), np.zeros(2, np.uint32)
    p = one.ctypes.data
    f = mfk.lib.mf_chunk_plan_build_host
    assert f(None, p, 1, 8, 2, 16, 0, 0, 1, None, 0, begin.ctypes.data) == 0
    for bad in ((1, 7, 2, 16, 1), (1, 8, 0, 16, 1), (1, 8, 2, 0, 1), (1, 8, 2, 16, 0), (1, 0, 2, 16, 1), (1, 130, 2, 16, 1)):
        batch, hq, hkv, page, ctas = bad
        assert f(p, p, batch, hq, hkv, page, 0, 0, ctas, None, 0, begin.ctypes.data) == 0


@pytest.mark.parametrize("q_len,kv_len", [((1 << 30) + 1, 1 << 30), (0xFFFFFFFF, 5), (1, (1 << 30) + 1), (1, 0xFFFFFFFF)])
def test_lengths_past_the_limit(mfk, q_len, kv_len):
    items, begin = mfk.build_chunk_plan_host([q_len], [kv_len], n_heads=8, n_kv_heads=2, page_size=16, n_ctas=4)
    assert len(items) == 0 and not begin.any()


@pytest.mark.parametrize("n_ctas", [1, 7, 148])
def test_units_without_keys_are_in_the_plan(mfk, n_ctas):
    """New tokens of a sequence without rows come out as zeros: someone has to write them, wherever a span ends."""
    rng = np.random.default_rng(5)
    for batch in (1, 60, 300):
        kv_lens = np.where(rng.random(batch) < 0.5, 0, rng.integers(1, 900, batch))
        q_lens = rng.integers(0, 40, batch)
        items, begin = mfk.build_chunk_plan_host(q_lens, kv_lens, n_heads=14, n_kv_heads=2, page_size=16, n_ctas=n_ctas)
        assert begin[0] == 0 and begin[-1] == len(items) and (np.diff(begin.astype(int)) >= 0).all()
        first = items[items[:, 8] == 0]  # the piece of a unit that starts at its first tile
        written = np.zeros((2, q_lens.sum()), int)
        for it in first:
            written[it[1], it[2]:it[2] + it[3]] += 1
        assert (written == 1).all()
