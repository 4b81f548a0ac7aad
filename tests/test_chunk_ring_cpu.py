"""The ring of K/V tiles of the ragged attention, run on the host: the streams' own walk (csrc/chunk_ring.hpp, the code that
the kernel compiles) against loads that land in any order, products and softmax steps of any length.  Barriers are modelled
as the hardware has them: a wait knows its phase by parity alone."""
import ctypes as C
import heapq
import random
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parent.parent / "test-burn_b200" / "csrc" / "chunk_ring.hpp"
WAIT, PASS, USE_K, USE_V, FIT = range(5)

# A stream's steps in the order in which the kernel's issuing warp takes them: (what, slot, parity).
SOURCE = r"""
#include "%s"
using namespace mf;
template <uint32_t S> static uint32_t walk(uint32_t stream, uint32_t items, const uint32_t *tiles, const uint32_t *rows, uint32_t *out)
{
    RingReader<S> reader;
    uint32_t m = 0;
    auto put = [&](uint32_t what, uint32_t slot, uint32_t phase) { out[3 * m] = what, out[3 * m + 1] = slot, out[3 * m + 2] = phase, ++m; };
    auto landed = [&](uint32_t slot, uint32_t phase) { put(0, slot, phase); };
    auto pass = [&](uint32_t slot) { put(1, slot, 0); };
    for (uint32_t i = 0; i < items; ++i) {
        const uint32_t n = tiles[i], mine = rows[i] ? n : (n + 1 - stream) / 2;
        if (n == 0) continue;
        auto next = [&]() { return reader.next(rows[i] != 0, n, stream, landed, pass); };
        if (mine) put(2, next(), 0);
        for (uint32_t j = 0; j < mine; ++j) {
            const uint32_t v = next();
            put(4, v, reader.last_phase());
            put(3, v, 0);
            if (j + 1 < mine) put(2, next(), 0);
        }
        reader.finish(n, landed, pass);
    }
    return m;
}
extern "C" uint32_t ring_walk(uint32_t slots, uint32_t stream, uint32_t items, const uint32_t *tiles, const uint32_t *rows, uint32_t *out)
{
    return slots == 5 ? walk<5>(stream, items, tiles, rows, out) : slots == 10 ? walk<10>(stream, items, tiles, rows, out) : 0;
}
extern "C" uint32_t v_tile(uint32_t rows, uint32_t n, uint32_t load) { return ring_v_tile(rows != 0, n, load); }
extern "C" uint32_t uses(uint32_t rows, uint32_t n, uint32_t stream, uint32_t load) { return ring_uses(rows != 0, n, stream, load); }
"""


@pytest.fixture(scope="module")
def ring(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text(SOURCE % HEADER)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(d / "ring.cpp"), "-o", str(d / "ring.so")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return C.CDLL(str(d / "ring.so"))


def steps(ring, slots, stream, items):
    n = (C.c_uint32 * len(items))(*[t for t, _ in items])
    rows = (C.c_uint32 * len(items))(*[int(r) for _, r in items])
    out = (C.c_uint32 * (3 * 12 * (sum(t for t, _ in items) + 1)))()
    m = ring.ring_walk(slots, stream, len(items), n, rows, out)
    return [tuple(out[3 * i:3 * i + 3]) for i in range(m)]


def v_loads(ring, n, rows, stream):
    """The V loads that a stream uses, in order, counted from the item's first load."""
    return [x for x in range(2 * n) if ring.v_tile(int(rows), n, x) < n and ring.uses(int(rows), n, stream, x)]


def own_waits_only(slots, stream, items):
    """A walk with a mistake: a stream waits for its own loads alone and hands them back for both."""
    out, base = [], 0
    for n, rows in items:
        mine = list(range(n)) if rows else list(range(stream, n, 2))
        def load(t, v):
            return 2 * t + v if rows else (4 * (t // 2) + (2 * v + t % 2 if t // 2 * 2 + 1 < n else v))
        def use(t, v):
            at = base + load(t, v)
            return [(WAIT, at % slots, at // slots & 1)] + [(FIT, at % slots, at // slots & 1)] * v + [(USE_V if v else USE_K, at % slots, 0 if rows else 1)]
        for j, t in enumerate(mine):
            if j == 0:
                out += use(t, 0)
            out += use(t, 1)
            if j + 1 < len(mine):
                out += use(mine[j + 1], 0)
        base += 2 * n
    return out


class Barrier:
    """Phases completed; `wait` is over when the phase in progress has the other parity."""

    def __init__(self, arrivals):
        self.arrivals, self.left, self.phase, self.waiting = arrivals, arrivals, 0, []

    def arrive(self, wake):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.arrivals, self.phase + 1
            for w in self.waiting:
                wake(w)
            self.waiting = []

    def over(self, parity):
        return (self.phase & 1) != parity


class EarlyWait(Exception):
    pass


def simulate(ring, slots, items, walks, seed):
    """Runs producer, two issuing warps, the warp that prepares V tiles, two softmax groups and the tensor pipe; raises EarlyWait when a wait returns before
    the load it is for has landed, or when a load lands in a tile that is still read."""
    rng = random.Random(seed)
    slow = rng.choice([0.0, 0.1, 0.3])
    delay = lambda mean: rng.expovariate(1 / mean) * (rng.choice([1, 20]) if rng.random() < slow else 1)  # noqa: E731
    full, empty = [Barrier(1) for _ in range(slots)], [Barrier(3) for _ in range(slots)]
    loads = 2 * sum(n for n, _ in items)
    landed, issued = [False] * loads, [False] * loads
    readers = [0] * loads
    events, now, seq = [], 0.0, 0

    def at(t, fn):
        nonlocal seq
        heapq.heappush(events, (t, seq, fn))
        seq += 1

    def wake(fn):
        at(now, fn)

    def run(gen):
        for op in gen:
            if isinstance(op, float):
                at(now + op, lambda: run(gen))
                return
            bar, parity = op
            if not bar.over(parity):
                bar.waiting.append(lambda: again(gen, op))
                return

    def again(gen, op):
        bar, parity = op
        if not bar.over(parity):
            bar.waiting.append(lambda: again(gen, op))
        else:
            run(gen)

    def land(load):
        landed[load] = True
        full[load % slots].arrive(wake)

    def producer():
        for load in range(loads):
            slot = load % slots
            yield empty[slot], (load // slots & 1) ^ 1
            if load >= slots and (readers[load - slots] or not landed[load - slots]):
                raise EarlyWait(f"load {load} goes into a tile that is in use")
            issued[load] = True
            at(now + delay(1.0), lambda load=load: land(load))
            yield delay(0.05)

    def check(load, who):
        if not landed[load]:
            raise EarlyWait(f"{who}: load {load} has not landed")
        if load + slots < loads and issued[load + slots]:
            raise EarlyWait(f"{who}: load {load} has been replaced")

    # what the streams' uses are, in the order of their walks: loads of K and V tiles; which V tiles need preparing
    def uses(stream):
        base = 0
        for n, rows in items:
            for j, v in enumerate(v_loads(ring, n, rows, stream)):
                yield base + v - (2 if not rows and 2 * j + 1 < n else 1), base + v
            base += 2 * n

    prepared = {load for load in range(loads) if rng.random() < 0.4}

    scores, weights, fit = [Barrier(1) for _ in range(2)], [Barrier(1) for _ in range(2)], [Barrier(1) for _ in range(slots)]

    def issuer(s, walk):
        mine = list(uses(s))
        order = []
        base_tiles = 0
        for n, rows in items:
            count = n if rows else (n + 1 - s) // 2
            for j in range(count):
                k, v = mine[base_tiles + j]
                if j == 0:
                    order.append(k)
                order.append(v)
                if j + 1 < count:
                    order.append(mine[base_tiles + j + 1][0])
            base_tiles += count
        done_v, pipe = 0, 0.0
        at_use = 0
        for what, slot, extra in walk:
            if what == WAIT:
                yield full[slot], extra
            elif what == PASS:
                empty[slot].arrive(wake)
            elif what == FIT:
                load = order[at_use]
                if load in prepared:
                    yield fit[slot], extra
                    if load not in ready:
                        raise EarlyWait(f"stream {s}: load {load} has not been prepared")
            else:
                load = order[at_use]
                at_use += 1
                assert load % slots == slot
                check(load, f"stream {s}")
                if what == USE_V:
                    yield weights[s], done_v & 1
                    done_v += 1
                    check(load, f"stream {s}, product")
                readers[load] += 1
                pipe = max(pipe, now) + delay(0.3)

                def over(load=load, slot=slot, what=what, extra=extra):
                    check(load, f"stream {s}, end of a product")
                    readers[load] -= 1
                    for _ in range(1 + extra):
                        empty[slot].arrive(wake)
                    if what == USE_K:
                        scores[s].arrive(wake)
                at(pipe, over)
                yield delay(0.05)
        assert at_use == len(order)

    ready = set()

    def preparer():
        base = 0
        for n, rows in items:
            for x in range(2 * n):
                load = base + x
                yield full[load % slots], load // slots & 1
                check(load, "preparing")
                if load in prepared and ring.v_tile(int(rows), n, x) < n:
                    yield delay(0.2)
                    check(load, "preparing")
                    ready.add(load)
                fit[load % slots].arrive(wake)
                empty[load % slots].arrive(wake)
            base += 2 * n

    def softmax(s):
        for t in range(len(list(uses(s)))):
            yield scores[s], t & 1
            yield delay(0.5)
            weights[s].arrive(wake)

    run(producer())
    run(preparer())
    for s in range(2):
        run(issuer(s, walks[s]))
        run(softmax(s))
    while events:
        now, _, fn = heapq.heappop(events)
        fn()
    assert all(landed) and not any(readers), "the ring stood still"
    assert [b.phase for b in empty] == [len(range(x, loads, slots)) for x in range(slots)] and all(b.left == 3 for b in empty)


def items_of(rng, count, most):
    return [(rng.randint(0, most), rng.random() < 0.4) for _ in range(count)]


@pytest.mark.parametrize("slots", [5, 10])
def test_uses_of_an_item(ring, slots):
    """Every load is some stream's; a stream's V load is one it uses; the walk takes each load once and in order."""
    for n in range(1, 41):
        for rows in (0, 1):
            for load in range(2 * n):
                used = [ring.uses(rows, n, s, load) for s in range(2)]
                assert used == [1, 1] if rows else sum(used) == 1
            for s in range(2):
                mine = n if rows else (n + 1 - s) // 2
                v = v_loads(ring, n, rows, s)
                assert [ring.v_tile(rows, n, x) for x in v] == [j if rows else 2 * j + s for j in range(mine)]
                walk = steps(ring, slots, s, [(n, rows)])
                waits = [(slot, phase) for what, slot, phase in walk if what == WAIT]
                assert waits == [(x % slots, x // slots & 1) for x in range(2 * n)]


@pytest.mark.parametrize("slots", [5, 10])
@pytest.mark.parametrize("rows", [False, True])
def test_no_wait_returns_early(ring, slots, rows):
    for n in range(1, 41):
        walks = [steps(ring, slots, s, [(n, rows)]) for s in range(2)]
        for seed in range(6):
            simulate(ring, slots, [(n, rows)], walks, seed)


@pytest.mark.parametrize("slots", [5, 10])
def test_no_wait_returns_early_over_items_of_both_kinds(ring, slots):
    rng = random.Random(3)
    for seed in range(150):
        items = items_of(rng, rng.randint(2, 9), rng.choice([2, 5, 12]))
        simulate(ring, slots, items, [steps(ring, slots, s, items) for s in range(2)], seed)


def test_the_model_sees_a_stream_that_waits_for_its_own_loads_only(ring):
    caught = 0
    for seed in range(60):
        items = [(16, False)]
        try:
            simulate(ring, 5, items, [own_waits_only(5, s, items) for s in range(2)], seed)
        except (EarlyWait, AssertionError):
            caught += 1
    assert caught > 10
    for seed in range(20):  # the same walk is sound where both streams use every load
        items = [(16, True)]
        simulate(ring, 5, items, [own_waits_only(5, s, items) for s in range(2)], seed)
