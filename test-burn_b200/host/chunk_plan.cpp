// Planner of a ragged batch's attention: which CTA walks which key tiles of which rows.
#include <algorithm>
#include <new>
#include <vector>

#include "../../include/metallic_cuda.h"
#include "../csrc/chunk_plan.hpp"

namespace mf {
namespace {

// Costs in a common unit of about a quarter of a microsecond: a tile of a unit with more than 128 rows (two query tiles on
// every key tile: 2.3 us, the softmax's pace), a tile of a unit with at most that (1.4 us, the memory's pace), and what
// an item costs its CTA beyond its tiles (q, draining the products, writing the rows, joining: about 4 us).  With equal
// costs for all tiles the CTAs that had a mixed step's prompt rows ended 90 us behind the others.  Measured at head_dim 128
// and used for 64, too, where a tile has half the bytes and the same exponentials.
constexpr uint32_t kRowsTileCost = 9, kKeysTileCost = 5, kItemCost = 16;
// Shortest piece a unit is cut into when every CTA has several units, in tiles.
constexpr uint32_t kMinPiece = 2;

}  // namespace

uint64_t chunk_item_capacity(uint32_t batch, uint64_t max_tokens, uint32_t n_kv_heads, uint32_t group, uint32_t n_ctas)
{
    const uint32_t per_unit = 2 * (kChunkTile / group);
    return (uint64_t)n_kv_heads * (std::min<uint64_t>(batch, max_tokens) + max_tokens / per_unit) + 2 * (uint64_t)n_ctas;
}

void build_chunk_plan(const uint32_t *q_lens, const uint32_t *kv_lens, uint32_t batch, uint32_t n_kv_heads, uint32_t group,
                      uint32_t page_size, uint32_t window, uint32_t n_sinks, uint32_t n_ctas, std::vector<ChunkItem> &items,
                      std::vector<uint32_t> &cta_begin)
{
    const uint32_t per_unit = 2 * (kChunkTile / group), P = page_size;
    auto tile_cost = [&](const ChunkItem &u) { return u.n_tok > per_unit / 2 ? kRowsTileCost : kKeysTileCost; };
    std::vector<ChunkItem> units;
    uint64_t cost = 0;
    uint32_t tok = 0;
    for (uint32_t b = 0; b < batch; ++b) {
        for (uint32_t h = 0; h < n_kv_heads; ++h)
            for (uint32_t t = 0; t < q_lens[b]; t += per_unit) {
                ChunkItem u{};
                u.seq = b;
                u.kvh = h;
                u.tok0 = tok + t;
                u.n_tok = std::min(per_unit, q_lens[b] - t);
                u.pos0 = (int32_t)((int64_t)kv_lens[b] - q_lens[b] + t);
                u.n_parts = 1;
                const int64_t last = (int64_t)u.pos0 + u.n_tok - 1;
                if (last >= 0) {
                    const uint32_t first_pos = (uint32_t)std::max(u.pos0, 0);
                    const uint32_t first_seen = window && first_pos >= window ? first_pos - window + 1 : 0;
                    const uint32_t sinks = (uint32_t)std::min<int64_t>(n_sinks, last + 1);
                    const uint32_t sink_pages = (sinks + P - 1) / P;
                    u.first_page = first_seen / P;
                    if (sink_pages >= u.first_page) u.first_page = 0;
                    else u.n_sink_pages = sink_pages;
                    u.n_pages = u.n_sink_pages + (uint32_t)(last / P) - u.first_page + 1;
                    u.tile_end = (uint32_t)(((uint64_t)u.n_pages * P + kChunkTile - 1) / kChunkTile);
                }
                cost += (uint64_t)u.tile_end * tile_cost(u) + kItemCost;
                units.push_back(u);
            }
        tok += q_lens[b];
    }
    items.clear();
    cta_begin.assign(n_ctas + 1, 0);
    uint32_t slots = 0, counters = 0;
    // `parts` consecutive items of unit u are at the end of the list
    auto number_parts = [&](size_t first) {
        const uint32_t parts = (uint32_t)(items.size() - first);
        if (parts < 2) return;
        for (size_t i = first; i < items.size(); ++i) {
            items[i].n_parts = parts;
            items[i].first_slot = slots;
            items[i].slot = slots + (uint32_t)(i - first);
            items[i].counter = counters;
        }
        slots += parts;
        ++counters;
    };
    auto parts_of = [&](const ChunkItem &u, uint32_t most) {
        const uint32_t tiles = most / tile_cost(u);
        return std::max(1u, (u.tile_end + tiles - 1) / tiles);
    };
    uint32_t lo = 1;
    bool pieces = units.size() <= n_ctas;
    if (pieces) {
        // Few units: one item per CTA, every unit cut into even pieces that cost at most `lo`, the smallest number for
        // which there are CTAs enough - unless unequal units leave some CTA more than an equal span would.
        lo = 2 * kKeysTileCost;  // (the two streams of a small unit take two tiles in about the time of one)
        uint32_t hi = lo;
        for (const ChunkItem &u : units) hi = std::max(hi, u.tile_end * tile_cost(u));
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            uint64_t need = 0;
            for (const ChunkItem &u : units) need += parts_of(u, mid);
            if (need <= n_ctas) hi = mid;
            else lo = mid + 1;
        }
        pieces = lo + kItemCost <= cost / n_ctas + 2 * kItemCost;  // (spans pay an item more per CTA)
    }
    if (pieces) {
        for (const ChunkItem &u : units) {
            const uint32_t parts = parts_of(u, lo);
            const size_t first = items.size();
            for (uint32_t i = 0; i < parts; ++i) {
                ChunkItem it = u;
                it.tile_begin = (uint32_t)((uint64_t)u.tile_end * i / parts);
                it.tile_end = (uint32_t)((uint64_t)u.tile_end * (i + 1) / parts);
                items.push_back(it);
            }
            number_parts(first);
        }
        for (uint32_t c = 0; c <= n_ctas; ++c) cta_begin[c] = (uint32_t)std::min<size_t>(c, items.size());
        return;
    }
    // Spans over the list of units, cut where a span is full; the smallest span for which the CTAs suffice.  fill() walks the
    // list with spans of cost `span` and returns how many there are (n_ctas + 1: too many).
    auto fill = [&](uint64_t span, bool emit) {
        uint32_t cta = 0;
        uint64_t room = span;
        for (const ChunkItem &u : units) {
            const uint32_t w = tile_cost(u);
            const size_t first = items.size();
            uint32_t at = 0;
            for (bool whole = false; !whole;) {
                const uint32_t rest = u.tile_end - at;
                uint32_t take = room > kItemCost ? (uint32_t)std::min<uint64_t>(rest, (room - kItemCost) / w) : 0;
                if (take < rest && rest - take < kMinPiece) take = rest > kMinPiece ? rest - kMinPiece : 0;
                if (take < rest && take < kMinPiece) take = 0;
                const bool fits = room >= kItemCost && (take > 0 || rest == 0);
                if (!fits) {
                    if (++cta == n_ctas) return n_ctas + 1;
                    if (emit) cta_begin[cta] = (uint32_t)items.size();
                    room = span;
                    continue;  // (a unit without tiles, too: its rows are written)
                }
                if (emit) {
                    ChunkItem it = u;
                    it.tile_begin = at;
                    it.tile_end = at + take;
                    items.push_back(it);
                }
                room -= kItemCost + (uint64_t)take * w;
                at += take;
                whole = at >= u.tile_end;
            }
            if (emit) number_parts(first);
        }
        if (emit)
            while (cta < n_ctas) cta_begin[++cta] = (uint32_t)items.size();
        return cta + 1;
    };
    uint64_t low = std::max<uint64_t>(cost / n_ctas, kItemCost + kMinPiece * kRowsTileCost), high = low;
    while (fill(high, false) > n_ctas) {
        low = high + 1;
        high += high / 8 + 1;
    }
    while (low + low / 256 < high) {  // within half a percent
        const uint64_t mid = low + (high - low) / 2;
        if (fill(mid, false) > n_ctas) low = mid + 1;
        else high = mid;
    }
    fill(high, true);
}

}  // namespace mf

extern "C" uint32_t mf_chunk_plan_build_host(const uint32_t *q_lens, const uint32_t *kv_lens, uint32_t batch, uint32_t n_heads,
                                             uint32_t n_kv_heads, uint32_t page_size, uint32_t window, uint32_t n_sinks,
                                             uint32_t n_ctas, uint32_t *items_out, uint32_t item_capacity, uint32_t *cta_begin_out)
{
    if (!q_lens || !kv_lens || !cta_begin_out || n_kv_heads == 0 || n_heads % n_kv_heads || n_heads / n_kv_heads == 0 ||
        n_heads / n_kv_heads > 64 || page_size == 0 || n_ctas == 0 || n_ctas > mf::kChunkMaxCtas)
        return 0;
    uint64_t tokens = 0;
    for (uint32_t b = 0; b < batch; ++b) {
        if (q_lens[b] > mf::kChunkMaxLen || kv_lens[b] > mf::kChunkMaxLen) return 0;
        tokens += q_lens[b];
    }
    if (tokens > mf::kChunkMaxLen || mf::chunk_item_capacity(batch, tokens, n_kv_heads, n_heads / n_kv_heads, n_ctas) > UINT32_MAX) return 0;
    try {
        std::vector<mf::ChunkItem> items;
        std::vector<uint32_t> begin;
        mf::build_chunk_plan(q_lens, kv_lens, batch, n_kv_heads, n_heads / n_kv_heads, page_size, window, n_sinks, n_ctas, items, begin);
        if (items_out && items.size() <= item_capacity)
            std::copy(reinterpret_cast<const uint32_t *>(items.data()),
                      reinterpret_cast<const uint32_t *>(items.data() + items.size()), items_out);
        std::copy(begin.begin(), begin.end(), cta_begin_out);
        return (uint32_t)items.size();
    } catch (const std::bad_alloc &) {
        return 0;
    }
}
