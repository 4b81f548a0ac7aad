// Work list of a ragged batch's attention (host/chunk_plan.cpp builds it, csrc/chunk_attention.cu walks it).
#pragma once
#include <stdint.h>

#include <vector>

namespace mf {

constexpr uint32_t kChunkTile = 128;  // keys per tile and query rows per stream
constexpr uint32_t kChunkMaxLen = 1u << 30;  // positions and tile arithmetic stay inside 32 bits

// A unit is the attention of up to 2 * (128 / G) consecutive new tokens of one sequence with the G query heads of one
// kv head: the rows (token, head) fill one or two 128-row query tiles ("streams").  The keys some row of the unit sees
// are listed page by page: first n_sink_pages pages from the start of the sequence, then the pages from first_page on;
// column x of this list (row x % P of its page x / P) is what the tiles are cut from.  An item is a range of a unit's
// tiles, processed by one CTA.
struct ChunkItem {
    uint32_t seq, kvh;
    uint32_t tok0;          // first token of the unit in the packed batch
    uint32_t n_tok;
    int32_t pos0;           // its position (negative: the first rows stand before the start of the cache)
    uint32_t n_sink_pages, first_page, n_pages;
    uint32_t tile_begin, tile_end;
    uint32_t slot, first_slot, n_parts;  // partial results, when the unit was cut
    uint32_t counter;       // ticket of a cut unit
    uint32_t reserved[2];
};
static_assert(sizeof(ChunkItem) == 64, "one item is four 16-byte loads");

constexpr uint32_t kChunkMaxCtas = 1u << 16;
// Most items a step of max_tokens new tokens can have.  Items are numbered in 32 bits.
uint64_t chunk_item_capacity(uint32_t batch, uint64_t max_tokens, uint32_t n_kv_heads, uint32_t group, uint32_t n_ctas);
// Partial slots and tickets: a boundary between two CTAs cuts at most one unit.
inline uint32_t chunk_slots(uint32_t n_ctas) { return 2 * n_ctas; }

// cta_begin: n_ctas + 1 entries.
void build_chunk_plan(const uint32_t *q_lens, const uint32_t *kv_lens, uint32_t batch, uint32_t n_kv_heads, uint32_t group,
                      uint32_t page_size, uint32_t window, uint32_t n_sinks, uint32_t n_ctas, std::vector<ChunkItem> &items,
                      std::vector<uint32_t> &cta_begin);

}  // namespace mf
