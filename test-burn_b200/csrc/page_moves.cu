// Pages copied in all layers of a model at once: forks (private copies of a shared page) and compaction.
//
// The pairs come from the host's page allocator and travel as kernel parameters: no upload, no device list that
// would have to outlive the call, and a captured launch keeps its own.
#include <algorithm>
#include <new>
#include <vector>

#include "internal.hpp"

namespace mf {
namespace {

constexpr uint32_t kMovePools = 128;   // pools per launch: 64 layers of an f16 cache, 32 of an 8-bit one
constexpr uint32_t kUnroll = 8;        // 16-byte units a lane has in flight
constexpr uint32_t kSegment = 32 * kUnroll;  // units a warp copies at a time (4 KB)

// Kernel parameters may take 32 764 bytes.  Two sizes: a fork's few pairs should not pay for a compaction's parameters.
template <uint32_t PAIRS>
struct MoveParams {
    uint4 *pool[kMovePools];
    uint32_t n_wide;       // pools [0, n_wide) have pages of units[0] 16-byte units, the others of units[1]
    uint32_t n_pools, n_pairs;
    uint32_t units[2];
    uint32_t src[PAIRS], dst[PAIRS];
};

// A warp copies a segment of one page of one pool: eight independent 16-byte loads a lane, then eight stores.  Bound by
// HBM (every byte read once and written once); the segments of one page are neighbours, so pages stream.  Measured: 1 000
// pages of 8 layers (1.05 GB moved) 173 us, 0.93 of the copy rate; 777 pages of 28 8-bit layers (0.73 GB, with scales
// of 256 bytes a page) 125 us, 0.90; 8 pages of 36 layers (9.4 MB) 2.5 us.
template <uint32_t PAIRS>
__global__ void __launch_bounds__(256) move_pages_kernel(const __grid_constant__ MoveParams<PAIRS> p)
{
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x / 32);
    const uint64_t first = (uint64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
#pragma unroll 1
    for (uint32_t kind = 0; kind < 2; ++kind) {
        const uint32_t units = p.units[kind], pool0 = kind ? p.n_wide : 0, pools = kind ? p.n_pools - p.n_wide : p.n_wide;
        const uint32_t segments = (units + kSegment - 1) / kSegment;
        const uint64_t total = (uint64_t)pools * p.n_pairs * segments;
#pragma unroll 1
        for (uint64_t x = first; x < total; x += warps) {
            const uint64_t page = x / segments;
            const uint32_t at = (uint32_t)(x - page * segments) * kSegment + lane, pool = (uint32_t)(page / p.n_pairs);
            const uint32_t pair = (uint32_t)(page - (uint64_t)pool * p.n_pairs);
            uint4 *base = p.pool[pool0 + pool];
            const uint4 *src = base + (size_t)p.src[pair] * units;
            uint4 *dst = base + (size_t)p.dst[pair] * units;
            uint4 r[kUnroll];
#pragma unroll
            for (uint32_t i = 0; i < kUnroll; ++i)
                if (at + i * 32 < units) r[i] = __ldcs(src + at + i * 32);
#pragma unroll
            for (uint32_t i = 0; i < kUnroll; ++i)
                if (at + i * 32 < units) dst[at + i * 32] = r[i];
        }
    }
}

struct PoolRef {
    void *base;
    uint64_t page_bytes;
};

template <uint32_t PAIRS>
mf_status launch_moves(MfContext *ctx, const PoolRef *pools, uint32_t n_pools, const uint32_t *src, const uint32_t *dst, uint32_t n)
{
    MoveParams<PAIRS> p;
    p.n_pools = n_pools;
    p.n_pairs = n;
    p.n_wide = 0;
    p.units[0] = (uint32_t)(pools[0].page_bytes / 16);
    p.units[1] = (uint32_t)(pools[n_pools - 1].page_bytes / 16);
    while (p.n_wide < n_pools && pools[p.n_wide].page_bytes == pools[0].page_bytes) ++p.n_wide;
    for (uint32_t j = 0; j < n_pools; ++j) p.pool[j] = static_cast<uint4 *>(pools[j].base);
    std::copy(src, src + n, p.src);
    std::copy(dst, dst + n, p.dst);
    uint64_t segments = 0;
    for (uint32_t k = 0; k < 2; ++k)
        segments += (uint64_t)(k ? n_pools - p.n_wide : p.n_wide) * n * ((p.units[k] + kSegment - 1) / kSegment);
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((segments + 7) / 8, (uint64_t)std::max(1, ctx->sm_count) * 8);
    move_pages_kernel<PAIRS><<<blocks, 256, 0, ctx->stream>>>(p);
    const mf_status st = check_launch(ctx, "move_pages_kernel");
    if (st == MF_OK) ctx->note_plain_launch(true);
    return st;
}

// pools: at most two page sizes, those of one size together.
mf_status move_pages(MfContext *ctx, const std::vector<PoolRef> &pools, uint32_t n_pages, const uint32_t *src, const uint32_t *dst,
                     uint32_t n, const char *what)
{
    for (uint32_t i = 0; i < n; ++i)
        if (src[i] >= n_pages || dst[i] >= n_pages)
            return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: pair %u (%u -> %u) outside the pool of %u pages", what, i, src[i], dst[i], n_pages);
    // Destinations are distinct and no source is one: the copies may then run in any order.
    std::vector<uint32_t> written(dst, dst + n);
    std::sort(written.begin(), written.end());
    const auto twice = std::adjacent_find(written.begin(), written.end());
    if (twice != written.end()) return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: page %u is written twice", what, *twice);
    for (uint32_t i = 0; i < n; ++i)
        if (std::binary_search(written.begin(), written.end(), src[i]))
            return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: page %u is read and written", what, src[i]);
    DeviceScope scope(ctx->device);
    for (size_t p0 = 0; p0 < pools.size(); p0 += kMovePools) {
        const uint32_t np = (uint32_t)std::min<size_t>(kMovePools, pools.size() - p0);
        for (uint32_t i0 = 0; i0 < n;) {
            const uint32_t ni = std::min(n - i0, n - i0 <= 64 ? 64u : 2048u);
            const mf_status st = n - i0 <= 64 ? launch_moves<64>(ctx, &pools[p0], np, src + i0, dst + i0, ni)
                                              : launch_moves<2048>(ctx, &pools[p0], np, src + i0, dst + i0, ni);
            if (st != MF_OK) return st;
            i0 += ni;
        }
    }
    return MF_OK;
}

template <class Cache>
mf_status check_layers(MfContext *ctx, const Cache *layers, uint32_t n_layers, const uint32_t *src, const uint32_t *dst, uint32_t n,
                       const char *what)
{
    if (!layers || n_layers == 0 || (n && (!src || !dst))) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "%s: null input", what);
    for (uint32_t i = 0; i < n_layers; ++i) {
        if (!layers[i].k_pool || !layers[i].v_pool) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "%s: pools of layer %u", what, i);
        if (layers[i].n_pages != layers[0].n_pages || layers[i].n_kv_heads != layers[0].n_kv_heads ||
            layers[i].page_size != layers[0].page_size || layers[i].head_dim != layers[0].head_dim)
            return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: layer %u has another geometry than layer 0", what, i);
    }
    return MF_OK;
}

mf_status check_pool(MfContext *ctx, const PoolRef &r, const char *what)
{
    if (reinterpret_cast<uintptr_t>(r.base) & 15u) return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: pools must be 16-byte aligned", what);
    if (r.page_bytes == 0 || r.page_bytes % 16 || r.page_bytes / 16 > 0xFFFFFFFFull)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: pages of %llu bytes", what, (unsigned long long)r.page_bytes);
    return MF_OK;
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" {

mf_status mf_paged_move_pages(MfContext *ctx, const MfPagedKv *layers, uint32_t n_layers, const uint32_t *src, const uint32_t *dst,
                              uint32_t n)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    mf_status st = check_layers(ctx, layers, n_layers, src, dst, n, "move pages");
    if (st != MF_OK) return st;
    try {
        std::vector<PoolRef> pools;
        pools.reserve(2 * (size_t)n_layers);
        const uint64_t bytes = (uint64_t)layers[0].n_kv_heads * layers[0].page_size * layers[0].head_dim * 2;
        for (uint32_t i = 0; i < n_layers; ++i)
            for (void *base : {layers[i].k_pool, layers[i].v_pool}) {
                pools.push_back({base, bytes});
                if ((st = check_pool(ctx, pools.back(), "move pages")) != MF_OK) return st;
            }
        return move_pages(ctx, pools, layers[0].n_pages, src, dst, n, "move pages");
    } catch (const std::bad_alloc &) {
        return fail(ctx, MF_ERR_OUT_OF_MEMORY, "move pages: host memory");
    }
}

mf_status mf_paged_kv8_move_pages(MfContext *ctx, const MfPagedKv8 *layers, uint32_t n_layers, const uint32_t *src,
                                  const uint32_t *dst, uint32_t n)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    mf_status st = check_layers(ctx, layers, n_layers, src, dst, n, "move pages (8-bit)");
    if (st != MF_OK) return st;
    try {
        std::vector<PoolRef> pools;
        const uint64_t rows = (uint64_t)layers[0].n_kv_heads * layers[0].page_size;
        constexpr uint32_t kGroup = kMovePools / 4;  // layers per launch: their byte pools, then their scales
        for (uint32_t i = 0; i < n_layers; ++i)
            if (!layers[i].k_scales || !layers[i].v_scales)
                return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "move pages (8-bit): scales of layer %u", i);
        pools.reserve(4 * (size_t)n_layers);
        for (uint32_t g = 0; g < n_layers; g += kGroup) {
            const uint32_t end = std::min(n_layers, g + kGroup);
            for (uint32_t i = g; i < end; ++i)
                for (void *base : {layers[i].k_pool, layers[i].v_pool}) pools.push_back({base, rows * layers[0].head_dim});
            for (uint32_t i = g; i < end; ++i)
                for (float *base : {layers[i].k_scales, layers[i].v_scales}) pools.push_back({base, rows * 4});
        }
        for (const PoolRef &r : pools)
            if ((st = check_pool(ctx, r, "move pages (8-bit)")) != MF_OK) return st;
        return move_pages(ctx, pools, layers[0].n_pages, src, dst, n, "move pages (8-bit)");
    } catch (const std::bad_alloc &) {
        return fail(ctx, MF_ERR_OUT_OF_MEMORY, "move pages (8-bit): host memory");
    }
}

}  // extern "C"
