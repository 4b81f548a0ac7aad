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

constexpr uint32_t kMovePools = 64;    // pools per launch
constexpr uint32_t kMovePairs = 256;   // pairs per launch

struct MoveParams {
    uint4 *pool[kMovePools];
    uint32_t chunks[kMovePools];  // 16-byte units of a page in this pool
    uint32_t src[kMovePairs], dst[kMovePairs];
};

// blockIdx: (pair, pool)
__global__ void __launch_bounds__(256) move_pages_kernel(const __grid_constant__ MoveParams p)
{
    const uint32_t n = p.chunks[blockIdx.y];
    uint4 *pool = p.pool[blockIdx.y];
    const uint4 *src = pool + (size_t)p.src[blockIdx.x] * n;
    uint4 *dst = pool + (size_t)p.dst[blockIdx.x] * n;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) dst[i] = src[i];
}

struct PoolRef {
    void *base;
    uint64_t page_bytes;
};

mf_status move_pages(MfContext *ctx, const std::vector<PoolRef> &pools, uint32_t n_pages, const uint32_t *src, const uint32_t *dst,
                     uint32_t n, const char *what)
{
    // Destinations are distinct and no source is one: the copies may then run in any order.
    std::vector<uint8_t> seen(n_pages, 0);
    for (uint32_t i = 0; i < n; ++i) {
        if (src[i] >= n_pages || dst[i] >= n_pages)
            return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: pair %u (%u -> %u) outside the pool of %u pages", what, i, src[i], dst[i], n_pages);
        if (seen[dst[i]]) return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: page %u is written twice", what, dst[i]);
        seen[dst[i]] = 1;
    }
    for (uint32_t i = 0; i < n; ++i)
        if (seen[src[i]]) return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: page %u is read and written", what, src[i]);
    DeviceScope scope(ctx->device);
    for (size_t p0 = 0; p0 < pools.size(); p0 += kMovePools)
        for (uint32_t i0 = 0; i0 < n; i0 += kMovePairs) {
            MoveParams p;
            const uint32_t np = (uint32_t)std::min<size_t>(kMovePools, pools.size() - p0), ni = std::min(kMovePairs, n - i0);
            for (uint32_t j = 0; j < np; ++j) {
                p.pool[j] = static_cast<uint4 *>(pools[p0 + j].base);
                p.chunks[j] = (uint32_t)(pools[p0 + j].page_bytes / 16);
            }
            std::copy(src + i0, src + i0 + ni, p.src);
            std::copy(dst + i0, dst + i0 + ni, p.dst);
            move_pages_kernel<<<dim3(ni, np), 256, 0, ctx->stream>>>(p);
            const mf_status st = check_launch(ctx, "move_pages_kernel");
            if (st != MF_OK) return st;
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
        for (uint32_t i = 0; i < n_layers; ++i) {
            if (!layers[i].k_scales || !layers[i].v_scales)
                return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "move pages (8-bit): scales of layer %u", i);
            for (void *base : {layers[i].k_pool, layers[i].v_pool}) pools.push_back({base, rows * layers[0].head_dim});
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
