// Attention of a ragged batch of new tokens over a paged cache: causal, optionally with a sliding window and
// first tokens that stay visible (sinks).
//
//   out[t, h] = sum_k w_k V[k] / sum_k w_k,   w_k = exp(scale * q[t, h] . K[k] - max_k),   k visible to t
//
// One warp per (token, query head) walks the visible keys with a running maximum and sum (f32), every lane
// holding D / 32 dims of q and of the accumulator.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "internal.hpp"
#include "ptx.cuh"

struct MfChunkPlan {
    uint32_t batch = 0, n_heads = 0, n_kv_heads = 0, head_dim = 0, page_size = 0, window = 0, n_sinks = 0;
    uint32_t max_tokens = 0, tokens = 0, max_pages = 0;
    int device = 0;
    uint32_t *d_meta = nullptr;  // [batch + 1] q_begin, [batch] kv_lens
    uint32_t *pinned[2] = {nullptr, nullptr};
    cudaEvent_t staged[2] = {nullptr, nullptr};
    uint32_t next_stage = 0;
};

namespace mf {
namespace {

constexpr uint32_t kMaxGroup = 64;
constexpr uint32_t kMaxLen = 1u << 30;  // positions and tile arithmetic stay inside 32 bits

struct ChunkParams {
    const __half *q;
    __half *out;
    const __half *k_pool, *v_pool;
    const uint32_t *page_table, *q_begin, *kv_lens;
    uint32_t *status;
    uint64_t q_stride_t, q_stride_h, out_stride_t, out_stride_h;
    uint32_t batch, n_heads, n_kv_heads, group, page_size, pt_stride, n_pages, window, n_sinks;
    float scale_log2;
};

template <uint32_t D>
__global__ void __launch_bounds__(256) chunk_rows_kernel(const ChunkParams p)
{
    constexpr uint32_t E = D / 32;  // dims per lane: [lane * E, lane * E + E)
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t wid = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const uint32_t h = (uint32_t)(wid % p.n_heads);
    const uint64_t t = wid / p.n_heads;
    if (t >= p.q_begin[p.batch]) return;
    uint32_t lo = 0, hi = p.batch;  // the sequence whose tokens hold t
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (p.q_begin[mid] <= t) lo = mid;
        else hi = mid;
    }
    const uint32_t b = lo, kvh = h / p.group;
    const int64_t pos = (int64_t)p.kv_lens[b] - (p.q_begin[b + 1] - t);
    float q[E], acc[E];
    const __half *qp = p.q + t * p.q_stride_t + h * p.q_stride_h + lane * E;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        q[e] = __half2float(qp[e]);
        acc[e] = 0.f;
    }
    float m = -1e30f, l = 0.f;
    const uint32_t *table = p.page_table + (size_t)b * p.pt_stride;
    auto walk = [&](int64_t k0, int64_t k1) {
        for (int64_t k = k0; k < k1; ++k) {
            const uint32_t page = table[k / p.page_size];
            if (page >= p.n_pages) {
                if (lane == 0) atomicOr(p.status, kStatusBadPage);
                continue;
            }
            const size_t row = (((size_t)page * p.n_kv_heads + kvh) * p.page_size + k % p.page_size) * D + lane * E;
            float s = 0.f;
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) s = fmaf(q[e], __half2float(p.k_pool[row + e]), s);
#pragma unroll
            for (uint32_t o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            s *= p.scale_log2;
            const float m_new = fmaxf(m, s), a = exp2f(m - m_new), w = exp2f(s - m_new);
            l = l * a + w;
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) acc[e] = fmaf(w, __half2float(p.v_pool[row + e]), acc[e] * a);
            m = m_new;
        }
    };
    const int64_t first = p.window ? (pos - (int64_t)p.window + 1 > 0 ? pos - (int64_t)p.window + 1 : 0) : 0;
    walk(0, min((int64_t)p.n_sinks, first));
    walk(first, pos + 1);
    const float inv = l != 0.f ? 1.f / l : 0.f;
    __half *op = p.out + t * p.out_stride_t + h * p.out_stride_h + lane * E;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) op[e] = __float2half_rn(acc[e] * inv);
}

mf_status check_lens(MfContext *ctx, const uint32_t *q_lens, const uint32_t *kv_lens, uint32_t batch, uint64_t *tokens,
                     uint32_t *max_kv)
{
    *tokens = 0;
    *max_kv = 0;
    for (uint32_t b = 0; b < batch; ++b) {
        if (q_lens[b] > kMaxLen || kv_lens[b] > kMaxLen)
            return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: sequence %u has %u new tokens and %u keys (limit %u)", b,
                        q_lens[b], kv_lens[b], kMaxLen);
        *tokens += q_lens[b];
        *max_kv = std::max(*max_kv, q_lens[b] ? kv_lens[b] : 0u);
    }
    if (*tokens > kMaxLen) return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: %llu new tokens", (unsigned long long)*tokens);
    return MF_OK;
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" {

void mf_chunk_plan_destroy(MfContext *ctx, MfChunkPlan *pl)
{
    if (!pl) return;
    DeviceScope scope(pl->device);
    if (ctx) cudaStreamSynchronize(ctx->stream);
    for (int i = 0; i < 2; ++i) {
        if (pl->staged[i]) cudaEventDestroy(pl->staged[i]);
        if (pl->pinned[i]) cudaFreeHost(pl->pinned[i]);
    }
    if (pl->d_meta) cudaFree(pl->d_meta);
    delete pl;
}

mf_status mf_chunk_plan_update(MfContext *ctx, MfChunkPlan *pl, const uint32_t *q_lens, const uint32_t *kv_lens)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (!pl || !q_lens || !kv_lens) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "chunk plan: null input");
    DeviceScope scope(ctx->device);
    uint64_t tokens;
    uint32_t max_kv;
    mf_status st = check_lens(ctx, q_lens, kv_lens, pl->batch, &tokens, &max_kv);
    if (st != MF_OK) return st;
    if (tokens > pl->max_tokens)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: %llu new tokens, made for %u", (unsigned long long)tokens, pl->max_tokens);
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if ((st = check_cuda(ctx, cudaStreamIsCapturing(ctx->stream, &cap), "cudaStreamIsCapturing")) != MF_OK) return st;
    if (cap != cudaStreamCaptureStatusNone)
        return fail(ctx, MF_ERR_INVALID_OPERATION, "chunk plan: no update while the stream is being captured");
    const uint32_t s = pl->next_stage;
    if ((st = check_cuda(ctx, cudaEventSynchronize(pl->staged[s]), "chunk plan: staging")) != MF_OK) return st;
    uint32_t *w = pl->pinned[s];
    w[0] = 0;
    for (uint32_t b = 0; b < pl->batch; ++b) w[b + 1] = w[b] + q_lens[b];
    for (uint32_t b = 0; b < pl->batch; ++b) w[pl->batch + 1 + b] = kv_lens[b];
    st = check_cuda(ctx, cudaMemcpyAsync(pl->d_meta, w, 4 * (2 * (size_t)pl->batch + 1), cudaMemcpyHostToDevice, ctx->stream),
                    "chunk plan: upload");
    if (st != MF_OK) return st;
    if ((st = check_cuda(ctx, cudaEventRecord(pl->staged[s], ctx->stream), "chunk plan: upload")) != MF_OK) return st;
    pl->next_stage = s ^ 1;
    pl->tokens = (uint32_t)tokens;
    pl->max_pages = (max_kv + pl->page_size - 1) / pl->page_size;
    return MF_OK;
}

mf_status mf_chunk_plan_create(MfContext *ctx, const uint32_t *q_lens, const uint32_t *kv_lens, uint32_t batch, uint32_t n_heads,
                               uint32_t n_kv_heads, uint32_t head_dim, uint32_t page_size, uint32_t window, uint32_t n_sinks,
                               uint32_t max_tokens, MfChunkPlan **out)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (!q_lens || !kv_lens || !out) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "chunk plan: null input");
    *out = nullptr;
    if (batch == 0 || n_kv_heads == 0 || n_heads == 0 || n_heads % n_kv_heads != 0)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: batch %u, n_heads %u, n_kv_heads %u", batch, n_heads, n_kv_heads);
    if (head_dim != 64 && head_dim != 128)
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "chunk plan: head_dim %u (64 or 128)", head_dim);
    if (n_heads / n_kv_heads > kMaxGroup)
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "chunk plan: group size %u > %u", n_heads / n_kv_heads, kMaxGroup);
    if (page_size < 8 || page_size > 128 || (page_size & (page_size - 1)))
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "chunk plan: page_size %u (8, 16, 32, 64 or 128)", page_size);
    if (n_sinks && !window) return fail(ctx, MF_ERR_INVALID_OPERATION, "chunk plan: %u sinks without a window", n_sinks);
    uint64_t tokens;
    uint32_t max_kv;
    mf_status st = check_lens(ctx, q_lens, kv_lens, batch, &tokens, &max_kv);
    if (st != MF_OK) return st;
    if (max_tokens > kMaxLen) return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: max_tokens %u", max_tokens);
    DeviceScope scope(ctx->device);
    MfChunkPlan *pl = new (std::nothrow) MfChunkPlan();
    if (!pl) return fail(ctx, MF_ERR_OUT_OF_MEMORY, "chunk plan");
    pl->batch = batch;
    pl->n_heads = n_heads;
    pl->n_kv_heads = n_kv_heads;
    pl->head_dim = head_dim;
    pl->page_size = page_size;
    pl->window = window;
    pl->n_sinks = n_sinks;
    pl->max_tokens = max_tokens ? max_tokens : (uint32_t)tokens;
    pl->device = ctx->device;
    cudaError_t e = cudaSuccess;
    auto ok = [&](cudaError_t r) {
        if (e == cudaSuccess) e = r;
    };
    const size_t words = 2 * (size_t)batch + 1;
    for (int i = 0; i < 2; ++i) {
        ok(cudaMallocHost(reinterpret_cast<void **>(&pl->pinned[i]), 4 * words));
        ok(cudaEventCreateWithFlags(&pl->staged[i], cudaEventDisableTiming));
    }
    ok(cudaMalloc(reinterpret_cast<void **>(&pl->d_meta), 4 * words));
    st = e == cudaSuccess ? mf_chunk_plan_update(ctx, pl, q_lens, kv_lens) : check_cuda(ctx, e, "chunk plan allocation");
    if (st != MF_OK) {
        mf_chunk_plan_destroy(ctx, pl);
        return st;
    }
    *out = pl;
    return MF_OK;
}

uint32_t mf_chunk_plan_tokens(const MfChunkPlan *pl) { return pl ? pl->tokens : 0; }

mf_status mf_paged_chunk_attention(MfContext *ctx, const MfChunkPlan *pl, const MfPagedKv *c, const MfPagedChunkArgs *a)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (!pl || !c || !c->k_pool || !c->v_pool || !c->page_table || !a || (pl->tokens && (!a->q || !a->out)))
        return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "paged chunk attention: null input");
    if (c->batch != pl->batch || c->n_kv_heads != pl->n_kv_heads || c->head_dim != pl->head_dim || c->page_size != pl->page_size)
        return fail(ctx, MF_ERR_INVALID_SHAPE,
                    "paged chunk attention: the cache (batch %u, %u kv heads, head_dim %u, pages of %u) is not the plan's (%u, %u, %u, %u)",
                    c->batch, c->n_kv_heads, c->head_dim, c->page_size, pl->batch, pl->n_kv_heads, pl->head_dim, pl->page_size);
    if (pl->device != ctx->device) return fail(ctx, MF_ERR_INVALID_OPERATION, "paged chunk attention: the plan is another device's");
    if (pl->max_pages > c->page_table_stride)
        return fail(ctx, MF_ERR_INVALID_OPERATION, "paged chunk attention: %u pages exceed the page table's %u", pl->max_pages,
                    c->page_table_stride);
    if (c->n_pages == 0 || (uint64_t)c->n_pages * c->n_kv_heads >= (1ull << 31))
        return fail(ctx, MF_ERR_INVALID_SHAPE, "paged chunk attention: %u pages of %u kv heads", c->n_pages, c->n_kv_heads);
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(c->k_pool) |
         reinterpret_cast<uintptr_t>(c->v_pool)) & 15u)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "paged chunk attention: q, out and the pools must be 16-byte aligned");
    if ((a->q_stride_t | a->q_stride_h | a->out_stride_t | a->out_stride_h) & 7u)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "paged chunk attention: strides must be multiples of 8 elements");
    if (!(a->scale >= 0.f) || !std::isfinite(a->scale))
        return fail(ctx, MF_ERR_INVALID_OPERATION, "paged chunk attention: scale %g", (double)a->scale);
    if (pl->max_tokens == 0 || !a->q || !a->out) return MF_OK;
    DeviceScope scope(ctx->device);
    ChunkParams p{};
    p.q = static_cast<const __half *>(a->q);
    p.out = static_cast<__half *>(a->out);
    p.k_pool = static_cast<const __half *>(c->k_pool);
    p.v_pool = static_cast<const __half *>(c->v_pool);
    p.page_table = c->page_table;
    p.q_begin = pl->d_meta;
    p.kv_lens = pl->d_meta + pl->batch + 1;
    p.status = ctx->d_status;
    p.q_stride_t = a->q_stride_t;
    p.q_stride_h = a->q_stride_h;
    p.out_stride_t = a->out_stride_t;
    p.out_stride_h = a->out_stride_h;
    p.batch = pl->batch;
    p.n_heads = pl->n_heads;
    p.n_kv_heads = pl->n_kv_heads;
    p.group = pl->n_heads / pl->n_kv_heads;
    p.page_size = pl->page_size;
    p.pt_stride = c->page_table_stride;
    p.n_pages = c->n_pages;
    p.window = pl->window;
    p.n_sinks = pl->n_sinks;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    const uint64_t blocks = ((uint64_t)pl->max_tokens * pl->n_heads + 7) / 8;
    if (blocks > 0x7FFFFFFFull) return fail(ctx, MF_ERR_INVALID_SHAPE, "paged chunk attention: %u tokens", pl->max_tokens);
    if (pl->head_dim == 128) chunk_rows_kernel<128><<<(uint32_t)blocks, 256, 0, ctx->stream>>>(p);
    else chunk_rows_kernel<64><<<(uint32_t)blocks, 256, 0, ctx->stream>>>(p);
    return check_launch(ctx, "chunk_rows_kernel");
}

}  // extern "C"
