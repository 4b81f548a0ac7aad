// Append of a ragged batch of new tokens to a paged cache (f16 or 8-bit) with rotary positions on several axes.
//
// Frequency j of a head turns by row positions[axis[j]][t] of the cos / sin tables; the cache row of a token counts
// tokens, not positions.  Products and sums in f32 from f16 operands, one rounding to f16 (append.cuh); the 8-bit
// cache quantises the rounded K row and the V row: scale = max|x| / 448, byte = e4m3(x / scale).
//
// One warp per (token, head slot).
#include <cuda_fp8.h>

#include "append.cuh"
#include "internal.hpp"

namespace mf {
namespace {

struct MropeParams {
    const __half *q, *k, *v;
    __half *q_rot;
    void *k_pool, *v_pool;
    float *k_scales, *v_scales;
    const __half *cos_t, *sin_t;
    const uint32_t *positions, *q_begin, *page_table, *kv_lens;
    uint32_t *status;
    uint64_t q_stride, k_stride, v_stride, q_rot_stride;
    uint32_t tokens, batch, n_heads, n_kv_heads, head_dim, page_size, pt_stride, n_pages, pos_stride, table_rows, rope_mode;
    uint8_t axis[64];
};

// Byte of (row r of the page, dim d) in the dim-major 16-key blocks of a V page of 128-wide heads.
__device__ __forceinline__ uint32_t v_block_offset(uint32_t r, uint32_t d) { return (r / 16) * 2048 + d * 16 + r % 16; }

template <bool K8>
__global__ void __launch_bounds__(256) mrope_append_kernel(const __grid_constant__ MropeParams p)
{
    const uint32_t lane = threadIdx.x & 31, D = p.head_dim;
    const uint64_t wid = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const uint32_t q_slots = p.q_rot ? p.n_heads : 0, slots = q_slots + 2 * p.n_kv_heads;
    if (wid >= (uint64_t)p.tokens * slots) return;
    const uint32_t t = (uint32_t)(wid / slots), slot = (uint32_t)(wid % slots);
    const bool is_q = slot < q_slots, is_v = slot >= q_slots + p.n_kv_heads;
    const uint32_t head = is_q ? slot : (is_v ? slot - q_slots - p.n_kv_heads : slot - q_slots);
    const __half *src = is_q ? p.q + t * p.q_stride + head * D : is_v ? p.v + t * p.v_stride + head * D : p.k + t * p.k_stride + head * D;
    __half x[2], y[2];
    __half a[2][2];  // pairs lane and lane + 32: (first, second)
    const uint32_t half = D / 2;
    auto dim = [&](uint32_t pr, uint32_t second) { return p.rope_mode == MF_ROPE_MODE_NEOX ? pr + second * half : 2 * pr + second; };
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t pr = lane + 32 * i;
        a[i][0] = a[i][1] = __float2half_rn(0.f);
        if (pr >= half) continue;
        x[0] = src[dim(pr, 0)];
        x[1] = src[dim(pr, 1)];
        y[0] = x[0];
        y[1] = x[1];
        if (!is_v) {
            const uint32_t row = p.positions[(size_t)p.axis[pr] * p.pos_stride + t];
            if (row >= p.table_rows) {
                atomicOr(p.status, kStatusBadPage);
            } else {
                const float c = __half2float(p.cos_t[(size_t)row * half + pr]), s = __half2float(p.sin_t[(size_t)row * half + pr]);
                y[0] = rot_first(__half2float(x[0]), __half2float(x[1]), c, s);
                y[1] = rot_second(__half2float(x[0]), __half2float(x[1]), c, s);
            }
        }
        a[i][0] = y[0];
        a[i][1] = y[1];
    }
    if (is_q) {
        __half *dst = p.q_rot + t * p.q_rot_stride + head * D;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (lane + 32 * i < half) {
                dst[dim(lane + 32 * i, 0)] = a[i][0];
                dst[dim(lane + 32 * i, 1)] = a[i][1];
            }
        return;
    }
    // the sequence whose tokens hold t, and the token's row in its cache
    uint32_t lo = 0, hi = p.batch;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (p.q_begin[mid] <= t) lo = mid;
        else hi = mid;
    }
    const uint32_t behind = p.q_begin[lo + 1] - t, len = p.kv_lens[lo];
    uint32_t page = 0xFFFFFFFFu, row = 0;
    if (t < p.q_begin[lo + 1] && behind <= len && (len - behind) / p.page_size < p.pt_stride) {
        row = len - behind;
        page = p.page_table[(size_t)lo * p.pt_stride + row / p.page_size];
        row %= p.page_size;
    }
    if (page >= p.n_pages) {
        if (lane == 0) atomicOr(p.status, kStatusBadPage);
        return;
    }
    const size_t run = ((size_t)page * p.n_kv_heads + head) * p.page_size;  // first row of the (page, kv head) run
    if (!K8) {
        __half *dst = static_cast<__half *>(is_v ? p.v_pool : p.k_pool) + (run + row) * D;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (lane + 32 * i < half) {
                dst[dim(lane + 32 * i, 0)] = a[i][0];
                dst[dim(lane + 32 * i, 1)] = a[i][1];
            }
        return;
    }
    float amax = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) amax = fmaxf(amax, fmaxf(fabsf(__half2float(a[i][0])), fabsf(__half2float(a[i][1]))));
#pragma unroll
    for (uint32_t o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = amax > 0.f ? __fdiv_rn(amax, 448.f) : 1.f;
    uint8_t *dst = static_cast<uint8_t *>(is_v ? p.v_pool : p.k_pool) + run * D;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s) {
            const uint32_t d = dim(lane + 32 * i, s);
            dst[is_v ? v_block_offset(row, d) : row * D + d] =
                (uint8_t)__nv_cvt_float_to_fp8(__fdiv_rn(__half2float(a[i][s]), scale), __NV_SATFINITE, __NV_E4M3);
        }
    if (lane == 0) (is_v ? p.v_scales : p.k_scales)[run + row] = scale;
}

template <class Cache>
mf_status mrope_params(MfContext *ctx, const Cache *c, const MfMropeAppendArgs *a, MropeParams &p, const char *what)
{
    if (!c || !c->k_pool || !c->v_pool || !c->page_table || !c->kv_lens || !a || !a->cos || !a->sin || !a->q_begin ||
        (a->tokens && (!a->k || !a->v || !a->positions)))
        return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "%s: null input", what);
    if (a->tokens && a->q_rot && !a->q) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "%s: q_rot without q", what);
    if (c->batch == 0 || c->n_kv_heads == 0 || c->page_size == 0 || c->n_pages == 0 || (a->q_rot && a->n_heads == 0))
        return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: batch %u, n_heads %u, n_kv_heads %u, page_size %u, %u pages", what, c->batch,
                    a->n_heads, c->n_kv_heads, c->page_size, c->n_pages);
    if (a->rope_mode > 1) return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: rope_mode %u", what, a->rope_mode);
    if (a->n_axes == 0 || a->n_axes > MF_MAX_ROPE_AXES) return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: %u axes", what, a->n_axes);
    for (uint32_t j = 0; j < c->head_dim / 2; ++j)
        if (a->axis[j] >= a->n_axes)
            return fail(ctx, MF_ERR_INVALID_OPERATION, "%s: frequency %u on axis %u of %u", what, j, a->axis[j], a->n_axes);
    if (a->position_stride < a->tokens)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: %u positions an axis for %u tokens", what, a->position_stride, a->tokens);
    if (a->table_rows == 0) return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: empty cos / sin tables", what);
    if (((a->q_rot ? a->q_stride | a->q_rot_stride : 0) | a->k_stride | a->v_stride) & 7u)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: strides must be multiples of 8 elements", what);
    const void *ptrs[] = {a->q_rot ? a->q : nullptr, a->k, a->v, a->q_rot, a->cos, a->sin, c->k_pool, c->v_pool};
    for (const void *x : ptrs)
        if (reinterpret_cast<uintptr_t>(x) & 15u) return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: tensors must be 16-byte aligned", what);
    p.q = static_cast<const __half *>(a->q);
    p.k = static_cast<const __half *>(a->k);
    p.v = static_cast<const __half *>(a->v);
    p.q_rot = static_cast<__half *>(a->q_rot);
    p.k_pool = c->k_pool;
    p.v_pool = c->v_pool;
    p.cos_t = static_cast<const __half *>(a->cos);
    p.sin_t = static_cast<const __half *>(a->sin);
    p.positions = a->positions;
    p.q_begin = a->q_begin;
    p.page_table = c->page_table;
    p.kv_lens = c->kv_lens;
    p.status = ctx->d_status;
    p.q_stride = a->q_stride;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.q_rot_stride = a->q_rot_stride;
    p.tokens = a->tokens;
    p.batch = c->batch;
    p.n_heads = a->n_heads;
    p.n_kv_heads = c->n_kv_heads;
    p.head_dim = c->head_dim;
    p.page_size = c->page_size;
    p.pt_stride = c->page_table_stride;
    p.n_pages = c->n_pages;
    p.pos_stride = a->position_stride;
    p.table_rows = a->table_rows;
    p.rope_mode = a->rope_mode;
    for (uint32_t j = 0; j < 64; ++j) p.axis[j] = a->axis[j];
    return MF_OK;
}

template <bool K8>
mf_status launch_mrope(MfContext *ctx, const MropeParams &p, const char *what)
{
    if (p.tokens == 0) return MF_OK;
    const uint64_t warps = (uint64_t)p.tokens * ((p.q_rot ? p.n_heads : 0) + 2 * (uint64_t)p.n_kv_heads);
    if ((warps + 7) / 8 > 0x7FFFFFFFull) return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: %u tokens", what, p.tokens);
    DeviceScope scope(ctx->device);
    mrope_append_kernel<K8><<<(uint32_t)((warps + 7) / 8), 256, 0, ctx->stream>>>(p);
    return check_launch(ctx, "mrope_append_kernel");
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" {

mf_status mf_paged_mrope_append(MfContext *ctx, const MfPagedKv *c, const MfMropeAppendArgs *a)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (c && (c->head_dim != 64 && c->head_dim != 128))
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "mrope append: head_dim %u (64 or 128)", c->head_dim);
    MropeParams p{};
    const mf_status st = mrope_params(ctx, c, a, p, "mrope append");
    return st != MF_OK ? st : launch_mrope<false>(ctx, p, "mrope append");
}

mf_status mf_paged_kv8_mrope_append(MfContext *ctx, const MfPagedKv8 *c, const MfMropeAppendArgs *a)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (c && c->head_dim != 128)
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "mrope append (8-bit): the 8-bit cache supports head_dim 128, got %u", c->head_dim);
    if (c && (c->page_size < 16 || c->page_size > 64 || (c->page_size & (c->page_size - 1))))
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "mrope append (8-bit): page_size %u (16, 32 or 64)", c->page_size);
    MropeParams p{};
    const mf_status st = mrope_params(ctx, c, a, p, "mrope append (8-bit)");
    if (st != MF_OK) return st;
    if (!c->k_scales || !c->v_scales) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "mrope append (8-bit): scales");
    p.k_scales = c->k_scales;
    p.v_scales = c->v_scales;
    return launch_mrope<true>(ctx, p, "mrope append (8-bit)");
}

}  // extern "C"
