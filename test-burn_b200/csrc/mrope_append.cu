// Append of a ragged batch of new tokens to a paged cache (f16 or 8-bit) with rotary positions on several axes.
//
// Frequency j of a head turns by row positions[axis[j]][t] of the cos / sin tables; the cache row of a token counts
// tokens, not positions.  Products and sums in f32 from f16 operands, one rounding to f16 (append.cuh); the 8-bit
// cache quantises the rounded K row and the V row: scale = max|x| / 448, byte = e4m3(x / scale).
//
// Bound by HBM: every row is read once and written once.  A CTA has the new tokens of one sequence that fall into one
// aligned block of cache rows (8 rows; 16 for the 8-bit cache, whose V bytes lie in 16-row blocks): it gathers the cos /
// sin rows of its tokens into shared memory once for all heads, and finds its sequence once.  A thread turns two 16-byte
// chunks at a time (append.cuh), several in flight.  V bytes of the 8-bit cache are transposed through shared memory: a
// whole block goes out as 16-byte words, a part of one byte by byte.
//
// Measured: 8.5k tokens of 32/8 heads of 128 (210 MB) 39.4 us, 5.3 TB/s, 0.81 of the copy rate; 4.8k tokens of 16/2 heads
// into the 8-bit cache (47 MB) 17 us - two thirds of it launch, the chain of loads before a CTA's first row (sequence,
// page, positions, tables) and the drain; one token of each of 64 sequences 3.3 us.
#include <cuda_fp8.h>

#include <algorithm>

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
    uint32_t slots_per_part;  // head slots a CTA takes
    uint8_t axis[64];
};

// scale of the 128-wide row whose chunk pairs eight neighbouring threads hold; every lane of the warp takes part
__device__ __forceinline__ float row_scale(const Chunk &a, const Chunk &c, bool live)
{
    float amax = 0.f;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(fabsf(__half2float(a.h[e])), fabsf(__half2float(c.h[e]))));
    if (!live) amax = 0.f;
#pragma unroll
    for (uint32_t o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    return amax > 0.f ? __fdiv_rn(amax, 448.f) : 1.f;
}
__device__ __forceinline__ uint2 bytes_of(const Chunk &x, float scale)
{
    union {
        uint2 u;
        uint8_t b[8];
    } r;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) r.b[e] = (uint8_t)__nv_cvt_float_to_fp8(__fdiv_rn(__half2float(x.h[e]), scale), __NV_SATFINITE, __NV_E4M3);
    return r.u;
}

constexpr uint32_t kThreads = 256;
__host__ __device__ constexpr uint32_t in_flight(bool k8) { return k8 ? 2 : 3; }  // chunk pairs a thread has in flight
constexpr uint32_t kVHeads = 8;     // 8-bit V: kv heads transposed at a time

// First block index of sequence b.  The tokens [q_begin[b], q_begin[b + 1]) touch at most (their number) / R + 2 aligned
// blocks of R cache rows, and these starts are at least that far apart, whatever the lengths are.
__host__ __device__ __forceinline__ uint64_t first_block(uint64_t begin, uint32_t b, uint32_t rows) { return begin / rows + 3ull * b; }

// blockIdx: (block of rows, part of the head slots); the last part of the 8-bit form has the V rows.
template <uint32_t D, bool K8>
__global__ void __launch_bounds__(kThreads, 5) mrope_append_kernel(const __grid_constant__ MropeParams p)
{
    constexpr uint32_t R = K8 ? 16 : 8, half = D / 2, cpr = D / 16;  // cpr: chunk pairs per head row
    __shared__ __align__(16) __half cos_s[R * half], sin_s[R * half];
    __shared__ uint4 found_s;  // sequence, its tokens [y, z), its length
    __shared__ __align__(16) uint8_t v_s[K8 ? kVHeads * 128 * 16 : 16];
    const uint32_t tid = threadIdx.x;
    // The sequence whose blocks hold this one, found by the thread that looks at it (a binary search would be a chain of
    // loads, most of a decode step's launch).
    if (tid == 0) found_s = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (uint32_t b = tid; b < p.batch; b += kThreads) {
        const uint32_t b0 = __ldg(p.q_begin + b), b1 = min(__ldg(p.q_begin + b + 1), p.tokens), kv = __ldg(p.kv_lens + b);
        const uint64_t mine = first_block(b0, b, R);
        if (b0 < b1 && mine <= blockIdx.x && blockIdx.x - mine <= (b1 - b0) / R + 1) found_s = make_uint4(b, b0, b1, kv);
    }
    __syncthreads();
    const uint32_t lo = found_s.x, begin = found_s.y, end = found_s.z, len = found_s.w;
    if (begin >= end) return;
    const uint32_t n_new = end - begin, which = blockIdx.x - (uint32_t)first_block(begin, lo, R);
    // Cache rows of this block's tokens.  A sequence shorter than its new tokens has no row for them: they are reported,
    // their q is turned all the same (row numbers count from there).
    const bool has_rows = n_new <= len;
    const uint32_t start = has_rows ? len - n_new : 0, row0 = (start / R + which) * R;
    const uint32_t first = max(row0, start), last = min(row0 + R, start + n_new);  // rows [first, last)
    if (first >= last) return;
    const uint32_t n_tok = last - first, t0 = begin + (first - start);
    const bool in_table = has_rows && first / p.page_size < p.pt_stride;
    const uint32_t page = in_table ? __ldg(p.page_table + (size_t)lo * p.pt_stride + first / p.page_size) : 0xFFFFFFFFu;
    const uint32_t in_page = first % p.page_size;
    const uint32_t q_slots = p.q_rot ? p.n_heads : 0;
    const uint32_t slots = q_slots + (K8 ? p.n_kv_heads : 2 * p.n_kv_heads);  // 8-bit V rows take their own way below
    const uint32_t part0 = blockIdx.y * p.slots_per_part, width = part0 < slots ? min(p.slots_per_part, slots - part0) : 0;
    // Pair x of the part: chunk j = x % cpr of slot part0 + (x / cpr) % width of token x / cpr / width.  A thread's pairs
    // are kThreads apart: j stays, (token, slot) advance without a division.
    const uint32_t j = tid % cpr, rows = n_tok * width;
    struct At {
        uint32_t row, tok, slot;
    };
    auto advance = [&](At &at) {
        at.row += kThreads / cpr;
        at.slot += kThreads / cpr;
        while (at.slot >= width && at.row < rows) at.slot -= width, ++at.tok;
    };
    At in{tid / cpr, 0, tid / cpr};
    while (in.slot >= width && in.row < rows) in.slot -= width, ++in.tok;
    At out = in;
    constexpr uint32_t kInFlight = in_flight(K8);
    Chunk a[kInFlight], c[kInFlight];
    auto fetch = [&]() {
#pragma unroll
        for (uint32_t u = 0; u < kInFlight; ++u, advance(in)) {
            if (in.row >= rows) continue;
            const uint64_t t = t0 + in.tok;
            const uint32_t slot = part0 + in.slot;
            const __half *src = slot < q_slots ? p.q + t * p.q_stride + slot * D
                                : slot < q_slots + p.n_kv_heads ? p.k + t * p.k_stride + (slot - q_slots) * D
                                                                : p.v + t * p.v_stride + (slot - q_slots - p.n_kv_heads) * D;
            a[u].u = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * j));
            c[u].u = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * j + half));
        }
    };
    fetch();  // on their way while the tables are gathered
    for (uint32_t x = tid; x < (width ? n_tok * half : 0); x += kThreads) {
        const uint32_t tok = x / half, j = x - tok * half;
        const uint32_t row = __ldg(p.positions + (size_t)p.axis[j] * p.pos_stride + t0 + tok);
        __half cv = __float2half_rn(1.f), sv = __float2half_rn(0.f);
        if (row < p.table_rows) {
            cv = p.cos_t[(size_t)row * half + j];
            sv = p.sin_t[(size_t)row * half + j];
        } else {
            atomicOr(p.status, kStatusBadPage);  // left as it is
        }
        cos_s[tok * half + j] = cv;
        sin_s[tok * half + j] = sv;
    }
    const bool store = page < p.n_pages;
    const size_t run = (size_t)page * p.n_kv_heads * p.page_size + in_page;  // row `first` of kv head 0 in its page
    if (!store && tid == 0) atomicOr(p.status, kStatusBadPage);
    __syncthreads();
    for (uint32_t r0 = 0; r0 < rows; r0 += kInFlight * (kThreads / cpr)) {
        if (r0) fetch();
#pragma unroll
        for (uint32_t u = 0; u < kInFlight; ++u, advance(out)) {
            const bool live = out.row < rows;
            if (!K8 && !live) continue;
            const uint32_t tok = out.tok, slot = part0 + out.slot;
            const bool is_q = slot < q_slots, is_v = slot >= q_slots + p.n_kv_heads;
            if (live && !is_v) rope_chunks(a[u], c[u], cos_s + tok * half, sin_s + tok * half, j, D, p.rope_mode);
            if (live && is_q) {
                __half *dst = p.q_rot + (t0 + (uint64_t)tok) * p.q_rot_stride + slot * D;
                *reinterpret_cast<uint4 *>(dst + 8 * j) = a[u].u;
                *reinterpret_cast<uint4 *>(dst + 8 * j + half) = c[u].u;
            }
            const uint32_t head = is_v ? slot - q_slots - p.n_kv_heads : slot - q_slots;
            if (!K8) {
                if (!is_q && store) {
                    __half *dst = static_cast<__half *>(is_v ? p.v_pool : p.k_pool) + (run + (size_t)head * p.page_size + tok) * D;
                    *reinterpret_cast<uint4 *>(dst + 8 * j) = a[u].u;
                    *reinterpret_cast<uint4 *>(dst + 8 * j + half) = c[u].u;
                }
            } else {
                // the eight threads of a row sit side by side
                if (!__any_sync(0xffffffffu, live && !is_q)) continue;
                const float scale = row_scale(a[u], c[u], live);
                if (live && !is_q && store) {
                    uint8_t *dst = static_cast<uint8_t *>(p.k_pool) + (run + (size_t)head * p.page_size + tok) * 128;
                    *reinterpret_cast<uint2 *>(dst + 8 * j) = bytes_of(a[u], scale);
                    *reinterpret_cast<uint2 *>(dst + 8 * j + 64) = bytes_of(c[u], scale);
                    if (j == 0) p.k_scales[run + (size_t)head * p.page_size + tok] = scale;
                }
            }
        }
    }
    if constexpr (K8) {
        if (!store || width) return;
        // 8-bit V: [kv head][dim][16 rows of the block]
        for (uint32_t h0 = 0; h0 < p.n_kv_heads; h0 += kVHeads) {
            const uint32_t heads = min(kVHeads, p.n_kv_heads - h0), pairs = n_tok * heads * 8;
            if (h0) __syncthreads();
            for (uint32_t x0 = 0; x0 < pairs; x0 += kThreads) {
                const uint32_t x = x0 + tid;
                const bool live = x < pairs;
                const uint32_t j = x % 8, head = x / 8 % heads, tok = x / 8 / heads;
                Chunk va, vc;
                va.u = vc.u = make_uint4(0, 0, 0, 0);
                if (live) {
                    const __half *src = p.v + (t0 + (uint64_t)tok) * p.v_stride + (h0 + head) * 128;
                    va.u = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * j));
                    vc.u = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * j + 64));
                }
                const float scale = row_scale(va, vc, live);
                if (!live) continue;
                union {
                    uint2 u[2];
                    uint8_t b[16];
                } by;
                by.u[0] = bytes_of(va, scale);
                by.u[1] = bytes_of(vc, scale);
    #pragma unroll
                for (uint32_t e = 0; e < 16; ++e) v_s[(head * 128 + (e / 8) * 64 + 8 * j + e % 8) * 16 + tok] = by.b[e];
                if (j == 0) p.v_scales[run + (size_t)(h0 + head) * p.page_size + tok] = scale;
            }
            __syncthreads();
            const uint32_t r = in_page % 16;  // row of the block that token 0 goes to (0 where the block is whole)
            for (uint32_t x = tid; x < heads * 128; x += kThreads) {
                const uint32_t head = x / 128, d = x % 128;
                uint8_t *dst = static_cast<uint8_t *>(p.v_pool) + (run - in_page + (size_t)(h0 + head) * p.page_size) * 128 + in_page / 16 * 2048 + d * 16 + r;
                if (n_tok == 16) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(v_s + x * 16);
                else
                    for (uint32_t t = 0; t < n_tok; ++t) dst[t] = v_s[x * 16 + t];
            }
        }
    }
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
mf_status launch_mrope(MfContext *ctx, MropeParams &p, const char *what)
{
    if (p.tokens == 0) return MF_OK;
    const uint32_t R = K8 ? 16 : 8, cpr = p.head_dim / 16;
    const uint64_t blocks = first_block(p.tokens, p.batch, R) + 1;
    const uint64_t slots = (p.q_rot ? p.n_heads : 0) + (uint64_t)(K8 ? 1 : 2) * p.n_kv_heads;
    // Prompts: so many parts that a whole block leaves every thread two rounds of loads (one round: 41 and 18 us for 8.5k
    // tokens of 32/8 heads and 4.8k tokens into the 8-bit cache, two: 39.6 and 17, no parts at all: 57 and 26).  Decode
    // steps (a token or few per sequence) have little for a CTA as it is.
    const uint64_t per_part = 2ull * in_flight(K8) * kThreads;
    uint64_t parts = 1;
    if (p.tokens >= 4ull * p.batch) parts = std::min<uint64_t>((R * slots * cpr + per_part - 1) / per_part, 64);
    p.slots_per_part = (uint32_t)((slots + parts - 1) / parts);
    parts = (slots + p.slots_per_part - 1) / p.slots_per_part + (K8 ? 1 : 0);
    if (blocks > 0x7FFFFFFFull) return fail(ctx, MF_ERR_INVALID_SHAPE, "%s: %u tokens of %u sequences", what, p.tokens, p.batch);
    DeviceScope scope(ctx->device);
    const dim3 grid((uint32_t)blocks, (uint32_t)parts);
    if (p.head_dim == 128) mrope_append_kernel<128, K8><<<grid, kThreads, 0, ctx->stream>>>(p);
    else if constexpr (!K8) mrope_append_kernel<64, false><<<grid, kThreads, 0, ctx->stream>>>(p);
    const mf_status st = check_launch(ctx, "mrope_append_kernel");
    if (st == MF_OK) ctx->note_plain_launch(true);
    return st;
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" {

mf_status mf_paged_mrope_append(MfContext *ctx, const MfPagedKv *c, const MfMropeAppendArgs *a)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (c && c->page_size % 8)
        return fail(ctx, MF_ERR_OPERATION_NOT_SUPPORTED, "mrope append: page_size %u (a multiple of 8)", c->page_size);
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
