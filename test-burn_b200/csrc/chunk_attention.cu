// Attention of a ragged batch of new tokens over a paged cache on the tcgen05 tensor cores: causal, optionally with a
// sliding window and first tokens that stay visible (sinks).
//
//   out[t, h] = sum_k w_k V[k] / sum_k w_k,   w_k = exp(scale * q[t, h] . K[k] - max_k),   k visible to t
//
// One persistent CTA per SM walks its items of the plan (chunk_plan.hpp).  The rows of a unit are (token, query head of
// the kv head) pairs, so that one pass over a kv head's keys serves all its query heads, and the causal diagonal and
// the window's edge are 128 / G tokens wide instead of 128.
//
// Two streams, each a 128-row score tile S_s and an output tile O_s in TMEM with a softmax group of its own:
//   more than 128 rows   the streams are the two query tiles, both work on every key tile ("paired rows")
//   up to 128 rows       both streams hold the same rows, stream s takes the key tiles s, s + 2, ... and the two states
//                        are merged when the item ends ("paired keys"): decode and short chunks
// A stream takes its key tiles in two halves of 64 keys, each with score columns of its own: S = Q K^T -> max, exp, P (f16,
// over S) -> O += P V -> the same half of the next tile.  While a softmax group works on one half, the tensor pipe has
// the other half and the other stream; a group waits for nothing but its own two halves.
//
//   warps 0-3, 4-7  softmax groups (one thread per row = TMEM lane)   warp 8   TMA producer, one copy per page and tile
//   warps 9, 10     issue the products of streams 0, 1                warp 11  loads q, prepares V tiles, allocates TMEM
//
// K and V tiles share one ring in the order in which the products want them (chunk_ring.hpp).  A (page, kv head) run lands as
// [8-row group][half][8 rows][128 bytes], so the 128 rows of a tile are evenly spaced 8-row groups whatever the page
// size, and both operands (K by rows, V by columns) take one descriptor per tile.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last rescale.  Weights carry a constant
// factor of 2^7 (it cancels in the division): at most 2^15, they are rounded to f16 for the product (2^-11 of each, 2^-32 of
// the reference maximum below 2^-21 of it), sums, maxima and accumulators are f32.
//
// Rows of a tile that no row of the unit sees (the end of the cache, the edge of the window) are cleared in V: their
// weight is zero, but zero times a stale NaN is not.  For the same reason elements that are not finite are taken out of the
// value rows that some rows of the unit see and others do not (along the diagonal and the window's edge: at most as many
// keys as the unit has tokens, each; none for a single token), and added to the rows that do see them when the item's rows
// are in memory (add_hidden).  What every row sees stays as it is.  Warp 11 does both while the softmax groups are at work
// (done by the groups it is 53 instead of 44 us for a prompt step of 14/2 heads of 64, window 512).
//
// What bounds it (measured on a B200):
//   long prompts (6.8k new tokens over 8k keys, 16/2 heads of 128; 319 GFLOP): 323 us in bursts at 1.97 GHz, 337-348
//     us when the power limit brings the clock to 1.7 GHz: 920-990 TFLOP/s.  Tensor pipe and
//     exponential unit are both at 0.5; a softmax group takes some 2 000 cycles for 64 keys and never waits.  Tried: sixteen
//     softmax warps (one group per stream and half), one softmax step per 128 keys with the issue in strict turns,
//     part of the exponentials as a cubic on the FMA pipe: none is faster over long blocks.
//   decode (64 sequences, window 4 096, 177 MB): 40 us in a graph, 4.4 TB/s; from the first tile (4 us after the launch) to
//     the last (33 us) the keys stream at 0.9 of the copy rate, the rest is start, drain and joining of cut units.
//   one token, 1 028 keys: 9.0-10.0 us, of which the last piece's joining is 2 and fence and ticket 1.  Five drafted tokens of
//     each of 8 sequences: 13.2-13.9.  A half tile in which no row sees a key (behind the last one) is left out, 1.1 us of either.
//
// TMEM columns (512): halves 0, 1 of S_0/P_0 [0,64) [64,128), of S_1/P_1 [128,192) [192,256), O_0 [256,384)  O_1 [384,512).
#include <algorithm>
#include <cstring>
#include <new>
#include <vector>

#include "chunk_plan.hpp"
#include "chunk_ring.hpp"
#include "internal.hpp"
#include "ptx.cuh"
#include "tcgen05.cuh"

struct MfChunkPlan {
    uint32_t batch = 0, n_heads = 0, n_kv_heads = 0, head_dim = 0, page_size = 0, window = 0, n_sinks = 0;
    uint32_t max_tokens = 0, tokens = 0, max_pages = 0;
    uint32_t n_ctas = 0, begin_words = 0;  // cta_begin, padded to whole items; the last word is the number of tokens
    uint64_t item_capacity = 0;
    int device = 0;
    std::vector<mf::ChunkItem> h_items;
    std::vector<uint32_t> h_begin;
    // [begin_words], [item_capacity] items; two pinned copies used in turn, each guarded by the event
    // recorded after its upload.  One allocation on the device, one on the host.
    void *device_block = nullptr;
    uint32_t *d_list = nullptr;
    uint32_t *pinned[2] = {nullptr, nullptr};
    cudaEvent_t staged[2] = {nullptr, nullptr};
    uint32_t next_stage = 0;
    float *d_acc = nullptr, *d_ml = nullptr;  // partial results: [slot][D / 4][256 rows][4], [slot][256 rows][2]
    uint32_t *d_tickets = nullptr;
    // Launches on another stream than the last update's wait for its upload, and the next update waits for them.
    cudaStream_t updated_on = nullptr;
    cudaEvent_t used = nullptr;
    mutable bool used_elsewhere = false;
    bool updated = false;  // an update has been made
};

namespace mf {
namespace {

constexpr uint32_t kMaxGroup = 64;
constexpr uint32_t kMaxLen = kChunkMaxLen;
constexpr uint32_t kTile = kChunkTile;
constexpr uint32_t kThreads = 384;
constexpr uint32_t kProducerWarp = 8, kIssuerWarp = 9, kQWarp = 11;
constexpr uint64_t kWaitNs = 2000000000ull;  // a wait that takes longer sets its bit of the status word and gives up
constexpr float kNegInf = -1e30f;  // a row's maximum before its first key
// Products of f16 rows of 128 are below 2^39: with this scale every finite score stays above kNegInf.
constexpr float kMaxScale = 1e18f;
constexpr float kRescaleThreshold = 8.0f;  // log2 of the largest growth of a row's maximum without a rescale
constexpr float kWeightShift = 7.0f;       // log2 of the weight of the reference maximum: 2^(8 + 7) fits f16
constexpr uint32_t kHalfTile = kTile * 128;

__host__ __device__ constexpr uint32_t tile_bytes(uint32_t d) { return kTile * d * 2; }
__host__ __device__ constexpr uint32_t ring_slots(uint32_t d) { return d == 128 ? 5 : 10; }
enum Bar : uint32_t {
    kSFull = 0,   // [stream * 2 + half] scores of the next tile's half are in S
    kPFull = 4,   // [stream * 2 + half] weights are in P, O has been rescaled if needed
    kODone = 8,   // [stream] a P V has completed (one phase per half tile)
    kOFull = 10,  // [stream] the item's last P V has completed (2 arrivals: with the issuing warp's own)
    kOFree = 12,  // [stream] the item's O has been read (8 arrivals)
    kQFull = 14,
    kQFree = 15,  // 2 arrivals: the streams' last Q K^T of the item
    kFull = 16    // [slots], then empty [slots] (3 arrivals: the streams and warp 11), then fit [slots] (warp 11 is through with it)
};
__host__ __device__ constexpr uint32_t num_bars(uint32_t d) { return kFull + 3 * ring_slots(d); }
constexpr uint32_t kMlBytes = 2 * kTile * 8;  // (m, l) of the two streams' rows
// Words behind the barriers: TMEM address, abort flag, "last piece of the unit", and the last four items (their number + 1)
// in which elements were taken out of V rows.  (Warp 11 is at most three items ahead of a softmax group: an item's q goes to
// shared memory when the one before has been multiplied, and that waits for the weights of the one before it.)
enum Word : uint32_t { kTmem = 0, kAbort = 1, kLast = 2, kTaken = 4, kNumWords = 8 };
__host__ __device__ constexpr uint32_t smem_bytes(uint32_t d)
{
    return tile_bytes(d) * (2 + ring_slots(d)) + kMlBytes + num_bars(d) * 8 + kNumWords * 4;
}
static_assert(smem_bytes(128) <= 227 * 1024 && smem_bytes(64) <= 227 * 1024, "shared memory");

struct ChunkParams {
    const __half *q;
    __half *out;
    const __half *v_pool;  // add_hidden only
    const uint32_t *page_table;
    const uint32_t *list;  // cta_begin, then the items
    float *acc, *ml;
    uint32_t *tickets, *status;
    uint64_t q_stride_t, q_stride_h, out_stride_t, out_stride_h;
    uint32_t begin_words, n_kv_heads, group, page_shift, pt_stride, n_pages, window, n_sinks;
    uint32_t q_tokens;  // tokens that the maps of q cover; 0: q is loaded without them
    float scale_log2;
};

__device__ __forceinline__ ChunkItem load_item(const ChunkParams &p, uint32_t i)
{
    ChunkItem it;
    const uint4 *src = reinterpret_cast<const uint4 *>(p.list + p.begin_words) + (size_t)i * 4;
    uint4 *dst = reinterpret_cast<uint4 *>(&it);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) dst[j] = __ldg(src + j);
    return it;
}

// (the next item, on its way while this one's rows are written)
__device__ __forceinline__ void prefetch_item(const ChunkParams &p, uint32_t i)
{
    asm volatile("prefetch.global.L1 [%0];" ::"l"(p.list + p.begin_words + (size_t)i * 16));
}

// What a row at position pos sees, in columns of the unit's page list: [0, a) and [b, c).
struct Visible {
    int32_t a, b, c;
};
__device__ __forceinline__ Visible visible(const ChunkParams &p, const ChunkItem &it, int32_t pos)
{
    Visible v{0, 0, 0};
    if (pos < 0) return v;
    const int32_t lo = p.window && (uint32_t)pos >= p.window ? pos - (int32_t)p.window + 1 : 0;
    const int32_t shift = ((int32_t)it.first_page - (int32_t)it.n_sink_pages) << p.page_shift;
    v.a = min((int32_t)min(p.n_sinks, 0x7FFFFFFFu), lo);
    v.b = lo - shift;
    v.c = pos + 1 - shift;
    if (v.a >= v.b) v.a = v.b = 0;  // the sinks reach the window: one range
    return v;
}
__device__ __forceinline__ uint32_t page_entry(const ChunkItem &it, uint32_t v)
{
    return v < it.n_sink_pages ? v : v - it.n_sink_pages + it.first_page;
}
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

// 1 / the sum of a row's weights.  A row before the start of the cache sees nothing and comes out as zeros; any other sees
// its own key at least: a sum of 0 means that all its scores are -inf, which is as little a number as a NaN among them.
__device__ __forceinline__ float inverse_sum(float sum, int32_t pos)
{
    if (sum > 0.f) return 1.f / sum;
    return pos < 0 ? 0.f : __int_as_float(0x7FFFFFFF);
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Past 2^24 the rounding of a reference maximum alone is worth a factor of two and more.
__device__ __forceinline__ bool is_far(float m_ref) { return fabsf(m_ref) > 16777216.f && m_ref > kNegInf; }

// The weights of a half tile in which some row of the warp has a reference maximum so far from 0: it is subtracted before the
// scaling.  Reads the scores from TMEM once more, writes the weights over them, returns their sum.
__device__ __noinline__ float far_weights(uint32_t tm, const Visible vis, int32_t x0, bool valid, float m_ref, float m_raw, float scale)
{
    const bool far = is_far(m_ref);
    const float sub = far ? m_raw : 0.f, shift = far ? kWeightShift : kWeightShift - m_ref;
    float sum = 0.f;
#pragma unroll 1
    for (uint32_t c = 0; c < 2; ++c) {
        const int32_t x = x0 + (int32_t)c * 32;
        const uint32_t see = valid ? low_bits(vis.a - x) | (low_bits(vis.c - x) & ~low_bits(vis.b - x)) : 0xFFFFFFFFu;
        uint32_t r[32], pk[16];
        tmem_ld32(tm + c * 32, r);
        tc_wait_ld();
#pragma unroll
        for (uint32_t q = 0; q < 32; ++q) {
            const float w = (see >> q) & 1u ? fast_exp2(fmaf(__uint_as_float(r[q]) - sub, scale, shift)) : 0.f;
            sum += w;
            r[q] = __float_as_uint(w);
        }
#pragma unroll
        for (uint32_t q = 0; q < 16; ++q) pk[q] = pack_f16x2(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
        tmem_st16(tm + c * 16, pk);
    }
    return sum;
}

// Means of f16 values stay in f16's range: the rounding of the weights (2^-11 of each) can carry one past its end, where the
// rounding to f16 would make it an infinity.  (0.06 us of a small call, 2 % of window 512 prompts; a look at the packed words
// and a second pass over TMEM for the rows that need it cost the same and more.)
template <uint32_t N>
__device__ __forceinline__ void keep_inside(float (&o)[N])
{
    float top = 0.f;
#pragma unroll
    for (uint32_t q = 0; q < N; q += 2) top = max3(top, fabsf(o[q]), fabsf(o[q + 1]));
    if (top > 65504.f) {
#pragma unroll
        for (uint32_t q = 0; q < N; ++q)
            if (fabsf(o[q]) < 65600.f) o[q] = fminf(fmaxf(o[q], -65504.f), 65504.f);
    }
}

// Columns of a unit's page list by who sees them.  [gap0, gap1) and what lies behind `end`: no row.  [sink0, sink1),
// [edge0, edge1), [diag0, diag1): some rows.  All others: every row.  (Rows only gain keys at the diagonal and lose keys at
// the window's edge: the first and the last row have them all.)
struct Cuts {
    int32_t gap0, gap1, end;
    int32_t sink0, sink1, edge0, edge1, diag0, diag1;
    // whether the V tile at column x has such rows; its second half is not used when no row sees it
    __device__ __forceinline__ bool tile(int32_t x) const
    {
        const int32_t y = used(x);
        return end < y || max(gap0, x) < min(gap1, y) || max(sink0, x) < min(sink1, y) || max(edge0, x) < min(edge1, y) ||
               max(diag0, x) < min(diag1, y);
    }
    __device__ __forceinline__ int32_t used(int32_t x) const { return x + (int32_t)(end > x + (int32_t)kTile / 2 ? kTile : kTile / 2); }
};
__device__ __forceinline__ Cuts cuts_of(const ChunkParams &p, const ChunkItem &it)
{
    const Visible first = visible(p, it, it.pos0), last = visible(p, it, it.pos0 + (int32_t)it.n_tok - 1);
    const int32_t any_b = visible(p, it, max(it.pos0, 0)).b;
    Cuts c;
    c.gap0 = last.a;
    c.gap1 = any_b;
    c.end = last.c;
    c.sink0 = min(last.a, first.c);
    c.sink1 = last.a;
    c.edge0 = max(any_b, last.a);
    c.edge1 = min(last.b, last.c);
    c.diag0 = max(max(first.c, any_b), last.b);
    c.diag1 = last.c;
    return c;
}

// Makes the V tile at column x fit for the products, by one warp: rows that no row of the unit sees become 0, and so do
// elements that are not finite in rows that some of them see.  Returns whether there were such elements.
template <uint32_t D>
__device__ __noinline__ bool prepare_values(uint8_t *tile, const Cuts cuts, int32_t x)
{
    constexpr uint32_t C = D / 8, kStep = 32 / C;  // 16-byte units per row, rows a step
    const uint32_t lane = threadIdx.x & 31, c = lane % C;
    const int32_t y = cuts.used(x);
    auto at = [&](int32_t col) {
        const uint32_t r = (uint32_t)(col - x);
        return reinterpret_cast<uint4 *>(tile + (r >> 3) * (16 * D) + (c >> 3) * 1024 + (r & 7) * 128 + (c & 7) * 16);
    };
    auto clear = [&](int32_t lo, int32_t hi) {
        for (int32_t col = max(lo, x) + (int32_t)(lane / C); col < min(hi, y); col += kStep) *at(col) = make_uint4(0, 0, 0, 0);
    };
    clear(cuts.gap0, cuts.gap1);
    clear(cuts.end, y);
    bool found = false;
    // an exponent of all ones carries into the sign's place
    auto odd = [](uint32_t w) { return ((w & 0x7FFF7FFFu) + 0x04000400u) & 0x80008000u; };
    auto without = [&](uint32_t w) {
        const uint32_t o = odd(w);
        return w & ~((o & 0x8000u ? 0xFFFFu : 0u) | (o & 0x80000000u ? 0xFFFF0000u : 0u));
    };
    auto take_out = [&](int32_t lo, int32_t hi) {
        constexpr int32_t kBatch = 8;
        hi = min(hi, y);
        for (int32_t col = max(lo, x) + (int32_t)(lane / C); col < hi; col += kBatch * kStep) {
            uint4 v[kBatch];
#pragma unroll
            for (int32_t k = 0; k < kBatch; ++k) {
                v[k] = make_uint4(0, 0, 0, 0);
                if (col + k * (int32_t)kStep < hi) v[k] = *at(col + k * (int32_t)kStep);
            }
            uint32_t any = 0;
#pragma unroll
            for (int32_t k = 0; k < kBatch; ++k) any |= odd(v[k].x) | odd(v[k].y) | odd(v[k].z) | odd(v[k].w);
            if (any) {
                found = true;
#pragma unroll
                for (int32_t k = 0; k < kBatch; ++k)
                    if (odd(v[k].x) | odd(v[k].y) | odd(v[k].z) | odd(v[k].w))
                        *at(col + k * (int32_t)kStep) = make_uint4(without(v[k].x), without(v[k].y), without(v[k].z), without(v[k].w));
            }
        }
    };
    take_out(cuts.sink0, cuts.sink1);
    take_out(cuts.edge0, cuts.edge1);
    take_out(cuts.diag0, cuts.diag1);
    fence_proxy_async();
    return __any_sync(0xffffffffu, found);
}

// What prepare_values took out, added to the rows that see it: a warp's 32 rows, `dims` dims from d0 on.  Such an element
// decides its row's output in that dim whatever its weight is (the weight of a visible key is positive): added as it is.
// to: element 0 of the lane's row (f16), or of its partial result (f32, in groups of four dims); null: no row.
template <uint32_t D, bool CUT>
__device__ __noinline__ void add_hidden(const ChunkParams &p, uint32_t item, int32_t pos, uint32_t d0, uint32_t dims, void *to)
{
    const ChunkItem it = load_item(p, item);
    const Visible vis = visible(p, it, pos);
    const Cuts cuts = cuts_of(p, it);
    const uint32_t lane = threadIdx.x & 31, E = dims / 32, P = 1u << p.page_shift;
    __syncwarp();  // the rows were written by other lanes of the warp
    for (uint32_t k = 0; k < 3; ++k) {
        const int32_t lo = max((int32_t)(it.tile_begin * kTile), k == 0 ? cuts.sink0 : k == 1 ? cuts.edge0 : cuts.diag0);
        const int32_t hi = min((int32_t)(it.tile_end * kTile), k == 0 ? cuts.sink1 : k == 1 ? cuts.edge1 : cuts.diag1);
        for (int32_t x = lo; x < hi; ++x) {
            const uint32_t entry = page_entry(it, (uint32_t)x >> p.page_shift);
            const uint32_t page = entry < p.pt_stride ? p.page_table[(size_t)it.seq * p.pt_stride + entry] : 0xFFFFFFFFu;
            if (page >= p.n_pages) continue;
            const __half *v = p.v_pool + ((((size_t)page * p.n_kv_heads + it.kvh) << p.page_shift) + ((uint32_t)x & (P - 1))) * D + d0;
            float value[D / 32];
            bool odd = false;
#pragma unroll
            for (uint32_t e = 0; e < D / 32; ++e) {
                value[e] = e < E ? __half2float(v[e * 32 + lane]) : 0.f;
                odd |= !(fabsf(value[e]) <= 65504.f);
            }
            if (!__any_sync(0xffffffffu, odd)) continue;
            uint32_t rows = __ballot_sync(0xffffffffu, to && (x < vis.a || (x >= vis.b && x < vis.c)));
            while (rows) {
                const uint32_t src = __ffs(rows) - 1;
                rows &= rows - 1;
                void *row = reinterpret_cast<void *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), src));
#pragma unroll
                for (uint32_t e = 0; e < D / 32; ++e) {
                    const uint32_t d = e * 32 + lane;
                    if (fabsf(value[e]) <= 65504.f) continue;
                    if (CUT) {
                        float *o = static_cast<float *>(row) + (size_t)(d / 4) * (2 * kTile) * 4 + d % 4;
                        __stcg(o, __ldcg(o) + value[e]);
                    } else {
                        __half *o = static_cast<__half *>(row) + d;
                        *o = __float2half_rn(__half2float(*o) + value[e]);
                    }
                }
            }
        }
    }
    __syncwarp();
}

template <uint32_t D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_q,
                const __grid_constant__ CUtensorMap tm_q1, const __grid_constant__ ChunkParams p)
{
    constexpr uint32_t kBytes = tile_bytes(D), kSlots = ring_slots(D);
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + 2 * kBytes;
    float2 *ml_s = reinterpret_cast<float2 *>(smem + kBytes * (2 + kSlots));  // [stream][row]
    const uint32_t bars = q_smem + kBytes * (2 + kSlots) + kMlBytes;
    volatile uint32_t *words = reinterpret_cast<volatile uint32_t *>(smem + kBytes * (2 + kSlots) + kMlBytes + num_bars(D) * 8);
    volatile uint32_t *abort_flag = words + kAbort;
    auto bar = [&](uint32_t i) { return bars + i * 8; };
    // (the warp's number by a shuffle: known to be the same in all its lanes, so that what the issuing warp computes stays
    // in uniform registers)
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t G = p.group, half_tok = kTile / G;
    const uint32_t item0 = __ldg(p.list + blockIdx.x), item1 = __ldg(p.list + blockIdx.x + 1);
    if (item0 >= item1) return;
    if (q_smem & 1023u) {  // the swizzled tiles need it; dynamic shared memory starts there when nothing is static
        if (tid == 0) atomicOr(p.status, 1u);
        return;
    }
    if (tid == 0) {
        for (uint32_t s = 0; s < 4; ++s) {
            mbar_init(bar(kSFull + s), 1);
            mbar_init(bar(kPFull + s), 4);
        }
        for (uint32_t s = 0; s < 2; ++s) {
            mbar_init(bar(kODone + s), 1);
            mbar_init(bar(kOFull + s), 2);
            mbar_init(bar(kOFree + s), 8);
        }
        mbar_init(bar(kQFull), 1);
        mbar_init(bar(kQFree), 2);
        for (uint32_t s = 0; s < kSlots; ++s) {
            mbar_init(bar(kFull + s), 1);
            mbar_init(bar(kFull + kSlots + s), 3);
            mbar_init(bar(kFull + 2 * kSlots + s), 1);
        }
        *abort_flag = 0;
        for (uint32_t x = kTaken; x < kNumWords; ++x) words[x] = 0;
        mbar_fence_init();
        fence_proxy_async();
    }
    if (warp == kQWarp) {
        tmem_alloc(smem_u32(const_cast<uint32_t *>(words)), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[kTmem];

    auto wait = [&](uint32_t b, uint32_t parity, uint32_t code) {
        if (mbar_try_wait(b, parity)) return;
        if (!*abort_flag && !mbar_wait_bounded(b, parity, kWaitNs)) {
            *abort_flag = 1;
            atomicOr(p.status, code);
        }
    };

    if (warp == kProducerWarp) {
        // ------------------------------------------------------------------ K/V producer (whole warp) ---
        const uint32_t per_tile = kTile >> p.page_shift, page_bytes = D * 2u << p.page_shift;
        const uint32_t none = p.n_pages * p.n_kv_heads;  // coordinate behind the pool: arrives as zeros
        uint32_t slot = 0, phase = 0;
        auto read_id = [&](const ChunkItem &it, uint32_t t) -> uint32_t {
            const uint32_t v = t * per_tile + lane;
            if (lane >= per_tile || v >= it.n_pages) return 0u;
            // (a replayed launch can meet a plan whose sequences have outgrown the captured table)
            const uint32_t entry = page_entry(it, v);
            return entry < p.pt_stride ? __ldg(p.page_table + (size_t)it.seq * p.pt_stride + entry) : 0xFFFFFFFFu;
        };
        auto load = [&](const CUtensorMap *tm, const ChunkItem &it, uint32_t t, uint32_t id) {
            const uint32_t n = min(per_tile, it.n_pages - t * per_tile);
            if (lane == 0) {
                wait(bar(kFull + kSlots + slot), phase ^ 1, 2u);
                mbar_arrive_expect_tx(bar(kFull + slot), n * page_bytes);
            }
            __syncwarp();
            if (lane < n) {
                if (id >= p.n_pages) atomicOr(p.status, kStatusBadPage);
                tma_load_5d_last(ring + slot * kBytes + lane * page_bytes, tm, (int32_t)(id < p.n_pages ? id * p.n_kv_heads + it.kvh : none),
                                 bar(kFull + slot));
            }
            if (++slot == kSlots) slot = 0, phase ^= 1;
        };
        if (lane == 0) {
            tma_prefetch_desc(&tm_k);
            tma_prefetch_desc(&tm_v);
        }
        ChunkItem it = load_item(p, item0);
        uint32_t id0 = read_id(it, it.tile_begin), id1 = read_id(it, it.tile_begin + 1);
        for (uint32_t i = item0; i < item1; ++i) {
            const ChunkItem next = i + 1 < item1 ? load_item(p, i + 1) : it;
            const uint32_t step = it.n_tok > half_tok ? 1 : 2;
            for (uint32_t t = it.tile_begin; t < it.tile_end; t += step) {
                // page ids of the following tiles are requested before this one's copies wait for their slots
                const bool last = t + step >= it.tile_end;
                const uint32_t n0 = last ? read_id(next, next.tile_begin) : read_id(it, t + step);
                const uint32_t n1 = last ? read_id(next, next.tile_begin + 1) : read_id(it, t + step + 1);
                const bool two = step == 2 && t + 1 < it.tile_end;
                load(&tm_k, it, t, id0);
                if (two) load(&tm_k, it, t + 1, id1);
                load(&tm_v, it, t, id0);
                if (two) load(&tm_v, it, t + 1, id1);
                id0 = n0;
                id1 = n1;
            }
            if (it.tile_begin == it.tile_end) {
                id0 = read_id(next, next.tile_begin);
                id1 = read_id(next, next.tile_begin + 1);
            }
            it = next;
        }
        // Nothing may still be on its way into this CTA's shared memory when it ends (it is not, unless a wait ran out).
        if (lane == 0 && *abort_flag)
            for (uint32_t s = 0; s < kSlots; ++s) mbar_wait_bounded(bar(kFull + s), s < slot ? phase : phase ^ 1, kWaitNs / 16);
    } else if (warp == kQWarp) {
        // ------------------------------------------------------------- q and V tiles (whole warp) ---
        uint32_t used = 0, slot = 0, phase = 0;
        // This item's loads in turn, like the streams: a tile that some row must not see in part is made fit for the products.
        auto prepare = [&](uint32_t i, const ChunkItem &it) {
            const uint32_t n = it.tile_end - it.tile_begin;
            const bool paired_rows = it.n_tok > half_tok;
            const Cuts cuts = cuts_of(p, it);
            for (uint32_t load = 0; load < 2 * n; ++load) {
                wait(bar(kFull + slot), phase, 8u);
                const uint32_t t = ring_v_tile(paired_rows, n, load);
                const int32_t x = (int32_t)((it.tile_begin + t) * kTile);
                if (t < n && cuts.tile(x)) {
                    const bool found = prepare_values<D>(smem + (2 + slot) * kBytes, cuts, x);
                    __syncwarp();
                    if (found && lane == 0) words[kTaken + used % 4] = i + 1;
                }
                if (lane == 0) {
                    mbar_arrive(bar(kFull + 2 * kSlots + slot));
                    mbar_arrive(bar(kFull + kSlots + slot));
                }
                if (++slot == kSlots) slot = 0, phase ^= 1;
            }
        };
        // A replayed launch can meet a plan with more tokens than q had when it was captured: then without the maps.
        const bool by_map = __ldg(p.list + p.begin_words - 1) <= p.q_tokens;
        for (uint32_t i = item0; i < item1; ++i) {
            const ChunkItem it = load_item(p, i);
            if (it.tile_begin == it.tile_end) continue;
            if (used) wait(bar(kQFree), (used - 1) & 1, 4u);
            ++used;
            if (by_map) {
                // the tokens of a stream in one copy per column half; what lies behind the unit's is loaded too and
                // computed on, and no one reads it
                if (lane == 0) {
                    const uint32_t streams = it.n_tok > half_tok ? 2 : 1, box = (it.n_tok == 1 ? 1 : half_tok) * G * 128;
                    const CUtensorMap *tm = it.n_tok == 1 ? &tm_q1 : &tm_q;
                    mbar_arrive_expect_tx(bar(kQFull), streams * (D / 64) * box);
                    for (uint32_t x = 0; x < streams; ++x)
#pragma unroll
                        for (uint32_t h = 0; h < D / 64; ++h)
                            tma_load_4d_box(q_smem + x * kBytes + h * kHalfTile, tm, 0, (int32_t)(it.kvh * G), (int32_t)(it.tok0 + x * half_tok),
                                            (int32_t)h, bar(kQFull));
                }
                __syncwarp();
                prepare(i, it);
                continue;
            }
            constexpr uint32_t C = D / 8;
            const uint32_t rows = it.n_tok * G, per_stream = half_tok * G;
            for (uint32_t x = lane; x < rows * C; x += 32) {
                uint32_t r = x / C;
                const uint32_t c = x % C, tok = r / G, g = r - tok * G;
                uint32_t dst = q_smem;
                if (r >= per_stream) r -= per_stream, dst += kBytes;
                cp_async16(dst + (c >> 3) * kHalfTile + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                           p.q + (it.tok0 + (uint64_t)tok) * p.q_stride_t + (uint64_t)(it.kvh * G + g) * p.q_stride_h + c * 8);
            }
            cp_async16_wait_all();
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kQFull));
            prepare(i, it);
        }
    } else if (warp >= kIssuerWarp) {
        // -------------------------------------------------------- the products of one stream (whole warp) ---
        // P V of a half tile and Q K^T of the same half of the stream's next tile, in turn for the two halves.  A warp per
        // stream: what the issue of a block costs (some 1 000 cycles with its waits) is as long as the block itself, and one
        // warp for both would be the kernel's pace.
        const uint32_t s = warp - kIssuerWarp, elected = elect_one_sync();
        constexpr uint32_t kIdescQK = instr_desc_f16(kTile, kTile / 2, 0), kIdescPV = instr_desc_f16(kTile, D, 1);
        constexpr uint32_t kGroupStride = 16 * D;  // bytes between 8-row groups of a K or V tile
        RingReader<kSlots> reader;
        auto landed = [&](uint32_t slot, uint32_t phase) { wait(bar(kFull + slot), phase, 16u); };
        auto pass = [&](uint32_t slot) {
            if (elected) mbar_arrive(bar(kFull + kSlots + slot));
        };
        uint32_t q_phase = 0, p_phase = 0, o_uses = 0;
        for (uint32_t i = item0; i < item1; ++i) {
            const ChunkItem it = load_item(p, i);
            const uint32_t n = it.tile_end - it.tile_begin;
            if (n == 0) continue;
            const bool paired_rows = it.n_tok > half_tok;
            const uint32_t tiles = paired_rows ? n : (n + 1 - s) / 2;
            // the item's last tile, if no row sees its second half (the softmax groups leave that half out, too)
            const Cuts cuts = cuts_of(p, it);
            const uint32_t half_tile = cuts.end <= (int32_t)(it.tile_end * kTile - kTile / 2) ? n - 1 : n;
            const uint64_t q_desc = smem_desc(q_smem + (paired_rows ? s * kBytes : 0), 16, 1024);
            uint32_t k = 0, v = 0;  // slots of the stream's K and V tile
            auto next = [&]() { return reader.next(paired_rows, n, s, landed, pass); };
            auto release = [&](uint32_t slot) { tc_commit_elected(elected, bar(kFull + kSlots + slot)); };
            auto scores = [&](uint32_t h) {
                if (h == 0) k = next();
                const uint64_t k_desc = smem_desc(ring + k * kBytes + h * 8 * kGroupStride, 16, kGroupStride);
                tc_fence_after();
#pragma unroll
                for (uint32_t kk = 0; kk < D / 16; ++kk)
                    tc_mma_ss_elected(elected, tmem + s * 128 + h * 64, q_desc + (((kk >> 2) * kHalfTile + (kk & 3) * 32) >> 4),
                                      k_desc + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4), kIdescQK, kk > 0);
                tc_commit_elected(elected, bar(kSFull + s * 2 + h));
                if (h == 1) release(k);
            };
            wait(bar(kQFull), q_phase, 32u);
            q_phase ^= 1;
            if (tiles) {
                scores(0);
                scores(1);
            }
            if (tiles <= 1) tc_commit_elected(elected, bar(kQFree));
            for (uint32_t j = 0; j < tiles; ++j) {
                const bool more = j + 1 < tiles;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    if (h == 0) {
                        v = next();
                        // (a slot's use is handed back by warp 11 when that is through with it: its phase cannot be two behind)
                        if (cuts.tile((int32_t)((it.tile_begin + (paired_rows ? j : 2 * j + s)) * kTile)))
                            wait(bar(kFull + 2 * kSlots + v), reader.last_phase(), 1024u);
                    }
                    const uint64_t v_desc = smem_desc(ring + v * kBytes + h * 8 * kGroupStride, 1024, kGroupStride);
                    wait(bar(kPFull + s * 2 + h), p_phase, 64u);
                    if (j == 0 && h == 0 && o_uses) wait(bar(kOFree + s), (o_uses - 1) & 1, 128u);
                    tc_fence_after();
                    if (h == 0 || (paired_rows ? j : 2 * j + s) != half_tile) {
#pragma unroll
                        for (uint32_t kk = 0; kk < kTile / 32; ++kk)
                            tc_mma_ts_elected(elected, tmem + 256 + s * 128, tmem + s * 128 + h * 64 + kk * 8,
                                              v_desc + ((kk * 2 * kGroupStride) >> 4), kIdescPV, (j > 0 || h > 0 || kk > 0) ? 1u : 0u);
                    }
                    tc_commit_elected(elected, bar(kODone + s));
                    if (h == 1) release(v);
                    if (more) scores(h);
                }
                p_phase ^= 1;
                if (!more) {
                    tc_commit_elected(elected, bar(kOFull + s));
                    if (elected) mbar_arrive(bar(kOFull + s));  // (what warp 11 has written is the softmax groups' to read)
                }
                if (j + 2 == tiles) tc_commit_elected(elected, bar(kQFree));
            }
            o_uses += tiles > 0;
            reader.finish(n, landed, pass);
        }
        // The products have to be over before the TMEM goes back (they are, unless a wait ran out).
        if (o_uses) wait(bar(kOFull + s), (o_uses - 1) & 1, 256u);
    } else {
        // -------------------------------------------------------------- softmax groups / epilogue ---
        const uint32_t s = warp >> 2, quad = warp & 3, r_in = quad * 32 + lane, gtid = tid & 127;
        const uint32_t lane_base = (quad * 32u) << 16;
        const uint32_t s_tm = tmem + lane_base + s * 128, o_base = tmem + lane_base + 256;
        const uint32_t row_tok = r_in / G, row_g = r_in - row_tok * G;  // row = (token, query head)
        uint32_t s_phase = 0, pv = 0, o_phase = 0;  // pv: this stream's P V so far
        for (uint32_t i = item0; i < item1; ++i) {
            ChunkItem it = load_item(p, i);
            const uint32_t n = it.tile_end - it.tile_begin, x_item = it.tile_begin * kTile;
            const bool paired_rows = it.n_tok > half_tok;
            const uint32_t tok_first = paired_rows ? s * half_tok : 0;
            const uint32_t rows = min(half_tok, it.n_tok - tok_first) * G;
            const bool valid = r_in < rows, busy = quad * 32 < rows;  // busy: the warp has rows
            const uint32_t tok = tok_first + (valid ? row_tok : 0), head = it.kvh * G + (valid ? row_g : 0);
            const int32_t pos = it.pos0 + (int32_t)tok;
            const Visible vis = visible(p, it, pos);
            const int32_t any_c = visible(p, it, it.pos0 + (int32_t)it.n_tok - 1).c;  // columns from here on: no row of the unit
            const uint32_t mine = paired_rows ? n : (n + 1 - s) / 2;
            float m_ref = kNegInf, m_raw = 0.f, l = 0.f;  // the reference maximum, with and without the scale
            bool far = false;  // some row of the warp has one far from 0
            for (uint32_t j = 0; j < mine; ++j) {
                const uint32_t t = paired_rows ? j : 2 * j + s;
#pragma unroll 1
                for (uint32_t h = 0; h < 2; ++h, ++pv) {
                    constexpr uint32_t N = kTile / 2;
                    const int32_t x0 = (int32_t)(x_item + t * kTile + h * N);
                    const uint32_t sp_tm = s_tm + h * N;
                    wait(bar(kSFull + s * 2 + h), s_phase, 512u);
                    tc_fence_after();
                    // (a tile's first half is not left out: the item's first product also clears O)
                    const bool seen = h == 0 || any_c > x0;
                    if (busy && seen) {
                        const bool whole = __all_sync(0xffffffffu, !valid || (vis.b <= x0 && vis.c >= x0 + (int32_t)N) || vis.a >= x0 + (int32_t)N);
                        uint32_t r[N];
#pragma unroll
                        for (uint32_t c = 0; c < N / 32; ++c) tmem_ld32(sp_tm + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
                        tc_wait_ld();
                        if (!whole) {
#pragma unroll
                            for (uint32_t c = 0; c < N / 32; ++c) {
                                const int32_t xc = x0 + (int32_t)c * 32;
                                const uint32_t see = valid ? low_bits(vis.a - xc) | (low_bits(vis.c - xc) & ~low_bits(vis.b - xc)) : 0xFFFFFFFFu;
                                if (__all_sync(0xffffffffu, see == 0xFFFFFFFFu)) continue;
#pragma unroll
                                for (uint32_t q = 0; q < 32; ++q)
                                    if (!((see >> q) & 1u)) r[c * 32 + q] = 0xFF800000u;  // -inf: weight exactly 0
                            }
                        }
                        float mx0 = -3.0e38f, mx1 = -3.0e38f, mx2 = -3.0e38f, mx3 = -3.0e38f;
#pragma unroll
                        for (uint32_t q = 0; q < N; q += 8) {
                            mx0 = max3(mx0, __uint_as_float(r[q]), __uint_as_float(r[q + 1]));
                            mx1 = max3(mx1, __uint_as_float(r[q + 2]), __uint_as_float(r[q + 3]));
                            mx2 = max3(mx2, __uint_as_float(r[q + 4]), __uint_as_float(r[q + 5]));
                            mx3 = max3(mx3, __uint_as_float(r[q + 6]), __uint_as_float(r[q + 7]));
                        }
                        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
                        const float m_new = mx > -3.0e38f ? mx * p.scale_log2 : kNegInf;
                        const bool grow = valid && m_new > m_ref + kRescaleThreshold;
                        const float m_old = m_ref;
                        if (grow) m_ref = m_new, m_raw = mx;
                        if (__any_sync(0xffffffffu, grow)) {
                            if (j > 0 || h > 0) {
                                // O has to hold every earlier P V before it is scaled.  The one before the last has completed
                                // (its half's scores were issued behind it), so the parity is unambiguous.
                                wait(bar(kODone + s), (pv - 1) & 1, 16384u);
                                tc_fence_after();
                                const float alpha = fast_exp2(m_old - m_ref);
                                l *= alpha;
#pragma unroll 1
                                for (uint32_t c = 0; c < D / 32; ++c) {
                                    uint32_t ob[32];
                                    tmem_ld32(o_base + s * 128 + c * 32, ob);
                                    tc_wait_ld();
#pragma unroll
                                    for (uint32_t q = 0; q < 32; ++q) ob[q] = __float_as_uint(__uint_as_float(ob[q]) * alpha);
                                    tmem_st32(o_base + s * 128 + c * 32, ob);
                                }
                                tc_wait_st();
                            }
                            far = __any_sync(0xffffffffu, is_far(m_ref));
                        }
                        if (far) {
                            l += far_weights(sp_tm, vis, x0, valid, m_ref, m_raw, p.scale_log2);
                        } else {
                            const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), nm2 = make_float2(kWeightShift - m_ref, kWeightShift - m_ref);
                            float2 acc_a = make_float2(0.f, 0.f), acc_b = make_float2(0.f, 0.f);
#pragma unroll
                            for (uint32_t c = 0; c < N / 32; ++c) {
                                uint32_t pk[16];
#pragma unroll
                                for (uint32_t q = 0; q < 16; ++q) {
                                    const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c * 32 + 2 * q]), __uint_as_float(r[c * 32 + 2 * q + 1])), sc2, nm2);
                                    float2 w;
                                    w.x = fast_exp2(x.x);
                                    w.y = fast_exp2(x.y);
                                    if (q & 1) acc_b = __fadd2_rn(acc_b, w);
                                    else acc_a = __fadd2_rn(acc_a, w);
                                    pk[q] = pack_f16x2(w.x, w.y);
                                }
                                tmem_st16(sp_tm + c * 16, pk);
                            }
                            const float2 acc = __fadd2_rn(acc_a, acc_b);
                            l += acc.x + acc.y;
                        }
                    }
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(kPFull + s * 2 + h));
                }
                s_phase ^= 1;
            }
            if (i + 1 < item1) prefetch_item(p, i + 1);
            it = load_item(p, i);  // rather than kept in registers across the tiles

            // ---- the item's rows ------------------------------------------------------------------------
            // paired rows: group s has all D dims of its own rows; paired keys: dims [s * D/2, (s + 1) * D/2) of the
            // same rows, from both streams' states.
            float f0 = 1.f, f1 = 0.f;  // factors of O_own / (O_0, O_1)
            if (!paired_rows) {
                ml_s[s * kTile + r_in] = make_float2(m_ref, l);
                if (mine) wait(bar(kOFull + s), o_phase, 2048u);
                named_bar_sync(9, 256);
                const float2 x0 = ml_s[r_in], x1 = ml_s[kTile + r_in];
                named_bar_sync(10, 256);  // the next item may publish
                m_ref = fmaxf(x0.x, x1.x);
                f0 = fast_exp2(x0.x - m_ref);
                f1 = fast_exp2(x1.x - m_ref);
                l = x0.y * f0 + x1.y * f1;
            } else if (n) {
                wait(bar(kOFull + s), o_phase, 2048u);
            }
            if (mine) o_phase ^= 1;
            tc_fence_after();
            const bool cut = it.n_parts > 1;
            const float norm = cut ? 1.f : inverse_sum(l, pos);
            f0 *= norm;
            f1 *= norm;
            const uint32_t d0 = paired_rows ? 0 : s * (D / 2), dims = paired_rows ? D : D / 2;
            const uint32_t slot_row = (paired_rows ? s * kTile : 0) + r_in;
            // partial results lie by row inside a group of four dims, so that neighbouring threads write neighbouring words
            float4 *part_row = reinterpret_cast<float4 *>(p.acc) + ((size_t)it.slot * (D / 4) + d0 / 4) * (2 * kTile) + slot_row;
            __half *dst = p.out + (it.tok0 + (uint64_t)tok) * p.out_stride_t + (uint64_t)head * p.out_stride_h + d0;
            if (busy) {
                // Rows go out four lanes to a row: the lanes of a quad swap their 16-byte blocks, lane q then has block q
                // of each of the quad's rows and four lanes store 64 consecutive bytes.
                __half *quad_dst[4];
                bool quad_valid[4];
#pragma unroll
                for (uint32_t t = 0; t < 4; ++t) {
                    const uint32_t src = (lane & ~3u) + t;
                    quad_dst[t] = reinterpret_cast<__half *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), src)) + (lane & 3) * 8;
                    quad_valid[t] = __shfl_sync(0xffffffffu, (uint32_t)valid, src) != 0;
                }
#pragma unroll 1
                for (uint32_t c = 0; c < dims / 32; ++c) {
                    float o[32];
#pragma unroll
                    for (uint32_t q = 0; q < 32; ++q) o[q] = 0.f;
                    if (n) {
                        tmem_ld32(o_base + (paired_rows ? s * 128 : 0) + d0 + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
                        tc_wait_ld();
#pragma unroll
                        for (uint32_t q = 0; q < 32; ++q) o[q] *= f0;
                        if (!paired_rows && n > 1) {
                            uint32_t o1[32];
                            tmem_ld32(o_base + 128 + d0 + c * 32, o1);
                            tc_wait_ld();
#pragma unroll
                            for (uint32_t q = 0; q < 32; ++q) o[q] = fmaf(__uint_as_float(o1[q]), f1, o[q]);
                        }
                    }
                    if (cut) {
                        if (valid) {
#pragma unroll
                            for (uint32_t q = 0; q < 32; q += 4)
                                __stcg(part_row + (c * 8 + q / 4) * (2 * kTile), make_float4(o[q], o[q + 1], o[q + 2], o[q + 3]));
                        }
                        continue;
                    }
                    keep_inside(o);
                    uint32_t w[16];
#pragma unroll
                    for (uint32_t q = 0; q < 16; ++q) w[q] = pack_f16x2(o[2 * q], o[2 * q + 1]);
#pragma unroll
                    for (uint32_t bit = 1; bit <= 2; bit <<= 1) {
                        const bool upper = lane & bit;
#pragma unroll
                        for (uint32_t t = 0; t < 4; ++t) {
                            if (t & bit) continue;
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) {
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[t * 4 + e] : w[(t | bit) * 4 + e], bit);
                                if (upper) w[t * 4 + e] = got;
                                else w[(t | bit) * 4 + e] = got;
                            }
                        }
                    }
#pragma unroll
                    for (uint32_t t = 0; t < 4; ++t)
                        if (quad_valid[t])
                            *reinterpret_cast<uint4 *>(quad_dst[t] + c * 32) = make_uint4(w[t * 4], w[t * 4 + 1], w[t * 4 + 2], w[t * 4 + 3]);
                }
            }
            // O has been read: the next item's first product may overwrite it.
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && n) {
                if (paired_rows) {
                    mbar_arrive_n(bar(kOFree + s), 2);
                } else {
                    mbar_arrive(bar(kOFree));
                    if (n > 1) mbar_arrive(bar(kOFree + 1));
                }
            }
            const bool taken = words[kTaken] == i + 1 || words[kTaken + 1] == i + 1 || words[kTaken + 2] == i + 1 || words[kTaken + 3] == i + 1;
            if (taken && busy) {
                if (cut) add_hidden<D, true>(p, i, pos, d0, dims, valid ? part_row : nullptr);
                else add_hidden<D, false>(p, i, pos, d0, dims, valid ? dst : nullptr);
            }
            if (cut) {
                if (valid && (paired_rows || s == 0))
                    __stcg(reinterpret_cast<float2 *>(p.ml) + (size_t)it.slot * 2 * kTile + slot_row, make_float2(m_ref, l));
                __threadfence();
                named_bar_sync(9, 256);
                if (tid == 0) {
                    const uint32_t done = atomicAdd(p.tickets + it.counter, 1u) + 1;
                    words[kLast] = done == it.n_parts;
                    if (done == it.n_parts) p.tickets[it.counter] = 0;  // for the next launch
                }
                named_bar_sync(10, 256);
                if (words[kLast]) {
                    // the last piece of the unit: all partial results are in memory
                    __threadfence();
                    // a thread takes 16 dims of a row; everything a piece has for it is requested at once
                    const uint32_t r0 = min(half_tok, it.n_tok) * G, total = it.n_tok * G;
                    for (uint32_t x = tid; x < total * (D / 16); x += 256) {
                        const uint32_t grp = x / total, row = x - grp * total, sr = row < r0 ? row : kTile + row - r0;
                        const float2 *ml = reinterpret_cast<const float2 *>(p.ml) + (size_t)it.first_slot * (2 * kTile) + sr;
                        const float4 *acc = reinterpret_cast<const float4 *>(p.acc) + ((size_t)it.first_slot * (D / 4) + grp * 4) * (2 * kTile) + sr;
                        float m = kNegInf, sum = 0.f, o[16];
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll 2
                        for (uint32_t k = 0; k < it.n_parts; ++k) {
                            const float2 z = __ldcg(ml + (size_t)k * (2 * kTile));
                            float4 a[4];
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) a[e] = __ldcg(acc + ((size_t)k * (D / 4) + e) * (2 * kTile));
                            const float m_new = fmaxf(m, z.x), f_old = fast_exp2(m - m_new), f = fast_exp2(z.x - m_new);
                            m = m_new;
                            sum = fmaf(z.y, f, sum * f_old);
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) {
                                o[4 * e] = fmaf(a[e].x, f, o[4 * e] * f_old);
                                o[4 * e + 1] = fmaf(a[e].y, f, o[4 * e + 1] * f_old);
                                o[4 * e + 2] = fmaf(a[e].z, f, o[4 * e + 2] * f_old);
                                o[4 * e + 3] = fmaf(a[e].w, f, o[4 * e + 3] * f_old);
                            }
                        }
                        const uint32_t tk = row / G;
                        const float inv = inverse_sum(sum, it.pos0 + (int32_t)tk);
                        uint4 *to = reinterpret_cast<uint4 *>(p.out + (it.tok0 + (uint64_t)tk) * p.out_stride_t +
                                                              (uint64_t)(it.kvh * G + row - tk * G) * p.out_stride_h + grp * 16);
#pragma unroll
                        for (uint32_t e = 0; e < 16; ++e) o[e] *= inv;
                        keep_inside(o);
#pragma unroll
                        for (uint32_t e = 0; e < 2; ++e)
                            to[e] = make_uint4(pack_f16x2(o[8 * e], o[8 * e + 1]), pack_f16x2(o[8 * e + 2], o[8 * e + 3]),
                                               pack_f16x2(o[8 * e + 4], o[8 * e + 5]), pack_f16x2(o[8 * e + 6], o[8 * e + 7]));
                    }
                }
                named_bar_sync(9, 256);  // words[kLast] and the partial rows are free again
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kQWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

auto *chunk_kernel(uint32_t head_dim) { return head_dim == 128 ? chunk_tc_kernel<128> : chunk_tc_kernel<64>; }

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

mf_status refuse_in_capture(MfContext *ctx, const char *what)
{
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    const mf_status st = check_cuda(ctx, cudaStreamIsCapturing(ctx->stream, &cap), "cudaStreamIsCapturing");
    if (st != MF_OK) return st;
    if (cap != cudaStreamCaptureStatusNone)
        return fail(ctx, MF_ERR_INVALID_OPERATION, "chunk plan: %s while the stream is being captured", what);
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
    if (pl->used_elsewhere) cudaEventSynchronize(pl->used);
    for (int i = 0; i < 2; ++i)
        if (pl->staged[i]) cudaEventDestroy(pl->staged[i]);
    if (pl->used) cudaEventDestroy(pl->used);
    if (pl->pinned[0]) cudaFreeHost(pl->pinned[0]);
    if (pl->device_block) cudaFree(pl->device_block);
    delete pl;
}

mf_status mf_chunk_plan_update(MfContext *ctx, MfChunkPlan *pl, const uint32_t *q_lens, const uint32_t *kv_lens)
{
    if (!ctx) return MF_ERR_INPUT_NOT_FOUND;
    if (!pl || !q_lens || !kv_lens) return fail(ctx, MF_ERR_INPUT_NOT_FOUND, "chunk plan: null input");
    if (pl->device != ctx->device) return fail(ctx, MF_ERR_INVALID_OPERATION, "chunk plan: the plan is another device's");
    DeviceScope scope(ctx->device);
    uint64_t tokens;
    uint32_t max_kv;
    mf_status st = check_lens(ctx, q_lens, kv_lens, pl->batch, &tokens, &max_kv);
    if (st != MF_OK) return st;
    if (tokens > pl->max_tokens)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: %llu new tokens, made for %u", (unsigned long long)tokens, pl->max_tokens);
    if ((st = refuse_in_capture(ctx, "no update")) != MF_OK) return st;
    try {
        build_chunk_plan(q_lens, kv_lens, pl->batch, pl->n_kv_heads, pl->n_heads / pl->n_kv_heads, pl->page_size, pl->window, pl->n_sinks,
                         pl->n_ctas, pl->h_items, pl->h_begin);
    } catch (const std::bad_alloc &) {
        return fail(ctx, MF_ERR_OUT_OF_MEMORY, "chunk plan: host memory");
    }
    if (pl->h_items.size() > pl->item_capacity)
        return fail(ctx, MF_ERR_INVALID_OPERATION, "chunk plan: %zu items, room for %llu", pl->h_items.size(), (unsigned long long)pl->item_capacity);
    const uint32_t s = pl->next_stage;
    if ((st = check_cuda(ctx, cudaEventSynchronize(pl->staged[s]), "chunk plan: staging")) != MF_OK) return st;
    uint32_t *w = pl->pinned[s];
    if (pl->used_elsewhere && (st = check_cuda(ctx, cudaStreamWaitEvent(ctx->stream, pl->used, 0), "chunk plan: order")) != MF_OK) return st;
    pl->used_elsewhere = false;
    // (a second update from another stream follows the first)
    if (pl->updated && pl->updated_on != ctx->stream &&
        (st = check_cuda(ctx, cudaStreamWaitEvent(ctx->stream, pl->staged[s ^ 1], 0), "chunk plan: order")) != MF_OK)
        return st;
    const size_t item_bytes = pl->h_items.size() * sizeof(ChunkItem);
    memcpy(w, pl->h_begin.data(), 4 * pl->h_begin.size());
    w[pl->begin_words - 1] = (uint32_t)tokens;
    if (item_bytes) memcpy(w + pl->begin_words, pl->h_items.data(), item_bytes);
    st = check_cuda(ctx, cudaMemcpyAsync(pl->d_list, w, 4 * (size_t)pl->begin_words + item_bytes, cudaMemcpyHostToDevice, ctx->stream),
                    "chunk plan: upload");
    if (st != MF_OK) return st;
    // (every launch leaves the tickets at zero, one whose waits ran out may not)
    if ((st = check_cuda(ctx, cudaMemsetAsync(pl->d_tickets, 0, 4 * (size_t)pl->n_ctas, ctx->stream), "chunk plan: tickets")) != MF_OK) return st;
    if ((st = check_cuda(ctx, cudaEventRecord(pl->staged[s], ctx->stream), "chunk plan: upload")) != MF_OK) return st;
    pl->next_stage = s ^ 1;
    pl->updated_on = ctx->stream;
    pl->updated = true;
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
    if (chunk_item_capacity(batch, max_tokens ? max_tokens : tokens, n_kv_heads, n_heads / n_kv_heads, (uint32_t)ctx->sm_count) > UINT32_MAX)
        return fail(ctx, MF_ERR_INVALID_SHAPE, "chunk plan: %llu tokens of %u kv heads", (unsigned long long)(max_tokens ? max_tokens : tokens), n_kv_heads);
    DeviceScope scope(ctx->device);
    // (an allocation would end the capture with an error)
    if ((st = refuse_in_capture(ctx, "no plan is made")) != MF_OK) return st;
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
    pl->n_ctas = (uint32_t)ctx->sm_count;
    pl->begin_words = (pl->n_ctas + 2 + 15) / 16 * 16;
    pl->item_capacity = chunk_item_capacity(batch, pl->max_tokens, n_kv_heads, n_heads / n_kv_heads, pl->n_ctas);
    const size_t list_bytes = (4 * (size_t)pl->begin_words + pl->item_capacity * sizeof(ChunkItem) + 255) / 256 * 256;
    const size_t rows = (size_t)chunk_slots(pl->n_ctas) * 2 * kTile, acc_bytes = rows * head_dim * 4, ml_bytes = rows * 8;
    // the GPU's memory first: what it cannot hold is not asked of the host, twice as large and pinned
    ok(cudaMalloc(&pl->device_block, acc_bytes + ml_bytes + list_bytes + 4 * (size_t)pl->n_ctas));
    if (e == cudaSuccess) ok(cudaMallocHost(reinterpret_cast<void **>(&pl->pinned[0]), 2 * list_bytes));
    for (cudaEvent_t *event : {&pl->staged[0], &pl->staged[1], &pl->used})
        if (e == cudaSuccess) ok(cudaEventCreateWithFlags(event, cudaEventDisableTiming));
    if (e == cudaSuccess) {
        char *at = static_cast<char *>(pl->device_block);
        pl->pinned[1] = pl->pinned[0] + list_bytes / 4;
        pl->d_acc = reinterpret_cast<float *>(at);
        pl->d_ml = reinterpret_cast<float *>(at + acc_bytes);
        pl->d_list = reinterpret_cast<uint32_t *>(at + acc_bytes + ml_bytes);
        pl->d_tickets = reinterpret_cast<uint32_t *>(at + acc_bytes + ml_bytes + list_bytes);
    }
    // (here rather than at the first launch, which may be inside a stream capture)
    if (e == cudaSuccess) ok(cudaFuncSetAttribute(chunk_kernel(head_dim), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(head_dim)));
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
    if (!(a->scale >= 0.f && a->scale <= kMaxScale))
        return fail(ctx, MF_ERR_INVALID_OPERATION, "paged chunk attention: scale %g", (double)a->scale);
    if (pl->max_tokens == 0 || !a->q || !a->out) return MF_OK;
    DeviceScope scope(ctx->device);
    ChunkParams p{};
    p.q = static_cast<const __half *>(a->q);
    p.out = static_cast<__half *>(a->out);
    p.v_pool = static_cast<const __half *>(c->v_pool);
    p.page_table = c->page_table;
    p.list = pl->d_list;
    p.acc = pl->d_acc;
    p.ml = pl->d_ml;
    p.tickets = pl->d_tickets;
    p.begin_words = pl->begin_words;
    p.status = ctx->d_status;
    p.q_stride_t = a->q_stride_t;
    p.q_stride_h = a->q_stride_h;
    p.out_stride_t = a->out_stride_t;
    p.out_stride_h = a->out_stride_h;
    p.n_kv_heads = pl->n_kv_heads;
    p.group = pl->n_heads / pl->n_kv_heads;
    for (p.page_shift = 0; (1u << p.page_shift) < pl->page_size; ++p.page_shift) {}
    p.pt_stride = c->page_table_stride;
    p.n_pages = c->n_pages;
    p.window = pl->window;
    p.n_sinks = pl->n_sinks;
    // scale 0 (every visible key counts alike): a factor that keeps -inf * factor = -inf in the masked columns
    p.scale_log2 = std::max(a->scale * 1.4426950408889634f, 1e-30f);
    CUtensorMap tm_k, tm_v;
    const uint64_t rows = (uint64_t)c->n_pages * c->n_kv_heads * c->page_size;
    mf_status st = get_tensor_map(ctx, c->k_pool, rows, c->head_dim, c->page_size, 64, &tm_k, 2);
    if (st == MF_OK) st = get_tensor_map(ctx, c->v_pool, rows, c->head_dim, c->page_size, 64, &tm_v, 2);
    if (st != MF_OK) return st;
    // q as (64 columns, heads, tokens, column halves): a box is the kv head's query heads of a stream's tokens (tm_q) or of
    // one token (tm_q1) and lands as rows (token, head) of 128 bytes
    CUtensorMap tm_q{}, tm_q1{};
    if (pl->tokens) {
        const uint64_t dims[4] = {64, pl->n_heads, pl->tokens, c->head_dim / 64};
        const uint64_t strides[3] = {a->q_stride_h * 2, a->q_stride_t * 2, 128};
        const uint32_t box[4] = {64, p.group, kTile / p.group, 1}, box1[4] = {64, p.group, 1, 1};
        bool ok = false, ok1 = false;
        st = encode_f16_map(ctx, &tm_q, a->q, 4, dims, strides, box, &ok);
        if (st == MF_OK) st = encode_f16_map(ctx, &tm_q1, a->q, 4, dims, strides, box1, &ok1);
        if (st != MF_OK) return st;
        if (ok && ok1) p.q_tokens = pl->tokens;
    }
    // A captured launch is not ordered here: it follows the plan as it stands at the replay.
    const bool elsewhere = pl->updated_on != ctx->stream && !mf_is_capturing(ctx);
    if (elsewhere) {
        if ((st = check_cuda(ctx, cudaStreamWaitEvent(ctx->stream, pl->staged[pl->next_stage ^ 1], 0), "chunk plan: order")) != MF_OK) return st;
        // (the event below stands for all such launches: a second stream's follow the first's)
        if (pl->used_elsewhere && (st = check_cuda(ctx, cudaStreamWaitEvent(ctx->stream, pl->used, 0), "chunk plan: order")) != MF_OK) return st;
    }
    auto *kern = chunk_kernel(c->head_dim);
    const uint32_t smem = smem_bytes(c->head_dim);
    kern<<<pl->n_ctas, kThreads, smem, ctx->stream>>>(tm_k, tm_v, tm_q, tm_q1, p);
    st = check_launch(ctx, "chunk_tc_kernel");
    if (st != MF_OK) return st;
    ctx->note_plain_launch(false);
    if (elsewhere) {
        if ((st = check_cuda(ctx, cudaEventRecord(pl->used, ctx->stream), "chunk plan: order")) != MF_OK) return st;
        pl->used_elsewhere = true;
    }
    return MF_OK;
}

}  // extern "C"
