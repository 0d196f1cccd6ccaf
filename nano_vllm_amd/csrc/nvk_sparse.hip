// nvk_sparse.hip -- decode attention over the cache blocks that a cheap score selects (nvk_block_index_*, nvk_sparse_decode*).
//
// The index keeps, for every block, kv-head and channel, the least and the largest key element: lo and hi.  For a query
// head q, q . k <= sum_c max(q_c, 0) hi_c + min(q_c, 0) lo_c for every key k of the block; the largest of these bounds over the
// group's query heads is the block's score for that kv-head.  A decode call reads the first blocks, the last blocks and the
// best-scored others, and attends to their tokens alone (Attention::paged_attention, include/core/attention.hpp:82-159, over
// a subset): with block_size 16 it moves 1/16 of the cache for the scores and top / blocks of it for the attention.
//
// Kernels: nvk_index_update_kernel behind an append, and for a decode call score and attend, with the selection and the join of
// chunks inside or beside the latter.  gfx950 only; no CPU path.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "nvk_addr.hip.h"
#include "nvk_chunk_join.hip.h"
#include "nvk_hip_util.h"

struct nvk_block_index
{
    nvk_pool *pool = nullptr;
    int       n_layers = 0, num_blocks = 0, block_size = 0, n_kv_heads = 0, head_dim = 0, device = 0;
    size_t    layer_floats = 0; // num_blocks * n_kv_heads * 2 * head_dim
    float    *base = nullptr;   // [layer][block][kv-head][lo | hi][head_dim]
    float    *ws = nullptr;     // scores | chosen blocks | partial results
    size_t    ws_floats = 0;
    int      *arrivals = nullptr; // of the join inside the attention kernel, zero between launches
    size_t    arrivals_cap = 0;
    long long ws_generation = 0;
};

namespace nvk {

constexpr int kSparseWaves = 4;

struct SparseArgs
{
    const float *k, *v;    // the layer's slabs [block][offset][kv-head][head_dim]
    float       *bounds;   // the layer's index
    const float *q;        // [num_seqs, n_heads, head_dim]
    float       *out;
    const int   *tables, *ctx_lens, *starts; // starts: index update only
    int          num_seqs, max_blocks, n_heads, group, n_kv_heads, head_dim, num_blocks, block_size;
    int          top, first, last;
    float       *scores;   // [num_seqs, n_kv_heads, max_nb]
    int         *chosen;   // [num_seqs, n_kv_heads, top]: what the selection kernel makes, of lines with more blocks than `top`
    int         *selected; // the caller's list of the same shape, of all lines, or null
    int          max_nb;                   // blocks of the longest context
    int          blocks_per_wave;          // score
    int          blocks_per_chunk, chunks; // attend
    int          head_sets;                // attend: workgroups along the group's heads
    float        scale_log2e;
    float       *ws_o, *ws_ml;
    int         *arrivals; // one for each (sequence, set of heads, kv-head), or null: the join kernel follows
};

typedef float  f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// rows of keys, values and bounds are read once by a launch: not worth keeping in the caches
__device__ __forceinline__ float4 load_once(const float *p)
{
    const f32x4 t = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p));
    return make_float4(t.x, t.y, t.z, t.w);
}

// Exchanges inside a row of sixteen lanes, on the vector pipe.
// lane ^ 1, lane ^ 2, lane ^ 7, and turned by 4 and by 8
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kFlip8 = 0x141, kTurn4 = 0x124, kTurn8 = 0x128;
template <int C> __device__ __forceinline__ float across(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), C, 0xF, 0xF, true));
}
template <int C> __device__ __forceinline__ double across(double x)
{
    const long long b = __double_as_longlong(x);
    const int       lo = __builtin_amdgcn_update_dpp(0, (int)b, C, 0xF, 0xF, true);
    const int       hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), C, 0xF, 0xF, true);
    return __longlong_as_double((long long)hi << 32 | (unsigned)lo);
}
// Sums of a over lanes l and l ^ 32 in the lower half of the wave, of b in the upper; of a over l and l ^ 16 in rows 0 and 2, of
// b in rows 1 and 3.
__device__ __forceinline__ float fold32(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float fold16(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Of a value that lane l carries for head l % HG: head h's (a constant after unrolling), in every lane of the quad.
template <int HG> __device__ __forceinline__ float of_head(float x, int h)
{
    if constexpr (HG == 1)
        return x;
    return h == 0 ? across<0x00>(x) : h == 1 ? across<0x55>(x) : h == 2 ? across<0xAA>(x) : across<0xFF>(x);
}

__device__ __forceinline__ int context_of(const SparseArgs &a, int seq)
{
    const int64_t room = (int64_t)min(a.max_nb, a.max_blocks) * a.block_size;
    return (int)min((int64_t)max(a.ctx_lens[seq], 0), room);
}

// ---- the index: lo and hi of each block that the tokens [starts[s], ctx_lens[s]) lie in, from all its tokens ------------
// SHARED: a workgroup takes 256 channels of a block's rows (all kv-heads side by side), its waves every fourth token each, and they
// meet in LDS; otherwise 1024 channels, a wave 256 for all tokens.  Bound by the keys it reads.
// Long blocks, and fewer blocks than CUs, are shared.  (8 kv-heads of 128 channels; 64 blocks of 16 tokens: 4.4 us shared, 5.3 not; 512
// blocks: 10.0 and 8.6; 8192 blocks: 127 and 128, 4.7 TB/s; of 64 tokens: 64 blocks 6.4 and 11.0, 2048 blocks 105 and 114.)
template <bool SHARED> __global__ void __launch_bounds__(64 * kSparseWaves) nvk_index_update_kernel(const SparseArgs a, int slots, int runs)
{
    constexpr int W = SHARED ? kSparseWaves : 1; // waves that share tokens
    __shared__ __attribute__((aligned(16))) float s_lo[W][256], s_hi[W][256];
    unsigned  id = blockIdx.x;
    const int run = (int)(id % (unsigned)runs);
    id /= (unsigned)runs;
    const int slot = (int)(id % (unsigned)slots), seq = (int)(id / (unsigned)slots);
    const int bs = a.block_size;
    const int end = (int)min((int64_t)a.ctx_lens[seq], (int64_t)a.max_blocks * bs), begin = max(a.starts[seq], 0);
    const int b = begin / bs + slot;
    if (end <= begin || (int64_t)b * bs >= end)
        return;
    const int pb = a.tables[(int64_t)seq * a.max_blocks + b];
    if (pb < 0 || pb >= a.num_blocks)
        return;
    const int    held = min(bs, end - b * bs), row = a.n_kv_heads * a.head_dim;
    const int    lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (SHARED ? run : run * kSparseWaves + wave) * 256 + 4 * lane;
    const float *k = a.k + (int64_t)pb * bs * row + c;
    // a NaN stays: x < lo is false for it, and lo < x once lo is one
    auto take = [](float &lo, float &hi, float x, float y) {
        lo = (x < lo || x != x) ? x : lo;
        hi = (y > hi || y != y) ? y : hi;
    };
    float4 lo = make_float4(INFINITY, INFINITY, INFINITY, INFINITY), hi = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (c < row) {
#pragma unroll 8
        for (int t = SHARED ? wave : 0; t < held; t += W) {
            const float4 x = *reinterpret_cast<const float4 *>(k + (int64_t)t * row);
            take(lo.x, hi.x, x.x, x.x), take(lo.y, hi.y, x.y, x.y), take(lo.z, hi.z, x.z, x.z), take(lo.w, hi.w, x.w, x.w);
        }
    }
    if constexpr (SHARED) {
        *reinterpret_cast<float4 *>(&s_lo[wave][4 * lane]) = lo, *reinterpret_cast<float4 *>(&s_hi[wave][4 * lane]) = hi;
        __syncthreads();
        if (wave > 0)
            return;
#pragma unroll
        for (int w = 1; w < W; w++) {
            const float4 x = *reinterpret_cast<const float4 *>(&s_lo[w][4 * lane]), y = *reinterpret_cast<const float4 *>(&s_hi[w][4 * lane]);
            take(lo.x, hi.x, x.x, y.x), take(lo.y, hi.y, x.y, y.y), take(lo.z, hi.z, x.z, y.z), take(lo.w, hi.w, x.w, y.w);
        }
    }
    if (c >= row)
        return;
    float *to = a.bounds + ((int64_t)pb * a.n_kv_heads + c / a.head_dim) * 2 * a.head_dim + c % a.head_dim;
    *reinterpret_cast<float4 *>(to)              = lo;
    *reinterpret_cast<float4 *>(to + a.head_dim) = hi;
}

// min(q, 0) for the least key element, max(q, 0) for the largest; a NaN stays one (fminf and fmaxf would make it 0; comparisons
// instead become branches around the loads: 1 x 8192 21.9 us for 18.8)
__device__ __forceinline__ float weight_of(float q, bool low)
{
    return low ? __builtin_elementwise_minimum(q, 0.f) : __builtin_elementwise_maximum(q, 0.f);
}

// ---- scores ---------------------------------------------------------------------------------------------------------
// With w = [min(q, 0) | max(q, 0)] a bound is the dot product of w with a block's [lo | hi], 2 head_dim contiguous floats.  It is
// summed in 64 bits (every product of two fp32 numbers is exact there) and rounded once: which of two close blocks is
// read does not hang on the order of a sum.  Sixteen lanes share a block, four blocks a wave; w stays in registers for HG
// query heads at a time.  NV = float4s of [lo | hi] per lane.  Bound by the bounds it reads: 16 sequences of 2048 blocks, eight kv-heads
// of 128 channels, four heads each: 268 MB in 47.5 us, 5.6 TB/s, with two groups of bounds on their way.
template <int NV, int HG> __global__ void __launch_bounds__(64 * kSparseWaves) nvk_block_score_kernel(const SparseArgs a, int slots)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, sub = lane >> 4;
    unsigned  id = blockIdx.x;
    const int kvh = (int)(id % (unsigned)a.n_kv_heads);
    id /= (unsigned)a.n_kv_heads;
    const int slot = (int)(id % (unsigned)slots), seq = (int)(id / (unsigned)slots);
    const int ctx = context_of(a, seq), nb = (ctx + a.block_size - 1) / a.block_size;
    const int begin = (slot * kSparseWaves + wave) * a.blocks_per_wave, end = min(begin + a.blocks_per_wave, nb);
    if (nb <= a.top || begin >= end) // everything is read: no scores needed
        return;
    const int  hd = a.head_dim;
    float     *score = a.scores + ((int64_t)seq * a.n_kv_heads + kvh) * a.max_nb;
    // (a wave's blocks are at most 128: a lane keeps the place of two)
    int entry[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        entry[i] = min(max(a.tables[(int64_t)seq * a.max_blocks + min(begin + 64 * i + lane, end - 1)], 0), a.num_blocks - 1);
    for (int h0 = 0; h0 < a.group; h0 += HG) {
        double w[HG][NV][4];
#pragma unroll
        for (int h = 0; h < HG; h++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (l16 + 16 * j) * 4; // place in [lo | hi]
                float4    x = make_float4(0.f, 0.f, 0.f, 0.f);
                // (a set that ends beyond the group repeats its last head: the maximum is the same)
                if (c < 2 * hd)
                    x = *reinterpret_cast<const float4 *>(
                        a.q + ((int64_t)seq * a.n_heads + kvh * a.group + min(h0 + h, a.group - 1)) * hd + (c < hd ? c : c - hd));
                const bool low = c < hd;
                w[h][j][0] = weight_of(x.x, low), w[h][j][1] = weight_of(x.y, low);
                w[h][j][2] = weight_of(x.z, low), w[h][j][3] = weight_of(x.w, low);
            }
        constexpr int RING = NV < 8 ? 3 : 2; // groups of four blocks: one in work, the others on their way
        float4        x[RING][NV];
        auto   fetch = [&](float4 (&to)[NV], int b0) {
            const int    at = min(b0 + sub, end - 1) - begin, lo = __shfl(entry[0], at & 63), hi = __shfl(entry[1], at & 63);
            const int    pb = at < 64 ? lo : hi;
            const float *src = a.bounds + ((int64_t)pb * a.n_kv_heads + kvh) * 2 * hd;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const int c = (l16 + 16 * j) * 4;
                to[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c < 2 * hd)
                    to[j] = load_once(src + c);
            }
        };
        auto take = [&](const float4 (&x)[NV], int b0) {
            double s[HG];
#pragma unroll
            for (int h = 0; h < HG; h++)
                s[h] = 0.0;
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int h = 0; h < HG; h++) {
                    s[h] = fma(w[h][j][0], (double)x[j].x, s[h]), s[h] = fma(w[h][j][1], (double)x[j].y, s[h]);
                    s[h] = fma(w[h][j][2], (double)x[j].z, s[h]), s[h] = fma(w[h][j][3], (double)x[j].w, s[h]);
                }
            // sums over the block's sixteen lanes; with several heads, each exchange halves the heads a lane carries
            double mine;
            if constexpr (HG == 4) {
                const bool   o1 = lane & 1, o2 = lane & 2;
                const double t0 = (o1 ? s[2] : s[0]) + across<kSwap1>(o1 ? s[0] : s[2]);
                const double t1 = (o1 ? s[3] : s[1]) + across<kSwap1>(o1 ? s[1] : s[3]);
                mine = (o2 ? t1 : t0) + across<kSwap2>(o2 ? t0 : t1);
            }
            else if constexpr (HG == 2) {
                const bool o1 = lane & 1;
                mine = (o1 ? s[1] : s[0]) + across<kSwap1>(o1 ? s[0] : s[1]);
                mine += across<kSwap2>(mine);
            }
            else {
                mine = s[0] + across<kSwap1>(s[0]);
                mine += across<kSwap2>(mine);
            }
            mine += across<kTurn4>(mine);
            mine += across<kTurn8>(mine);
            float best = (float)mine;
            best       = best != best ? INFINITY : best; // no number: as high as can be
            best       = fmaxf(best, across<kSwap1>(best));
            best       = fmaxf(best, across<kSwap2>(best));
            if (l16 == 0 && b0 + sub < end)
                score[b0 + sub] = h0 > 0 ? fmaxf(score[b0 + sub], best) : best;
        };
#pragma unroll
        for (int d = 0; d + 1 < RING; d++)
            if (begin + 4 * d < end)
                fetch(x[d], begin + 4 * d);
        for (int b0 = begin; b0 < end; b0 += 4 * RING) {
#pragma unroll
            for (int d = 0; d < RING; d++)
                if (b0 + 4 * d < end) {
                    if (b0 + 4 * (d + RING - 1) < end)
                        fetch(x[(d + RING - 1) % RING], b0 + 4 * (d + RING - 1));
                    take(x[d], b0 + 4 * d);
                }
        }
    }
}

// The same for groups of more than four heads, on fp64 matrix instructions: heads are the rows, sixteen blocks the columns of a
// product, so that the bounds are read once for sixteen heads.  The order of a contraction is free: a lane holds four
// neighbouring bounds of its block, and the weights are laid out to match.  An instruction reads half a line of each block, so the
// loads go through the caches (past them 4 % more time).  (Whole calls, this kernel and the one above in two passes: 16 x 32768, 8
// kv-heads of 8 heads and 128 channels 150 and 167 us; 30 x 9000, 4 of 7 and 64 channels 32 and 46; 4 of 5 and 32 channels 25 and 36.)
template <int NV>
__global__ void __launch_bounds__(64 * kSparseWaves, NV == 4 ? 1 : 2) nvk_block_score_wide_kernel(const SparseArgs a, int slots)
{
    constexpr int J = 4 * NV; // float4s of [lo | hi] per lane
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    unsigned  id = blockIdx.x;
    const int kvh = (int)(id % (unsigned)a.n_kv_heads);
    id /= (unsigned)a.n_kv_heads;
    const int slot = (int)(id % (unsigned)slots), seq = (int)(id / (unsigned)slots);
    const int ctx = context_of(a, seq), nb = (ctx + a.block_size - 1) / a.block_size;
    const int begin = (slot * kSparseWaves + wave) * a.blocks_per_wave, end = min(begin + a.blocks_per_wave, nb);
    if (nb <= a.top || begin >= end) // everything is read: no scores needed
        return;
    const int hd = a.head_dim;
    float    *score = a.scores + ((int64_t)seq * a.n_kv_heads + kvh) * a.max_nb;
    int       entry[2]; // (a wave's blocks are at most 128)
#pragma unroll
    for (int i = 0; i < 2; i++)
        entry[i] = min(max(a.tables[(int64_t)seq * a.max_blocks + min(begin + 64 * i + lane, end - 1)], 0), a.num_blocks - 1);
    const int tiles = (end - begin + 15) / 16;
    for (int h0 = 0; h0 < a.group; h0 += 16) {
        double w[J][4];
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int c = 16 * j + 4 * g; // place in [lo | hi]
            float4    x = make_float4(0.f, 0.f, 0.f, 0.f);
            // (a set that ends beyond the group repeats its last head: the maximum is the same)
            if (c < 2 * hd)
                x = *reinterpret_cast<const float4 *>(
                    a.q + ((int64_t)seq * a.n_heads + kvh * a.group + min(h0 + l16, a.group - 1)) * hd + (c < hd ? c : c - hd));
            const bool low = c < hd;
            w[j][0] = weight_of(x.x, low), w[j][1] = weight_of(x.y, low);
            w[j][2] = weight_of(x.z, low), w[j][3] = weight_of(x.w, low);
        }
        auto fetch = [&](float4 (&to)[J], int t) {
            const int    at = min(16 * t + l16, end - 1 - begin), lo = __shfl(entry[0], at & 63), hi = __shfl(entry[1], at & 63);
            const float *src = a.bounds + ((int64_t)(at < 64 ? lo : hi) * a.n_kv_heads + kvh) * 2 * hd;
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int c = 16 * j + 4 * g;
                to[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c < 2 * hd)
                    to[j] = *reinterpret_cast<const float4 *>(src + c);
            }
        };
        // (no branch between the products and what reads them: a wait for a result was once seen lost across one)
        auto take = [&](const float4 (&x)[J], int t) {
            f64x4 s0 = {0.0, 0.0, 0.0, 0.0}, s1 = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int j = 0; j < J; j++) {
                s0 = __builtin_amdgcn_mfma_f64_16x16x4f64(w[j][0], (double)x[j].x, s0, 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f64_16x16x4f64(w[j][1], (double)x[j].y, s1, 0, 0, 0);
                s0 = __builtin_amdgcn_mfma_f64_16x16x4f64(w[j][2], (double)x[j].z, s0, 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f64_16x16x4f64(w[j][3], (double)x[j].w, s1, 0, 0, 0);
            }
            float best = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float r = (float)(s0[i] + s1[i]);
                best = fmaxf(best, r != r ? INFINITY : r); // no number: as high as can be
            }
            best = fmaxf(best, __shfl_xor(best, 16));
            best = fmaxf(best, __shfl_xor(best, 32));
            const int b = begin + 16 * t + l16;
            if (g == 0 && b < end)
                score[b] = h0 > 0 ? fmaxf(score[b], best) : best;
        };
        float4 one[J], two[J]; // in turn
        fetch(one, 0);
        for (int t = 0; t < tiles; t += 2) {
            if (t + 1 < tiles)
                fetch(two, t + 1);
            take(one, t);
            if (t + 1 < tiles) {
                if (t + 2 < tiles)
                    fetch(one, t + 2);
                take(two, t + 1);
            }
        }
    }
}

// ---- selection --------------------------------------------------------------------------------------------------------
// The key of the last block that is read is found by counting passes over the four bytes of the keys; read are the blocks above
// it, and as many of those level with it as are left, lowest first, in ascending order.  Where the 256 threads of an attention
// workgroup can keep all keys (2048 blocks, eight each) every one of them selects for itself (1 x 8192: 18.8 us, with a launch for
// the selection 23.6; 16 x 32768: 104.5 and 108).  Beyond that a kernel of its own does, with keys in registers up to 32768 blocks
// (1 x 131072: 42.5 us, 57.7 with keys made again for every pass).  Bound by latency: counting in LDS between barriers.
constexpr int kHeldKeys  = 8;
constexpr int kHeldBlocks = 64 * kSparseWaves * kHeldKeys;

__device__ __forceinline__ unsigned block_key(const SparseArgs &a, const float *score, int b, int nb)
{
    if (b < a.first || b >= nb - a.last)
        return 0xffffffffu; // read always (no score maps there)
    const unsigned u = __float_as_uint(score[b] + 0.f); // (-0 is 0)
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// sum over the lanes up to and with this one
__device__ __forceinline__ int scan_wave(int x)
{
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false); // from 1, 2, 4, 8 lanes below in the row
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); // the last lane of row 0 to row 1, of row 2 to row 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); // the last lane of the lower half to the upper
    return x;
}

// One pass, after the counts of byte (key >> shift) of the keys with this prefix are complete: extends the prefix by the byte
// in which the `left`-th key from above lies, and takes the keys above it off `left`.  Every wave does it for itself.
__device__ __forceinline__ void next_byte(const int *count, int shift, unsigned &prefix, int &left)
{
    const int  lane = threadIdx.x & 63;
    const int4 c4 = *reinterpret_cast<const int4 *>(count + 252 - 4 * lane); // bins from the top: four to a lane
    const int  c[4] = {c4.w, c4.z, c4.y, c4.x};
    const int  sum = (c[0] + c[1]) + (c[2] + c[3]);
    int        before = scan_wave(sum) - sum; // of the lanes before this one
    int        bin = -1, rest = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (before < left && before + c[i] >= left) // exactly one bin of one lane
            bin = 255 - (4 * lane + i), rest = left - before;
        before += c[i];
    }
    const int from = __ffsll((unsigned long long)__ballot(bin >= 0)) - 1;
    prefix |= (unsigned)__builtin_amdgcn_readlane(bin, from) << shift;
    left = __builtin_amdgcn_readlane(rest, from);
}

// The selection by a workgroup of WAVES waves that keep KEYS keys a thread: take(at, block, i) for each block that is read, `at` its
// place in ascending order, i the number among the thread's blocks, which are first .. first + share - 1.
template <int WAVES, int KEYS> struct HeldSelection
{
    int      first, share;
    unsigned key[KEYS];
    __device__ __forceinline__ bool there(int i, int nb) const { return i < share && first + i < nb; }
    __device__ __forceinline__ HeldSelection(const SparseArgs &a, const float *score, int nb)
    {
        share = (nb + 64 * WAVES - 1) / (64 * WAVES), first = share * (int)threadIdx.x;
#pragma unroll
        for (int i = 0; i < KEYS; i++)
            key[i] = there(i, nb) ? block_key(a, score, first + i, nb) : 0u;
    }
    template <class F> __device__ __forceinline__ void run(int top, int nb, F &&take)
    {
        __shared__ __attribute__((aligned(16))) int s_count[4][256];
        __shared__ int s_wave[2][WAVES];
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        for (int i = tid; i < 4 * 256; i += 64 * WAVES)
            s_count[i >> 8][i & 255] = 0;
        __syncthreads();
        unsigned edge = 0;
        int      ties = top;
        // The upper bytes of scores are mostly one or two: counted by the wave, one addition for each.
#pragma unroll
        for (int i = 0; i < KEYS; i++)
            if (i < share) {
                unsigned long long left = __ballot(first + i < nb);
                while (left) {
                    const unsigned           top_byte = (unsigned)__builtin_amdgcn_readlane((int)key[i], __ffsll(left) - 1) >> 24;
                    const unsigned long long same = __ballot((key[i] >> 24) == top_byte) & left;
                    if (lane == 0)
                        atomicAdd(&s_count[0][top_byte], __popcll(same));
                    left &= ~same & (left - 1); // (the first one is among the same)
                }
            }
        __syncthreads();
        next_byte(s_count[0], 24, edge, ties);
#pragma unroll
        for (int pass = 1; pass < 4; pass++) {
            const int shift = 24 - 8 * pass;
#pragma unroll
            for (int i = 0; i < KEYS; i++)
                if (there(i, nb) && (key[i] >> (shift + 8)) == (edge >> (shift + 8)))
                    atomicAdd(&s_count[pass][(key[i] >> shift) & 255u], 1);
            __syncthreads();
            next_byte(s_count[pass], shift, edge, ties);
            if (s_count[pass][(edge >> shift) & 255u] == ties) { // all of the edge's bin is read: the bytes below do not matter
                ties = nb;
                break;
            }
        }
        int above = 0, even = 0;
#pragma unroll
        for (int i = 0; i < KEYS; i++)
            above += there(i, nb) && key[i] > edge, even += there(i, nb) && key[i] == edge;
        int pa = scan_wave(above), pe = scan_wave(even);
        if (lane == 63)
            s_wave[0][wave] = pa, s_wave[1][wave] = pe;
        __syncthreads();
        pa -= above, pe -= even;
#pragma unroll
        for (int w = 0; w < WAVES; w++)
            pa += w < wave ? s_wave[0][w] : 0, pe += w < wave ? s_wave[1][w] : 0;
#pragma unroll
        for (int i = 0; i < KEYS; i++) {
            const bool hi = there(i, nb) && key[i] > edge, level = there(i, nb) && key[i] == edge;
            if (hi || (level && pe < ties))
                take(pa + min(pe, ties), first + i, i);
            pa += hi, pe += level;
        }
    }
};

constexpr int kSelectThreads = 1024;

// a workgroup per (sequence, kv-head)
template <int KEYS> __global__ void __launch_bounds__(kSelectThreads) nvk_block_select_held_kernel(const SparseArgs a)
{
    const int line = blockIdx.x, ctx = context_of(a, line / a.n_kv_heads), nb = (ctx + a.block_size - 1) / a.block_size;
    if (nb <= a.top)
        return;
    int *chosen = a.chosen + (int64_t)line * a.top;
    HeldSelection<kSelectThreads / 64, KEYS> held(a, a.scores + (int64_t)line * a.max_nb, nb);
    held.run(a.top, nb, [&](int at, int b, int) { chosen[at] = b; });
}

// the same for any number of blocks, whose keys are made again for every pass
__global__ void __launch_bounds__(kSelectThreads) nvk_block_select_kernel(const SparseArgs a)
{
    constexpr int W = kSelectThreads / 64;
    __shared__ __attribute__((aligned(16))) int s_count[4][256];
    __shared__ int s_wave[2][2][W];
    const int    line = blockIdx.x, seq = line / a.n_kv_heads;
    const int    tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int    ctx = context_of(a, seq), nb = (ctx + a.block_size - 1) / a.block_size;
    int         *chosen = a.chosen + (int64_t)line * a.top;
    const float *score = a.scores + (int64_t)line * a.max_nb;
    if (nb <= a.top)
        return;
    s_count[tid >> 8][tid & 255] = 0;
    __syncthreads();
    unsigned edge = 0;
    int      ties = a.top; // in the end: of the blocks with the edge's key, so many are read
#pragma unroll
    for (int pass = 0; pass < 4; pass++) {
        const int shift = 24 - 8 * pass;
        for (int b = tid; b < nb; b += kSelectThreads) {
            const unsigned key = block_key(a, score, b, nb);
            if (pass == 0 || (key >> (shift + 8)) == (edge >> (shift + 8)))
                atomicAdd(&s_count[pass][(key >> shift) & 255u], 1);
        }
        __syncthreads();
        next_byte(s_count[pass], shift, edge, ties);
    }
    int placed = 0, level = 0;
    for (int b0 = 0, turn = 0; b0 < nb; b0 += kSelectThreads, turn ^= 1) { // (the counts alternate between two places)
        const int      b = b0 + tid;
        const unsigned key = b < nb ? block_key(a, score, b, nb) : 0u;
        const bool     above = b < nb && key > edge, even = b < nb && key == edge;
        const unsigned long long below = ((unsigned long long)1 << lane) - 1;
        const unsigned long long ma = __ballot(above), me = __ballot(even);
        if (lane == 0)
            s_wave[turn][0][wave] = __popcll(ma), s_wave[turn][1][wave] = __popcll(me);
        __syncthreads();
        int pa = 0, pe = 0, ta = 0, te = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            pa += w < wave ? s_wave[turn][0][w] : 0, pe += w < wave ? s_wave[turn][1][w] : 0;
            ta += s_wave[turn][0][w], te += s_wave[turn][1][w];
        }
        pa += __popcll(ma & below), pe += __popcll(me & below);
        // before this block: pa above it, and of the pe level ones those that are among the first `ties`
        if (above || (even && level + pe < ties))
            chosen[placed + pa + min(max(ties - level, 0), pe)] = b;
        placed += ta + min(max(ties - level, 0), te);
        level += te;
    }
}

// ---- attention over the chosen blocks -----------------------------------------------------------------------------------
// A wave takes eight tokens a step, eight lanes each: a lane holds NV float4s of the row (lane 8 apart: whole lines per
// token), dots them with HG query heads, and keeps maximum, sum and output of its own eight-lane group -- nothing
// crosses the groups before the end.  Bound by the keys and values it reads, behind the latency of the selection: 128 of 2048
// blocks of 16 sequences, eight kv-heads of 128 channels: 268 MB in 54 us, 48 (5.6 TB/s) where contexts are read whole.
template <int NV, int HG, bool SELECT>
__global__ void __launch_bounds__(64 * kSparseWaves, NV == 1 ? 4 : NV <= 4 || HG == 1 ? 2 : 1) nvk_sparse_attn_kernel(const SparseArgs a)
{
    constexpr int kMostBlocks = 64; // of a chunk
    __shared__ int   s_phys[kMostBlocks], s_first[kMostBlocks];
    __shared__ float s_m[kSparseWaves][HG], s_l[kSparseWaves][HG];
    __shared__ __attribute__((aligned(16))) float s_o[kSparseWaves][HG][32 * NV];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l8 = lane & 7, tg = lane >> 3;
    unsigned  id = blockIdx.x;
    const int kvh = (int)(id % (unsigned)a.n_kv_heads);
    id /= (unsigned)a.n_kv_heads;
    const int set = (int)(id % (unsigned)a.head_sets);
    id /= (unsigned)a.head_sets;
    const int chunk = (int)(id % (unsigned)a.chunks), seq = (int)(id / (unsigned)a.chunks);
    const int hd = a.head_dim, bs = a.block_size;
    const int ctx = context_of(a, seq), nb = (ctx + bs - 1) / bs, n = min(nb, a.top);
    const int begin = chunk * a.blocks_per_chunk, count = min(a.blocks_per_chunk, n - begin);
    const int parts = max((n + a.blocks_per_chunk - 1) / a.blocks_per_chunk, 1);
    if (chunk >= parts)
        return;
    const int64_t pair = (int64_t)seq * a.n_kv_heads + kvh;
    const int    *table = a.tables + (int64_t)seq * a.max_blocks;
    int          *selected = a.selected && chunk == 0 && set == 0 ? a.selected + pair * a.top : nullptr; // one workgroup tells
    if (nb <= a.top) { // everything is read
        if ((int)threadIdx.x < count)
            s_first[threadIdx.x] = begin + threadIdx.x, s_phys[threadIdx.x] = table[begin + threadIdx.x];
        if (selected)
            for (int i = threadIdx.x; i < a.top; i += 64 * kSparseWaves)
                selected[i] = i < nb ? i : -1;
    }
    else if constexpr (SELECT) {
        HeldSelection<kSparseWaves, kHeldKeys> held(a, a.scores + pair * a.max_nb, nb);
        int entry[kHeldKeys]; // (of all the thread's blocks, while the keys are counted, rather than of the picks behind it)
#pragma unroll
        for (int i = 0; i < kHeldKeys; i++)
            entry[i] = held.there(i, nb) ? table[held.first + i] : 0;
        held.run(a.top, nb, [&](int at, int b, int i) {
            if (at >= begin && at < begin + count)
                s_first[at - begin] = b, s_phys[at - begin] = entry[i];
            if (selected)
                selected[at] = b;
        });
    }
    else if ((int)threadIdx.x < count) { // (the list is the selection kernel's)
        const int b = min(max(a.chosen[pair * a.top + begin + threadIdx.x], 0), nb - 1);
        s_first[threadIdx.x] = b, s_phys[threadIdx.x] = table[b];
    }
    __syncthreads();
    if ((int)threadIdx.x < count)
        s_first[threadIdx.x] *= bs, s_phys[threadIdx.x] = min(max(s_phys[threadIdx.x], 0), a.num_blocks - 1);
    __syncthreads();

    const int head0 = kvh * a.group + set * HG, heads = min(HG, a.group - set * HG);
    float4    q[HG][NV], o[HG][NV];
#pragma unroll
    for (int h = 0; h < HG; h++)
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (l8 + 8 * j) * 4;
            q[h][j] = make_float4(0.f, 0.f, 0.f, 0.f), o[h][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (h < heads && c < hd)
                q[h][j] = *reinterpret_cast<const float4 *>(a.q + ((int64_t)seq * a.n_heads + head0 + h) * hd + c);
        }
    // each lane carries the statistics of head lane % HG of its eight-lane group
    float m = -INFINITY, l = 0.f;

    const int tokens = max(count, 0) * bs, steps = (tokens + 7) / 8;
    auto fetch = [&](int step, float4 (&k)[NV], float4 (&v)[NV]) -> bool {
        const int  t = step * 8 + tg;
        const int  e = min(t / bs, max(count - 1, 0)), off = t - t / bs * bs;
        const bool there = t < tokens && s_first[e] + off < ctx;
        const int64_t at = (((int64_t)s_phys[e] * bs + off) * a.n_kv_heads + kvh) * hd;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int c = (l8 + 8 * j) * 4;
            k[j] = make_float4(0.f, 0.f, 0.f, 0.f), v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (there && c < hd) {
                k[j] = load_once(a.k + at + c);
                v[j] = load_once(a.v + at + c);
            }
        }
        return there;
    };
    constexpr int AHEAD = NV == 1 ? 4 : 1; // steps on their way: of narrow rows more
    float4        kn[AHEAD][NV], vn[AHEAD][NV];
    bool          next_there[AHEAD];
#pragma unroll
    for (int d = 0; d < AHEAD; d++) {
        next_there[d] = false;
        if (wave + d * kSparseWaves < steps)
            next_there[d] = fetch(wave + d * kSparseWaves, kn[d], vn[d]);
    }
    auto work = [&](const float4 (&k)[NV], const float4 (&v)[NV], const bool there) {
        float s[HG];
#pragma unroll
        for (int h = 0; h < HG; h++) {
            s[h] = 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                s[h] = fmaf(q[h][j].x, k[j].x, s[h]), s[h] = fmaf(q[h][j].y, k[j].y, s[h]);
                s[h] = fmaf(q[h][j].z, k[j].z, s[h]), s[h] = fmaf(q[h][j].w, k[j].w, s[h]);
            }
        }
        // over the token's eight lanes (l and l ^ 7 first); afterwards lane l carries head l % HG
#pragma unroll
        for (int h = 0; h < HG; h++)
            s[h] += across<kFlip8>(s[h]);
        float mine;
        if constexpr (HG == 4) {
            const bool  o1 = lane & 1, o2 = lane & 2;
            const float t0 = (o1 ? s[1] : s[0]) + across<kSwap1>(o1 ? s[0] : s[1]);
            const float t1 = (o1 ? s[3] : s[2]) + across<kSwap1>(o1 ? s[2] : s[3]);
            mine = (o2 ? t1 : t0) + across<kSwap2>(o2 ? t0 : t1);
        }
        else if constexpr (HG == 2) {
            const bool o1 = lane & 1;
            mine = (o1 ? s[1] : s[0]) + across<kSwap1>(o1 ? s[0] : s[1]);
            mine += across<kSwap2>(mine);
        }
        else {
            mine = s[0] + across<kSwap1>(s[0]);
            mine += across<kSwap2>(mine);
        }
        const float t = there ? mine * a.scale_log2e : -INFINITY;
        if (__any(t > m)) {
            const float m_new = fmaxf(m, t);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int h = 0; h < HG; h++) {
                const float x = of_head<HG>(alpha, h);
#pragma unroll
                for (int j = 0; j < NV; j++)
                    o[h][j].x *= x, o[h][j].y *= x, o[h][j].z *= x, o[h][j].w *= x;
            }
        }
        const float p = there ? __builtin_amdgcn_exp2f(t - (m == -INFINITY ? 0.f : m)) : 0.f;
        l += p;
#pragma unroll
        for (int h = 0; h < HG; h++) {
            const float x = of_head<HG>(p, h);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                o[h][j].x = fmaf(x, v[j].x, o[h][j].x), o[h][j].y = fmaf(x, v[j].y, o[h][j].y);
                o[h][j].z = fmaf(x, v[j].z, o[h][j].z), o[h][j].w = fmaf(x, v[j].w, o[h][j].w);
            }
        }
    };
    for (int step = wave; step < steps; step += AHEAD * kSparseWaves)
#pragma unroll
        for (int d = 0; d < AHEAD; d++)
            if (d == 0 || step + d * kSparseWaves < steps) {
                float4 k[NV], v[NV];
#pragma unroll
                for (int j = 0; j < NV; j++)
                    k[j] = kn[d][j], v[j] = vn[d][j];
                const bool there = next_there[d];
                if (step + (d + AHEAD) * kSparseWaves < steps)
                    next_there[d] = fetch(step + (d + AHEAD) * kSparseWaves, kn[d], vn[d]);
                work(k, v, there);
            }

    // the eight groups of the wave, then the waves
    float M = m;
    M       = fmaxf(M, __shfl_xor(M, 8));
    M       = fmaxf(M, __shfl_xor(M, 16));
    M       = fmaxf(M, __shfl_xor(M, 32));
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    l *= alpha;
    l += __shfl_xor(l, 8);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < HG)
        s_m[wave][lane] = M, s_l[wave][lane] = l;
#pragma unroll
    for (int h = 0; h < HG; h++) {
        const float x = of_head<HG>(alpha, h);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            // row r of the wave ends with component r, twice in its sixteen lanes
            float y = fold16(fold32(o[h][j].x * x, o[h][j].z * x), fold32(o[h][j].y * x, o[h][j].w * x));
            y += across<kTurn8>(y);
            if ((lane & 8) == 0)
                s_o[wave][h][(l8 + 8 * j) * 4 + (lane >> 4)] = y;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < heads * (hd / 2); e += 64 * kSparseWaves) {
        const int h = e / (hd / 2), c = e % (hd / 2) * 2;
        float     Mh = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kSparseWaves; w++)
            Mh = fmaxf(Mh, s_m[w][h]);
#pragma unroll
        for (int w = 0; w < kSparseWaves; w++) {
            const float f = s_m[w][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][h] - Mh);
            L += s_l[w][h] * f;
            x += s_o[w][h][c] * f, y += s_o[w][h][c + 1] * f;
        }
        const int64_t line = (int64_t)seq * a.n_heads + head0 + h;
        if (parts > 1) {
            store_through(a.ws_o + (line * a.chunks + chunk) * hd + c, x, y);
            if (c == 0)
                store_through(a.ws_ml + (line * a.chunks + chunk) * 2, Mh, L);
        }
        else { // (no token: zeros; scores that are all -infinity: 0 / 0)
            a.out[line * hd + c]     = ctx == 0 ? 0.f : x / L;
            a.out[line * hd + c + 1] = ctx == 0 ? 0.f : y / L;
        }
    }
    if (parts == 1 || !a.arrivals || !arrived_last(a.arrivals + ((int64_t)seq * a.head_sets + set) * a.n_kv_heads + kvh, parts))
        return;
    for (int e = threadIdx.x; e < heads * (hd / 4); e += 64 * kSparseWaves) {
        const int64_t line = (int64_t)seq * a.n_heads + head0 + e / (hd / 4);
        const int     c = e % (hd / 4) * 4;
        const float4  x = join_few<true>(a.ws_o + line * a.chunks * hd + c, a.ws_ml + line * a.chunks * 2, parts, hd, false);
        store_four(a.out + line * hd + c, x.x, x.y, x.z, x.w);
    }
}

// a workgroup per (sequence, head)
__global__ void __launch_bounds__(kJoinThreads) nvk_sparse_join_kernel(const SparseArgs a)
{
    const int64_t line = blockIdx.x;
    const int     ctx = context_of(a, (int)(line / a.n_heads)), nb = (ctx + a.block_size - 1) / a.block_size;
    const int     n = max((min(nb, a.top) + a.blocks_per_chunk - 1) / a.blocks_per_chunk, 1);
    if (n == 1)
        return; // (written straight to `out`)
    join_chunks(a.ws_o + line * a.chunks * a.head_dim, a.ws_ml + line * a.chunks * 2, n, a.head_dim, false, a.out + line * a.head_dim);
}

} // namespace nvk

namespace {

using nvk::SparseArgs;

constexpr int kCus = 256; // MI355X

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

struct SparseShape
{
    int    max_nb = 0, blocks_per_wave = 4, score_slots = 1, blocks_per_chunk = 1, chunks = 1, head_sets = 1, hg = 1;
    bool   wide = false; // scores on matrix instructions
    bool   inside = false, select_inside = false; // the attention kernel joins the chunks itself, selects itself
    size_t score_floats = 0, chosen_ints = 0, part_floats = 0, arrivals = 0;
    size_t floats() const { return score_floats + chosen_ints + part_floats; }
};

size_t to_line(size_t floats) { return (floats + 31) / 32 * 32; }

SparseShape sparse_shape(const nvk_block_index *x, int num_seqs, int n_heads, int max_ctx, int top)
{
    SparseShape s;
    const int   group = n_heads / x->n_kv_heads;
    s.max_nb = (int)ceil_div(max_ctx, x->block_size);
    s.hg     = group == 1 ? 1 : group == 2 ? 2 : 4;
    if (x->head_dim > 128) // registers
        s.hg = std::min(s.hg, 2);
    s.head_sets = (int)ceil_div(group, s.hg);
    // scores: four blocks a wave at least, 128 at most, in between two workgroups for every CU: one round of the chip.  (16 sequences
    // of 2048 blocks, eight kv-heads: 47.5 us with 128 blocks a wave, 53.2 in two rounds of 64.)
    const long long lines = (long long)num_seqs * x->n_kv_heads;
    s.wide = group > 4 && x->head_dim <= 128;
    const long long per = lines * s.max_nb / ((s.wide && x->head_dim > 64 ? 1LL : 2LL) * kCus * nvk::kSparseWaves), unit = s.wide ? 16 : 4;
    s.blocks_per_wave = (int)std::min(128LL, std::max(unit, per / unit * unit));
    s.score_slots     = (int)std::max(1LL, ceil_div(s.max_nb, (long long)s.blocks_per_wave * nvk::kSparseWaves));
    // attention: the chosen blocks are cut while all workgroups still run at once (two fit a CU, of narrow rows four, of the widest
    // one), into pieces of eight tokens a wave at least and 64 blocks at most.  Four would fit with 64 channels too, but each
    // selects for itself.  (32 channels, 166 and 500 blocks: 34 and 46 us with four, 44 and 51 with two; 64 channels, 500 blocks: 31.7
    // and 27.6; 256 channels, heads by two: 84 us with one, 97 with two.)
    const int       n = std::max(1, std::min(s.max_nb, top));
    const long long tasks = lines * s.head_sets;
    const int       per_cu = x->head_dim <= 32 ? 4 : x->head_dim <= 128 || s.hg == 1 ? 2 : 1;
    const long long fit = std::max(1LL, (long long)per_cu * kCus / std::max(tasks, 1LL));
    const long long least = ceil_div(8LL * nvk::kSparseWaves, x->block_size);
    s.blocks_per_chunk = (int)std::min(64LL, std::max(least, ceil_div(n, fit)));
    // (rather sixteen pieces, which the kernel joins itself, than more short ones)
    if (ceil_div(n, s.blocks_per_chunk) > nvk::kJoinInside && ceil_div(n, nvk::kJoinInside) * x->block_size <= 256)
        s.blocks_per_chunk = (int)std::min(64LL, ceil_div(n, nvk::kJoinInside));
    s.blocks_per_chunk = std::max(1, s.blocks_per_chunk);
    s.chunks           = (int)ceil_div(n, s.blocks_per_chunk);
    s.score_floats     = s.max_nb > top ? to_line((size_t)lines * s.max_nb) : 0;
    s.select_inside    = s.max_nb <= nvk::kHeldBlocks;
    s.chosen_ints      = s.select_inside || s.max_nb <= top ? 0 : to_line((size_t)lines * top);
    s.inside           = s.chunks > 1 && s.chunks <= nvk::kJoinInside;
    s.arrivals         = s.inside ? (size_t)tasks : 0;
    s.part_floats      = s.chunks > 1 ? (size_t)num_seqs * n_heads * s.chunks * (x->head_dim + 2) : 0;
    return s;
}

int reserve(nvk_block_index *x, size_t floats, size_t arrivals, hipStream_t st, const char *who)
{
    const int rc = nvk::grow_buffer(&x->ws, &x->ws_floats, &x->ws_generation, floats, st, who);
    return rc != NVK_OK ? rc : nvk::grow_counters(&x->arrivals, &x->arrivals_cap, &x->ws_generation, arrivals, st, who);
}

// What no call of up to this shape passes, fewer sequences (which are cut into more chunks) and fewer blocks among them: as
// sparse_shape cuts, lines times chunks are at most the workgroups that fit the chip times the heads of one, or chunks are 64 blocks.
size_t most_floats(const nvk_block_index *x, int num_seqs, int n_heads, int max_ctx, int top)
{
    const SparseShape s = sparse_shape(x, num_seqs, n_heads, max_ctx, top);
    const size_t      lines = (size_t)num_seqs * x->n_kv_heads;
    const long long   parts = std::max(4LL * kCus * s.hg, (long long)num_seqs * n_heads * ceil_div(std::min(s.max_nb, top), 64));
    return to_line(lines * s.max_nb) + to_line(lines * std::min(s.max_nb, top)) + (size_t)parts * (x->head_dim + 2);
}

template <int NV, int HG> void launch_sparse(const SparseArgs &a, const SparseShape &s, bool score, hipStream_t st)
{
    const unsigned lines = (unsigned)a.num_seqs * (unsigned)a.n_kv_heads;
    const dim3 scores(lines * (unsigned)s.score_slots), threads(64 * nvk::kSparseWaves);
    if constexpr (NV < 8 && HG == 4)
        if (score && s.wide)
            hipLaunchKernelGGL((nvk::nvk_block_score_wide_kernel<NV>), scores, threads, 0, st, a, s.score_slots);
    if (score && !s.wide)
        hipLaunchKernelGGL((nvk::nvk_block_score_kernel<NV, HG>), scores, threads, 0, st, a, s.score_slots);
    const dim3 grid(lines * (unsigned)s.head_sets * (unsigned)s.chunks), block(64 * nvk::kSparseWaves);
    if (s.select_inside)
        hipLaunchKernelGGL((nvk::nvk_sparse_attn_kernel<NV, HG, true>), grid, block, 0, st, a);
    else {
        if (score) { // (4 x 4096 blocks: 56.5 us with 16 keys a thread, 63.0 with 32; 18750 blocks: 43.3 with 32, 79.4 with none)
            const dim3 all(nvk::kSelectThreads);
            if (s.max_nb <= 16 * nvk::kSelectThreads)
                hipLaunchKernelGGL(nvk::nvk_block_select_held_kernel<16>, dim3(lines), all, 0, st, a);
            else if (s.max_nb <= 32 * nvk::kSelectThreads)
                hipLaunchKernelGGL(nvk::nvk_block_select_held_kernel<32>, dim3(lines), all, 0, st, a);
            else
                hipLaunchKernelGGL(nvk::nvk_block_select_kernel, dim3(lines), all, 0, st, a);
        }
        hipLaunchKernelGGL((nvk::nvk_sparse_attn_kernel<NV, HG, false>), grid, block, 0, st, a);
    }
}

template <int NV> void launch_heads(const SparseArgs &a, const SparseShape &s, bool score, hipStream_t st)
{
    if constexpr (NV < 8)
        if (s.hg == 4) {
            launch_sparse<NV, 4>(a, s, score, st);
            return;
        }
    if (s.hg == 2)
        launch_sparse<NV, 2>(a, s, score, st);
    else
        launch_sparse<NV, 1>(a, s, score, st);
}

int check_index(const nvk_block_index *x, int layer, const char *who)
{
    if (!x)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null index", who);
    if (layer < 0 || layer >= x->n_layers)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: layer %d outside [0,%d)", who, layer, x->n_layers);
    return NVK_OK;
}

int fill_args(const nvk_block_index *x, int layer, SparseArgs *a)
{
    void     *k = nullptr, *v = nullptr;
    const int rc = nvk_pool_layer_ptrs(x->pool, layer, &k, &v);
    if (rc != NVK_OK)
        return rc;
    a->k = (const float *)k, a->v = (const float *)v, a->bounds = x->base + (size_t)layer * x->layer_floats;
    a->n_kv_heads = x->n_kv_heads, a->head_dim = x->head_dim, a->num_blocks = x->num_blocks, a->block_size = x->block_size;
    return NVK_OK;
}

int pool_stream(const nvk_block_index *x, void *stream, hipStream_t *st)
{
    if (stream) {
        *st = (hipStream_t)stream;
        return NVK_OK;
    }
    void     *own = nullptr;
    const int rc = nvk_pool_stream(x->pool, &own);
    *st          = (hipStream_t)own;
    return rc;
}

int enqueue_update(nvk_block_index *x, int layer, int num_seqs, const int *tables, int max_blocks, const int *starts,
                   const int *ctx_lens, int max_new, hipStream_t st, const char *who)
{
    SparseArgs a{};
    const int  rc = fill_args(x, layer, &a);
    if (rc != NVK_OK)
        return rc;
    a.tables = tables, a.max_blocks = max_blocks, a.starts = starts, a.ctx_lens = ctx_lens, a.num_seqs = num_seqs;
    // max_new tokens lie in at most this many blocks
    const long long slots = std::min((long long)max_blocks, ceil_div((long long)max_new + x->block_size - 1, x->block_size));
    const bool      shared = x->block_size > 16 || slots * num_seqs < kCus;
    const long long runs = ceil_div((long long)x->n_kv_heads * x->head_dim, shared ? 256 : 256 * nvk::kSparseWaves), groups = slots * num_seqs * runs;
    if (!nvk::grid_fits(groups, 64 * nvk::kSparseWaves))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: %lld blocks", who, slots * num_seqs);
    if (shared)
        hipLaunchKernelGGL(nvk::nvk_index_update_kernel<true>, dim3((unsigned)groups), dim3(64 * nvk::kSparseWaves), 0, st, a, (int)slots, (int)runs);
    else
        hipLaunchKernelGGL(nvk::nvk_index_update_kernel<false>, dim3((unsigned)groups), dim3(64 * nvk::kSparseWaves), 0, st, a, (int)slots, (int)runs);
    NVK_HIP_TRY(hipGetLastError());
    return NVK_OK;
}

int check_sparse(const nvk_block_index *x, int layer, int num_seqs, int n_heads, int max_blocks, int max_ctx, int top, int first,
                 int last, const char *who)
{
    const int rc = check_index(x, layer, who);
    if (rc != NVK_OK)
        return rc;
    if (num_seqs < 0 || max_blocks <= 0 || max_ctx < 0 || (long long)max_blocks * x->block_size > nvk::kMostTokens
        || max_ctx > nvk::kMostTokens)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: bad sizes (num_seqs %d, max_blocks %d, max_ctx %d)", who, num_seqs, max_blocks, max_ctx);
    if (n_heads <= 0 || n_heads % x->n_kv_heads != 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: n_heads %d is no multiple of n_kv_heads %d", who, n_heads, x->n_kv_heads);
    if (first < 0 || last < 1 || top < 1 || (long long)first + last > top)
        return nvk::fail(NVK_ERR_INVALID_ARG,
                         "%s: first %d, last %d (at least 1: the newest block is always read) and top %d (at least both)", who,
                         first, last, top);
    return NVK_OK;
}

int enqueue_sparse(nvk_block_index *x, int layer, int num_seqs, int n_heads, const float *q, const int *tables, int max_blocks,
                   const int *ctx_lens, int max_ctx, int top, int first, int last, float *out, int *selected, hipStream_t st,
                   const char *who)
{
    if (!selected) // (a list of its own is no wider than the longest context)
        top = std::min(top, std::max((int)ceil_div(max_ctx, x->block_size), 1));
    const SparseShape s = sparse_shape(x, num_seqs, n_heads, max_ctx, top);
    const long long   lines = (long long)num_seqs * x->n_kv_heads;
    const bool        joins = s.chunks > 1 && !s.inside;
    if (!nvk::grid_fits(lines * s.score_slots, 64 * nvk::kSparseWaves) || !nvk::grid_fits(lines * s.head_sets * s.chunks, 64 * nvk::kSparseWaves)
        || (!s.select_inside && !nvk::grid_fits(lines, nvk::kSelectThreads)) || (joins && !nvk::grid_fits((long long)num_seqs * n_heads, nvk::kJoinThreads)))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: too many workgroups", who);
    int rc = reserve(x, s.floats(), s.arrivals, st, who);
    if (rc != NVK_OK)
        return rc;
    SparseArgs a{};
    rc = fill_args(x, layer, &a);
    if (rc != NVK_OK)
        return rc;
    a.q = q, a.out = out, a.tables = tables, a.max_blocks = max_blocks, a.ctx_lens = ctx_lens, a.num_seqs = num_seqs;
    a.n_heads = n_heads, a.group = n_heads / x->n_kv_heads, a.top = top, a.first = first, a.last = last;
    a.max_nb = s.max_nb, a.blocks_per_wave = s.blocks_per_wave, a.blocks_per_chunk = s.blocks_per_chunk, a.chunks = s.chunks;
    a.head_sets = s.head_sets, a.scale_log2e = (float)(1.4426950408889634 / std::sqrt((double)x->head_dim));
    a.scores = x->ws;
    a.selected = selected, a.chosen = selected ? selected : (int *)(x->ws + s.score_floats);
    a.ws_o   = x->ws + s.score_floats + s.chosen_ints;
    a.ws_ml  = a.ws_o + (size_t)num_seqs * n_heads * s.chunks * x->head_dim;
    a.arrivals = s.inside ? x->arrivals : nullptr;
    const bool score = s.max_nb > top;
    const int  nv = x->head_dim <= 32 ? 1 : x->head_dim <= 64 ? 2 : x->head_dim <= 128 ? 4 : 8;
    switch (nv) {
    case 1: launch_heads<1>(a, s, score, st); break;
    case 2: launch_heads<2>(a, s, score, st); break;
    case 4: launch_heads<4>(a, s, score, st); break;
    default: launch_heads<8>(a, s, score, st); break;
    }
    NVK_HIP_TRY(hipGetLastError());
    if (joins) {
        hipLaunchKernelGGL(nvk::nvk_sparse_join_kernel, dim3((unsigned)(num_seqs * n_heads)), dim3(nvk::kJoinThreads), 0, st, a);
        NVK_HIP_TRY(hipGetLastError());
    }
    return NVK_OK;
}

} // namespace

extern "C" {

int nvk_block_index_create(nvk_pool *pool, nvk_block_index **out_index)
{
    if (!out_index)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_block_index_create: out_index is null");
    *out_index = nullptr;
    int g[6];
    if (!pool || nvk_pool_geometry(pool, g) != NVK_OK)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_block_index_create: null pool");
    if (g[4] % 4 != 0 || g[4] > 256)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_block_index_create: head_dim %d (a multiple of 4, at most 256)", g[4]);
    nvk_block_index *x = new (std::nothrow) nvk_block_index();
    if (!x)
        return nvk::fail(NVK_ERR_OOM, "nvk_block_index_create: host allocation failed");
    x->pool = pool, x->n_layers = g[0], x->num_blocks = g[1], x->block_size = g[2], x->n_kv_heads = g[3], x->head_dim = g[4];
    x->device = g[5], x->layer_floats = (size_t)g[1] * g[3] * 2 * g[4];
    nvk::DeviceScope scope(x->device);
    const size_t     bytes = x->layer_floats * (size_t)x->n_layers * sizeof(float);
    hipError_t       e = scope.ok ? hipMalloc((void **)&x->base, bytes) : hipErrorInvalidDevice;
    if (e == hipSuccess)
        e = hipMemset(x->base, 0, bytes); // the bounds of the zeros that a pool starts with
    if (e == hipSuccess)
        e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        const int rc = nvk::fail(e == hipErrorOutOfMemory ? NVK_ERR_OOM : NVK_ERR_HIP, "nvk_block_index_create: %s (%zu bytes requested)",
                                 hipGetErrorString(e), bytes);
        (void)hipGetLastError();
        nvk_block_index_destroy(x);
        return rc;
    }
    *out_index = x;
    return NVK_OK;
}

int nvk_block_index_destroy(nvk_block_index *index)
{
    if (!index)
        return NVK_OK;
    nvk::DeviceScope scope(index->device); // (a release path: goes on whatever the switch returned)
    (void)hipDeviceSynchronize();          // launches on any stream may still use it
    if (index->base)
        (void)hipFree(index->base);
    if (index->ws)
        (void)hipFree(index->ws);
    if (index->arrivals)
        (void)hipFree(index->arrivals);
    delete index;
    return NVK_OK;
}

int nvk_block_index_layer_ptr(const nvk_block_index *index, int layer, void **bounds_dev)
{
    const int rc = check_index(index, layer, "nvk_block_index_layer_ptr");
    if (rc != NVK_OK)
        return rc;
    if (!bounds_dev)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_block_index_layer_ptr: null pointer");
    *bounds_dev = index->base + (size_t)layer * index->layer_floats;
    return NVK_OK;
}

long long nvk_block_index_workspace_generation(const nvk_block_index *index) { return index ? index->ws_generation : -1; }

int nvk_block_index_reserve_workspace(nvk_block_index *index, int num_seqs, int n_heads, int max_ctx, int top_blocks)
{
    const char *who = "nvk_block_index_reserve_workspace";
    const int   rc = check_sparse(index, 0, num_seqs, n_heads, 1, max_ctx, top_blocks, 0, 1, who);
    if (rc != NVK_OK)
        return rc;
    NVK_SCOPE(index->device);
    hipStream_t st = nullptr;
    const int   rs = pool_stream(index, nullptr, &st);
    if (rs != NVK_OK)
        return rs;
    const size_t tasks = (size_t)num_seqs * n_heads; // (no more workgroups meet than there are heads)
    return reserve(index, most_floats(index, num_seqs, n_heads, max_ctx, top_blocks), std::max(tasks, 4 * (size_t)kCus), st, who);
}

int nvk_block_index_update(nvk_block_index *index, int layer, int num_seqs, const int *block_tables, int max_blocks,
                           const int *starts, const int *ctx_lens, int max_new, int ptr_kind, void *stream)
{
    const char *who = "nvk_block_index_update";
    int         rc = check_index(index, layer, who);
    if (rc != NVK_OK)
        return rc;
    if (ptr_kind != NVK_PTR_HOST && ptr_kind != NVK_PTR_DEVICE)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: ptr_kind %d", who, ptr_kind);
    if (num_seqs < 0 || max_blocks <= 0 || max_new < 0 || (long long)max_blocks * index->block_size > nvk::kMostTokens)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: bad sizes (num_seqs %d, max_blocks %d, max_new %d)", who, num_seqs, max_blocks, max_new);
    if (num_seqs == 0 || (max_new == 0 && ptr_kind == NVK_PTR_DEVICE))
        return NVK_OK;
    if (!block_tables || !starts || !ctx_lens)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pointer", who);
    NVK_SCOPE(index->device);
    hipStream_t st = nullptr;
    rc             = pool_stream(index, ptr_kind == NVK_PTR_DEVICE ? stream : nullptr, &st);
    if (rc != NVK_OK)
        return rc;
    if (ptr_kind == NVK_PTR_DEVICE)
        return enqueue_update(index, layer, num_seqs, block_tables, max_blocks, starts, ctx_lens, max_new, st, who);

    rc = nvk::check_tables(block_tables, num_seqs, max_blocks, ctx_lens, index->block_size, index->num_blocks, who);
    if (rc != NVK_OK)
        return rc;
    int most = 0;
    for (int s = 0; s < num_seqs; s++) {
        if (starts[s] < 0 || starts[s] > ctx_lens[s])
            return nvk::fail(NVK_ERR_INVALID_ARG, "%s: start %d of sequence %d, whose context is %d tokens", who, starts[s], s, ctx_lens[s]);
        most = std::max(most, ctx_lens[s] - starts[s]);
    }
    if (most == 0)
        return NVK_OK;
    nvk::Staging g;
    const int    it = g.add(block_tables, (size_t)num_seqs * max_blocks * sizeof(int)), is = g.add(starts, (size_t)num_seqs * sizeof(int)),
              ic = g.add(ctx_lens, (size_t)num_seqs * sizeof(int));
    NVK_HIP_TRY(g.upload(st));
    rc = enqueue_update(index, layer, num_seqs, g.at<int>(it), max_blocks, g.at<int>(is), g.at<int>(ic), most, st, who);
    NVK_HIP_TRY(hipStreamSynchronize(st));
    return rc;
}

int nvk_sparse_decode_device(nvk_block_index *index, int layer, int num_seqs, int n_heads, const float *q_dev,
                             const int *block_tables_dev, int max_blocks, const int *ctx_lens_dev, int max_ctx, int top_blocks,
                             int first_blocks, int last_blocks, float *out_dev, int *selected_dev, void *stream)
{
    const char *who = "nvk_sparse_decode_device";
    int         rc = check_sparse(index, layer, num_seqs, n_heads, max_blocks, max_ctx, top_blocks, first_blocks, last_blocks, who);
    if (rc != NVK_OK || num_seqs == 0)
        return rc;
    if (!q_dev || !block_tables_dev || !ctx_lens_dev || !out_dev)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pointer", who);
    if ((uintptr_t)q_dev % 16 != 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: q is not 16-byte aligned", who);
    if (!nvk::for_floats(out_dev))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: out is not aligned to its type", who);
    NVK_SCOPE(index->device);
    hipStream_t st = nullptr;
    rc             = pool_stream(index, stream, &st);
    if (rc != NVK_OK)
        return rc;
    return enqueue_sparse(index, layer, num_seqs, n_heads, q_dev, block_tables_dev, max_blocks, ctx_lens_dev, max_ctx, top_blocks,
                          first_blocks, last_blocks, out_dev, selected_dev, st, who);
}

int nvk_sparse_decode(nvk_block_index *index, int layer, int num_seqs, int n_heads, const float *q, const int *block_tables,
                      int max_blocks, const int *ctx_lens, int top_blocks, int first_blocks, int last_blocks, float *out,
                      int *selected)
{
    const char *who = "nvk_sparse_decode";
    int         rc = check_sparse(index, layer, num_seqs, n_heads, max_blocks, 0, top_blocks, first_blocks, last_blocks, who);
    if (rc != NVK_OK || num_seqs == 0)
        return rc;
    if (!q || !block_tables || !ctx_lens || !out)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pointer", who);
    rc = nvk::check_tables(block_tables, num_seqs, max_blocks, ctx_lens, index->block_size, index->num_blocks, who);
    if (rc != NVK_OK)
        return rc;
    NVK_SCOPE(index->device);
    hipStream_t st = nullptr;
    rc             = pool_stream(index, nullptr, &st);
    if (rc != NVK_OK)
        return rc;
    const int    max_ctx = *std::max_element(ctx_lens, ctx_lens + num_seqs);
    const size_t qb = (size_t)num_seqs * n_heads * index->head_dim * sizeof(float);
    const size_t sb = (size_t)num_seqs * index->n_kv_heads * top_blocks * sizeof(int);
    nvk::Staging g;
    const int    iq = g.add(q, qb), io = g.add(nullptr, qb), it = g.add(block_tables, (size_t)num_seqs * max_blocks * sizeof(int)),
              ic = g.add(ctx_lens, (size_t)num_seqs * sizeof(int)), is = g.add(nullptr, selected ? sb : 0);
    NVK_HIP_TRY(g.upload(st));
    rc = enqueue_sparse(index, layer, num_seqs, n_heads, g.at<float>(iq), g.at<int>(it), max_blocks, g.at<int>(ic), max_ctx, top_blocks,
                        first_blocks, last_blocks, g.at<float>(io), selected ? g.at<int>(is) : nullptr, st, who);
    if (rc == NVK_OK) {
        NVK_HIP_TRY(hipMemcpyAsync(out, g.at<float>(io), qb, hipMemcpyDeviceToHost, st));
        if (selected)
            NVK_HIP_TRY(hipMemcpyAsync(selected, g.at<int>(is), sb, hipMemcpyDeviceToHost, st));
    }
    NVK_HIP_TRY(hipStreamSynchronize(st));
    return rc;
}

} // extern "C"
