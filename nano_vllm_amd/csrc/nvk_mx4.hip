// nvk_mx4.hip -- the 4-bit paged KV pool (nvk_mx4_pool_*) and attention over it (nvk_mx4_decode*, nvk_mx4_prefill*).
//
// out[r, h] = softmax(q[r, h] . K^T / sqrt(head_dim)) V over the tokens that row r sees, K and V behind a block table, the
// group of n_heads / n_kv_heads query heads sharing a kv-head (Attention::paged_attention, include/core/attention.hpp:82-159,
// over another cache).  Codes times a power of two are bf16 numbers exactly, and a query element or a probability is exactly
// the sum of three bf16 numbers (its mantissa cut into three bytes), so both products run on bf16 matrix instructions
// with fp32 accumulators and no rounding of their own: three instructions for one, still five times the fp32 matrix rate.
// gfx950 only; no CPU path.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "nvk_hip_util.h"
#include "nvk_mx4.hip.h"

namespace nvk {

#ifndef MX4_AHEAD
#define MX4_AHEAD 1
#endif
#ifndef MX4_WGS
#define MX4_WGS 2LL
#endif
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float  f32x4 __attribute__((ext_vector_type(4)));

struct Mx4AttnArgs
{
    Mx4Layer     mx;
    const float *q;   // [rows, n_heads, head_dim]
    float       *out; // the same
    const int   *row_offsets; // [num_seqs + 1] or null: row s belongs to sequence s
    const int   *tables, *ctx_lens;
    int          num_seqs, max_blocks, n_heads, group, total_rows;
    int          col_blocks;   // workgroups along a sequence's (row, head) columns
    int          chunk_tokens; // tokens a workgroup takes (a multiple of 32)
    int          chunks;       // chunks along the longest context
    float        scale_log2e;  // log2(e) / sqrt(head_dim)
    float       *ws_o, *ws_ml; // partial results where chunks > 1: [rows * heads][chunks][head_dim], [..][2]
};

// The three bf16 numbers whose sum is x, packed for two values at a time.  Truncation: each residual is exact.
__device__ __forceinline__ unsigned high_halves(float lo, float hi)
{
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float residual(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

struct Pieces // eight values in three bf16 vectors
{
    bf16x8 p[3];
};
__device__ __forceinline__ Pieces split8(const float (&x)[8])
{
    union
    {
        unsigned u[4];
        bf16x8   v;
    } w[3];
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        r[i] = x[i];
#pragma unroll
    for (int s = 0; s < 3; s++) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[s].u[i] = high_halves(r[2 * i], r[2 * i + 1]);
        if (s < 2)
#pragma unroll
            for (int i = 0; i < 8; i++)
                r[i] = residual(r[i]);
    }
    Pieces o;
    o.p[0] = w[0].v, o.p[1] = w[1].v, o.p[2] = w[2].v;
    return o;
}

// two channels of byte `B` of a dword of codes, times the scale
template <int B> __device__ __forceinline__ unsigned two_values(unsigned codes, float scale)
{
    const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B);
    return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned two_values_at(unsigned codes, float scale, int b)
{
    switch (b) { // (b is a constant after unrolling)
    case 0: return two_values<0>(codes, scale);
    case 1: return two_values<1>(codes, scale);
    case 2: return two_values<2>(codes, scale);
    default: return two_values<3>(codes, scale);
    }
}
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// What a lane holds of one tile.
template <int KK> struct Mx4Raw
{
    static constexpr int KS = KK == 8 ? 2 : 1; // groups that a lane's channels of K lie in
    unsigned k[KK], v[KK], vs;
    unsigned ks[KS];
};

template <int KK> __device__ __forceinline__ void load_tile(Mx4Raw<KK> &r, const unsigned char *tile, int lane)
{
    const int g = lane >> 4, l16 = lane & 15;
    const unsigned *kc = reinterpret_cast<const unsigned *>(tile + l16 * 16 * KK + g * 4 * KK);
    const unsigned *vc = reinterpret_cast<const unsigned *>(tile + mx4_v_at(KK) + lane * 4 * KK);
    if constexpr (KK >= 4) {
#pragma unroll
        for (int i = 0; i < KK; i += 4) {
            const uint4 a = *reinterpret_cast<const uint4 *>(kc + i), b = *reinterpret_cast<const uint4 *>(vc + i);
            r.k[i] = a.x, r.k[i + 1] = a.y, r.k[i + 2] = a.z, r.k[i + 3] = a.w;
            r.v[i] = b.x, r.v[i + 1] = b.y, r.v[i + 2] = b.z, r.v[i + 3] = b.w;
        }
    }
    else if constexpr (KK == 2) {
        const uint2 a = *reinterpret_cast<const uint2 *>(kc), b = *reinterpret_cast<const uint2 *>(vc);
        r.k[0] = a.x, r.k[1] = a.y, r.v[0] = b.x, r.v[1] = b.y;
    }
    else
        r.k[0] = kc[0], r.v[0] = vc[0];
    // K: channels g*8*KK .. of token l16; V: channels l16*2*KK .. of tokens 4g .. 4g+3
    if constexpr (KK == 8) {
        r.ks[0] = tile[mx4_ks_at(KK) + (2 * g) * kMx4Tile + l16];
        r.ks[1] = tile[mx4_ks_at(KK) + (2 * g + 1) * kMx4Tile + l16];
    }
    else
        r.ks[0] = tile[mx4_ks_at(KK) + (g * KK / 4) * kMx4Tile + l16];
    r.vs = *reinterpret_cast<const unsigned *>(tile + mx4_vs_at(KK) + (l16 * KK / 16) * kMx4Tile + 4 * g);
}

// One wave: NC * 16 columns ((row, head of the group) pairs of one kv-head) against the tokens of its part of a chunk.
//   S^T = K Q^T     A = K [16 tokens x 32 channels], B = Q^T [32 channels x 16 columns] -> lane (g, col): tokens 4g .. 4g+3
//   O^T = V^T P^T   A = V^T [16 channels x 32 tokens], B = P^T [32 tokens x 16 columns]
// The order of channels (in S) and of tokens (in O) along a contraction is free, so it is chosen such that the lane that holds
// a probability after S is the lane that needs it for O: the softmax touches no LDS, and a column's statistics need
// two lane exchanges a step.  WT waves of a workgroup take steps of 32 tokens in turn (few columns: decode) and join through
// LDS at the end, or WC waves take different columns over the same tokens (prefill).
template <int KK, int NC, int WT, int WC>
__global__ void __launch_bounds__(64 * WT * WC, KK == 8 ? 1 : 2) nvk_mx4_attn_kernel(const Mx4AttnArgs a)
{
    constexpr int HDP = 32 * KK;
    constexpr int AHEAD = MX4_AHEAD;
    static_assert(WT == 1 || (WC == 1 && NC == 1), "waves share either the tokens or the columns");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    const int wt = WT > 1 ? wave : 0, wc = WC > 1 ? wave : 0;

    // workgroup -> (sequence, column block, chunk, kv-head); kv-heads change fastest: eight kv-heads are eight XCDs, and the
    // column blocks of one kv-head meet in the L2 of one
    unsigned  id = blockIdx.x;
    const int kvh = (int)(id % (unsigned)a.mx.n_kv_heads);
    id /= (unsigned)a.mx.n_kv_heads;
    const int chunk = (int)(id % (unsigned)a.chunks);
    id /= (unsigned)a.chunks;
    const int cb = (int)(id % (unsigned)a.col_blocks);
    const int seq = (int)(id / (unsigned)a.col_blocks);

    int row0 = seq, rows = 1;
    if (a.row_offsets) {
        row0 = a.row_offsets[seq];
        rows = min(a.row_offsets[seq + 1], a.total_rows) - row0;
        if (row0 < 0 || rows <= 0)
            return;
    }
    const int bs = a.mx.block_size;
    const int ctx = min(max(a.ctx_lens[seq], 0), (int)min((int64_t)a.max_blocks * bs, (int64_t)0x7fffffff));
    const int columns = rows * a.group;
    const int col0 = (cb * WC + wc) * 16 * NC;
    if (cb * WC * 16 * NC >= columns)
        return;

    // a column's row sees the tokens below `limit`: all up to its own, its place being at the end of the context
    int limit[NC], out_row[NC], out_head[NC];
    int most = 0; // the largest limit of the wave's columns, and of the workgroup's
    const int last_row = min((cb + 1) * WC * 16 * NC - 1, columns - 1) / a.group;
    const int block_most = max(ctx - rows + last_row + 1, 0);
#pragma unroll
    for (int n = 0; n < NC; n++) {
        const int col = col0 + 16 * n + l16, r = col / a.group;
        out_row[n] = col < columns ? row0 + r : -1;
        out_head[n] = kvh * a.group + col % a.group;
        limit[n] = col < columns ? max(ctx - rows + r + 1, 0) : 0;
    }
    {
        const int r = min(col0 + 16 * NC - 1, columns - 1) / a.group;
        most = col0 < columns ? max(ctx - rows + r + 1, 0) : 0;
    }
    const int least = col0 < columns ? max(ctx - rows + col0 / a.group + 1, 0) : 0; // the smallest limit
    const int begin = chunk * a.chunk_tokens;
    if (chunk > 0 && begin >= block_most) // nothing of this chunk is seen (the first one writes rows that see nothing)
        return;
    const int end = min(begin + a.chunk_tokens, most);

    // Q^T operands: column l16, channels g*8*KK + kk*8 ..
    Pieces q[NC][KK];
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            float x[8];
            const int c0 = g * 8 * KK + kk * 8;
#pragma unroll
            for (int i = 0; i < 8; i++)
                x[i] = 0.f;
            if (out_row[n] >= 0 && c0 < a.mx.head_dim) {
                const float *src = a.q + ((int64_t)out_row[n] * a.n_heads + out_head[n]) * a.mx.head_dim + c0;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    x[i] = src[i];
            }
            q[n][kk] = split8(x);
        }

    f32x4 acc[NC][2 * KK];
    float m[NC], l[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) {
        m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
        for (int ct = 0; ct < 2 * KK; ct++)
            acc[n][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    unsigned poisoned[NC]; // channel groups in which a token that the column sees holds no number
#pragma unroll
    for (int n = 0; n < NC; n++)
        poisoned[n] = 0;

    // tiles of this wave: its step i covers the 32 tokens from begin + 32 * (wt + WT * i)
    const int     steps = max(0, (end - begin + 31) / 32 - wt + WT - 1) / WT;
    const int     last_tile = max((min(end, ctx) - 1) / kMx4Tile, 0);
    const int     tiles_per_block = bs / kMx4Tile;
    const int64_t head_at = (int64_t)kvh * mx4_tile_bytes(KK), tile_stride = (int64_t)a.mx.n_kv_heads * mx4_tile_bytes(KK);
    const int    *table = a.tables + (int64_t)seq * a.max_blocks;
    int           entry = 0; // lane L: the tile number in the layer of tile L % 2 of the wave's step (i & ~31) + L / 2
    auto refill = [&](int i) {
        const int t = min((begin >> 4) + 2 * (wt + WT * (i + (lane >> 1))) + (lane & 1), last_tile);
        const int b = t / tiles_per_block;
        entry = min(max(table[b], 0), a.mx.num_blocks - 1) * tiles_per_block + t % tiles_per_block;
    };
    auto fetch = [&](Mx4Raw<KK> (&r)[2], int i) {
        if ((i & 31) == 0)
            refill(i);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int e = __builtin_amdgcn_readlane(entry, 2 * (i & 31) + j);
            load_tile<KK>(r[j], a.mx.base + e * tile_stride + head_at, lane);
        }
    };

    Mx4Raw<KK> ahead[AHEAD][2]; // tiles on their way: steps i, i + 1, ..
#pragma unroll
    for (int d = 0; d < AHEAD; d++)
        if (d < steps)
            fetch(ahead[d], d);
    for (int i = 0; i < steps; i++) {
        Mx4Raw<KK> raw[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            raw[j] = ahead[0][j];
#pragma unroll
            for (int d = 0; d + 1 < AHEAD; d++)
                ahead[d][j] = ahead[d + 1][j];
        }
        if (i + AHEAD < steps)
            fetch(ahead[AHEAD - 1], i + AHEAD);
        const int t0 = begin + 32 * (wt + WT * i);

        // A group of K or V that holds no number (scale byte 255) is dealt with before any product: this compiler does not
        // keep the wait between a matrix instruction and the first read of its result across a branch, so none may stand there.
        unsigned vs[2] = {raw[0].vs, raw[1].vs};
        unsigned odd = 0; // bits 0..7: byte b of tile j's V scales; 8 + 2 j + u: K scale u of tile j
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int b = 0; b < 4; b++)
                odd |= (((vs[j] >> (8 * b)) & 255u) == 255u) ? 1u << (4 * j + b) : 0u;
#pragma unroll
            for (int u = 0; u < Mx4Raw<KK>::KS; u++)
                odd |= raw[j].ks[u] == 255u ? 1u << (8 + 2 * j + u) : 0u;
        }
        // K, one operand after another; a token whose group of K holds no number has no scores either
        bf16x8 k[2][KK];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                const float sc = scale_of(raw[j].ks[KK == 8 ? kk / 4 : 0]);
                union
                {
                    unsigned u[4];
                    bf16x8   v;
                } w;
#pragma unroll
                for (int b = 0; b < 4; b++)
                    w.u[b] = two_values_at(raw[j].k[kk], sc, b);
                k[j][kk] = w.v;
            }
        if (__any(odd != 0)) {
            const unsigned nan2 = 0x7fc07fc0u;
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
                    if ((odd >> (8 + 2 * j + (KK == 8 ? kk / 4 : 0))) & 1u)
                        k[j][kk] = __builtin_bit_cast(bf16x8, make_uint4(nan2, nan2, nan2, nan2));
                // V: the scale is taken as 0, and the columns that see the token are marked
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    unsigned long long who = __ballot((odd >> (4 * j + b)) & 1u);
                    if ((odd >> (4 * j + b)) & 1u)
                        vs[j] &= ~(255u << (8 * b));
                    for (; who; who &= who - 1) { // lane (quad, c16) tells: token 4 quad + b of tile j, group of c16
                        const int from = __ffsll((long long)who) - 1;
                        const int token = t0 + 16 * j + 4 * (from >> 4) + b;
#pragma unroll
                        for (int n = 0; n < NC; n++)
                            if (token < limit[n])
                                poisoned[n] |= 1u << ((from & 15) * KK / 16);
                    }
                }
            }
        }

        // scores
        f32x4 s[NC][2];
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                s[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int p = 2; p >= 0; p--) // small pieces first
#pragma unroll
                for (int n = 0; n < NC; n++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        s[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[j][kk], q[n][kk].p[p], s[n][j], 0, 0, 0);

        // softmax, in powers of two; p[n][j * 4 + i]: token t0 + 16 j + 4 g + i
        Pieces p[NC];
#pragma unroll
        for (int n = 0; n < NC; n++) {
            float t[8], top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; e++)
                t[e] = s[n][e >> 2][e & 3] * a.scale_log2e;
            if (t0 + 32 > least) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (t0 + 16 * (e >> 2) + 4 * g + (e & 3) >= limit[n])
                        t[e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 8; e++)
                top = fmaxf(top, t[e]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (__any(top > m[n])) {
                const float m_new = fmaxf(m[n], top);
                const float alpha = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - m_new);
                m[n] = m_new;
                l[n] *= alpha;
#pragma unroll
                for (int ct = 0; ct < 2 * KK; ct++)
                    acc[n][ct] *= alpha;
            }
            const float base = m[n] == -INFINITY ? 0.f : m[n];
            float       sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                t[e] = __builtin_amdgcn_exp2f(t[e] - base);
                sum += t[e];
            }
            l[n] += sum;
            p[n] = split8(t);
        }

        // O += P V, two channels of a lane at a time
#pragma unroll
        for (int b = 0; b < KK; b++) {
            unsigned w[2][4]; // tile, token: channels 2b and 2b + 1 of the lane's run
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int t = 0; t < 4; t++)
                    w[j][t] = two_values_at(raw[j].v[(t * KK + b) / 4], scale_of((vs[j] >> (8 * t)) & 255u), (t * KK + b) % 4);
            union
            {
                unsigned u[4];
                bf16x8   v;
            } lo, hi;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int t = 0; t < 4; t += 2) {
                    lo.u[2 * j + t / 2] = __builtin_amdgcn_perm(w[j][t + 1], w[j][t], 0x05040100u);
                    hi.u[2 * j + t / 2] = __builtin_amdgcn_perm(w[j][t + 1], w[j][t], 0x07060302u);
                }
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int e = 2; e >= 0; e--) {
                    acc[n][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo.v, p[n].p[e], acc[n][2 * b], 0, 0, 0);
                    acc[n][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi.v, p[n].p[e], acc[n][2 * b + 1], 0, 0, 0);
                }
        }
    }

    // column sums over the four lane groups; marked groups become NaN.  acc[n][ct][i]: channel (4 g + i) * 2 KK + ct
#pragma unroll
    for (int n = 0; n < NC; n++) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (poisoned[n])
#pragma unroll
            for (int ct = 0; ct < 2 * KK; ct++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if ((poisoned[n] >> (((4 * g + i) * 2 * KK + ct) / 32)) & 1u)
                        acc[n][ct][i] = __uint_as_float(0x7fc00000u);
    }

    if constexpr (WT == 1) {
#pragma unroll
        for (int n = 0; n < NC; n++) {
            if (out_row[n] < 0)
                continue;
            const int64_t line = (int64_t)out_row[n] * a.n_heads + out_head[n];
            float        *dst = a.out + line * a.mx.head_dim;
            float         norm = l[n] == 0.f ? 0.f : 1.f / l[n];
            if (a.chunks > 1) {
                dst = a.ws_o + (line * a.chunks + chunk) * a.mx.head_dim;
                norm = 1.f;
                if (g == 0) {
                    a.ws_ml[(line * a.chunks + chunk) * 2] = m[n];
                    a.ws_ml[(line * a.chunks + chunk) * 2 + 1] = l[n];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int ct = 0; ct < 2 * KK; ct++) {
                    const int c = (4 * g + i) * 2 * KK + ct;
                    if (c < a.mx.head_dim)
                        dst[c] = acc[n][ct][i] * norm;
                }
        }
    }
    else {
        // join the waves: common maximum, then a sum over LDS, 16 columns x HDP channels in passes of one wave's results
        __shared__ float s_m[WT][16], s_l[WT][16];
        __shared__ __attribute__((aligned(16))) float s_o[WT][16][HDP + 4];
        if (g == 0)
            s_m[wave][l16] = m[0], s_l[wave][l16] = l[0];
        __syncthreads();
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WT; w++)
            M = fmaxf(M, s_m[w][l16]);
        const float alpha = m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[0] - M);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int ct = 0; ct < 2 * KK; ct++)
                s_o[wave][l16][(4 * g + i) * 2 * KK + ct] = acc[0][ct][i] * alpha;
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * (HDP / 4); e += 64 * WT) {
            const int c16 = e / (HDP / 4), c = (e % (HDP / 4)) * 4;
            const int col = col0 + c16;
            if (col >= columns || c >= a.mx.head_dim)
                continue;
            float Mc = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < WT; w++)
                Mc = fmaxf(Mc, s_m[w][c16]);
            f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WT; w++) {
                L += s_m[w][c16] == -INFINITY ? 0.f : s_l[w][c16] * __builtin_amdgcn_exp2f(s_m[w][c16] - Mc);
                o += *reinterpret_cast<const f32x4 *>(&s_o[w][c16][c]);
            }
            const int64_t line = (int64_t)(row0 + col / a.group) * a.n_heads + kvh * a.group + col % a.group;
            float        *dst = a.out + line * a.mx.head_dim + c;
            if (a.chunks > 1) {
                dst = a.ws_o + (line * a.chunks + chunk) * a.mx.head_dim + c;
                if (c == 0) {
                    a.ws_ml[(line * a.chunks + chunk) * 2] = Mc;
                    a.ws_ml[(line * a.chunks + chunk) * 2 + 1] = L;
                }
            }
            else
                o *= L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int i = 0; i < 4; i++)
                dst[i] = o[i];
        }
    }
}

// Joins the chunks of a (row, head): one wave each.
__global__ void __launch_bounds__(256) nvk_mx4_merge_kernel(const Mx4AttnArgs a)
{
    const int64_t line = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int     lane = threadIdx.x & 63;
    if (line >= (int64_t)a.total_rows * a.n_heads)
        return;
    const int row = (int)(line / a.n_heads);
    int       seq = row, rows = 1, row0 = row;
    if (a.row_offsets) { // the sequence whose rows hold this one
        int lo = 0, hi = a.num_seqs; // offsets[lo] <= row < offsets[hi]
        if (row < a.row_offsets[0] || row >= a.row_offsets[a.num_seqs])
            return;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.row_offsets[mid] <= row)
                lo = mid;
            else
                hi = mid;
        }
        seq = lo, row0 = a.row_offsets[lo], rows = min(a.row_offsets[lo + 1], a.total_rows) - row0;
    }
    const int ctx = min(max(a.ctx_lens[seq], 0), (int)min((int64_t)a.max_blocks * a.mx.block_size, (int64_t)0x7fffffff));
    const int limit = max(ctx - rows + (row - row0) + 1, 0);
    const int n = min(max((limit + a.chunk_tokens - 1) / a.chunk_tokens, 1), a.chunks);
    const float *ml = a.ws_ml + line * a.chunks * 2, *o = a.ws_o + line * a.chunks * a.mx.head_dim;
    // a lane takes every 64th chunk's maximum, then its weight; the outputs are summed in chunk order
    float M = -INFINITY, L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = lane; c < n; c += 64)
        M = fmaxf(M, ml[2 * c]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        M = fmaxf(M, __shfl_xor(M, o));
    for (int c0 = 0; c0 < n; c0 += 64) {
        float w = 0.f;
        if (c0 + lane < n) {
            const float m = ml[2 * (c0 + lane)];
            w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
            L += ml[2 * (c0 + lane) + 1] * w;
        }
        const int some = min(64, n - c0);
#pragma unroll 4
        for (int c = 0; c < some; c++) {
            const float f = __shfl(w, c);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (lane + 64 * i < a.mx.head_dim)
                    x[i] += o[(int64_t)(c0 + c) * a.mx.head_dim + lane + 64 * i] * f;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        L += __shfl_xor(L, o);
    const float norm = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < a.mx.head_dim)
            a.out[line * a.mx.head_dim + lane + 64 * i] = x[i] * norm;
}

} // namespace nvk

namespace {

using nvk::Mx4AttnArgs;

constexpr int kDecodeWaves = 4, kPrefillWaves = 4;
constexpr int prefill_cols(int kk) { return kk == 8 ? 1 : 2; } // columns of a prefill wave: 16 times this (registers)

struct Mx4Shape
{
    bool   prefill = false;
    int    col_blocks = 1, chunk_tokens = 32, chunks = 1;
    size_t ws_floats = 0;
};

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// How a call is cut into workgroups: columns first, then chunks of the context until the chip is full.
Mx4Shape mx4_shape(const nvk_mx4_pool *pool, int num_seqs, int n_heads, int total_rows, int max_rows, int max_ctx)
{
    Mx4Shape  s;
    const int group = n_heads / pool->n_kv_heads;
    // Waves that share the tokens while one wave holds a sequence's columns; else waves that share the columns.
    s.prefill    = (long long)max_rows * group > 16;
    const int cols = s.prefill ? 16 * prefill_cols(pool->kk) * kPrefillWaves : 16;
    s.col_blocks = ceil_div((long long)max_rows * group, cols);
    const long long tasks = (long long)num_seqs * pool->n_kv_heads * s.col_blocks;
    // workgroups wanted: four to a CU; a chunk is worth its start and its join from 256 tokens on
    const int wanted = ceil_div(MX4_WGS * pool->num_cus, std::max(tasks, 1LL));
    const int most = std::max(1, max_ctx / 256);
    s.chunks       = std::max(1, std::min(wanted, most));
    s.chunk_tokens = std::max(32, ceil_div(ceil_div(max_ctx, s.chunks), 32) * 32);
    s.chunks       = std::max(1, ceil_div(max_ctx, s.chunk_tokens));
    s.ws_floats    = s.chunks > 1 ? (size_t)total_rows * n_heads * s.chunks * (pool->head_dim + 2) : 0;
    return s;
}

template <int KK> void launch_attn(const Mx4AttnArgs &a, const Mx4Shape &s, unsigned blocks, hipStream_t st)
{
    if (s.prefill)
        hipLaunchKernelGGL((nvk::nvk_mx4_attn_kernel<KK, prefill_cols(KK), 1, kPrefillWaves>), dim3(blocks),
                           dim3(64 * kPrefillWaves), 0, st, a);
    else
        hipLaunchKernelGGL((nvk::nvk_mx4_attn_kernel<KK, 1, kDecodeWaves, 1>), dim3(blocks), dim3(64 * kDecodeWaves), 0, st, a);
}

int check_attention(const nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, int total_rows, int max_rows, int max_blocks,
                    int max_ctx, const char *who)
{
    if (!pool)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pool", who);
    if (layer < 0 || layer >= pool->n_layers)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: layer %d outside [0,%d)", who, layer, pool->n_layers);
    if (num_seqs < 0 || total_rows < 0 || max_rows < 0 || max_blocks <= 0 || max_ctx < 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: negative size", who);
    if (n_heads <= 0 || n_heads % pool->n_kv_heads != 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: n_heads %d is no multiple of n_kv_heads %d", who, n_heads, pool->n_kv_heads);
    if ((long long)max_blocks * pool->block_size > 0x7fffffffLL || (long long)max_rows * n_heads > 0x3fffffffLL
        || max_ctx > 0x7fffff00)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: more than 2^31 tokens in a table, or 2^30 columns in a sequence", who);
    return NVK_OK;
}

int enqueue_attention(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, int total_rows, const float *q,
                      const int *row_offsets, int max_rows, const int *tables, int max_blocks, const int *ctx_lens, int max_ctx,
                      float *out, hipStream_t st, const char *who)
{
    const Mx4Shape  s = mx4_shape(pool, num_seqs, n_heads, total_rows, max_rows, max_ctx);
    const long long blocks = (long long)num_seqs * pool->n_kv_heads * s.col_blocks * s.chunks;
    if (blocks > 0x7fffffffLL)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: %lld workgroups", who, blocks);
    int rc = nvk::grow_workspace(&pool->ws, &pool->ws_floats, &pool->ws_generation, s.ws_floats, st, who);
    if (rc != NVK_OK)
        return rc;
    Mx4AttnArgs a{};
    a.mx = pool->layer(layer), a.q = q, a.out = out, a.row_offsets = row_offsets, a.tables = tables, a.ctx_lens = ctx_lens;
    a.num_seqs = num_seqs, a.max_blocks = max_blocks, a.n_heads = n_heads, a.group = n_heads / pool->n_kv_heads;
    a.total_rows = total_rows, a.col_blocks = s.col_blocks, a.chunk_tokens = s.chunk_tokens, a.chunks = s.chunks;
    a.scale_log2e = (float)(1.4426950408889634 / std::sqrt((double)pool->head_dim));
    if (s.chunks > 1) {
        a.ws_o  = pool->ws;
        a.ws_ml = pool->ws + (size_t)total_rows * n_heads * s.chunks * pool->head_dim;
    }
    switch (pool->kk) {
    case 1: launch_attn<1>(a, s, (unsigned)blocks, st); break;
    case 2: launch_attn<2>(a, s, (unsigned)blocks, st); break;
    case 4: launch_attn<4>(a, s, (unsigned)blocks, st); break;
    default: launch_attn<8>(a, s, (unsigned)blocks, st); break;
    }
    NVK_HIP_TRY(hipGetLastError());
    if (s.chunks > 1) {
        hipLaunchKernelGGL(nvk::nvk_mx4_merge_kernel, dim3((unsigned)(((long long)total_rows * n_heads + 3) / 4)), dim3(256), 0, st, a);
        NVK_HIP_TRY(hipGetLastError());
    }
    return NVK_OK;
}

// the host-pointer forms of both
int attention_host(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, const float *q, const int *chunk_lens,
                   const int *tables, int max_blocks, const int *ctx_lens, float *out, const char *who)
{
    int rc = check_attention(pool, layer, num_seqs, n_heads, 0, 0, max_blocks, 0, who);
    if (rc != NVK_OK)
        return rc;
    if (num_seqs == 0)
        return NVK_OK;
    if (!q || !tables || !ctx_lens || !out)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pointer", who);
    rc = nvk::check_tables(tables, num_seqs, max_blocks, ctx_lens, pool->block_size, pool->num_blocks, who);
    if (rc != NVK_OK)
        return rc;
    long long total = 0;
    int       max_rows = 1, max_ctx = 0;
    int      *offsets = new (std::nothrow) int[(size_t)num_seqs + 1];
    if (!offsets)
        return nvk::fail(NVK_ERR_OOM, "%s: host allocation failed", who);
    for (int s = 0; s < num_seqs && rc == NVK_OK; s++) {
        const int n = chunk_lens ? chunk_lens[s] : 1;
        offsets[s]  = (int)total;
        if (n < 0 || (chunk_lens && n > ctx_lens[s]))
            rc = nvk::fail(NVK_ERR_INVALID_ARG, "%s: %d rows of sequence %d, whose context is %d tokens", who, n, s, ctx_lens[s]);
        total += n;
        if (total * n_heads > 0x7fffffffLL)
            rc = nvk::fail(NVK_ERR_INVALID_ARG, "%s: too many rows", who);
        max_rows = std::max(max_rows, n), max_ctx = std::max(max_ctx, ctx_lens[s]);
    }
    offsets[num_seqs] = (int)total;
    if (rc != NVK_OK || total == 0) {
        delete[] offsets;
        return rc;
    }
    rc = [&]() -> int {
        NVK_SCOPE(pool->device);
        const size_t qb = (size_t)total * n_heads * pool->head_dim * sizeof(float);
        nvk::Staging st;
        const int    iq = st.add(q, qb), io = st.add(nullptr, qb), it = st.add(tables, (size_t)num_seqs * max_blocks * sizeof(int)),
                  ic = st.add(ctx_lens, (size_t)num_seqs * sizeof(int)), ir = st.add(offsets, ((size_t)num_seqs + 1) * sizeof(int));
        NVK_HIP_TRY(st.upload(pool->stream));
        const int e = enqueue_attention(pool, layer, num_seqs, n_heads, (int)total, st.at<float>(iq),
                                        chunk_lens ? st.at<int>(ir) : nullptr, max_rows, st.at<int>(it), max_blocks, st.at<int>(ic),
                                        max_ctx, st.at<float>(io), pool->stream, who);
        if (e == NVK_OK)
            NVK_HIP_TRY(hipMemcpyAsync(out, st.at<float>(io), qb, hipMemcpyDeviceToHost, pool->stream));
        NVK_HIP_TRY(hipStreamSynchronize(pool->stream));
        return e;
    }();
    delete[] offsets;
    return rc;
}

} // namespace

extern "C" {

int nvk_mx4_pool_create(int n_layers, int num_blocks, int block_size, int n_kv_heads, int head_dim, int device,
                        nvk_mx4_pool **out_pool)
{
    if (!out_pool)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_create: out_pool is null");
    *out_pool = nullptr;
    if (n_layers <= 0 || num_blocks <= 0 || n_kv_heads <= 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_create: non-positive size");
    if (block_size <= 0 || block_size % nvk::kMx4Tile != 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_create: block_size %d is no multiple of %d", block_size, nvk::kMx4Tile);
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 256)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_create: head_dim %d (a multiple of 8, at most 256)", head_dim);
    if ((long long)num_blocks * (block_size / nvk::kMx4Tile) > 0x7fffffffLL || (long long)n_kv_heads * head_dim > 0x7fffffffLL)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_create: more than 2^31 tiles in a layer");
    if (device < 0 || device >= nvk::device_count_cached())
        return nvk::fail(nvk::device_count_cached() ? NVK_ERR_INVALID_ARG : NVK_ERR_NO_DEVICE,
                         "nvk_mx4_pool_create: device %d outside [0,%d)", device, nvk::device_count_cached());
    const int    kk = nvk::mx4_kk(head_dim);
    const double bytes = (double)n_layers * num_blocks * (block_size / nvk::kMx4Tile) * n_kv_heads * nvk::mx4_tile_bytes(kk);
    if (bytes > 1e15)
        return nvk::fail(NVK_ERR_OOM, "nvk_mx4_pool_create: %.3g bytes requested", bytes);
    nvk_mx4_pool *pool = new (std::nothrow) nvk_mx4_pool();
    if (!pool)
        return nvk::fail(NVK_ERR_OOM, "nvk_mx4_pool_create: host allocation failed");
    pool->n_layers = n_layers, pool->num_blocks = num_blocks, pool->block_size = block_size, pool->n_kv_heads = n_kv_heads;
    pool->head_dim = head_dim, pool->device = device, pool->kk = kk;
    pool->layer_bytes = (size_t)num_blocks * (block_size / nvk::kMx4Tile) * n_kv_heads * nvk::mx4_tile_bytes(kk);
    nvk::DeviceScope scope(device);
    hipDeviceProp_t  prop;
    if (hipGetDeviceProperties(&prop, device) == hipSuccess && prop.multiProcessorCount > 0)
        pool->num_cus = prop.multiProcessorCount;
    hipError_t e = scope.ok ? hipSuccess : hipErrorInvalidDevice;
    if (e == hipSuccess)
        e = hipMalloc((void **)&pool->base, pool->layer_bytes * (size_t)n_layers);
    if (e == hipSuccess)
        e = hipStreamCreateWithFlags(&pool->stream, hipStreamNonBlocking);
    // zeros are values of 0 (and keep channels of padding at 0)
    if (e == hipSuccess)
        e = hipMemsetAsync(pool->base, 0, pool->layer_bytes * (size_t)n_layers, pool->stream);
    if (e == hipSuccess)
        e = hipStreamSynchronize(pool->stream);
    if (e != hipSuccess) {
        const int rc = nvk::fail(e == hipErrorOutOfMemory ? NVK_ERR_OOM : NVK_ERR_HIP, "nvk_mx4_pool_create: %s (%zu bytes requested)",
                                 hipGetErrorString(e), pool->layer_bytes * (size_t)n_layers);
        (void)hipGetLastError();
        nvk_mx4_pool_destroy(pool);
        return rc;
    }
    *out_pool = pool;
    return NVK_OK;
}

int nvk_mx4_pool_destroy(nvk_mx4_pool *pool)
{
    if (!pool)
        return NVK_OK;
    nvk::DeviceScope scope(pool->device); // (a release path: goes on whatever the switch returned)
    (void)hipDeviceSynchronize();         // launches on any stream may still use it
    if (pool->base)
        (void)hipFree(pool->base);
    if (pool->ws)
        (void)hipFree(pool->ws);
    if (pool->stream)
        (void)hipStreamDestroy(pool->stream);
    delete pool;
    return NVK_OK;
}

int nvk_mx4_pool_geometry(const nvk_mx4_pool *pool, int *out6)
{
    if (!pool || !out6)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_geometry: null argument");
    const int g[6] = {pool->n_layers, pool->num_blocks, pool->block_size, pool->n_kv_heads, pool->head_dim, pool->device};
    std::copy(g, g + 6, out6);
    return NVK_OK;
}

long long nvk_mx4_pool_layer_bytes(const nvk_mx4_pool *pool) { return pool ? (long long)pool->layer_bytes : -1; }

int nvk_mx4_pool_layer_ptr(const nvk_mx4_pool *pool, int layer, void **base_dev)
{
    if (!pool || !base_dev || layer < 0 || layer >= pool->n_layers)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_layer_ptr: bad arguments");
    *base_dev = pool->base + (size_t)layer * pool->layer_bytes;
    return NVK_OK;
}

int nvk_mx4_pool_stream(const nvk_mx4_pool *pool, void **stream)
{
    if (!pool || !stream)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_stream: null argument");
    *stream = (void *)pool->stream;
    return NVK_OK;
}

int nvk_mx4_pool_synchronize(nvk_mx4_pool *pool)
{
    if (!pool)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_pool_synchronize: null pool");
    NVK_SCOPE(pool->device);
    NVK_HIP_TRY(hipStreamSynchronize(pool->stream));
    return NVK_OK;
}

long long nvk_mx4_pool_workspace_generation(const nvk_mx4_pool *pool) { return pool ? pool->ws_generation : -1; }

int nvk_mx4_pool_reserve_workspace(nvk_mx4_pool *pool, int num_seqs, int n_heads, int total_rows, int max_rows, int max_ctx)
{
    const char *who = "nvk_mx4_pool_reserve_workspace";
    const int   rc = check_attention(pool, 0, num_seqs, n_heads, total_rows, max_rows, 1, max_ctx, who);
    if (rc != NVK_OK)
        return rc;
    NVK_SCOPE(pool->device);
    const Mx4Shape s = mx4_shape(pool, num_seqs, n_heads, total_rows, std::max(max_rows, 1), max_ctx);
    return nvk::grow_workspace(&pool->ws, &pool->ws_floats, &pool->ws_generation, s.ws_floats, pool->stream, who);
}

int nvk_mx4_decode_device(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, const float *q_dev,
                          const int *block_tables_dev, int max_blocks, const int *ctx_lens_dev, int max_ctx, float *out_dev,
                          void *stream)
{
    const char *who = "nvk_mx4_decode_device";
    const int   rc = check_attention(pool, layer, num_seqs, n_heads, num_seqs, 1, max_blocks, max_ctx, who);
    if (rc != NVK_OK)
        return rc;
    if (num_seqs == 0)
        return NVK_OK;
    if (!q_dev || !block_tables_dev || !ctx_lens_dev || !out_dev)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pointer", who);
    NVK_SCOPE(pool->device);
    return enqueue_attention(pool, layer, num_seqs, n_heads, num_seqs, q_dev, nullptr, 1, block_tables_dev, max_blocks, ctx_lens_dev,
                             max_ctx, out_dev, stream ? (hipStream_t)stream : pool->stream, who);
}

int nvk_mx4_prefill_device(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, int total_rows, const float *q_dev,
                           const int *row_offsets_dev, int max_rows, const int *block_tables_dev, int max_blocks,
                           const int *ctx_lens_dev, int max_ctx, float *out_dev, void *stream)
{
    const char *who = "nvk_mx4_prefill_device";
    const int   rc = check_attention(pool, layer, num_seqs, n_heads, total_rows, max_rows, max_blocks, max_ctx, who);
    if (rc != NVK_OK)
        return rc;
    if (num_seqs == 0 || total_rows == 0 || max_rows == 0)
        return NVK_OK;
    if (!q_dev || !row_offsets_dev || !block_tables_dev || !ctx_lens_dev || !out_dev)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pointer", who);
    NVK_SCOPE(pool->device);
    return enqueue_attention(pool, layer, num_seqs, n_heads, total_rows, q_dev, row_offsets_dev, max_rows, block_tables_dev,
                             max_blocks, ctx_lens_dev, max_ctx, out_dev, stream ? (hipStream_t)stream : pool->stream, who);
}

int nvk_mx4_decode(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, const float *q, const int *block_tables,
                   int max_blocks, const int *ctx_lens, float *out)
{
    return attention_host(pool, layer, num_seqs, n_heads, q, nullptr, block_tables, max_blocks, ctx_lens, out, "nvk_mx4_decode");
}

int nvk_mx4_prefill(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, const float *q, const int *block_tables,
                    int max_blocks, const int *chunk_lens, const int *ctx_lens, float *out)
{
    if (num_seqs > 0 && !chunk_lens)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_mx4_prefill: null pointer");
    return attention_host(pool, layer, num_seqs, n_heads, q, chunk_lens, block_tables, max_blocks, ctx_lens, out, "nvk_mx4_prefill");
}

} // extern "C"
