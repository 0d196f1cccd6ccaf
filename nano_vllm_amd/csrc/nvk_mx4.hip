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

#include "nvk_addr.hip.h"
#include "nvk_chunk_join.hip.h"
#include "nvk_hip_util.h"
#include "nvk_mx4.hip.h"

namespace nvk {

constexpr int kDecodeWaves = 4, kPrefillWaves = 4;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float  f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct Mx4AttnArgs
{
    Mx4Layer     mx;
    const float *q;   // [rows, n_heads, head_dim]
    float       *out; // the same
    const int   *row_offsets; // [num_seqs + 1] or null: row s belongs to sequence s
    const int   *tables, *ctx_lens;
    int          num_seqs, max_blocks, n_heads, group, total_rows;
    int          col_blocks;   // prefill: workgroups along a sequence's (row, head) columns
    int          chunk_tokens; // tokens a workgroup takes (a multiple of 32)
    int          chunks;       // chunks along the longest context
    float        scale_log2e;  // log2(e) / sqrt(head_dim)
    float       *ws_o, *ws_ml; // partial results where chunks > 1: [rows * heads][chunks][head_dim], [..][2]
    int          whole_lines;  // the decode kernel ran
    int         *arrivals;     // decode: one for each (sequence, kv-head), or null: the join kernel follows
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
// The conversion looks at the exponent field of its scale alone (any sign and mantissa do), and makes NaN of exponent 255: a
// scale byte needs a shift and no mask.
__device__ __forceinline__ float scale_at(unsigned bytes, int b)
{
    return __uint_as_float(b < 3 ? bytes << (23 - 8 * b) : bytes >> 1);
}
// Non-zero where a byte of x is 255.
__device__ __forceinline__ unsigned byte_255(unsigned x) { return (0xfefefefeu - x) & x & 0x80808080u; }

// Over the four lanes of a quad.
__device__ __forceinline__ float sum_of_quad(float x)
{
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, true)); // lanes 1 0 3 2
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, true)); // lanes 2 3 0 1
    return x;
}
// The largest of x over the four lanes (g, l16), g = 0 .. 3; their sum.
__device__ __forceinline__ float max_of_g(float x)
{
    const unsigned u = __float_as_uint(x);
    const auto     a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto     b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// What a lane holds of one tile.
template <int KK> struct Mx4Raw
{
    static constexpr int KS = KK == 8 ? 2 : 1; // groups that a lane's channels of K lie in
    unsigned k[KK], v[KK], vs;
    unsigned ks[KS];
};

// Byte offsets of a lane's parts inside a tile: K, channels g*8*KK .. of token l16; V, channels l16*2*KK .. of tokens
// 4g .. 4g+3; the scales of both.
template <int KK> struct Mx4Places
{
    unsigned k, v, ks[Mx4Raw<KK>::KS], vs;
    __device__ __forceinline__ explicit Mx4Places(int lane)
    {
        const int g = lane >> 4, l16 = lane & 15;
        k = l16 * 16 * KK + g * 4 * KK;
        v = mx4_v_at(KK) + lane * 4 * KK;
#pragma unroll
        for (int u = 0; u < Mx4Raw<KK>::KS; u++)
            ks[u] = mx4_ks_at(KK) + (g * KK / 4 + u) * kMx4Tile + l16;
        vs = mx4_vs_at(KK) + (l16 * KK / 16) * kMx4Tile + 4 * g;
    }
};

// All of it.  (Each code is read by one wave of the launch: not worth keeping in the caches.)
template <int KK> __device__ __forceinline__ void load_tile(Mx4Raw<KK> &r, const unsigned char *tile, const Mx4Places<KK> &at)
{
    const unsigned *kc = reinterpret_cast<const unsigned *>(tile + at.k);
    const unsigned *vc = reinterpret_cast<const unsigned *>(tile + at.v);
    if constexpr (KK >= 4) {
#pragma unroll
        for (int i = 0; i < KK; i += 4) {
            const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kc + i));
            const u32x4 y = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vc + i));
#pragma unroll
            for (int u = 0; u < 4; u++)
                r.k[i + u] = x[u], r.v[i + u] = y[u];
        }
    }
    else
#pragma unroll
        for (int i = 0; i < KK; i++)
            r.k[i] = kc[i], r.v[i] = vc[i];
#pragma unroll
    for (int u = 0; u < Mx4Raw<KK>::KS; u++)
        r.ks[u] = tile[at.ks[u]];
    r.vs = *reinterpret_cast<const unsigned *>(tile + at.vs);
}
// K where asked for, V where asked for, the V scales always.  (Read by many workgroups.)
template <int KK>
__device__ __forceinline__ void load_tile_part(Mx4Raw<KK> &r, const unsigned char *tile, const Mx4Places<KK> &at, bool k, bool v)
{
    auto codes = [](unsigned (&to)[KK], const unsigned char *from) {
        if constexpr (KK >= 4) {
#pragma unroll
            for (int i = 0; i < KK; i += 4) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(from + 4 * i);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    to[i + u] = x[u];
            }
        }
        else
#pragma unroll
            for (int i = 0; i < KK; i++)
                to[i] = reinterpret_cast<const unsigned *>(from)[i];
    };
    if (k) {
        codes(r.k, tile + at.k);
#pragma unroll
        for (int u = 0; u < Mx4Raw<KK>::KS; u++)
            r.ks[u] = tile[at.ks[u]];
    }
    if (v)
        codes(r.v, tile + at.v);
    r.vs = *reinterpret_cast<const unsigned *>(tile + at.vs);
}

// ---- what both kernels are made of ------------------------------------------------------------------------------------
// A wave holds a tile of 16 columns, a column being a (row, head of the group) pair of one kv-head, and takes 32 tokens a step:
//   S^T = K Q^T     A = K [16 tokens x 32 channels], B = Q^T [32 channels x 16 columns] -> lane (g, col): tokens 4g .. 4g+3
//   O^T = V^T P^T   A = V^T [16 channels x 32 tokens], B = P^T [32 tokens x 16 columns]
// The order of channels (in S) and of tokens (in O) along a contraction is free, so it is chosen such that the lane that holds
// a probability after S is the lane that needs it for O: the softmax touches no LDS, and a column's maximum takes two lane
// exchanges a step.
// PACK: up to four columns, each four times in a tile: the first three copies carry one piece of q and of the probabilities
// each, whose products then take a third of the instructions and registers, and the copies of a column are added (a quad of
// lanes).
template <int KK, bool PACK> struct Mx4Wave
{
    static constexpr int COLS   = PACK ? 4 : 16; // columns of a tile
    static constexpr int PIECES = PACK ? 1 : 3;

    int      lane, g, l16, lcol, piece; // lcol: the lane's column of a tile; PACK: `piece` is which copy of it
    int      limit, out_row, out_head; // the lane's column: its row sees the tokens below `limit`, all up to its own
    int      most, least;              // the largest and the smallest limit of the wave's columns
    bf16x8   q[KK][PIECES];
    f32x4    acc[2 * KK]; // [ct][i]: channel (4 g + i) * 2 KK + ct
    // m: what scores are taken relative to, a score that was the largest once (0 while lim is -inf: no token yet).  It is moved
    // only where a score passes it by more than 8: probabilities up to 2^8 are as exact as those up to 1.
    float    m, lim, l;
    unsigned poisoned;   // channel groups in which a token that the column sees holds no number
    unsigned cut1, cut2; // PACK: what a probability loses to become the lane's piece (the fourth copy's result is dropped)

    __device__ __forceinline__ void start(const Mx4AttnArgs &a, int row0, int rows, int ctx, int kvh, int col0)
    {
        lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
        lcol = PACK ? l16 >> 2 : l16, piece = l16 & 3;
        cut1 = piece > 0 ? 0xffff0000u : 0u, cut2 = piece > 1 ? 0xffff0000u : 0u;
        const int columns = rows * a.group;
        const int last = min(col0 + COLS - 1, columns - 1) / a.group;
        most  = col0 < columns ? max(ctx - rows + last + 1, 0) : 0;
        least = col0 < columns ? max(ctx - rows + col0 / a.group + 1, 0) : 0;
        const int col = col0 + lcol, r = col / a.group;
        out_row  = col < columns ? row0 + r : -1;
        out_head = kvh * a.group + col % a.group;
        limit    = col < columns ? max(ctx - rows + r + 1, 0) : 0;
        // Q^T: channels g*8*KK + kk*8 .. of the column, in units in which a probability is a power of two
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            float     x[8];
            const int c0 = g * 8 * KK + kk * 8;
#pragma unroll
            for (int i = 0; i < 8; i++)
                x[i] = 0.f;
            if (out_row >= 0 && c0 < a.mx.head_dim) {
                const float *src = a.q + ((int64_t)out_row * a.n_heads + out_head) * a.mx.head_dim + c0;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    x[i] = src[i] * a.scale_log2e;
            }
            const Pieces three = split8(x);
            if constexpr (PACK) {
                const u32x4 none = {0, 0, 0, 0};
                const u32x4 one  = piece == 0   ? __builtin_bit_cast(u32x4, three.p[0])
                                   : piece == 1 ? __builtin_bit_cast(u32x4, three.p[1])
                                   : piece == 2 ? __builtin_bit_cast(u32x4, three.p[2]) : none;
                q[kk][0] = __builtin_bit_cast(bf16x8, one);
            }
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    q[kk][e] = three.p[e];
        }
        m = 0.f, lim = -INFINITY, l = 0.f, poisoned = 0;
#pragma unroll
        for (int ct = 0; ct < 2 * KK; ct++)
            acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // A group of V that holds no number (scale byte 255): its scale is taken as 0, and the columns that see the token are marked.
    // (One of K makes its token's scores NaN by itself.)  `vs`: the lane's V scales of the two tiles from token t0 on.
    // Before any product of a step: an earlier form of these kernels had its branches behind the score products, with results in
    // accumulation registers, and a first read one slot behind across a branch; its scores differed from run to run.  Where
    // a branch stands there now (`softmax`) the compiler pads both ways; a walk over every path of the built kernels checks it.
    __device__ __forceinline__ void mark(unsigned (&vs)[2], int t0)
    {
        if (__any((byte_255(vs[0]) | byte_255(vs[1])) != 0)) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const bool         odd = ((vs[j] >> (8 * b)) & 255u) == 255u;
                    unsigned long long who = __ballot(odd);
                    if (odd)
                        vs[j] &= ~(255u << (8 * b));
                    for (; who; who &= who - 1) { // lane (quad, c16) tells: token 4 quad + b of tile j, group of c16
                        const int from = __ffsll((long long)who) - 1;
                        const int token = t0 + 16 * j + 4 * (from >> 4) + b;
                        if (token < limit)
                            poisoned |= 1u << ((from & 15) * KK / 16);
                    }
                }
        }
    }

    // Where scores start: relative to m.
    __device__ __forceinline__ f32x4 origin() const { return PACK && piece ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{-m, -m, -m, -m}; }

    // Scores (s[j][i]: token t0 + 16 j + 4 g + i) -> the pieces of its probabilities; maximum, sum and output follow.
    __device__ __forceinline__ void softmax(const f32x4 (&s)[2], int t0, bf16x8 (&p)[PIECES])
    {
        float t[8], top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            t[e] = s[e >> 2][e & 3];
            if constexpr (PACK)
                t[e] = sum_of_quad(t[e]);
        }
        if (t0 + 32 > least) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (t0 + 16 * (e >> 2) + 4 * g + (e & 3) >= limit)
                    t[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
            top = fmaxf(top, t[e]);
        top = max_of_g(top);
        if (__any(top > lim)) {
            const bool  over = top > lim;
            const float up = over ? top : 0.f;
            const float alpha = lim == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-up);
            m += up;
            lim = over ? 8.f : lim;
            l *= alpha;
#pragma unroll
            for (int ct = 0; ct < 2 * KK; ct++)
                acc[ct] *= alpha;
#pragma unroll
            for (int e = 0; e < 8; e++)
                t[e] -= up;
        }
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            t[e] = __builtin_amdgcn_exp2f(t[e]);
            sum += t[e];
        }
        l += sum;
        if constexpr (PACK) { // the lane's own piece: what as many truncations leave
            union
            {
                unsigned u[4];
                bf16x8   v;
            } w;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                t[e] -= __uint_as_float(__float_as_uint(t[e]) & cut1);
                t[e] -= __uint_as_float(__float_as_uint(t[e]) & cut2);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                w.u[e] = high_halves(t[2 * e], t[2 * e + 1]);
            p[0] = w.v;
        }
        else {
            const Pieces three = split8(t);
#pragma unroll
            for (int e = 0; e < 3; e++)
                p[e] = three.p[e];
        }
    }

    // After the last token: sums over the lanes that share a column; marked groups become NaN; m is -inf where no token was seen.
    __device__ __forceinline__ void finish()
    {
        if constexpr (PACK) // the three copies of a column
#pragma unroll
            for (int ct = 0; ct < 2 * KK; ct++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[ct][i] = sum_of_quad(piece == 3 ? 0.f : acc[ct][i]);
        if (lim == -INFINITY)
            m = -INFINITY;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (poisoned)
#pragma unroll
            for (int ct = 0; ct < 2 * KK; ct++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if ((poisoned >> (((4 * g + i) * 2 * KK + ct) / 32)) & 1u)
                        acc[ct][i] = __uint_as_float(0x7fc00000u);
    }
};

// K of a tile: 8 channels from one dword of codes.
__device__ __forceinline__ bf16x8 k_operand(unsigned codes, float scale)
{
    union
    {
        unsigned u[4];
        bf16x8   v;
    } w;
#pragma unroll
    for (int b = 0; b < 4; b++)
        w.u[b] = two_values_at(codes, scale, b);
    return w.v;
}
// V of two tiles: channels 2b and 2b + 1 of the lane's run, for its eight tokens.
template <int KK>
__device__ __forceinline__ void v_operands(const unsigned (&v0)[KK], const unsigned (&v1)[KK], const unsigned (&vs)[2], int b, bf16x8 &even,
                                           bf16x8 &odd)
{
    unsigned w[2][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        w[0][t] = two_values_at(v0[(t * KK + b) / 4], scale_at(vs[0], t), (t * KK + b) % 4);
        w[1][t] = two_values_at(v1[(t * KK + b) / 4], scale_at(vs[1], t), (t * KK + b) % 4);
    }
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
    even = lo.v, odd = hi.v;
}

// Where a workgroup's piece of context lies: tile `t` of the context -> its address.  A lane keeps one entry of the block
// table; 64 tiles at a time.
struct Mx4Tiles
{
    const unsigned char *base; // the layer, at the kv-head
    const int           *table;
    int64_t              stride; // bytes from one tile of the layer to the next
    int                  per_block, last, num_blocks; // last: the last tile that may be asked for

    __device__ __forceinline__ Mx4Tiles(const Mx4AttnArgs &a, int seq, int kvh, int last_tile)
    {
        base       = a.mx.base + (int64_t)kvh * mx4_tile_bytes(a.mx.kk);
        table      = a.tables + (int64_t)seq * a.max_blocks;
        stride     = (int64_t)a.mx.n_kv_heads * mx4_tile_bytes(a.mx.kk);
        per_block  = a.mx.block_size / kMx4Tile;
        last       = max(last_tile, 0);
        num_blocks = a.mx.num_blocks;
    }
    // the tile's number in the layer (out of bounds entries are clamped)
    __device__ __forceinline__ int entry(int t) const
    {
        t           = min(t, last);
        const int b = t / per_block;
        return min(max(table[b], 0), num_blocks - 1) * per_block + t % per_block;
    }
    __device__ __forceinline__ const unsigned char *at(int number) const { return base + number * stride; }
};

__device__ __forceinline__ int mx4_context(const Mx4AttnArgs &a, int seq)
{
    return min(max(a.ctx_lens[seq], 0), (int)min((int64_t)a.max_blocks * a.mx.block_size, (int64_t)0x7fffffff));
}
// rows of a sequence: [row0, row0 + rows)
__device__ __forceinline__ int mx4_rows(const Mx4AttnArgs &a, int seq, int &row0)
{
    row0 = seq;
    if (!a.row_offsets)
        return 1;
    row0 = a.row_offsets[seq];
    return row0 < 0 ? 0 : min(a.row_offsets[seq + 1], a.total_rows) - row0;
}

// ---- few columns: the waves of a workgroup share the tokens --------------------------------------------------------------
// Bound by the codes it reads while everything beside the loads hides behind them; what does not is the vector work of a
// step.  The waves take steps of 32 tokens in turn and join through LDS.  Of 128 channels, groups of four heads, eight kv-heads: 64 x
// 2048 tokens 28.5 us (144 MB, 5.1 TB/s), 16 x 32768 98.5 us (574 MB, 5.8 TB/s; its loads alone, with nothing done to them, 91).  PACK
// takes 16 products a step instead of 48 and 158 registers instead of 198, so that three workgroups fit a CU and not two: 16 x 32768
// 115 us without, 105 with it, 102 in one round of three a CU.  Tried and no faster: two or three steps on their way (30.8 and 31.2
// for the 28.4 of 64 x 2048), workgroups of three, six or twelve waves (45, 37 and 36 us).
template <int KK, bool PACK>
__global__ void __launch_bounds__(64 * kDecodeWaves, KK == 8 ? 1 : PACK ? 3 : 2) nvk_mx4_decode_kernel(const Mx4AttnArgs a)
{
    using Wave = Mx4Wave<KK, PACK>;
    constexpr int HDP = 32 * KK, COLS = Wave::COLS, W = kDecodeWaves;
    const int     wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroup -> (sequence, chunk, kv-head); a sequence's columns are one tile.  Consecutive workgroups go to the eight XCDs in
    // turn.  Where the pieces of context come out even over the XCDs, the kv-heads of one are put side by side on one XCD, which
    // then reads whole blocks of the cache (64 x 2048: 3 % less time); elsewhere that would leave an XCD with more
    // workgroups than there is room for (42 pieces of 6 kv-heads with 256 channels: 29.9 us, 18.6 in plain order).
    const unsigned n_kv = (unsigned)a.mx.n_kv_heads, pieces = (unsigned)a.num_seqs * (unsigned)a.chunks, rest = blockIdx.x / 8u;
    const bool     even = pieces % 8u == 0;
    const int      kvh = (int)((even ? rest : blockIdx.x) % n_kv);
    const unsigned unit = even ? rest / n_kv * 8u + blockIdx.x % 8u : blockIdx.x / n_kv;
    const int      chunk = (int)(unit % (unsigned)a.chunks), seq = (int)(unit / (unsigned)a.chunks);
    int       row0;
    const int rows = mx4_rows(a, seq, row0), columns = rows * a.group;
    if (rows <= 0)
        return;
    const int ctx = mx4_context(a, seq);
    const int begin = chunk * a.chunk_tokens;
    Wave      w;
    w.start(a, row0, rows, ctx, kvh, 0);
    // the chunks that some column sees; the first one writes rows that see nothing
    const int parts = max(min((w.most + a.chunk_tokens - 1) / a.chunk_tokens, a.chunks), 1);
    if (chunk >= parts)
        return;
    const int end = min(begin + a.chunk_tokens, w.most);

    // step i of this wave covers the 32 tokens from begin + 32 * (wave + W * i)
    const int             steps = max(0, (end - begin + 31) / 32 - wave + W - 1) / W;
    const Mx4Tiles        tiles(a, seq, kvh, (min(end, ctx) - 1) / kMx4Tile);
    const Mx4Places<KK>   places(w.lane);
    int                   entry = 0; // lane L: tile L % 2 of the wave's step (i & ~31) + L / 2
    auto                  fetch = [&](Mx4Raw<KK> (&r)[2], int i) {
        if ((i & 31) == 0)
            entry = tiles.entry((begin >> 4) + 2 * (wave + W * (i + (w.lane >> 1))) + (w.lane & 1));
#pragma unroll
        for (int j = 0; j < 2; j++)
            load_tile<KK>(r[j], tiles.at(__builtin_amdgcn_readlane(entry, 2 * (i & 31) + j)), places);
    };
    // one step on `raw`, while the next one's tiles are on their way into `next`
    auto step = [&](int i, const Mx4Raw<KK> (&raw)[2], Mx4Raw<KK> (&next)[2]) {
        if (i + 1 < steps)
            fetch(next, i + 1);
        const int t0 = begin + 32 * (wave + W * i);
        unsigned  vs[2] = {raw[0].vs, raw[1].vs};
        w.mark(vs, t0);
        bf16x8 k[2][KK];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
                k[j][kk] = k_operand(raw[j].k[kk], scale_at(raw[j].ks[KK == 8 ? kk / 4 : 0], 0));
        // the large pieces of q first: the sums of the small ones then round at the size of what is left
        f32x4 s[2] = {w.origin(), w.origin()};
#pragma unroll
        for (int e = 0; e < Wave::PIECES; e++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[j][kk], w.q[kk][e], s[j], 0, 0, 0);
        bf16x8 p[Wave::PIECES];
        w.softmax(s, t0, p);
#pragma unroll
        for (int b = 0; b < KK; b++) {
            bf16x8 even, odd;
            v_operands<KK>(raw[0].v, raw[1].v, vs, b, even, odd);
#pragma unroll
            for (int e = Wave::PIECES - 1; e >= 0; e--) {
                w.acc[2 * b]     = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, p[e], w.acc[2 * b], 0, 0, 0);
                w.acc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, p[e], w.acc[2 * b + 1], 0, 0, 0);
            }
        }
    };
    Mx4Raw<KK> one[2], two[2]; // in turn: no copies between the steps
    if (steps > 0)
        fetch(one, 0);
    for (int i = 0; i < steps; i += 2) {
        step(i, one, two);
        if (i + 1 < steps)
            step(i + 1, two, one);
    }
    w.finish();

    // join the waves: common maximum, then a sum over LDS
    __shared__ float s_m[W][COLS], s_l[W][COLS];
    __shared__ __attribute__((aligned(16))) float s_o[W][COLS][HDP + 4];
    const bool writes = !PACK || w.piece == 0;
    if (w.g == 0 && writes)
        s_m[wave][w.lcol] = w.m, s_l[wave][w.lcol] = w.l;
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < W; x++)
        M = fmaxf(M, s_m[x][w.lcol]);
    const float alpha = w.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - M);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int ct = 0; ct < 2 * KK; ct++)
            if (writes)
                s_o[wave][w.lcol][(4 * w.g + i) * 2 * KK + ct] = w.acc[ct][i] * alpha;
    __syncthreads();
    // (zeros for a row that sees no token; one whose scores are all -infinity is 0 / 0, no number)
    auto sees_none = [&](int col) { return ctx - rows + col / a.group + 1 <= 0; };
    for (int e = threadIdx.x; e < COLS * (HDP / 4); e += 64 * W) {
        const int col = e / (HDP / 4), c = (e % (HDP / 4)) * 4;
        if (col >= columns || c >= a.mx.head_dim)
            continue;
        float Mc = -INFINITY, L = 0.f;
#pragma unroll
        for (int x = 0; x < W; x++)
            Mc = fmaxf(Mc, s_m[x][col]);
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < W; x++) {
            L += s_m[x][col] == -INFINITY ? 0.f : s_l[x][col] * __builtin_amdgcn_exp2f(s_m[x][col] - Mc);
            o += *reinterpret_cast<const f32x4 *>(&s_o[x][col][c]);
        }
        const int64_t line = (int64_t)(row0 + col / a.group) * a.n_heads + kvh * a.group + col % a.group;
        if (parts > 1) {
            float *dst = a.ws_o + (line * a.chunks + chunk) * a.mx.head_dim + c, *ml = a.ws_ml + (line * a.chunks + chunk) * 2;
            store_through(dst, o[0], o[1]), store_through(dst + 2, o[2], o[3]);
            if (c == 0)
                store_through(ml, Mc, L);
        }
        else {
            o = sees_none(col) ? f32x4{0.f, 0.f, 0.f, 0.f} : o * (1.f / L);
            store_four(a.out + line * a.mx.head_dim + c, o[0], o[1], o[2], o[3]);
        }
    }
    if (parts == 1 || !a.arrivals || !arrived_last(a.arrivals + (int64_t)seq * a.mx.n_kv_heads + kvh, parts))
        return;
    for (int e = threadIdx.x; e < COLS * (HDP / 4); e += 64 * W) {
        const int col = e / (HDP / 4), c = (e % (HDP / 4)) * 4;
        if (col >= columns || c >= a.mx.head_dim)
            continue;
        const int64_t line = (int64_t)(row0 + col / a.group) * a.n_heads + kvh * a.group + col % a.group;
        // (a row of a short context was not seen by the later chunks of a longer one: they hold nothing for it)
        const float4 o = join_few<true>(a.ws_o + line * a.chunks * a.mx.head_dim + c, a.ws_ml + line * a.chunks * 2, parts, a.mx.head_dim,
                                        sees_none(col));
        store_four(a.out + line * a.mx.head_dim + c, o.x, o.y, o.z, o.w);
    }
}

// ---- many columns: the waves of a workgroup share the operands -------------------------------------------------------------
// Bound by the matrix instructions (48 for a tile of columns, a step and 128 channels) once the codes are turned into operands
// only once: the four waves of a workgroup convert a quarter of a step's K and V each into LDS, a step ahead, and read all
// of it as 16-byte operands.  One barrier a step: a buffer is written while the other is read.  Three chunks of up to 1500 rows
// behind up to 4000 tokens, 32 heads of 128 channels: 433 us for 497 GFLOP of products, 1150 TFLOP/s, where a large library
// product of bf16 reaches 1180 (each wave converting for itself: 684 us).  Two tiles of columns a wave halve the operands read but leave
// room for two workgroups a CU and not three: as fast there, and 34 us instead of 26 for a prompt of 512 tokens, 135 instead of 100 for 2048.
// With 64 channels and fewer neither pipe is full: a step is one chain (operands from LDS, score products, maximum, exponentials,
// pieces, output products) between barriers.  (1157 rows of 16 heads of 48 channels: waves wait 48 % of their time, the vector pipe is
// busy 34 % of the kernel's and the matrix pipe 16 %.)
template <int KK> __global__ void __launch_bounds__(64 * kPrefillWaves, KK == 8 ? 1 : 3) nvk_mx4_prefill_kernel(const Mx4AttnArgs a)
{
    using Wave = Mx4Wave<KK, false>;
    constexpr int COLS = Wave::COLS, W = kPrefillWaves;
    __shared__ __attribute__((aligned(16))) bf16x8 s_k[2][2 * KK][64], s_v[2][2 * KK][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroup -> (kv-head, column block, chunk, sequence): kv-heads in turn, so that with eight of them the column blocks
    // that read the same codes meet in the L2 of one XCD; the last column blocks, which see the most tokens, first.
    unsigned  id = blockIdx.x;
    const int kvh = (int)(id % (unsigned)a.mx.n_kv_heads);
    id /= (unsigned)a.mx.n_kv_heads;
    const int seq = (int)(id % (unsigned)a.num_seqs);
    id /= (unsigned)a.num_seqs;
    const int chunk = (int)(id % (unsigned)a.chunks);
    const int cb = a.col_blocks - 1 - (int)(id / (unsigned)a.chunks);
    int       row0;
    const int rows = mx4_rows(a, seq, row0), columns = rows * a.group;
    if (rows <= 0 || cb * W * COLS >= columns)
        return;
    const int ctx = mx4_context(a, seq);
    const int begin = chunk * a.chunk_tokens;
    const int last_row = min((cb + 1) * W * COLS - 1, columns - 1) / a.group;
    const int block_most = max(ctx - rows + last_row + 1, 0); // the largest limit of the workgroup's columns
    if (chunk > 0 && begin >= block_most)
        return;
    Wave w;
    w.start(a, row0, rows, ctx, kvh, (cb * W + wave) * COLS);
    const int end = min(begin + a.chunk_tokens, block_most);
    const int steps = max(0, (end - begin + 31) / 32);

    // This wave's share of a step: K operands kk of tile j for item = wave, wave + W, .. of (kk, j), V channel pairs b = wave, ..
    const Mx4Tiles      tiles(a, seq, kvh, (min(end, ctx) - 1) / kMx4Tile);
    const Mx4Places<KK> places(w.lane);
    const int           tile_j = wave & 1; // (W is even: all K items of a wave lie in one tile)
    constexpr int       AHEAD = KK == 2 ? 2 : 1; // steps whose codes are on their way (two: 64 channels 3 % less time, 32 and 128 a sixth more and beyond)
    Mx4Raw<KK>          ring[AHEAD][2];
    int                 entry = 0; // lane L: tile L of the current 32 steps
    auto                fetch = [&](int i, Mx4Raw<KK> (&raw)[2]) {
        if ((i & 31) == 0)
            entry = tiles.entry((begin >> 4) + 2 * i + w.lane);
#pragma unroll
        for (int j = 0; j < 2; j++)
            load_tile_part<KK>(raw[j], tiles.at(__builtin_amdgcn_readlane(entry, 2 * (i & 31) + j)), places, j == tile_j, wave < KK);
    };
    auto convert = [&](int i, const Mx4Raw<KK> (&raw)[2]) {
        unsigned vs[2] = {raw[0].vs, raw[1].vs};
        w.mark(vs, begin + 32 * i);
        const int   buf = i & 1;
        const auto &mine = tile_j ? raw[1] : raw[0];
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
            if ((kk * 2 + tile_j) % W == wave)
                s_k[buf][kk * 2 + tile_j][w.lane] = k_operand(mine.k[kk], scale_at(mine.ks[KK == 8 ? kk / 4 : 0], 0));
#pragma unroll
        for (int b = 0; b < KK; b++)
            if (b % W == wave) {
                bf16x8 even, odd;
                v_operands<KK>(raw[0].v, raw[1].v, vs, b, even, odd);
                s_v[buf][2 * b][w.lane] = even, s_v[buf][2 * b + 1][w.lane] = odd;
            }
    };
    if (steps > 0) {
        fetch(0, ring[0]);
        convert(0, ring[0]);
#pragma unroll
        for (int d = 1; d <= AHEAD; d++)
            if (d < steps)
                fetch(d, ring[d % AHEAD]);
    }
    __syncthreads();
    auto step = [&](int i, Mx4Raw<KK> (&raw)[2]) { // raw: the codes of step i + 1
        if (i + 1 < steps) {
            convert(i + 1, raw);
            if (i + 1 + AHEAD < steps)
                fetch(i + 1 + AHEAD, raw);
        }
        const int t0 = begin + 32 * i, buf = i & 1;
        if (t0 < w.most) {
            f32x4 s[2] = {w.origin(), w.origin()};
#pragma unroll
            for (int e = 0; e < 3; e++)
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(s_k[buf][kk * 2 + j][w.lane], w.q[kk][e], s[j], 0, 0, 0);
            bf16x8 p[3];
            w.softmax(s, t0, p);
#pragma unroll
            for (int ct = 0; ct < 2 * KK; ct++) {
                const bf16x8 v = s_v[buf][ct][w.lane];
#pragma unroll
                for (int e = 2; e >= 0; e--)
                    w.acc[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[e], w.acc[ct], 0, 0, 0);
            }
        }
        __syncthreads();
    };
    for (int i = 0; i < steps; i += AHEAD)
#pragma unroll
        for (int d = 0; d < AHEAD; d++)
            if (d == 0 || i + d < steps)
                step(i + d, ring[(d + 1) % AHEAD]);
    w.finish();

    if (w.out_row < 0)
        return;
    const int64_t line = (int64_t)w.out_row * a.n_heads + w.out_head;
    float        *dst = a.out + line * a.mx.head_dim;
    float         norm = w.limit == 0 ? 0.f : 1.f / w.l; // (no token seen: zeros; scores that are all -infinity: 0 / 0)
    if (a.chunks > 1) {
        dst  = a.ws_o + (line * a.chunks + chunk) * a.mx.head_dim;
        norm = 1.f;
        if (w.g == 0) {
            a.ws_ml[(line * a.chunks + chunk) * 2]     = w.m;
            a.ws_ml[(line * a.chunks + chunk) * 2 + 1] = w.l;
        }
    }
    // (a lane holds runs of 2 KK channels: a run, or a half of sixteen, is in the row as a whole)
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int ct = 0; ct < 2 * KK; ct += KK == 1 ? 2 : 4) {
            const int c = (4 * w.g + i) * 2 * KK + ct;
            if (c < a.mx.head_dim) {
                if constexpr (KK == 1)
                    dst[c] = w.acc[ct][i] * norm, dst[c + 1] = w.acc[ct + 1][i] * norm;
                else
                    store_four(dst + c, w.acc[ct][i] * norm, w.acc[ct + 1][i] * norm, w.acc[ct + 2][i] * norm, w.acc[ct + 3][i] * norm);
            }
        }
}

// How many chunks the line of a (row, head) has, 0 where nothing is to be joined; `empty`: its row sees no token.
__device__ __forceinline__ int mx4_line_chunks(const Mx4AttnArgs &a, int64_t line, bool &empty)
{
    const int row = (int)(line / a.n_heads);
    int       seq = row, rows = 1, row0 = row;
    if (a.row_offsets) { // the sequence whose rows hold this one: offsets[lo] <= row < offsets[hi]
        int lo = 0, hi = a.num_seqs;
        if (row < a.row_offsets[0] || row >= a.row_offsets[a.num_seqs])
            return 0;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.row_offsets[mid] <= row)
                lo = mid;
            else
                hi = mid;
        }
        seq  = lo;
        rows = mx4_rows(a, seq, row0);
    }
    const int ctx = mx4_context(a, seq), limit = max(ctx - rows + (row - row0) + 1, 0);
    empty = limit == 0;
    if (a.whole_lines && min(max((ctx + a.chunk_tokens - 1) / a.chunk_tokens, 1), a.chunks) == 1)
        return 0; // (decode writes a sequence of one chunk straight to `out`)
    return min(max((limit + a.chunk_tokens - 1) / a.chunk_tokens, 1), a.chunks);
}

// Many chunks: a workgroup per line.
__global__ void __launch_bounds__(kJoinThreads) nvk_mx4_join_kernel(const Mx4AttnArgs a)
{
    const int64_t line = blockIdx.x;
    bool          empty = true;
    const int     n = mx4_line_chunks(a, line, empty);
    if (n > 0)
        join_chunks(a.ws_o + line * a.chunks * a.mx.head_dim, a.ws_ml + line * a.chunks * 2, n, a.mx.head_dim, empty, a.out + line * a.mx.head_dim);
}

// Up to kJoinInside chunks (of many lines: a prefill's): a thread per four channels of a line.  (4088 rows of 8 heads of 80 channels, two
// chunks: 9.4 us, a workgroup per line 45.6.)
__global__ void __launch_bounds__(kJoinThreads) nvk_mx4_join_few_kernel(const Mx4AttnArgs a, unsigned lines)
{
    const unsigned quads = a.mx.head_dim >> 2;
    const int64_t  id = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x, line = id / quads;
    if (line >= lines)
        return;
    bool      empty = true;
    const int n = mx4_line_chunks(a, line, empty), c = (int)(id - line * quads) * 4;
    if (n > 0) {
        const float4 o = join_few<false>(a.ws_o + line * a.chunks * a.mx.head_dim + c, a.ws_ml + line * a.chunks * 2, n, a.mx.head_dim, empty);
        store_four(a.out + line * a.mx.head_dim + c, o.x, o.y, o.z, o.w);
    }
}

} // namespace nvk

namespace {

using nvk::Mx4AttnArgs;

using nvk::kDecodeWaves, nvk::kPrefillWaves;

struct Mx4Shape
{
    bool   prefill = false, pack = false, inside = false; // inside: the decode kernel joins the chunks itself
    int    col_blocks = 1, chunk_tokens = 32, chunks = 1;
    size_t ws_floats = 0, arrivals = 0;
};

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// How a call is cut into workgroups: columns first, then chunks of the context until the chip is full.
Mx4Shape mx4_shape(const nvk_mx4_pool *pool, int num_seqs, int n_heads, int total_rows, int max_rows, int max_ctx)
{
    Mx4Shape  s;
    const int group = n_heads / pool->n_kv_heads;
    // Waves that share the tokens while one wave holds a sequence's columns; else waves that share the columns, of which one alone
    // would work on up to 16.
    s.prefill = (long long)max_rows * group > 16;
    s.pack    = (long long)max_rows * group <= 4;
    s.col_blocks = s.prefill ? ceil_div((long long)max_rows * group, 16 * kPrefillWaves) : 1;
    const long long tasks = (long long)num_seqs * pool->n_kv_heads * s.col_blocks;
    // Cut the context while everything still runs at once (workgroups of four waves: so many fit a CU), into chunks of 192
    // tokens at least (a step of the four waves is 128; prefill's waves share the tokens: 64); not into more than can be joined
    // inside unless those were long.  (In chunks of 64, 128, 192, 256 tokens: 1 x 200 7.4, 6.3, 6.3, 6.2 us, 1 x 1000 8.6, 8.6, 8.3,
    // 9.0, 230 x 256 9.7, 9.7, 7.0, 7.1; 64 x 2048, two workgroups a CU: 28.1 us uncut, 39.6 in two rounds.)
    // Prompts with narrow heads are cut finer, more workgroups fit.  (1157 rows of 48 channels: 36.8 us uncut, 31.6 in 2, 26.9 in 3.)
    const long long per_cu = pool->kk == 8 ? 1 : s.prefill ? (pool->kk <= 2 ? 4 : 2) : s.pack ? 3 : 2, fit = per_cu * pool->num_cus;
    s.chunks = (int)std::max(1LL, std::min(fit / std::max(tasks, 1LL), (long long)max_ctx / (s.prefill ? 64 : 192)));
    // A prompt is cut where that saves more than the join costs: a step of 32 tokens takes about 1 us, the join 4 us and its reads and
    // writes at 5 TB/s.  (128 rows of 32 heads of 128 channels: 10.4 us uncut, 13.3 in 2; 256: 15.5 and 20.7 in 4; 512: 25.9 and 32.5 in 2;
    // 512 behind 1536: 82.7 and 69.5 in 2.  16 heads of 48: 128 rows 7.8 and 10.7, 1157 rows 37.5 and 27.3, 128 behind 896 31.1 and 14.9.)
    // The step is that of 128 channels.  Narrower ones are shorter, and the widest take about 2 us, so that the rule errs by up to a
    // fifth where the two sides are close: 512 rows of 32 heads of 64 are cut (23.1 us, uncut 19.1), 256 and 512 of 16 heads of 256
    // are not (26.6 and 45.7 us, cut 21.5 and 39.4).
    if (s.prefill && s.chunks > 1
        && (max_ctx - max_ctx / s.chunks) / 32 < 4 + (long long)total_rows * n_heads * pool->head_dim * s.chunks * 8 / 5000000)
        s.chunks = 1;
    if (!s.prefill && s.chunks > nvk::kJoinInside && max_ctx <= 512 * nvk::kJoinInside)
        s.chunks = nvk::kJoinInside;
    s.chunk_tokens = std::max(32, ceil_div(ceil_div(max_ctx, s.chunks), 32) * 32);
    s.chunks       = std::max(1, ceil_div(max_ctx, s.chunk_tokens));
    s.inside       = !s.prefill && s.chunks > 1 && s.chunks <= nvk::kJoinInside;
    s.arrivals     = s.inside ? (size_t)tasks : 0;
    s.ws_floats    = s.chunks > 1 ? (size_t)total_rows * n_heads * s.chunks * (pool->head_dim + 2) : 0;
    return s;
}

int reserve(nvk_mx4_pool *pool, size_t floats, size_t arrivals, hipStream_t st, const char *who)
{
    const int rc = nvk::grow_buffer(&pool->ws, &pool->ws_floats, &pool->ws_generation, floats, st, who);
    return rc != NVK_OK ? rc : nvk::grow_counters(&pool->arrivals, &pool->arrivals_cap, &pool->ws_generation, arrivals, st, who);
}

// What no call of up to this shape passes, fewer sequences (which are cut into more chunks) among them: as mx4_shape cuts, lines times
// chunks are at most the workgroups that fit the chip times the columns of one.
size_t most_floats(const nvk_mx4_pool *pool, int n_heads, int total_rows, int max_rows, int max_ctx)
{
    const long long columns = (long long)max_rows * (n_heads / pool->n_kv_heads), lines = (long long)total_rows * n_heads;
    long long       most = std::max(3 * std::min(columns, 4LL), 2 * std::min(columns, 16LL));
    if (columns > 16)
        most = std::max(most, 4 * std::min(columns, 16LL * kPrefillWaves));
    return (size_t)std::min(most * pool->num_cus, lines * (max_ctx / 64)) * (size_t)(pool->head_dim + 2);
}

template <int KK> void launch_attn(const Mx4AttnArgs &a, const Mx4Shape &s, unsigned blocks, hipStream_t st)
{
    if (s.prefill)
        hipLaunchKernelGGL(nvk::nvk_mx4_prefill_kernel<KK>, dim3(blocks), dim3(64 * kPrefillWaves), 0, st, a);
    else if (s.pack)
        hipLaunchKernelGGL((nvk::nvk_mx4_decode_kernel<KK, true>), dim3(blocks), dim3(64 * kDecodeWaves), 0, st, a);
    else
        hipLaunchKernelGGL((nvk::nvk_mx4_decode_kernel<KK, false>), dim3(blocks), dim3(64 * kDecodeWaves), 0, st, a);
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
    if ((long long)max_blocks * pool->block_size > nvk::kMostTokens || (long long)max_rows * n_heads > 0x3fffffffLL
        || max_ctx > nvk::kMostTokens)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: more than 2^31 tokens in a table, or 2^30 columns in a sequence", who);
    return NVK_OK;
}

int enqueue_attention(nvk_mx4_pool *pool, int layer, int num_seqs, int n_heads, int total_rows, const float *q,
                      const int *row_offsets, int max_rows, const int *tables, int max_blocks, const int *ctx_lens, int max_ctx,
                      float *out, hipStream_t st, const char *who)
{
    total_rows = (int)std::min((long long)total_rows, (long long)num_seqs * max_rows); // (rows behind these belong to nobody)
    const Mx4Shape  s = mx4_shape(pool, num_seqs, n_heads, total_rows, max_rows, max_ctx);
    const long long units = (long long)num_seqs * s.col_blocks * s.chunks;
    const long long blocks = units * pool->n_kv_heads;
    const long long lines = (long long)total_rows * n_heads, few = (lines * (pool->head_dim / 4) + nvk::kJoinThreads - 1) / nvk::kJoinThreads;
    if (!nvk::grid_fits(blocks, 64 * kDecodeWaves) || (s.chunks > 1 && !nvk::grid_fits(lines, nvk::kJoinThreads))
        || (s.chunks > 1 && !nvk::grid_fits(few, nvk::kJoinThreads)))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: %lld workgroups", who, blocks);
    int rc = reserve(pool, s.ws_floats, s.arrivals, st, who);
    if (rc != NVK_OK)
        return rc;
    Mx4AttnArgs a{};
    a.mx = pool->layer(layer), a.q = q, a.out = out, a.row_offsets = row_offsets, a.tables = tables, a.ctx_lens = ctx_lens;
    a.num_seqs = num_seqs, a.max_blocks = max_blocks, a.n_heads = n_heads, a.group = n_heads / pool->n_kv_heads;
    a.total_rows = total_rows, a.col_blocks = s.col_blocks, a.chunk_tokens = s.chunk_tokens, a.chunks = s.chunks;
    a.scale_log2e = (float)(1.4426950408889634 / std::sqrt((double)pool->head_dim));
    a.whole_lines = !s.prefill;
    a.arrivals    = s.inside ? pool->arrivals : nullptr;
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
    if (s.chunks > 1 && !s.inside) {
        if (s.chunks <= nvk::kJoinInside)
            hipLaunchKernelGGL(nvk::nvk_mx4_join_few_kernel, dim3((unsigned)few), dim3(nvk::kJoinThreads), 0, st, a, (unsigned)lines);
        else
            hipLaunchKernelGGL(nvk::nvk_mx4_join_kernel, dim3((unsigned)lines), dim3(nvk::kJoinThreads), 0, st, a);
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
    if (rc == NVK_OK)
        rc = check_attention(pool, layer, num_seqs, n_heads, (int)total, max_rows, max_blocks, max_ctx, who);
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
    if (pool->arrivals)
        (void)hipFree(pool->arrivals);
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
    return reserve(pool, most_floats(pool, n_heads, total_rows, max_rows, max_ctx), 3 * (size_t)pool->num_cus, pool->stream, who);
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
    if (!nvk::for_floats(q_dev) || !nvk::for_floats(out_dev))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: q or out is not aligned to its type", who);
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
    if (!nvk::for_floats(q_dev) || !nvk::for_floats(out_dev))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: q or out is not aligned to its type", who);
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
