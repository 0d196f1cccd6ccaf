// nvk_rotary.hip -- from projected rows to the paged cache in one launch: RMS norm of each query and key head, rotary
// positions, append (nvk_rope_*, nvk_pool_norm_rope_append, nvk_mx4_pool_norm_rope_append), and the way back from the 4-bit
// cache (nvk_mx4_pool_read_rows).
//
// The mathematics, for one head row x of a token at position p:
//     y = x / sqrt(mean(x^2) + eps) * w                       (only where a weight is given)
//     (a, b) -> (a c - b s, a s + b c),  c = m cos(p f_i), s = m sin(p f_i), i = 0 .. rotary_dim / 2 - 1
// Pair i is (y[2i], y[2i+1]) or (y[i], y[i + rotary_dim/2]); channels from rotary_dim on pass through.  The reference knows
// the first pairing over the whole head, unscaled and without a norm (Ops::apply_rope, include/ops/positional.hpp:13-39).
//
// Everything between the loaded row and the stored value is computed in 64 bits and rounded once: a key that is stored in
// 4 bits is then the nearest code of the exact value, whatever the order of the sums, and the angle of a far position keeps
// its fraction (p f to 2^-53 relative; in fp32 a position of 100 000 would leave 2^-7 of a radian).  It costs little: the
// kernel is bound by the rows it moves, and MI355X adds and multiplies fp64 at the unpacked fp32 rate.  (8192 rows of 32 + 8 + 8 heads
// of 128 channels, normed and rotated: 80 us for 403 MB, 5.0 TB/s; a large copy moves 4.7.  131072 rows of 8 + 8 heads into the 4-bit
// cache: 300 us for 1.2 GB.  One row: 3.9 us, the launch and its dependent loads.)
// gfx950 only; no CPU path.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include "nvk_addr.hip.h"
#include "nvk_hip_util.h"
#include "nvk_mx4.hip.h"

struct nvk_rope
{
    int                 head_dim = 0, rotary_dim = 0, layout = 0, device = 0;
    double              factor   = 1.0; // m, on cos and sin
    double             *freq_dev = nullptr; // half turns per position: no reduction by pi on the device
    std::vector<double> freq;
};

namespace nvk {

constexpr int kRotaryMaxHead = 256; // channels of a head row
constexpr int kRotaryBatch   = 512; // values a wave holds at a time: 8 per lane
constexpr int kRotaryWaves   = 4;

struct RotaryArgs
{
    const float  *q, *k, *v;   // [rows, heads, head_dim]; q or (k and v) may be null
    float        *q_out;
    const float  *q_weight, *k_weight; // [head_dim] or null
    double        eps, inv_head_dim;
    const double *freq; // [rotary_dim / 2], in half turns per position; or null
    double        factor;
    int           rotary_dim, half_layout;
    const int    *row_seqs, *positions, *tables;
    int           num_seqs, max_blocks, n_heads;
    float        *k_slab, *v_slab; // fp32 cache
    Mx4Layer      mx;              // its geometry also for the fp32 cache; base and kk only for the 4-bit one
};

// channels of pair p of a head row: rotated pairs first, then what is left two by two
__device__ __forceinline__ void pair_channels(const RotaryArgs &a, int p, int &ia, int &ib)
{
    const int half = a.rotary_dim >> 1;
    if (p < half && a.half_layout)
        ia = p, ib = p + half;
    else
        ia = 2 * p, ib = 2 * p + 1;
}

// Exchanges of doubles on the vector pipe: lane ^ 1, lane ^ 2, turns by 4 and 8 inside sixteen lanes, a quad's lane to all four.
template <int C> __device__ __forceinline__ double across(double x)
{
    const long long b = __double_as_longlong(x);
    const int       lo = __builtin_amdgcn_update_dpp(0, (int)b, C, 0xF, 0xF, true);
    const int       hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), C, 0xF, 0xF, true);
    return __longlong_as_double((long long)hi << 32 | (unsigned)lo);
}
// x of this lane and of lane ^ 16 (ROW) or lane ^ 32, added
template <bool ROW> __device__ __forceinline__ double fold(double x)
{
    const unsigned long long b = (unsigned long long)__double_as_longlong(x);
    const unsigned           lo = (unsigned)b, hi = (unsigned)(b >> 32);
    const auto l = ROW ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto h = ROW ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return __longlong_as_double((long long)((unsigned long long)h[0] << 32 | l[0]))
           + __longlong_as_double((long long)((unsigned long long)h[1] << 32 | l[1]));
}
template <int W> __device__ __forceinline__ double sum_over(double x) // over W = 16, 32 or 64 neighbouring lanes
{
    x += across<0xB1>(x);
    x += across<0x4E>(x);
    x += across<0x124>(x);
    x += across<0x128>(x);
    if constexpr (W >= 32)
        x = fold<true>(x);
    if constexpr (W >= 64)
        x = fold<false>(x);
    return x;
}

// A wave takes a row, or one of `parts` shares of its heads where rows are few (each share computes the row's angles again, side
// by side); its heads come in batches of kRotaryBatch values, the next one on its way while one is worked on.  W lanes hold
// one head row, PPL pairs each, so that a lane's angles stay in its registers; U head rows are in flight in a lane.
// For the 4-bit cache a batch of keys or values then crosses LDS, after which a lane holds eight neighbouring channels: one
// dword of codes.
template <int W, int PPL, bool MX4>
__global__ void __launch_bounds__(64 * kRotaryWaves) nvk_norm_rope_append_kernel(const RotaryArgs a, int rows, int parts)
{
    constexpr int U = PPL == 2 ? 2 : 4; // head rows per lane at a time
    constexpr int R = 64 / W;           // head rows side by side in a wave
    constexpr int HB = U * R;           // head rows per batch
    __shared__ __attribute__((aligned(16))) float s_row[MX4 ? kRotaryWaves : 1][MX4 ? kRotaryBatch : 4];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = blockIdx.x * kRotaryWaves + wave;
    const int row = id / parts, part = id - row * parts;
    if (row >= rows)
        return;
    // everything that does not hang on the row's place is on its way before the place is known
    const int pos = a.positions[row];
    const int seq = a.row_seqs ? a.row_seqs[row] : row;
    const int bs = a.mx.block_size, hd = a.mx.head_dim, pairs = hd >> 1, kv = a.mx.n_kv_heads;
    const int lane = threadIdx.x & 63;
    const int sub = lane / W, lw = lane % W; // which of the wave's head rows, and the lane's place in it
    int       ia[PPL], ib[PPL];
#pragma unroll
    for (int j = 0; j < PPL; j++)
        pair_channels(a, lw + j * W, ia[j], ib[j]);
    const int turned = a.freq ? a.rotary_dim >> 1 : 0;
    double    freq[PPL];
#pragma unroll
    for (int j = 0; j < PPL; j++)
        freq[j] = lw + j * W < turned ? a.freq[lw + j * W] : 0.0;

    // batches: keys, values, queries; this wave's are part, part + parts, ..
    const int kb = a.k ? (kv + HB - 1) / HB : 0, qb = a.q ? (a.n_heads + HB - 1) / HB : 0;
    const int batches = 2 * kb + qb;
    auto      kind_of = [&](int t) { return t < kb ? 0 : t < 2 * kb ? 1 : 2; }; // key, value, query
    auto      fetch = [&](int t, float2 (&x)[U][PPL], float2 (&w)[PPL]) {
        const int    kind = kind_of(t);
        const int    head0 = (t - kind * kb) * HB, heads = kind == 2 ? a.n_heads : kv;
        const float *src = (kind == 0 ? a.k : kind == 1 ? a.v : a.q) + (int64_t)row * heads * hd;
        const float *weight = kind == 0 ? a.k_weight : kind == 1 ? nullptr : a.q_weight;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < PPL; j++) {
                const int head = head0 + u * R + sub;
                x[u][j] = make_float2(0.f, 0.f);
                if (head < heads && lw + j * W < pairs)
                    x[u][j] = make_float2(src[head * hd + ia[j]], src[head * hd + ib[j]]);
            }
#pragma unroll
        for (int j = 0; j < PPL; j++) {
            w[j] = make_float2(1.f, 1.f);
            if (weight && lw + j * W < pairs)
                w[j] = make_float2(weight[ia[j]], weight[ib[j]]);
        }
    };
    float2 next[U][PPL], next_w[PPL];
    int    t = part;
    if (t < batches)
        fetch(t, next, next_w);

    // rows of padding, and rows that have no place in their table, are left alone
    if (pos < 0 || (a.k && (seq < 0 || seq >= a.num_seqs || pos / bs >= a.max_blocks)))
        return;
    const int  block = a.k ? a.tables[(int64_t)seq * a.max_blocks + pos / bs] : 0;
    const int  offset = pos % bs;
    const bool keep = a.k && block >= 0 && block < a.mx.num_blocks;
    double     cs[PPL], sn[PPL];
#pragma unroll
    for (int j = 0; j < PPL; j++) {
        cs[j] = 1.0, sn[j] = 0.0;
        if (lw + j * W < turned) {
            sincospi((double)pos * freq[j], &sn[j], &cs[j]);
            cs[j] *= a.factor, sn[j] *= a.factor;
        }
    }

    // one batch of keys, values or queries
    auto work = [&](auto k_, int t, const float2 (&x)[U][PPL], const float2 (&wt)[PPL]) {
        constexpr int kind = decltype(k_)::value;
        const int     head0 = (t - kind * kb) * HB, heads = kind == 2 ? a.n_heads : kv;
        const bool    weight = kind == 0 ? a.k_weight != nullptr : kind == 2 && a.q_weight != nullptr;
        double scale = 1.0; // of head row u: in lane u of every quad
        if (weight) {
            double ss[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                ss[u] = 0.0;
#pragma unroll
                for (int j = 0; j < PPL; j++)
                    ss[u] = fma((double)x[u][j].x, (double)x[u][j].x, fma((double)x[u][j].y, (double)x[u][j].y, ss[u]));
                ss[u] = sum_over<W>(ss[u]);
            }
            double mine = ss[0];
#pragma unroll
            for (int u = 1; u < U; u++)
                mine = (lane & 3) == u ? ss[u] : mine;
            scale = rsqrt(fma(mine, a.inv_head_dim, a.eps));
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int    head = head0 + u * R + sub;
            const double by = u == 0 ? across<0x00>(scale) : u == 1 ? across<0x55>(scale) : u == 2 ? across<0xAA>(scale) : across<0xFF>(scale);
#pragma unroll
            for (int j = 0; j < PPL; j++) {
                const bool there = head < heads && lw + j * W < pairs, turns = kind != 1 && lw + j * W < turned;
                float      xa = x[u][j].x, xb = x[u][j].y;
                if (weight || turns) { // (others keep what they hold: no 0 * infinity)
                    double ya = xa, yb = xb;
                    if (weight)
                        ya = ya * by * (double)wt[j].x, yb = yb * by * (double)wt[j].y;
                    if (turns) {
                        const double na = ya * cs[j] - yb * sn[j];
                        yb              = ya * sn[j] + yb * cs[j];
                        ya              = na;
                    }
                    const bool cut = MX4 && kind == 0;
                    xa = cut ? mx4_cut(ya) : (float)ya, xb = cut ? mx4_cut(yb) : (float)yb;
                }
                if (!there)
                    continue;
                if (MX4 && kind < 2) {
                    s_row[wave][(u * R + sub) * hd + ia[j]] = xa;
                    s_row[wave][(u * R + sub) * hd + ib[j]] = xb;
                }
                else {
                    float *dst;
                    if (kind == 2)
                        dst = a.q_out + ((int64_t)row * heads + head) * hd;
                    else
                        dst = (kind == 0 ? a.k_slab : a.v_slab) + row_float_index(block, offset, head, bs, kv, hd);
                    dst[ia[j]] = xa, dst[ib[j]] = xb;
                }
            }
        }
        if constexpr (MX4 && kind < 2) { // (the wave's own part of LDS: written and read by the same wave, in order)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int  octets = hd >> 3; // dwords of codes per head row
            const int  mine = lane / octets, c0 = (lane % octets) * 8, head = head0 + mine;
            const bool there = mine < HB && head < heads;
            float      y[8];
            unsigned   amax = 0; // as bits: an infinity or a NaN is larger than any number
#pragma unroll
            for (int i = 0; i < 8; i++) {
                y[i] = there ? s_row[wave][mine * hd + c0 + i] : 0.f;
                amax = max(amax, __float_as_uint(y[i]) & 0x7fffffffu);
            }
            // the group of 32 channels is four lanes, or what is left of the row
            const int group = c0 / 32;
            if (octets % 4 == 0) {
                amax = max(amax, (unsigned)__builtin_amdgcn_update_dpp(0, (int)amax, 0xB1, 0xF, 0xF, true));
                amax = max(amax, (unsigned)__builtin_amdgcn_update_dpp(0, (int)amax, 0x4E, 0xF, 0xF, true));
            }
            else { // (rows of 48 or 56 channels are 6 or 7 lanes: partners go by the place in the row, each lane asks all of them)
                const unsigned own = amax;
#pragma unroll
                for (int o = 1; o <= 3; o++) {
                    const int pc = (((c0 >> 3) & 3) ^ o) + 4 * group;
                    amax = max(amax, (unsigned)__shfl((int)own, pc < octets ? mine * octets + pc : lane));
                }
            }
            if (there) {
                const unsigned sb = mx4_scale_byte(amax), word = sb == 255u ? 0u : mx4_codes(y, sb);
                const int      kk = a.mx.kk, tok = offset % kMx4Tile;
                unsigned char *tile = a.mx.tile(block, offset, head);
                if (kind == 0)
                    *reinterpret_cast<unsigned *>(tile + tok * 16 * kk + c0 / 2) = word;
                else if (kk >= 4)
                    *reinterpret_cast<unsigned *>(tile + mx4_v_at(kk) + mx4_v_byte(tok, c0, kk)) = word;
                else
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        tile[mx4_v_at(kk) + mx4_v_byte(tok, c0 + 2 * i, kk)] = (unsigned char)(word >> (8 * i));
                if (c0 % 32 == 0)
                    tile[(kind == 0 ? mx4_ks_at(kk) : mx4_vs_at(kk)) + group * kMx4Tile + tok] = (unsigned char)sb;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    for (; t < batches; t += parts) {
        float2 x[U][PPL], wt[PPL];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < PPL; j++)
                x[u][j] = next[u][j];
#pragma unroll
        for (int j = 0; j < PPL; j++)
            wt[j] = next_w[j];
        if (t + parts < batches)
            fetch(t + parts, next, next_w);
        const int kind = kind_of(t);
        if (kind == 2)
            work(std::integral_constant<int, 2>(), t, x, wt);
        else if (keep && kind == 0)
            work(std::integral_constant<int, 0>(), t, x, wt);
        else if (keep)
            work(std::integral_constant<int, 1>(), t, x, wt);
    }
}

// ---- the values of cached rows: one thread per 8 channels of (row, kv-head).  Bound by the fp32 it writes; 3001 rows of 6 heads of 48
// channels (7 MB) take 4.8 us, which is the launch and its dependent loads --------------------------------------------------
__global__ void __launch_bounds__(256)
    nvk_mx4_read_rows_kernel(const Mx4Layer mx, int rows, const int *__restrict__ row_seqs, const int *__restrict__ positions,
                             const int *__restrict__ tables, int num_seqs, int max_blocks, float *__restrict__ k_out,
                             float *__restrict__ v_out)
{
    const unsigned octets = mx.head_dim >> 3, per_row = mx.n_kv_heads * octets;
    const int64_t  id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t  row = id / per_row;
    if (row >= rows)
        return;
    const unsigned i = (unsigned)(id - row * per_row);
    const int      pos = positions[row], seq = row_seqs ? row_seqs[row] : (int)row, bs = mx.block_size;
    if (pos < 0 || seq < 0 || seq >= num_seqs || pos / bs >= max_blocks)
        return;
    const int block = tables[(int64_t)seq * max_blocks + pos / bs], offset = pos % bs, tok = offset % kMx4Tile;
    if (block < 0 || block >= mx.num_blocks)
        return;
    const int            head = i / octets, c0 = (i % octets) * 8, kk = mx.kk;
    const unsigned char *tile = mx.tile(block, offset, head);
    unsigned             kw = *reinterpret_cast<const unsigned *>(tile + tok * 16 * kk + c0 / 2), vw = 0;
    if (kk >= 4)
        vw = *reinterpret_cast<const unsigned *>(tile + mx4_v_at(kk) + mx4_v_byte(tok, c0, kk));
    else
#pragma unroll
        for (int j = 0; j < 4; j++)
            vw |= (unsigned)tile[mx4_v_at(kk) + mx4_v_byte(tok, c0 + 2 * j, kk)] << (8 * j);
    const unsigned ks = tile[mx4_ks_at(kk) + (c0 / 32) * kMx4Tile + tok], vs = tile[mx4_vs_at(kk) + (c0 / 32) * kMx4Tile + tok];
    const int64_t  at = (row * mx.n_kv_heads + head) * mx.head_dim + c0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float4 k, v;
        k.x = mx4_value((kw >> (16 * h)) & 15u, ks), k.y = mx4_value((kw >> (16 * h + 4)) & 15u, ks);
        k.z = mx4_value((kw >> (16 * h + 8)) & 15u, ks), k.w = mx4_value((kw >> (16 * h + 12)) & 15u, ks);
        v.x = mx4_value((vw >> (16 * h)) & 15u, vs), v.y = mx4_value((vw >> (16 * h + 4)) & 15u, vs);
        v.z = mx4_value((vw >> (16 * h + 8)) & 15u, vs), v.w = mx4_value((vw >> (16 * h + 12)) & 15u, vs);
        store_four(k_out + at + 4 * h, k.x, k.y, k.z, k.w);
        store_four(v_out + at + 4 * h, v.x, v.y, v.z, v.w);
    }
}

} // namespace nvk

namespace {

using nvk::RotaryArgs;

constexpr int kCus = 256; // MI355X

template <bool MX4> void launch_rotary(const RotaryArgs &a, int rows, hipStream_t st)
{
    const int hd = a.mx.head_dim, pairs = hd / 2;
    const int w = pairs <= 16 ? 16 : pairs <= 32 ? 32 : 64;
    const int hb = pairs > 64 ? 2 : 4 * (64 / w);
    const int batches = (a.k ? 2 * ((a.mx.n_kv_heads + hb - 1) / hb) : 0) + (a.q ? (a.n_heads + hb - 1) / hb : 0);
    // Few rows: a row's batches are spread over several waves, one each at most, while there are no more than sixteen waves for
    // every CU; up to 32 where three are left to each, which pays for its angles.  (3001 rows of three batches: 10.6 us a wave a
    // row, 12.9 two, 13.9 three; 256 rows of twelve: 7.9 us; 2111 rows of nine: 20.0 us a wave a row, 16.2 three.)
    const int  parts = (int)std::max({1LL, std::min((long long)batches, 16LL * kCus / rows), std::min(batches / 3LL, 32LL * kCus / rows)});
    const dim3 grid((unsigned)(((long long)rows * parts + nvk::kRotaryWaves - 1) / nvk::kRotaryWaves)), block(64 * nvk::kRotaryWaves);
    if (pairs > 64)
        hipLaunchKernelGGL((nvk::nvk_norm_rope_append_kernel<64, 2, MX4>), grid, block, 0, st, a, rows, parts);
    else if (w == 64)
        hipLaunchKernelGGL((nvk::nvk_norm_rope_append_kernel<64, 1, MX4>), grid, block, 0, st, a, rows, parts);
    else if (w == 32)
        hipLaunchKernelGGL((nvk::nvk_norm_rope_append_kernel<32, 1, MX4>), grid, block, 0, st, a, rows, parts);
    else
        hipLaunchKernelGGL((nvk::nvk_norm_rope_append_kernel<16, 1, MX4>), grid, block, 0, st, a, rows, parts);
}

// Host-pointer calls: every row has a place of its own.  (Two rows in one slot: whichever comes last would stay, or a mix.)
int check_rows(int rows, const int *row_seqs, const int *positions, const int *tables, int num_seqs, int max_blocks,
               int block_size, int num_blocks, bool own_slots, const char *who)
{
    try {
        std::vector<long long> slots;
        for (int r = 0; r < rows; r++) {
            const int pos = positions[r], seq = row_seqs ? row_seqs[r] : r;
            if (pos < 0)
                continue; // padding
            if (seq < 0 || seq >= num_seqs || pos / block_size >= max_blocks)
                return nvk::fail(NVK_ERR_INVALID_ARG, "%s: row %d: position %d of sequence %d outside its table", who, r, pos, seq);
            const int pb = tables[(size_t)seq * max_blocks + pos / block_size];
            if (pb < 0 || pb >= num_blocks)
                return nvk::fail(NVK_ERR_BAD_BLOCK, "%s: block %d of sequence %d outside [0,%d)", who, pb, seq, num_blocks);
            slots.push_back((long long)pb * block_size + pos % block_size);
        }
        if (own_slots) {
            std::sort(slots.begin(), slots.end());
            if (std::adjacent_find(slots.begin(), slots.end()) != slots.end())
                return nvk::fail(NVK_ERR_INVALID_ARG, "%s: two rows share one slot of the cache", who);
        }
    }
    catch (const std::bad_alloc &) {
        return nvk::fail(NVK_ERR_OOM, "%s: host allocation failed", who);
    }
    return NVK_OK;
}

// The part that the two caches share: checks, staging of host arrays, launch.
template <bool MX4>
int norm_rope_append(RotaryArgs a, int device, hipStream_t own_stream, const nvk_rope *rope, int rows,
                     int ptr_kind, void *stream, const char *who)
{
    const int hd = a.mx.head_dim, bs = a.mx.block_size, kv = a.mx.n_kv_heads;
    if (ptr_kind != NVK_PTR_HOST && ptr_kind != NVK_PTR_DEVICE)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: ptr_kind %d", who, ptr_kind);
    if (rows < 0 || a.num_seqs < 0 || (a.k && a.max_blocks <= 0) || a.n_heads <= 0 || !(a.eps >= 0.0))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: bad arguments (rows %d, num_seqs %d, max_blocks %d, n_heads %d)", who, rows,
                         a.num_seqs, a.max_blocks, a.n_heads);
    if ((long long)a.n_heads * hd > 0x7fffffffLL)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: n_heads %d", who, a.n_heads);
    if (hd % 2 != 0 || hd > nvk::kRotaryMaxHead)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: head_dim %d (even, at most %d)", who, hd, nvk::kRotaryMaxHead);
    if (a.k && (long long)a.max_blocks * bs > nvk::kMostTokens)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: a table of %d blocks of %d tokens passes 2^31 tokens", who, a.max_blocks, bs);
    if (rope && (rope->head_dim != hd || rope->device != device))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: the rotary table is for head_dim %d on device %d, the pool has %d on %d", who,
                         rope->head_dim, rope->device, hd, device);
    if (rows == 0)
        return NVK_OK;
    if (!nvk::grid_fits((rows + (long long)nvk::kRotaryWaves - 1) / nvk::kRotaryWaves, 64 * nvk::kRotaryWaves))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: %d rows", who, rows);
    if ((!a.q && !a.k) || (a.q != nullptr) != (a.q_out != nullptr) || (a.k != nullptr) != (a.v != nullptr))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: q and q_out, k_rows and v_rows come in pairs, at least one of them", who);
    if (!a.positions || (a.k && !a.tables))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: positions or block_tables missing", who);
    if (!nvk::for_floats(a.q) || !nvk::for_floats(a.q_out) || !nvk::for_floats(a.k) || !nvk::for_floats(a.v))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: rows are not aligned to their type", who);

    if (!a.k) // (positions alone matter: what else is given may be of any size)
        a.row_seqs = a.tables = nullptr;

    NVK_SCOPE(device);
    hipStream_t st = (ptr_kind == NVK_PTR_DEVICE && stream) ? (hipStream_t)stream : own_stream;
    a.inv_head_dim = 1.0 / hd;
    a.freq = rope ? rope->freq_dev : nullptr;
    a.factor = rope ? rope->factor : 1.0;
    a.rotary_dim = rope ? rope->rotary_dim : 0;
    a.half_layout = rope ? (rope->layout == NVK_ROPE_HALF) : 0;
    if (ptr_kind == NVK_PTR_DEVICE) {
        launch_rotary<MX4>(a, rows, st);
        NVK_HIP_TRY(hipGetLastError());
        return NVK_OK;
    }

    if (a.k) {
        const int rc = check_rows(rows, a.row_seqs, a.positions, a.tables, a.num_seqs, a.max_blocks, bs, a.mx.num_blocks, true, who);
        if (rc != NVK_OK)
            return rc;
    }
    float       *q_host = a.q_out;
    const size_t qb = a.q ? (size_t)rows * a.n_heads * hd * sizeof(float) : 0, kb = a.k ? (size_t)rows * kv * hd * sizeof(float) : 0;
    const size_t rb = (size_t)rows * sizeof(int), tb = a.tables ? (size_t)a.num_seqs * a.max_blocks * sizeof(int) : 0;
    nvk::Staging s;
    const int    iq = s.add(a.q, qb), ik = s.add(a.k, kb), iv = s.add(a.v, kb), ip = s.add(a.positions, rb),
              is = s.add(a.row_seqs, a.row_seqs ? rb : 0), it = s.add(a.tables, tb),
              iw = s.add(a.q_weight, a.q_weight ? hd * sizeof(float) : 0), ix = s.add(a.k_weight, a.k_weight ? hd * sizeof(float) : 0);
    NVK_HIP_TRY(s.upload(st));
    if (a.q)
        a.q = s.at<float>(iq), a.q_out = s.at<float>(iq); // in place: a row is read whole before it is written
    if (a.k)
        a.k = s.at<float>(ik), a.v = s.at<float>(iv);
    a.positions = s.at<int>(ip);
    a.row_seqs  = a.row_seqs ? s.at<int>(is) : nullptr;
    a.tables    = s.at<int>(it);
    a.q_weight  = a.q_weight ? s.at<float>(iw) : nullptr;
    a.k_weight  = a.k_weight ? s.at<float>(ix) : nullptr;
    launch_rotary<MX4>(a, rows, st);
    NVK_HIP_TRY(hipGetLastError());
    // (rows of padding come back as they went)
    if (q_host && a.q)
        NVK_HIP_TRY(hipMemcpyAsync(q_host, a.q_out, qb, hipMemcpyDeviceToHost, st));
    NVK_HIP_TRY(hipStreamSynchronize(st));
    return NVK_OK;
}

} // namespace

extern "C" {

int nvk_rope_create(int head_dim, int rotary_dim, int layout, double theta, int scaling, double factor, int original_len,
                    int device, nvk_rope **out_rope)
{
    if (!out_rope)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: out_rope is null");
    *out_rope = nullptr;
    if (head_dim <= 0 || head_dim > nvk::kRotaryMaxHead || head_dim % 2 != 0 || rotary_dim <= 0 || rotary_dim > head_dim
        || rotary_dim % 2 != 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: head_dim %d, rotary_dim %d (both even, at most %d)", head_dim,
                         rotary_dim, nvk::kRotaryMaxHead);
    if (layout != NVK_ROPE_INTERLEAVED && layout != NVK_ROPE_HALF)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: layout %d", layout);
    if (scaling < NVK_ROPE_SCALE_NONE || scaling > NVK_ROPE_SCALE_YARN)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: scaling %d", scaling);
    if (!(theta > 0.0) || !std::isfinite(theta))
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: theta %g", theta);
    if (scaling != NVK_ROPE_SCALE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: factor %g (1 or more)", factor);
    if (scaling == NVK_ROPE_SCALE_NTK && rotary_dim <= 2)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: a changed base needs more than one pair (rotary_dim %d)", rotary_dim);
    if (scaling == NVK_ROPE_SCALE_YARN && original_len <= 0)
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_create: original_len %d", original_len);
    if (device < 0 || device >= nvk::device_count_cached())
        return nvk::fail(nvk::device_count_cached() ? NVK_ERR_INVALID_ARG : NVK_ERR_NO_DEVICE,
                         "nvk_rope_create: device %d outside [0,%d)", device, nvk::device_count_cached());
    nvk_rope *r = nullptr;
    try {
        r = new nvk_rope();
        r->head_dim = head_dim, r->rotary_dim = rotary_dim, r->layout = layout, r->device = device;
        const double base = scaling == NVK_ROPE_SCALE_NTK
                                ? theta * std::pow(factor, (double)rotary_dim / (double)(rotary_dim - 2)) : theta;
        for (int i = 0; i < rotary_dim; i += 2) {
            double f = std::pow(base, -(double)i / rotary_dim);
            if (scaling == NVK_ROPE_SCALE_LINEAR)
                f /= factor;
            else if (scaling == NVK_ROPE_SCALE_YARN) {
                // turns a pair makes over the trained context: up to 1 slowed down, from 32 on kept, a ramp between
                const double turns = original_len * f / (2.0 * M_PI);
                const double kept  = std::min(1.0, std::max(0.0, (turns - 1.0) / 31.0));
                f                  = (1.0 - kept) * f / factor + kept * f;
            }
            r->freq.push_back(f);
        }
        if (scaling == NVK_ROPE_SCALE_YARN)
            r->factor = 0.1 * std::log(factor) + 1.0;
    }
    catch (const std::bad_alloc &) {
        delete r;
        return nvk::fail(NVK_ERR_OOM, "nvk_rope_create: host allocation failed");
    }
    double half_turns[nvk::kRotaryMaxHead / 2];
    for (size_t i = 0; i < r->freq.size(); i++)
        half_turns[i] = r->freq[i] / M_PI;
    nvk::DeviceScope scope(device);
    hipError_t       e = scope.ok ? hipSuccess : hipErrorInvalidDevice;
    if (e == hipSuccess)
        e = hipMalloc((void **)&r->freq_dev, r->freq.size() * sizeof(double));
    if (e == hipSuccess)
        e = hipMemcpy(r->freq_dev, half_turns, r->freq.size() * sizeof(double), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        const int rc = nvk::fail(e == hipErrorOutOfMemory ? NVK_ERR_OOM : NVK_ERR_HIP, "nvk_rope_create: %s", hipGetErrorString(e));
        if (r->freq_dev)
            (void)hipFree(r->freq_dev);
        delete r;
        return rc;
    }
    *out_rope = r;
    return NVK_OK;
}

int nvk_rope_destroy(nvk_rope *rope)
{
    if (!rope)
        return NVK_OK;
    nvk::DeviceScope scope(rope->device); // (a release path: goes on whatever the switch returned)
    (void)hipDeviceSynchronize();         // launches on any stream may still read the table
    (void)hipFree(rope->freq_dev);
    delete rope;
    return NVK_OK;
}

int nvk_rope_frequencies(const nvk_rope *rope, double *freq, int cap, double *factor)
{
    if (!rope || cap < 0 || (cap > 0 && !freq))
        return nvk::fail(NVK_ERR_INVALID_ARG, "nvk_rope_frequencies: bad arguments");
    for (int i = 0; i < std::min(cap, (int)rope->freq.size()); i++)
        freq[i] = rope->freq[(size_t)i];
    if (factor)
        *factor = rope->factor;
    return (int)rope->freq.size();
}

int nvk_pool_norm_rope_append(nvk_pool *pool, int layer, const nvk_rope *rope, int rows, int n_heads, const float *q,
                              float *q_out, const float *k_rows, const float *v_rows, const float *q_weight,
                              const float *k_weight, float eps, const int *row_seqs, const int *positions,
                              const int *block_tables, int num_seqs, int max_blocks, int ptr_kind, void *stream)
{
    const char *who = "nvk_pool_norm_rope_append";
    int         g[6];
    int         rc = pool ? nvk_pool_geometry(pool, g) : nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pool", who);
    if (rc != NVK_OK)
        return rc;
    void *k = nullptr, *v = nullptr, *own = nullptr;
    if ((rc = nvk_pool_layer_ptrs(pool, layer, &k, &v)) != NVK_OK || (rc = nvk_pool_stream(pool, &own)) != NVK_OK)
        return rc;
    RotaryArgs a{};
    a.q = q, a.q_out = q_out, a.k = k_rows, a.v = v_rows, a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps;
    a.row_seqs = row_seqs, a.positions = positions, a.tables = block_tables, a.num_seqs = num_seqs, a.max_blocks = max_blocks;
    a.n_heads = n_heads, a.k_slab = (float *)k, a.v_slab = (float *)v;
    a.mx.num_blocks = g[1], a.mx.block_size = g[2], a.mx.n_kv_heads = g[3], a.mx.head_dim = g[4];
    return norm_rope_append<false>(a, g[5], (hipStream_t)own, rope, rows, ptr_kind, stream, who);
}

int nvk_mx4_pool_norm_rope_append(nvk_mx4_pool *pool, int layer, const nvk_rope *rope, int rows, int n_heads, const float *q,
                                  float *q_out, const float *k_rows, const float *v_rows, const float *q_weight,
                                  const float *k_weight, float eps, const int *row_seqs, const int *positions,
                                  const int *block_tables, int num_seqs, int max_blocks, int ptr_kind, void *stream)
{
    const char *who = "nvk_mx4_pool_norm_rope_append";
    if (!pool)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pool", who);
    if (layer < 0 || layer >= pool->n_layers)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: layer %d outside [0,%d)", who, layer, pool->n_layers);
    RotaryArgs a{};
    a.q = q, a.q_out = q_out, a.k = k_rows, a.v = v_rows, a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps;
    a.row_seqs = row_seqs, a.positions = positions, a.tables = block_tables, a.num_seqs = num_seqs, a.max_blocks = max_blocks;
    a.n_heads = n_heads, a.mx = pool->layer(layer);
    return norm_rope_append<true>(a, pool->device, pool->stream, rope, rows, ptr_kind, stream, who);
}

int nvk_mx4_pool_read_rows(nvk_mx4_pool *pool, int layer, int rows, const int *row_seqs, const int *positions,
                           const int *block_tables, int num_seqs, int max_blocks, float *k_out, float *v_out, int ptr_kind,
                           void *stream)
{
    const char *who = "nvk_mx4_pool_read_rows";
    if (!pool)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: null pool", who);
    if (layer < 0 || layer >= pool->n_layers)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: layer %d outside [0,%d)", who, layer, pool->n_layers);
    if (ptr_kind != NVK_PTR_HOST && ptr_kind != NVK_PTR_DEVICE)
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: ptr_kind %d", who, ptr_kind);
    if (rows < 0 || num_seqs < 0 || max_blocks <= 0 || (long long)max_blocks * pool->block_size > nvk::kMostTokens
        || (rows > 0 && (!positions || !block_tables || !k_out || !v_out)))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: bad arguments", who);
    if (rows == 0)
        return NVK_OK;
    if (!nvk::for_floats(k_out) || !nvk::for_floats(v_out))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: rows are not aligned to their type", who);
    NVK_SCOPE(pool->device);
    hipStream_t st = (ptr_kind == NVK_PTR_DEVICE && stream) ? (hipStream_t)stream : pool->stream;
    const long long threads = (long long)rows * pool->n_kv_heads * (pool->head_dim / 8);
    if (!nvk::grid_fits((threads + 255) / 256, 256))
        return nvk::fail(NVK_ERR_INVALID_ARG, "%s: %d rows", who, rows);
    const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
    if (ptr_kind == NVK_PTR_DEVICE) {
        hipLaunchKernelGGL(nvk::nvk_mx4_read_rows_kernel, grid, block, 0, st, pool->layer(layer), rows, row_seqs, positions,
                           block_tables, num_seqs, max_blocks, k_out, v_out);
        NVK_HIP_TRY(hipGetLastError());
        return NVK_OK;
    }
    const int rc = check_rows(rows, row_seqs, positions, block_tables, num_seqs, max_blocks, pool->block_size, pool->num_blocks,
                              false, who);
    if (rc != NVK_OK)
        return rc;
    const size_t kb = (size_t)rows * pool->n_kv_heads * pool->head_dim * sizeof(float), rb = (size_t)rows * sizeof(int);
    nvk::Staging s;
    const int    ik = s.add(k_out, kb), iv = s.add(v_out, kb), ip = s.add(positions, rb), is = s.add(row_seqs, row_seqs ? rb : 0),
              it = s.add(block_tables, (size_t)num_seqs * max_blocks * sizeof(int));
    NVK_HIP_TRY(s.upload(st));
    hipLaunchKernelGGL(nvk::nvk_mx4_read_rows_kernel, grid, block, 0, st, pool->layer(layer), rows,
                       row_seqs ? s.at<int>(is) : (const int *)nullptr, s.at<int>(ip), s.at<int>(it), num_seqs, max_blocks,
                       s.at<float>(ik), s.at<float>(iv));
    NVK_HIP_TRY(hipGetLastError());
    NVK_HIP_TRY(hipMemcpyAsync(k_out, s.at<float>(ik), kb, hipMemcpyDeviceToHost, st));
    NVK_HIP_TRY(hipMemcpyAsync(v_out, s.at<float>(iv), kb, hipMemcpyDeviceToHost, st));
    NVK_HIP_TRY(hipStreamSynchronize(st));
    return NVK_OK;
}

} // extern "C"
