// nvk_mx4.hip.h -- the 4-bit paged KV cache: its layout, its codes, and the pool behind nvk_mx4_*.
//
// A cached value is sign * {0, .5, 1, 1.5, 2, 3, 4, 6} * 2^e (e2m1 elements under one shared e8m0 exponent per 32 channels of
// a row): 17/32 byte a value instead of 4, and a bf16 number exactly, which is what lets the attention multiply it on
// bf16 matrix instructions without an error of its own.
//
// Layout.  The unit is a tile: 16 tokens of one kv-head, laid out in the order the matrix instruction's operands take, so
// that every lane of a wave fetches its part of a tile with one wide load and the tile with contiguous ones.
// With HDP = head_dim rounded up to 32, 64, 128 or 256 and KK = HDP / 32:
//     K codes   [token 16][HDP / 2 bytes]                  256 * KK bytes   (lane (g, token): channels g*8*KK ...)
//     V codes   [token quad 4][c16][token 4][KK bytes]     256 * KK bytes   (lane (quad, c16): channels c16*2*KK ...)
//     K scales  [group KK][token 16]                        16 * KK bytes
//     V scales  [group KK][token 16]                        16 * KK bytes
// in all 544 * KK bytes, 2176 = 17 whole 128-byte lines for head_dim 128.  A layer is [block][tile of the block][kv-head].
// A byte holds channels 2i (low nibble) and 2i + 1; padding channels stay zero.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "nvk_internal.h"

namespace nvk {

constexpr int kMx4Tile = 16; // tokens of a tile

// bytes of a tile for KK 32-channel groups
__host__ __device__ constexpr int mx4_tile_bytes(int kk) { return 544 * kk; }
__host__ __device__ constexpr int mx4_v_at(int kk) { return 256 * kk; }
__host__ __device__ constexpr int mx4_ks_at(int kk) { return 512 * kk; }
__host__ __device__ constexpr int mx4_vs_at(int kk) { return 528 * kk; }
inline int mx4_kk(int head_dim) { return head_dim <= 32 ? 1 : head_dim <= 64 ? 2 : head_dim <= 128 ? 4 : 8; }

// byte of channel pair (channel, channel + 1) of `tok` inside the V codes; channel even
__device__ __forceinline__ int mx4_v_byte(int tok, int channel, int kk)
{
    const int c16 = channel / (2 * kk), b = (channel % (2 * kk)) / 2;
    return (((tok >> 2) * 16 + c16) * 4 + (tok & 3)) * kk + b;
}

// Where the rows of a layer lie, for kernels that write or read single rows.
struct Mx4Layer
{
    unsigned char *base;
    int            num_blocks, block_size, n_kv_heads, head_dim, kk;
    // tile of (block, offset in the block, kv-head)
    __device__ __forceinline__ unsigned char *tile(int block, int offset, int kv_head) const
    {
        const int64_t t = (int64_t)block * (block_size / kMx4Tile) + offset / kMx4Tile;
        return base + (t * n_kv_heads + kv_head) * (int64_t)mx4_tile_bytes(kk);
    }
};

// The value of a code under a scale byte; byte 255 is a group that held an infinity or a NaN.
__device__ __forceinline__ float mx4_value(unsigned code, unsigned scale_byte)
{
    const unsigned mag  = code & 7u;
    // 0 .5 1 1.5 2 3 4 6: halves 0 1 2 3 4 6 8 12
    const unsigned half = mag < 4u ? mag : (mag < 6u ? 2u * (mag - 2u) : 4u * (mag - 4u));
    // * 2^(byte - 127), as a product of two factors that are both normal for every byte in [0, 254]
    const int   e = (int)scale_byte - 127;
    const float v = ((float)half * 0.5f) * __uint_as_float((unsigned)(127 + (e >> 1)) << 23)
                    * __uint_as_float((unsigned)(127 + (e - (e >> 1))) << 23);
    const float s = (code & 8u) ? -v : v;
    return scale_byte == 255u ? __uint_as_float(0x7fc00000u) : s;
}

// y in the 24 bits of a float, cut and not rounded, the last bit set where anything was cut off: above, at or below any number of
// few bits exactly where y is, so that what is decided on it is decided on y.  (Below 2^-126 the conversion rounds.  From 2^128 on
// y is an infinity, as it is in an fp32 cache.)
__device__ __forceinline__ float mx4_cut(double y)
{
    const unsigned long long bits = (unsigned long long)__double_as_longlong(y);
    const float f = (float)__longlong_as_double((long long)(bits & ~0x1fffffffULL));
    return __uint_as_float(__float_as_uint(f) | (((unsigned)bits & 0x1fffffffu) != 0u ? 1u : 0u));
}

// The scale byte of a group from the largest of its values' bits without their signs: the smallest e with amax <= 7 * 2^e, as e + 127;
// 255 where the group holds an infinity or a NaN.
// 7 and not 6: up to 7 the largest code, 6, is off by at most one unit of 2^e, which is what rounding between 4 and 6 costs
// anyway; beyond 7 clipping would cost more than the next exponent.  At most 125: 6 * 2^125 is the largest level below 2^128,
// and a value that is finite stays so (a stale infinity behind a context would reach its rows as 0 * infinity).
__device__ __forceinline__ unsigned mx4_scale_byte(unsigned amax)
{
    const int e = (int)(amax >> 23) - 129 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0); // over 1.75 * 2^ex
    return amax >= 0x7f800000u ? 255u : (unsigned)(min(max(e, -126), 125) + 127); // (0 or below the range: the smallest exponent)
}

// The codes of eight values under a scale byte up to 252: to the nearest, ties to the even code, 6 at most.  The conversion does
// just that, checked on every tie and its neighbours under every exponent.
__device__ __forceinline__ unsigned mx4_codes(const float (&x)[8], unsigned scale_byte)
{
    const float scale = __uint_as_float(scale_byte << 23);
    unsigned    word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[0], x[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[2], x[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[4], x[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[6], x[7], scale, 3);
    return word;
}

} // namespace nvk

struct nvk_mx4_pool
{
    int            n_layers = 0, num_blocks = 0, block_size = 0, n_kv_heads = 0, head_dim = 0, device = 0, kk = 0;
    size_t         layer_bytes = 0;
    unsigned char *base        = nullptr;
    hipStream_t    stream      = nullptr;
    int            num_cus     = 256;
    // partial results of sequences that are cut into chunks (grown on demand, never under stream capture)
    float    *ws            = nullptr;
    size_t    ws_floats     = 0;
    int      *arrivals      = nullptr; // of the join inside the decode kernel, zero between launches
    size_t    arrivals_cap  = 0;
    long long ws_generation = 0;

    nvk::Mx4Layer layer(int l) const
    {
        return {base + (size_t)l * layer_bytes, num_blocks, block_size, n_kv_heads, head_dim, kk};
    }
};
