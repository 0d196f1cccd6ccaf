// nvk_chunk_join.hip.h -- joining the partial results of a query whose tokens were cut into chunks (device code).
//
// Chunk c of a line, a (row, head), left o_c = sum p v, m_c and l_c = sum p with p = 2^(score - m_c); the result is
// sum_c w_c o_c / sum_c w_c l_c with w_c = 2^(m_c - max m).  Sums run in a fixed order.
// Up to kJoinInside chunks it is done by the workgroup that finishes last (no launch of its own: 2-3 us less), beyond that
// by a kernel whose workgroups spread over the chip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nvk {

constexpr int kJoinThreads = 256; // a workgroup per line; head_dim <= 256

// `o` [n][hd] and `ml` [n][2] of the line -> out [hd].  `empty`: a line that sees no token gives zeros (one whose scores are all
// -infinity is 0 / 0, no number).
__device__ __forceinline__ void join_chunks(const float *__restrict__ o, const float *__restrict__ ml, int n, int hd, bool empty,
                                            float *__restrict__ out)
{
    constexpr int W = kJoinThreads / 64;
    __shared__ float s_o[W][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // a lane takes every 64th chunk's maximum, then its weight
    float M = -INFINITY, L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = lane; c < n; c += 64)
        M = fmaxf(M, ml[2 * c]);
#pragma unroll
    for (int e = 32; e > 0; e >>= 1)
        M = fmaxf(M, __shfl_xor(M, e));
    for (int c0 = 0; c0 < n; c0 += 64) {
        float w = 0.f;
        if (c0 + lane < n) {
            const float m = ml[2 * (c0 + lane)];
            w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
            L += ml[2 * (c0 + lane) + 1] * w;
        }
        // the waves take chunks in turn, four at a time
        const int some = min(64, n - c0);
        for (int c = wave; c < some; c += 4 * W) {
            float f[4], y[4][4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int at = c + u * W;
                f[u] = at < some ? __shfl(w, at & 63) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    y[u][i] = at < some && lane + 64 * i < hd ? o[(int64_t)(c0 + at) * hd + lane + 64 * i] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    x[i] += y[u][i] * f[u];
        }
    }
#pragma unroll
    for (int e = 32; e > 0; e >>= 1)
        L += __shfl_xor(L, e);
#pragma unroll
    for (int i = 0; i < 4; i++)
        s_o[wave][lane + 64 * i] = x[i];
    __syncthreads();
    for (int c = threadIdx.x; c < hd; c += kJoinThreads) {
        const float sum = (s_o[0][c] + s_o[1][c]) + (s_o[2][c] + s_o[3][c]);
        out[c]          = empty ? 0.f : sum / L;
    }
}

// ---- inside the kernel that made the partial results ------------------------------------------------------------------
// Partial results are stored write-through (agent scope); every wave waits for its stores, the workgroup meets, one lane counts
// it in.  Who finds all others counted reads them, past the caches as they were stored.  Nobody waits for anybody, and the
// counter is zero again for the next launch.  (No acquire fence, which would drop what the XCD's L2 holds, for every
// workgroup that joins: 230 joins of two chunks took 14 us with it.)
constexpr int kJoinInside = 16; // chunks

// two floats at an address that is aligned to both
__device__ __forceinline__ void store_through(float *p, float x, float y)
{
    const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_through(const float *p)
{
    const unsigned long long v =
        __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32)));
}

// Whether this workgroup, whose partial results have just been stored, is the last of `n`.  Called by all its threads.
__device__ __forceinline__ bool arrived_last(int *counter, int n)
{
    __shared__ int s_last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const int last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        if (last)
            __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = last;
    }
    __syncthreads();
    return s_last;
}

// Four channels of a line from its n <= kJoinInside chunks, stored hd (o) and 2 (ml) floats apart; THROUGH: by other workgroups
// of this launch.
template <bool THROUGH> __device__ __forceinline__ float4 join_few(const float *o, const float *ml, int n, int hd, bool empty)
{
    float4 y[kJoinInside];
    float2 w[kJoinInside];
#pragma unroll
    for (int c = 0; c < kJoinInside; c++)
        if (c < n) {
            if constexpr (THROUGH) {
                const float2 a = load_through(o + (int64_t)c * hd), b = load_through(o + (int64_t)c * hd + 2);
                w[c] = load_through(ml + 2 * c);
                y[c] = make_float4(a.x, a.y, b.x, b.y);
            }
            else {
                w[c] = *reinterpret_cast<const float2 *>(ml + 2 * c);
                y[c] = *reinterpret_cast<const float4 *>(o + (int64_t)c * hd);
            }
        }
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int c = 0; c < kJoinInside; c++)
        if (c < n)
            M = fmaxf(M, w[c].x);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kJoinInside; c++)
        if (c < n) {
            const float f = w[c].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w[c].x - M);
            L += w[c].y * f;
            x.x += y[c].x * f, x.y += y[c].y * f, x.z += y[c].z * f, x.w += y[c].w * f;
        }
    return empty ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x / L, x.y / L, x.z / L, x.w / L);
}

} // namespace nvk
