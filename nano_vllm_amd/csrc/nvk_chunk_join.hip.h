// nvk_chunk_join.hip.h -- joining the partial results of a query whose tokens were cut into chunks (device code).
//
// Chunk c of a line, a (row, head), left o_c = sum p v, m_c and l_c = sum p with p = 2^(score - m_c); the result is
// sum_c w_c o_c / sum_c w_c l_c with w_c = 2^(m_c - max m).  Sums run in a fixed order.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nvk {

constexpr int kJoinThreads = 256; // a workgroup per line; head_dim <= 256

// `o` [n][hd] and `ml` [n][2] of the line -> out [hd].  A line without a token (every l_c 0) gives zeros.
__device__ __forceinline__ void join_chunks(const float *__restrict__ o, const float *__restrict__ ml, int n, int hd, float *__restrict__ out)
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
        out[c]          = L == 0.f ? sum : sum / L; // (no token: 0, or no number where one was met)
    }
}

} // namespace nvk
