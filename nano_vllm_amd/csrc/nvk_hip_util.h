// nvk_hip_util.h -- small host helpers of the operator translation units (HIP only).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>

#include "nvk_device_scope.h"
#include "nvk_internal.h"
#include "nvk_launch.h"

#define NVK_HIP_TRY(expr)                                                                                              \
    do {                                                                                                               \
        hipError_t e__ = (expr);                                                                                       \
        if (e__ != hipSuccess)                                                                                         \
            return nvk::fail(e__ == hipErrorOutOfMemory ? NVK_ERR_OOM : NVK_ERR_HIP, "%s failed: %s (%s:%d)", #expr,  \
                             hipGetErrorString(e__), __FILE__, __LINE__);                                              \
    } while (0)

namespace nvk {

// Tokens that a block table, a context may hold: an int has room for a tile, a chunk's rounding or a step more.
constexpr long long kMostTokens = 0x7fff0000LL;
// Whether a launch of `groups` workgroups of `threads` is one: the threads of a grid are counted in 32 bits.
inline bool grid_fits(long long groups, int threads) { return groups >= 0 && groups <= 0xffffffffLL / threads; }

inline bool for_floats(const void *p) { return ((uintptr_t)p & 3) == 0; } // aligned to one

// Whether launches on `stream` go into a graph and not to the device: captured by the caller, or recorded by this thread.
inline bool stream_is_capturing(hipStream_t stream)
{
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (Recording::of(stream))
        return true;
    return stream && hipStreamIsCapturing(stream, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

// A buffer of at least `want` elements, freed and allocated again when it has to grow.  Never while `stream` records a graph
// (the graph would keep the old address; hipMalloc is not capturable): refused, with the remedy in the message.
// The generation moves before the old buffer goes, not with the new one: where no memory is left for that, a graph which holds
// the old address must not be replayed either.
template <class T>
inline int grow_buffer(T **buf, size_t *have, long long *generation, size_t want, hipStream_t stream, const char *who)
{
    if (want <= *have)
        return NVK_OK;
    if (stream_is_capturing(stream))
        return fail(NVK_ERR_INVALID_ARG,
                    "%s: the workspace would have to grow while the stream is being captured: size it first, outside the "
                    "capture (the reserve_workspace entry point, or one direct call of the same shape)", who);
    if (*buf) {
        NVK_HIP_TRY(hipDeviceSynchronize()); // launches on any stream may still use the old buffer
        ++*generation;
        NVK_HIP_TRY(hipFree(*buf));
        *buf = nullptr, *have = 0;
    }
    NVK_HIP_TRY(hipMalloc((void **)buf, want * sizeof(T)));
    *have = want;
    ++*generation;
    return NVK_OK;
}

// Counters that every launch finds at zero and leaves at zero, grown like a workspace.
inline int grow_counters(int **counters, size_t *have, long long *generation, size_t want, hipStream_t stream, const char *who)
{
    if (want <= *have)
        return NVK_OK;
    want = want < 4096 ? 4096 : want;
    const int rc = grow_buffer(counters, have, generation, want, stream, who);
    if (rc != NVK_OK)
        return rc;
    // (the fill may still run when hipMemset returns, and a non-blocking stream does not wait for it)
    hipError_t e = hipMemset(*counters, 0, want * sizeof(int));
    if (e == hipSuccess)
        e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        (void)hipFree(*counters);
        *counters = nullptr, *have = 0;
        return fail(NVK_ERR_HIP, "%s: clearing the counters failed: %s", who, hipGetErrorString(e));
    }
    return NVK_OK;
}

// Device copies of a host-pointer call's arrays: one allocation, freed with the scope.
class Staging
{
    static constexpr int kMost = 16;
    char *dev_ = nullptr;
    struct Part
    {
        size_t at, bytes;
        const void *from;
    } part_[kMost];
    int    n_    = 0;
    size_t size_ = 0;

  public:
    Staging() = default;
    ~Staging()
    {
        if (dev_)
            (void)hipFree(dev_);
    }
    Staging(const Staging &)            = delete;
    Staging &operator=(const Staging &) = delete;
    // announces an array (`from` null: only room); returns its number
    int add(const void *from, size_t bytes)
    {
        part_[n_] = {size_, bytes, from};
        size_ += (bytes + 255) / 256 * 256;
        return n_++;
    }
    hipError_t upload(hipStream_t stream)
    {
        hipError_t e = hipMalloc((void **)&dev_, size_ + 256);
        for (int i = 0; e == hipSuccess && i < n_; i++)
            if (part_[i].from && part_[i].bytes)
                e = hipMemcpyAsync(dev_ + part_[i].at, part_[i].from, part_[i].bytes, hipMemcpyHostToDevice, stream);
        return e;
    }
    template <class T> T *at(int i) const { return reinterpret_cast<T *>(dev_ + part_[i].at); }
};

// Host-pointer calls: every used table entry and every row's place has to exist.
inline int check_tables(const int *tables, int num_seqs, int max_blocks, const int *ctx_lens, int block_size, int num_blocks,
                        const char *who)
{
    for (int s = 0; s < num_seqs; s++) {
        if (ctx_lens[s] < 0 || (long long)ctx_lens[s] > (long long)max_blocks * block_size)
            return fail(NVK_ERR_INVALID_ARG, "%s: sequence %d holds %d tokens, its table has room for %lld", who, s, ctx_lens[s],
                        (long long)max_blocks * block_size);
        const int need = (int)(((long long)ctx_lens[s] + block_size - 1) / block_size);
        for (int b = 0; b < need; b++) {
            const int id = tables[(size_t)s * max_blocks + b];
            if (id < 0 || id >= num_blocks)
                return fail(NVK_ERR_BAD_BLOCK, "%s: block %d of sequence %d outside [0,%d)", who, id, s, num_blocks);
        }
    }
    return NVK_OK;
}

} // namespace nvk
