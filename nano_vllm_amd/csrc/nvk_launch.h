// nvk_launch.h -- kernel launches and copies that go to a stream or, while the calling thread records a step, into a graph.
//
// A model's decode step is recorded once and replayed.  It is not recorded by capturing its stream: while any stream of the
// process captures, ROCm 7.2 refuses null-stream calls and device-wide waits of every thread, the application's among them, and
// such a call invalidates the capture and leaves the capturing stream unusable for good (tools/capture_recovery_probe.hip).  Here
// the launches of the recording thread on the recorded stream become nodes of a graph, each behind the one before; no stream
// is in another state than usual meanwhile, and other threads notice nothing.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <tuple>
#include <utility>

namespace nvk {

class Recording
{
    inline static thread_local Recording *current_ = nullptr;
    hipStream_t    stream_;
    hipGraph_t     graph_ = nullptr;
    hipGraphNode_t last_  = nullptr;
    hipError_t     error_;

    template <class F> void add(F &&node)
    {
        hipGraphNode_t fresh = nullptr;
        if (error_ == hipSuccess)
            error_ = node(&fresh, last_ ? &last_ : nullptr, (size_t)(last_ ? 1 : 0));
        if (error_ == hipSuccess)
            last_ = fresh;
    }

  public:
    explicit Recording(hipStream_t stream) : stream_(stream), error_(hipGraphCreate(&graph_, 0)) { current_ = this; }
    ~Recording()
    {
        current_ = nullptr;
        if (graph_)
            (void)hipGraphDestroy(graph_);
    }
    Recording(const Recording &)            = delete;
    Recording &operator=(const Recording &) = delete;

    // the calling thread's recording of `stream`, or null
    static Recording *of(hipStream_t stream) { return current_ && current_->stream_ == stream ? current_ : nullptr; }

    void kernel(const void *function, dim3 grid, dim3 block, size_t lds, void **args)
    {
        add([&](hipGraphNode_t *node, const hipGraphNode_t *behind, size_t n) {
            hipKernelNodeParams p{};
            p.func = const_cast<void *>(function), p.gridDim = grid, p.blockDim = block, p.sharedMemBytes = (unsigned)lds;
            p.kernelParams = args; // (their values are copied into the node)
            return hipGraphAddKernelNode(node, graph_, behind, n, &p);
        });
    }
    void copy(void *to, const void *from, size_t bytes, hipMemcpyKind kind)
    {
        add([&](hipGraphNode_t *node, const hipGraphNode_t *behind, size_t n) {
            return hipGraphAddMemcpyNode1D(node, graph_, behind, n, to, from, bytes, kind);
        });
    }
    // Ends the recording; what was recorded in `exec`, or the first error.
    hipError_t finish(hipGraphExec_t *exec)
    {
        current_ = nullptr;
        return error_ != hipSuccess ? error_ : hipGraphInstantiate(exec, graph_, nullptr, nullptr, 0);
    }
};

// hipLaunchKernelGGL, or a node of the thread's recording of `stream`; errors are left for hipGetLastError, or for finish().
template <class... P, class... A>
inline void launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, A &&...a)
{
    static_assert(sizeof...(P) == sizeof...(A), "one argument for each parameter");
    std::tuple<P...> values(static_cast<P>(std::forward<A>(a))...);
    std::apply(
        [&](P &...value) {
            void *args[] = {const_cast<void *>(static_cast<const volatile void *>(&value))..., nullptr};
            if (Recording *r = Recording::of(stream))
                r->kernel(reinterpret_cast<const void *>(kernel), grid, block, lds, args);
            else
                (void)hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, args, lds, stream);
        },
        values);
}

// hipMemcpyAsync likewise
inline hipError_t copy_async(void *to, const void *from, size_t bytes, hipMemcpyKind kind, hipStream_t stream)
{
    Recording *r = Recording::of(stream);
    if (!r)
        return hipMemcpyAsync(to, from, bytes, kind, stream);
    r->copy(to, from, bytes, kind);
    return hipSuccess;
}

} // namespace nvk
