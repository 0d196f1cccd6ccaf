// recording_driver.cpp -- test infrastructure: nvk_launch.h over a HIP runtime that only writes down its calls, without a device.
// tests/test_step_recording.py builds and runs it; prints one line per mistake.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <thread>
#include <vector>

#include "nvk_launch.h"

struct Params // a kernel's argument block
{
    int    n;
    double x;
};
static void one(const Params, float *) {}
static void two(unsigned, const int *, double) {}

static std::vector<std::string> g_calls; // in order
static std::vector<std::intptr_t>  g_behind;
static int  g_nodes = 0, g_graphs = 0, g_fail_at = -1;
static int  g_wrong = 0;

static void expect(bool ok, const char *what)
{
    if (!ok)
        std::printf("%s\n", what), g_wrong++;
}
static std::string values(const void *f, void **a)
{
    char s[96] = "?";
    if (f == reinterpret_cast<const void *>(&one)) {
        const Params *p = static_cast<Params *>(a[0]);
        std::snprintf(s, sizeof s, "one(%d,%g,%d)", p->n, p->x, *static_cast<float **>(a[1]) != nullptr);
    }
    else if (f == reinterpret_cast<const void *>(&two))
        std::snprintf(s, sizeof s, "two(%u,%d,%g)", *static_cast<unsigned *>(a[0]), *static_cast<int **>(a[1]) != nullptr, *static_cast<double *>(a[2]));
    return s;
}
static hipError_t node(hipGraphNode_t *out, const hipGraphNode_t *behind, size_t n, const std::string &what)
{
    if (g_nodes == g_fail_at)
        return hipErrorOutOfMemory;
    g_behind.push_back(n == 1 ? reinterpret_cast<std::intptr_t>(behind[0]) : -(std::intptr_t)n);
    *out = reinterpret_cast<hipGraphNode_t>((std::intptr_t)++g_nodes);
    g_calls.push_back("node " + what);
    return hipSuccess;
}
extern "C" {
hipError_t hipGraphCreate(hipGraph_t *g, unsigned) { return *g = reinterpret_cast<hipGraph_t>(8), g_graphs++, hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t) { return g_graphs--, hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t *e, hipGraph_t, hipGraphNode_t *, char *, size_t)
{
    return *e = reinterpret_cast<hipGraphExec_t>(16), g_calls.push_back("instantiate"), hipSuccess;
}
hipError_t hipGraphAddKernelNode(hipGraphNode_t *out, hipGraph_t, const hipGraphNode_t *behind, size_t n, const hipKernelNodeParams *p)
{
    char shape[64];
    std::snprintf(shape, sizeof shape, " %ux%u+%u", p->gridDim.x, p->blockDim.x, p->sharedMemBytes);
    return node(out, behind, n, values(p->func, p->kernelParams) + shape);
}
hipError_t hipGraphAddMemcpyNode1D(hipGraphNode_t *out, hipGraph_t, const hipGraphNode_t *behind, size_t n, void *, const void *, size_t bytes, hipMemcpyKind)
{
    return node(out, behind, n, "copy " + std::to_string(bytes));
}
hipError_t hipLaunchKernel(const void *f, dim3, dim3, void **a, size_t, hipStream_t) { return g_calls.push_back("run " + values(f, a)), hipSuccess; }
hipError_t hipMemcpyAsync(void *, const void *, size_t bytes, hipMemcpyKind, hipStream_t) { return g_calls.push_back("move " + std::to_string(bytes)), hipSuccess; }
}

int main()
{
    hipStream_t const st = reinterpret_cast<hipStream_t>(64), other = reinterpret_cast<hipStream_t>(128);
    float             y = 0.f;
    auto              step = [&](hipStream_t s) {
        Params p{3, 0.5};
        nvk::launch(one, dim3(2), dim3(64), 0, s, p, &y);
        p.n = 9; // (the value at the call is what counts)
        expect(nvk::copy_async(&y, &p, 4, hipMemcpyHostToDevice, s) == hipSuccess, "copy");
        nvk::launch(two, dim3(5), dim3(256), 1024, s, 7, nullptr, 2.f); // int, nullptr and float become the kernel's types
    };
    const std::vector<std::string> direct = {"run one(3,0.5,1)", "move 4", "run two(7,0,2)"};

    step(st);
    expect(g_calls == direct, "without a recording everything goes to the stream");

    hipGraphExec_t exec = nullptr;
    g_calls.clear();
    {
        nvk::Recording r(st);
        expect(nvk::Recording::of(st) == &r && !nvk::Recording::of(other), "recording of its stream");
        step(st);
        expect(g_calls == std::vector<std::string>({"node one(3,0.5,1) 2x64+0", "node copy 4", "node two(7,0,2) 5x256+1024"}), "three nodes");
        expect(g_behind == std::vector<std::intptr_t>({0, 1, 2}), "each behind the one before");
        g_calls.clear();
        step(other);
        expect(g_calls == direct, "another stream's launches run");
        g_calls.clear();
        std::thread([&] {
            expect(!nvk::Recording::of(st), "another thread records nothing");
            step(st);
        }).join();
        expect(g_calls == direct, "another thread's launches run");
        expect(r.finish(&exec) == hipSuccess && exec && g_calls.back() == "instantiate", "finished");
        g_calls.clear();
        step(st);
        expect(g_calls == direct && !nvk::Recording::of(st), "after the end everything goes to the stream");
    }
    expect(g_graphs == 0, "the graph is gone");

    g_calls.clear(), exec = nullptr, g_nodes = 0, g_fail_at = 1;
    {
        nvk::Recording r(st);
        step(st);
        expect(g_calls.size() == 1, "nothing is added behind a node that failed, and nothing runs");
        expect(r.finish(&exec) == hipErrorOutOfMemory && !exec, "the first error is the result");
    }
    expect(g_graphs == 0, "the graph is gone after an error");
    {
        nvk::Recording r(st); // given up
    }
    expect(g_graphs == 0 && !nvk::Recording::of(st), "a recording that is given up leaves nothing");
    return g_wrong ? 1 : 0;
}
