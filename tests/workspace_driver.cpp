// workspace_driver.cpp -- test infrastructure: the growing buffers of nvk_hip_util.h over an allocator that can be told to fail,
// without a device.  tests/test_workspace_growth.py builds and runs it; prints one line per mistake.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <set>

#include "nvk_hip_util.h"

static std::set<void *> g_live;
static long             g_mallocs_left = -1, g_memsets_left = -1, g_frees_left = -1; // calls until one fails; -1: none does
static bool             g_capturing = false;
static int              g_wrong = 0;

static bool fails(long &left) { return left >= 0 && left-- == 0; }

extern "C" {
hipError_t hipMalloc(void **p, size_t n)
{
    if (fails(g_mallocs_left))
        return hipErrorOutOfMemory;
    g_live.insert(*p = std::malloc(n));
    return hipSuccess;
}
hipError_t hipFree(void *p)
{
    if (fails(g_frees_left))
        return hipErrorUnknown;
    if (!g_live.erase(p))
        std::printf("freed what was not there\n"), g_wrong++;
    std::free(p);
    return hipSuccess;
}
hipError_t hipMemset(void *, int, size_t) { return fails(g_memsets_left) ? hipErrorUnknown : hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s)
{
    *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
const char *hipGetErrorString(hipError_t) { return "told to fail"; }
}
int nvk::fail(int code, const char *, ...) { return code; }

static void expect(bool ok, const char *what)
{
    if (!ok)
        std::printf("%s\n", what), g_wrong++;
}

// `grow` one of the two; whoever remembers the generation with the address has to learn that the address went
template <class T, class F> static void check(const char *name, F grow)
{
    hipStream_t const st = reinterpret_cast<hipStream_t>(8);
    T        *buf = nullptr;
    size_t    have = 0;
    long long generation = 0;
    std::printf("# %s\n", name);
    expect(grow(&buf, &have, &generation, (size_t)5000, st) == NVK_OK && buf && have >= 5000, "first allocation");
    T *const        held = buf;
    const long long seen = generation;
    expect(seen > 0, "the first allocation is counted");
    expect(grow(&buf, &have, &generation, (size_t)4000, st) == NVK_OK && buf == held && generation == seen, "a smaller one moves nothing");
    g_capturing = true;
    expect(grow(&buf, &have, &generation, (size_t)6000, st) == NVK_ERR_INVALID_ARG && buf == held && generation == seen && g_live.count(held),
           "refused under capture, the buffer as it was");
    g_capturing = false;

    g_frees_left = 0;
    expect(grow(&buf, &have, &generation, (size_t)6000, st) != NVK_OK && buf == held && g_live.count(held), "a buffer that cannot be freed stays");
    g_frees_left = -1;

    const long long before = generation;
    g_mallocs_left = 0;
    expect(grow(&buf, &have, &generation, (size_t)7000, st) == NVK_ERR_OOM, "no memory: says so");
    g_mallocs_left = -1;
    expect(g_live.count(held) || generation != before, "the old buffer is gone and the generation has not moved");
    expect(g_live.count(held) ? buf == held : !buf && have == 0, "what is remembered is what is there");
    expect(grow(&buf, &have, &generation, (size_t)100, st) == NVK_OK && buf && have >= 100, "works again when there is memory");

    const long long again = generation;
    T *const        second = buf;
    expect(grow(&buf, &have, &generation, have + 1, st) == NVK_OK && generation != again && second != nullptr, "a move is counted");
    (void)hipFree(buf);
    expect(g_live.empty(), "nothing is left");
}

int main()
{
    check<float>("workspace", [](float **b, size_t *h, long long *g, size_t n, hipStream_t st) { return nvk::grow_buffer(b, h, g, n, st, "test"); });
    auto counters = [](int **b, size_t *h, long long *g, size_t n, hipStream_t st) { return nvk::grow_counters(b, h, g, n, st, "test"); };
    check<int>("counters", counters);

    int      *buf = nullptr;
    size_t    have = 0;
    long long generation = 0;
    expect(counters(&buf, &have, &generation, 10, nullptr) == NVK_OK, "counters");
    const long long seen = generation;
    g_memsets_left = 0;
    expect(counters(&buf, &have, &generation, 9000, nullptr) != NVK_OK, "a failed fill is an error");
    expect(!buf && have == 0 && g_live.empty() && generation != seen, "counters that were not cleared are not kept, and the old ones' end is counted");
    return g_wrong ? 1 : 0;
}
