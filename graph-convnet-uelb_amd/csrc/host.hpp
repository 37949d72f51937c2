// Host-side helpers of the translation units behind the C ABI: the error message of the calling thread, the optional
// per-kernel timing and the launch macros.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_ext.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

namespace gcn_host {

inline thread_local char g_err[512] = "";

// Measurement overrides (grid sizes, chunk lengths, probes) exist only in builds made with -DGCN_TUNING
// (tools/build_tuning_lib.sh); the product library reads no environment variable.
#ifdef GCN_TUNING
inline const char* tune_env(const char* name) { return getenv(name); }
#else
inline const char* tune_env(const char*) { return nullptr; }
#endif

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

// ---- optional per-kernel timing with HIP events (used by bench.py; off by default) -----------------
// gcn_prof_begin(substr) arms it: every later launch whose name contains substr is bracketed by two
// events on its own stream.  gcn_prof_end() synchronises those events and returns the summed time.
struct ProfEvents {
    hipEvent_t e0, e1, e2;      // e0, e1: an empty bracket recorded right before the launch; e1, e2: the launch
};
struct ProfState {
    bool on = false;
    char match[64] = "";
    std::vector<ProfEvents> ev;
    hipEvent_t pending = nullptr;
};
inline ProfState g_prof;

inline void prof_pre(const char* name, hipStream_t st) {
    if (!g_prof.on || strstr(name, g_prof.match) == nullptr) return;
    ProfEvents p;
    if (hipEventCreate(&p.e0) != hipSuccess || hipEventCreate(&p.e1) != hipSuccess || hipEventCreate(&p.e2) != hipSuccess) return;
    (void)hipEventRecord(p.e0, st);
    (void)hipEventRecord(p.e1, st);
    g_prof.ev.push_back(p);
    g_prof.pending = p.e2;
}
// For launches made with hipExtLaunchKernelGGL: the two events receive the kernel's own begin and end time
// stamps (what a kernel trace reports), so no bracket cost is involved.  e0 == nullptr marks such an entry.
inline void prof_ext(const char* name, hipEvent_t* start, hipEvent_t* stop) {
    *start = nullptr; *stop = nullptr;
    if (!g_prof.on || strstr(name, g_prof.match) == nullptr) return;
    ProfEvents p;
    p.e0 = nullptr;
    if (hipEventCreate(&p.e1) != hipSuccess || hipEventCreate(&p.e2) != hipSuccess) return;
    g_prof.ev.push_back(p);
    *start = p.e1; *stop = p.e2;
}
inline void prof_post(hipStream_t st) {
    if (g_prof.pending) { (void)hipEventRecord(g_prof.pending, st); g_prof.pending = nullptr; }
}

#define GCN_PROF_PRE(name) prof_pre(name, (hipStream_t)GCN_STREAM)
#define GCN_CHECK_LAUNCH(name)                                                                   \
    do {                                                                                         \
        prof_post((hipStream_t)GCN_STREAM);                                                      \
        hipError_t e_ = hipGetLastError();                                                       \
        if (e_ != hipSuccess) return fail(-3, "launch of %s failed: %s", name, hipGetErrorString(e_)); \
    } while (0)

#define GCN_STREAM st

// launch of one of the main kernels, timed by its own time stamps when the profiler is armed for its name
#define GCN_LAUNCH_TIMED_LDS(name, kern, grid, block, lds, ...)                                   \
    do {                                                                                         \
        hipEvent_t es_ = nullptr, ee_ = nullptr;                                                 \
        prof_ext(name, &es_, &ee_);                                                              \
        hipExtLaunchKernelGGL(kern, dim3(grid), dim3(block), lds, (hipStream_t)GCN_STREAM, es_, ee_, 0, __VA_ARGS__); \
        hipError_t e_ = hipGetLastError();                                                       \
        if (e_ != hipSuccess) return fail(-3, "launch of %s failed: %s", name, hipGetErrorString(e_)); \
    } while (0)
#define GCN_LAUNCH_TIMED(name, kern, grid, block, ...) GCN_LAUNCH_TIMED_LDS(name, kern, grid, block, 0, __VA_ARGS__)

}  // namespace gcn_host

using namespace gcn_host;
