// What the host sides of the entry points share: the message of the last error, the launch call, settings and addresses
// kept per context, argument checks.
#pragma once
#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <utility>

#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/kf_b200.h"

namespace kf {
namespace host {

inline thread_local char g_err[512] = "";

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

// `dependent`: launch as a programmatic dependent of the kernel before it in the stream (the grid may start while
// that kernel still runs and must order its reads of that kernel's output with griddepcontrol.wait).
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel_ex(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool dependent,
                             Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    if (dependent) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
    return launch_kernel_ex(kern, grid, block, smem, st, false, std::forward<Args>(args)...);
}

// Identity of the calling thread's CUDA context: never used again in a process, and a new one after a device reset.
// 0: unknown (no context yet), to be treated as one never seen.
inline unsigned long long context_id() {
    using Fn = CUresult (*)(CUcontext, unsigned long long*);
    static std::atomic<Fn> cached{nullptr};
    Fn fn = cached.load(std::memory_order_acquire);
    if (fn == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuCtxGetId", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return 0;
        fn = reinterpret_cast<Fn>(p);
        cached.store(fn, std::memory_order_release);
    }
    unsigned long long id = 0;
    return fn(nullptr, &id) == CUDA_SUCCESS ? id : 0;
}

// Let a kernel use `bytes` of dynamic shared memory.  The setting belongs to the context: made at the kernel's first
// launch in each (0.6 us).
template <auto KERN> cudaError_t allow_smem(int bytes) {
    static std::atomic<unsigned long long> done[64];  // contexts by id (two threads may both set it)
    const unsigned long long id = context_id();
    if (id != 0 && done[id % 64].load(std::memory_order_acquire) == id) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done[id % 64].store(id, std::memory_order_release);
    return e;
}

// Device address, in the current context, of a variable of the library image; looked up once per context.  And the context's
// number.
struct SymbolCache {
    std::atomic_flag busy = ATOMIC_FLAG_INIT;
    unsigned long long id[64];
    void* at[64];
};
inline cudaError_t symbol_address(SymbolCache& c, const void* symbol, void** out,
                                  unsigned long long* context = nullptr) {
    unsigned long long id = context_id();
    const int i = static_cast<int>(id % 64);
    auto locked = [&](auto&& body) {
        while (c.busy.test_and_set(std::memory_order_acquire)) {}
        body();
        c.busy.clear(std::memory_order_release);
    };
    void* p = nullptr;
    locked([&] { if (id != 0 && c.id[i] == id) p = c.at[i]; });
    if (p == nullptr) {
        cudaError_t e = cudaGetSymbolAddress(&p, symbol);
        if (e != cudaSuccess) return e;
        id = context_id();  // (the call may have made the context)
        if (id != 0) locked([&] { c.id[id % 64] = id; c.at[id % 64] = p; });
    }
    *out = p;
    if (context != nullptr) *context = id;
    return cudaSuccess;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Element stride of a dimension of extent n: a multiple of 8 (16 bytes), positive unless the dimension has a
// single entry.  A zero stride over n > 1 entries (an expanded / broadcast view) is refused: the TMA maps
// describe distinct rows and would walk past the allocation.
inline bool stride_ok(int64_t s, int64_t n) { return (s % 8) == 0 && (s > 0 || (s == 0 && n == 1)); }

inline int check_device() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(KF_ECUDA, "cudaGetDevice failed");
    static int cached_major[64];
    if (dev < 0 || dev >= 64) return fail(KF_ECUDA, "device ordinal %d out of range", dev);
    if (cached_major[dev] == 0) {
        int major = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
            return fail(KF_ECUDA, "cannot query the compute capability");
        cached_major[dev] = major;
    }
    if (cached_major[dev] != 10) return fail(KF_ENOSUP, "this library is built for sm_100a (compute capability 10.x)");
    return KF_OK;
}

inline int sm_count() {
    static int cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (cached[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cached[dev] = n;
    }
    return cached[dev];
}

// Slots of a table in device memory that captured launches own: a captured launch runs again with every replay of its
// graph, next to whatever else is running, so it gets a slot for itself, which the graph, its clones and its executable
// forms own together and give back when the last of them is destroyed.  (Plain data: graphs may outlive static objects.)
template <int N> struct GraphSlots {
    std::atomic_flag busy = ATOMIC_FLAG_INIT;
    int back[N], n_back, n_taken;  // slots given back; slots taken at least once
    int take() {                   // -1: none left
        while (busy.test_and_set(std::memory_order_acquire)) {}
        const int s = n_back > 0 ? back[--n_back] : n_taken < N ? n_taken++ : -1;
        busy.clear(std::memory_order_release);
        return s;
    }
    void give_back(int slot) {
        while (busy.test_and_set(std::memory_order_acquire)) {}
        back[n_back++] = slot;
        busy.clear(std::memory_order_release);
    }
};

// Slots that launches into streams use: one for each stream, as launches of one stream never run at the same time, while those
// of two may, however far apart they were enqueued (one may wait for an event while thousands go through the other).  A stream is
// known by its context's and its own number, which are never used again in a process.  (Plain data.)
template <int N> struct StreamSlots {
    std::atomic_flag busy = ATOMIC_FLAG_INIT;
    unsigned long long context[N], stream[N];  // context 0: nobody's slot
    int of(unsigned long long ctx, unsigned long long id) {  // -1: every slot belongs to another stream
        const unsigned int first = static_cast<unsigned int>((ctx * 31 + id) * 2654435761u >> 7) % N;
        while (busy.test_and_set(std::memory_order_acquire)) {}
        int at = -1;
        for (int i = 0; i < N && at < 0; ++i) {
            const int k = static_cast<int>((first + i) % N);
            if (context[k] == 0) {
                context[k] = ctx;
                stream[k] = id;
            }
            if (context[k] == ctx && stream[k] == id) at = k;
        }
        busy.clear(std::memory_order_release);
        return at;
    }
};

// The slot of the launch about to be made into `st` in context `ctx`: its stream's, or, while the stream is being captured, one of GRAPH's behind
// all of those; -1 when every slot of the kind is taken, or the stream cannot be told from others.
template <auto& STREAM, auto& GRAPH> int launch_slot(cudaStream_t st, unsigned long long ctx, int* out) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaGraph_t graph = nullptr;
    if (cudaStreamGetCaptureInfo_v2(st, &capture, nullptr, &graph, nullptr, nullptr) != cudaSuccess) {
        cudaGetLastError();  // (the legacy stream next to a capture elsewhere: the launch itself reports that)
        capture = cudaStreamCaptureStatusNone;
    }
    *out = -1;
    if (capture != cudaStreamCaptureStatusActive) {
        unsigned long long id = 0;
        if (ctx == 0) return KF_OK;
        if (cudaStreamGetId(st, &id) != cudaSuccess) {
            cudaGetLastError();
            return KF_OK;
        }
        *out = STREAM.of(ctx, id);
        return KF_OK;
    }
    const int slot = GRAPH.take();
    if (slot < 0) return KF_OK;
    cudaUserObject_t owner = nullptr;
    cudaError_t e = cudaUserObjectCreate(&owner, reinterpret_cast<void*>(static_cast<intptr_t>(slot)),
                                         [](void* tag) { GRAPH.give_back(static_cast<int>(reinterpret_cast<intptr_t>(tag))); }, 1,
                                         cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
        GRAPH.give_back(slot);
        return fail(KF_ECUDA, "cudaUserObjectCreate failed: %s", cudaGetErrorString(e));
    }
    e = cudaGraphRetainUserObject(graph, owner, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
        cudaUserObjectRelease(owner, 1);  // (gives the slot back)
        return fail(KF_ECUDA, "cudaGraphRetainUserObject failed: %s", cudaGetErrorString(e));
    }
    *out = static_cast<int>(sizeof(STREAM.stream) / sizeof(STREAM.stream[0])) + slot;
    return KF_OK;
}

}  // namespace host
}  // namespace kf
