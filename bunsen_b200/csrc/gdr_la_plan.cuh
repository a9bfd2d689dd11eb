// Work lists of the decayed linear attention's chunked kernels: sequences, or
// segments of them, and the states between segments.
#pragma once

#include <atomic>

#include "gdr_la.cuh"

namespace gdr {

constexpr int kLaChunk = 128;  // segments are whole chunks of the largest kernel

// w^n for n below 2^24, 1 for n <= 0 (minus infinity included): the exponent's
// rounding error goes in as a factor, e^(p + d) = e^p (1 + d).
__device__ __forceinline__ float la_power(float g, int n) {
    if (n <= 0) return 1.f;
    const float p = g * n;
    if (p < -104.f) return 0.f;  // below the smallest f32
    const float e = expf(p);
    return fmaf(e, fmaf(g, static_cast<float>(n), -p), e);
}

// w^n in two parts, hi + lo.
__device__ __forceinline__ float2 la_power2(float g, int n) {
    const double f = exp(static_cast<double>(g) * n);
    const float hi = static_cast<float>(f);
    return make_float2(hi, static_cast<float>(f - hi));
}

// A list of work in device memory, made by la_plan: entries of positions and states,
// each for every head, the longest first. null: one job a CTA, its sequence and
// head by its index.
struct LaWork {
    int32_t count;    // entries
    int32_t next;     // the next job not handed out (entry x heads + head)
};
struct LaEntry {
    int32_t start, len, in, out;
};

// States by index: the call's own of sequence x >= 0, none (-1: zeros, or not
// wanted), or segment -2 - x's in the scratch. Null, or row `r` columns `c` apart.
struct LaState {
    const float* ptr;
    int64_t row, col;
};
__device__ __forceinline__ LaState la_state(const LaCore& p, int x, int h, const float* own,
                                            const float* scratch) {
    const int64_t size = static_cast<int64_t>(p.d_b) * p.d_c;
    const float* base = x >= 0 ? own : x == -1 ? nullptr : scratch;
    const bool turned = x >= 0 ? p.state_t : p.scratch_t;
    return {base != nullptr
                ? base + (static_cast<int64_t>(x >= 0 ? x : -2 - x) * p.heads + h) * size
                : nullptr,
            turned ? 1 : p.d_c, turned ? p.d_b : 1};
}

struct LaSplit {
    int32_t base, parts, seq, unused;  // segment r's state: slot base + r (r = 0: in place only)
};
struct LaPlan {
    LaWork main[2], states;  // (main: for either of two launches that share the lists)
    int32_t splits, seg_tokens;
};

// How a kernel's segments cost: in chunks of its main pass, a chunk of the pass
// that finds the segments' states, and what that pass and the scan cost at all.
struct LaSplitCost {
    bool may, must;  // sequences may go in segments; do even where it looks slower
    int forced;      // segment length in chunks, or 0
    float state_cost, fixed_cost;
};

// The lists of one call, in scratch from the library's pool (none when every job has a
// CTA of its own: plan is null).
struct LaLists {
    void* mem = nullptr;
    LaPlan* plan = nullptr;
    LaEntry *main = nullptr, *states = nullptr;
    LaSplit* splits = nullptr;
    float* slots = nullptr;
    bool split = false;  // some sequences may be in segments: run the states' pass
    int uses = 0;        // launches that have used them
};
// grid: CTAs of the persistent kernels; blocks: jobs of each (entry, head); shared: two
// launches will use the lists.
cudaError_t la_prepare(const LaCore& p, int grid, int blocks, LaSplitCost o, bool shared,
                       bool chained, LaLists& lists, cudaStream_t stream);
cudaError_t la_scan_states(const LaCore& p, const LaLists& lists, cudaStream_t stream);
cudaError_t la_release(const LaLists& lists, cudaStream_t stream);
int la_sm_count();
// A launch that may begin while the kernel before it in the stream, one of this call's, still
// runs: each of them lets the next one in at once and waits, before it reads or writes
// anything in global memory, for all of the one before (which has waited for its own).
// Saves the 2 us between two kernels.
template <typename... P, typename... A>
cudaError_t la_launch_next(void (*kernel)(P...), int grid, int threads, int smem,
                           cudaStream_t stream, A... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &a;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}
__device__ __forceinline__ void after_last_kernel() {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}
// A kernel's dynamic shared memory, allowed once a device (the call costs a launch's time).
template <typename K>
cudaError_t la_allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
// Two cores whose lists would be the same (jobs of 128 columns).
inline bool la_same_lists(const LaCore& x, const LaCore& y) {
    return (x.d_c + 127) / 128 == (y.d_c + 127) / 128;
}

}  // namespace gdr
