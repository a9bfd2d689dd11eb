// The work lists of gdr_la_plan.cuh.
#include <algorithm>
#include <cmath>

#include "gdr_la_plan.cuh"

namespace gdr {

cudaError_t library_pool(cudaMemPool_t* pool, bool create);

namespace {

constexpr int64_t kStateBudget = int64_t{2} << 30;  // scratch states of a call, bytes

// ---- sequences in segments ------------------------------------------------------
// A state passes through positions as S -> w^n S + B, B what they reach from zero.
// So a long sequence, which one CTA would walk alone, goes in segments of L chunks:
// one pass finds the B of every segment but the last (in the order of time), a
// scan the states before the segments, and the main pass runs all segments at once.
// The first pass reads b and c again: it is worth it where the longest
// sequences would bound the call. la_plan decides from the lengths, which only
// the device has.
constexpr int kPlanThreads = 1024, kBuckets = 1024;
constexpr float kLinkCost = 0.05f;  // of the scan, a link, in chunks of the main pass

// The longest time of a CTA, in chunks, with sequences in segments of L chunks: `sum`
// chunks altogether, the longest sequence `most` of them, `each` jobs a CTA for an
// entry; of the sequences above L, `again` chunks go through the states' pass, `whole`
// segments are whole (or nearly), one sequence has `parts` segments at most.
__host__ __device__ inline float split_time(const LaSplitCost& how, float each, int L, int sum,
                                            int most, int again, int whole, int parts) {
    // A pass takes the work's share of a CTA, and at least the most whole segments
    // that fall to one.
    const float longest = static_cast<float>(L < most ? L : most);
    float t = fmaxf(fmaxf(longest * ceilf(whole * each), sum * each * 1.03f + 1.f), longest);
    if (again > 0)
        t += how.state_cost * fmaxf(longest * ceilf(again * each / L), again * each * 1.03f) +
             how.fixed_cost + kLinkCost * parts;
    return t;
}
__host__ __device__ inline float whole_time(float each, int sum, int most) {
    return fmaxf(static_cast<float>(most), sum * each * 1.03f + 1.f);
}
// The lengths that are tried: 32, from l_min to the longest sequence.
__host__ __device__ inline int candidate_length(int i, int l_min, int most) {
    const float range = fmaxf(1.f, static_cast<float>(most) / l_min);
    const int L = static_cast<int>(l_min * powf(range, i / 31.f));
    return L > l_min ? L : l_min;
}
constexpr float kWorthIt = 0.97f;  // of the time without segments

// The block's sum (op 0) or maximum (op 1) of x.
__device__ int block_reduce(int x, bool maximum, int* ws) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 16; o > 0; o >>= 1) {
        const int y = __shfl_xor_sync(0xffffffffu, x, o);
        x = maximum ? max(x, y) : x + y;
    }
    __syncthreads();
    if (lane == 0) ws[warp] = x;
    __syncthreads();
    x = ws[lane];
    for (int o = 16; o > 0; o >>= 1) {
        const int y = __shfl_xor_sync(0xffffffffu, x, o);
        x = maximum ? max(x, y) : x + y;
    }
    return x;
}

// A state updated in place: the last segment writes what the first one reads, and may do
// so first. The scan copies it, to the slot of segment 0.
__device__ __forceinline__ bool in_place(const LaCore& p) {
    return p.state_in != nullptr && p.state_in == p.state_out;
}

// The work lists: every sequence of more than p.steps_most positions, or its segments, the
// longest first (by buckets of chunk counts), and the first pass's segments. seg_cap: state
// slots; 0: no splitting. forced: a given segment length.
__global__ void __launch_bounds__(kPlanThreads)
la_plan(const LaCore p, LaPlan* plan, LaEntry* main, LaEntry* states, LaSplit* splits, int32_t* base,
        int grid, int blocks, int l_min, int seg_cap, LaSplitCost how) {
    const int forced = how.forced;
    const bool must = how.must;
    __shared__ int ws[32], hist[kBuckets], slots, n_splits, n_states;
    __shared__ float cost[32];
    __shared__ int counts[kPlanThreads];  // the first sequences' chunks
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    after_last_kernel();
    auto chunks = [&](int s, int64_t& start, int64_t& len) {
        int64_t end;
        la_span(p, s, start, end);
        len = end - start;
        if (len <= p.steps_most) return -1;  // another launch's
        return static_cast<int>((len + kLaChunk - 1) / kLaChunk);
    };
    int64_t start, len;
    auto count = [&](int s) {
        if (s < kPlanThreads) return counts[s];
        int64_t x, y;
        return chunks(s, x, y);
    };
    int sum = 0, most = 0, listed = 0;
    for (int s = tid; s < p.n_seqs; s += kPlanThreads) {
        const int c = chunks(s, start, len);
        if (s < kPlanThreads) counts[s] = c;
        if (c < 0) continue;
        ++listed;
        sum += c;
        most = max(most, c);
    }
    listed = block_reduce(listed, false, ws);
    sum = block_reduce(sum, false, ws);
    most = block_reduce(most, true, ws);
    // Candidate lengths from l_min to the longest sequence, one a warp.
    const float each = static_cast<float>(p.heads) * blocks / grid;
    auto candidate = [&](int i) { return forced > 0 ? forced : candidate_length(i, l_min, most); };
    {
        const int L = candidate(warp);
        int again = 0, parts_most = 0, segs = 0, whole = 0;  // whole: segments of L chunks
        for (int s = lane; s < p.n_seqs; s += 32) {
            const int c = count(s);
            if (c > L) {
                const int parts = (c + L - 1) / L;
                again += (parts - 1) * L;
                segs += parts;
                whole += (c + L / 3) / L;  // (a part of two thirds too)
                parts_most = max(parts_most, parts);
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            again += __shfl_xor_sync(0xffffffffu, again, o);
            segs += __shfl_xor_sync(0xffffffffu, segs, o);
            whole += __shfl_xor_sync(0xffffffffu, whole, o);
            parts_most = max(parts_most, __shfl_xor_sync(0xffffffffu, parts_most, o));
        }
        float t = split_time(how, each, L, sum, most, again, whole, parts_most);
        if (segs > seg_cap) t = INFINITY;
        if (lane == 0) cost[warp] = t;
    }
    __syncthreads();
    int L = most > 0 ? most : 1;  // not split
    if (seg_cap > 0) {
        float t = cost[lane];
        int best = lane;
        for (int o = 16; o > 0; o >>= 1) {
            const float u = __shfl_xor_sync(0xffffffffu, t, o);
            const int other = __shfl_xor_sync(0xffffffffu, best, o);
            if (u < t || (u == t && other < best)) {
                t = u;
                best = other;
            }
        }
        if (t < (must || forced > 0 ? INFINITY : kWorthIt * whole_time(each, sum, most)))
            L = candidate(best);
    }
    const int shift = max(0, 32 - __clz(min(L, most)) - 10);  // bucket: chunks >> shift
    for (int i = tid; i < kBuckets; i += kPlanThreads) hist[i] = 0;
    if (tid == 0) slots = n_splits = n_states = 0;
    __syncthreads();
    auto bucket = [&](int c) { return kBuckets - 1 - (c >> shift); };  // longest first
    for (int s = tid; s < p.n_seqs; s += kPlanThreads) {
        const int c = count(s);
        if (c < 0) continue;
        int parts = c > L ? (c + L - 1) / L : 1, at = 0;
        if (parts > 1) at = atomicAdd(&slots, parts);
        base[s] = at;
        if (parts > 1) {
            atomicAdd(&hist[bucket(L)], parts - 1);
            atomicAdd(&hist[bucket(c - (parts - 1) * L)], 1);
        } else {
            atomicAdd(&hist[bucket(c)], 1);
        }
    }
    __syncthreads();
    // Exclusive scan of the buckets (as many as threads).
    int x = hist[tid];
    const int mine = x;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) ws[warp] = x;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < warp; ++i) before += ws[i];
    __syncthreads();
    hist[tid] = before + x - mine;
    __syncthreads();
    for (int s = tid; s < p.n_seqs; s += kPlanThreads) {
        const int c = count(s);
        if (c < 0 || c > L) continue;
        chunks(s, start, len);
        main[atomicAdd(&hist[bucket(c)], 1)] = {static_cast<int32_t>(start),
                                                static_cast<int32_t>(len), s, s};
    }
    // Sequences in segments, a warp each.
    for (int s = warp; s < p.n_seqs; s += kPlanThreads / 32) {
        const int c = count(s);
        if (c <= L) continue;
        chunks(s, start, len);
        const int parts = (c + L - 1) / L, at = base[s];
        if (lane == 0) splits[atomicAdd(&n_splits, 1)] = {at, parts, s, 0};
        for (int r = lane; r < parts; r += 32) {  // in the order of time
            const int part = p.reverse ? parts - 1 - r : r;
            const int from = part * L, n = min(L, c - from);
            const int32_t t0 = static_cast<int32_t>(start) + from * kLaChunk;
            const int32_t tokens = min(n * kLaChunk, static_cast<int32_t>(len) - from * kLaChunk);
            main[atomicAdd(&hist[bucket(n)], 1)] = {t0, tokens,
                                                    r == 0 && !in_place(p) ? s : -2 - (at + r),
                                                    r == parts - 1 ? s : -1};
            if (r < parts - 1)
                states[atomicAdd(&n_states, 1)] = {t0, tokens, -1, -2 - (at + r + 1)};
        }
    }
    __syncthreads();
    if (tid == 0) {
        plan->main[0] = plan->main[1] = {listed + slots - n_splits, grid};
        plan->states = {n_states, grid};
        plan->splits = n_splits;
        plan->seg_tokens = L * kLaChunk;
    }
}

// S_{r+1} = w^(tokens of r) S_r + B_r, in place: slot base + r + 1 holds B_r. kVec
// elements of a row a thread, the links' loads issued ahead of the products.
template <int kVec>
__global__ void __launch_bounds__(256)
la_scan(const LaCore p, const LaPlan* plan, const LaSplit* splits, float* scratch) {
    after_last_kernel();
    const int size = p.d_b * p.d_c, tiles = (size + 256 * kVec - 1) / (256 * kVec);
    const int64_t jobs = static_cast<int64_t>(plan->splits) * p.heads * tiles;
    for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int tile = static_cast<int>(job % tiles);
        const int h = static_cast<int>(job / tiles % p.heads);
        const LaSplit sp = splits[job / tiles / p.heads];
        const int e = (tile * 256 + threadIdx.x) * kVec;
        if (e >= size) continue;
        float x[kVec];
        const LaState in = la_state(p, sp.seq, h, p.state_in, scratch);
#pragma unroll
        for (int v = 0; v < kVec; ++v)
            x[v] = in.ptr != nullptr ? in.ptr[(e / p.d_c) * in.row + (e % p.d_c + v) * in.col] : 0.f;
        int64_t start, end;
        la_span(p, sp.seq, start, end);
        const float g = p.log_decay[h];
        const int last = static_cast<int>(end - start) - (sp.parts - 1) * plan->seg_tokens;
        const float w = la_power(g, plan->seg_tokens);
        const int64_t step = static_cast<int64_t>(p.heads) * size;
        float* slot = scratch + (static_cast<int64_t>(sp.base) * p.heads + h) * size + e;
        if (in_place(p)) {
#pragma unroll
            for (int v = 0; v < kVec; ++v) slot[v] = x[v];
        }
        slot += step;
#pragma unroll 4
        for (int r = 0; r < sp.parts - 1; ++r, slot += step) {
            const float f = p.reverse && r == 0 ? la_power(g, last) : w;
            if constexpr (kVec == 4) {
                const float4 b = *reinterpret_cast<const float4*>(slot);
                x[0] = fmaf(f, x[0], b.x), x[1] = fmaf(f, x[1], b.y);
                x[2] = fmaf(f, x[2], b.z), x[3] = fmaf(f, x[3], b.w);
                *reinterpret_cast<float4*>(slot) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
                x[0] = fmaf(f, x[0], *slot);
                *slot = x[0];
            }
        }
    }
}

}  // namespace

int la_sm_count() {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

cudaError_t la_prepare(const LaCore& p, int grid, int blocks, LaSplitCost o, bool shared,
                       bool chained, LaLists& out, cudaStream_t stream) {
    if (shared) {  // two passes over the segments for one that finds their states
        o.state_cost *= 0.5f;
        o.fixed_cost *= 0.5f;
    }
    // What splitting could bring: no sequence is longer than `longest` chunks, and the
    // work fills every CTA for `each` chunks or fewer.
    const int64_t tokens = la_tokens(p);
    const int64_t longest = ((p.cu_seqlens ? tokens : p.seq_len) + kLaChunk - 1) / kLaChunk;
    const int64_t most = p.cu_seqlens ? tokens / kLaChunk + p.n_seqs : longest * p.n_seqs;
    const double each = static_cast<double>(most) * p.heads * blocks / grid;
    const int l_min = o.forced > 0 ? o.forced : std::max(2, static_cast<int>(each / 4));
    bool split = o.may && longest > l_min &&
                 (o.must || longest > 2 * l_min + static_cast<int>(o.fixed_cost));
    if (split && !o.must && o.forced == 0 && p.cu_seqlens == nullptr) {
        // Dense lengths are known here.
        const int c = static_cast<int>(longest), n = p.n_seqs;
        const float per = static_cast<float>(p.heads) * blocks / grid;
        float best = kWorthIt * whole_time(per, n * c, c);
        split = false;
        for (int i = 0; i < 32 && !split; ++i) {
            const int L = candidate_length(i, l_min, c);
            if (L >= c) continue;
            const int parts = (c + L - 1) / L;
            split = split_time(o, per, L, n * c, c, n * (parts - 1) * L, n * ((c + L / 3) / L), parts) < best;
        }
    }
    if (!split && p.steps_most < 0 && static_cast<int64_t>(p.n_seqs) * p.heads * blocks <= grid)
        return cudaSuccess;
    const size_t size = sizeof(float) * p.heads * p.d_b * p.d_c;
    // A split sequence of c > L chunks has ceil(c / L) < 2 c / L segments.
    const int64_t cap = split ? std::min<int64_t>(2 * most / l_min + 2, kStateBudget / size) : 0;
    auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
    const size_t o_main = up(sizeof(LaPlan)),
                 o_states = o_main + up(sizeof(LaEntry) * (p.n_seqs + cap)),
                 o_splits = o_states + up(sizeof(LaEntry) * cap),
                 o_base = o_splits + up(sizeof(LaSplit) * (cap / 2 + 1)),
                 o_slots = o_base + up(sizeof(int32_t) * p.n_seqs), bytes = o_slots + cap * size;
    cudaMemPool_t pool;
    cudaError_t e = library_pool(&pool, true);
    if (e == cudaSuccess) e = cudaMallocFromPoolAsync(&out.mem, bytes, pool, stream);
    if (e != cudaSuccess) return e;
    uint8_t* at = static_cast<uint8_t*>(out.mem);
    out.plan = reinterpret_cast<LaPlan*>(at);
    out.main = reinterpret_cast<LaEntry*>(at + o_main);
    out.states = reinterpret_cast<LaEntry*>(at + o_states);
    out.splits = reinterpret_cast<LaSplit*>(at + o_splits);
    out.slots = reinterpret_cast<float*>(at + o_slots);
    out.split = split;
    int32_t* base = reinterpret_cast<int32_t*>(at + o_base);
    if (chained)
        return la_launch_next(la_plan, 1, kPlanThreads, 0, stream, p, out.plan, out.main, out.states,
                              out.splits, base, grid, blocks, l_min, static_cast<int>(cap), o);
    la_plan<<<1, kPlanThreads, 0, stream>>>(p, out.plan, out.main, out.states, out.splits, base, grid,
                                            blocks, l_min, static_cast<int>(cap), o);
    return cudaGetLastError();
}

cudaError_t la_scan_states(const LaCore& p, const LaLists& lists, cudaStream_t stream) {
    return la_launch_next(p.d_c % 4 == 0 ? la_scan<4> : la_scan<1>, 4 * la_sm_count(), 256, 0, stream,
                          p, lists.plan, lists.splits, lists.slots);
}

cudaError_t la_release(const LaLists& lists, cudaStream_t stream) {
    return lists.mem != nullptr ? cudaFreeAsync(lists.mem, stream) : cudaSuccess;
}

}  // namespace gdr
