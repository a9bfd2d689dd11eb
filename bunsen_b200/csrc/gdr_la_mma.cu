// The decayed linear attention core (gdr_la.cuh) in chunks at f32 accuracy: f32 and
// f16 operands, and bf16 ones of widths the tensor-memory kernel does not take;
// d_b up to 128, d_c up to 256.
//
// The same sums as gdr_la_tc.cu in chunks of C = 64 positions:
//   out_i = tau [ w^{i+1} a_i . S + sum_{j<=i} sigma w^{i-j} (a_i.b_j) c_j ]
//   S'    = w^C S + sum_j sigma w^{C-1-j} b_j c_j^T
// (backward in time their mirror image). Every product runs on the tensor cores as
// tf32 mma.sync in parts: x = hi + lo, each 11 bits, hi hi + hi lo + lo hi leaves
// 2^-22 of a product; 16-bit operands are one part exactly, so a b is one
// product for them, the others two. mma.sync at tf32 measures 488 products a
// cycle and SM, three of them 163 f32 ones, against 117 of FFMA, whose operands
// cost more loads besides.
//
// A CTA of eight warps takes one (sequence or segment, head) and 64 columns of the
// state, which are independent of the others (a b is computed again for each
// 64 columns: a sixth of the work). The state stays in registers as the update's
// accumulators, a copy of it in shared memory as the inter product's operand.
// Per chunk three barrier-separated stages: scores (into P), the outputs, the
// update. Bound by mma.sync: 11 300 cycles a chunk and 64 columns at f32.
#include <type_traits>

#include "gdr_f32x2.cuh"
#include "gdr_la.cuh"
#include "gdr_la_plan.cuh"

namespace gdr {

namespace {

constexpr int kC = 64, kCols = 64;
// Rows padded so that a fragment's 32 lanes fall on different banks.
constexpr int kLdC = kCols + 8, kLdP = kC + 4;

template <int kDb>
constexpr int smem_floats() {
    return 2 * kC * (kDb + 4) + kC * kLdC + kDb * kLdC + kC * kLdP + 2 * (kC + 8);
}

// x in one or two parts of 11 bits (tf32), the first rounded to the nearest by
// carrying into the bits that stay, the second cut: what is left out is below 2^-22 of
// x, of either sign. (cvt.rna.tf32 is two instructions more a part.)
template <int kParts>
struct Parts {
    uint32_t v[kParts];
};
template <int kParts>
__device__ __forceinline__ Parts<kParts> parts(float x) {
    Parts<kParts> p;
    if constexpr (kParts == 1) {
        p.v[0] = __float_as_uint(x);
    } else {
        p.v[0] = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
        p.v[1] = __float_as_uint(x - __uint_as_float(p.v[0])) & 0xffffe000u;
    }
    return p;
}

// c (+)= A B of one 16 x 8 x 8 step.
template <bool kAdd>
__device__ __forceinline__ void mma_step(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kAdd)
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3},"
            " {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3},"
            " {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// sum += A B, A and B in parts, the smallest products first. The step's own sum
// starts at zero and is added by FADD: the tensor cores' adds round towards zero,
// which over 48 of them in one accumulator made an error of 2.2e-6 (against 2e-7 so).
template <int kA, int kB>
__device__ __forceinline__ void mma(float (&sum)[4], const Parts<kA> (&a)[4],
                                    const Parts<kB> (&b)[2]) {
    float c[4];
    auto with = [&](int i, int j, auto add) {
        mma_step<decltype(add)::value>(c, a[0].v[i], a[1].v[i], a[2].v[i], a[3].v[i], b[0].v[j],
                                       b[1].v[j]);
    };
    if constexpr (kA == 2) with(1, 0, std::false_type{});
    if constexpr (kB == 2) with(0, 1, std::bool_constant<kA == 2>{});
    with(0, 0, std::bool_constant<kA == 2 || kB == 2>{});
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        unpair(add2(pair(sum[i], sum[i + 1]), pair(c[i], c[i + 1])), sum[i], sum[i + 1]);
    }
}

// A thread's share of kC rows x kWidth columns from [T, heads, d], rows [row0, row0 +
// rows) and columns from col0, zeros past the rows and past d: fetched into
// registers ahead of the chunk, four elements at once, and put into a tile.
template <typename T, int kWidth, int kThreads>
struct Share {
    static constexpr int kN = kC * kWidth / 4 / kThreads;
    using Raw = std::conditional_t<sizeof(T) == 4, float4, uint2>;
    Raw v[kN];

    __device__ __forceinline__ void fetch(const void* base, int64_t row0, int rows, int heads, int h,
                                          int d, int col0, bool vec) {
        const int64_t step = static_cast<int64_t>(heads) * d;
        const int c = threadIdx.x % (kWidth / 4) * 4, r0 = threadIdx.x / (kWidth / 4);
        const T* src = static_cast<const T*>(base) + (row0 * heads + h) * d + col0 + c;
#pragma unroll
        for (int x = 0; x < kN; ++x) {
            const int r = r0 + x * (kThreads * 4 / kWidth);
            Raw f{};
            if (r < rows && col0 + c < d) {
                const T* at = src + r * step;
                if (vec) {  // (d is a multiple of 4 then)
                    f = *reinterpret_cast<const Raw*>(at);
                } else {
                    T* e = reinterpret_cast<T*>(&f);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col0 + c + j < d) e[j] = at[j];
                }
            }
            v[x] = f;
        }
    }
    template <int kLd>
    __device__ __forceinline__ void put(float* dst) const {
        const int c = threadIdx.x % (kWidth / 4) * 4, r0 = threadIdx.x / (kWidth / 4);
#pragma unroll
        for (int x = 0; x < kN; ++x) {
            const T* e = reinterpret_cast<const T*>(&v[x]);
            *reinterpret_cast<float4*>(dst + (r0 + x * (kThreads * 4 / kWidth)) * kLd + c) =
                make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
        }
    }
};

template <int kDb>
constexpr int threads_of() {
    return kDb == 64 ? 256 : 512;
}

template <typename T, int kDb, bool kRev>
__global__ void __launch_bounds__(threads_of<kDb>(), kDb == 64 ? 2 : 1)
la_mma(const LaCore p, LaWork* work, const LaEntry* entries, float* scratch, bool state_only,
       bool vec_ab, bool vec_c) {
    constexpr int kThreads = threads_of<kDb>();
    constexpr int kIn = sizeof(T) == 4 ? 2 : 1;  // parts of an input
    constexpr int kLdA = kDb + 4;
    constexpr int kOn = kDb == 64 ? 4 : 2;  // 8-column tiles of scores and outputs a warp holds
    constexpr int kUn = 4;                  // and of the state
    extern __shared__ __align__(16) float smem[];
    float* as = smem;              // [kC][kLdA]
    float* bs = as + kC * kLdA;    // [kC][kLdA]
    float* cs = bs + kC * kLdA;    // [kC][kLdC]
    float* ss = cs + kC * kLdC;    // [kDb][kLdC]
    float* ps = ss + kDb * kLdC;   // [kC][kLdP]
    float* pw = ps + kC * kLdP;    // w^0 .. w^kC
    __shared__ int next_job;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    // Scores, outputs: 16 rows from m0 x 8 kOn columns from c0. Warps with the same
    // warp % 4 share a scheduler: each gets every row block once (two of them, the first
    // with the last, in the narrow form), so that the mask leaves all four the same work.
    const int q = warp >> 2;
    const int turn = kDb == 64 ? (q == 0 ? warp & 3 : 3 - (warp & 3))
                               : ((warp & 3) + (0x1203 >> 4 * q)) & 3;
    const int m0 = 16 * (kRev ? 3 - turn : turn);
    const int c0 = 8 * kOn * (kRev ? (kDb == 64 ? 1 : 3) - q : q);
    // The update: 16 rows, kUn x 8 columns.
    const int um0 = 16 * (warp % (kDb / 16)), un0 = 32 * (warp / (kDb / 16));
    const int blocks = (p.d_c + kCols - 1) / kCols;
    const int jobs = (work != nullptr ? work->count : p.n_seqs) * p.heads * blocks;
    int id = blockIdx.x;
    while (id < jobs) {
        const int n0 = id % blocks * kCols, h = id / blocks % p.heads, e = id / blocks / p.heads;
        LaEntry it;
        if (work != nullptr) {
            it = entries[e];
        } else {
            int64_t start, end;
            la_span(p, e, start, end);
            it = {static_cast<int32_t>(start), static_cast<int32_t>(end - start), e, e};
        }
        const int nch = (it.len + kC - 1) / kC;
        Share<T, kDb, kThreads> va, vb;
        Share<T, kCols, kThreads> vc;
        auto fetch = [&](int c) {
            const int x0 = kRev ? nch - 1 - c : c;
            const int64_t row = static_cast<int64_t>(it.start) + x0 * kC;
            const int len = min(kC, it.len - x0 * kC);
            if (!state_only)
                va.fetch(p.a, row, len, p.heads_a, h / (p.heads / p.heads_a), p.d_b, 0, vec_ab);
            vb.fetch(p.b, row, len, p.heads_b, h / (p.heads / p.heads_b), p.d_b, 0, vec_ab);
            vc.fetch(p.c, row, len, p.heads_c, h / (p.heads / p.heads_c), p.d_c, n0, vec_c);
        };
        const float decay = p.log_decay[h];
        __syncthreads();  // the last job's last reads
        if (tid <= kC) pw[tid] = la_power(decay, tid);
        float s[kUn][4];  // the state: rows um0 + g (+ 8), columns n0 + un0 + 8 n + 2 t (+ 1)
        const LaState in = la_state(p, it.in, h, p.state_in, scratch);
#pragma unroll
        for (int n = 0; n < kUn; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = um0 + g + 8 * (x >> 1), col = n0 + un0 + 8 * n + 2 * t + (x & 1);
                s[n][x] = in.ptr != nullptr && row < p.d_b && col < p.d_c
                              ? in.ptr[row * in.row + col * in.col]
                              : 0.f;
            }
        float2 f{1.f, 0.f};  // w^len of a chunk, in two parts
        int known = 0;
        for (int c = -1; c < nch; ++c) {  // (before the first chunk, only its fetch)
            const int x0 = kRev ? nch - 1 - c : c;
            const int64_t row = static_cast<int64_t>(it.start) + x0 * kC;
            const int len = min(kC, it.len - x0 * kC);
            float o[kOn][4] = {};
            if (c >= 0) {
                if (len != known) {
                    f = la_power2(decay, len);
                    known = len;
                }
                vb.template put<kLdA>(bs);
                vc.template put<kLdC>(cs);
                if (!state_only) {
                    va.template put<kLdA>(as);
    #pragma unroll
                    for (int n = 0; n < kUn; ++n) {
                        float* dst = ss + (um0 + g) * kLdC + un0 + 8 * n + 2 * t;
                        *reinterpret_cast<float2*>(dst) = make_float2(s[n][0], s[n][1]);
                        *reinterpret_cast<float2*>(dst + 8 * kLdC) = make_float2(s[n][2], s[n][3]);
                    }
                }
                __syncthreads();
                if (!state_only) {
                    // Scores, where the mask leaves any, and a . S.
                    float acc[kOn][4] = {};
                    const bool some = kRev ? c0 + 8 * kOn - 1 >= m0 : c0 <= m0 + 15;
    #pragma unroll 2
                    for (int k = 0; k < kDb; k += 8) {
                        const float* ap = as + (m0 + g) * kLdA + k + t;
                        const Parts<kIn> a[4] = {parts<kIn>(ap[0]), parts<kIn>(ap[8 * kLdA]),
                                                 parts<kIn>(ap[4]), parts<kIn>(ap[8 * kLdA + 4])};
    #pragma unroll
                        for (int n = 0; n < kOn; ++n) {
                            const float* bp = ss + (k + t) * kLdC + c0 + 8 * n + g;
                            const Parts<2> b[2] = {parts<2>(bp[0]), parts<2>(bp[4 * kLdC])};
                            mma(o[n], a, b);
                        }
                        if (some)
    #pragma unroll
                            for (int n = 0; n < kOn; ++n) {
                                const float* bp = bs + (c0 + 8 * n + g) * kLdA + k + t;
                                const Parts<kIn> b[2] = {parts<kIn>(bp[0]), parts<kIn>(bp[4])};
                                mma(acc[n], a, b);
                            }
                    }
                    if (some) {
    #pragma unroll
                        for (int n = 0; n < kOn; ++n)
    #pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const int i = m0 + g + 8 * (x >> 1), j = c0 + 8 * n + 2 * t + (x & 1);
                                const int apart = kRev ? j - i : i - j;
                                acc[n][x] = apart >= 0 ? acc[n][x] * (p.sigma * pw[apart]) : 0.f;
                            }
    #pragma unroll
                        for (int n = 0; n < kOn; ++n) {
                            float* dst = ps + (m0 + g) * kLdP + c0 + 8 * n + 2 * t;
                            *reinterpret_cast<float2*>(dst) = make_float2(acc[n][0], acc[n][1]);
                            *reinterpret_cast<float2*>(dst + 8 * kLdP) =
                                make_float2(acc[n][2], acc[n][3]);
                        }
                    }
    #pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int i = m0 + g + 8 * (x >> 1);
                        const float ahead = pw[kRev ? max(len - 1 - i, 0) : i + 1];
    #pragma unroll
                        for (int n = 0; n < kOn; ++n) o[n][x] *= ahead;
                    }
                    __syncthreads();
                }
            }
            if (c + 1 < nch) fetch(c + 1);
            if (c < 0) continue;
            if (!state_only) {
                // The scores' part: the mask leaves columns up to m0 + 15, or from m0 on.
                for (int k = kRev ? m0 : 0; k < (kRev ? kC : m0 + 16); k += 8) {
                    const float* ap = ps + (m0 + g) * kLdP + k + t;
                    const Parts<2> a[4] = {parts<2>(ap[0]), parts<2>(ap[8 * kLdP]), parts<2>(ap[4]),
                                           parts<2>(ap[8 * kLdP + 4])};
#pragma unroll
                    for (int n = 0; n < kOn; ++n) {
                        const float* bp = cs + (k + t) * kLdC + c0 + 8 * n + g;
                        const Parts<kIn> b[2] = {parts<kIn>(bp[0]), parts<kIn>(bp[4 * kLdC])};
                        mma(o[n], a, b);
                    }
                }
#pragma unroll
                for (int n = 0; n < kOn; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int i = m0 + g + 8 * (x >> 1);
                        const int col = n0 + c0 + 8 * n + 2 * t + (x & 1);
                        if (i >= len || col >= p.d_c) continue;
                        const int64_t at = ((row + i) * p.heads + h) * p.d_c + col;
                        const float y = o[n][x] * p.tau;
                        if (p.out_f32) static_cast<float*>(p.out)[at] = y;
                        else static_cast<T*>(p.out)[at] = from_f32<T>(y);
                    }
            }
            // The update: 16 rows of the weighted b^T x c.
#pragma unroll
            for (int n = 0; n < kUn; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[n][x] = fmaf(s[n][x], f.x, s[n][x] * f.y);
#pragma unroll 2
            for (int k = 0; k < len; k += 8) {
                const float* ap = bs + (k + t) * kLdA + um0 + g;
                const float w0 = p.sigma * pw[kRev ? k + t + 1 : max(len - 1 - k - t, 0)];
                const float w1 = p.sigma * pw[kRev ? k + t + 5 : max(len - 5 - k - t, 0)];
                const Parts<2> a[4] = {parts<2>(ap[0] * w0), parts<2>(ap[8] * w0),
                                       parts<2>(ap[4 * kLdA] * w1),
                                       parts<2>(ap[4 * kLdA + 8] * w1)};
#pragma unroll
                for (int n = 0; n < kUn; ++n) {
                    const float* bp = cs + (k + t) * kLdC + un0 + 8 * n + g;
                    const Parts<kIn> b[2] = {parts<kIn>(bp[0]), parts<kIn>(bp[4 * kLdC])};
                    mma(s[n], a, b);
                }
            }
            __syncthreads();  // before the next chunk's tiles
        }
        const LaState out = la_state(p, it.out, h, p.state_out, scratch);
        if (out.ptr != nullptr)
#pragma unroll
            for (int n = 0; n < kUn; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int row = um0 + g + 8 * (x >> 1), col = n0 + un0 + 8 * n + 2 * t + (x & 1);
                    if (row < p.d_b && col < p.d_c)
                        const_cast<float*>(out.ptr)[row * out.row + col * out.col] = s[n][x];
                }
        if (work == nullptr) break;  // one job a CTA
        if (tid == 0) next_job = atomicAdd(&work->next, 1);
        __syncthreads();
        id = next_job;
        __syncthreads();
    }
}

template <typename T, int kDb, bool kRev>
cudaError_t start(const LaCore& p, LaSplitCost how, cudaStream_t stream) {
    auto* kernel = la_mma<T, kDb, kRev>;
    constexpr int kSmem = static_cast<int>(sizeof(float)) * smem_floats<kDb>();
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    const uintptr_t unit = 4 * sizeof(T) - 1;
    const bool vec_ab = p.d_b % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.a) |
                                            reinterpret_cast<uintptr_t>(p.b)) & unit) == 0;
    const bool vec_c = p.d_c % 4 == 0 && (reinterpret_cast<uintptr_t>(p.c) & unit) == 0;
    const int grid = la_sm_count() * (kDb == 64 ? 2 : 1), blocks = (p.d_c + kCols - 1) / kCols;
    LaLists lists;
    if ((e = la_prepare(p, grid, blocks, how, lists, stream)) != cudaSuccess) return e;
    if (lists.split) {
        kernel<<<grid, threads_of<kDb>(), kSmem, stream>>>(p, &lists.plan->states, lists.states, lists.slots,
                                                  true, vec_ab, vec_c);
        la_scan_states(p, lists, stream);
    }
    const int64_t jobs = static_cast<int64_t>(p.n_seqs) * p.heads * blocks;
    kernel<<<lists.plan != nullptr ? grid : static_cast<int>(jobs), threads_of<kDb>(), kSmem, stream>>>(
        p, lists.plan != nullptr ? &lists.plan->main : nullptr, lists.main, lists.slots, false,
        vec_ab, vec_c);
    e = cudaGetLastError();
    const cudaError_t f = la_release(lists, stream);
    return e != cudaSuccess ? e : f;
}

template <typename T>
cudaError_t pick(const LaCore& p, LaSplitCost how, cudaStream_t stream) {
    if (p.d_b <= 64)
        return p.reverse ? start<T, 64, true>(p, how, stream) : start<T, 64, false>(p, how, stream);
    return p.reverse ? start<T, 128, true>(p, how, stream) : start<T, 128, false>(p, how, stream);
}

}  // namespace

bool la_mma_supports(const LaCore& p) {
    return p.d_b <= 128 && p.d_c <= kLaMaxD && la_tokens(p) < (int64_t{1} << 31) - 2 * kLaChunk &&
           static_cast<int64_t>(p.n_seqs) * p.heads < (int64_t{1} << 28);
}

cudaError_t launch_la_mma(const LaCore& p, cudaStream_t stream) {
    // A chunk of the states' pass is a third of one of the main pass.
    const LaSplitCost how{true, false, 0, 0.35f, 2.f};
    switch (p.dtype) {
        case GDR_DTYPE_BF16: return pick<__nv_bfloat16>(p, how, stream);
        case GDR_DTYPE_F16: return pick<__half>(p, how, stream);
        default: return pick<float>(p, how, stream);
    }
}

}  // namespace gdr
