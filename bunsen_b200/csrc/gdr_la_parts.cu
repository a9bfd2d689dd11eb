// The decayed linear attention core (gdr_la.cuh) in chunks at f32 accuracy, on the tensor
// cores: f32 and f16 operands, and bf16 ones of widths gdr_la_tc.cu does not take;
// d_b up to 128, d_c up to 256.
//
// The same sums as gdr_la_tc.cu in chunks of C = 64 positions:
//   out_i = tau [ w^{i+1} a_i . S + sum_{j<=i} sigma w^{i-j} (a_i.b_j) c_j ]
//   S'    = w^C S + sum_j sigma w^{C-1-j} b_j c_j^T
// (backward in time their mirror image). Every operand goes in as bf16 parts, x = x0 +
// x1 + x2 with 8 bits each (f16: two parts exactly, bf16: one), which keep f32's range
// at any magnitude; of a product the parts x_i y_j with i + j <= 2 leave 2^-24 of it,
// six products for f32. tcgen05.mma at 4096 bf16 products a cycle and SM makes that 680
// f32 ones; three tf32 products by mma.sync make 163, FFMA 117.
//
// One CTA an SM takes a (sequence or segment, head) and 128 columns of the state:
//   16 warps convert: a, b and the weighted b to parts in shared memory, c to TMEM with the
//            columns of c on the lanes, the state's copy to TMEM (its third part to shared
//            memory); they turn scores into P, write the outputs, and hold the
//            state, 32 values a thread
//   1 warp   issues the products
//   3 warps  bring the lines of the chunk after the next to L2
// The products of a chunk, N positions or rows of b on the columns of TMEM:
//   scores = A B^T          64 x 64
//   O1^T   = S^T A^T        128 x 64, the state's copy as the first operand
//   O2^T   = C^T P^T        128 x 64, over the scores
//   U^T    = C^T (w B)      128 x d_b
// c never is in shared memory: a thread reads one column of it, 16 positions,
// neighbouring lanes neighbouring columns, and that is how TMEM wants it; outputs go out
// the same way. A product with both operands in shared memory reads 6 KiB of it in the 32
// cycles of 128 x 64 x 16, half again what it delivers, so what can be comes from
// TMEM (the state's copy wholly in shared memory: 221 us for 8192 packed positions and
// 16 heads, against 194 us). A chunk's loads go out in the waits for the products, a early,
// b and c late: all at once they wait for one another.
//
// TMEM (512 columns): scores and O2 64, O1 64, U 128, c three parts of 32, the state's copy two
// of 64.
//
// Bound: 5000 tensor cycles a chunk at f32 and 128 x 128, 2.9 us, where a chunk takes 5.8 us
// (8192 packed positions, 16 heads, d = 128: 182 us; with mma.sync in three tf32 products and
// shared memory alone 988 us): issue slots, 0.67 of them taken by conversions and the address
// work around them, in a chain with the products.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "gdr_la.cuh"
#include "gdr_la_plan.cuh"
#include "gdr_la_sm100.cuh"

namespace gdr {

// As g_la_error in gdr_la_tc.cu.
__device__ int g_la_parts_error;

namespace {

using namespace sm100;

constexpr int kC = 64, kCols = 128;
constexpr int kWarps = 16, kThreads = 32 * (kWarps + 4);
constexpr uint32_t kRows64 = 64 * 128, kRows128 = 128 * 128;  // bytes of a tile 64 wide
constexpr uint32_t kColSc = 0, kColO2 = 0, kColO1 = 64, kColU = 128, kColC = 256, kColS = 352;

template <typename T, int kDb, bool kStateOnly>
struct Layout {
    static constexpr int kIn = sizeof(T) == 4 ? 3 : std::is_same_v<T, __half> ? 2 : 1;
    // P and the state's copy, and the parts' products: outputs of 16 bits need 16. Each is off by
    // 2^-16 of itself at most, and so is each product of two parts left out: 2^-16 of the
    // sums of absolute terms for bf16, three times that for f16, where rounding the output takes
    // 2^-8 and 2^-11 of what has not cancelled.
    static constexpr int kPs = sizeof(T) == 4 ? 3 : 2;
    static constexpr int kHalves = kDb / 64;
    static constexpr uint32_t kTileAb = kHalves * kRows64, kTileS = kHalves * kRows128;
    // a, b, the weighted b, the third part of the state's copy, P; or two weighted b.
    static constexpr uint32_t kA = 0, kB = kA + kIn * kTileAb;
    static constexpr uint32_t kBw = kStateOnly ? 0 : kB + kIn * kTileAb;
    static constexpr uint32_t kS = kBw + (kStateOnly ? 6 : 3) * kTileAb;
    static constexpr uint32_t kP = kS + (kStateOnly || kPs < 3 ? 0 : kTileS);
    static constexpr uint32_t kMisc = kP + (kStateOnly ? 0 : kPs * kRows64);
    static constexpr uint32_t kBytes = kMisc + 2048;
};

struct Misc {
    // Powers for a job's whole chunks, and for its short one:
    alignas(16) float wt[2][kC];     // sigma w^{len-1-j}, the weights of b (backward w^{j+1})
    alignas(16) float ahead[2][kC];  // tau w^{i+1}, of a_i . S (backward w^{len-1-i})
    float2 f[2];                     // w^len, in two parts
    float decay[kC];                 // sigma w^0 .. w^{kC-1}
    uint64_t ab_ready, s_ready, p_ready, w_ready[2], sc_full, o_full, u_full[2], drain;
    uint32_t tmem;
    uint32_t scored;  // chunks whose scores' product is issued
    int next;
};
static_assert(sizeof(Misc) <= 2048, "its room");

// 2 kN values in kParts bf16 parts each, put(k, part k of the pairs) part by part.
// (Volatile: kN chains at once and no more, or the registers run out. Scalar
// differences: pairs of f32 took more moves and registers than they saved.)
template <int kParts, int kN, typename F>
__device__ __forceinline__ void split(float (&v)[kN], F&& put) {
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
        uint32_t r[kN / 2];
#pragma unroll
        for (int j = 0; j < kN / 2; ++j)
            asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r[j]) : "f"(v[2 * j + 1]), "f"(v[2 * j]));
        put(k, r);
        if (k + 1 < kParts)
#pragma unroll
            for (int j = 0; j < kN / 2; ++j) {
                v[2 * j] -= low_f32(r[j]);
                v[2 * j + 1] -= high_f32(r[j]);
            }
    }
}

// D (+)= A B over 16 kSteps of K, both K-major in shared memory in tiles 64 wide, kJump*
// bytes apart. (Addresses step inside the assembly: four instructions a product.)
template <int kHalves, uint32_t kJumpA, uint32_t kJumpB>
__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "mov.b64 a, %1;\n\tmov.b64 b, %2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
    if constexpr (kHalves == 2)
        product_ss<1, 0, 0>(d, a + kJumpA / 16, b + kJumpB / 16, idesc, 1);
}
// D (+)= A B over 64 of K: A in TMEM, B's steps kStep bytes apart.
template <uint32_t kStep>
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tmov.b32 a, %1;\n\tmov.b64 b, %2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, %5;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, %5;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, %5;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(kStep / 16)
        : "memory");
}
// The parts (i, j) of a product with i + j <= kOrder, the smallest first.
template <int kX, int kY, int kOrder, typename F>
__device__ __forceinline__ void each_part(F&& f) {
    bool first = true;
#pragma unroll
    for (int o = kOrder; o >= 0; --o)
#pragma unroll
        for (int i = 0; i <= o; ++i)
            if (i < kX && o - i < kY) {
                f(i, o - i, first ? 0u : 1u);
                first = false;
            }
}

// x, unknown to the compiler: what follows from it is computed where it is used and not
// kept in registers over the chunks (as hoisted addresses it spilled).
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+r"(x));
    return x;
}

// (Volatile: in the order written, so that one store's values at a time are in registers.)
__device__ __forceinline__ void st_shared(uint32_t at, uint32_t x, uint32_t y, uint32_t z,
                                          uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

// Eight neighbours of a row, as read.
template <typename T>
struct Eight {
    T v[8];
};
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* at, int left, bool vec) {
    Eight<T> e{};
    if (left <= 0) return e;
    if (vec) {  // (d is a multiple of 8 then, and rows begin on 16 bytes)
        constexpr int kV = sizeof(Eight<T>) / 16;
#pragma unroll
        for (int i = 0; i < kV; ++i)
            reinterpret_cast<uint4*>(e.v)[i] = reinterpret_cast<const uint4*>(at)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) e.v[i] = at[i];
    }
    return e;
}

template <typename T, int kN>
struct Operand {
    Eight<T> v[kN];
};

template <typename T, int kDb, bool kRev, bool kStateOnly>
__global__ void __launch_bounds__(kThreads, 1)
la_parts(const LaCore p, LaWork* work, const LaEntry* entries, float* scratch, bool vec) {
    using L = Layout<T, kDb, kStateOnly>;
    constexpr int kIn = L::kIn, kPs = L::kPs, kOrder = kPs - 1, kHalves = L::kHalves;
    constexpr int kEights = kC * kDb / 8 / (32 * kWarps);  // of a and of b, a thread
    constexpr int kMine = kDb / 4;                         // the state's rows of a thread
    extern __shared__ __align__(1024) uint8_t sm[];
    Misc& M = *reinterpret_cast<Misc*>(sm + L::kMisc);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        M.scored = 0;
        mbar_init(&M.ab_ready, kWarps);
        mbar_init(&M.s_ready, kWarps);
        mbar_init(&M.p_ready, kWarps);
        mbar_init(&M.w_ready[0], kWarps);
        mbar_init(&M.w_ready[1], kWarps);
        mbar_init(&M.sc_full, 1);
        mbar_init(&M.o_full, 1);
        mbar_init(&M.u_full[0], 1);
        mbar_init(&M.u_full[1], 1);
        mbar_init(&M.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarps) {
        tmem_alloc(&M.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    after_last_kernel();
    __syncthreads();
    tc_fence_after();
    bool ok = M.tmem == 0 && (smem_u32(sm) & 1023) == 0;  // (all columns: they begin at 0)
    const int blocks = (p.d_c + kCols - 1) / kCols;
    const int jobs = (work != nullptr ? work->count : p.n_seqs) * p.heads * blocks;
    const int quarter = warp & 3, part = warp >> 2;
    const uint32_t base = smem_u32(sm);
    const uint32_t quad = static_cast<uint32_t>(quarter) << 21;  // this warp's lanes
    uint32_t n = 0;                                              // chunks before
    // The jobs, one after the other: body(entry, head, first column, chunks).
    auto each_job = [&](auto&& body) {
        int id = blockIdx.x;
#pragma unroll 1
        while (id < jobs) {
            const int e = id / blocks / p.heads;
            LaEntry it;
            if (work != nullptr) {
                it = entries[e];
            } else {
                int64_t start, end;
                la_span(p, e, start, end);
                it = {static_cast<int32_t>(start), static_cast<int32_t>(end - start), e, e};
            }
            const int nch = (it.len + kC - 1) / kC;
            body(it, id / blocks % p.heads, id % blocks * kCols, nch);
            n += nch;
            if (tid == 0) M.next = work != nullptr ? atomicAdd(&work->next, 1) : jobs;
            if (!__syncthreads_and(ok)) break;
            id = M.next;
            __syncthreads();
        }
    };
    // The launch gives each thread 96 registers, 480 for the five warpgroups' lanes together:
    // 4 x 112 + 32.
    if (warp >= kWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        each_job([&](const LaEntry& it, int h, int n0, int nch) {
            // ---- the products ------------------------------------------------------
            constexpr uint32_t kScores = idesc_bf16(64, kC, 0, 0, 0);
            constexpr uint32_t kKK = idesc_bf16(128, kC, 0, 0, 0);
            constexpr uint32_t kKMn = idesc_bf16(128, kDb, 0, 1, 0);
            auto update = [&](uint32_t b_at, uint32_t c_at, uint32_t u_at) {
                each_part<kIn, 3, 2>([&](int i, int j, uint32_t acc) {
                    product_ts<2048>(u_at, c_at + 32 * i,
                                     sdesc_sw128(b_at + j * L::kTileAb, kRows64, 1024), kKMn, acc);
                });
            };
            __syncthreads();  // (the converting warps' one at a job's start)
#pragma unroll 1
            for (int c = 0; warp == kWarps && ok && c < nch; ++c) {
                const uint32_t ph = (n + c) & 1, base = here(smem_u32(sm));
                if constexpr (kStateOnly) {
                    if (!(ok = warp_wait(&M.w_ready[ph], ((n + c) >> 1) & 1))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        update(base + ph * 3 * L::kTileAb, kColC + 96 * ph, 128 * ph);
                        umma_commit(&M.u_full[ph]);
                    }
                } else {
                    if (!(ok = warp_wait(&M.ab_ready, ph))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        each_part<kIn, kIn, kOrder>([&](int i, int j, uint32_t acc) {
                            product_ss<kHalves, kRows64, kRows64>(
                                kColSc, sdesc_sw128(base + L::kA + i * L::kTileAb, 16, 1024),
                                sdesc_sw128(base + L::kB + j * L::kTileAb, 16, 1024), kScores, acc);
                        });
                        umma_commit(&M.sc_full);
                        *const_cast<volatile uint32_t*>(&M.scored) = n + c + 1;
                    }
                    if (!(ok = warp_wait(&M.s_ready, ph))) break;
                    tc_fence_after();
                    if (elect_one())
                        each_part<kPs, kIn, kOrder>([&](int i, int j, uint32_t acc) {
                            const uint32_t a_at = base + L::kA + j * L::kTileAb;
                            if (i == 2) {
                                product_ss<kHalves, kRows128, kRows64>(
                                    kColO1, sdesc_sw128(base + L::kS, 16, 1024),
                                    sdesc_sw128(a_at, 16, 1024), kKK, acc);
                                return;
                            }
#pragma unroll
                            for (int x = 0; x < kHalves; ++x)
                                product_ts<32>(kColO1, kColS + kDb / 2 * i + 32 * x,
                                               sdesc_sw128(a_at + x * kRows64, 16, 1024), kKK,
                                               x == 0 ? acc : 1);
                        });
                    if (!(ok = warp_wait(&M.p_ready, ph))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        each_part<kIn, kPs, kOrder>([&](int i, int j, uint32_t acc) {
                            product_ts<32>(kColO2, kColC + 32 * i,
                                           sdesc_sw128(base + L::kP + j * kRows64, 16, 1024), kKK,
                                           acc);
                        });
                        umma_commit(&M.o_full);
                    }
                    if (!(ok = warp_wait(&M.w_ready[0], ph))) break;
                    tc_fence_after();
                    if (elect_one()) {
                        update(base + L::kBw, kColC, kColU);
                        umma_commit(&M.u_full[0]);
                    }
                }
            }
            // Lines to L2, by the group's other warps, two chunks ahead: the loads come in bursts,
            // of every SM at about the same time, and HBM would not keep up with them.
#pragma unroll 1
            for (int c = 1; !kStateOnly && warp > kWarps && c < nch; ++c) {
                // (By a count, not by a phase: these warps may fall behind by more than
                // one. Nothing hangs on them: they go on when the tries run out.)
                for (int tries = 0; tries < 4096; ++tries) {
                    if (static_cast<int32_t>(*const_cast<volatile uint32_t*>(&M.scored) - (n + c)) >= -1)
                        break;
                    __nanosleep(200);
                }
                constexpr int kLine = 128 / static_cast<int>(sizeof(T));
                const int x0 = kRev ? nch - 1 - c : c;
                const int64_t row = static_cast<int64_t>(it.start) + x0 * kC;
                const int len = min(kC, it.len - x0 * kC);
                auto lines = [&](const void* of, int heads, int d, int from, int width) {
                    const T* src = static_cast<const T*>(of) +
                                   (row * heads + h / (p.heads / heads)) * d + from;
                    const int each = (min(width, d - from) + kLine - 1) / kLine;
#pragma unroll 1
                    for (int x = tid - 32 * (kWarps + 1); x < len * each; x += 96)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(
                            src + x / each * (heads * d) + x % each * kLine));
                };
                lines(p.a, p.heads_a, p.d_b, 0, kDb);
                lines(p.c, p.heads_c, p.d_c, n0, kCols);
                lines(p.b, p.heads_b, p.d_b, 0, kDb);
            }
        });
        if (warp == kWarps) {  // nothing of this CTA's may be in flight when it ends
            if (elect_one()) umma_commit(&M.drain);
            warp_wait(&M.drain, 0);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        each_job([&](const LaEntry& it, int h, int n0, int nch) {
            // ---- conversions, outputs, the state -----------------------------------------
            const int col = 32 * quarter + lane;  // this thread's column of c, of 128
            const bool mine = n0 + col < p.d_c;
            const int ha = h / (p.heads / p.heads_a), hb = h / (p.heads / p.heads_b),
                      hc = h / (p.heads / p.heads_c);
            // Operands on their way. (Fetched after the last chunk too, as zeros: behind
            // conditions they took more registers.)
            using Ab = Operand<T, kEights>;
            using Column = Operand<T, 2>;
            auto chunk_at = [&](int c, int64_t& row, int& len) {
                const int x = kRev ? nch - 1 - c : c;
                row = static_cast<int64_t>(it.start) + x * kC;
                len = c < nch ? min(kC, it.len - x * kC) : 0;  // (after the last chunk: nothing)
            };
            auto fetch = [&](const void* base, int heads, int head, int c) {
                Ab o;
                int64_t row;
                int len;
                chunk_at(c, row, len);
                const int tid = here(threadIdx.x), step = heads * p.d_b;
                const T* src = static_cast<const T*>(base) + (row * heads + head) * p.d_b;
#pragma unroll
                for (int i = 0; i < kEights; ++i) {
                    const int at = tid + 32 * kWarps * i, r = at / (kDb / 8), d = at % (kDb / 8) * 8;
                    o.v[i] = load8(src + (r * step + d), r < len ? p.d_b - d : 0, here(vec));
                }
                return o;
            };
            auto fetch_c = [&](int c) {
                Column o;
                int64_t row;
                int len;
                chunk_at(c, row, len);
                const int step = p.heads_c * p.d_c;  // (64 of them are below 2^31)
                const T* src = static_cast<const T*>(p.c) + (row * p.heads_c + hc) * p.d_c + n0 +
                               32 * quarter + here(lane) + 16 * part * step;
                const int live = mine ? len - 16 * part : 0;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    o.v[j >> 3].v[j & 7] = j < live ? src[j * step] : T(0.f);
                return o;
            };
            // Parts of a or b, or of b with weights: rows of 128 bytes, 16 of them
            // exchanged by the row's number.
            auto put = [&](uint32_t at, const Ab& from, auto parts, const float* weights) {
                const int tid = here(threadIdx.x);
#pragma unroll
                for (int i = 0; i < kEights; ++i) {
                    const int x = tid + 32 * kWarps * i, r = x / (kDb / 8), d = x % (kDb / 8);
                    const float w = weights != nullptr ? weights[r] : 1.f;
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[j] = to_f32(from.v[i].v[j]);
                        if (weights != nullptr) v[j] *= w;
                    }
                    const uint32_t dst = base + at + (d >> 3) * kRows64 + r * 128 + (((d ^ r) & 7) << 4);
                    split<decltype(parts)::value>(v, [&](int k, const uint32_t(&r)[4]) {
                        st_shared(dst + k * L::kTileAb, r[0], r[1], r[2], r[3]);
                    });
                }
            };
            constexpr std::integral_constant<int, kIn> as_read{};
            constexpr std::integral_constant<int, 3> weighted{};
            auto put_c = [&](uint32_t at, const Column& vc) {
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = to_f32(vc.v[j >> 3].v[j & 7]);
                split<kIn>(v, [&](int k, const uint32_t(&r)[8]) {
                    tmem_st8(quad + at + 32 * k + 8 * part, r);
                });
            };
            auto arrive = [&](uint64_t* bar) {  // all of this warp's writes before
                tmem_wait_st();
                tc_fence_before();
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            Ab va;
            if (!kStateOnly) va = fetch(p.a, p.heads_a, ha, 0);
            Ab vb = fetch(p.b, p.heads_b, hb, 0);
            Column vc = fetch_c(0);  // positions 16 part .. + 15 of this thread's column
            const float decay = p.log_decay[h];
            {
                const int len = tid < 4 * kC / 2 || it.len % kC == 0 ? kC : it.len % kC;
                const int j = tid % kC, up = j + 1, down = max(len - 1 - j, 0);
                if (tid < 4 * kC) {
                    const bool wt = tid / kC % 2 == 0;
                    const float f = la_power(decay, wt == kRev ? up : down);
                    if (wt) M.wt[tid / (2 * kC)][j] = p.sigma * f;
                    else M.ahead[tid / (2 * kC)][j] = p.tau * f;
                } else if (tid < 5 * kC) {
                    M.decay[j] = p.sigma * la_power(decay, j);
                }
                if (j == 0 && tid <= 2 * kC) M.f[tid / (2 * kC)] = la_power2(decay, len);
            }
            uint64_t s[kMine / 2];  // rows kMine part .. of the state, pairs
            const LaState in = la_state(p, it.in, h, p.state_in, scratch);
            {
                const int b0 = kMine * part;
                const float* src = in.ptr + (n0 + col) * in.col + b0 * in.row;
                const bool any = in.ptr != nullptr && mine;
#pragma unroll
                for (int j = 0; j < kMine / 2; ++j, src += 2 * in.row)
                    s[j] = pair(any && b0 + 2 * j < p.d_b ? src[0] : 0.f,
                                any && b0 + 2 * j + 1 < p.d_b ? src[in.row] : 0.f);
            }
            __syncthreads();  // the powers
            auto add_update = [&](uint32_t at, int len) {
                const float2 f = M.f[len < kC];
                const uint64_t hi2 = pair(f.x, f.x), lo2 = pair(f.y, f.y);
#pragma unroll
                for (int blk = 0; blk < kMine / 8; ++blk) {
                    uint64_t u[4];
                    tmem_ld8(quad + at + kMine * part + 8 * blk, u);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[4 * blk + j] = fma2(s[4 * blk + j], hi2, fma2(s[4 * blk + j], lo2, u[j]));
                }
                tc_fence_before();  // (before this warp's next arrival)
            };
            auto len_of = [&](int c) { return min(kC, it.len - (kRev ? nch - 1 - c : c) * kC); };
            if constexpr (kStateOnly) {
                // The conversions of a chunk run beside the product of the one before.
#pragma unroll 1
                for (int c = 0; c < nch; ++c) {
                    const uint32_t ph = (n + c) & 1;
                    put(ph * 3 * L::kTileAb, vb, weighted, M.wt[len_of(c) < kC]);
                    put_c(kColC + 96 * ph, vc);
                    // (By buffer: a warp may be a chunk ahead of another, and must not arrive
                    // in its place.)
                    arrive(&M.w_ready[ph]);
                    vb = fetch(p.b, p.heads_b, hb, c + 1);
                    vc = fetch_c(c + 1);
                    if (c > 0) {
                        if (!(ok = warp_wait(&M.u_full[ph ^ 1], ((n + c - 1) >> 1) & 1))) break;
                        tc_fence_after();
                        add_update(128 * (ph ^ 1), len_of(c - 1));
                    }
                }
                if (ok && nch > 0) {
                    const uint32_t m = n + nch - 1;
                    if ((ok = warp_wait(&M.u_full[m & 1], (m >> 1) & 1))) {
                        tc_fence_after();
                        add_update(128 * (m & 1), len_of(nch - 1));
                    }
                }
            } else {
                put(L::kA, va, as_read, nullptr);
#pragma unroll 1
                for (int c = 0; c < nch; ++c) {
                    const uint32_t ph = (n + c) & 1;
                    const int x = kRev ? nch - 1 - c : c, len = len_of(c);
                    put(L::kB, vb, as_read, nullptr);
                    arrive(&M.ab_ready);
                    // The state's copy: two parts on TMEM's lanes, the third in shared memory,
                    // which the scores' product keeps busy.
#pragma unroll
                    for (int m = 0; m < kMine / 16; ++m) {
                        const int col = 32 * quarter + here(lane);
                        const int at = kMine * part + 16 * m;  // rows
                        float v[16];
#pragma unroll
                        for (int j = 0; j < 8; ++j) unpair(s[8 * m + j], v[2 * j], v[2 * j + 1]);
                        split<kPs>(v, [&](int k, const uint32_t(&r)[8]) {
                            if (k < 2) {
                                tmem_st8(quad + kColS + kDb / 2 * k + at / 2, r);
                                return;
                            }
                            const uint32_t dst = base + L::kS + (at >> 6) * kRows128 + col * 128;
                            const int x = at >> 3 & 7;
                            st_shared(dst + ((x ^ col) & 7) * 16, r[0], r[1], r[2], r[3]);
                            st_shared(dst + (((x + 1) ^ col) & 7) * 16, r[4], r[5], r[6], r[7]);
                        });
                    }
                    arrive(&M.s_ready);
                    put_c(kColC, vc);
                    // (The next chunk's loads go out in the waits: all at once they took 4000
                    // cycles of the L2's time.)
                    const Ab na = fetch(p.a, p.heads_a, ha, c + 1);
                    {
                        // P: the scores' 64 rows are the first 16 lanes of every quarter; the others
                        // take half of their 16 columns. What the mask leaves, decayed.
                        const int i = 16 * quarter + here(lane & 15);
                        const int j0 = 16 * part + (lane & 16) / 2;
                        if (!(ok = warp_wait(&M.sc_full, ph))) break;
                        tc_fence_after();
                        uint64_t near[4], far[4];
                        tmem_ld8(quad + kColSc + 16 * part, near);
                        tmem_ld8(quad + kColSc + 16 * part + 8, far);
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint64_t other = __shfl_sync(0xffffffffu, far[j], lane & 15);
                            unpair(lane < 16 ? near[j] : other, v[2 * j], v[2 * j + 1]);
                            const int e0 = kRev ? j0 + 2 * j - i : i - j0 - 2 * j;
                            const int e1 = kRev ? e0 + 1 : e0 - 1;
                            v[2 * j] = e0 >= 0 ? v[2 * j] * M.decay[e0] : 0.f;
                            v[2 * j + 1] = e1 >= 0 ? v[2 * j + 1] * M.decay[e1] : 0.f;
                        }
                        const uint32_t dst = base + L::kP + i * 128 + (((j0 >> 3) ^ i) & 7) * 16;
                        split<kPs>(v, [&](int k, const uint32_t(&r)[4]) {
                            st_shared(dst + k * kRows64, r[0], r[1], r[2], r[3]);
                        });
                        arrive(&M.p_ready);
                    }
                    put(L::kBw, vb, weighted, M.wt[len < kC]);
                    arrive(&M.w_ready[0]);
                    vb = fetch(p.b, p.heads_b, hb, c + 1);
                    vc = fetch_c(c + 1);
                    if (!(ok = warp_wait(&M.o_full, ph))) break;
                    tc_fence_after();
                    {
                        const int step = p.heads * p.d_c;
                        const int col = 32 * quarter + here(lane);
                        const int64_t at =
                            static_cast<int64_t>(it.start + x * kC + 16 * part) * step +
                            static_cast<int64_t>(h) * p.d_c + n0 + col;
                        const int live = mine ? len - 16 * part : 0;
                        auto outputs = [&](auto* to) {
                            const uint64_t tau = pair(p.tau, p.tau);
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                uint64_t u[4], v[4];
                                tmem_ld8(quad + kColO1 + 16 * part + 8 * m, u);
                                tmem_ld8(quad + kColO2 + 16 * part + 8 * m, v);
                                const ulonglong2* ahead = reinterpret_cast<const ulonglong2*>(
                                    &M.ahead[len < kC][16 * part + 8 * m]);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const uint64_t f = j & 1 ? ahead[j >> 1].y : ahead[j >> 1].x;
                                    float y[2];
                                    unpair(fma2(u[j], f, mul2(v[j], tau)), y[0], y[1]);
#pragma unroll
                                    for (int k = 0; k < 2; ++k)
                                        if (8 * m + 2 * j + k < live)
                                            to[(8 * m + 2 * j + k) * step] =
                                                from_f32<std::remove_reference_t<decltype(*to)>>(y[k]);
                                }
                            }
                        };
                        if (here(p.out_f32)) outputs(static_cast<float*>(p.out) + at);
                        else outputs(static_cast<T*>(p.out) + at);
                    }
                    put(L::kA, na, as_read, nullptr);
                    if (!(ok = warp_wait(&M.u_full[0], ph))) break;
                    tc_fence_after();
                    add_update(kColU, len);
                }
            }
            const LaState out = la_state(p, it.out, h, p.state_out, scratch);
            if (ok && out.ptr != nullptr && mine) {
                const int b0 = kMine * part;
                float* dst = const_cast<float*>(out.ptr) + (n0 + col) * out.col + b0 * out.row;
#pragma unroll
                for (int j = 0; j < kMine / 2; ++j, dst += 2 * out.row) {
                    float f[2];
                    unpair(s[j], f[0], f[1]);
                    if (b0 + 2 * j < p.d_b) dst[0] = f[0];
                    if (b0 + 2 * j + 1 < p.d_b) dst[out.row] = f[1];
                }
            }
        });
    }
    if (!ok && lane == 0) atomicOr(&g_la_parts_error, 1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kWarps) tmem_dealloc(M.tmem, 512);
}

template <typename T, int kDb, bool kRev>
cudaError_t start(const LaCore& p, LaLists* shared, bool chained, cudaStream_t stream) {
    auto* full = la_parts<T, kDb, kRev, false>;
    auto* states = la_parts<T, kDb, kRev, true>;
    constexpr int kFull = static_cast<int>(Layout<T, kDb, false>::kBytes),
                  kStates = static_cast<int>(Layout<T, kDb, true>::kBytes);
    static std::atomic<uint64_t> full_done{0}, states_done{0};
    cudaError_t e = la_allow_smem(full, kFull, full_done);
    if (e == cudaSuccess) e = la_allow_smem(states, kStates, states_done);
    if (e != cudaSuccess) return e;
    const bool vec = p.d_b % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.a) |
                                         reinterpret_cast<uintptr_t>(p.b)) & 15) == 0;
    const int grid = la_sm_count(), blocks = (p.d_c + kCols - 1) / kCols;
    // In chunks of 128: 13 us at one CTA an SM, 0.3 of that in the states' pass, whose start,
    // the list's kernel and the scan are 2.
    LaLists own;
    LaLists& lists = shared != nullptr ? *shared : own;
    if (lists.uses == 0) {
        e = la_prepare(p, grid, blocks, {true, false, 0, 0.3f, 2.f}, shared != nullptr, chained, lists,
                       stream);
        if (e != cudaSuccess) return e;
        if (lists.split) {
            e = la_launch_next(states, grid, kThreads, kStates, stream, p, &lists.plan->states,
                               lists.states, lists.slots, vec);
            if (e == cudaSuccess) e = la_scan_states(p, lists, stream);
        }
    }
    const int64_t jobs = static_cast<int64_t>(p.n_seqs) * p.heads * blocks;
    if (e == cudaSuccess && lists.plan != nullptr)
        e = la_launch_next(full, grid, kThreads, kFull, stream, p, &lists.plan->main[lists.uses],
                           lists.main, lists.slots, vec);
    else if (e == cudaSuccess)
        full<<<static_cast<int>(jobs), kThreads, kFull, stream>>>(p, nullptr, nullptr, nullptr, vec);
    ++lists.uses;
    if (e == cudaSuccess) e = cudaGetLastError();
    const cudaError_t f = la_release(own, stream);
    return e != cudaSuccess ? e : f;
}

template <typename T>
cudaError_t pick(const LaCore& p, LaLists* shared, bool chained, cudaStream_t stream) {
    if (p.d_b <= 64)
        return (p.reverse ? start<T, 64, true> : start<T, 64, false>)(p, shared, chained, stream);
    return (p.reverse ? start<T, 128, true> : start<T, 128, false>)(p, shared, chained, stream);
}

}  // namespace

bool la_parts_supports(const LaCore& p) {
    return p.d_b <= 128 && p.d_c <= kLaMaxD && la_tokens(p) < (int64_t{1} << 31) - 2 * kLaChunk &&
           static_cast<int64_t>(p.n_seqs) * p.heads < (int64_t{1} << 28);
}

cudaError_t launch_la_parts(const LaCore& p, cudaStream_t stream, LaLists* shared, bool chained) {
    switch (p.dtype) {
        case GDR_DTYPE_BF16: return pick<__nv_bfloat16>(p, shared, chained, stream);
        case GDR_DTYPE_F16: return pick<__half>(p, shared, chained, stream);
        default: return pick<float>(p, shared, chained, stream);
    }
}

cudaError_t take_la_parts_error(int* flag) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_la_parts_error, sizeof(int));
    if (e != cudaSuccess || *flag == 0) return e;
    const int zero = 0;
    return cudaMemcpyToSymbol(g_la_parts_error, &zero, sizeof(int));
}

}  // namespace gdr
