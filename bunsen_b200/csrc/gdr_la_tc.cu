// The decayed linear attention core (gdr_la.cuh) on the tensor cores: bf16
// operands, d_b and d_c up to 128 (multiples of 8), f32 states.
//
// Per (sequence, head) the positions go in chunks of C = 128 (forward in time;
// the mirror image backward), S the state before the chunk, i, j in the chunk:
//   out_i = tau [ w^{i+1} a_i . S + sum_{j<=i} sigma w^{i-j} (a_i.b_j) c_j ]
//   S'    = w^C S + sum_j sigma w^{C-1-j} b_j c_j^T.
// Every decay is a power with a non-negative exponent, so none overflows; w^0
// is 1 for any decay, minus infinity included.
//
// One CTA per SM, persistent over (sequence, head) items, warp-specialised, so
// that the loads, the matrix products and the conversions of consecutive
// chunks run beside one another:
//   warps 0-7    scores -> decayed bf16 P; outputs (scaled, converted, staged)
//   warps 8-15   the state, f32 in registers (64 values a thread): adds a
//                chunk's update, writes the bf16 copy; initial and final states
//   warps 16-23  the update's operand, c scaled by w^{C-1-j}
//   warp 24      TMA loads of the a, b, c tiles, two stages of 96 KiB
//   warp 25      issues the products of the outputs
//   warp 26      issues the products of the update
//   warp 27      TMA stores of the outputs (stored from registers, 32 bytes of 32
//                rows at a time, they kept the load-store unit busy for 2000
//                cycles a chunk)
// The products of a chunk, M = N = 128 each, f32 accumulators in TMEM:
//   scores = A B^T              both from shared memory
//   O      = A Sb               Sb the state's bf16 copy (K-major rows of c)
//   O     += P C                P from TMEM, C read MN-major
//   U^T    = (w c)^T B          (w c)^T from TMEM, B read MN-major
// TMEM (512 columns): U^T 128, scores with P over them 128, O 128, (w c)^T two
// buffers of 48 (32 positions in three parts).
// Two issuing warps, because a wait and a commit cost their thread 100 to 200
// cycles each beside products that keep shared memory busy, 17 of them a
// chunk; the state in registers rather than scaled in TMEM, because there the
// next update waited for the scaling (5.4 us a chunk with one issuer and the
// state in TMEM, 3.7 us so).
//
// What is rounded: P and Sb to bf16 (2^-8 relative each, on disjoint parts of
// an output, which is itself rounded to bf16: inputs are bf16, so another
// half-step of theirs; a second part of either would be a product more, 32 KiB of
// shared memory that is not there, and a third less error). The state accumulates
// in f32 over every chunk, so its operand is not rounded: w c goes in as three bf16
// parts, 24 bits. Measured against 64 bits: outputs 2.3e-3 (a bf16 rounding alone:
// 1.7e-3), states 3.2e-7.
//
// Jobs come from a list, the longest first, handed out by a counter; long sequences
// go in segments whose states a pass of their own finds (kStateOnly: loads, (w c)^T and
// the update alone; gdr_la_plan.cu).
//
// Bound: HBM, at 128 x (768 to 1024) bytes a chunk and head (q and k shared or not),
// 2.2 to 3.0 us per SM at the measured copy rate; six products are 3100 tensor cycles, 1.8 us;
// shared memory moves 480 KiB a chunk, 3800 cycles. A chunk takes 3.8 us (131072
// packed positions, 32 heads: 852 us, 4.1 TB/s, 0.63 of the copy rate, one call at a
// time; 1049 us, 0.51, among other calls, at lower clocks): the chains between the roles,
// 250 cycles from a commit to the waiting warp's next instruction, are what is left. The
// states' pass takes 1.7 to 2 us a chunk.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "gdr_la.cuh"
#include "gdr_la_plan.cuh"
#include "gdr_la_sm100.cuh"

namespace gdr {

// Device-side failures since the last gdr_device_error: bit 0, a bounded wait
// ran out.
__device__ int g_la_error;

namespace {

using namespace sm100;

constexpr int kC = kLaChunk, kD = 128;
constexpr int kThreads = 896;
constexpr uint32_t kTile = 32768;         // 128 positions x 128 bf16, two 64-wide halves
constexpr uint32_t kHalf = kTile / 2;
constexpr uint32_t kStage = 3 * kTile;    // a, b, c
constexpr uint32_t kOffSb = 2 * kStage, kOffMisc = kOffSb + kTile;
constexpr uint32_t kSmemBytes = kOffMisc + 512;
constexpr uint32_t kColU = 0, kColP = 128, kColO = 256, kColWBuf = 48;


// What a CTA works on next: the positions [start, start + len) of a sequence with
// head h, from state `in` to state `out` (see la_state); len < 0: nothing more.
struct Job {
    int start, len, h, in, out;
};
constexpr int kJobs = 4;  // in flight between the loading warp and the other roles

constexpr int kRingMost = 8;

struct Bars {
    uint64_t a_full[2], b_full[2], c_full[2], a_free[2], c_read[2], o_staged[2];
    uint64_t in_full[2], o_full[2], u_full[2];
    uint64_t sc_full, pa_ready, sb_ready, o_free, u_free, fix[2], drain[2];
    uint64_t wv_full[kRingMost], wv_free[kRingMost];
    uint64_t job_full[kJobs], job_free[kJobs];
    uint32_t tmem;
    Job jobs[kJobs];
};

// Where the x-th 128 bytes of the features of a stage's outputs are staged: the
// a tile's halves, f32 outputs in the c tile's too.
__device__ __forceinline__ uint8_t* staged(uint8_t* stage, int x) {
    return stage + (x >> 1) * 2 * kTile + (x & 1) * kHalf;
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0,
                                             int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
        " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
        "r"(v[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint64_t (&v)[8]) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[2 * i] = static_cast<uint32_t>(v[i]);
        r[2 * i + 1] = static_cast<uint32_t>(v[i] >> 32);
    }
    tmem_st16(taddr, r);
}

// 16 lanes x 16 columns: thread t's register 2 i holds lane t / 4, column 4 i +
// t % 4, and register 2 i + 1 the lane 8 below it.
__device__ __forceinline__ void tmem_st_16x128(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
        : "memory");
}

// The products of a chunk, 128 x 128 each, issued by one elected thread. The
// operands' addresses step inside the assembly, which takes four instructions a
// product; stepped outside, or in a branch on the stage, two to four times that.

// D = A B over 128 of K: both K-major in shared memory (two 64-wide halves).
__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, 0, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "mov.b64 a, %1;\n\tmov.b64 b, %2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 1018;\n\tadd.s64 b, b, 1018;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
        "}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc)
        : "memory");
}
// D += A B over 128 of K: A in TMEM (its rows the lanes; the second half 64
// columns from the first), B MN-major.
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred t;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\t"
        "setp.eq.b32 t, 0, 0;\n\tmov.b32 a, %1;\n\tmov.b64 b, %2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 40;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 8;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc)
        : "memory");
}
// D = (or +=) (A1 + A2 + A3) B over 32 of K: the parts 16 columns apart in TMEM.
__device__ __forceinline__ void product_ts3(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tmov.b32 a, %1;\n\tmov.b64 b, %2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p;\n\t"
        "add.u32 a, a, 16;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 16;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "sub.u32 a, a, 24;\n\tadd.s64 b, b, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 16;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "add.u32 a, a, 16;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
        "}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The n lowest bits (all 32 from n = 32 on).
__device__ __forceinline__ uint32_t low_bits(uint32_t n) {
    uint32_t r;
    asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(r) : "r"(n));
    return r;
}

// Moves registers between the roles: the launch gives each thread 72, 504 for
// the seven warpgroups' lanes together: 2 x 72 + 2 x 96 + 2 x 64 + 40, and in the
// states' pass 2 x 24 + 2 x 104 + 2 x 96 + 40.
template <int kRegs>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Chunk c of an item, in the order they run: its length, and its first row.
template <bool kRev>
__device__ __forceinline__ int chunk_len(const Job& it, int nch, int c) {
    return min(kC, it.len - (kRev ? nch - 1 - c : c) * kC);
}
template <bool kRev>
__device__ __forceinline__ void chunk_of(const Job& it, int nch, int c,
                                         int64_t& row, int& len) {
    const int x = kRev ? nch - 1 - c : c;
    row = static_cast<int64_t>(it.start) + x * kC;
    len = min(kC, it.len - x * kC);
}

// kStateOnly: only the state after the positions is wanted (no a, no output).
template <bool kRev, bool kStateOnly>
__global__ void __launch_bounds__(kThreads, 1)
la_tc(const LaCore p, const __grid_constant__ CUtensorMap ma,
      const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap mc,
      const __grid_constant__ CUtensorMap mo, LaWork* work, const LaEntry* entries, float* scratch) {
    extern __shared__ __align__(1024) uint8_t sm[];  // (checked below: swizzled tiles need it)
    Bars& B = *reinterpret_cast<Bars*>(sm + kOffMisc);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.a_full[i], 1);
            mbar_init(&B.b_full[i], 1);
            mbar_init(&B.a_free[i], 1);
            mbar_init(&B.o_staged[i], 8);
            mbar_init(&B.c_full[i], 1);
            mbar_init(&B.c_read[i], 8);
            mbar_init(&B.in_full[i], 1);
            mbar_init(&B.o_full[i], 1);
            mbar_init(&B.u_full[i], 1);
            mbar_init(&B.fix[i], 8);
            mbar_init(&B.drain[i], 1);
        }
        for (int i = 0; i < kRingMost; ++i) {
            mbar_init(&B.wv_full[i], 8);
            mbar_init(&B.wv_free[i], 1);
        }
        for (int i = 0; i < kJobs; ++i) {
            mbar_init(&B.job_full[i], 1);
            mbar_init(&B.job_free[i], kStateOnly ? 17 : 27);  // every warp that reads it
        }
        mbar_init(&B.sc_full, 1);
        mbar_init(&B.pa_ready, 8);
        mbar_init(&B.o_free, 8);
        mbar_init(&B.sb_ready, 8);
        mbar_init(&B.u_free, 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 26) {
        tmem_alloc(&B.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    after_last_kernel();
    __syncthreads();
    tc_fence_after();
    bool ok = true;  // false: a wait ran out, and its role with it
    // All 512 columns are this CTA's, so they begin at 0: a constant, as the
    // tiles' addresses are, keeps the products' operands in uniform registers.
    constexpr uint32_t tm = 0;
    // Buffers of (w c)^T: the room beside U^T, or what the scores and O leave.
    constexpr uint32_t kRing = kStateOnly ? kRingMost : 2, kColW = kStateOnly ? 128 : 384;
    if (B.tmem != 0 || (smem_u32(sm) & 1023) != 0) ok = false;  // never: nothing would be right
    // The job of a slot that is full, and the slot given back (its warp converged).
    auto take = [&](uint32_t slot) {
        const Job j = B.jobs[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.job_free[slot]);
        return j;
    };
    const uint32_t quad = tm + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's lanes

    if (warp >= 24) {
        give_registers<40>();
        if (warp == 24) {
            // ---- loads -------------------------------------------------------------
            {
                uint32_t n = 0;
                const int heads = p.heads;
                const int jobs = work != nullptr ? work->count * heads : p.n_seqs * heads;
#pragma unroll 1
                for (uint32_t k = 0; ok; ++k) {
                    const uint32_t slot = k % kJobs;
                    if (k >= kJobs && !(ok = warp_wait(&B.job_free[slot], (k / kJobs & 1) ^ 1))) break;
                    int id = k == 0 ? static_cast<int>(blockIdx.x) : jobs;
                    if (work != nullptr && k > 0) {
                        if (lane == 0) id = atomicAdd(&work->next, 1);
                        id = __shfl_sync(0xffffffffu, id, 0);
                    }
                    Job it{0, -1, 0, -1, -1};
                    if (id < jobs) {
                        const int e = id / heads;
                        it.h = id - e * heads;
                        if (work != nullptr) {
                            const LaEntry x = entries[e];
                            it.start = x.start, it.len = x.len, it.in = x.in, it.out = x.out;
                        } else {
                            int64_t start, end;
                            la_span(p, e, start, end);
                            it.start = static_cast<int>(start);
                            it.len = static_cast<int>(end - start);
                            it.in = it.out = e;
                        }
                    }
                    if (lane == 0) {
                        B.jobs[slot] = it;
                        mbar_arrive(&B.job_full[slot]);
                    }
                    __syncwarp();
                    if (it.len < 0) break;
                    const int nch = (it.len + kC - 1) / kC;
                    const int ha = it.h / (p.heads / p.heads_a), hb = it.h / (p.heads / p.heads_b),
                              hc = it.h / (p.heads / p.heads_c);
#pragma unroll 1
                    for (int c = 0; ok && c < nch; ++c, ++n) {
                        const int st = n & 1;
                        const uint32_t ph = ((n >> 1) & 1) ^ 1;
                        int64_t row;
                        int len;
                        chunk_of<kRev>(it, nch, c, row, len);
                        const int r = static_cast<int>(row);
                        uint8_t* base = sm + st * kStage;
                        auto load = [&](uint64_t* full, uint8_t* dst, const CUtensorMap* map,
                                        int head) {
                            if (elect_one()) {
                                mbar_expect_tx(full, kTile);
                                tma_load_3d(dst, map, full, 0, head, r);
                                tma_load_3d(dst + kHalf, map, full, 64, head, r);
                            }
                        };
                        // Chunk n - 2: its products with b and with c are done, its operand's
                        // warps have read c, and its output has left the tiles.
                        if (!kStateOnly && n >= 2 && !(ok = warp_wait(&B.in_full[st], ph))) break;
                        if (n >= 2 && !(ok = warp_wait(&B.u_full[st], ph))) break;
                        load(&B.b_full[st], base + kTile, &mb, hb);
                        if (!kStateOnly && n >= 2) {
                            if (p.out_f32 && !(ok = warp_wait(&B.a_free[st], ph))) break;
                            if (!(ok = warp_wait(&B.o_full[st], ph))) break;
                        }
                        if (n >= 2 && !(ok = warp_wait(&B.c_read[st], ph))) break;
                        load(&B.c_full[st], base + 2 * kTile, &mc, hc);
                        if (kStateOnly) continue;
                        if (n >= 2 && !(ok = warp_wait(&B.a_free[st], ph))) break;
                        load(&B.a_full[st], base, &ma, ha);
                    }
                }
                // Nothing of this CTA's may be in flight when it ends.
#pragma unroll 1
                for (uint32_t i = n >= 2 ? n - 2 : 0; i < n + (ok ? 0 : 1); ++i)
                    for (uint64_t* full : {B.b_full, B.c_full, kStateOnly ? B.b_full : B.a_full})
                        warp_wait(&full[i & 1], (i >> 1) & 1);
            }
            __syncwarp();
        } else if (!kStateOnly && warp == 25) {
            // ---- the outputs' products -------------------------------------------------
            {
                constexpr uint32_t kKK = idesc_bf16(128, 128, 0, 0, 0);
                constexpr uint32_t kKMn = idesc_bf16(128, 128, 0, 1, 0);
                const uint32_t base = smem_u32(sm);
                auto from_a = [&](uint32_t st, uint32_t d, uint32_t b_tile) {
                    product_ss(tm + d, sdesc_sw128(base + st * kStage, 16, 1024),
                               sdesc_sw128(b_tile, 16, 1024), kKK);
                };
                auto from_p = [&](uint32_t st) {
                    product_ts(tm + kColO, tm + kColP,
                               sdesc_sw128(base + st * kStage + 2 * kTile, kHalf, 1024), kKMn);
                };
                uint32_t n = 0, tails = 0;
#pragma unroll 1
                for (uint32_t k = 0; ok; ++k) {
                    if (!(ok = warp_wait(&B.job_full[k % kJobs], k / kJobs & 1))) break;
                    const Job it = take(k % kJobs);
                    if (it.len < 0) break;
                    const int nch = (it.len + kC - 1) / kC;
#pragma unroll 1
                    for (int c = 0; c < nch; ++c, ++n) {
                        const uint32_t st = n & 1, ph = n & 1;
                        if (!(ok = warp_wait(&B.b_full[st], (n >> 1) & 1))) break;
                        if (!(ok = warp_wait(&B.a_full[st], (n >> 1) & 1))) break;
                        if (chunk_len<kRev>(it, nch, c) < kC) {  // (by stage: bits of `tails`)
                            if (!(ok = warp_wait(&B.fix[st], (tails >> st) & 1))) break;
                            tails ^= 1u << st;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            from_a(st, kColP, base + st * kStage + kTile);
                            umma_commit(&B.sc_full);
                        }
                        if (!(ok = warp_wait(&B.sb_ready, ph))) break;
                        if (n > 0 && !(ok = warp_wait(&B.o_free, ph ^ 1))) break;
                        tc_fence_after();
                        if (elect_one()) {
                            from_a(st, kColO, base + kOffSb);
                            umma_commit(&B.in_full[st]);
                        }
                        // (P is written, and the c tile is there: its warps waited for it.)
                        if (!(ok = warp_wait(&B.pa_ready, ph))) break;
                        tc_fence_after();
                        if (elect_one()) {
                            from_p(st);
                            umma_commit(&B.o_full[st]);
                        }
                    }
                }
                if (elect_one()) umma_commit(&B.drain[0]);
                warp_wait(&B.drain[0], 0);
            }
            __syncwarp();
        } else if (warp == 26) {
            // ---- the update's products -------------------------------------------------
            {
                constexpr uint32_t kKMn = idesc_bf16(128, 128, 0, 1, 0);
                const uint32_t base = smem_u32(sm);
                auto update = [&](uint32_t st, uint32_t q, uint32_t buf) {  // 32 positions
                    product_ts3(tm + kColU, tm + kColW + buf * kColWBuf,
                                sdesc_sw128(base + st * kStage + kTile + q * 4096, kHalf, 1024), kKMn,
                                q);
                };
                uint32_t n = 0, w = 0, tails = 0;
#pragma unroll 1
                for (uint32_t k = 0; ok; ++k) {
                    if (!(ok = warp_wait(&B.job_full[k % kJobs], k / kJobs & 1))) break;
                    const Job it = take(k % kJobs);
                    if (it.len < 0) break;
                    const int nch = (it.len + kC - 1) / kC;
#pragma unroll 1
                    for (int c = 0; c < nch; ++c, ++n) {
                        const uint32_t st = n & 1;
                        if (!(ok = warp_wait(&B.b_full[st], (n >> 1) & 1))) break;
                        if (chunk_len<kRev>(it, nch, c) < kC) {  // (by stage: bits of `tails`)
                            if (!(ok = warp_wait(&B.fix[st], (tails >> st) & 1))) break;
                            tails ^= 1u << st;
                        }
                        if (n > 0 && !(ok = warp_wait(&B.u_free, (n & 1) ^ 1))) break;
#pragma unroll 1
                        for (uint32_t q = 0; q < 4; ++q, ++w) {
                            const uint32_t buf = w % kRing;
                            if (!(ok = warp_wait(&B.wv_full[buf], w / kRing & 1))) break;
                            tc_fence_after();
                            if (elect_one()) {
                                update(st, q, buf);
                                umma_commit(&B.wv_free[buf]);
                                if (q == 3) umma_commit(&B.u_full[st]);
                            }
                        }
                        if (!ok) break;
                    }
                }
                if (elect_one()) umma_commit(&B.drain[1]);
                warp_wait(&B.drain[1], 0);
            }
            __syncwarp();
        } else if (!kStateOnly && warp == 27) {
            // ---- the outputs' stores -----------------------------------------------------
            uint32_t n = 0;
#pragma unroll 1
            for (uint32_t k = 0; ok; ++k) {
                if (!(ok = warp_wait(&B.job_full[k % kJobs], k / kJobs & 1))) break;
                const Job it = take(k % kJobs);
                if (it.len < 0) break;
                const int nch = (it.len + kC - 1) / kC;
#pragma unroll 1
                for (int c = 0; c < nch; ++c, ++n) {
                    const uint32_t st = n & 1;
                    int64_t row;
                    int len;
                    chunk_of<kRev>(it, nch, c, row, len);
                    if (!(ok = warp_wait(&B.o_staged[st], (n >> 1) & 1))) break;
                    uint8_t* tile = sm + st * kStage;
                    // Boxes of 32 positions, 128 bytes of features each; the last rows one
                    // by one: behind them another sequence's stay as they are.
                    const int whole = len & ~31, boxes = p.out_f32 ? 4 : 2, width = p.out_f32 ? 32 : 64;
                    if (lane == 0) {
#pragma unroll 1
                        for (int x = 0; x < boxes && x * width < p.d_c; ++x)
#pragma unroll 1
                            for (int r = 0; r < whole; r += 32)
                                tma_store_3d(&mo, staged(tile, x) + r * 128, x * width, it.h,
                                             static_cast<int>(row) + r);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    const int piece = p.out_f32 ? 4 : 8;  // features in 16 bytes
                    uint8_t* out = static_cast<uint8_t*>(p.out);
#pragma unroll 1
                    for (int r = whole; r < len; ++r) {
                        const int64_t at = ((row + r) * p.heads + it.h) * p.d_c + lane * piece;
                        if (lane * piece < p.d_c)
                            *reinterpret_cast<uint4*>(out + at * (16 / piece)) =
                                *reinterpret_cast<const uint4*>(staged(tile, lane >> 3) + r * 128 +
                                                                (((lane & 7) ^ (r & 7)) << 4));
                    }
                    fence_proxy_async();  // the tile's next writer is the async proxy
                    __syncwarp();
                    if (lane == 0) {
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        mbar_arrive(&B.a_free[st]);
                    }
                }
            }
            if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            __syncwarp();
        }
    } else if (warp < 8) {
        if constexpr (kStateOnly) give_registers<24>();
        // ---- scores and outputs -------------------------------------------------------
        // Scores are scaled by w^{i-j} and the inter product, before P C is added to it, by
        // rows: a pass over O, but every factor is at most 1, so nothing overflows that
        // the result does not. (With the powers out of the sums, w^{-(j+1)} on the scores'
        // columns and w^{i+1} on O's rows at its end, scores above 2e16 did at a log decay of
        // -0.4; the 131072 packed positions took 814 us so, 852 us now.)
        // A block's 32 column factors run from the largest exponent down by
        // products with w^2 in registers: a table in shared memory waits there
        // behind the tensor cores' operands.
        // Two warps share 32 rows: of the scores blocks 0, 1 and 2, 3 (P goes over the
        // first scores of either pair), of the outputs 64 features each.
        const int quarter = warp & 3, half = warp >> 2, i = 32 * quarter + lane;
        // This warp's blocks that the mask leaves: [first, last).
        const int first = kRev ? max(2 * half, quarter) : 2 * half;
        const int last = kRev ? 2 * half + 2 : min(2 * half + 2, quarter + 1);
        const uint32_t pcol = quad + kColP + 64 * half;  // P's and the scores' columns
        uint32_t n = 0;
#pragma unroll 1
        for (uint32_t k = 0; !kStateOnly && ok; ++k) {
            if (!(ok = warp_wait(&B.job_full[k % kJobs], k / kJobs & 1))) break;
            const Job it = take(k % kJobs);
            if (it.len < 0) break;
            const int nch = (it.len + kC - 1) / kC;
            const float g = p.log_decay[it.h], w = la_power(g, 1);
            const uint64_t step = pair(w * w, w * w);
            const float w16 = la_power(g, 16);
            // Of the diagonal block, its half that is farther from the diagonal.
            const float steep = p.sigma * p.tau * la_power(g, kRev ? max(16 - lane, 0)
                                                                : max(lane - 15, 0));
            // Off the diagonal block: w^{i-j} splits in two exponents that are not
            // negative, rows' and columns'; the blocks' first column factors.
            const float edge = p.sigma * p.tau * la_power(g, kRev ? 32 - lane : lane + 1);
            float fb[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int cb = 2 * half + x, apart = kRev ? cb - quarter : quarter - cb;
                fb[x] = edge * la_power(g, 32 * (apart - 1));
            }
            float ahead = 0.f;  // O's row factor
            int known = 0;      // the chunk length it is for
#pragma unroll 1
            for (int c = 0; c < nch; ++c, ++n) {
                const uint32_t st = n & 1, ph = n & 1, ph2 = (n >> 1) & 1;
                const int len = chunk_len<kRev>(it, nch, c);
                if (len != known) {
                    ahead = p.tau * la_power(g, kRev ? max(len - 1 - i, 0) : i + 1);
                    known = len;
                }
                if (!(ok = warp_wait(&B.sc_full, ph))) break;
                tc_fence_after();
#pragma unroll 1
                for (int cb = first; cb < last; ++cb) {
#pragma unroll
                    for (int hb = 0; hb < 2; ++hb) {  // half blocks: 16 scores a thread
                        const int x = cb & 1;
                        const bool diag = cb == quarter;
                        uint64_t s[8];
                        tmem_ld16(pcol + 32 * x + 16 * hb, s);
                        uint32_t packed[8];
                        // The powers run from the larger exponents' side of either half.
                        const bool far = kRev ? hb == 1 : hb == 0;
                        const int me = lane - 16 * hb;  // this row's column in the half, if diag
                        if (!diag) {
                            float f = x == 0 ? fb[0] : fb[1];
                            if (far) f *= w16;
                            uint64_t f2 = kRev ? pair(f, f * w) : pair(f * w, f);
#pragma unroll
                            for (int t = 0; t < 8; ++t) {
                                const int j = kRev ? t : 7 - t;
                                packed[j] = pack_bf16(mul2(s[j], f2));
                                f2 = mul2(f2, step);
                            }
                        } else {
                            float f = far ? steep : p.sigma * p.tau;
#pragma unroll
                            for (int t = 0; t < 8; ++t) {
                                const int j = kRev ? t : 7 - t;
                                float u, v;
                                unpair(s[j], u, v);
                                (kRev ? u : v) *= f;
                                if (kRev ? 2 * j >= me : 2 * j + 1 <= me) f *= w;
                                (kRev ? v : u) *= f;
                                if (kRev ? 2 * j + 1 >= me : 2 * j <= me) f *= w;
                                packed[j] = pack_bf16(u, v);
                            }
                        }
                        if (diag) {  // j <= i, or j >= i
                            const int edge16 = 16 * (kRev ? me : me + 1);  // bits kept, or not
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t low = low_bits(max(edge16 - 32 * j, 0));
                                packed[j] &= kRev ? ~low : low;
                            }
                        }
                        tmem_st8(pcol + 16 * x + 8 * hb, packed);
                    }
                }
                uint32_t zero[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) zero[j] = 0;
#pragma unroll 1
                for (int cb = 2 * half; cb < 2 * half + 2; ++cb)
                    if (cb < first || cb >= last) tmem_st16(pcol + 16 * (cb & 1), zero);
                if (!(ok = warp_wait(&B.in_full[st], ph2))) break;
                tc_fence_after();
#pragma unroll 1
                for (int blk = 0; blk < 4; ++blk) {
                    const uint32_t at = quad + kColO + 64 * half + 16 * blk;
                    uint64_t o[8];
                    tmem_ld16(at, o);
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] = mul2(o[j], pair(ahead, ahead));
                    tmem_st16(at, o);
                }
                if (!(ok = warp_wait(&B.c_full[st], ph2))) break;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.pa_ready);

                // The output: converted, staged where a was (f32: and c).
                if (!(ok = warp_wait(&B.o_full[st], ph2))) break;
                if (p.out_f32 && !(ok = warp_wait(&B.c_read[st], ph2))) break;
                tc_fence_after();
                uint8_t* tile = sm + st * kStage;
#pragma unroll 1
                for (int blk = 0; blk < 4; ++blk) {
                    uint64_t u[8];
                    tmem_ld16(quad + kColO + 64 * half + 16 * blk, u);
                    if (blk == 3) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&B.o_free);
                    }
                    if (p.out_f32) {
                        uint8_t* dst = staged(tile, 2 * half + (blk >> 1)) + i * 128;
#pragma unroll
                        for (int m = 0; m < 4; ++m)
                            *reinterpret_cast<ulonglong2*>(
                                dst + ((((blk & 1) * 4 + m) ^ (i & 7)) << 4)) =
                                make_ulonglong2(u[2 * m], u[2 * m + 1]);
                    } else {
                        uint8_t* dst = staged(tile, half) + i * 128;
#pragma unroll
                        for (int m = 0; m < 2; ++m)
                            *reinterpret_cast<uint4*>(dst + (((blk * 2 + m) ^ (i & 7)) << 4)) =
                                make_uint4(pack_bf16(u[4 * m]), pack_bf16(u[4 * m + 1]),
                                           pack_bf16(u[4 * m + 2]), pack_bf16(u[4 * m + 3]));
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.o_staged[st]);
            }
        }
    } else if (warp < 16) {
        take_registers<kStateOnly ? 104 : 96>();
        // ---- the state -----------------------------------------------------------
        const int col = 32 * (warp & 3) + lane;  // this thread's column of S (row of U^T),
        const int half = (warp - 8) >> 2, b0 = 64 * half;  // and its rows b0 .. b0 + 63
        // Its row of Sb: 16 bytes at x are at (row's first) ^ x.
        const uint32_t sb =
            smem_u32(sm + kOffSb) + half * kHalf + col * 128 + ((col & 7) << 4);
        uint32_t n = 0;  // chunks begun
        uint64_t s[32];  // pairs of its rows
#pragma unroll 1
        for (uint32_t k = 0; ok; ++k) {
            if (!(ok = warp_wait(&B.job_full[k % kJobs], k / kJobs & 1))) break;
            const Job it = take(k % kJobs);
            if (it.len < 0) break;
            const int nch = (it.len + kC - 1) / kC;
            const float g = p.log_decay[it.h];
            const bool mine = col < p.d_c;
            {
                const LaState in = la_state(p, it.in, it.h, p.state_in, scratch);
                if (in.ptr != nullptr && mine) {
                    const float* src = in.ptr + col * in.col + b0 * in.row;
#pragma unroll
                    for (int j = 0; j < 32; ++j, src += 2 * in.row)
                        s[j] = pair(b0 + 2 * j < p.d_b ? src[0] : 0.f,
                                    b0 + 2 * j + 1 < p.d_b ? src[in.row] : 0.f);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] = 0;
                }
            }
            uint64_t hi2 = 0, lo2 = 0;  // w^len in two parts: it is applied chunk after chunk
            int known = 0;
#pragma unroll 1
            for (int c = 0; c < nch; ++c, ++n) {
                if constexpr (!kStateOnly) {
                    // The bf16 copy, once the last chunk's product has read its own.
                    if (n > 0 && !(ok = warp_wait(&B.in_full[(n - 1) & 1], ((n - 1) >> 1) & 1))) break;
                    uint32_t to = sb;
                    asm volatile("" : "+r"(to));  // (eight addresses kept would be registers)
#pragma unroll
                    for (int m = 0; m < 8; ++m)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to ^ (m << 4)),
                                     "r"(pack_bf16(s[4 * m])), "r"(pack_bf16(s[4 * m + 1])),
                                     "r"(pack_bf16(s[4 * m + 2])), "r"(pack_bf16(s[4 * m + 3]))
                                     : "memory");
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.sb_ready);
                }
                const int len = chunk_len<kRev>(it, nch, c);
                if (len != known) {
                    const float2 f = la_power2(g, len);
                    hi2 = pair(f.x, f.x);
                    lo2 = pair(f.y, f.y);
                    known = len;
                }
                if (!(ok = warp_wait(&B.u_full[n & 1], (n >> 1) & 1))) break;
                tc_fence_after();
#pragma unroll
                for (int blk = 0; blk < 8; ++blk) {
                    uint64_t u[4];
                    tmem_ld8(quad + kColU + b0 + 8 * blk, u);
                    if (blk == 7) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&B.u_free);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[4 * blk + j] = fma2(s[4 * blk + j], hi2, fma2(s[4 * blk + j], lo2, u[j]));
                }
            }
            const LaState out = la_state(p, it.out, it.h, p.state_out, scratch);
            if (ok && out.ptr != nullptr && mine) {
                float* dst = const_cast<float*>(out.ptr) + col * out.col + b0 * out.row;
#pragma unroll
                for (int m = 0; m < 8; ++m) {  // (d_b is a multiple of 8)
                    if (b0 + 8 * m >= p.d_b) break;
#pragma unroll
                    for (int j = 4 * m; j < 4 * m + 4; ++j, dst += 2 * out.row)
                        unpair(s[j], dst[0], dst[out.row]);
                }
            }
        }
    } else {
        if constexpr (kStateOnly) take_registers<96>();
        else give_registers<64>();
        // ---- the update's operand ----------------------------------------------------
        // (w c)^T, features on the TMEM lanes: 8 x 8 blocks of the c tile come
        // transposed from ldmatrix, thread t holding feature t / 4 (and + 8)
        // at positions 2 (t % 4), + 1 of each 8, which is where tcgen05.st's
        // 16x128b shape puts them; a thread's weights stay in registers.
        const int wc = warp & 3, half = (warp - 16) >> 2;  // 32 features, 16 of them
        const int row = ((lane >> 4) << 3) + (lane & 7);  // ldmatrix row of this lane
        const uint32_t src0 = smem_u32(sm) + 2 * kTile + (wc >> 1) * kHalf + row * 128;
        const int chunk0 = 4 * (wc & 1) + 2 * half + ((lane >> 3) & 1);
        const uint64_t minus = pair(-1.f, -1.f);
        uint32_t n = 0, w = 0;
#pragma unroll 1
        for (uint32_t k = 0; ok; ++k) {
            if (!(ok = warp_wait(&B.job_full[k % kJobs], k / kJobs & 1))) break;
            const Job it = take(k % kJobs);
            if (it.len < 0) break;
            const int nch = (it.len + kC - 1) / kC;
            const float g = p.log_decay[it.h];
            // Of position j = 32 q + jj, jj = 8 k + 2 (t % 4) + e, in a whole chunk:
            // w^(127 - j) = w^(96 - 32 q) w^(31 - jj), backward w^(32 q) w^(jj + 1).
            const int j0 = 2 * (lane & 3);
            const float mine = la_power(g, lane);  // w^lane, for the other lanes
            auto small = [&](int n) { return __shfl_sync(0xffffffffu, mine, n & 31); };
            uint64_t wt[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = 8 * k + j0;
                wt[k] = kRev ? pair(small(j) * small(1), small(j + 1) * small(1))
                             : pair(small(31 - j), small(30 - j));
            }
            const float w32 = la_power(g, 32), w64 = la_power(g, 64), w96 = la_power(g, 96);
#pragma unroll 1
            for (int c = 0; c < nch; ++c, ++n) {
                const int st = n & 1;
                const int len = chunk_len<kRev>(it, nch, c);
                if (!(ok = warp_wait(&B.c_full[st], (n >> 1) & 1))) break;
                if (len < kC) {
                    if (!(ok = warp_wait(&B.b_full[st], (n >> 1) & 1))) break;
                    // The rows past the sequence hold another's (or anything):
                    // zeros, so that no product of theirs is NaN.
                    uint8_t* bt = sm + st * kStage + kTile;
                    uint8_t* tile = lane < 16 ? bt : bt + kTile;
#pragma unroll 1
                    for (int r = len + warp - 16; r < kC; r += 8)
                        *reinterpret_cast<uint4*>(tile + ((lane & 15) >> 3) * kHalf + r * 128 +
                                                  (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.fix[st]);
                }
                // A quarter's values; in the states' pass, which has registers for them,
                // the next one's on their way.
                auto fetch = [&](int q, uint32_t (&x)[8]) {
#pragma unroll
                    for (int g2 = 0; g2 < 2; ++g2)
                        asm volatile(
                            "ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16"
                            " {%0, %1, %2, %3}, [%4];"
                            : "=r"(x[4 * g2]), "=r"(x[4 * g2 + 1]), "=r"(x[4 * g2 + 2]),
                              "=r"(x[4 * g2 + 3])
                            : "r"(src0 + st * kStage + (32 * q + 16 * g2) * 128 +
                                  ((chunk0 ^ (lane & 7)) << 4))
                            : "memory");
                };
                uint32_t next[8];
                if constexpr (kStateOnly) fetch(0, next);
#pragma unroll 1
                for (int q = 0; q < 4; ++q, ++w) {
                    const uint32_t buf = w % kRing;
                    uint32_t x[8];
                    if constexpr (kStateOnly) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = next[i];
                        if (q < 3) fetch(q + 1, next);
                    } else {
                        fetch(q, x);
                    }
                    if (q == 3) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&B.c_read[st]);
                    }
                    uint64_t f[4];
                    if (len == kC) {
                        const int e = kRev ? q : 3 - q;
                        const float base =
                            p.sigma * (e == 0 ? 1.f : e == 1 ? w32 : e == 2 ? w64 : w96);
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[k] = mul2(wt[k], pair(base, base));
                    } else {
                        // A short chunk: its own powers, nothing past its end
                        // (where another sequence's values may be).
                        const int live = len - 32 * q;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int j = 8 * k + j0;
                            float v[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                // w^(32 m + rest), the rest from its lane.
                                const int n = kRev ? 32 * q + j + e : max(live - 1 - j - e, 0);
                                const int m = n >> 5;
                                v[e] = p.sigma * small(n) * (kRev ? small(1) : 1.f) *
                                       (m == 0 ? 1.f : m == 1 ? w32 : m == 2 ? w64 : w96);
                            }
                            f[k] = pair(v[0], v[1]);
                            const uint32_t keep =
                                (j < live ? 0xffffu : 0u) | (j + 1 < live ? 0xffff0000u : 0u);
                            x[2 * k] &= keep;
                            x[2 * k + 1] &= keep;
                        }
                    }
                    if (w >= kRing &&
                        !(ok = warp_wait(&B.wv_free[buf], (w / kRing & 1) ^ 1)))
                        break;
                    tc_fence_after();
                    uint32_t mid[8], lo[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint64_t v = mul2(widen(x[k]), f[k >> 1]);
                        x[k] = pack_bf16(v);
                        v = fma2(widen(x[k]), minus, v);
                        mid[k] = pack_bf16(v);
                        lo[k] = pack_bf16(fma2(widen(mid[k]), minus, v));
                    }
                    const uint32_t at =
                        quad + (static_cast<uint32_t>(half) << 20) + kColW + buf * kColWBuf;
                    tmem_st_16x128(at, x);
                    tmem_st_16x128(at + 16, mid);
                    tmem_st_16x128(at + 32, lo);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.wv_full[buf]);
                }
                if (!ok) break;
            }
        }
    }
    if (!ok && lane == 0) atomicOr(&g_la_error, 1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 26) tmem_dealloc(B.tmem, 512);
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            ptr = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    }();
    return fn;
}

// [tokens, heads, d] bf16 or f32 in boxes of 128 bytes of features x 1 head x
// `rows` positions; features past d read as zeros and are not written.
bool tile_map(CUtensorMap* map, const void* base, int64_t tokens, int heads, int d, int rows,
              bool f32 = false) {
    auto encode = encoder();
    if (encode == nullptr) return false;
    const cuuint64_t es = f32 ? 4 : 2;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {d * es, static_cast<cuuint64_t>(heads) * d * es};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / es), 1,
                               static_cast<cuuint32_t>(rows)};
    const cuuint32_t estride[3] = {1, 1, 1};
    return encode(map,
                  f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                  const_cast<void*>(base), dims, strides, box, estride,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool la_tc_supports(const LaCore& p) {
    const uintptr_t align = reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) |
                            reinterpret_cast<uintptr_t>(p.c) | reinterpret_cast<uintptr_t>(p.out);
    return p.dtype == GDR_DTYPE_BF16 && p.d_b <= kD && p.d_c <= kD && p.d_b % 8 == 0 &&
           p.d_c % 8 == 0 && (align & 15) == 0 && la_tokens(p) > 0 &&
           la_tokens(p) < (int64_t{1} << 31) - 2 * kC &&
           static_cast<int64_t>(p.n_seqs) * p.heads < (int64_t{1} << 30);
}

cudaError_t launch_la_tc(const LaCore& p, bool split, bool must, int forced, cudaStream_t stream,
                         LaLists* shared, bool chained) {
    CUtensorMap ma, mb, mc, mo;
    const int64_t tokens = la_tokens(p);
    if (!tile_map(&ma, p.a, tokens, p.heads_a, p.d_b, kC) ||
        !tile_map(&mb, p.b, tokens, p.heads_b, p.d_b, kC) ||
        !tile_map(&mc, p.c, tokens, p.heads_c, p.d_c, kC) ||
        !tile_map(&mo, p.out, tokens, p.heads, p.d_c, 32, p.out_f32 != 0))
        return cudaErrorInvalidValue;
    auto* full = p.reverse ? la_tc<true, false> : la_tc<false, false>;
    auto* states = p.reverse ? la_tc<true, true> : la_tc<false, true>;
    static std::atomic<uint64_t> done[2][2];
    cudaError_t e = la_allow_smem(full, static_cast<int>(kSmemBytes), done[p.reverse != 0][0]);
    if (e == cudaSuccess)
        e = la_allow_smem(states, static_cast<int>(kSmemBytes), done[p.reverse != 0][1]);
    if (e != cudaSuccess) return e;
    // In chunks of the main pass, 3.8 us: one of the states' pass 0.45; that pass's start, the
    // list's kernel and the scan 11 (9 and 12 us the last two, cold).
    const int sms = la_sm_count();
    LaLists own;
    LaLists& lists = shared != nullptr ? *shared : own;
    if (lists.uses == 0) {
        e = la_prepare(p, sms, 1, {split, must, forced, 0.45f, 11.f}, shared != nullptr, chained,
                       lists, stream);
        if (e != cudaSuccess) return e;
        if (lists.split) {
            e = la_launch_next(states, sms, kThreads, static_cast<int>(kSmemBytes), stream, p, ma, mb,
                               mc, mo, &lists.plan->states, lists.states, lists.slots);
            if (e == cudaSuccess) e = la_scan_states(p, lists, stream);
        }
    }
    const int64_t jobs = static_cast<int64_t>(p.n_seqs) * p.heads;
    if (e == cudaSuccess && lists.plan != nullptr)
        e = la_launch_next(full, sms, kThreads, static_cast<int>(kSmemBytes), stream, p, ma, mb, mc,
                           mo, &lists.plan->main[lists.uses], lists.main, lists.slots);
    else if (e == cudaSuccess)
        full<<<static_cast<int>(jobs), kThreads, kSmemBytes, stream>>>(p, ma, mb, mc, mo, nullptr,
                                                                       nullptr, nullptr);
    ++lists.uses;
    if (e == cudaSuccess) e = cudaGetLastError();
    const cudaError_t f = la_release(own, stream);
    return e != cudaSuccess ? e : f;
}

cudaError_t take_la_error(int* flag) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_la_error, sizeof(int));
    if (e != cudaSuccess || *flag == 0) return e;
    const int zero = 0;
    return cudaMemcpyToSymbol(g_la_error, &zero, sizeof(int));
}

}  // namespace gdr
