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
//   warps 0-3    scores -> decayed bf16 P
//   warps 4-11   the state, f32 in registers (64 values a thread): adds a
//                chunk's update, writes the bf16 copy; initial and final states;
//                the output (scaled, converted, stored)
//   warps 12-15  the update's operand, c scaled by w^{C-1-j}
//   warp 16      TMA loads of the a, b, c tiles, two stages of 96 KiB
//   warp 17      issues the products of the outputs
//   warp 18      issues the products of the update
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
// next update waited for the scaling (4.0 us a chunk with one issuer and the
// state in TMEM, TIMEUS so).
//
// What is rounded: P and Sb to bf16 (2^-8 relative each, on disjoint parts of
// an output, which is itself rounded to bf16: inputs are bf16, so another
// half-step of theirs; f32 operands would halve the tensor rate for a third
// less error). The state accumulates in f32 over every chunk, so its operand
// is not rounded: w c goes in as three bf16 parts, 24 bits. Measured against
// 64 bits: outputs 2.3e-3 (a bf16 rounding alone: 1.7e-3), states below 1e-6.
//
// Bound: by HBM at 128 x (768 to 1024) bytes a chunk and head (q and k shared
// or not), 2.2 to 3.0 us per SM at the measured copy rate, against 6 products of
// 512 tensor cycles, 1.6 us.
#include <cudaTypedefs.h>

#include <algorithm>

#include "gdr_la.cuh"
#include "gdr_sm100.cuh"

namespace gdr {

// Device-side failures since the last gdr_device_error: bit 0, a bounded wait
// ran out.
__device__ int g_la_error;

namespace {

using namespace sm100;

constexpr int kC = 128, kD = 128;
constexpr int kThreads = 640;
constexpr uint32_t kTile = 32768;         // 128 positions x 128 bf16, two 64-wide halves
constexpr uint32_t kHalf = kTile / 2;
constexpr uint32_t kStage = 3 * kTile;    // a, b, c
constexpr uint32_t kOffSb = 2 * kStage, kOffMisc = kOffSb + kTile;
constexpr uint32_t kSmemBytes = kOffMisc + 512 + 1024;  // + alignment slack
constexpr uint32_t kColU = 0, kColP = 128, kColO = 256, kColW = 384, kColWBuf = 48;
constexpr int kWaitTries = 1 << 20;  // seconds

struct Bars {
    uint64_t a_full[2], b_full[2], c_full[2], a_free[2], b_free[2], c_free[2];
    uint64_t sc_full, in_full, o_full, o_free, pa_ready, sb_ready, u_full, u_free, fix[2], drain[2];
    uint64_t wv_full[2], wv_free[2];
    uint32_t tmem;
};

// One (sequence or segment, head) of a pass.
struct Item {
    int64_t start;
    int len, h;
    const float* in;  // state before it (null: zeros)
    float* out;       // state after it (null: not wanted)
    bool in_t, out_t;  // stored [d_c, d_b]
};

// Waits for a phase; false once the tries ran out, which is recorded. The
// hardware suspends a try for some microseconds, without issuing anything (a
// try with a time of its own became a loop of sleeps: a third of all
// instructions). Tries are counted rather than timed to keep the code small: six
// roles' loops share one instruction cache.
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < kWaitTries; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    atomicOr(&g_la_error, 1);
    return false;
}
// The same for a whole warp together: false for every lane.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, lane_wait(bar, parity));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
        : "memory");
}

// 32 lanes x 16 columns, as pairs of columns, arrived. (The loads take some 30
// cycles; several in flight gained nothing.)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint64_t (&v)[8]) {
    asm volatile(
        "{\n\t.reg .b32 r<16>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        " {r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {r0, r1};\n\tmov.b64 %1, {r2, r3};\n\t"
        "mov.b64 %2, {r4, r5};\n\tmov.b64 %3, {r6, r7};\n\t"
        "mov.b64 %4, {r8, r9};\n\tmov.b64 %5, {r10, r11};\n\t"
        "mov.b64 %6, {r12, r13};\n\tmov.b64 %7, {r14, r15};\n\t}"
        : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3]), "=l"(v[4]), "=l"(v[5]), "=l"(v[6]),
          "=l"(v[7])
        : "r"(taddr)
        : "memory");
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

// D[tmem] = A[tmem] B (+ D): A's rows are the lanes, K pairs its columns.
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Two f32 as bf16, x in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
__device__ __forceinline__ float low_f32(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_f32(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// Moves registers between the roles: the launch gives each thread 96, 480 for
// the five warpgroups' lanes together; 40 + 80 + 2 x 128 + 96 = 472 of them.
template <int kRegs>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Pairs of f32 in one 64-bit register: one instruction for two products or sums.
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(uint64_t p) {
    float x, y;
    unpair(p, x, y);
    return pack_bf16(x, y);
}
__device__ __forceinline__ uint64_t widen(uint32_t p) { return pair(low_f32(p), high_f32(p)); }

// w^n for 0 <= n <= 128, 1 for n = 0 (minus infinity included): the exponent's
// rounding error goes in as a factor, e^(p + d) = e^p (1 + d).
__device__ __forceinline__ float power(float g, int n) {
    if (n <= 0) return 1.f;
    const float p = g * n;
    if (p < -104.f) return 0.f;  // below the smallest f32
    const float e = expf(p);
    return fmaf(e, fmaf(g, static_cast<float>(n), -p), e);
}

// w^n in two parts, hi + lo.
__device__ __forceinline__ float2 power2(float g, int n) {
    const double f = exp(static_cast<double>(g) * n);
    const float hi = static_cast<float>(f);
    return make_float2(hi, static_cast<float>(f - hi));
}

// Heads whose decay's powers to w^-128 are far from overflow (e^51).
__device__ __forceinline__ bool is_gentle(float g) { return g >= -0.4f && g <= 0.4f; }

// tau times the decay of the state before the chunk at its row i.
template <bool kRev>
__device__ __forceinline__ float row_factor(const LaCore& p, float g, int len, int i) {
    return p.tau * power(g, kRev ? max(len - 1 - i, 0) : i + 1);
}

__device__ __forceinline__ Item item_of(const LaCore& p, int id) {
    Item it;
    const int s = id / p.heads;
    it.h = id - s * p.heads;
    int64_t end;
    la_span(p, s, it.start, end);
    it.len = static_cast<int>(end - it.start);
    const int64_t at = static_cast<int64_t>(id) * p.d_b * p.d_c;
    it.in = p.state_in != nullptr ? p.state_in + at : nullptr;
    it.out = p.state_out != nullptr ? p.state_out + at : nullptr;
    it.in_t = it.out_t = p.state_t != 0;
    return it;
}

// Chunk c of an item, in the order they run: its length, and its first row.
template <bool kRev>
__device__ __forceinline__ int chunk_len(const Item& it, int nch, int c) {
    return min(kC, it.len - (kRev ? nch - 1 - c : c) * kC);
}
template <bool kRev>
__device__ __forceinline__ void chunk_of(const Item& it, int nch, int c,
                                         int64_t& row, int& len) {
    const int x = kRev ? nch - 1 - c : c;
    row = it.start + static_cast<int64_t>(x) * kC;
    len = min(kC, it.len - x * kC);
}

template <bool kRev>
__global__ void __launch_bounds__(kThreads, 1)
la_tc(const LaCore p, const __grid_constant__ CUtensorMap ma,
      const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap mc, int items) {
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
    Bars& B = *reinterpret_cast<Bars*>(sm + kOffMisc);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.a_full[i], 1);
            mbar_init(&B.b_full[i], 1);
            mbar_init(&B.c_full[i], 1);
            mbar_init(&B.a_free[i], 1);
            mbar_init(&B.b_free[i], 1);
            mbar_init(&B.c_free[i], 5);  // its product's end, and the operand's warps
            mbar_init(&B.drain[i], 1);
            mbar_init(&B.fix[i], 4);
            mbar_init(&B.wv_full[i], 4);
            mbar_init(&B.wv_free[i], 1);
        }
        mbar_init(&B.sc_full, 1);
        mbar_init(&B.in_full, 1);
        mbar_init(&B.o_full, 1);
        mbar_init(&B.o_free, 8);
        mbar_init(&B.pa_ready, 4);
        mbar_init(&B.sb_ready, 8);
        mbar_init(&B.u_full, 1);
        mbar_init(&B.u_free, 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 18) {
        tmem_alloc(&B.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = B.tmem;
    const uint32_t quad = tm + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's lanes

    if (warp >= 16) {
        give_registers<40>();
    if (warp == 16) {
        // ---- loads -------------------------------------------------------------
        if (lane == 0) {
            uint32_t n = 0;
            bool ok = true;
#pragma unroll 1
            for (int id = blockIdx.x; ok && id < items; id += gridDim.x) {
                const Item it = item_of(p, id);
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
                    auto load = [&](uint64_t* full, uint64_t* free, uint8_t* dst,
                                    const CUtensorMap* map, int head) {
                        if (n >= 2 && !(ok = lane_wait(free, ph))) return;
                        mbar_expect_tx(full, kTile);
                        tma_load_3d(dst, map, full, 0, head, r);
                        tma_load_3d(dst + kHalf, map, full, 64, head, r);
                    };
                    // a is free after the scores' and the inter product, b then after
                    // the update's, c after P C and the operand's warps.
                    uint8_t* base = sm + st * kStage;
                    load(&B.a_full[st], &B.a_free[st], base, &ma, ha);
                    if (ok) load(&B.b_full[st], &B.b_free[st], base + kTile, &mb, hb);
                    if (ok) load(&B.c_full[st], &B.c_free[st], base + 2 * kTile, &mc, hc);
                    if (!ok) break;
                }
            }
            // Nothing of this CTA's may be in flight when it ends.
#pragma unroll 1
            for (uint32_t i = n >= 2 ? n - 2 : 0; i < n + (ok ? 0 : 1); ++i)
                for (uint64_t* full : {B.a_full, B.b_full, B.c_full})
                    lane_wait(&full[i & 1], (i >> 1) & 1);
        }
        __syncwarp();
    } else if (warp == 17) {
        // ---- the outputs' products -------------------------------------------------
        if (lane == 0) {
            constexpr uint32_t kKK = idesc_bf16(128, 128, 0, 0, 0);
            constexpr uint32_t kKMn = idesc_bf16(128, 128, 0, 1, 0);
            const uint64_t tile0 = sdesc_sw128(smem_u32(sm), 16, 1024);
            const uint64_t sb = sdesc_sw128(smem_u32(sm + kOffSb), 16, 1024);
            const uint64_t mn0 = sdesc_sw128(smem_u32(sm), kHalf, 1024);
            uint32_t n = 0, tails = 0;
            bool ok = true;
#pragma unroll 1
            for (int id = blockIdx.x; ok && id < items; id += gridDim.x) {
                const Item it = item_of(p, id);
                const int nch = (it.len + kC - 1) / kC;
#pragma unroll 1
                for (int c = 0; c < nch; ++c, ++n) {
                    const uint32_t st = n & 1, ph = n & 1;
                    const uint64_t a = tile0 + st * (kStage >> 4), bt = a + (kTile >> 4);
                    if (!(ok = lane_wait(&B.a_full[st], (n >> 1) & 1))) break;
                    if (!(ok = lane_wait(&B.b_full[st], (n >> 1) & 1))) break;
                    if (chunk_len<kRev>(it, nch, c) < kC) {  // (by stage: bits of `tails`)
                        if (!(ok = lane_wait(&B.fix[st], (tails >> st) & 1))) break;
                        tails ^= 1u << st;
                    }
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t off = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
                        umma_bf16(tm + kColP, a + off, bt + off, kKK, k);
                    }
                    umma_commit(&B.sc_full);
                    if (!(ok = lane_wait(&B.sb_ready, ph))) break;
                    if (n > 0 && !(ok = lane_wait(&B.o_free, ph ^ 1))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t off = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
                        umma_bf16(tm + kColO, a + off, sb + off, kKK, k);
                    }
                    umma_commit(&B.in_full);
                    umma_commit(&B.a_free[st]);
                    if (!(ok = lane_wait(&B.c_full[st], (n >> 1) & 1))) break;
                    if (!(ok = lane_wait(&B.pa_ready, ph))) break;
                    tc_fence_after();
                    const uint64_t v = mn0 + ((st * kStage + 2 * kTile) >> 4);
#pragma unroll 1
                    for (uint32_t k = 0; k < 8; ++k)
                        umma_bf16_ts(tm + kColO, tm + kColP + 8 * k, v + k * (2048 >> 4), kKMn, 1);
                    umma_commit(&B.o_full);
                    umma_commit(&B.c_free[st]);
                }
            }
            umma_commit(&B.drain[0]);
            lane_wait(&B.drain[0], 0);
        }
        __syncwarp();
    } else if (warp == 18) {
        // ---- the update's products -------------------------------------------------
        if (lane == 0) {
            constexpr uint32_t kKMn = idesc_bf16(128, 128, 0, 1, 0);
            const uint64_t mn0 = sdesc_sw128(smem_u32(sm) + kTile, kHalf, 1024);
            uint32_t n = 0, w = 0, tails = 0;
            bool ok = true;
#pragma unroll 1
            for (int id = blockIdx.x; ok && id < items; id += gridDim.x) {
                const Item it = item_of(p, id);
                const int nch = (it.len + kC - 1) / kC;
#pragma unroll 1
                for (int c = 0; c < nch; ++c, ++n) {
                    const uint32_t st = n & 1;
                    const uint64_t bt = mn0 + st * (kStage >> 4);
                    if (!(ok = lane_wait(&B.b_full[st], (n >> 1) & 1))) break;
                    if (chunk_len<kRev>(it, nch, c) < kC) {  // (by stage: bits of `tails`)
                        if (!(ok = lane_wait(&B.fix[st], (tails >> st) & 1))) break;
                        tails ^= 1u << st;
                    }
                    if (n > 0 && !(ok = lane_wait(&B.u_free, (n & 1) ^ 1))) break;
#pragma unroll 1
                    for (uint32_t q = 0; q < 4; ++q, ++w) {
                        const uint32_t buf = w & 1;
                        if (!(ok = lane_wait(&B.wv_full[buf], (w >> 1) & 1))) break;
                        tc_fence_after();
                        const uint32_t op = tm + kColW + buf * kColWBuf;
#pragma unroll 1
                        for (uint32_t k = 0; k < 2; ++k) {
                            const uint64_t d = bt + (2 * q + k) * (2048 >> 4);
#pragma unroll
                            for (uint32_t t = 0; t < 3; ++t)
                                umma_bf16_ts(tm + kColU, op + 16 * t + 8 * k, d, kKMn, q | k | t);
                        }
                        umma_commit(&B.wv_free[buf]);
                    }
                    if (!ok) break;
                    umma_commit(&B.u_full);
                    umma_commit(&B.b_free[st]);
                }
            }
            umma_commit(&B.drain[1]);
            lane_wait(&B.drain[1], 0);
        }
        __syncwarp();
    }
    } else if (warp < 4) {
        give_registers<80>();
        // ---- scores -----------------------------------------------------------------
        // Where w^-128 is far from overflow, the powers come out of the sums:
        //   out_i = tau w^{i+1} [ a_i . S + sum_{j<=i} sigma w^{-(j+1)} (a_i.b_j) c_j ]
        // (backward w^{len-1-i} and w^{-(len-1-j)}): one column factor on the
        // scores, one row factor on the output, the inter product untouched. Each row's
        // terms keep their ratios, so no bits are lost. Steeper heads scale scores by
        // w^{i-j} and the inter product by rows, a pass over O more.
        // A block's 32 column factors run from the largest exponent down by
        // products with w^2 in registers: a table in shared memory waits there
        // behind the tensor cores' operands.
        const int i = 32 * warp + lane;  // this thread's row of the chunk
        const int blocks = kRev ? 4 - warp : warp + 1, cb0 = kRev ? warp : 0;  // not masked
        uint32_t n = 0;
        bool ok = true;
#pragma unroll 1
        for (int id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const Item it = item_of(p, id);
            const int nch = (it.len + kC - 1) / kC;
            const float g = p.log_decay[it.h], w = power(g, 1);
            const bool gentle = is_gentle(g);
            const uint64_t step = pair(w * w, w * w);
            const float w16 = power(g, 16), steep = power(g, kRev ? max(16 - lane, 0)
                                                                  : max(lane - 15, 0));
            float ahead = 0.f, fb[4];  // steep: O's row factor; each block's first column factor
            int known = 0;             // the chunk length they are for
#pragma unroll 1
            for (int c = 0; c < nch; ++c, ++n) {
                const uint32_t ph = n & 1;
                const int len = chunk_len<kRev>(it, nch, c);
                if (len != known) {
                    ahead = row_factor<kRev>(p, g, len, i);
                    // Steep, off the diagonal block: w^{i-j} splits in two
                    // exponents that are not negative, rows' and columns'.
                    const float edge = p.sigma * p.tau * power(g, kRev ? 32 - lane : lane + 1);
#pragma unroll
                    for (int cb = 0; cb < 4; ++cb) {
                        const int e = kRev ? len - 1 - 32 * cb : 32 * cb + 32;
                        const int apart = kRev ? cb - warp : warp - cb;
                        fb[cb] = (gentle ? p.sigma : edge) *
                                 power(gentle && e >= 0 ? -g : g,
                                       gentle ? abs(e) : 32 * (apart - 1));
                    }
                    known = len;
                }
                // Half block y = 2 x + (upper half), 16 scores a thread. The powers run
                // from the larger exponents' side ...
                auto decay = [&](int y, uint64_t (&s)[8]) {
                    const int x = y >> 1, hb = y & 1, cb = cb0 + x;
                    const bool diag = kRev ? x == 0 : x == blocks - 1;
                    const bool far = kRev ? hb == 1 : hb == 0;
                    uint32_t packed[8];
                    if (gentle || !diag) {
                        float f = cb < 2 ? (cb == 0 ? fb[0] : fb[1]) : (cb == 2 ? fb[2] : fb[3]);
                        if (far) f *= w16;
                        uint64_t f2 = kRev ? pair(f, f * w) : pair(f * w, f);
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            const int j = kRev ? t : 7 - t;
                            packed[j] = pack_bf16(mul2(s[j], f2));
                            f2 = mul2(f2, step);
                        }
                    } else {
                        const int me = lane - 16 * hb;  // this row's column in the half
                        float f = p.sigma * p.tau * (far ? steep : 1.f);
#pragma unroll
                        for (int t = 0; t < 8; ++t) {
                            const int j = kRev ? t : 7 - t;
                            float x, y2;
                            unpair(s[j], x, y2);
                            (kRev ? x : y2) *= f;
                            if (kRev ? 2 * j >= me : 2 * j + 1 <= me) f *= w;
                            (kRev ? y2 : x) *= f;
                            if (kRev ? 2 * j + 1 >= me : 2 * j <= me) f *= w;
                            packed[j] = pack_bf16(x, y2);
                        }
                    }
                    if (diag) {  // j <= i, or j >= i
                        const int me = lane - 16 * hb;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const bool k0 = kRev ? 2 * j >= me : 2 * j <= me;
                            const bool k1 = kRev ? 2 * j + 1 >= me : 2 * j + 1 <= me;
                            packed[j] &= (k0 ? 0xffffu : 0u) | (k1 ? 0xffff0000u : 0u);
                        }
                    }
                    tmem_st8(quad + kColP + 16 * cb + 8 * hb, packed);
                };
                if (!(ok = warp_wait(&B.sc_full, ph))) break;
                tc_fence_after();
                // ... and P goes over the scores in their order, over blocks that are
                // read by then.
                const uint32_t scores = quad + kColP + 32 * cb0;
#pragma unroll 1
                for (int y = 0; y < 2 * blocks; ++y) {
                    uint64_t s[8];
                    tmem_ld16(scores + 16 * y, s);
                    decay(y, s);
                }
                uint32_t zero[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) zero[j] = 0;
#pragma unroll 1
                for (int cb = kRev ? 0 : blocks; cb < (kRev ? cb0 : 4); ++cb)
                    tmem_st16(quad + kColP + 16 * cb, zero);
                if (!gentle) {
                    if (!(ok = warp_wait(&B.in_full, ph))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int cb = 0; cb < 4; ++cb) {
                        float o[32];
                        tmem_ld32(quad + kColO + 32 * cb, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= ahead;
                        tmem_st32(quad + kColO + 32 * cb, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.pa_ready);
            }
        }
    } else if (warp < 12) {
        take_registers<128>();
        // ---- the state and the outputs ----------------------------------------------
        const int col = 32 * (warp & 3) + lane;  // this thread's column of S (row of U^T),
        const int half = (warp - 4) >> 2, b0 = 64 * half;  // and its rows b0 .. b0 + 63; of the
        uint8_t* sb = sm + kOffSb + half * kHalf + col * 128;  // output, row col of the chunk
        uint32_t n = 0;  // chunks begun                       // and those features
        bool ok = true;
        // 32-byte stores where every row piece is so aligned.
        const bool wide = p.d_c % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;
        uint64_t s[32];  // pairs of its rows
#pragma unroll 1
        for (int id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const Item it = item_of(p, id);
            const int nch = (it.len + kC - 1) / kC;
            const float g = p.log_decay[it.h];
            const bool gentle = is_gentle(g);
            const int64_t rs_in = it.in_t ? 1 : p.d_c, rs_out = it.out_t ? 1 : p.d_c;
            const bool mine = col < p.d_c;
            if (it.in != nullptr && mine) {
                const float* src = it.in + (it.in_t ? col * p.d_b : col) + b0 * rs_in;
#pragma unroll
                for (int j = 0; j < 32; ++j, src += 2 * rs_in)
                    s[j] = pair(b0 + 2 * j < p.d_b ? src[0] : 0.f,
                                b0 + 2 * j + 1 < p.d_b ? src[rs_in] : 0.f);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) s[j] = 0;
            }
            // w^len in two parts (it is applied chunk after chunk); the output's
            // row factor.
            uint64_t hi2 = 0, lo2 = 0;
            float ahead = 1.f;
            int known = 0;
#pragma unroll 1
            for (int c = -1; c < nch; ++c) {
                // The state's bf16 copy for chunk c + 1, once chunk c's product has read its own.
                if (c >= 0) {
                    const int len = chunk_len<kRev>(it, nch, c);
                    if (len != known) {
                        const float2 f = power2(g, len);
                        hi2 = pair(f.x, f.x);
                        lo2 = pair(f.y, f.y);
                        ahead = gentle ? row_factor<kRev>(p, g, len, col) : 1.f;
                        known = len;
                    }
                    if (!(ok = warp_wait(&B.u_full, n & 1))) break;
                    tc_fence_after();
#pragma unroll
                    for (int blk = 0; blk < 4; ++blk) {
                        uint64_t u[8];
                        tmem_ld16(quad + kColU + b0 + 16 * blk, u);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            s[8 * blk + j] =
                                fma2(s[8 * blk + j], hi2, fma2(s[8 * blk + j], lo2, u[j]));
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.u_free);
                }
                if (c + 1 < nch) {
                    const uint32_t before = c >= 0 ? n : n - 1;  // the last chunk begun
                    if (n > 0 || c >= 0)
                        if (!(ok = warp_wait(&B.in_full, before & 1))) break;
#pragma unroll
                    for (int m = 0; m < 8; ++m)
                        *reinterpret_cast<uint4*>(sb + ((m ^ (col & 7)) << 4)) =
                            make_uint4(pack_bf16(s[4 * m]), pack_bf16(s[4 * m + 1]),
                                       pack_bf16(s[4 * m + 2]), pack_bf16(s[4 * m + 3]));
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.sb_ready);
                }
                if (c < 0) continue;
                // The output: scaled, converted, stored from registers, 16 features
                // of a row (one 32-byte sector) at a time; only rows of the sequence.
                int64_t row;
                int len;
                chunk_of<kRev>(it, nch, c, row, len);
                if (!(ok = warp_wait(&B.o_full, n & 1))) break;
                tc_fence_after();
                const bool live = col < len;
                const uint64_t scale = pair(ahead, ahead);
                const int64_t at = ((row + col) * p.heads + it.h) * p.d_c + b0;
#pragma unroll 1
                for (int blk = 0; blk < 4; ++blk) {
                    uint64_t u[8];
                    tmem_ld16(quad + kColO + b0 + 16 * blk, u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] = mul2(u[j], scale);
                    const int left = p.d_c - b0 - 16 * blk;  // features of the row from here
                    if (!live || left <= 0) continue;
                    if (p.out_f32) {
                        float* o = static_cast<float*>(p.out) + at + 16 * blk;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (4 * j < left) {
                                float4 x;
                                unpair(u[2 * j], x.x, x.y);
                                unpair(u[2 * j + 1], x.z, x.w);
                                reinterpret_cast<float4*>(o)[j] = x;
                            }
                    } else {
                        uint32_t x[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = pack_bf16(u[j]);
                        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + at + 16 * blk;
                        if (wide) {
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                                         ::"l"(o), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]),
                                         "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                                         : "memory");
                        } else {
                            reinterpret_cast<uint4*>(o)[0] = make_uint4(x[0], x[1], x[2], x[3]);
                            if (left > 8)
                                reinterpret_cast<uint4*>(o)[1] = make_uint4(x[4], x[5], x[6], x[7]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.o_free);
                ++n;
            }
            if (ok && it.out != nullptr && mine) {
                float* dst = it.out + (it.out_t ? col * p.d_b : col) + b0 * rs_out;
#pragma unroll
                for (int j = 0; j < 32; ++j, dst += 2 * rs_out) {
                    float x, y;
                    unpair(s[j], x, y);
                    if (b0 + 2 * j < p.d_b) dst[0] = x;
                    if (b0 + 2 * j + 1 < p.d_b) dst[rs_out] = y;
                }
            }
        }
    } else {
        // ---- the update's operand ----------------------------------------------------
        // (w c)^T, features on the TMEM lanes: 8 x 8 blocks of the c tile come
        // transposed from ldmatrix, thread t holding feature t / 4 (and + 8)
        // at positions 2 (t % 4), + 1 of each 8, which is where tcgen05.st's
        // 16x128b shape puts them; a thread's weights stay in registers.
        const int wc = warp - 12;
        const int row = ((lane >> 4) << 3) + (lane & 7);  // ldmatrix row of this lane
        const uint32_t src0 = smem_u32(sm) + 2 * kTile + (wc >> 1) * kHalf + row * 128;
        const int chunk0 = 4 * (wc & 1) + ((lane >> 3) & 1);
        const uint64_t minus = pair(-1.f, -1.f);
        uint32_t n = 0, w = 0;
        bool ok = true;
#pragma unroll 1
        for (int id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const Item it = item_of(p, id);
            const int nch = (it.len + kC - 1) / kC;
            const float g = p.log_decay[it.h];
            // Of position j = 32 q + jj, jj = 8 k + 2 (t % 4) + e, in a whole chunk:
            // w^(127 - j) = w^(96 - 32 q) w^(31 - jj), backward w^(32 q) w^(jj + 1).
            const int j0 = 2 * (lane & 3);
            const float mine = power(g, lane);  // w^lane, for the other lanes
            auto small = [&](int n) { return __shfl_sync(0xffffffffu, mine, n & 31); };
            uint64_t wt[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = 8 * k + j0;
                wt[k] = kRev ? pair(small(j) * small(1), small(j + 1) * small(1))
                             : pair(small(31 - j), small(30 - j));
            }
            const float w32 = power(g, 32), w64 = power(g, 64), w96 = power(g, 96);
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
                    for (int r = len + wc; r < kC; r += 4)
                        *reinterpret_cast<uint4*>(tile + ((lane & 15) >> 3) * kHalf + r * 128 +
                                                  (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.fix[st]);
                }
#pragma unroll 1
                for (int q = 0; q < 4; ++q, ++w) {
                    const int buf = w & 1;
                    uint32_t x[2][8];
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int g2 = 0; g2 < 2; ++g2)
                            asm volatile(
                                "ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16"
                                " {%0, %1, %2, %3}, [%4];"
                                : "=r"(x[half][4 * g2]), "=r"(x[half][4 * g2 + 1]),
                                  "=r"(x[half][4 * g2 + 2]), "=r"(x[half][4 * g2 + 3])
                                : "r"(src0 + st * kStage + (32 * q + 16 * g2) * 128 +
                                      (((chunk0 + 2 * half) ^ (lane & 7)) << 4))
                                : "memory");
                    if (q == 3) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&B.c_free[st]);
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
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                x[half][2 * k] &= keep;
                                x[half][2 * k + 1] &= keep;
                            }
                        }
                    }
                    if (w >= 2 && !(ok = warp_wait(&B.wv_free[buf], ((w >> 1) & 1) ^ 1))) break;
                    tc_fence_after();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t mid[8], lo[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            uint64_t v = mul2(widen(x[half][k]), f[k >> 1]);
                            x[half][k] = pack_bf16(v);
                            v = fma2(widen(x[half][k]), minus, v);
                            mid[k] = pack_bf16(v);
                            lo[k] = pack_bf16(fma2(widen(mid[k]), minus, v));
                        }
                        const uint32_t at =
                            quad + (static_cast<uint32_t>(half) << 20) + kColW + buf * kColWBuf;
                        tmem_st_16x128(at, x[half]);
                        tmem_st_16x128(at + 16, mid);
                        tmem_st_16x128(at + 32, lo);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.wv_full[buf]);
                }
                if (!ok) break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 18) tmem_dealloc(tm, 512);
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

// [tokens, heads, d] bf16 in boxes of 64 features x 1 head x 128 positions;
// features past d read as zeros.
bool tile_map(CUtensorMap* map, const void* base, int64_t tokens, int heads, int d) {
    auto encode = encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(d) * 2,
                                   static_cast<cuuint64_t>(heads) * d * 2};
    const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(kC)};
    const cuuint32_t estride[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides,
                  box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
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

cudaError_t launch_la_tc(const LaCore& p, cudaStream_t stream) {
    CUtensorMap ma, mb, mc;
    const int64_t tokens = la_tokens(p);
    if (!tile_map(&ma, p.a, tokens, p.heads_a, p.d_b) ||
        !tile_map(&mb, p.b, tokens, p.heads_b, p.d_b) ||
        !tile_map(&mc, p.c, tokens, p.heads_c, p.d_c))
        return cudaErrorInvalidValue;
    auto* kernel = p.reverse ? la_tc<true> : la_tc<false>;
    const cudaError_t e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes));
    if (e != cudaSuccess) return e;
    const int64_t items = static_cast<int64_t>(p.n_seqs) * p.heads;
    const int grid = static_cast<int>(std::min<int64_t>(items, sm_count()));
    kernel<<<grid, kThreads, kSmemBytes, stream>>>(p, ma, mb, mc, static_cast<int>(items));
    return cudaGetLastError();
}

cudaError_t take_la_error(int* flag) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_la_error, sizeof(int));
    if (e != cudaSuccess || *flag == 0) return e;
    const int zero = 0;
    return cudaMemcpyToSymbol(g_la_error, &zero, sizeof(int));
}

}  // namespace gdr
