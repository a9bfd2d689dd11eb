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
// that the loads, the matrix products and the three conversions of
// consecutive chunks run beside one another:
//   warp 12      TMA loads of the a, b, c tiles, two stages of 96 KiB
//   warp 13      issues every tcgen05.mma
//   warps 0-3    scores -> decayed bf16 P; the inter product's row scale; the
//                output (converted, staged in the stage's a tile, TMA store)
//   warps 4-7    the state: f32 in TMEM -> its bf16 copy in shared memory, and
//                scaled by w^C in TMEM; initial and final states
//   warps 8-11   the update's operand, c scaled by w^{C-1-j}
// The products of a chunk, M = N = 128 each, f32 accumulators in TMEM:
//   scores = A B^T              both from shared memory
//   O      = A Sb               Sb the state's bf16 copy (K-major rows of c)
//   S^T   += (w c)^T B          (w c)^T from TMEM, B read MN-major
//   O     += P C                P from TMEM, C read MN-major
// TMEM (512 columns): S^T 128, scores with P over them 128, O 128, (w c)^T two
// buffers of 48 (32 positions in three parts).
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
constexpr int kThreads = 448;
constexpr uint32_t kTile = 32768;         // 128 positions x 128 bf16, two 64-wide halves
constexpr uint32_t kHalf = kTile / 2;
constexpr uint32_t kStage = 3 * kTile;    // a, b, c
constexpr uint32_t kOffSb = 2 * kStage, kOffMisc = kOffSb + kTile;
constexpr uint32_t kSmemBytes = kOffMisc + 2048 + 1024;  // + alignment slack
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256, kColW = 384, kColWBuf = 48;
constexpr uint64_t kWaitLimitNs = 2000000000ull;

struct Bars {
    uint64_t full[2], kv_free[2], q_free[2];
    uint64_t sc_full, in_full, o_full, o_free, pa_ready, st_ready, st_full, fix, drain;
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

// Waits for a phase, the whole warp together; false (for every lane) once the
// limit ran out, which is recorded.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_wait(bar, parity, kWaitLimitNs);
    if (!ok) atomicOr(&g_la_error, 1);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_wait(bar, parity, kWaitLimitNs);
    if (!ok) atomicOr(&g_la_error, 1);
    return ok;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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

// w^n to f32 accuracy (the exponent in f64), 1 for n = 0.
__device__ __forceinline__ double power(double g, int n) { return n <= 0 ? 1.0 : exp(g * n); }

__device__ __forceinline__ Item item_of(const LaCore& p, int64_t id) {
    Item it;
    const int s = static_cast<int>(id / p.heads);
    it.h = static_cast<int>(id - static_cast<int64_t>(s) * p.heads);
    int64_t end;
    la_span(p, s, it.start, end);
    it.len = static_cast<int>(end - it.start);
    const int64_t at = id * p.d_b * p.d_c;
    it.in = p.state_in != nullptr ? p.state_in + at : nullptr;
    it.out = p.state_out != nullptr ? p.state_out + at : nullptr;
    it.in_t = it.out_t = p.state_t != 0;
    return it;
}

// Chunk c of an item, in the order they run.
__device__ __forceinline__ void chunk_of(const LaCore& p, const Item& it, int nch, int c,
                                         int64_t& row, int& len) {
    const int x = p.reverse ? nch - 1 - c : c;
    row = it.start + static_cast<int64_t>(x) * kC;
    len = min(kC, it.len - x * kC);
}

__global__ void __launch_bounds__(kThreads, 1)
la_tc(const LaCore p, const __grid_constant__ CUtensorMap ma,
      const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap mc,
      const __grid_constant__ CUtensorMap mo, int64_t items) {
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
    Bars& B = *reinterpret_cast<Bars*>(sm + kOffMisc);
    float* tables = reinterpret_cast<float*>(sm + kOffMisc + 512);  // [8 warps][32]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.full[i], 1);
            mbar_init(&B.kv_free[i], 1);
            mbar_init(&B.q_free[i], 4);
            mbar_init(&B.wv_full[i], 4);
            mbar_init(&B.wv_free[i], 1);
        }
        mbar_init(&B.sc_full, 1);
        mbar_init(&B.in_full, 1);
        mbar_init(&B.o_full, 1);
        mbar_init(&B.o_free, 4);
        mbar_init(&B.pa_ready, 4);
        mbar_init(&B.st_ready, 4);
        mbar_init(&B.st_full, 1);
        mbar_init(&B.fix, 4);
        mbar_init(&B.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 13) {
        tmem_alloc(&B.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = B.tmem;
    const uint32_t quad = tm + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's lanes

    if (warp == 12) {
        // ---- loads -------------------------------------------------------------
        if (lane == 0) {
            uint32_t n = 0;
            bool ok = true;
            for (int64_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
                const Item it = item_of(p, id);
                const int nch = (it.len + kC - 1) / kC;
                const int ha = it.h / (p.heads / p.heads_a), hb = it.h / (p.heads / p.heads_b),
                          hc = it.h / (p.heads / p.heads_c);
                for (int c = 0; c < nch; ++c, ++n) {
                    const int st = n & 1;
                    const uint32_t ph = ((n >> 1) & 1) ^ 1;
                    int64_t row;
                    int len;
                    chunk_of(p, it, nch, c, row, len);
                    uint8_t* base = sm + st * kStage;
                    if (n >= 2 && !(ok = lane_wait(&B.kv_free[st], ph))) break;
                    mbar_expect_tx(&B.full[st], kStage);
                    const int r = static_cast<int>(row);
                    tma_load_3d(base + kTile, &mb, &B.full[st], 0, hb, r);
                    tma_load_3d(base + kTile + kHalf, &mb, &B.full[st], 64, hb, r);
                    tma_load_3d(base + 2 * kTile, &mc, &B.full[st], 0, hc, r);
                    tma_load_3d(base + 2 * kTile + kHalf, &mc, &B.full[st], 64, hc, r);
                    if (n >= 2 && !(ok = lane_wait(&B.q_free[st], ph))) break;
                    tma_load_3d(base, &ma, &B.full[st], 0, ha, r);
                    tma_load_3d(base + kHalf, &ma, &B.full[st], 64, ha, r);
                }
            }
            // Nothing of this CTA's may be in flight when it ends.
            for (uint32_t i = n >= 2 ? n - 2 : 0; i < n; ++i)
                lane_wait(&B.full[i & 1], (i >> 1) & 1);
        }
        __syncwarp();
    } else if (warp == 13) {
        // ---- products ------------------------------------------------------------
        if (lane == 0) {
            constexpr uint32_t kKK = idesc_bf16(128, 128, 0, 0, 0);
            constexpr uint32_t kKMn = idesc_bf16(128, 128, 0, 1, 0);
            const uint32_t sb = smem_u32(sm + kOffSb);
            uint32_t n = 0, w = 0, tails = 0;
            bool ok = true;
            for (int64_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
                const Item it = item_of(p, id);
                const int nch = (it.len + kC - 1) / kC;
                for (int c = 0; c < nch; ++c, ++n) {
                    const int st = n & 1;
                    const uint32_t ph = n & 1;
                    int64_t row;
                    int len;
                    chunk_of(p, it, nch, c, row, len);
                    const uint32_t a = smem_u32(sm + st * kStage), b = a + kTile, v = b + kTile;
                    if (!(ok = lane_wait(&B.full[st], (n >> 1) & 1))) break;
                    if (len < kC && !(ok = lane_wait(&B.fix, tails++ & 1))) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
                        umma_bf16(tm + kColP, sdesc_sw128(a + off, 16, 1024),
                                  sdesc_sw128(b + off, 16, 1024), kKK, k > 0);
                    }
                    umma_commit(&B.sc_full);
                    if (!(ok = lane_wait(&B.st_ready, ph))) break;
                    if (n > 0 && !(ok = lane_wait(&B.o_free, ph ^ 1))) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
                        umma_bf16(tm + kColO, sdesc_sw128(a + off, 16, 1024),
                                  sdesc_sw128(sb + off, 16, 1024), kKK, k > 0);
                    }
                    umma_commit(&B.in_full);
                    for (int q = 0; ok && q < 4; ++q, ++w) {
                        const int buf = w & 1;
                        if (!(ok = lane_wait(&B.wv_full[buf], (w >> 1) & 1))) break;
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint64_t d = sdesc_sw128(b + (32 * q + 16 * k) * 128, kHalf, 1024);
#pragma unroll
                            for (int t = 0; t < 3; ++t)
                                umma_bf16_ts(tm + kColS, tm + kColW + buf * kColWBuf + 16 * t + 8 * k,
                                             d, kKMn, 1);
                        }
                        umma_commit(&B.wv_free[buf]);
                    }
                    if (!ok) break;
                    umma_commit(&B.st_full);
                    if (!(ok = lane_wait(&B.pa_ready, ph))) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        umma_bf16_ts(tm + kColO, tm + kColP + 8 * k,
                                     sdesc_sw128(v + 16 * k * 128, kHalf, 1024), kKMn, 1);
                    umma_commit(&B.o_full);
                    umma_commit(&B.kv_free[st]);
                }
            }
            umma_commit(&B.drain);
            lane_wait(&B.drain, 0);
        }
        __syncwarp();
    } else if (warp < 4) {
        // ---- scores, outputs -------------------------------------------------------
        float* tab = tables + 32 * warp;  // w^n, n < 32
        const int i = 32 * warp + lane;   // this thread's row of the chunk
        uint32_t n = 0;
        bool ok = true, pending = false;
        int pending_st = 0;
        for (int64_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const Item it = item_of(p, id);
            const int nch = (it.len + kC - 1) / kC;
            const double g = p.log_decay[it.h];
            __syncwarp();
            tab[lane] = static_cast<float>(power(g, lane));
            __syncwarp();
            // Off the diagonal block the exponent splits in two that are not
            // negative: (row part, 32 m) and the column's, from the table.
            const float edge = static_cast<float>(power(g, p.reverse ? 32 - lane : lane + 1));
            const float w32 = static_cast<float>(power(g, 32)), w64 = static_cast<float>(power(g, 64));
            float ahead = 0.f;  // the inter product's row scale
            int known = 0;      // the chunk length it is for
            for (int c = 0; c < nch; ++c, ++n) {
                const uint32_t ph = n & 1;
                const int st = n & 1;
                int64_t row;
                int len;
                chunk_of(p, it, nch, c, row, len);
                if (len != known) {
                    ahead = static_cast<float>(power(g, p.reverse ? max(len - 1 - i, 0) : i + 1));
                    known = len;
                }
                if (!(ok = warp_wait(&B.sc_full, ph))) break;
                tc_fence_after();
#pragma unroll 1
                for (int cb = 0; cb < 4; ++cb) {
                    const int apart = p.reverse ? cb - warp : warp - cb;  // blocks apart
                    uint32_t packed[16];
                    if (apart < 0) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) packed[j] = 0;
                    } else {
                        float s[32];
                        tmem_ld32(quad + kColP + 32 * cb, s);
                        tmem_wait_ld();
                        if (apart > 0) {
                            const float f = p.sigma * edge *
                                            (apart == 1 ? 1.f : apart == 2 ? w32 : w64);
#pragma unroll
                            for (int j4 = 0; j4 < 8; ++j4) {
                                const float4 x = reinterpret_cast<const float4*>(
                                    tab)[p.reverse ? j4 : 7 - j4];
                                const float y[4] = {p.reverse ? x.x : x.w, p.reverse ? x.y : x.z,
                                                    p.reverse ? x.z : x.y, p.reverse ? x.w : x.x};
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[4 * j4 + j] *= f * y[j];
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const int e = p.reverse ? j - lane : lane - j;
                                s[j] = e >= 0 ? s[j] * (p.sigma * tab[e & 31]) : 0.f;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) packed[j] = pack_bf16(s[2 * j], s[2 * j + 1]);
                    }
                    tmem_st16(quad + kColP + 16 * cb, packed);
                }
                if (pending) {  // the store of the last chunk has left its tile
                    if (lane == 0) {
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        mbar_arrive(&B.q_free[pending_st]);
                    }
                    pending = false;
                }
                if (!(ok = warp_wait(&B.in_full, ph))) break;
                tc_fence_after();
#pragma unroll 1
                for (int cb = 0; cb < 4; ++cb) {
                    float s[32];
                    tmem_ld32(quad + kColO + 32 * cb, s);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] *= ahead;
                    tmem_st32(quad + kColO + 32 * cb, s);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.pa_ready);
                if (!(ok = warp_wait(&B.o_full, ph))) break;
                tc_fence_after();
                uint8_t* tile = sm + st * kStage;  // a's, read by now
                const int live = min(max(len - 32 * warp, 0), 32);
                const int64_t orow = (row + i) * p.heads + it.h;
#pragma unroll 1
                for (int cb = 0; cb < 4; ++cb) {
                    float s[32];
                    tmem_ld32(quad + kColO + 32 * cb, s);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] *= p.tau;
                    if (p.out_f32) {
                        float* o = static_cast<float*>(p.out) + orow * p.d_c + 32 * cb;
                        if (lane < live)
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (32 * cb + 4 * j < p.d_c)
                                    reinterpret_cast<float4*>(o)[j] = make_float4(
                                        s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]);
                    } else {
                        uint8_t* dst = tile + (cb >> 1) * kHalf + i * 128;
#pragma unroll
                        for (int m = 0; m < 4; ++m)
                            *reinterpret_cast<uint4*>(dst + ((((cb & 1) * 4 + m) ^ (i & 7)) << 4)) =
                                make_uint4(pack_bf16(s[8 * m], s[8 * m + 1]),
                                           pack_bf16(s[8 * m + 2], s[8 * m + 3]),
                                           pack_bf16(s[8 * m + 4], s[8 * m + 5]),
                                           pack_bf16(s[8 * m + 6], s[8 * m + 7]));
                    }
                }
                tc_fence_before();
                if (!p.out_f32 && live == 32) fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.o_free);
                if (!p.out_f32 && live == 32) {
                    if (lane == 0) {
                        const uint8_t* src = tile + 32 * warp * 128;
                        const int r = static_cast<int>(row) + 32 * warp;
                        tma_store_3d(&mo, src, 0, it.h, r);
                        if (p.d_c > 64) tma_store_3d(&mo, src + kHalf, 64, it.h, r);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    pending = true;
                    pending_st = st;
                } else {
                    // A part of a tile: the rows of other sequences stay as
                    // they are.
                    if (!p.out_f32) {
                        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out);
                        const int ch = lane & 15;
                        for (int r = lane >> 4; r < live; r += 2) {
                            const int ri = 32 * warp + r;
                            if (8 * ch < p.d_c)
                                *reinterpret_cast<uint4*>(
                                    o + ((row + ri) * p.heads + it.h) * p.d_c + 8 * ch) =
                                    *reinterpret_cast<const uint4*>(
                                        tile + (ch >> 3) * kHalf + ri * 128 +
                                        (((ch & 7) ^ (ri & 7)) << 4));
                        }
                        // The tile's next writer is the async proxy.
                        fence_proxy_async();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.q_free[st]);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (pending && lane == 0) mbar_arrive(&B.q_free[pending_st]);
    } else if (warp < 8) {
        // ---- the state -----------------------------------------------------------
        const int col = 32 * (warp - 4) + lane;  // this thread's column of S (row of S^T)
        uint8_t* sb = sm + kOffSb + col * 128;
        uint32_t n = 0;
        bool ok = true;
        for (int64_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const Item it = item_of(p, id);
            const int nch = (it.len + kC - 1) / kC;
            const double g = p.log_decay[it.h];
            const int rs_in = it.in_t ? 1 : p.d_c, rs_out = it.out_t ? 1 : p.d_c;
            const float* src = it.in ? it.in + (it.in_t ? col * p.d_b : col) : nullptr;
            float* dst = it.out ? it.out + (it.out_t ? col * p.d_b : col) : nullptr;
            float hi = 1.f, lo = 0.f;  // w^len, in two parts: it is applied every chunk
            int known = 0;             // the chunk length they are for
            for (int c = 0; c <= nch; ++c) {
                if (c < nch) {
                    int64_t row;
                    int len;
                    chunk_of(p, it, nch, c, row, len);
                    if (len != known) {
                        const double f = power(g, len);
                        hi = static_cast<float>(f);
                        lo = static_cast<float>(f - hi);
                        known = len;
                    }
                }
                if (c > 0) {
                    if (!(ok = warp_wait(&B.st_full, (n - 1) & 1))) break;
                    tc_fence_after();
                }
                const bool last = c == nch;
#pragma unroll 1
                for (int blk = 0; blk < 4; ++blk) {
                    float s[32];
                    if (c > 0) {
                        tmem_ld32(quad + kColS + 32 * blk, s);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const int b = 32 * blk + j;
                            s[j] = src != nullptr && col < p.d_c && b < p.d_b
                                       ? src[static_cast<int64_t>(b) * rs_in]
                                       : 0.f;
                        }
                    }
                    if (last) {
                        if (dst != nullptr && col < p.d_c)
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const int b = 32 * blk + j;
                                if (b < p.d_b) dst[static_cast<int64_t>(b) * rs_out] = s[j];
                            }
                        continue;
                    }
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        *reinterpret_cast<uint4*>(sb + (blk >> 1) * kHalf +
                                                  ((((blk & 1) * 4 + m) ^ (col & 7)) << 4)) =
                            make_uint4(pack_bf16(s[8 * m], s[8 * m + 1]),
                                       pack_bf16(s[8 * m + 2], s[8 * m + 3]),
                                       pack_bf16(s[8 * m + 4], s[8 * m + 5]),
                                       pack_bf16(s[8 * m + 6], s[8 * m + 7]));
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] = fmaf(s[j], hi, s[j] * lo);
                    tmem_st32(quad + kColS + 32 * blk, s);
                }
                if (last) {
                    tc_fence_before();
                    break;
                }
                tmem_wait_st();
                fence_proxy_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.st_ready);
                ++n;
            }
        }
    } else {
        // ---- the update's operand ----------------------------------------------------
        float* tab = tables + 32 * (warp - 4);
        const int col = 32 * (warp - 8) + lane;  // this thread's feature of c
        const int cx = ((col & 63) >> 3) << 4, cy = (col >> 6) * kHalf + (col & 7) * 2;
        uint32_t n = 0, w = 0;
        bool ok = true;
        for (int64_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const Item it = item_of(p, id);
            const int nch = (it.len + kC - 1) / kC;
            const double g = p.log_decay[it.h];
            __syncwarp();  // every lane has read the last item's table
            tab[lane] = static_cast<float>(power(g, p.reverse ? lane + 1 : 31 - lane));
            __syncwarp();
            const float w32 = static_cast<float>(power(g, 32)), w64 = static_cast<float>(power(g, 64)),
                        w96 = static_cast<float>(power(g, 96));
            for (int c = 0; c < nch; ++c, ++n) {
                const int st = n & 1;
                int64_t row;
                int len;
                chunk_of(p, it, nch, c, row, len);
                uint8_t* bt = sm + st * kStage + kTile;
                uint8_t* ct = bt + kTile;
                if (!(ok = warp_wait(&B.full[st], (n >> 1) & 1))) break;
                if (len < kC) {
                    // The rows past the sequence hold another's (or anything):
                    // zeros, so that no product of theirs is NaN.
                    for (int r = len + (warp - 8); r < kC; r += 4) {
                        uint8_t* tile = lane < 16 ? bt : ct;
                        *reinterpret_cast<uint4*>(tile + ((lane & 15) >> 3) * kHalf + r * 128 +
                                                  (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.fix);
                }
                for (int q = 0; ok && q < 4; ++q, ++w) {
                    const int buf = w & 1;
                    if (w >= 2 && !(ok = warp_wait(&B.wv_free[buf], ((w >> 1) & 1) ^ 1))) break;
                    tc_fence_after();
                    const uint8_t* src = ct + 32 * q * 128 + cy;
                    uint32_t hi[16], mid[16], lo[16];
                    auto split = [&](int j2, float x0, float x1) {
                        hi[j2] = pack_bf16(x0, x1);
                        x0 -= low_f32(hi[j2]);
                        x1 -= high_f32(hi[j2]);
                        mid[j2] = pack_bf16(x0, x1);
                        lo[j2] = pack_bf16(x0 - low_f32(mid[j2]), x1 - high_f32(mid[j2]));
                    };
                    auto value = [&](int j) {
                        return __uint_as_float(
                            static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(
                                src + j * 128 + (cx ^ ((j & 7) << 4))))
                            << 16);
                    };
                    if (len == kC) {
                        // w^(127 - j) = w^(96 - 32 q) w^(31 - jj), and
                        // w^(j + 1) = w^(32 q) w^(jj + 1).
                        const int e = p.reverse ? q : 3 - q;
                        const float base =
                            p.sigma * (e == 0 ? 1.f : e == 1 ? w32 : e == 2 ? w64 : w96);
#pragma unroll
                        for (int j4 = 0; j4 < 8; ++j4) {
                            const float4 t = reinterpret_cast<const float4*>(tab)[j4];
                            split(2 * j4, value(4 * j4) * (base * t.x),
                                  value(4 * j4 + 1) * (base * t.y));
                            split(2 * j4 + 1, value(4 * j4 + 2) * (base * t.z),
                                  value(4 * j4 + 3) * (base * t.w));
                        }
                    } else {
                        // A short chunk: w^(len - 1 - j), the table shifted in
                        // its last quarter; zeros past it.
                        const int live = len - 32 * q;
                        const float base = p.sigma * static_cast<float>(power(
                                                         g, p.reverse ? 32 * q : max(live - 32, 0)));
                        const int shift = p.reverse || live >= 32 ? 0 : 32 - live;
#pragma unroll
                        for (int j2 = 0; j2 < 16; ++j2) {
                            const int j = 2 * j2;
                            split(j2, j < live ? value(j) * (base * tab[(j + shift) & 31]) : 0.f,
                                  j + 1 < live ? value(j + 1) * (base * tab[(j + 1 + shift) & 31])
                                               : 0.f);
                        }
                    }
                    const uint32_t at = quad + kColW + buf * kColWBuf;
                    tmem_st16(at, hi);
                    tmem_st16(at + 16, mid);
                    tmem_st16(at + 32, lo);
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
    if (warp == 13) tmem_dealloc(tm, 512);
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

// [tokens, heads, d] bf16 in boxes of 64 features x 1 head x `rows` positions;
// features past d read as zeros and are not written.
bool tile_map(CUtensorMap* map, const void* base, int64_t tokens, int heads, int d, int rows) {
    auto encode = encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(d) * 2,
                                   static_cast<cuuint64_t>(heads) * d * 2};
    const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)};
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
           la_tokens(p) < (int64_t{1} << 31) - 2 * kC;
}

cudaError_t launch_la_tc(const LaCore& p, cudaStream_t stream) {
    CUtensorMap ma, mb, mc, mo;
    const int64_t tokens = la_tokens(p);
    if (!tile_map(&ma, p.a, tokens, p.heads_a, p.d_b, kC) ||
        !tile_map(&mb, p.b, tokens, p.heads_b, p.d_b, kC) ||
        !tile_map(&mc, p.c, tokens, p.heads_c, p.d_c, kC))
        return cudaErrorInvalidValue;
    if (p.out_f32)
        mo = mc;  // not used
    else if (!tile_map(&mo, p.out, tokens, p.heads, p.d_c, 32))
        return cudaErrorInvalidValue;
    cudaError_t e = cudaFuncSetAttribute(la_tc, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(kSmemBytes));
    if (e != cudaSuccess) return e;
    const int64_t items = static_cast<int64_t>(p.n_seqs) * p.heads;
    const int grid = static_cast<int>(std::min<int64_t>(items, sm_count()));
    la_tc<<<grid, kThreads, kSmemBytes, stream>>>(p, ma, mb, mc, mo, items);
    return cudaGetLastError();
}

cudaError_t take_la_error(int* flag) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_la_error, sizeof(int));
    if (e != cudaSuccess || *flag == 0) return e;
    const int zero = 0;
    return cudaMemcpyToSymbol(g_la_error, &zero, sizeof(int));
}

}  // namespace gdr
