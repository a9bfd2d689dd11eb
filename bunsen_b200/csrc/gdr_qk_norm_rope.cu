// RMS norm of every query and key head with the position rotation in the
// same pass, and its gradient.
//
// A head vector x of d features, r = 1 / sqrt(mean(x^2) + eps), weight u:
//   n = x r u;  the first `rot` features of n rotate in pairs by the
//   position's angles: (y1, y2) = (n1 cos - n2 sin, n2 cos + n1 sin),
// the pairs (i, i + rot/2), or (2i, 2i+1) when interleaved. The gradient:
//   dn = rotation by the opposite angles of dy;  du = sum over rows x r dn;
//   dx = r (u dn - x r^2 mean(x u dn)).
// Every sum and product is f32; the one rounding is the output's own.
//
// Bound by HBM: one read and one write of q and k (for the gradient two reads
// and one write). The vector kernels give a lane 8 features, both of every pair it
// rotates among them (two runs of four: 8-byte accesses for 16-bit types), 8,
// 16 or 32 lanes to a row, so a warp covers one to four rows per instruction,
// the row's sums by shuffles inside its lanes; products by f32 pairs. (With 8
// consecutive features a lane, partners by shuffle and single products it was
// bound by instructions: 165 us for 32768 x 32 heads of 128, against 102 us, 5.4 TB/s,
// 0.83 of the copy rate; the gradient of 16384 x 32 heads 230 us against 98 us, 4.2 TB/s.)
// A warp takes kRows rows of one token per lane group, all of their loads issued before
// any is computed; the token's angles are read once for them. Other shapes (odd
// widths, unaligned rows) take one warp per row, scalar accesses.
//
// The weights' gradient is summed without atomics, so equal calls give equal
// bits: a fixed grid, each lane's sums over its rows in registers, each
// block's in shared memory in warp order, then one kernel over the blocks.
#include "gdr_common.cuh"
#include "gdr_f32x2.cuh"
#include "gdr_qk_norm_rope.cuh"

namespace gdr {

// Device-side failures since the last gdr_device_error: bit 1, a position
// outside the angle tables (its rows are left unwritten).
__device__ int g_rope_error;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxD = 256;
constexpr int kWaves = 4;  // of CTAs of the outputs' kernels

// The 8 features of a lane: two runs of four, at `o0` and `o1`, so that both
// features of a rotated pair are one lane's: 4 li and rot / 2 + 4 li of the rotated
// part, 8 li and 8 li + 4 behind it or where pairs are neighbours.
template <typename T>
struct Raw {
    uint2 v[sizeof(T) == 4 ? 4 : 2];  // as loaded, so that several rows are in flight
};
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int o0, int o1) {
    Raw<T> r;
    if constexpr (sizeof(T) == 4) {
        const uint4 a = *reinterpret_cast<const uint4*>(row + o0);
        const uint4 b = *reinterpret_cast<const uint4*>(row + o1);
        r.v[0] = make_uint2(a.x, a.y), r.v[1] = make_uint2(a.z, a.w);
        r.v[2] = make_uint2(b.x, b.y), r.v[3] = make_uint2(b.z, b.w);
    } else {
        r.v[0] = *reinterpret_cast<const uint2*>(row + o0);
        r.v[1] = *reinterpret_cast<const uint2*>(row + o1);
    }
    return r;
}
// As pairs of f32.
template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, uint64_t (&x)[4]) {
    const T* e = reinterpret_cast<const T*>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = pair(to_f32(e[2 * i]), to_f32(e[2 * i + 1]));
}
template <typename T>
__device__ __forceinline__ void store(T* row, int o0, int o1, const uint64_t (&x)[4]) {
    Raw<T> r;
    T* e = reinterpret_cast<T*>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float u, v;
        unpair(x[i], u, v);
        e[2 * i] = from_f32<T>(u);
        e[2 * i + 1] = from_f32<T>(v);
    }
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint4*>(row + o0) = make_uint4(r.v[0].x, r.v[0].y, r.v[1].x, r.v[1].y);
        *reinterpret_cast<uint4*>(row + o1) = make_uint4(r.v[2].x, r.v[2].y, r.v[3].x, r.v[3].y);
    } else {
        *reinterpret_cast<uint2*>(row + o0) = r.v[0];
        *reinterpret_cast<uint2*>(row + o1) = r.v[1];
    }
}
__device__ __forceinline__ void load_pairs(const float* row, int o0, int o1, uint64_t (&x)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(row + o0);
    const float4 b = *reinterpret_cast<const float4*>(row + o1);
    x[0] = pair(a.x, a.y), x[1] = pair(a.z, a.w), x[2] = pair(b.x, b.y), x[3] = pair(b.z, b.w);
}
__device__ __forceinline__ float sum_pair(uint64_t x) {
    float u, v;
    unpair(x, u, v);
    return u + v;
}

template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The angles of a lane's four pairs, as its features' products want them: neighbours
// (u, v) -> (u, v) (c, c) + (v, u) (-s, s); else pairs of the two runs.
template <bool kInter>
struct Angles {
    uint64_t c[kInter ? 4 : 2], s[kInter ? 4 : 2], n[kInter ? 1 : 2];
};
template <bool kInter>
__device__ __forceinline__ Angles<kInter> angles(const float4& c, const float4& s) {
    Angles<kInter> a;
    if constexpr (kInter) {
        a.c[0] = pair(c.x, c.x), a.c[1] = pair(c.y, c.y), a.c[2] = pair(c.z, c.z), a.c[3] = pair(c.w, c.w);
        a.s[0] = pair(-s.x, s.x), a.s[1] = pair(-s.y, s.y), a.s[2] = pair(-s.z, s.z), a.s[3] = pair(-s.w, s.w);
    } else {
        a.c[0] = pair(c.x, c.y), a.c[1] = pair(c.z, c.w);
        a.s[0] = pair(s.x, s.y), a.s[1] = pair(s.z, s.w);
        a.n[0] = pair(-s.x, -s.y), a.n[1] = pair(-s.z, -s.w);
    }
    return a;
}
template <bool kInter>
__device__ __forceinline__ void rotate(const Angles<kInter>& a, uint64_t (&x)[4]) {
    if constexpr (kInter) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u, v;
            unpair(x[i], u, v);
            x[i] = fma2(x[i], a.c[i], mul2(pair(v, u), a.s[i]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t u = x[i], v = x[2 + i];
            x[i] = fma2(u, a.c[i], mul2(v, a.n[i]));
            x[2 + i] = fma2(v, a.c[i], mul2(u, a.s[i]));
        }
    }
}

__device__ __forceinline__ bool in_tables(const NormRope& p, int pos) {
    return pos >= 0 && pos < p.table_rows;
}
__device__ __forceinline__ void report_position() {
    if ((threadIdx.x & 31) == 0) atomicOr(&g_rope_error, 2);
}

// The weights' sums of a block into its row of `part` [gridDim.x][2][d]: the
// warps' sums in warp order.
__device__ __forceinline__ void block_weights(const NormRope& p, float (*acc)[kMaxD], float* part) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += kThreads) {
        const int which = i / p.d, e = i - which * p.d;
        float s = 0.f;
        for (int w = 0; w < kWarps; ++w) s += acc[2 * w + which][e];
        part[static_cast<int64_t>(blockIdx.x) * 2 * p.d + i] = s;
    }
}

// The outputs, or (kGrad) the gradients. A warp works on q or on k throughout (in
// proportion to their units; its weights stay in registers), a unit of kRows x
// (32 / G) heads of one token at a time, every load before the first use.
// `q_warps` of all warps work on q. Rows past the last head are the last again,
// not stored.
template <typename T, int G, int kRows, bool kInter, bool kGrad>
__global__ void __launch_bounds__(kThreads, kGrad ? 2 : 4)
norm_rope_vec(const NormRope p, uint32_t q_warps, float* part) {
    constexpr int kSub = 32 / G, kPer = kSub * kRows;
    __shared__ float acc[kGrad ? 2 * kWarps : 1][kMaxD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int li = lane % G, sub = lane / G;
    const bool live = 8 * li < p.d, turned = 8 * li < p.rot;
    int o0 = 8 * li, o1 = 8 * li + 4;
    if (turned && !kInter) o0 = 4 * li, o1 = p.rot / 2 + 4 * li;
    if (!live) o0 = o1 = 0;
    const uint32_t me = blockIdx.x * kWarps + warp;
    const bool is_k = me >= q_warps;
    const int heads = is_k ? p.heads_k : p.heads_q;
    const uint32_t each = (heads + kPer - 1) / kPer;  // units of a token
    const uint32_t units = static_cast<uint32_t>(p.tokens) * each;
    const uint32_t step = is_k ? gridDim.x * kWarps - q_warps : q_warps;
    const T* x = static_cast<const T*>(is_k ? p.k : p.q);
    const T* dy = static_cast<const T*>(is_k ? p.dk_out : p.dq_out);
    T* y = static_cast<T*>(is_k ? p.k_out : p.q_out);
    const int64_t token_stride = is_k ? p.k_token : p.q_token, head_stride = is_k ? p.k_head : p.q_head;
    const float* weight = is_k ? p.k_weight : p.q_weight;
    uint64_t wt[4], wsum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) wt[j] = pair(1.f, 1.f), wsum[j] = 0;
    if (weight != nullptr) load_pairs(weight, o0, o1, wt);
    const float inv_d = 1.f / p.d;
    const uint32_t first = is_k ? me - q_warps : me;
    // The gradient's CTAs are few and stay (their weights' sums): a unit ahead they read
    // its position, which the angles' loads wait for. (Its rows too: 113 us against 98.)
    int next = kGrad && first < units ? p.positions[first / each] : 0;
#pragma unroll 1
    for (uint32_t u = first; u < units; u += step) {
        const uint32_t token = u / each;
        const int head0 = static_cast<int>(u - token * each) * kPer + sub;
        const T* row = x + token * token_stride;
        const int64_t flat = static_cast<int64_t>(token) * heads;
        Raw<T> rx[kRows], rd[kGrad ? kRows : 1];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int h = min(head0 + i * kSub, heads - 1);
            rx[i] = load_raw(row + h * head_stride, o0, o1);
            if constexpr (kGrad) rd[i] = load_raw(dy + (flat + h) * p.d, o0, o1);
        }
        const int pos = kGrad ? next : p.positions[token];
        if (kGrad && u + step < units) next = p.positions[(u + step) / each];
        if (!in_tables(p, pos)) {
            report_position();
            continue;
        }
        float4 c = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
        if (turned) {
            const int64_t at = static_cast<int64_t>(pos) * (p.rot / 2) + 4 * li;
            c = *reinterpret_cast<const float4*>(p.cos + at);
            sn = *reinterpret_cast<const float4*>(p.sin + at);
            if (kGrad) sn = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);  // the opposite angles
        }
        const Angles<kInter> a = angles<kInter>(c, sn);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            uint64_t v[4], ss = 0;
            unpack(rx[i], v);
#pragma unroll
            for (int j = 0; j < 4; ++j) ss = fma2(v[j], v[j], ss);
            const bool mine = live && head0 + i * kSub < heads;
            if constexpr (!kGrad) {
                const float r =
                    rsqrtf(fmaf(group_sum<G>(live ? sum_pair(ss) : 0.f), inv_d, p.eps));
                const uint64_t rr = pair(r, r);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], mul2(wt[j], rr));
                rotate(a, v);
            } else {
                uint64_t g[4], t[4], dot = 0;
                unpack(rd[i], g);
                rotate(a, g);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    t[j] = mul2(v[j], g[j]);
                    dot = fma2(t[j], wt[j], dot);
                }
                const float r =
                    rsqrtf(fmaf(group_sum<G>(live ? sum_pair(ss) : 0.f), inv_d, p.eps));
                // (Step by step: r^3 leaves f32 where r and the gradient do not.)
                const float back =
                    -group_sum<G>(live ? sum_pair(dot) : 0.f) * inv_d * r * r * r;
                const float r_own = mine ? r : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    wsum[j] = fma2(t[j], pair(r_own, r_own), wsum[j]);
                    v[j] = fma2(v[j], pair(back, back), mul2(g[j], mul2(wt[j], pair(r, r))));
                }
            }
            if (mine) store(y + (flat + head0 + i * kSub) * p.d, o0, o1, v);
        }
    }
    if constexpr (kGrad) {
        if (part == nullptr) return;
        for (int e = lane; e < p.d; e += 32) acc[2 * warp + !is_k][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float u, v;
            unpair(wsum[j >> 1], u, v);
            float t = j & 1 ? v : u;
#pragma unroll
            for (int o = G; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (sub == 0 && live) acc[2 * warp + is_k][(j < 4 ? o0 : o1 - 4) + j] = t;
        }
        block_weights(p, acc, part);
    }
}

// Any width up to 256, any strides: one warp per row, lane l holding features
// l, l + 32, ...; a rotation partner is read again from the row.
template <typename T, bool kGrad>
__global__ void __launch_bounds__(kThreads)
norm_rope_any(const NormRope p, int64_t rows, float* part) {
    constexpr int kE = kMaxD / 32;
    __shared__ float acc[kGrad ? 2 * kWarps : 1][kMaxD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.rot / 2;
    float wsum[2][kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) wsum[0][j] = wsum[1][j] = 0.f;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp; row < rows; row += step) {
        const int64_t token = row / (p.heads_q + p.heads_k);
        int h = static_cast<int>(row - token * (p.heads_q + p.heads_k));
        const bool is_k = h >= p.heads_q;
        if (is_k) h -= p.heads_q;
        const int64_t pos = p.positions[token];
        if (!in_tables(p, static_cast<int>(pos))) {
            report_position();
            continue;
        }
        const T* x = is_k ? static_cast<const T*>(p.k) + token * p.k_token + h * p.k_head
                          : static_cast<const T*>(p.q) + token * p.q_token + h * p.q_head;
        const int64_t flat = (token * (is_k ? p.heads_k : p.heads_q) + h) * p.d;
        const T* dy = kGrad ? static_cast<const T*>(is_k ? p.dk_out : p.dq_out) + flat : nullptr;
        T* y = static_cast<T*>(is_k ? p.k_out : p.q_out) + flat;
        const float* weight = is_k ? p.k_weight : p.q_weight;
        auto wt = [&](int e) { return weight != nullptr ? weight[e] : 1.f; };
        float v[kE], ss = 0.f;
#pragma unroll
        for (int j = 0; j < kE; ++j) {
            const int e = lane + 32 * j;
            v[j] = e < p.d ? to_f32(x[e]) : 0.f;
            ss = fmaf(v[j], v[j], ss);
        }
        const float r = 1.f / sqrtf(warp_sum(ss) / p.d + p.eps);
        float g[kE], dot = 0.f;  // the output, or the gradient of n
#pragma unroll
        for (int j = 0; j < kE; ++j) {
            const int e = lane + 32 * j;
            g[j] = 0.f;
            if (e >= p.d) continue;
            const float own = kGrad ? to_f32(dy[e]) : v[j] * r * wt(e);
            g[j] = own;
            if (e < p.rot) {
                const bool low = p.interleaved ? (e & 1) == 0 : e < half;
                const int pe = p.interleaved ? e ^ 1 : (low ? e + half : e - half);
                const int ai = p.interleaved ? e / 2 : (low ? e : e - half);
                const float other = kGrad ? to_f32(dy[pe]) : to_f32(x[pe]) * r * wt(pe);
                const float c = p.cos[pos * half + ai], s = p.sin[pos * half + ai];
                g[j] = own * c + (low == kGrad ? other : -other) * s;
            }
            if (kGrad) dot = fmaf(v[j] * wt(e), g[j], dot);
        }
        const float back = kGrad ? warp_sum(dot) / p.d * r * r : 0.f;
#pragma unroll
        for (int j = 0; j < kE; ++j) {
            const int e = lane + 32 * j;
            if (e >= p.d) continue;
            if (kGrad) {
                const float t = v[j] * r * g[j];
                if (is_k) wsum[1][j] += t;
                else wsum[0][j] += t;
                y[e] = from_f32<T>(r * (wt(e) * g[j] - v[j] * back));
            } else {
                y[e] = from_f32<T>(g[j]);
            }
        }
    }
    if constexpr (kGrad) {
        if (part == nullptr) return;
#pragma unroll
        for (int j = 0; j < kE; ++j) {
            acc[2 * warp][lane + 32 * j] = wsum[0][j];
            acc[2 * warp + 1][lane + 32 * j] = wsum[1][j];
        }
        block_weights(p, acc, part);
    }
}

// d_weight[e] = sum over the blocks' rows of `part`: 8 columns a CTA, 32 runs of rows
// joined in order.
__global__ void __launch_bounds__(kThreads)
sum_weights(const float* part, int blocks, int d, float* dq_weight, float* dk_weight) {
    __shared__ float run[kThreads];
    const int c = threadIdx.x & 7, r = threadIdx.x >> 3;
    const int i = blockIdx.x * 8 + c;  // of 2 d
    float s = 0.f;
    if (i < 2 * d)
#pragma unroll 4
        for (int b = r; b < blocks; b += kThreads / 8) s += part[static_cast<int64_t>(b) * 2 * d + i];
    run[threadIdx.x] = s;
    __syncthreads();
    if (r != 0 || i >= 2 * d) return;
    s = 0.f;
    for (int w = 0; w < kThreads / 8; ++w) s += run[8 * w + c];
    float* out = i < d ? dq_weight : dk_weight;
    if (out != nullptr) out[i < d ? i : i - d] = s;
}

// Accesses of four features need these; else the scalar kernel.
bool vectors(const NormRope& p) {
    if (p.d % 8 || p.rot % 8) return false;
    if (p.q_token % 4 || p.q_head % 4 || p.k_token % 4 || p.k_head % 4) return false;
    uintptr_t a = 0;
    for (const void* x : {p.q, p.k, static_cast<const void*>(p.q_out),
                          static_cast<const void*>(p.k_out), p.dq_out, p.dk_out,
                          static_cast<const void*>(p.cos), static_cast<const void*>(p.sin),
                          static_cast<const void*>(p.q_weight),
                          static_cast<const void*>(p.k_weight)})
        a |= reinterpret_cast<uintptr_t>(x);
    return (a & 15) == 0;
}

// What a call launches.
struct Launch {
    int blocks;
    uint32_t q_warps;  // vector kernels
};

int sm_count() {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

int lanes_of(const NormRope& p) { return p.d <= 64 ? 8 : p.d <= 128 ? 16 : 32; }
// Rows a lane group takes at once: four (the gradient's at 128 registers a thread, two CTAs
// an SM: 98 us where three CTAs, two rows and 80 registers, which spilled, took 118); one
// where that leaves SMs without work.
int rows_of(const NormRope& p) {
    constexpr int rows = 4;
    const int64_t units =
        p.tokens * norm_rope_units(p.heads_q, p.heads_k, 32 / lanes_of(p) * rows);
    return units < 2 * kWarps * sm_count() ? 1 : rows;
}

Launch launch_of(const NormRope& p) {
    const int per = vectors(p) ? 32 / lanes_of(p) * rows_of(p) : 1;
    const int64_t units = p.tokens * norm_rope_units(p.heads_q, p.heads_k, per);
    const int64_t want = (units + kWarps) / kWarps;
    const int64_t most = static_cast<int64_t>(sm_count()) * (p.dq_out != nullptr ? 2 : kWaves * 4);
    Launch l;
    l.blocks = static_cast<int>(want < 1 ? 1 : want < most ? want : most);
    l.q_warps = norm_rope_q_warps(static_cast<int64_t>(l.blocks) * kWarps, p.heads_q, p.heads_k, per);
    return l;
}

template <typename T, int G, bool kInter>
void start_rows(const NormRope& p, float* part, Launch l, cudaStream_t s) {
    const bool one = rows_of(p) == 1;
    if (p.dq_out != nullptr)
        (one ? norm_rope_vec<T, G, 1, kInter, true> : norm_rope_vec<T, G, 4, kInter, true>)
            <<<l.blocks, kThreads, 0, s>>>(p, l.q_warps, part);
    else
        (one ? norm_rope_vec<T, G, 1, kInter, false> : norm_rope_vec<T, G, 4, kInter, false>)
            <<<l.blocks, kThreads, 0, s>>>(p, l.q_warps, nullptr);
}

template <typename T, int G>
void start_pairs(const NormRope& p, float* part, Launch l, cudaStream_t s) {
    p.interleaved ? start_rows<T, G, true>(p, part, l, s) : start_rows<T, G, false>(p, part, l, s);
}

template <typename T>
void start(const NormRope& p, float* part, Launch l, cudaStream_t s) {
    if (!vectors(p)) {
        const int64_t rows = p.tokens * (p.heads_q + p.heads_k);
        if (p.dq_out != nullptr)
            norm_rope_any<T, true><<<l.blocks, kThreads, 0, s>>>(p, rows, part);
        else
            norm_rope_any<T, false><<<l.blocks, kThreads, 0, s>>>(p, rows, nullptr);
        return;
    }
    switch (lanes_of(p)) {
        case 8: start_pairs<T, 8>(p, part, l, s); break;
        case 16: start_pairs<T, 16>(p, part, l, s); break;
        default: start_pairs<T, 32>(p, part, l, s);
    }
}

}  // namespace

int norm_rope_max_d() { return kMaxD; }

// Blocks of a gradient call: its weights' partial sums are one row of 2 d each.
int norm_rope_blocks(const NormRope& p) { return launch_of(p).blocks; }

cudaError_t launch_norm_rope(const NormRope& p, float* part, cudaStream_t s) {
    const Launch l = launch_of(p);
    switch (p.dtype) {
        case GDR_DTYPE_BF16: start<__nv_bfloat16>(p, part, l, s); break;
        case GDR_DTYPE_F16: start<__half>(p, part, l, s); break;
        default: start<float>(p, part, l, s); break;
    }
    if (part != nullptr)
        sum_weights<<<(2 * p.d + 7) / 8, kThreads, 0, s>>>(part, l.blocks, p.d, p.dq_weight,
                                                           p.dk_weight);
    return cudaGetLastError();
}

cudaError_t take_rope_error(int* flag) {
    cudaError_t e = cudaMemcpyFromSymbol(flag, g_rope_error, sizeof(int));
    if (e != cudaSuccess || *flag == 0) return e;
    const int zero = 0;
    return cudaMemcpyToSymbol(g_rope_error, &zero, sizeof(int));
}

}  // namespace gdr
