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
// and one write). The vector kernels give a lane 8 consecutive features (one
// 16-byte access for 16-bit types), 8, 16 or 32 lanes to a row, so a warp
// covers one to four rows per instruction, the row's sums by shuffles inside
// its lanes, a rotation partner by one shuffle (or in the lane itself when
// interleaved). A warp takes kRows rows of one token per lane group, all loads
// issued before any is used; the token's angles are read once for them. Other
// shapes (odd widths, unaligned rows) take one warp per row, scalar accesses.
//
// The weights' gradient is summed without atomics, so equal calls give equal
// bits: a fixed grid, each lane's sums over its rows in registers, each
// block's in shared memory in warp order, then one kernel over the blocks.
#include "gdr_common.cuh"
#include "gdr_qk_norm_rope.cuh"

namespace gdr {

// Device-side failures since the last gdr_device_error: bit 1, a position
// outside the angle tables (its rows are left unwritten).
__device__ int g_rope_error;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxD = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* src, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(src)[0];
        const float4 b = reinterpret_cast<const float4*>(src)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(src);
        const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 a;
        T* e = reinterpret_cast<T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
        *reinterpret_cast<uint4*>(dst) = a;
    }
}

// A raw row piece as loaded, so that several are in flight before one is used.
template <typename T>
struct Raw {
    uint4 v[sizeof(T) == 4 ? 2 : 1];
};
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* src) {
    Raw<T> r;
    r.v[0] = reinterpret_cast<const uint4*>(src)[0];
    if constexpr (sizeof(T) == 4) r.v[1] = reinterpret_cast<const uint4*>(src)[1];
    return r;
}
template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&x)[8]) {
    const T* e = reinterpret_cast<const T*>(r.v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}

template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The angles of a lane's 8 features: cos and sin for each, or, interleaved,
// for its 4 pairs (the other 4 unused). Lanes past the rotated part: none.
struct Angles {
    float c[8], s[8];
};

__device__ __forceinline__ void load_angles(const NormRope& p, int64_t pos, int e0, Angles& a) {
    const int half = p.rot / 2;
    if (e0 >= p.rot) return;
    if (p.interleaved) {
        const float4 c = *reinterpret_cast<const float4*>(p.cos + pos * half + e0 / 2);
        const float4 s = *reinterpret_cast<const float4*>(p.sin + pos * half + e0 / 2);
        a.c[0] = c.x; a.c[1] = c.y; a.c[2] = c.z; a.c[3] = c.w;
        a.s[0] = s.x; a.s[1] = s.y; a.s[2] = s.z; a.s[3] = s.w;
    } else {
        const int i = e0 < half ? e0 : e0 - half;
        load8(p.cos + pos * half + i, a.c);
        load8(p.sin + pos * half + i, a.s);
    }
}

// Rotates a lane's 8 features in place (sign -1: by the opposite angles).
// Every lane of the warp calls it: the partner features come by shuffle.
__device__ __forceinline__ void rotate8(const NormRope& p, int e0, const Angles& a, float sign,
                                        float (&x)[8]) {
    if (p.interleaved) {
        if (e0 < p.rot) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = x[2 * i], v = x[2 * i + 1], s = sign * a.s[i];
                x[2 * i] = u * a.c[i] - v * s;
                x[2 * i + 1] = v * a.c[i] + u * s;
            }
        }
        return;
    }
    const int half = p.rot / 2, lane = threadIdx.x & 31;
    const bool low = e0 < half;
    const int partner = e0 >= p.rot ? lane : low ? lane + half / 8 : lane - half / 8;
    const float s = low ? -sign : sign;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float other = __shfl_sync(0xffffffffu, x[i], partner);
        if (e0 < p.rot) x[i] = x[i] * a.c[i] + s * other * a.s[i];
    }
}

// Which rows a warp's unit of work covers: `per` heads of q, or of k, of one
// token.
struct Unit {
    int64_t token;
    int head0, heads;  // first head of the unit, heads of the tensor
    bool is_k;
};
__device__ __forceinline__ Unit unit_of(const NormRope& p, int64_t unit, int per) {
    const int nq = (p.heads_q + per - 1) / per, nk = (p.heads_k + per - 1) / per;
    Unit u;
    u.token = unit / (nq + nk);
    int b = static_cast<int>(unit - u.token * (nq + nk));
    u.is_k = b >= nq;
    if (u.is_k) b -= nq;
    u.head0 = b * per;
    u.heads = u.is_k ? p.heads_k : p.heads_q;
    return u;
}

__device__ __forceinline__ bool position_of(const NormRope& p, int64_t token, int64_t& pos) {
    pos = p.positions[token];
    if (pos >= 0 && pos < p.table_rows) return true;
    if ((threadIdx.x & 31) == 0) atomicOr(&g_rope_error, 2);
    return false;
}

template <typename T, int G, int kRows>
__global__ void __launch_bounds__(kThreads)
norm_rope_vec(const NormRope p, int64_t units) {
    constexpr int kPer = (32 / G) * kRows;
    const int lane = threadIdx.x & 31, li = lane % G, sub = lane / G, e0 = 8 * li;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
    if (unit >= units) return;
    const Unit u = unit_of(p, unit, kPer);
    int64_t pos;
    if (!position_of(p, u.token, pos)) return;
    const T* x = static_cast<const T*>(u.is_k ? p.k : p.q) +
                 u.token * (u.is_k ? p.k_token : p.q_token);
    const int64_t hstride = u.is_k ? p.k_head : p.q_head;
    T* y = static_cast<T*>(u.is_k ? p.k_out : p.q_out) + u.token * u.heads * p.d;
    const float* weight = u.is_k ? p.k_weight : p.q_weight;
    const bool live = e0 < p.d;
    Raw<T> raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        raw[i] = Raw<T>{};
        const int h = u.head0 + i * (32 / G) + sub;
        if (live && h < u.heads) raw[i] = load_raw(x + h * hstride + e0);
    }
    Angles a;
    load_angles(p, pos, e0, a);
    float wt[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wt[i] = 1.f;
    if (weight != nullptr && live) load8(weight + e0, wt);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int h = u.head0 + i * (32 / G) + sub;
        float v[8], ss = 0.f;
        unpack(raw[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        const float r = 1.f / sqrtf(group_sum<G>(ss) / p.d + p.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= r * wt[j];
        rotate8(p, e0, a, 1.f, v);
        if (live && h < u.heads) store8(y + static_cast<int64_t>(h) * p.d + e0, v);
    }
}

// The weights' sums of a block into its row of `part` [gridDim.x][2][d]: the
// warps' sums in warp order (row groups of a warp first).
__device__ __forceinline__ void block_weights(const NormRope& p, float (*acc)[kMaxD], float* part) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += kThreads) {
        const int which = i / p.d, e = i - which * p.d;
        float s = 0.f;
        for (int w = 0; w < kWarps; ++w) s += acc[2 * w + which][e];
        part[static_cast<int64_t>(blockIdx.x) * 2 * p.d + i] = s;
    }
}

template <typename T, int G, int kRows>
__global__ void __launch_bounds__(kThreads)
norm_rope_grad_vec(const NormRope p, int64_t units, float* part) {
    constexpr int kPer = (32 / G) * kRows;
    __shared__ float acc[2 * kWarps][kMaxD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int li = lane % G, sub = lane / G, e0 = 8 * li;
    const bool live = e0 < p.d;
    float wsum[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) wsum[0][j] = wsum[1][j] = 0.f;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
    for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp; unit < units;
         unit += step) {
        const Unit u = unit_of(p, unit, kPer);
        int64_t pos;
        if (!position_of(p, u.token, pos)) continue;
        const T* x = static_cast<const T*>(u.is_k ? p.k : p.q) +
                     u.token * (u.is_k ? p.k_token : p.q_token);
        const int64_t hstride = u.is_k ? p.k_head : p.q_head;
        const int64_t row0 = u.token * u.heads;
        const T* dy = static_cast<const T*>(u.is_k ? p.dk_out : p.dq_out);
        T* dx = static_cast<T*>(u.is_k ? p.k_out : p.q_out);
        const float* weight = u.is_k ? p.k_weight : p.q_weight;
        Raw<T> rx[kRows], rd[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            rx[i] = Raw<T>{};
            rd[i] = Raw<T>{};
            const int h = u.head0 + i * (32 / G) + sub;
            if (live && h < u.heads) {
                rx[i] = load_raw(x + h * hstride + e0);
                rd[i] = load_raw(dy + (row0 + h) * p.d + e0);
            }
        }
        Angles a;
        load_angles(p, pos, e0, a);
        float wt[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) wt[i] = 1.f;
        if (weight != nullptr && live) load8(weight + e0, wt);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int h = u.head0 + i * (32 / G) + sub;
            float v[8], g[8], ss = 0.f, dot = 0.f;
            unpack(rx[i], v);
            unpack(rd[i], g);
            rotate8(p, e0, a, -1.f, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ss = fmaf(v[j], v[j], ss);
                dot = fmaf(v[j] * wt[j], g[j], dot);
            }
            const float r = 1.f / sqrtf(group_sum<G>(ss) / p.d + p.eps);
            const float back = group_sum<G>(dot) / p.d * (r * r);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float t = v[j] * r * g[j];
                if (u.is_k) wsum[1][j] += t;
                else wsum[0][j] += t;
                v[j] = r * (wt[j] * g[j] - v[j] * back);
            }
            if (live && h < u.heads) store8(dx + (row0 + h) * p.d + e0, v);
        }
    }
    if (part == nullptr) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float x = wsum[w][j];
#pragma unroll
            for (int o = G; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            if (sub == 0 && live) acc[2 * warp + w][e0 + j] = x;
        }
    block_weights(p, acc, part);
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
        const Unit u = unit_of(p, row, 1);
        int64_t pos;
        if (!position_of(p, u.token, pos)) continue;
        const T* x = u.is_k ? static_cast<const T*>(p.k) + u.token * p.k_token + u.head0 * p.k_head
                            : static_cast<const T*>(p.q) + u.token * p.q_token + u.head0 * p.q_head;
        const int64_t flat = (u.token * u.heads + u.head0) * p.d;
        const T* dy = kGrad ? static_cast<const T*>(u.is_k ? p.dk_out : p.dq_out) + flat : nullptr;
        T* y = static_cast<T*>(u.is_k ? p.k_out : p.q_out) + flat;
        const float* weight = u.is_k ? p.k_weight : p.q_weight;
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
        const float back = kGrad ? warp_sum(dot) / p.d * (r * r) : 0.f;
#pragma unroll
        for (int j = 0; j < kE; ++j) {
            const int e = lane + 32 * j;
            if (e >= p.d) continue;
            if (kGrad) {
                const float t = v[j] * r * g[j];
                if (u.is_k) wsum[1][j] += t;
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

// d_weight[e] = sum over the blocks' rows of `part`, 8 warps each a run of
// blocks, joined in order.
__global__ void __launch_bounds__(kThreads)
sum_weights(const float* part, int blocks, int d, float* dq_weight, float* dk_weight) {
    __shared__ float run[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + lane;  // of 2 d
    const int each = (blocks + kWarps - 1) / kWarps;
    float s = 0.f;
    if (i < 2 * d)
        for (int b = warp * each; b < min(blocks, (warp + 1) * each); ++b)
            s += part[static_cast<int64_t>(b) * 2 * d + i];
    run[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || i >= 2 * d) return;
    s = 0.f;
    for (int w = 0; w < kWarps; ++w) s += run[w][lane];
    float* out = i < d ? dq_weight : dk_weight;
    if (out != nullptr) out[i < d ? i : i - d] = s;
}

int64_t unit_count(const NormRope& p, int per) {
    return p.tokens * ((p.heads_q + per - 1) / per + (p.heads_k + per - 1) / per);
}

// 16-byte accesses need these; else the scalar kernel.
bool vectors(const NormRope& p) {
    const int es = p.dtype == GDR_DTYPE_F32 ? 4 : 2, e16 = 16 / es;
    if (p.d % 8 || (p.interleaved ? p.rot % 8 : (p.rot / 2) % 8)) return false;
    if (p.q_token % e16 || p.q_head % e16 || p.k_token % e16 || p.k_head % e16) return false;
    uintptr_t a = 0;
    for (const void* x : {p.q, p.k, static_cast<const void*>(p.q_out),
                          static_cast<const void*>(p.k_out), p.dq_out, p.dk_out,
                          static_cast<const void*>(p.cos), static_cast<const void*>(p.sin),
                          static_cast<const void*>(p.q_weight),
                          static_cast<const void*>(p.k_weight)})
        a |= reinterpret_cast<uintptr_t>(x);
    return (a & 15) == 0;
}

template <typename T, int G, int kRows>
void start_vec(const NormRope& p, float* part, int blocks, cudaStream_t s) {
    const int64_t units = unit_count(p, (32 / G) * kRows);
    if (p.dq_out != nullptr)
        norm_rope_grad_vec<T, G, kRows><<<blocks, kThreads, 0, s>>>(p, units, part);
    else
        norm_rope_vec<T, G, kRows>
            <<<static_cast<unsigned>((units + kWarps - 1) / kWarps), kThreads, 0, s>>>(p, units);
}

template <typename T>
void start(const NormRope& p, float* part, int blocks, cudaStream_t s) {
    if (!vectors(p)) {
        const int64_t rows = unit_count(p, 1);
        if (p.dq_out != nullptr)
            norm_rope_any<T, true><<<blocks, kThreads, 0, s>>>(p, rows, part);
        else
            norm_rope_any<T, false><<<blocks, kThreads, 0, s>>>(p, rows, nullptr);
        return;
    }
    // Four rows per lane group, or one when that leaves SMs without work.
    const bool few = unit_count(p, (p.d <= 64 ? 4 : p.d <= 128 ? 2 : 1) * 4) < 148 * kWarps;
    if (p.d <= 64) few ? start_vec<T, 8, 1>(p, part, blocks, s) : start_vec<T, 8, 4>(p, part, blocks, s);
    else if (p.d <= 128) few ? start_vec<T, 16, 1>(p, part, blocks, s) : start_vec<T, 16, 4>(p, part, blocks, s);
    else few ? start_vec<T, 32, 1>(p, part, blocks, s) : start_vec<T, 32, 4>(p, part, blocks, s);
}

}  // namespace

int norm_rope_max_d() { return kMaxD; }

// Blocks of a gradient call (its weights' partial sums: one row of 2 d each)
// and of the scalar forward kernel.
int norm_rope_blocks(const NormRope& p) {
    const int64_t warps = (unit_count(p, 1) + 3) / 4;
    const int64_t want = (warps + kWarps - 1) / kWarps;
    return static_cast<int>(want < 148 * 4 ? (want > 0 ? want : 1) : 148 * 4);
}

cudaError_t launch_norm_rope(const NormRope& p, float* part, cudaStream_t s) {
    const int blocks = norm_rope_blocks(p);
    switch (p.dtype) {
        case GDR_DTYPE_BF16: start<__nv_bfloat16>(p, part, blocks, s); break;
        case GDR_DTYPE_F16: start<__half>(p, part, blocks, s); break;
        default: start<float>(p, part, blocks, s); break;
    }
    if (part != nullptr)
        sum_weights<<<(2 * p.d + 31) / 32, kThreads, 0, s>>>(part, blocks, p.d, p.dq_weight,
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
