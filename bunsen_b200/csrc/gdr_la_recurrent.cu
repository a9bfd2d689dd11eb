// The decayed linear attention core (gdr_la.cuh) one position at a time.
//
//   forward:   S <- w S + sigma b_t c_t^T;  out_t = tau a_t . S
//   backward:  S <- S + sigma b_t c_t^T;  out_t = tau a_t . S;  S <- w S
//
// A state's columns evolve independently (column j needs a, b and its own
// c[j]), so a CTA of 256 threads takes one (sequence, head) and a slab of
// columns, the slab's state in registers: kLanes lanes cover the slab's
// columns (kVec each), 256 / kLanes row groups take rows rg, rg + RG, ... .
// Per position one exchange of a and b and one of the partial sums over d_b.
//
// A decode step (one position a row) is bound by HBM: 8 d_b d_c bytes of
// state against a few hundred bytes of operands. Which slab: 128 columns
// (a warp reads whole 512-byte state rows) when that fills the GPU, else 32
// columns, four times the CTAs with a quarter of the loads each, for the
// latency of small batches. 256 rows of 32 heads, d = 128: 164 us, 6.6 TB/s, the copy
// rate; one row 3 us on the device.
#include "gdr_la.cuh"

namespace gdr {

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float la_load(const void* base, int64_t i) {
    return to_f32(static_cast<const T*>(base)[i]);
}

template <typename T, int kLanes, int kVec, int kRows>
__global__ void __launch_bounds__(kThreads)
la_recurrent(const LaCore p) {
    constexpr int kRG = kThreads / kLanes, kSlab = kLanes * kVec, kWarps = kThreads / 32;
    __shared__ float ab[2][2][kRG * kRows];  // [position parity][a, b][row]
    __shared__ float red[2][kWarps][kSlab];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int li = tid % kLanes, rg = tid / kLanes;
    const int h = blockIdx.x, s = blockIdx.y;
    const int col0 = static_cast<int>(blockIdx.z) * kSlab, col = col0 + li * kVec;
    int64_t t0, t1;
    la_span(p, s, t0, t1);
    if (p.steps_most >= 0 && t1 - t0 > p.steps_most) return;
    const int64_t hs = (static_cast<int64_t>(s) * p.heads + h) * p.d_b * p.d_c;
    const int64_t rs = p.state_t ? 1 : p.d_c, cs = p.state_t ? p.d_b : 1;  // state strides
    // The decay in two parts: applied position after position, the rounding of
    // one part would add up.
    const double wd = exp(static_cast<double>(p.log_decay[h]));
    const float w = static_cast<float>(wd), w_lo = static_cast<float>(wd - w);

    float st[kRows][kVec];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int row = rg + kRG * r;
#pragma unroll
        for (int v = 0; v < kVec; ++v) st[r][v] = 0.f;
        if (p.state_in != nullptr && row < p.d_b && col < p.d_c) {
            const float* src = p.state_in + hs + row * rs + col * cs;
            if constexpr (kVec == 4) {
                const float4 x = *reinterpret_cast<const float4*>(src);
                st[r][0] = x.x; st[r][1] = x.y; st[r][2] = x.z; st[r][3] = x.w;
            } else {
                st[r][0] = *src;
            }
        }
    }

    const int64_t len = t1 - t0;
    const int64_t ha = h / (p.heads / p.heads_a), hb = h / (p.heads / p.heads_b),
                  hc = h / (p.heads / p.heads_c);
    float na = 0.f, nb = 0.f, nc[kVec];  // the next position's operands
    auto load = [&](int64_t i) {
        const int64_t t = p.reverse ? t1 - 1 - i : t0 + i;
        if (tid < p.d_b) {
            na = la_load<T>(p.a, (t * p.heads_a + ha) * p.d_b + tid);
            nb = la_load<T>(p.b, (t * p.heads_b + hb) * p.d_b + tid);
        }
#pragma unroll
        for (int v = 0; v < kVec; ++v)
            nc[v] = col + v < p.d_c ? la_load<T>(p.c, (t * p.heads_c + hc) * p.d_c + col + v) : 0.f;
    };
    if (len > 0) load(0);
    for (int64_t i = 0; i < len; ++i) {
        const int par = static_cast<int>(i & 1);
        if (tid < kRG * kRows) {  // rows past d_b hold zeros
            ab[par][0][tid] = na;
            ab[par][1][tid] = nb * p.sigma;
        }
        float c[kVec];
#pragma unroll
        for (int v = 0; v < kVec; ++v) c[v] = nc[v];
        if (i + 1 < len) load(i + 1);
        __syncthreads();
        float acc[kVec];
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = 0.f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float ar = ab[par][0][rg + kRG * r], br = ab[par][1][rg + kRG * r];
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                if (!p.reverse) st[r][v] = fmaf(st[r][v], w, st[r][v] * w_lo);
                st[r][v] = fmaf(br, c[v], st[r][v]);
                acc[v] = fmaf(ar, st[r][v], acc[v]);
                if (p.reverse) st[r][v] = fmaf(st[r][v], w, st[r][v] * w_lo);
            }
        }
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], o);
            if (lane < kLanes) red[par][warp][li * kVec + v] = acc[v];
        }
        __syncthreads();
        if (tid < kSlab && col0 + tid < p.d_c) {
            float o = 0.f;
#pragma unroll
            for (int x = 0; x < kWarps; ++x) o += red[par][x][tid];
            o *= p.tau;
            const int64_t t = p.reverse ? t1 - 1 - i : t0 + i;
            const int64_t at = (t * p.heads + h) * p.d_c + col0 + tid;
            if (p.out_f32)
                static_cast<float*>(p.out)[at] = o;
            else
                static_cast<T*>(p.out)[at] = from_f32<T>(o);
        }
    }

    if (p.state_out == nullptr) return;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int row = rg + kRG * r;
        if (row < p.d_b && col < p.d_c) {
            float* dst = p.state_out + hs + row * rs + col * cs;
            if constexpr (kVec == 4)
                *reinterpret_cast<float4*>(dst) = make_float4(st[r][0], st[r][1], st[r][2], st[r][3]);
            else
                *dst = st[r][0];
        }
    }
}

template <typename T, int kLanes, int kVec, int kRows>
cudaError_t start(const LaCore& p, cudaStream_t stream) {
    constexpr int kSlab = kLanes * kVec;
    const dim3 grid(p.heads, p.n_seqs, (p.d_c + kSlab - 1) / kSlab);
    la_recurrent<T, kLanes, kVec, kRows><<<grid, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t pick(const LaCore& p, cudaStream_t stream) {
    const uintptr_t align =
        reinterpret_cast<uintptr_t>(p.state_in) | reinterpret_cast<uintptr_t>(p.state_out);
    const bool vec = p.d_c % 4 == 0 && !p.state_t && (align & 15) == 0;
    if (!vec) return p.d_b <= 128 ? start<T, 32, 1, 16>(p, stream) : start<T, 32, 1, 32>(p, stream);
    if (p.d_b > 128) return start<T, 8, 4, 8>(p, stream);
    const bool many = static_cast<int64_t>(p.n_seqs) * p.heads >= 2 * 148;
    return many && p.d_c > 32 ? start<T, 32, 4, 16>(p, stream) : start<T, 8, 4, 4>(p, stream);
}

}  // namespace

cudaError_t launch_la_recurrent(const LaCore& p, cudaStream_t stream) {
    switch (p.dtype) {
        case GDR_DTYPE_BF16: return pick<__nv_bfloat16>(p, stream);
        case GDR_DTYPE_F16: return pick<__half>(p, stream);
        default: return pick<float>(p, stream);
    }
}

}  // namespace gdr
