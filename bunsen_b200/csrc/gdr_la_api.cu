// The entry points of include/gdr.h for the decayed linear attention and for
// the head norms with rotation: argument checks, then the kernels.
#include <cmath>
#include <type_traits>

#include "gdr_la.cuh"
#include "gdr_la_plan.cuh"
#include "gdr_qk_norm_rope.cuh"

namespace gdr {
cudaError_t library_pool(cudaMemPool_t* pool, bool create);

namespace {

gdr_status la_status(cudaError_t e) {
    if (e == cudaErrorNotSupported) return GDR_ERR_UNSUPPORTED;  // run_core's: no such kernel
    return e == cudaSuccess ? GDR_OK : GDR_ERR_CUDA;
}

// out[t, j, :] = the sum over a key head's `group` value heads of the f32
// partials [T, heads, d], in head order, for the packed positions that belong
// to a sequence (the others are left as they are).
template <typename T>
__global__ void __launch_bounds__(256)
sum_group(const float* __restrict__ part, T* __restrict__ out, int heads_qk, int group, int d,
          int64_t tokens, const int32_t* cu, int n_seqs) {
    after_last_kernel();
    int64_t first = 0, last = tokens;
    if (cu != nullptr) {
        first = cu[0] < 0 ? 0 : cu[0];
        last = cu[n_seqs] < tokens ? cu[n_seqs] : tokens;
    }
    const int64_t row = static_cast<int64_t>(heads_qk) * d, n = (last - first) * row;
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += step) {
        const int64_t at = first * row + i, th = at / d;  // (position, key head)
        const float* src = part + th * group * d + (at - th * d);
        float s = 0.f;
        for (int g = 0; g < group; ++g) s += src[static_cast<int64_t>(g) * d];
        out[at] = from_f32<T>(s);
    }
}

cudaError_t launch_sum_group(int dtype, const float* part, void* out, int heads_qk, int group,
                             int d, int64_t tokens, const int32_t* cu, int n_seqs,
                             cudaStream_t s) {
    const int64_t want = (tokens * heads_qk * d + 255) / 256;
    const int blocks = static_cast<int>(want < 148 * 16 ? want : 148 * 16);
    auto go = [&](auto* to) {
        using T = std::remove_pointer_t<decltype(to)>;
        return la_launch_next(sum_group<T>, blocks, 256, 0, s, part, to, heads_qk, group, d, tokens, cu,
                              n_seqs);
    };
    switch (dtype) {
        case GDR_DTYPE_BF16: return go(static_cast<__nv_bfloat16*>(out));
        case GDR_DTYPE_F16: return go(static_cast<__half*>(out));
        default: return go(static_cast<float*>(out));
    }
}

gdr_status check_la(const gdr_la_params* params, const int32_t* cu_seqlens) {
    if (params == nullptr) return GDR_ERR_INVALID;
    const gdr_la_params& a = *params;
    if (a.heads_qk <= 0 || a.heads_v <= 0 || a.heads_v % a.heads_qk != 0) return GDR_ERR_INVALID;
    if (a.d_k <= 0 || a.d_v <= 0 || a.seq_len < 0) return GDR_ERR_INVALID;
    if (a.dtype != GDR_DTYPE_F32 && a.dtype != GDR_DTYPE_BF16 && a.dtype != GDR_DTYPE_F16)
        return GDR_ERR_INVALID;
    if (!std::isfinite(static_cast<float>(a.scale))) return GDR_ERR_INVALID;  // as the kernels have it
    if ((cu_seqlens == nullptr ? a.batch : a.n_seqs) < 0) return GDR_ERR_INVALID;
    if (a.algo < GDR_ALGO_AUTO || a.algo > GDR_ALGO_TENSOR_SPLIT || a.split_chunks < 0)
        return GDR_ERR_INVALID;
    const int64_t n = cu_seqlens == nullptr ? a.batch : a.n_seqs;
    if (n > 65535 || a.heads_v > 65535) return GDR_ERR_UNSUPPORTED;  // grid limits
    if (cu_seqlens == nullptr && n * a.seq_len >= (int64_t{1} << 31)) return GDR_ERR_UNSUPPORTED;
    if (a.d_k > kLaMaxD || a.d_v > kLaMaxD) return GDR_ERR_UNSUPPORTED;
    return GDR_OK;
}

LaCore core_of(const gdr_la_params& a, const int32_t* cu_seqlens, const float* log_decay) {
    LaCore p{};
    p.n_seqs = cu_seqlens ? a.n_seqs : a.batch;
    p.seq_len = a.seq_len;
    p.cu_seqlens = cu_seqlens;
    p.heads = a.heads_v;
    p.log_decay = log_decay;
    p.dtype = a.dtype;
    p.steps_most = -1;
    return p;
}

void operands(LaCore& p, const void* x, int hx, const void* y, int hy, const void* z, int hz,
              int d_b, int d_c) {
    p.a = x;
    p.heads_a = hx;
    p.b = y;
    p.heads_b = hy;
    p.c = z;
    p.heads_c = hz;
    p.d_b = d_b;
    p.d_c = d_c;
}

enum class Kernel { none, recurrent, tensor, parts, both };
constexpr int kFewEach = 4;  // positions of a sequence that step as fast as their chunk runs

Kernel kernel_of(const gdr_la_params& a, const LaCore& p, bool chunked) {
    const int64_t tokens = la_tokens(p);
    if (!chunked || tokens == 0) return Kernel::recurrent;
    const bool tc = la_tc_supports(p);
    if (!tc && a.algo >= GDR_ALGO_TENSOR) return Kernel::none;
    // A few positions step as fast as a chunk does, and in f32 (rounded to bf16, a chunk's few
    // scores would be most of some outputs); the others go in chunks. The lengths of a pack
    // are on the device: one with few positions a sequence on average may still hold a long
    // one, whose steps, 0.7 to 1.3 us each, would bound the call. So such a pack goes to both
    // kernels, each with the sequences that are its own, both at f32 accuracy: a prompt of
    // 3000 between 1000 single positions, 32 heads of 128, 4420 us in steps, 887 so. The second
    // kernel and its plan are 12 to 20 us where no sequence is theirs (256 single positions 181 and
    // 194 us): up to 64 positions, where no walk takes 80 us, steps alone.
    const bool few =
        tokens <= 16 || tokens <= kFewEach * static_cast<int64_t>(p.n_seqs);  // on average
    if (few && a.algo < GDR_ALGO_TENSOR) {
        const bool mixed = p.cu_seqlens != nullptr && tokens > 64 && la_parts_supports(p);
        return mixed ? Kernel::both : Kernel::recurrent;
    }
    // Nor do prompts of a chunk or less, where every sequence and head has an SM, gain from
    // bf16 scores and states: 12 us in parts, 10 us with them, and half their error in the
    // sums. (Several an SM do: 12 sequences of 64 heads 61 us against 40.)
    const bool exact = tokens <= 64 && a.algo == GDR_ALGO_AUTO && la_parts_supports(p) &&
                       static_cast<int64_t>(p.n_seqs) * p.heads <= la_sm_count();
    if (tc && a.algo != GDR_ALGO_CUDA_CORE && !exact) return Kernel::tensor;
    return la_parts_supports(p) ? Kernel::parts : Kernel::recurrent;
}

cudaError_t run_core(const gdr_la_params& a, const LaCore& p, bool chunked, cudaStream_t s,
                     LaLists* shared = nullptr, bool chained = false) {
    switch (kernel_of(a, p, chunked)) {
        case Kernel::none: return cudaErrorNotSupported;
        case Kernel::tensor:
            return launch_la_tc(p, a.algo != GDR_ALGO_TENSOR, a.algo == GDR_ALGO_TENSOR_SPLIT,
                                a.split_chunks, s, shared, chained);
        case Kernel::parts: return launch_la_parts(p, s, shared, chained);
        case Kernel::both: {
            LaCore two = p;
            two.steps_most = kFewEach;
            const cudaError_t e = launch_la_recurrent(two, s);
            return e != cudaSuccess ? e : launch_la_parts(two, s, shared, false);
        }
        default: return launch_la_recurrent(p, s);
    }
}

gdr_status forward(bool chunked, const gdr_la_params* params, const void* q, const void* k,
                   const void* v, const float* log_decay, const float* state_in, void* out,
                   float* state_out, const int32_t* cu_seqlens, void* stream) {
    const gdr_status st = check_la(params, cu_seqlens);
    if (st != GDR_OK) return st;
    LaCore p = core_of(*params, cu_seqlens, log_decay);
    const bool some = la_tokens(p) > 0;
    if (some && !(q && k && v && out)) return GDR_ERR_INVALID;
    if (p.n_seqs > 0 && !(state_out && log_decay)) return GDR_ERR_INVALID;
    if (p.n_seqs == 0) return GDR_OK;
    operands(p, q, params->heads_qk, k, params->heads_qk, v, params->heads_v, params->d_k,
             params->d_v);
    p.sigma = 1.f;
    p.tau = static_cast<float>(params->scale);
    p.state_in = state_in;
    p.state_out = state_out;
    p.out = out;
    return la_status(run_core(*params, p, chunked, static_cast<cudaStream_t>(stream)));
}

}  // namespace
}  // namespace gdr

extern "C" {

gdr_status gdr_la_recurrent(const gdr_la_params* params, const void* q, const void* k,
                            const void* v, const float* log_decay, const float* state_in,
                            void* out, float* state_out, const int32_t* cu_seqlens,
                            void* stream) {
    return gdr::forward(false, params, q, k, v, log_decay, state_in, out, state_out, cu_seqlens,
                        stream);
}

gdr_status gdr_la_chunked(const gdr_la_params* params, const void* q, const void* k, const void* v,
                          const float* log_decay, const float* state_in, void* out,
                          float* state_out, const int32_t* cu_seqlens, void* stream) {
    return gdr::forward(true, params, q, k, v, log_decay, state_in, out, state_out, cu_seqlens,
                        stream);
}

gdr_status gdr_la_backward(const gdr_la_params* params, const void* q, const void* k,
                           const void* v, const float* log_decay, const void* d_out,
                           const float* state_in, const float* d_state_out, void* dq, void* dk,
                           void* dv, float* d_state_in, const int32_t* cu_seqlens, void* stream) {
    using namespace gdr;
    const gdr_status st = check_la(params, cu_seqlens);
    if (st != GDR_OK) return st;
    const gdr_la_params& a = *params;
    const LaCore base = core_of(a, cu_seqlens, log_decay);
    const int64_t tokens = la_tokens(base);
    if (tokens > 0 && !(q && k && v && d_out && dq && dk && dv)) return GDR_ERR_INVALID;
    if (base.n_seqs > 0 && log_decay == nullptr) return GDR_ERR_INVALID;
    if (base.n_seqs == 0) return GDR_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const float scale = static_cast<float>(a.scale);
    const int group = a.heads_v / a.heads_qk;
    // Gradients of shared key heads: each value head's share in f32, then
    // their sum in head order.
    float* part = nullptr;
    cudaError_t e = cudaSuccess;
    if (group > 1 && tokens > 0) {
        cudaMemPool_t pool;
        if (library_pool(&pool, true) != cudaSuccess ||
            cudaMallocFromPoolAsync(reinterpret_cast<void**>(&part),
                                    sizeof(float) * tokens * a.heads_v * a.d_k, pool,
                                    s) != cudaSuccess)
            return GDR_ERR_CUDA;
    }
    // dv_t = D_t^T k_t, and the gradient of the initial state.
    LaCore v_core = base;
    operands(v_core, k, a.heads_qk, q, a.heads_qk, d_out, a.heads_v, a.d_k, a.d_v);
    v_core.sigma = scale;
    v_core.tau = 1.f;
    v_core.reverse = 1;
    v_core.state_in = d_state_out;
    v_core.state_out = d_state_in;
    v_core.out = dv;
    // dk_t = D_t v_t, D transposed.
    LaCore k_core = base;
    operands(k_core, v, a.heads_v, d_out, a.heads_v, q, a.heads_qk, a.d_v, a.d_k);
    k_core.sigma = scale;
    k_core.tau = 1.f;
    k_core.reverse = 1;
    k_core.state_t = 1;
    k_core.state_in = d_state_out;
    // dq_t = scale S_t do_t.
    LaCore q_core = base;
    operands(q_core, d_out, a.heads_v, v, a.heads_v, k, a.heads_qk, a.d_v, a.d_k);
    q_core.sigma = 1.f;
    q_core.tau = scale;
    q_core.state_t = 1;
    q_core.state_in = state_in;
    for (LaCore* c : {&k_core, &q_core}) {
        c->out = part != nullptr ? part : c == &k_core ? dk : dq;
        c->out_f32 = part != nullptr;
    }
    auto sum = [&](void* grad) {
        return part == nullptr ? cudaSuccess
                               : launch_sum_group(a.dtype, part, grad, a.heads_qk, group, a.d_k,
                                                  tokens, cu_seqlens, base.n_seqs, s);
    };
    // dv and dk run over the same D: one of them finds its states between segments.
    const Kernel kernel = kernel_of(a, v_core, true);
    const bool same = kernel != Kernel::none && kernel != Kernel::recurrent &&
                      kernel_of(a, k_core, true) == kernel && la_same_lists(v_core, k_core);
    LaLists lists;
    k_core.scratch_t = same;
    e = run_core(a, v_core, true, s, same ? &lists : nullptr);
    if (e == cudaSuccess && tokens > 0) {
        e = run_core(a, k_core, true, s, same ? &lists : nullptr);
        if (e == cudaSuccess) e = sum(dk);
    }
    const cudaError_t r = la_release(lists, s);
    if (e == cudaSuccess) e = r;
    if (e == cudaSuccess && tokens > 0) {
        e = run_core(a, q_core, true, s, nullptr, true);
        if (e == cudaSuccess) e = sum(dq);
    }
    if (part != nullptr) {
        const cudaError_t f = cudaFreeAsync(part, s);
        if (e == cudaSuccess) e = f;
    }
    return la_status(e);
}

}  // extern "C"

namespace {

gdr_status make_rope(const gdr_qk_norm_rope_params* params, const void* q, const void* k,
                     const int32_t* positions, const float* cos, const float* sin,
                     const float* q_weight, const float* k_weight, void* q_out, void* k_out,
                     gdr::NormRope& p) {
    if (params == nullptr) return GDR_ERR_INVALID;
    const gdr_qk_norm_rope_params& a = *params;
    if (a.tokens < 0 || a.heads_q <= 0 || a.heads_k <= 0 || a.head_dim <= 0) return GDR_ERR_INVALID;
    if (a.rotary_dim <= 0 || a.rotary_dim % 2 != 0 || a.rotary_dim > a.head_dim || a.table_rows <= 0)
        return GDR_ERR_INVALID;
    if (a.dtype != GDR_DTYPE_F32 && a.dtype != GDR_DTYPE_BF16 && a.dtype != GDR_DTYPE_F16)
        return GDR_ERR_INVALID;
    if (!(a.eps >= 0.0) || !std::isfinite(static_cast<float>(a.eps))) return GDR_ERR_INVALID;
    if (a.head_dim > gdr::norm_rope_max_d()) return GDR_ERR_UNSUPPORTED;
    if (a.tokens >= (int64_t{1} << 31) ||
        a.tokens * (static_cast<int64_t>(a.heads_q) + a.heads_k) >= (int64_t{1} << 31))
        return GDR_ERR_UNSUPPORTED;  // rows are counted in 32 bits
    if (a.tokens > 0 && !(q && k && positions && cos && sin && q_out && k_out))
        return GDR_ERR_INVALID;
    p.tokens = a.tokens;
    p.heads_q = a.heads_q;
    p.heads_k = a.heads_k;
    p.d = a.head_dim;
    p.rot = a.rotary_dim;
    p.table_rows = a.table_rows;
    p.interleaved = a.interleaved != 0;
    p.dtype = a.dtype;
    p.eps = static_cast<float>(a.eps);
    p.q = q;
    p.k = k;
    p.q_token = a.q_token_stride;
    p.q_head = a.q_head_stride;
    p.k_token = a.k_token_stride;
    p.k_head = a.k_head_stride;
    p.positions = positions;
    p.cos = cos;
    p.sin = sin;
    p.q_weight = q_weight;
    p.k_weight = k_weight;
    p.q_out = q_out;
    p.k_out = k_out;
    return GDR_OK;
}

}  // namespace

extern "C" {

gdr_status gdr_qk_norm_rope(const gdr_qk_norm_rope_params* params, const void* q, const void* k,
                            const int32_t* positions, const float* cos, const float* sin,
                            const float* q_weight, const float* k_weight, void* q_out,
                            void* k_out, void* stream) {
    gdr::NormRope p;
    const gdr_status st =
        make_rope(params, q, k, positions, cos, sin, q_weight, k_weight, q_out, k_out, p);
    if (st != GDR_OK || p.tokens == 0) return st;
    return gdr::la_status(gdr::launch_norm_rope(p, nullptr, static_cast<cudaStream_t>(stream)));
}

gdr_status gdr_qk_norm_rope_backward(const gdr_qk_norm_rope_params* params, const void* dq_out,
                                     const void* dk_out, const void* q, const void* k,
                                     const int32_t* positions, const float* cos, const float* sin,
                                     const float* q_weight, const float* k_weight, void* dq,
                                     void* dk, float* dq_weight, float* dk_weight, void* stream) {
    gdr::NormRope p;
    const gdr_status st =
        make_rope(params, q, k, positions, cos, sin, q_weight, k_weight, dq, dk, p);
    if (st != GDR_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p.tokens == 0) {  // no rows: the weights' gradients are zero
        cudaError_t e = cudaSuccess;
        for (float* w : {dq_weight, dk_weight})
            if (w != nullptr && e == cudaSuccess) e = cudaMemsetAsync(w, 0, sizeof(float) * p.d, s);
        return gdr::la_status(e);
    }
    if (dq_out == nullptr || dk_out == nullptr) return GDR_ERR_INVALID;
    p.dq_out = dq_out;
    p.dk_out = dk_out;
    p.dq_weight = dq_weight;
    p.dk_weight = dk_weight;
    void* part = nullptr;
    if (dq_weight != nullptr || dk_weight != nullptr) {
        cudaMemPool_t pool;
        const size_t bytes = sizeof(float) * 2 * p.d * gdr::norm_rope_blocks(p);
        if (gdr::library_pool(&pool, true) != cudaSuccess ||
            cudaMallocFromPoolAsync(&part, bytes, pool, s) != cudaSuccess)
            return GDR_ERR_CUDA;
    }
    cudaError_t e = gdr::launch_norm_rope(p, static_cast<float*>(part), s);
    if (part != nullptr) {
        const cudaError_t f = cudaFreeAsync(part, s);
        if (e == cudaSuccess) e = f;
    }
    return gdr::la_status(e);
}

}  // extern "C"
