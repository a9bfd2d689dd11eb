// Linear attention with a decay for each head: what its kernels share.
//
// Per (sequence, value head), w = exp(log_decay[h]):
//   S_t = w S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t.
// Its gradients are the same recurrence with other operands. With
// D_t = dL/dS_t = scale q_t do_t^T + w D_{t+1}:
//   dq_t = scale S_t do_t,   dk_t = D_t v_t,   dv_t = D_t^T k_t,
// so every kernel here computes one core,
//   out_t = tau a_t . S_t,   S built from sigma b_t c_t^T and the decay,
// forward in time (o: a, b, c = q, k, v; dq: do, v, k with the state
// transposed) or backward (dv: k, q, do; dk: v, do, q transposed).
#pragma once

#include "gdr_common.cuh"

namespace gdr {

struct LaCore {
    int32_t n_seqs, seq_len;    // as Problem: dense T, or T_total of a pack
    const int32_t* cu_seqlens;  // nullptr: dense
    int32_t heads;              // value heads: one state each
    int32_t heads_a, heads_b, heads_c;  // heads of each operand's tensor; each
                                        // divides `heads`, consecutive value
                                        // heads share one
    const void* a;              // [T, heads_a, d_b]
    const void* b;              // [T, heads_b, d_b]
    const void* c;              // [T, heads_c, d_c]
    int32_t d_b, d_c;           // the state is [d_b, d_c]
    const float* log_decay;     // [heads]
    float sigma, tau;
    int32_t reverse;            // backward in time
    int32_t state_t;            // state_in / state_out hold [d_c, d_b]
    const float* state_in;      // may be null (zeros)
    float* state_out;           // may be null (not wanted), may be state_in
    void* out;                  // [T, heads, d_c] in the operands' type, or f32
    int32_t out_f32;
    int32_t dtype;              // of a, b, c
    int32_t scratch_t;          // states between segments are there as [d_c, d_b]
    int32_t steps_most;         // a pack in two launches: sequences of at most so many
                                // positions are the recurrent one's, longer ones the
                                // chunked one's; -1: one launch takes them all
};

inline int64_t la_tokens(const LaCore& p) {
    return p.cu_seqlens ? p.seq_len : static_cast<int64_t>(p.n_seqs) * p.seq_len;
}

// [start, end) of sequence s, clamped as seq_span clamps.
__device__ __forceinline__ void la_span(const LaCore& p, int s, int64_t& start, int64_t& end) {
    if (p.cu_seqlens == nullptr) {
        start = static_cast<int64_t>(s) * p.seq_len;
        end = start + p.seq_len;
        return;
    }
    int64_t x = p.cu_seqlens[s], y = p.cu_seqlens[s + 1];
    x = x < 0 ? 0 : (x > p.seq_len ? p.seq_len : x);
    y = y < x ? x : (y > p.seq_len ? p.seq_len : y);
    start = x;
    end = y;
}

// Work lists of a call (gdr_la_plan.cuh). Two cores over the same positions in the same
// direction, whose states are each other's transposes, may share them: given to
// both launches, made by the first, with the states between segments.
struct LaLists;

// Kernels of the core (each its own file) and what they take.
cudaError_t launch_la_recurrent(const LaCore& p, cudaStream_t stream);
bool la_parts_supports(const LaCore& p);
cudaError_t launch_la_parts(const LaCore& p, cudaStream_t stream, LaLists* shared, bool chained);
bool la_tc_supports(const LaCore& p);
// split: long sequences may go in segments (scratch from the library's pool);
// must: they do even where it looks slower; forced: segment length in chunks, or 0.
// chained: the stream's last kernel is one of this call's that lets the next one in.
cudaError_t launch_la_tc(const LaCore& p, bool split, bool must, int forced, cudaStream_t stream,
                         LaLists* shared, bool chained);
cudaError_t take_la_error(int* flag);
constexpr int kLaMaxD = 256;  // d_k, d_v of any kernel here

}  // namespace gdr
