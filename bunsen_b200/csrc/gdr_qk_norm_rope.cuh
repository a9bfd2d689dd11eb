// The head norms with rotation: what the entry points hand to the kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace gdr {

struct NormRope {
    int64_t tokens;
    int32_t heads_q, heads_k, d, rot, table_rows, interleaved, dtype;
    float eps;
    const void* q;  // [tokens, heads, d]: token and head strides in elements
    const void* k;
    int64_t q_token, q_head, k_token, k_head;
    const int32_t* positions;  // [tokens]
    const float* cos;          // [table_rows, rot / 2]
    const float* sin;
    const float* q_weight;  // [d], or null (ones)
    const float* k_weight;
    const void* dq_out = nullptr;  // gradient calls: of the outputs, contiguous
    const void* dk_out = nullptr;
    void* q_out;  // contiguous: the outputs, or the gradients of q and k
    void* k_out;
    float* dq_weight = nullptr;  // gradient calls: [d] or null (not wanted)
    float* dk_weight = nullptr;
};

// The vector kernels' units of a token: `per` heads of q or of k, the last of either with
// fewer.
inline int64_t norm_rope_units(int heads_q, int heads_k, int per) {
    return (heads_q + per - 1) / per + (heads_k + per - 1) / per;
}
// How many of `warps` (two at least) work on q: its share of the units. (By its share of the
// heads, 32 heads of q and one of k left k's warps with eight times q's work: the gradient
// of 32768 tokens took 1008 us, now 223.)
inline uint32_t norm_rope_q_warps(int64_t warps, int heads_q, int heads_k, int per) {
    const int64_t q = warps * ((heads_q + per - 1) / per) / norm_rope_units(heads_q, heads_k, per);
    return static_cast<uint32_t>(q < 1 ? 1 : q > warps - 1 ? warps - 1 : q);
}

int norm_rope_max_d();
int norm_rope_blocks(const NormRope& p);
// `part`: null, or (gradient calls) f32 [norm_rope_blocks][2][d].
cudaError_t launch_norm_rope(const NormRope& p, float* part, cudaStream_t s);
cudaError_t take_rope_error(int* flag);

}  // namespace gdr
