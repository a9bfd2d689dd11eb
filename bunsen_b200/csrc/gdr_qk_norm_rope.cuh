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

int norm_rope_max_d();
int norm_rope_blocks(const NormRope& p);
// `part`: null, or (gradient calls) f32 [norm_rope_blocks][2][d].
cudaError_t launch_norm_rope(const NormRope& p, float* part, cudaStream_t s);
cudaError_t take_rope_error(int* flag);

}  // namespace gdr
