// qk_norm.hpp -- host-side contract of the norm of queries and keys.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "block_ops.hpp"
#include "gated_delta.hpp"

namespace cubf {

constexpr int kQkNormMaxDim = 256;

// q and k are (batch, tokens, heads, dim) with any strides, outputs and
// gradients contiguous.  The position of token t of batch row b on an axis is
// positions[axis * positions_axis + (b * tokens + t) % positions_period].
struct QkNormArgs {
    HeadTensor q, k, d_q_out, d_k_out;      // the last two: gradients of the outputs, backward only
    const void* q_weight;                   // (dim), or null: one
    const void* k_weight;
    const void* positions;                  // or null: no rotation
    const float* frequencies;               // (rotary / 2)
    const int* axes;                        // (rotary / 2), or null: axis 0
    void* q_out;
    void* k_out;
    void* d_q;
    void* d_k;
    void* d_q_weight;                       // in the weight's type; backward, where the weight is
    void* d_k_weight;
    float* partials;                        // (parts, 2, dim): the parameter gradients' sums
    size_t batch, tokens;
    size_t positions_axis, positions_period;
    int q_heads, k_heads, dim, rotary, axis_count, parts;
    float eps;
    bool length, interleaved, positions64, q_weight32, k_weight32;
};

// CTAs of the backward, one part of the parameter gradients each.
int qk_norm_parts(const QkNormArgs& args);
cudaError_t launch_qk_norm(BlockType type, const QkNormArgs& args, bool backward, cudaStream_t stream);

}  // namespace cubf
