// gated_delta.hpp -- host-side contract of the gated delta rule.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "block_ops.hpp"

namespace cubf {

constexpr int kDeltaChunk = 64;          // tokens a chunk
constexpr int kDeltaMaxDim = 128;        // of keys and of values
constexpr int kDeltaMaxLength = 1 << 30;
constexpr int kDeltaWaitLimit = 1 << 17;  // tries, of 8 us each where nothing comes: a second

// A (batch, token, head, channel) tensor: strides in elements, the channels adjacent.
struct HeadTensor {
    const void* p;
    size_t batch, token, head;
};

// Outputs and gradients are contiguous.  A chunk's place ("slot") among those
// of all sequences is base(j) + c for chunk c of sequence j: j ceil(length /
// 64) in a dense batch, floor(offsets[j] / 64) + j in a packed one, which
// leaves each sequence at least the places that it needs without a pass over
// the offsets.
struct GatedDeltaArgs {
    HeadTensor q, k, v, log_decay, beta, d_o;
    const float* initial;        // (states, heads, k_dim, v_dim) or null: zero
    const int* offsets;          // (sequences + 1) of a packed batch, or null
    void* o;                     // (batch, length, heads, v_dim)
    float* last;                 // (states, heads, k_dim, v_dim)
    const float* d_last;         // or null: zero
    void *d_q, *d_k, *d_v, *d_log_decay, *d_beta;
    float* d_initial;            // or null
    int batch, length, k_heads, heads, k_dim, v_dim, sequences;
    float scale;
    bool log_decay32, beta32;    // fp32 gates beside 16-bit tensors
    uint32_t wait_limit;         // tries of a wait on a barrier
    void* workspace;
};

struct GatedDeltaStepArgs {
    HeadTensor q, k, v, log_decay, beta;   // batch strides; token unused
    const float* state;          // (pool, heads, k_dim, v_dim)
    float* new_state;            // may be state
    const int* slots;            // or null: slot b of request b
    void* o;                     // (batch, heads, v_dim)
    size_t batch, pool;
    int k_heads, heads, k_dim, v_dim;
    float scale;
    bool log_decay32, beta32;
};

size_t gated_delta_workspace(BlockType type, const GatedDeltaArgs& args, bool backward);
cudaError_t launch_gated_delta(BlockType type, const GatedDeltaArgs& args, bool backward, cudaStream_t stream);
cudaError_t launch_gated_delta_step(BlockType type, const GatedDeltaStepArgs& args, cudaStream_t stream);

}  // namespace cubf
