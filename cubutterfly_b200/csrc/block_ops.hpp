// block_ops.hpp -- host-side contract of the block operators of recurrent
// language models: the gated linear recurrence and the block norm.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace cubf {

enum class BlockType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };

// ---- gated linear recurrence (gated_scan.cuh) ----------------------------
constexpr int kGatedScanChunk = 16;       // tokens per saved chunk state
constexpr int kGatedScanMaxLength = 1 << 30;

// Strides in elements; the channel stride of every tensor is one.  Outputs
// and gradients are contiguous (batch, length, dim).
struct GatedScanArgs {
    const void* x;
    const void* r;
    const void* i;
    const void* d_h;
    size_t x_batch, r_batch, i_batch, dh_batch;
    size_t x_token, r_token, i_token, dh_token;
    const float* decay;
    const float* initial;       // (states, dim) or null: zero
    const int* offsets;         // (sequences + 1) of a packed batch, or null
    void* h;
    float* last;                // (states, dim)
    float* chunk_states;        // (batch, chunks, dim): h before every 16th token; null where no gradient follows
    const float* d_last;        // or null: zero
    void* d_x;
    void* d_r;
    void* d_i;
    float* d_initial;           // or null
    float* d_decay;
    float* partials;            // (batch, dim)
    int batch, length, dim, sequences;
    float exponent;
};

struct GatedStepArgs {
    const void* x;
    const void* r;
    const void* i;
    size_t x_row, r_row, i_row;
    const float* decay;
    const float* state;
    float* new_state;           // may be state
    const int* slots;           // or null: slot b of request b
    void* h;
    size_t batch, pool;
    int dim;
    float exponent;
};

cudaError_t launch_gated_scan(BlockType type, const GatedScanArgs& args, bool backward, cudaStream_t stream);
cudaError_t launch_gated_scan_step(BlockType type, const GatedStepArgs& args, cudaStream_t stream);

// ---- block norm (block_norm.cuh) ------------------------------------------
enum GateMode : int { kGateNone = 0, kGateChannel = 1, kGateGroups = 2, kGateFull = 3 };
constexpr int kBlockNormMaxDim = 16384;
constexpr int kBlockNormMinRotate = 64;   // rotated rows: powers of two from here

// Outputs and gradients are contiguous.  The
// per-channel vectors are in the block's type or, flagged, in fp32.
struct BlockNormArgs {
    const void* x;              // residual type
    const void* y;              // block type; null: no block output, s = x
    const void* gate;
    const void* pre;
    const void* post;
    const void* scales;         // residual scale per channel, or null: `scale`
    const void* d_residual;     // or null: zero
    const void* d_normed;       // or null: zero
    size_t gate_row;            // elements, of a gate per group
    // from a row to the next, in bytes
    uint32_t x_bytes, y_bytes, gate_bytes, d_residual_bytes, d_normed_bytes;
    void* residual;             // or null: not written
    void* normed;               // or null: no norm of the sum
    float* r_post;              // r(y) and r(s) of every row, kept for the backward; or null
    float* r_pre;
    void* d_x;
    void* d_y;
    void* d_gate;
    void* d_pre;
    void* d_post;
    void* d_scale;
    float* partials;            // (parts, 3, dim)
    size_t rows, rows_per_gate;
    float scale, eps, rotate_scale;
    int dim, gate_mode, act, parts_per_group;
    bool post_norm, rotate, pre32, post32, scales32, gate32;
    bool need_p, need_q, need_z;
};

// CTAs per gate group that sum the parameter gradients (one part each).
int block_norm_parts(size_t rows_per_gate, size_t groups, int dim);
cudaError_t launch_block_norm(BlockType type, bool residual32, const BlockNormArgs& args, cudaStream_t stream);
cudaError_t launch_block_norm_backward(BlockType type, bool residual32, const BlockNormArgs& args, size_t groups,
                                       cudaStream_t stream);

}  // namespace cubf
