// launch_block_dispatch.cpp -- picks the unit of a type for the block norm, the
// gated linear recurrence and the gated delta rule.
#include <algorithm>

#include "block_ops.hpp"
#include "gated_delta.hpp"

namespace cubf {

template <int TYPE>
cudaError_t launch_block_norm_unit(const BlockNormArgs& a, cudaStream_t stream);
template <int TYPE>
cudaError_t launch_block_norm_backward_unit(const BlockNormArgs& a, size_t groups, cudaStream_t stream);

#define CUBF_BN_UNIT(TYPE)                                                                  \
    template <>                                                                             \
    cudaError_t launch_block_norm_unit<TYPE>(const BlockNormArgs&, cudaStream_t);           \
    template <>                                                                             \
    cudaError_t launch_block_norm_backward_unit<TYPE>(const BlockNormArgs&, size_t, cudaStream_t);
CUBF_BN_UNIT(0)
CUBF_BN_UNIT(1)
CUBF_BN_UNIT(2)
CUBF_BN_UNIT(3)
CUBF_BN_UNIT(4)
#undef CUBF_BN_UNIT

namespace {
int unit_of(BlockType type, bool residual32) {
    if (type == BlockType::kF32) return 4;
    return (type == BlockType::kBF16 ? 2 : 0) + (residual32 ? 1 : 0);
}
}  // namespace

int block_norm_parts(size_t rows_per_gate, size_t groups, int dim) {
    // A CTA of 512 threads takes 512 x 8 values of rows side by side; at least
    // two turns of it, and no more CTAs than SMs.
    const size_t side = std::max<size_t>(1, 4096 / static_cast<size_t>(dim));
    const size_t most = std::max<size_t>(1, (rows_per_gate + 2 * side - 1) / (2 * side));
    const size_t share = std::max<size_t>(1, (148 + groups - 1) / std::max<size_t>(1, groups));
    return static_cast<int>(std::min(most, share));
}

cudaError_t launch_block_norm(BlockType type, bool residual32, const BlockNormArgs& a, cudaStream_t stream) {
    switch (unit_of(type, residual32)) {
        case 0: return launch_block_norm_unit<0>(a, stream);
        case 1: return launch_block_norm_unit<1>(a, stream);
        case 2: return launch_block_norm_unit<2>(a, stream);
        case 3: return launch_block_norm_unit<3>(a, stream);
        default: return launch_block_norm_unit<4>(a, stream);
    }
}

cudaError_t launch_block_norm_backward(BlockType type, bool residual32, const BlockNormArgs& a, size_t groups,
                                       cudaStream_t stream) {
    switch (unit_of(type, residual32)) {
        case 0: return launch_block_norm_backward_unit<0>(a, groups, stream);
        case 1: return launch_block_norm_backward_unit<1>(a, groups, stream);
        case 2: return launch_block_norm_backward_unit<2>(a, groups, stream);
        case 3: return launch_block_norm_backward_unit<3>(a, groups, stream);
        default: return launch_block_norm_backward_unit<4>(a, groups, stream);
    }
}

template <int TYPE>
cudaError_t launch_gated_scan_unit(const GatedScanArgs& a, bool backward, cudaStream_t stream);
template <int TYPE>
cudaError_t launch_gated_scan_step_unit(const GatedStepArgs& a, cudaStream_t stream);

#define CUBF_GS_UNIT(TYPE)                                                                  \
    template <>                                                                             \
    cudaError_t launch_gated_scan_unit<TYPE>(const GatedScanArgs&, bool, cudaStream_t);     \
    template <>                                                                             \
    cudaError_t launch_gated_scan_step_unit<TYPE>(const GatedStepArgs&, cudaStream_t);
CUBF_GS_UNIT(0)
CUBF_GS_UNIT(1)
CUBF_GS_UNIT(2)
#undef CUBF_GS_UNIT

cudaError_t launch_gated_scan(BlockType type, const GatedScanArgs& a, bool backward, cudaStream_t stream) {
    switch (type) {
        case BlockType::kF16: return launch_gated_scan_unit<0>(a, backward, stream);
        case BlockType::kBF16: return launch_gated_scan_unit<1>(a, backward, stream);
        default: return launch_gated_scan_unit<2>(a, backward, stream);
    }
}

cudaError_t launch_gated_scan_step(BlockType type, const GatedStepArgs& a, cudaStream_t stream) {
    switch (type) {
        case BlockType::kF16: return launch_gated_scan_step_unit<0>(a, stream);
        case BlockType::kBF16: return launch_gated_scan_step_unit<1>(a, stream);
        default: return launch_gated_scan_step_unit<2>(a, stream);
    }
}

template <int TYPE, int KP>
cudaError_t launch_gated_delta_unit(const GatedDeltaArgs& a, bool backward, cudaStream_t stream);
template <int TYPE, int KP>
size_t gated_delta_workspace_unit(const GatedDeltaArgs& a, bool backward);
template <int TYPE>
cudaError_t launch_gated_delta_step_unit(const GatedDeltaStepArgs& a, cudaStream_t stream);

#define CUBF_GD_UNIT(TYPE, KP)                                                               \
    template <>                                                                              \
    cudaError_t launch_gated_delta_unit<TYPE, KP>(const GatedDeltaArgs&, bool, cudaStream_t); \
    template <>                                                                              \
    size_t gated_delta_workspace_unit<TYPE, KP>(const GatedDeltaArgs&, bool);
#define CUBF_GD_TYPE_UNITS(TYPE) \
    CUBF_GD_UNIT(TYPE, 64)       \
    CUBF_GD_UNIT(TYPE, 128)      \
    template <>                  \
    cudaError_t launch_gated_delta_step_unit<TYPE>(const GatedDeltaStepArgs&, cudaStream_t);
CUBF_GD_TYPE_UNITS(0)
CUBF_GD_TYPE_UNITS(1)
CUBF_GD_TYPE_UNITS(2)
#undef CUBF_GD_TYPE_UNITS
#undef CUBF_GD_UNIT

size_t gated_delta_workspace(BlockType type, const GatedDeltaArgs& a, bool backward) {
    const bool small = a.k_dim <= 64;
    switch (type) {
        case BlockType::kF16:
            return small ? gated_delta_workspace_unit<0, 64>(a, backward) : gated_delta_workspace_unit<0, 128>(a, backward);
        case BlockType::kBF16:
            return small ? gated_delta_workspace_unit<1, 64>(a, backward) : gated_delta_workspace_unit<1, 128>(a, backward);
        default:
            return small ? gated_delta_workspace_unit<2, 64>(a, backward) : gated_delta_workspace_unit<2, 128>(a, backward);
    }
}

cudaError_t launch_gated_delta(BlockType type, const GatedDeltaArgs& a, bool backward, cudaStream_t stream) {
    const bool small = a.k_dim <= 64;
    switch (type) {
        case BlockType::kF16:
            return small ? launch_gated_delta_unit<0, 64>(a, backward, stream)
                         : launch_gated_delta_unit<0, 128>(a, backward, stream);
        case BlockType::kBF16:
            return small ? launch_gated_delta_unit<1, 64>(a, backward, stream)
                         : launch_gated_delta_unit<1, 128>(a, backward, stream);
        default:
            return small ? launch_gated_delta_unit<2, 64>(a, backward, stream)
                         : launch_gated_delta_unit<2, 128>(a, backward, stream);
    }
}

cudaError_t launch_gated_delta_step(BlockType type, const GatedDeltaStepArgs& a, cudaStream_t stream) {
    switch (type) {
        case BlockType::kF16: return launch_gated_delta_step_unit<0>(a, stream);
        case BlockType::kBF16: return launch_gated_delta_step_unit<1>(a, stream);
        default: return launch_gated_delta_step_unit<2>(a, stream);
    }
}

}  // namespace cubf
