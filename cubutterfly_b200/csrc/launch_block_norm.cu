// launch_block_norm.cu -- launches of the block norm; compiled once per
// CUBF_BN_TYPE (0 fp16, 1 fp16 with an fp32 residual, 2 bf16, 3 bf16 with an
// fp32 residual, 4 fp32) and CUBF_BN_BACKWARD.
#include <algorithm>

#include "block_norm.cuh"
#include "launch_util.cuh"

#ifndef CUBF_BN_TYPE
#define CUBF_BN_TYPE 2
#endif
#ifndef CUBF_BN_BACKWARD
#define CUBF_BN_BACKWARD 0
#endif

namespace cubf {

template <int TYPE>
cudaError_t launch_block_norm_unit(const BlockNormArgs& a, cudaStream_t stream);
template <int TYPE>
cudaError_t launch_block_norm_backward_unit(const BlockNormArgs& a, size_t groups, cudaStream_t stream);

namespace {

using namespace norm;

constexpr int kType = CUBF_BN_TYPE;
using T = std::conditional_t<kType <= 1, __half, std::conditional_t<kType <= 3, __nv_bfloat16, float>>;
using R = std::conditional_t<kType == 1 || kType == 3 || kType == 4, float, T>;
constexpr int kVec = 16 / static_cast<int>(sizeof(T));
// values a thread of the backward: 16 fit the registers where every tensor is 16-bit
constexpr int kWide = sizeof(R) == 2 ? 16 : 8;

// Consecutive values that every row of every tensor is aligned for: whole
// 16-byte vectors (kVec), pairs, or one.
int alignment(const BlockNormArgs& a) {
    uintptr_t block = static_cast<uintptr_t>(a.dim) * sizeof(T);  // of 16-byte vectors of the block's type
    uintptr_t wide = static_cast<uintptr_t>(a.dim) * 4;           // of fp32 tensors beside 16-bit ones
    auto add = [](uintptr_t& bits, const void* p) { bits |= reinterpret_cast<uintptr_t>(p); };
    for (const void* p : {a.y, a.d_normed, static_cast<const void*>(a.normed), static_cast<const void*>(a.d_y)})
        add(block, p);
    block |= a.y_bytes | a.d_normed_bytes;
    uintptr_t& stream = sizeof(R) == 4 ? wide : block;
    for (const void* p : {a.x, a.d_residual, static_cast<const void*>(a.residual), static_cast<const void*>(a.d_x)})
        add(stream, p);
    stream |= a.x_bytes | a.d_residual_bytes;
    uintptr_t& gate = a.gate32 ? wide : block;
    add(gate, a.gate);
    add(gate, a.gate_mode == kGateFull ? a.d_gate : nullptr);
    gate |= a.gate_mode == kGateFull ? a.gate_bytes : a.gate_row * (a.gate32 ? 4 : sizeof(T));
    add(a.pre32 ? wide : block, a.pre);
    add(a.post32 ? wide : block, a.post);
    add(a.scales32 ? wide : block, a.scales);
    add(wide, a.partials);
    if (sizeof(T) == 4) block |= wide;
    if (((block | wide) & 15) == 0 && a.dim % kVec == 0) return kVec;
    // pairs: 2 values of the block's type, 8 bytes of fp32
    return (block & (2 * sizeof(T) - 1)) == 0 && (wide & 7) == 0 ? 2 : 1;
}

template <typename S, bool ROTATE>
cudaError_t run(const BlockNormArgs& a, size_t groups, cudaStream_t stream) {
    static KernelSetup setup;
#if CUBF_BN_BACKWARD
    auto kernel = &block_norm_backward_kernel<T, R, S, ROTATE>;
#else
    auto kernel = &block_norm_kernel<T, R, S, ROTATE>;
#endif
#if CUBF_BN_BACKWARD
    using Plan = BackwardPlan<S, ROTATE>;
    const int smem = 4 * Plan::floats_needed(a.need_z);
    constexpr int most = 4 * Plan::floats_needed(true);
#else
    constexpr int smem = 4 * ForwardPlan<S, ROTATE>::kFloats, most = smem;
#endif
    int cap = 0;
    cudaError_t e = setup_kernel(setup, kernel, S::kThreads, most, &cap, CUBF_BN_BACKWARD);
    if (e != cudaSuccess) return e;
#if CUBF_BN_BACKWARD
    (void)cap;
    const size_t grid = groups * a.parts_per_group;
#else
    (void)groups;
    const size_t grid = std::min<size_t>((a.rows + S::kRows - 1) / S::kRows, static_cast<size_t>(cap));
#endif
    if (grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    return launch_dependent(kernel, static_cast<unsigned>(grid), static_cast<unsigned>(S::kThreads), smem, stream, a);
}

template <int TPR, int EPT, int VW, bool ROTATE, int THREADS = 0>
cudaError_t shape(const BlockNormArgs& a, size_t groups, cudaStream_t stream) {
    return run<Shape<TPR, EPT, VW, THREADS>, ROTATE>(a, groups, stream);
}

cudaError_t dispatch(const BlockNormArgs& a, size_t groups, cudaStream_t s) {
    constexpr int V = kVec;
    const int width = alignment(a);
    const bool vec = width == V;
    const int d = a.dim;
    if (a.rotate) {
        if (vec && d >= 256) {
#if CUBF_BN_BACKWARD
            switch (d) {
                case 256: return shape<32, 8, V, true, 512>(a, groups, s);
                case 512: return shape<512 / kWide, kWide, V, true, 512>(a, groups, s);
                case 1024: return shape<1024 / kWide, kWide, V, true, 512>(a, groups, s);
                case 2048: return shape<2048 / kWide, kWide, V, true, 512>(a, groups, s);
                case 4096: return shape<4096 / kWide, kWide, V, true, 512>(a, groups, s);
                case 8192: return shape<512, 16, V, true>(a, groups, s);
                case 16384: return shape<1024, 16, V, true>(a, groups, s);
            }
#else
            if (a.rows > 296 || d < 2048) {
                switch (d) {
                    case 256: return shape<32, 8, V, true>(a, groups, s);
                    case 512: return shape<32, 16, V, true>(a, groups, s);
                    case 1024: return shape<32, 32, V, true, 256>(a, groups, s);
                    case 2048: return shape<64, 32, V, true, 512>(a, groups, s);
                    case 4096: return shape<128, 32, V, true, 512>(a, groups, s);
                    case 8192: return shape<256, 32, V, true, 512>(a, groups, s);
                    case 16384: return shape<512, 32, V, true>(a, groups, s);
                }
            }
            // few rows: more threads a row
            switch (d) {
                case 2048: return shape<256, 8, V, true>(a, groups, s);
                case 4096: return shape<512, 8, V, true>(a, groups, s);
                case 8192: return shape<1024, 8, V, true>(a, groups, s);
                case 16384: return shape<1024, 16, V, true>(a, groups, s);
            }
#endif
        }
        switch (d) {
            case 64: return shape<32, 2, 1, true>(a, groups, s);
            case 128: return shape<32, 4, 1, true>(a, groups, s);
            case 256: return shape<32, 8, 1, true>(a, groups, s);
            case 512: return shape<32, 16, 1, true>(a, groups, s);
            case 1024: return shape<64, 16, 1, true>(a, groups, s);
            case 2048: return shape<128, 16, 1, true>(a, groups, s);
            case 4096: return shape<256, 16, 1, true>(a, groups, s);
            case 8192: return shape<512, 16, 1, true>(a, groups, s);
            case 16384: return shape<1024, 16, 1, true>(a, groups, s);
        }
        return cudaErrorInvalidValue;
    }
#if CUBF_BN_BACKWARD
    constexpr int kThreads = 512;  // rows side by side, so that there is one part of the sums per SM
    if (vec) {
        if (d <= 256) return shape<32, 8, V, false, 512>(a, groups, s);
        if (d <= 512) return shape<512 / kWide, kWide, V, false, 512>(a, groups, s);
        if (d <= 1024) return shape<1024 / kWide, kWide, V, false, 512>(a, groups, s);
        if (d <= 2048) return shape<2048 / kWide, kWide, V, false, 512>(a, groups, s);
        if (d <= 4096) return shape<4096 / kWide, kWide, V, false, 512>(a, groups, s);
        if (d <= 8192) return shape<8192 / kWide, kWide, V, false>(a, groups, s);
#else
    constexpr int kThreads = 0;
    if (vec) {
        if (d <= 256) return shape<32, 8, V, false>(a, groups, s);
        if (d <= 512) return shape<64, 8, V, false>(a, groups, s);
        if (d <= 1024) return shape<128, 8, V, false>(a, groups, s);
        if (d <= 2048) return shape<256, 8, V, false>(a, groups, s);
        if (d <= 4096) return shape<512, 8, V, false>(a, groups, s);
        if (d <= 8192) return shape<1024, 8, V, false>(a, groups, s);
#endif
        if (d <= kBlockNormMaxDim) return shape<1024, 16, V, false>(a, groups, s);
    } else if (width == 2) {
        if (d <= 256) return shape<32, 8, 2, false, kThreads>(a, groups, s);
        if (d <= 1024) return shape<128, 8, 2, false, kThreads>(a, groups, s);
        if (d <= 2048) return shape<256, 8, 2, false, kThreads>(a, groups, s);
        if (d <= 4096) return shape<512, 8, 2, false>(a, groups, s);
        if (d <= 8192) return shape<1024, 8, 2, false>(a, groups, s);
        if (d <= kBlockNormMaxDim) return shape<1024, 16, 2, false>(a, groups, s);
    } else {
        if (d <= 256) return shape<32, 8, 1, false, kThreads>(a, groups, s);
        if (d <= 1024) return shape<128, 8, 1, false, kThreads>(a, groups, s);
        if (d <= 2048) return shape<256, 8, 1, false, kThreads>(a, groups, s);
        if (d <= 4096) return shape<512, 8, 1, false>(a, groups, s);
        if (d <= 8192) return shape<1024, 8, 1, false>(a, groups, s);
        if (d <= kBlockNormMaxDim) return shape<1024, 16, 1, false>(a, groups, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

#if CUBF_BN_BACKWARD
template <>
cudaError_t launch_block_norm_backward_unit<CUBF_BN_TYPE>(const BlockNormArgs& a, size_t groups, cudaStream_t stream) {
    cudaError_t e = dispatch(a, groups, stream);
    if (e != cudaSuccess || !(a.need_p || a.need_q || a.need_z)) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((a.dim + 31) / 32) *
                       (3u + (a.gate_mode == kGateGroups ? static_cast<unsigned>(groups) : 0u)));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, &block_norm_sums_kernel<T>, a, static_cast<int>(groups * a.parts_per_group));
}
#else
template <>
cudaError_t launch_block_norm_unit<CUBF_BN_TYPE>(const BlockNormArgs& a, cudaStream_t stream) {
    return dispatch(a, 1, stream);
}
#endif

}  // namespace cubf
