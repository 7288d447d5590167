// launch_gated_scan.cu -- launches of the gated linear recurrence; compiled
// once per CUBF_GS_TYPE (0 fp16, 1 bf16, 2 fp32).
#include <algorithm>

#include "gated_scan.cuh"
#include "launch_util.cuh"

#ifndef CUBF_GS_TYPE
#define CUBF_GS_TYPE 1
#endif

namespace cubf {

template <int TYPE>
cudaError_t launch_gated_scan_unit(const GatedScanArgs& a, bool backward, cudaStream_t stream);
template <int TYPE>
cudaError_t launch_gated_scan_step_unit(const GatedStepArgs& a, cudaStream_t stream);

namespace {

using namespace scan;
using T = std::conditional_t<CUBF_GS_TYPE == 0, __half, std::conditional_t<CUBF_GS_TYPE == 1, __nv_bfloat16, float>>;

constexpr int kTwoPerSM = 110 * 1024;  // dynamic shared memory of a CTA that fits twice beside the static 2 to 6 KB

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// The widest access, in bytes, that every row of every tensor is aligned for.
struct Alignment {
    uintptr_t bits = 0;  // of addresses and strides in bytes
    Alignment& pointer(const void* p) {
        bits |= reinterpret_cast<uintptr_t>(p);
        return *this;
    }
    Alignment& stride(size_t elements) {
        bits |= elements * sizeof(T);
        return *this;
    }
    int bytes() const { return static_cast<int>(16 | bits) & -static_cast<int>(16 | bits); }
};

int piece_of(const GatedScanArgs& a, bool backward) {
    Alignment v;
    v.stride(static_cast<size_t>(a.dim)).pointer(a.x).pointer(a.r).pointer(a.i);
    v.stride(a.x_batch).stride(a.r_batch).stride(a.i_batch).stride(a.x_token).stride(a.r_token).stride(a.i_token);
    if (backward)
        v.pointer(a.d_h).pointer(a.d_x).pointer(a.d_r).pointer(a.d_i).stride(a.dh_batch).stride(a.dh_token);
    else
        v.pointer(a.h);
    return v.bytes();
}

// Lane groups along time: each doubling makes twice as many CTAs, of half the
// channels and twice the tokens a round.  Whole rows of 64 channels run
// fastest once the CTAs fill the GPU (8 x 2048 x 2048 bf16, 256, 512, 1024 and
// 2048 CTAs: 60, 62, 69, 105 us forward, 101, 119, 122, 208 backward); below
// that more CTAs win (16384 x 4096, 64 to 512 CTAs: 230, 115, 119, 196 us
// forward and 402, 290, 246, 442 backward, whose turns want two CTAs per SM).
// Shifted rows take more shared memory: where only one CTA of twice the groups
// fits on an SM, those are taken while they make no second wave (13 x 8000 x 143
// bf16 backward, 117 and 234 CTAs: 259, 317 us; 32730 x 425, 27 and 54: 976, 588).
int lane_groups(const GatedScanArgs& a, bool backward, int piece) {
    const int steps = backward ? kBackwardSteps : piece < 16 ? kForwardSteps<T, 4> : kForwardSteps<T, 16>;
    const int tile = steps * kWarps;
    const int stage = (backward ? 4 * BackwardRows<T, 1, 16>::STAGES : 3 * ForwardRows<T, 1, 16>::STAGES) * tile;
    int g = 1;
    while (g < 8 && a.length > g * tile) {
        const int shared = stage * (kWarpChannels * static_cast<int>(sizeof(T)) + (piece < 16 ? 2 * g * 16 : 0));
        const int enough = shared > kTwoPerSM ? 74 : backward ? 240 : 120;
        if (ceil_div(a.dim, kWarpChannels / g) * static_cast<long long>(a.batch) >= enough) break;
        g *= 2;
    }
    return g;
}

template <bool PACKED, int GROUPS, int PIECE, bool BACKWARD>
cudaError_t launch_kernel(const GatedScanArgs& a, cudaStream_t stream) {
    static KernelSetup setup;
    const auto kernel = [] {
        if constexpr (BACKWARD)
            return &gated_scan_backward_kernel<T, PACKED, GROUPS, PIECE>;
        else
            return &gated_scan_kernel<T, PACKED, GROUPS, PIECE>;
    }();
    using Tile = std::conditional_t<BACKWARD, BackwardRows<T, GROUPS, PIECE>, ForwardRows<T, GROUPS, PIECE>>;
    constexpr int smem = kWarps * Tile::STAGES * Tile::kBytes;
    int cap = 0;
    // two CTAs per SM fit only in the largest carveout
    cudaError_t e = setup_kernel(setup, kernel, kWarps * 32, smem, &cap, true);
    if (e != cudaSuccess) return e;
    const int tiles = ceil_div(a.dim, Tile::kChannels);
    const size_t grid = static_cast<size_t>(tiles) * a.batch;
    if (grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    return launch_dependent(kernel, static_cast<unsigned>(grid), kWarps * 32u, smem, stream, a, tiles);
}

template <bool PACKED, bool BACKWARD>
cudaError_t launch_access(const GatedScanArgs& a, cudaStream_t stream) {
    const int piece = piece_of(a, BACKWARD);
    const int groups = lane_groups(a, BACKWARD, piece);
    if (piece >= 16) {
        switch (groups) {
            case 1: return launch_kernel<PACKED, 1, 16, BACKWARD>(a, stream);
            case 2: return launch_kernel<PACKED, 2, 16, BACKWARD>(a, stream);
            case 4: return launch_kernel<PACKED, 4, 16, BACKWARD>(a, stream);
            default: return launch_kernel<PACKED, 8, 16, BACKWARD>(a, stream);
        }
    }
    if (piece >= 4) {
        switch (groups) {
            case 1: return launch_kernel<PACKED, 1, 4, BACKWARD>(a, stream);
            case 2: return launch_kernel<PACKED, 2, 4, BACKWARD>(a, stream);
            case 4: return launch_kernel<PACKED, 4, 4, BACKWARD>(a, stream);
            default: return launch_kernel<PACKED, 8, 4, BACKWARD>(a, stream);
        }
    }
    if constexpr (sizeof(T) == 2) {
        switch (groups) {
            case 1: return launch_kernel<PACKED, 1, 2, BACKWARD>(a, stream);
            case 2: return launch_kernel<PACKED, 2, 2, BACKWARD>(a, stream);
            case 4: return launch_kernel<PACKED, 4, 2, BACKWARD>(a, stream);
            default: return launch_kernel<PACKED, 8, 2, BACKWARD>(a, stream);
        }
    }
    return cudaErrorMisalignedAddress;
}

}  // namespace

template <>
cudaError_t launch_gated_scan_unit<CUBF_GS_TYPE>(const GatedScanArgs& a, bool backward, cudaStream_t stream) {
    if (!backward) return a.offsets ? launch_access<true, false>(a, stream) : launch_access<false, false>(a, stream);
    const cudaError_t e = a.offsets ? launch_access<true, true>(a, stream) : launch_access<false, true>(a, stream);
    if (e != cudaSuccess) return e;
    return launch_dependent(&gated_scan_decay_kernel<T>, static_cast<unsigned>(ceil_div(a.dim, 32)), 256u, 0, stream, a,
                            a.batch);
}

template <>
cudaError_t launch_gated_scan_step_unit<CUBF_GS_TYPE>(const GatedStepArgs& a, cudaStream_t stream) {
    Alignment v;
    v.stride(static_cast<size_t>(a.dim)).pointer(a.x).pointer(a.r).pointer(a.i).pointer(a.h);
    v.stride(a.x_row).stride(a.r_row).stride(a.i_row);
    const int tiles = ceil_div(a.dim, kWarpChannels);
    // one request a warp while that is no more than 32 warps per SM
    const size_t groups = std::max<size_t>(1, static_cast<size_t>(148 * 32) / tiles);
    const size_t rows = (a.batch + groups - 1) / groups;
    const size_t tasks = (a.batch + rows - 1) / rows * tiles;
    const size_t grid = (tasks + 3) / 4;
    if (grid > 0x7fffffffULL || rows > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    const bool pairs = v.bytes() >= 2 * static_cast<int>(sizeof(T));
    const bool wide = a.dim % 2 == 0 &&
                      ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.new_state)) & 7u) == 0;
    const auto kernel = pairs ? (wide ? &gated_scan_step_kernel<T, true, true> : &gated_scan_step_kernel<T, true, false>)
                              : (wide ? &gated_scan_step_kernel<T, false, true> : &gated_scan_step_kernel<T, false, false>);
    return launch_dependent(kernel, static_cast<unsigned>(grid), 128u, 0, stream, a, tiles, static_cast<int>(rows));
}

}  // namespace cubf
