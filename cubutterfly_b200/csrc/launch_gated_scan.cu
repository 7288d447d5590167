// launch_gated_scan.cu -- launches of the gated linear recurrence.
#include <algorithm>
#include <cstdlib>

#include "gated_scan.cuh"
#include "launch_util.cuh"

namespace cubf {
namespace {

using namespace scan;
static_assert(kGatedScanBackwardTile == kBackwardSteps * kWarps, "the workspace is sized for the backward's clusters");

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename... Args>
cudaError_t launch_clusters(void (*kernel)(Args...), unsigned grid, unsigned threads, int smem, int cluster,
                            cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The widest access every row of every tensor is aligned for.
template <typename T>
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
    Access access() const {
        if ((bits & 15) == 0) return kAsync;
        return (bits & (2 * sizeof(T) - 1)) == 0 ? kPairs : kScalar;
    }
};

template <typename T>
Access access_of(const GatedScanArgs& a, bool backward) {
    Alignment<T> v;
    v.stride(static_cast<size_t>(a.dim)).pointer(a.x).pointer(a.r).pointer(a.i);
    v.stride(a.x_batch).stride(a.r_batch).stride(a.i_batch).stride(a.x_token).stride(a.r_token).stride(a.i_token);
    if (backward)
        v.pointer(a.d_h).pointer(a.d_x).pointer(a.d_r).pointer(a.d_i).stride(a.dh_batch).stride(a.dh_token);
    else
        v.pointer(a.h);
    return v.access();
}

template <typename T, bool PACKED, bool CLUSTER, Access ACCESS, bool BACKWARD>
cudaError_t launch_kernel(const GatedScanArgs& a, int cluster, cudaStream_t stream) {
    static KernelSetup setup;
    const auto kernel = [] {
        if constexpr (BACKWARD)
            return &gated_scan_backward_kernel<T, PACKED, CLUSTER, ACCESS>;
        else
            return &gated_scan_kernel<T, PACKED, CLUSTER, ACCESS>;
    }();
    using Tile = std::conditional_t<BACKWARD, BackwardRows<T, ACCESS>, ForwardRows<T, ACCESS>>;
    constexpr int smem = kWarps * Tile::STAGES * Tile::kBytes;
    int cap = 0;
    // two CTAs per SM fit only in the largest carveout
    cudaError_t e = setup_kernel(setup, kernel, kWarps * 32, smem, &cap, ACCESS == kAsync);
    if (e != cudaSuccess) return e;
    const int tiles = ceil_div(a.dim, kChannels);
    const size_t grid = static_cast<size_t>(tiles) * a.batch * cluster;
    if (grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    return launch_clusters(kernel, static_cast<unsigned>(grid), kWarps * 32u, smem, cluster, stream, a, cluster, tiles);
}

template <typename T, bool PACKED, Access ACCESS, bool BACKWARD>
cudaError_t launch_split(const GatedScanArgs& a, cudaStream_t stream) {
    const int tile = (BACKWARD ? kBackwardSteps : kForwardSteps<T>) * kWarps;
    const int cluster = gated_scan_cluster(a.batch, a.length, a.dim, tile);
    return cluster > 1 ? launch_kernel<T, PACKED, true, ACCESS, BACKWARD>(a, cluster, stream)
                       : launch_kernel<T, PACKED, false, ACCESS, BACKWARD>(a, 1, stream);
}

template <typename T, bool PACKED, bool BACKWARD>
cudaError_t launch_access(const GatedScanArgs& a, cudaStream_t stream) {
    switch (access_of<T>(a, BACKWARD)) {
        case kAsync: return launch_split<T, PACKED, kAsync, BACKWARD>(a, stream);
        case kPairs: return launch_split<T, PACKED, kPairs, BACKWARD>(a, stream);
        default: return launch_split<T, PACKED, kScalar, BACKWARD>(a, stream);
    }
}

template <typename T>
cudaError_t launch_typed(const GatedScanArgs& a, bool backward, cudaStream_t stream) {
    if (a.offsets) return backward ? launch_access<T, true, true>(a, stream) : launch_access<T, true, false>(a, stream);
    return backward ? launch_access<T, false, true>(a, stream) : launch_access<T, false, false>(a, stream);
}

cudaError_t launch_any(BlockType type, const GatedScanArgs& a, bool backward, cudaStream_t stream) {
    switch (type) {
        case BlockType::kF16: return launch_typed<__half>(a, backward, stream);
        case BlockType::kBF16: return launch_typed<__nv_bfloat16>(a, backward, stream);
        case BlockType::kF32: return launch_typed<float>(a, backward, stream);
    }
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t launch_step_typed(const GatedStepArgs& a, cudaStream_t stream) {
    Alignment<T> v;
    v.stride(static_cast<size_t>(a.dim)).pointer(a.x).pointer(a.r).pointer(a.i).pointer(a.h);
    v.stride(a.x_row).stride(a.r_row).stride(a.i_row);
    const int tiles = ceil_div(a.dim, kChannels);
    // about 32 warps per SM before a warp takes a second request
    const size_t groups = std::max<size_t>(1, static_cast<size_t>(148 * 32) / tiles);
    const size_t rows = (a.batch + groups - 1) / groups;
    const size_t tasks = (a.batch + rows - 1) / rows * tiles;
    const size_t grid = (tasks + 3) / 4;
    if (grid > 0x7fffffffULL || rows > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    return launch_dependent(v.access() == kScalar ? &gated_scan_step_kernel<T, kScalar> : &gated_scan_step_kernel<T, kPairs>,
                            static_cast<unsigned>(grid), 128u, 0, stream, a, tiles, static_cast<int>(rows));
}

}  // namespace

int gated_scan_cluster(int batch, int length, int dim, int tile) {
    if (getenv("CUBF_K")) return atoi(getenv("CUBF_K"));
    const size_t columns = static_cast<size_t>(ceil_div(dim, kChannels)) * batch;
    const int tiles = ceil_div(length, tile);
    int best = 1;
    double least = 0;
    for (int k = 1; k <= kGatedScanMaxCluster; k *= 2) {
        const double waves = static_cast<double>((columns * k + 295) / 296);
        const double cost = waves * ceil_div(tiles, k) * (k > 1 ? 1.15 : 1.0);
        if (k == 1 || cost < least) {
            best = k;
            least = cost;
        }
    }
    return best;
}

cudaError_t launch_gated_scan(BlockType type, const GatedScanArgs& a, cudaStream_t stream) {
    return launch_any(type, a, false, stream);
}

cudaError_t launch_gated_scan_backward(BlockType type, const GatedScanArgs& a, cudaStream_t stream) {
    cudaError_t e = launch_any(type, a, true, stream);
    if (e != cudaSuccess) return e;
    const int parts = a.batch * gated_scan_cluster(a.batch, a.length, a.dim, kGatedScanBackwardTile);
    return launch_dependent(&gated_scan_decay_kernel, static_cast<unsigned>(ceil_div(a.dim, 32)), 256u, 0, stream, a,
                            parts);
}

cudaError_t launch_gated_scan_step(BlockType type, const GatedStepArgs& a, cudaStream_t stream) {
    switch (type) {
        case BlockType::kF16: return launch_step_typed<__half>(a, stream);
        case BlockType::kBF16: return launch_step_typed<__nv_bfloat16>(a, stream);
        case BlockType::kF32: return launch_step_typed<float>(a, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace cubf
