// launch_gated_delta.cu -- launches of the gated delta rule; compiled once per
// CUBF_GD_TYPE (0 fp16, 1 bf16, 2 fp32) and CUBF_GD_K (64 or 128: the padded
// key size).
#include <algorithm>
#include <cmath>

#ifndef CUBF_GD_TYPE
#define CUBF_GD_TYPE 1
#endif
#ifndef CUBF_GD_K
#define CUBF_GD_K 128
#endif

// 16-bit tensors go through the 5th-generation tensor cores; three pieces of fp32 ones would not fit tensor memory.
#define CUBF_GD_TENSOR (CUBF_GD_TYPE != 2)
#if CUBF_GD_TENSOR
#include "gated_delta_tc.cuh"
#else
#include "gated_delta_fp32.cuh"
#endif
#include "launch_util.cuh"

namespace cubf {

template <int TYPE, int KP>
cudaError_t launch_gated_delta_unit(const GatedDeltaArgs& a, bool backward, cudaStream_t stream);
template <int TYPE, int KP>
size_t gated_delta_workspace_unit(const GatedDeltaArgs& a, bool backward);
template <int TYPE>
cudaError_t launch_gated_delta_step_unit(const GatedDeltaStepArgs& a, cudaStream_t stream);

namespace {

using namespace delta;
using T = std::conditional_t<CUBF_GD_TYPE == 0, __half, std::conditional_t<CUBF_GD_TYPE == 1, __nv_bfloat16, float>>;
constexpr int KP = CUBF_GD_K;

int ceil_div(int a, int b) { return (a + b - 1) / b; }

bool rows_aligned(const HeadTensor& t, int width) {
    const size_t bits = (t.batch | t.token | t.head | static_cast<size_t>(width)) * sizeof(T);
    return ((reinterpret_cast<uintptr_t>(t.p) | bits) & 15u) == 0;
}

int sequences_of(const GatedDeltaArgs& a) { return a.offsets ? a.sequences : a.batch; }

#if CUBF_GD_TENSOR
// Chunks a segment, 0 for none: the shortest time by what a chunk of a chain takes on one SM (2.4 us with its results
// forward, 2.9 backward, 1.9 without them), a state's join (4 us) and the CTAs that run at once, one per SM.  Of a packed
// batch the host knows the tokens and the sequences alone; n random cuts leave a longest piece of (1 + 1/2 + .. + 1/n) / n.
// Whole calls forward, one sequence of 16384 tokens: 32 heads 606 us in three segments against 804 in one, 12 heads 319 in
// seven against 705, 4 heads 192 in 16 against 649; forward and backward of 4 heads 582 in 12 against 1890.  Backward a
// chunk takes 4.5 us while every SM writes; but with 4.5 here the choices were the same or worse (training 4 x 4096 tokens of
// 20 heads 1615 us for 1490, 10007 tokens of 4 heads in 13 sequences 430 for 395).
int segment_length(const GatedDeltaArgs& a, bool backward) {
    double longest = ceil_div(a.length, C), all = longest * a.batch;
    const double sequences = sequences_of(a);
    if (a.offsets) {
        double share = 0;
        for (int n = 1; n <= a.sequences && n <= 1000; ++n) share += 1.0 / n;
        longest *= std::min(1.0, share / sequences);
    }
    if (longest < 16) return 0;
    const double full = backward ? 2.9 : 2.4;
    auto waves = [](double ctas) { return std::max(1.0, std::ceil(ctas / 148)); };
    double best = std::max(waves((backward ? 2 : 1) * sequences * a.heads) * all / sequences, longest) * full;
    int length = 0;
    for (int n = 2; n <= 64 && longest / n >= 4; ++n) {
        const int chunks = static_cast<int>(std::ceil(longest / n));
        const double segments = a.offsets ? all / chunks + sequences : sequences * std::ceil(longest / chunks);  // of all
        // of s segments, s - 1 ends, s - 2 maps and, backward, s - 1 ends of the reversed chain
        const double first = segments * a.heads * (backward ? 3 : 2) - (backward ? 4 : 3) * sequences * a.heads;
        const double time = waves(first) * chunks * 1.9 + (n - 2) * 4 + 10 +
                            waves((backward ? 2 : 1) * segments * a.heads) * chunks * full;
        if (time < 0.95 * best) best = time, length = chunks;
    }
    return length;
}
#endif

Places places_of(const GatedDeltaArgs& a, bool backward) {
    Places w{};
    w.slots = a.offsets ? a.length / C + a.sequences : a.batch * ceil_div(a.length, C);
    w.v_pitch = ceil_div(a.v_dim, 16) * 16;
    w.v_rows = ceil_div(a.v_dim, 64) * 64;
    w.state_piece = static_cast<size_t>(KP / 64) * w.v_rows * 128;
    const size_t chunks = static_cast<size_t>(w.slots) * a.heads, key_chunks = static_cast<size_t>(w.slots) * a.k_heads;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
#if CUBF_GD_TENSOR
    w.squares = (backward ? 6 : 4) * tc::kPanel;
    w.factors = take(chunks * kTcFactors * C * 4);
    w.solve = take(chunks * w.squares);
    w.packed = take(key_chunks * 2 * kInput<T> * KP * 128);
    w.values = take(chunks * w.v_rows * 128);
    w.segments.length = segment_length(a, backward);
    if (const int n = w.segments.length; n > 0) {
        w.segments.total = a.offsets ? (a.length / C + a.sequences) / n + a.sequences : a.batch * ceil_div(ceil_div(a.length, C), n);
        const size_t ends = static_cast<size_t>(w.segments.total) * a.heads;
        w.segments.ends = take(ends * a.k_dim * a.v_dim * 4);
        w.segments.maps = take(ends * KP * KP * 4);
        if (backward) w.segments.d_ends = take(ends * a.k_dim * a.v_dim * 4);
    }
    if (backward) {
        w.rows = take(chunks * kInput<T> * w.v_rows * 128);
        w.states = take(chunks * 2 * w.state_piece);
        w.d_states = take(chunks * 2 * w.state_piece);
        w.errors = take(chunks * 2 * w.v_rows * 128);
        w.d_writes = take(chunks * 2 * w.v_rows * 128);
    }
#else
    w.factors = take(chunks * kFactors * 4);
    w.solve = take(chunks * kPieces * kSquare * 2);
    w.attention = take(chunks * kPieces * kSquare * 2);
    w.packed = take(key_chunks * 2 * kPieces * C * KP * 2);
    if (backward) {
        w.states = take(chunks * w.v_pitch * KP * 4);
        w.d_states = take(chunks * w.v_pitch * KP * 4);
        w.errors = take(chunks * C * w.v_pitch * 4);
        w.d_writes = take(chunks * C * w.v_pitch * 4);
        if (a.heads != a.k_heads) {
            const size_t values = static_cast<size_t>(a.batch) * a.length * a.heads * a.k_dim;
            w.d_q = take(values * 4);
            w.d_k = take(values * 4);
        }
    }
#endif
    w.total = at;
    return w;
}

template <typename Kernel, typename... Args>
cudaError_t launch(KernelSetup& setup, Kernel kernel, size_t grid, int threads, int smem, cudaStream_t stream,
                   const Args&... args) {
    if (grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    int cap = 0;
    const cudaError_t e = setup_kernel(setup, kernel, threads, smem, &cap, true);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, static_cast<unsigned>(grid), static_cast<unsigned>(threads), smem, stream, args...);
}

#if !CUBF_GD_TENSOR
cudaError_t launch_chains(const GatedDeltaArgs& a, const Places& w, bool backward, cudaStream_t stream) {
    const int tiles = ceil_div(a.v_dim, 16), chains = sequences_of(a) * a.heads;
    ChainShape shape{};
    // a warp runs by itself: as many a CTA as fill the SMs, up to 8, which share the tiles of a chunk
    shape.warps = 8;
    while (shape.warps > 2 && (shape.warps / 2 >= tiles || static_cast<long long>(chains) * ceil_div(tiles, shape.warps) < 148))
        shape.warps /= 2;
    shape.warps = std::min(shape.warps, tiles);
    shape.slices = ceil_div(tiles, shape.warps);
    shape.wide_v = rows_aligned(a.v, a.v_dim);
    shape.wide_d = rows_aligned(a.d_o, a.v_dim);
    const HeadTensor out{backward ? a.d_v : a.o, 0, 0, static_cast<size_t>(a.v_dim)};
    shape.wide_o = rows_aligned(out, a.v_dim);
    const size_t grid = static_cast<size_t>(chains) * shape.slices;
    if (backward) {
        // set up for the largest CTA, launched with what this one's warps need
        static KernelSetup setup;
        constexpr int most = ChainTiles<KP>::bytes(8);
        int cap = 0;
        const auto kernel = &gated_delta_chains_kernel<KP>;
        const cudaError_t e = setup_kernel(setup, kernel, 256, most, &cap, true);
        if (e != cudaSuccess) return e;
        if (2 * grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
        return launch_dependent(kernel, static_cast<unsigned>(2 * grid), 32u * shape.warps,
                                ChainTiles<KP>::bytes(shape.warps), stream, a, w, shape);
    }
    static KernelSetup setup;
    constexpr int most = ChainTiles<KP>::bytes(8);
    int cap = 0;
    const auto kernel = &gated_delta_forward_kernel<KP>;
    const cudaError_t e = setup_kernel(setup, kernel, 256, most, &cap, true);
    if (e != cudaSuccess) return e;
    if (grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    return launch_dependent(kernel, static_cast<unsigned>(grid), 32u * shape.warps,
                             ChainTiles<KP>::bytes(shape.warps), stream, a, w, shape);
}
#endif

}  // namespace

template <>
size_t gated_delta_workspace_unit<CUBF_GD_TYPE, CUBF_GD_K>(const GatedDeltaArgs& a, bool backward) {
    return places_of(a, backward).total;
}

namespace {
cudaError_t launch_kernels(const GatedDeltaArgs& a, bool backward, cudaStream_t stream) {
    const Places w = places_of(a, backward);
    const size_t chunks = static_cast<size_t>(w.slots) * a.heads;
#if CUBF_GD_TENSOR
    const size_t key_chunks = static_cast<size_t>(w.slots) * a.k_heads;
    const int sequences = sequences_of(a);
    const size_t chains = static_cast<size_t>(w.segments.length ? w.segments.total : sequences) * a.heads;
    const bool wide_q = rows_aligned(a.q, a.k_dim) && rows_aligned(a.k, a.k_dim);
    const HeadTensor out{backward ? a.d_v : a.o, 0, 0, static_cast<size_t>(a.v_dim)};
    const bool wide_out = rows_aligned(out, a.v_dim);
    static KernelSetup prepare, prepare_backward, ends, join, forward, both, gradients;
    cudaError_t e = backward ? launch(prepare_backward, &gated_delta_tc_prepare_kernel<T, KP, true>, key_chunks, 128,
                                      sizeof(TcPrepareShared<T, KP, true>), stream, a, w, wide_q, rows_aligned(a.v, a.v_dim),
                                      rows_aligned(a.d_o, a.v_dim))
                             : launch(prepare, &gated_delta_tc_prepare_kernel<T, KP, false>, key_chunks, 128,
                                      sizeof(TcPrepareShared<T, KP, false>), stream, a, w, wide_q, rows_aligned(a.v, a.v_dim), false);
    if (e != cudaSuccess) return e;
    if (w.segments.length) {
        const int kinds = backward ? 3 : 2, slices = ceil_div(a.v_dim, kJoinColumns);
        e = launch(ends, &gated_delta_tc_ends_kernel<T, KP>, chains * kinds, kTcThreads, sizeof(TcShared<T, KP>), stream, a, w, kinds);
        if (e != cudaSuccess) return e;
        e = launch(join, &gated_delta_join_kernel<KP>, static_cast<size_t>(sequences) * a.heads * slices * (backward ? 2 : 1),
                   2 * KP, sizeof(JoinShared<KP>), stream, a, w, slices, backward);
        if (e != cudaSuccess) return e;
    }
    if (!backward)
        return launch(forward, &gated_delta_tc_forward_kernel<T, KP>, chains, kTcThreads, sizeof(TcShared<T, KP>), stream, a, w,
                      wide_out);
    e = launch(both, &gated_delta_tc_chains_kernel<T, KP>, 2 * chains, kTcThreads, sizeof(TcShared<T, KP>), stream, a, w, wide_out);
    if (e != cudaSuccess) return e;
    return launch(gradients, &gated_delta_tc_gradients_kernel<T, KP>, key_chunks, kGradientThreads,
                  sizeof(GradientShared<T, KP>), stream, a, w);
#else
    static KernelSetup prepare, gradients, share;
    cudaError_t e = launch(prepare, &gated_delta_prepare_kernel<KP>, chunks, 128, sizeof(PrepareShared<KP>), stream, a, w);
    if (e != cudaSuccess) return e;
    e = launch_chains(a, w, backward, stream);
    if (e != cudaSuccess || !backward) return e;
    constexpr int smem = sizeof(GradientsShared<KP>);
    e = launch(gradients, &gated_delta_gradients_kernel<KP>, chunks, 512, smem, stream, a, w);
    if (e != cudaSuccess || a.heads == a.k_heads) return e;
    const size_t values = static_cast<size_t>(a.batch) * a.length * a.k_heads * a.k_dim;
    return launch(share, &gated_delta_share_kernel, std::min<size_t>((values + 255) / 256, 148 * 8), 256, 0, stream, a, w,
                  values);
#endif
}
}  // namespace

template <>
cudaError_t launch_gated_delta_unit<CUBF_GD_TYPE, CUBF_GD_K>(const GatedDeltaArgs& a, bool backward, cudaStream_t stream) {
    const cudaError_t e = launch_kernels(a, backward, stream);
    if (e != cudaSuccess || !a.offsets) return e;
    static KernelSetup rest;
    return launch(rest, &gated_delta_rest_kernel<T>, 148, 256, 0, stream, a, backward);
}

#if CUBF_GD_K == 128
template <>
cudaError_t launch_gated_delta_step_unit<CUBF_GD_TYPE>(const GatedDeltaStepArgs& a, cudaStream_t stream) {
    const bool wide = a.v_dim % 4 == 0 &&
                      ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.new_state)) & 15u) == 0;
    const int slices = ceil_div(a.v_dim, wide ? 32 : 8);
    const size_t grid = a.batch * a.heads * slices;
    if (grid > 0x7fffffffULL) return cudaErrorInvalidConfiguration;
    const auto kernel = wide ? &gated_delta_step_kernel<T, 4> : &gated_delta_step_kernel<T, 1>;
    return launch_dependent(kernel, static_cast<unsigned>(grid), 128u, 0, stream, a, slices);
}
#endif

}  // namespace cubf
