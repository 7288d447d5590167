// launch_qk_norm.cu -- launches of the norm of queries and keys.
#include <algorithm>

#include "launch_util.cuh"
#include "qk_norm.cuh"

namespace cubf {
namespace {

using namespace qk;

// Whole 16-byte vectors of every head: both halves of the pairs in the vector's steps, and aligned.
template <typename T>
bool vectors(const QkNormArgs& a, bool backward) {
    constexpr size_t n = 16 / sizeof(T);
    const size_t half = a.rotary / 2, rest = a.dim - a.rotary;
    if (a.interleaved ? a.dim % (2 * n) != 0 : (half % n != 0 || rest % (2 * n) != 0)) return false;
    size_t bits = static_cast<size_t>(a.dim) * sizeof(T);
    auto take = [&](const HeadTensor& t) {
        bits |= reinterpret_cast<uintptr_t>(t.p) | (t.batch | t.token | t.head) * sizeof(T);
    };
    take(a.q);
    take(a.k);
    if (backward) {
        take(a.d_q_out);
        take(a.d_k_out);
    }
    for (const void* p : {a.q_out, a.k_out, a.d_q, a.d_k}) bits |= reinterpret_cast<uintptr_t>(p);
    return bits % 16 == 0;
}

template <typename T, int NP, bool VEC, bool WEIGHTED, bool TURNED>
cudaError_t launch_kernel(const QkNormArgs& a, bool backward, cudaStream_t stream) {
    if (backward)
        return launch_dependent(&qk_norm_backward_kernel<T, NP, VEC, WEIGHTED, TURNED>, static_cast<unsigned>(a.parts),
                                32u * kWarps, 0, stream, a);
    // all heads of a token a warp, fewer while that leaves an SM less than two turns of its 32 warps
    const size_t tokens = a.batch * a.tokens;
    const int heads = a.q_heads + a.k_heads;
    int lanes = 1;
    const int pairs = a.rotary / 2 + (a.dim - a.rotary + 1) / 2;
    while (lanes * NP < pairs) lanes *= 2;
    const int turn = 32 / lanes;                 // heads that a warp takes side by side
    int unit = (heads + turn - 1) / turn * turn;
    while (unit > turn && tokens * ((heads + unit - 1) / unit) < 148 * 64) unit = (unit / turn + 1) / 2 * turn;
    const int per_token = (heads + unit - 1) / unit;
    // At most two rounds of the four CTAs an SM, since each lays out weights and frequencies first.  One round of CTAs that stay
    // saves that (2500 tokens of 32 + 8 heads of 128 16.6 us for 18.6) but leaves the last turn's SMs idle (16384 tokens 86.7 for 78.8).
    const size_t grid = std::min<size_t>((tokens * per_token + kWarps - 1) / kWarps, 148 * 8);
    return launch_dependent(&qk_norm_kernel<T, NP, VEC, WEIGHTED, TURNED>, static_cast<unsigned>(grid), 32u * kWarps, 0, stream,
                            a, unit, per_token);
}

template <typename T, int NP, bool VEC>
cudaError_t launch_options(const QkNormArgs& a, bool backward, cudaStream_t stream) {
    if (a.q_weight || a.k_weight)
        return a.positions ? launch_kernel<T, NP, VEC, true, true>(a, backward, stream)
                           : launch_kernel<T, NP, VEC, true, false>(a, backward, stream);
    return a.positions ? launch_kernel<T, NP, VEC, false, true>(a, backward, stream)
                       : launch_kernel<T, NP, VEC, false, false>(a, backward, stream);
}

template <typename T>
cudaError_t launch(QkNormArgs a, bool backward, cudaStream_t stream) {
    if (a.rotary == 0) a.interleaved = true;     // any pairs do: adjacent ones are read in the widest pieces
    const cudaError_t e = vectors<T>(a, backward) ? launch_options<T, 16 / sizeof(T), true>(a, backward, stream)
                                                  : launch_options<T, 4, false>(a, backward, stream);
    if (e != cudaSuccess || !backward || (!a.q_weight && !a.k_weight)) return e;
    return launch_dependent(&qk_norm_weights_kernel<T>, static_cast<unsigned>((2 * a.dim + 31) / 32), 32u * kWarps, 0,
                            stream, a);
}

}  // namespace

int qk_norm_parts(const QkNormArgs& a) {
    // a token a warp, four CTAs of 8 warps per SM at most
    return static_cast<int>(std::min<size_t>((a.batch * a.tokens + kWarps - 1) / kWarps, 148 * 4));
}

cudaError_t launch_qk_norm(BlockType type, const QkNormArgs& a, bool backward, cudaStream_t stream) {
    switch (type) {
        case BlockType::kF16: return launch<__half>(a, backward, stream);
        case BlockType::kBF16: return launch<__nv_bfloat16>(a, backward, stream);
        default: return launch<float>(a, backward, stream);
    }
}

}  // namespace cubf
