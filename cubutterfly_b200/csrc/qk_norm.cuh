// qk_norm.cuh -- norms of queries and keys head by head, with the rotation by
// the tokens' positions in the same pass.
//
// Per head x of D values:  n = x r(x),  r = 1/sqrt(mean(x^2) + eps)  or, for
// heads of length one, 1/sqrt(sum(x^2) + eps);  y = n weight;  each rotated
// pair (a, b) of y with angle phi = position frequency becomes
// (a cos phi - b sin phi, b cos phi + a sin phi).
// Backward: the gradient of y is the output's rotated by -phi,
// d_weight = sum of d_y n, and with t = d_y weight:  d_x = r (t - n mean(t n))
// (sum in place of mean for heads of length one).
//
// Bounded by memory: every head is read once and written once.  A warp takes
// one token and runs through its heads, 32 / G at a time, a group of G lanes
// each, so that a lane's sines and cosines serve all heads of the token.  A
// lane holds pairs: of rotated halves the same 16 bytes of either half, of
// adjacent pairs 32 bytes side by side, so neither needs an exchange.
//
// Angles: a position times a frequency is taken modulo one turn in 64-bit
// integers (the frequency in turns times 2^64, from a product in fp64), so
// that far positions keep every bit: the angle's error is 2e-7 at position
// 2^31 and frequency 1, where fp32 products would be off by whole turns.
#pragma once

#include "common.cuh"
#include "qk_norm.hpp"

namespace cubf::qk {

constexpr int kWarps = 8;
constexpr int kMaxPairs = kQkNormMaxDim / 2;

// What a lane holds: pairs first(), first() + 1, ... (VEC) or every G-th one.
struct Layout {
    int dim, half, rest;                 // rotated pairs; pairs of what is not rotated
    int pairs, lanes;                    // all pairs; lanes of a head (a power of two)
    bool interleaved;
    CUBF_DEV int a(int p) const { return interleaved ? 2 * p : p < half ? p : half + p; }
    CUBF_DEV int b(int p) const { return interleaved ? 2 * p + 1 : p < half ? half + p : half + rest + p; }
};
CUBF_DEV Layout layout_of(const QkNormArgs& a, int per_lane) {
    Layout l{a.dim, a.rotary / 2, 0, 0, 1, a.interleaved};
    l.rest = (a.dim - a.rotary + 1) / 2;
    l.pairs = l.half + l.rest;
    while (l.lanes * per_lane < l.pairs) l.lanes *= 2;
    return l;
}

template <typename T, int NP, bool VEC>
struct Pairs {
    float a[NP], b[NP];
    static CUBF_DEV int pair(const Layout& l, int lane, int i) { return VEC ? lane * NP + i : lane + l.lanes * i; }

    CUBF_DEV void load(const T* p, const Layout& l, int lane) {
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
            static_assert(N == NP, "a vector of either half");
            Vec16<T> x{}, y{};
            const int first = lane * NP;
            if (first < l.pairs) {
                x = *reinterpret_cast<const Vec16<T>*>(p + l.a(first));
                y = *reinterpret_cast<const Vec16<T>*>(p + (l.interleaved ? 2 * first + N : l.b(first)));
            }
            if (l.interleaved) {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const Vec16<T>& v = i < NP / 2 ? x : y;
                    a[i] = Convert<T, float>::load(v.v[2 * i % N]);
                    b[i] = Convert<T, float>::load(v.v[2 * i % N + 1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    a[i] = Convert<T, float>::load(x.v[i]);
                    b[i] = Convert<T, float>::load(y.v[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int q = pair(l, lane, i);
                a[i] = q < l.pairs ? Convert<T, float>::load(p[l.a(q)]) : 0.f;
                b[i] = q < l.pairs && l.b(q) < l.dim ? Convert<T, float>::load(p[l.b(q)]) : 0.f;
            }
        }
    }
    CUBF_DEV void store(T* p, const Layout& l, int lane) const {
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
            const int first = lane * NP;
            if (first >= l.pairs) return;
            Vec16<T> x, y;
            if (l.interleaved) {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    Vec16<T>& v = i < NP / 2 ? x : y;
                    v.v[2 * i % N] = Convert<T, float>::store(a[i]);
                    v.v[2 * i % N + 1] = Convert<T, float>::store(b[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    x.v[i] = Convert<T, float>::store(a[i]);
                    y.v[i] = Convert<T, float>::store(b[i]);
                }
            }
            *reinterpret_cast<Vec16<T>*>(p + l.a(first)) = x;
            *reinterpret_cast<Vec16<T>*>(p + (l.interleaved ? 2 * first + N : l.b(first))) = y;
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int q = pair(l, lane, i);
                if (q < l.pairs) {
                    p[l.a(q)] = Convert<T, float>::store(a[i]);
                    if (l.b(q) < l.dim) p[l.b(q)] = Convert<T, float>::store(b[i]);
                }
            }
        }
    }
    CUBF_DEV void turn(const float (&c)[NP], const float (&s)[NP], float sign) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * c[i] - y * (s[i] * sign);
            b[i] = y * c[i] + x * (s[i] * sign);
        }
    }
};

struct Shared {
    alignas(16) float weight[2][2][kMaxPairs];      // q's and k's, of the pairs' first and second values
    unsigned long long turns[kMaxPairs];            // frequency / 2 pi, of a turn times 2^64
    int axis[kMaxPairs];
};

// Weights and frequencies in the order of the pairs.
template <typename T>
CUBF_DEV void prepare(const QkNormArgs& a, const Layout& l, Shared& sm) {
    for (int p = threadIdx.x; p < kMaxPairs; p += 32 * kWarps) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const void* w = which ? a.k_weight : a.q_weight;
            const bool wide = which ? a.k_weight32 : a.q_weight32;
            auto at = [&](int i) {
                if (!w || i >= l.dim) return 1.f;
                return wide ? static_cast<const float*>(w)[i] : Convert<T, float>::load(static_cast<const T*>(w)[i]);
            };
            sm.weight[which][0][p] = p < l.pairs ? at(l.a(p)) : 1.f;
            sm.weight[which][1][p] = p < l.pairs ? at(l.b(p)) : 1.f;
        }
        const bool turned = p < l.half;
        double x = turned ? static_cast<double>(a.frequencies[p]) * 0.15915494309189533577 : 0.0;
        x -= floor(x);                              // whole turns a position drop out
        sm.turns[p] = static_cast<unsigned long long>(x * 18446744073709551616.0);
        sm.axis[p] = turned && a.axes ? min(max(a.axes[p], 0), a.axis_count - 1) : 0;
    }
    __syncthreads();
}

template <typename T, int NP, bool VEC>
CUBF_DEV void angles(const QkNormArgs& a, const Layout& l, const Shared& sm, size_t token, int lane, float (&c)[NP],
                     float (&s)[NP]) {
    const size_t at = token % a.positions_period;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int p = min(Pairs<T, NP, VEC>::pair(l, lane, i), kMaxPairs - 1);
        const size_t place = sm.axis[p] * a.positions_axis + at;
        const long long position = a.positions64 ? static_cast<const long long*>(a.positions)[place]
                                                 : static_cast<const int*>(a.positions)[place];
        const unsigned long long phase = static_cast<unsigned long long>(position) * sm.turns[p];
        // -1 .. 1: half turns
        const float x = static_cast<float>(static_cast<int>(phase >> 32)) * 4.656612873077393e-10f;
        sincospif(x, &s[i], &c[i]);
    }
}

CUBF_DEV float group_sum(float v, int lanes) {
    for (int d = lanes / 2; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// `unit_heads` heads of a token a warp.
template <typename T, int NP, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) qk_norm_kernel(QkNormArgs a, int unit_heads, int units_per_token) {
    __shared__ Shared sm;
    pdl_begin();
    const Layout l = layout_of(a, NP);
    prepare<T>(a, l, sm);
    const int lane = threadIdx.x & 31, in_group = lane & (l.lanes - 1), group = lane / l.lanes, groups = 32 / l.lanes;
    const int all_heads = a.q_heads + a.k_heads;
    const float share = a.length ? 1.f : 1.f / static_cast<float>(a.dim);
    const size_t units = a.batch * a.tokens * units_per_token;
    for (size_t unit = static_cast<size_t>(blockIdx.x) * kWarps + threadIdx.x / 32; unit < units;
         unit += static_cast<size_t>(gridDim.x) * kWarps) {
        const size_t token = unit / units_per_token;
        const int first = static_cast<int>(unit % units_per_token) * unit_heads, last = min(first + unit_heads, all_heads);
        const size_t row = token / a.tokens, in_row = token % a.tokens;
        float c[NP], s[NP];
        if (a.positions) angles<T, NP, VEC>(a, l, sm, token, in_group, c, s);
        constexpr int TURN = 2;              // heads of a lane group loaded together
        for (int base = first; base < last; base += TURN * groups) {
            Pairs<T, NP, VEC> x[TURN];
#pragma unroll
            for (int u = 0; u < TURN; ++u) {
                const int head = min(base + u * groups + group, last - 1);
                const bool key = head >= a.q_heads;
                const HeadTensor& t = key ? a.k : a.q;
                x[u].load(static_cast<const T*>(t.p) + row * t.batch + in_row * t.token +
                              static_cast<size_t>(key ? head - a.q_heads : head) * t.head,
                          l, in_group);
            }
#pragma unroll
            for (int u = 0; u < TURN; ++u) {
                const int head = base + u * groups + group;
                const bool key = head >= a.q_heads;
                float squares = 0.f;
#pragma unroll
                for (int i = 0; i < NP; ++i) squares = fmaf(x[u].a[i], x[u].a[i], fmaf(x[u].b[i], x[u].b[i], squares));
                const float r = 1.f / sqrtf(fmaf(group_sum(squares, l.lanes), share, a.eps));
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const int p = min(Pairs<T, NP, VEC>::pair(l, in_group, i), kMaxPairs - 1);
                    x[u].a[i] *= r * sm.weight[key][0][p];
                    x[u].b[i] *= r * sm.weight[key][1][p];
                }
                if (a.positions) x[u].turn(c, s, 1.f);
                if (head < last) {
                    T* out = key ? static_cast<T*>(a.k_out) + (token * a.k_heads + head - a.q_heads) * a.dim
                                 : static_cast<T*>(a.q_out) + (token * a.q_heads + head) * a.dim;
                    x[u].store(out, l, in_group);
                }
            }
        }
    }
}

// The same walk; each CTA leaves its sums of the weights' gradients in `partials`.
template <typename T, int NP, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) qk_norm_backward_kernel(QkNormArgs a) {
    __shared__ Shared sm;
    __shared__ float sums[kWarps][2][2][kMaxPairs];
    pdl_begin();
    const Layout l = layout_of(a, NP);
    prepare<T>(a, l, sm);
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int in_group = lane & (l.lanes - 1), group = lane / l.lanes, groups = 32 / l.lanes;
    const float share = a.length ? 1.f : 1.f / static_cast<float>(a.dim);
    const size_t tokens = a.batch * a.tokens;
    float wa[2][NP] = {}, wb[2][NP] = {};
    for (size_t token = static_cast<size_t>(blockIdx.x) * kWarps + warp; token < tokens;
         token += static_cast<size_t>(gridDim.x) * kWarps) {
        const size_t row = token / a.tokens, in_row = token % a.tokens;
        float c[NP], s[NP];
        if (a.positions) angles<T, NP, VEC>(a, l, sm, token, in_group, c, s);
#pragma unroll
        for (int key = 0; key < 2; ++key) {
            const int heads = key ? a.k_heads : a.q_heads;
            const HeadTensor &t = key ? a.k : a.q, &d = key ? a.d_k_out : a.d_q_out;
            const T* const xs = static_cast<const T*>(t.p) + row * t.batch + in_row * t.token;
            const T* const ds = static_cast<const T*>(d.p) + row * d.batch + in_row * d.token;
            T* const out = static_cast<T*>(key ? a.d_k : a.d_q) + token * heads * a.dim;
            for (int base = 0; base < heads; base += groups) {
                const int head = base + group;
                const bool own = head < heads;
                Pairs<T, NP, VEC> x, g;
                x.load(xs + static_cast<size_t>(own ? head : heads - 1) * t.head, l, in_group);
                g.load(ds + static_cast<size_t>(own ? head : heads - 1) * d.head, l, in_group);
                if (a.positions) g.turn(c, s, -1.f);
                float squares = 0.f;
#pragma unroll
                for (int i = 0; i < NP; ++i) squares = fmaf(x.a[i], x.a[i], fmaf(x.b[i], x.b[i], squares));
                const float r = 1.f / sqrtf(fmaf(group_sum(squares, l.lanes), share, a.eps));
                float along = 0.f;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const int p = min(Pairs<T, NP, VEC>::pair(l, in_group, i), kMaxPairs - 1);
                    x.a[i] *= r;                    // n
                    x.b[i] *= r;
                    if (own) {
                        wa[key][i] = fmaf(g.a[i], x.a[i], wa[key][i]);
                        wb[key][i] = fmaf(g.b[i], x.b[i], wb[key][i]);
                    }
                    g.a[i] *= sm.weight[key][0][p];
                    g.b[i] *= sm.weight[key][1][p];
                    along = fmaf(g.a[i], x.a[i], fmaf(g.b[i], x.b[i], along));
                }
                along = group_sum(along, l.lanes) * share;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    g.a[i] = r * fmaf(-x.a[i], along, g.a[i]);
                    g.b[i] = r * fmaf(-x.b[i], along, g.b[i]);
                }
                if (own) g.store(out + static_cast<size_t>(head) * a.dim, l, in_group);
            }
        }
    }
    if (!a.q_weight && !a.k_weight) return;
    // lane groups, then warps
#pragma unroll
    for (int key = 0; key < 2; ++key)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            for (int d = l.lanes; d < 32; d *= 2) {
                wa[key][i] += __shfl_xor_sync(0xffffffffu, wa[key][i], d);
                wb[key][i] += __shfl_xor_sync(0xffffffffu, wb[key][i], d);
            }
            const int p = Pairs<T, NP, VEC>::pair(l, in_group, i);
            if (group == 0 && p < l.pairs) {
                sums[warp][key][0][p] = wa[key][i];
                sums[warp][key][1][p] = wb[key][i];
            }
        }
    __syncthreads();
    float* const part = a.partials + static_cast<size_t>(blockIdx.x) * 2 * a.dim;
    for (int e = threadIdx.x; e < 4 * l.pairs; e += 32 * kWarps) {
        const int key = e / (2 * l.pairs), second = e / l.pairs % 2, p = e % l.pairs;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sums[w][key][second][p];
        const int at = second ? l.b(p) : l.a(p);
        if (at < l.dim) part[key * a.dim + at] = v;
    }
}

// Sums of the CTAs' parts: a warp for 32 channels, its CTA's warps taking turns with the parts.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) qk_norm_weights_kernel(QkNormArgs a) {
    __shared__ float sums[kWarps][32];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int at = blockIdx.x * 32 + lane;       // of both weights side by side
    float v = 0.f;
    if (at < 2 * a.dim)
        for (int part = warp; part < a.parts; part += kWarps) v += a.partials[static_cast<size_t>(part) * 2 * a.dim + at];
    sums[warp][lane] = v;
    __syncthreads();
    if (warp > 0 || at >= 2 * a.dim) return;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v += sums[w][lane];
    const bool key = at >= a.dim;
    void* const out = key ? a.d_k_weight : a.d_q_weight;
    if (!out) return;
    const int i = key ? at - a.dim : at;
    if (key ? a.k_weight32 : a.q_weight32)
        static_cast<float*>(out)[i] = v;
    else
        static_cast<T*>(out)[i] = Convert<T, float>::store(v);
}

}  // namespace cubf::qk
