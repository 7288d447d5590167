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
// one token (of few tokens, a part of its heads) and runs through its heads, 32 / G at a time, a group of G lanes
// each; its sines and cosines are computed once, a pair a lane, into a table
// that all heads read.  A lane holds pairs: of rotated halves the same 16 bytes
// of either half, of adjacent pairs 32 bytes side by side, so neither needs an
// exchange.
//
// Angles: a position times a frequency is taken modulo one turn in 64-bit
// integers (the frequency in turns times 2^64, from a product of two fp64
// parts), so that far positions keep every bit: the angle's error is 1e-7, the
// half turn's rounding to fp32, up to position 2^31 and frequency 1, where fp32
// products would be off by whole turns.
#pragma once

#include "common.cuh"
#include "f32x2.cuh"
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

using f32x2::P;

// A lane's NP pairs of a head, firsts and seconds as packed fp32 pairs.
template <typename T, int NP, bool VEC>
struct Pairs {
    P a[NP / 2], b[NP / 2];
    static CUBF_DEV int pair(const Layout& l, int lane, int i) { return VEC ? lane * NP + i : lane + l.lanes * i; }

    CUBF_DEV void load(const T* p, const Layout& l, int lane) {
        float x[NP], y[NP];
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
            static_assert(N == NP, "a vector of either half");
            Vec16<T> u{}, w{};
            const int first = lane * NP;
            if (first < l.pairs) {
                u = *reinterpret_cast<const Vec16<T>*>(p + l.a(first));
                w = *reinterpret_cast<const Vec16<T>*>(p + (l.interleaved ? 2 * first + N : l.b(first)));
            }
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const Vec16<T>& v = i < NP / 2 ? u : w;
                x[i] = Convert<T, float>::load(l.interleaved ? v.v[2 * i % N] : u.v[i]);
                y[i] = Convert<T, float>::load(l.interleaved ? v.v[2 * i % N + 1] : w.v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int q = pair(l, lane, i);
                x[i] = q < l.pairs ? Convert<T, float>::load(p[l.a(q)]) : 0.f;
                y[i] = q < l.pairs && l.b(q) < l.dim ? Convert<T, float>::load(p[l.b(q)]) : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < NP / 2; ++i) {
            a[i] = f32x2::pk(x[2 * i], x[2 * i + 1]);
            b[i] = f32x2::pk(y[2 * i], y[2 * i + 1]);
        }
    }
    CUBF_DEV void store(T* p, const Layout& l, int lane) const {
        float x[NP], y[NP];
#pragma unroll
        for (int i = 0; i < NP / 2; ++i) {
            f32x2::up(a[i], x[2 * i], x[2 * i + 1]);
            f32x2::up(b[i], y[2 * i], y[2 * i + 1]);
        }
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
            const int first = lane * NP;
            if (first >= l.pairs) return;
            Vec16<T> u, w;
            if (l.interleaved) {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    Vec16<T>& v = i < NP / 2 ? u : w;
                    v.v[2 * i % N] = Convert<T, float>::store(x[i]);
                    v.v[2 * i % N + 1] = Convert<T, float>::store(y[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    u.v[i] = Convert<T, float>::store(x[i]);
                    w.v[i] = Convert<T, float>::store(y[i]);
                }
            }
            *reinterpret_cast<Vec16<T>*>(p + l.a(first)) = u;
            *reinterpret_cast<Vec16<T>*>(p + (l.interleaved ? 2 * first + N : l.b(first))) = w;
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int q = pair(l, lane, i);
                if (q < l.pairs) {
                    p[l.a(q)] = Convert<T, float>::store(x[i]);
                    if (l.b(q) < l.dim) p[l.b(q)] = Convert<T, float>::store(y[i]);
                }
            }
        }
    }
    // A table's values for the lane's pairs: `t` holds one a pair.
    static CUBF_DEV void table(const float* t, const Layout& l, int lane, P (&v)[NP / 2]) {
        if constexpr (VEC) {
            const float4* q = reinterpret_cast<const float4*>(t + min(lane * NP, kMaxPairs - NP));
#pragma unroll
            for (int i = 0; i < NP / 4; ++i) {
                const float4 x = q[i];
                v[2 * i] = f32x2::pk(x.x, x.y), v[2 * i + 1] = f32x2::pk(x.z, x.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP / 2; ++i)
                v[i] = f32x2::pk(t[min(pair(l, lane, 2 * i), kMaxPairs - 1)], t[min(pair(l, lane, 2 * i + 1), kMaxPairs - 1)]);
        }
    }
    // (a, b) -> (a c - b s, b c + a s); s negated turns back
    CUBF_DEV void turn(const P (&c)[NP / 2], const P (&s)[NP / 2]) {
#pragma unroll
        for (int i = 0; i < NP / 2; ++i) {
            const P x = a[i], y = b[i], minus = f32x2::mul2(s[i], f32x2::pk(-1.f, -1.f));
            a[i] = f32x2::fma2(x, c[i], f32x2::mul2(y, minus));
            b[i] = f32x2::fma2(y, c[i], f32x2::mul2(x, s[i]));
        }
    }
    // Sum of x a + y b over the lane's pairs.
    CUBF_DEV float dot(const P (&x)[NP / 2], const P (&y)[NP / 2]) const {
        P sum = f32x2::mul2(x[0], a[0]);
#pragma unroll
        for (int i = 0; i < NP / 2; ++i) {
            if (i) sum = f32x2::fma2(x[i], a[i], sum);
            sum = f32x2::fma2(y[i], b[i], sum);
        }
        float lo, hi;
        f32x2::up(sum, lo, hi);
        return lo + hi;
    }
    CUBF_DEV void scale(P f) {
#pragma unroll
        for (int i = 0; i < NP / 2; ++i) a[i] = f32x2::mul2(a[i], f), b[i] = f32x2::mul2(b[i], f);
    }
};

struct Shared {
    alignas(16) float weight[2][2][kMaxPairs];      // q's and k's, of the pairs' first and second values
    alignas(16) float turned[kWarps][2][kMaxPairs]; // cosines and sines of a warp's token
    unsigned long long turns[kMaxPairs];            // frequency / 2 pi, of a turn times 2^64
    int axis[kMaxPairs];
};

// Weights and frequencies in the order of the pairs.
template <typename T, bool WEIGHTED, bool TURNED>
CUBF_DEV void prepare(const QkNormArgs& a, const Layout& l, Shared& sm) {
    if (!WEIGHTED && !TURNED) return;
    for (int p = threadIdx.x; p < kMaxPairs; p += 32 * kWarps) {
        if (WEIGHTED) {
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
        }
        if (TURNED) {
            const bool turned = p < l.half;
            // 1 / 2 pi in two parts: rounded to one, times 2^31 positions, it alone would turn by 2e-7, the product as much
            constexpr double part = 0.15915494309189535, rest = -9.839338337591243e-18, turn = 18446744073709551616.0;
            const double frequency = turned ? static_cast<double>(a.frequencies[p]) : 0.0;
            double x = frequency * part;
            const double low = fma(frequency, part, -x) + frequency * rest;
            x -= rint(x);                           // whole turns a position drop out; exact, as less floor(x) is not below zero
            sm.turns[p] = static_cast<unsigned long long>(llrint(x * turn)) + static_cast<unsigned long long>(llrint(low * turn));
            sm.axis[p] = turned && a.axes ? min(max(a.axes[p], 0), a.axis_count - 1) : 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {      // what stays as it is beyond the rotated pairs
                sm.turned[w][0][p] = 1.f;
                sm.turned[w][1][p] = 0.f;
            }
        }
    }
    __syncthreads();
}

// Cosines and sines of a token's pairs, a lane each, into the warp's table.
CUBF_DEV void angles(const QkNormArgs& a, const Layout& l, Shared& sm, size_t token, int warp, int lane) {
    const size_t at = token < a.positions_period ? token : token % a.positions_period;
    __syncwarp();
    for (int p = lane; p < l.half; p += 32) {
        const size_t place = sm.axis[p] * a.positions_axis + at;
        const long long position = a.positions64 ? static_cast<const long long*>(a.positions)[place]
                                                 : static_cast<const int*>(a.positions)[place];
        const unsigned long long phase = static_cast<unsigned long long>(position) * sm.turns[p];
        // -1 .. 1: half turns
        const float x = static_cast<float>(static_cast<int>(phase >> 32)) * 4.656612873077393e-10f;
        sincospif(x, &sm.turned[warp][1][p], &sm.turned[warp][0][p]);
    }
    __syncwarp();
}

CUBF_DEV float group_sum(float v, int lanes) {
    for (int d = lanes / 2; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// `unit_heads` heads of a token a warp.
template <typename T, int NP, bool VEC, bool WEIGHTED, bool TURNED>
__global__ void __launch_bounds__(32 * kWarps, 4) qk_norm_kernel(QkNormArgs a, int unit_heads, int units_per_token) {
    __shared__ Shared sm;
    pdl_begin();
    using Head = Pairs<T, NP, VEC>;
    const Layout l = layout_of(a, NP);
    prepare<T, WEIGHTED, TURNED>(a, l, sm);
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int in_group = lane & (l.lanes - 1), group = lane / l.lanes, groups = 32 / l.lanes;
    const int all_heads = a.q_heads + a.k_heads;
    const float share = a.length ? 1.f : 1.f / static_cast<float>(a.dim);
    const size_t units = a.batch * a.tokens * units_per_token;
    for (size_t unit = static_cast<size_t>(blockIdx.x) * kWarps + warp; unit < units;
         unit += static_cast<size_t>(gridDim.x) * kWarps) {
        const size_t token = units_per_token == 1 ? unit : unit / units_per_token;
        const int first = units_per_token == 1 ? 0 : static_cast<int>(unit % units_per_token) * unit_heads;
        const int last = min(first + unit_heads, all_heads);
        const size_t row = a.batch == 1 ? 0 : token / a.tokens, in_row = token - row * a.tokens;
        const T* const q = static_cast<const T*>(a.q.p) + row * a.q.batch + in_row * a.q.token;
        const T* const k = static_cast<const T*>(a.k.p) + row * a.k.batch + in_row * a.k.token;
        T* const q_out = static_cast<T*>(a.q_out) + token * a.q_heads * a.dim;
        T* const k_out = static_cast<T*>(a.k_out) + token * a.k_heads * a.dim;
        if (TURNED) angles(a, l, sm, token, warp, lane);
        for (int base = first; base < last; base += groups) {
            const int head = min(base + group, last - 1);
            const bool key = head >= a.q_heads;
            Head x;
            x.load(key ? k + static_cast<size_t>(head - a.q_heads) * a.k.head : q + static_cast<size_t>(head) * a.q.head, l,
                   in_group);
            const float r = 1.f / sqrtf(fmaf(group_sum(x.dot(x.a, x.b), l.lanes), share, a.eps));
            if (WEIGHTED) {
                P w[NP / 2];
                Head::table(sm.weight[key][0], l, in_group, w);
#pragma unroll
                for (int i = 0; i < NP / 2; ++i) x.a[i] = f32x2::mul2(x.a[i], w[i]);
                Head::table(sm.weight[key][1], l, in_group, w);
#pragma unroll
                for (int i = 0; i < NP / 2; ++i) x.b[i] = f32x2::mul2(x.b[i], w[i]);
            }
            x.scale(f32x2::pk(r, r));
            if (TURNED) {
                P c[NP / 2], s[NP / 2];
                Head::table(sm.turned[warp][0], l, in_group, c);
                Head::table(sm.turned[warp][1], l, in_group, s);
                x.turn(c, s);
            }
            if (base + group < last)
                x.store(key ? k_out + static_cast<size_t>(head - a.q_heads) * a.dim : q_out + static_cast<size_t>(head) * a.dim, l,
                        in_group);
        }
    }
}

// The same walk; each CTA leaves its sums of the weights' gradients in `partials`.
template <typename T, int NP, bool VEC, bool WEIGHTED, bool TURNED>
__global__ void __launch_bounds__(32 * kWarps, WEIGHTED ? 2 : 4) qk_norm_backward_kernel(QkNormArgs a) {
    __shared__ Shared sm;
    pdl_begin();
    using Head = Pairs<T, NP, VEC>;
    const Layout l = layout_of(a, NP);
    prepare<T, WEIGHTED, TURNED>(a, l, sm);
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int in_group = lane & (l.lanes - 1), group = lane / l.lanes, groups = 32 / l.lanes;
    const float share = a.length ? 1.f : 1.f / static_cast<float>(a.dim);
    const size_t tokens = a.batch * a.tokens;
    P wa[2][NP / 2], wb[2][NP / 2];
    if (WEIGHTED) {
#pragma unroll
        for (int key = 0; key < 2; ++key)
#pragma unroll
            for (int i = 0; i < NP / 2; ++i) wa[key][i] = wb[key][i] = f32x2::pk(0.f, 0.f);
    }
    for (size_t token = static_cast<size_t>(blockIdx.x) * kWarps + warp; token < tokens;
         token += static_cast<size_t>(gridDim.x) * kWarps) {
        const size_t row = a.batch == 1 ? 0 : token / a.tokens, in_row = token - row * a.tokens;
        if (TURNED) angles(a, l, sm, token, warp, lane);
#pragma unroll
        for (int key = 0; key < 2; ++key) {
            const int heads = key ? a.k_heads : a.q_heads;
            const HeadTensor &t = key ? a.k : a.q, &d = key ? a.d_k_out : a.d_q_out;
            const T* const xs = static_cast<const T*>(t.p) + row * t.batch + in_row * t.token;
            const T* const ds = static_cast<const T*>(d.p) + row * d.batch + in_row * d.token;
            T* const out = static_cast<T*>(key ? a.d_k : a.d_q) + token * heads * a.dim;
            for (int base = 0; base < heads; base += groups) {
                const int head = min(base + group, heads - 1);
                const bool own = base + group < heads;
                Head x, g;
                x.load(xs + static_cast<size_t>(head) * t.head, l, in_group);
                g.load(ds + static_cast<size_t>(head) * d.head, l, in_group);
                if (TURNED) {
                    P c[NP / 2], s[NP / 2];
                    Head::table(sm.turned[warp][0], l, in_group, c);
                    Head::table(sm.turned[warp][1], l, in_group, s);
#pragma unroll
                    for (int i = 0; i < NP / 2; ++i) s[i] = f32x2::mul2(s[i], f32x2::pk(-1.f, -1.f));
                    g.turn(c, s);
                }
                const float r = 1.f / sqrtf(fmaf(group_sum(x.dot(x.a, x.b), l.lanes), share, a.eps));
                x.scale(f32x2::pk(r, r));        // n
                if (WEIGHTED) {
                    P w[NP / 2];
                    Head::table(sm.weight[key][0], l, in_group, w);
#pragma unroll
                    for (int i = 0; i < NP / 2; ++i) {
                        if (own) wa[key][i] = f32x2::fma2(g.a[i], x.a[i], wa[key][i]);
                        g.a[i] = f32x2::mul2(g.a[i], w[i]);
                    }
                    Head::table(sm.weight[key][1], l, in_group, w);
#pragma unroll
                    for (int i = 0; i < NP / 2; ++i) {
                        if (own) wb[key][i] = f32x2::fma2(g.b[i], x.b[i], wb[key][i]);
                        g.b[i] = f32x2::mul2(g.b[i], w[i]);
                    }
                }
                const float along = -group_sum(g.dot(x.a, x.b), l.lanes) * share;
                const P m2 = f32x2::pk(along, along);
#pragma unroll
                for (int i = 0; i < NP / 2; ++i) {
                    g.a[i] = f32x2::fma2(x.a[i], m2, g.a[i]);
                    g.b[i] = f32x2::fma2(x.b[i], m2, g.b[i]);
                }
                g.scale(f32x2::pk(r, r));
                if (own) g.store(out + static_cast<size_t>(head) * a.dim, l, in_group);
            }
        }
    }
    if constexpr (WEIGHTED) {
        // lane groups, then warps
        __shared__ float sums[kWarps][2][2][kMaxPairs];
#pragma unroll
        for (int key = 0; key < 2; ++key)
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                float x[2], y[2];
                f32x2::up(wa[key][i / 2], x[0], x[1]);
                f32x2::up(wb[key][i / 2], y[0], y[1]);
                float u = x[i % 2], v = y[i % 2];
                for (int d = l.lanes; d < 32; d *= 2) {
                    u += __shfl_xor_sync(0xffffffffu, u, d);
                    v += __shfl_xor_sync(0xffffffffu, v, d);
                }
                const int p = Head::pair(l, in_group, i);
                if (group == 0 && p < l.pairs) {
                    sums[warp][key][0][p] = u;
                    sums[warp][key][1][p] = v;
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
}

// Sums of the CTAs' parts: a warp for 32 channels, its CTA's warps taking turns with the parts.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) qk_norm_weights_kernel(QkNormArgs a) {
    __shared__ float sums[kWarps][32];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int at = blockIdx.x * 32 + lane;       // of both weights side by side
    float v = 0.f;
    if (at < 2 * a.dim) {
#pragma unroll 8
        for (int part = warp; part < a.parts; part += kWarps) v += a.partials[static_cast<size_t>(part) * 2 * a.dim + at];
    }
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
