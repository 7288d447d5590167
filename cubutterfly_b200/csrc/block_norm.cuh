// block_norm.cuh -- the boundary between two blocks of a language model: the
// block's output is RMS-normed, gated and added to the scaled residual
// stream, and the sum is RMS-normed and Hadamard-rotated for the next block.
//
//   n = y r(y) w_post,  r(v) = 1/sqrt(mean(v^2) + eps)
//   s = alpha x + act(gate) n
//   u = s r(s) w_pre,   u <- u H_D / sqrt(D) where the next block is rotated
//
// Rows are independent.  TPR threads hold a row in registers (EPT values
// each), so x and y are read once and s and u written once; the two row sums
// go through warp shuffles and, in rows of several warps, shared memory.  A
// CTA walks over rows and loads the next one while it works on this one.
#pragma once

#include "block_ops.hpp"
#include "common.cuh"

namespace cubf::norm {

// ---- memory access: VW consecutive values -----------------------------------------------------
// Values of a row as loaded, kept packed until they are used.
template <typename T, int VW>
struct Piece {
    static constexpr int kWords = VW * static_cast<int>(sizeof(T)) / 4 > 0 ? VW * static_cast<int>(sizeof(T)) / 4 : 1;
    uint32_t w[kWords];

    CUBF_DEV void clear() {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = 0;
    }
    CUBF_DEV void load(const T* p) {
        if constexpr (VW == 1 && sizeof(T) == 2) {
            w[0] = __ldcs(reinterpret_cast<const unsigned short*>(p));
        } else if constexpr (VW == 1) {
            w[0] = __ldcs(reinterpret_cast<const unsigned int*>(p));
        } else {
#pragma unroll
            for (int k = 0; k < kWords / 4; ++k) {
                const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p) + k);
                w[4 * k] = q.x;
                w[4 * k + 1] = q.y;
                w[4 * k + 2] = q.z;
                w[4 * k + 3] = q.w;
            }
        }
    }
    CUBF_DEV float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            const unsigned short h = static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)));
            T v;
            memcpy(&v, &h, 2);
            return Convert<T, float>::load(v);
        }
    }
};

template <typename T, int VW>
CUBF_DEV void store_values(T* p, const float (&v)[VW]) {
    if constexpr (VW == 1) {
        p[0] = Convert<T, float>::store(v[0]);
    } else {
        constexpr int kVec = 16 / sizeof(T);
        static_assert(VW % kVec == 0, "whole 16-byte vectors");
#pragma unroll
        for (int k = 0; k < VW / kVec; ++k) {
            Vec16<T> q;
#pragma unroll
            for (int e = 0; e < kVec; ++e) q.v[e] = Convert<T, float>::store(v[k * kVec + e]);
            stg_stream(reinterpret_cast<Vec16<T>*>(p) + k, q);
        }
    }
}

// VW consecutive values of a per-channel vector (in T, or in fp32), through L1.
template <typename T, int VW>
CUBF_DEV void load_vector(const void* base, bool is32, size_t idx, float (&v)[VW]) {
    if (is32) {
        const float* p = static_cast<const float*>(base) + idx;
        if constexpr (VW == 1) {
            v[0] = __ldg(p);
        } else {
#pragma unroll
            for (int k = 0; k < VW / 4; ++k) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(p) + k);
                v[4 * k] = q.x;
                v[4 * k + 1] = q.y;
                v[4 * k + 2] = q.z;
                v[4 * k + 3] = q.w;
            }
        }
    } else if constexpr (sizeof(T) == 2) {
        const T* p = static_cast<const T*>(base) + idx;
        if constexpr (VW == 1) {
            v[0] = Convert<T, float>::load(p[0]);
        } else {
#pragma unroll
            for (int k = 0; k < VW / 8; ++k) {
                Vec16<T> q;
                *reinterpret_cast<uint4*>(&q) = __ldg(reinterpret_cast<const uint4*>(p) + k);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * k + e] = Convert<T, float>::load(q.v[e]);
            }
        }
    }
}

CUBF_DEV float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// act(g), and its slope where SLOPE
template <bool SLOPE>
CUBF_DEV float activation(int act, float g) {
    if (act == 0) return SLOPE ? 1.f : g;
    const float s = sigmoid(g);
    if (act == 1) return SLOPE ? s * (1.f - s) : s;
    return SLOPE ? s * (1.f + g * (1.f - s)) : g * s;
}

// ---- a row over TPR threads -------------------------------------------------------------------
// Thread j holds chunks c = 0 .. C - 1 of VW consecutive values: value (c, e)
// is element (c TPR + j) VW + e of the row.
template <int TPR_, int EPT_, int VW_>
struct Shape {
    static constexpr int TPR = TPR_, EPT = EPT_, VW = VW_, C = EPT / VW;
    static constexpr int kThreads = TPR == 32 ? 128 : TPR;
    static constexpr int kRows = kThreads / TPR;    // rows a CTA works on at a time
    static constexpr int kWarps = TPR / 32 > 0 ? TPR / 32 : 1;
    static_assert(C * VW == EPT && TPR >= 32, "whole chunks over whole warps");
};

// Sum over the row's threads, the same in each.  Rows of several warps are
// alone in their CTA; `slot` (0, 1, ...) names the shared words used, so that
// sums in turn need one barrier each.
template <typename S>
CUBF_DEV float row_sum(float v, float* shared, int slot) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (S::kWarps > 1) {
        float* words = shared + slot * S::kWarps;
        if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int k = 0; k < S::kWarps; ++k) v += words[k];
    }
    return v;
}

constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// ---- Hadamard rotation of a row ---------------------------------------------------------------
// The row's index bits are held either by a thread's registers or by the
// thread number.  Butterflies run over the register bits; then the row is
// written to shared memory and read back with other bits in registers, until
// every bit has had its turn, and at the end back in the layout of the loads.
// Words are swizzled (the 16-byte group index is XORed with the index bits
// above it), and the thread bits are ordered so that the 32 lanes fall into
// different banks.
struct Layout {
    uint32_t regs;      // index bits held in registers, ascending
    int order[16];      // index bit of each thread bit
};
template <int LOGD, int LOGE>
constexpr Layout make_layout(uint32_t regs, bool vector) {
    Layout l{};
    l.regs = regs;
    bool used[16] = {};
    int n = 0;
    if (!vector) {
        // one thread bit for each bank bit: bits 0 .. 4 themselves, above them bit p falls on 2 + (p - 5) mod 3
        for (int bank = 0; bank < 5; ++bank)
            for (int p = 0; p < LOGD; ++p) {
                const int on = p < 5 ? p : 2 + (p - 5) % 3;
                if (on == bank && !((regs >> p) & 1u) && !used[p]) {
                    used[p] = true;
                    l.order[n++] = p;
                    break;
                }
            }
    }
    for (int p = 0; p < LOGD; ++p)
        if (!((regs >> p) & 1u) && !used[p]) l.order[n++] = p;
    return l;
}
// Index bits in registers in pass `k`: pass 0 is the layout of the loads (the
// low VB bits and the top bits); each later pass takes the next LOGE of the
// others, filled up with bits already done.
template <int LOGD, int LOGE, int VB>
constexpr uint32_t pass_bits(int k) {
    const uint32_t all = lowmask(LOGD);
    const uint32_t low = lowmask(VB), top = lowmask(LOGE - VB) << (LOGD - (LOGE - VB));
    if (k == 0) return low | top;
    const int tb = LOGD - LOGE;
    uint32_t m = 0;
    int first = (k - 1) * LOGE, count = tb - first < LOGE ? tb - first : LOGE;
    for (int i = 0; i < count; ++i) m |= 1u << (VB + first + i);
    for (int p = LOGD - 1; p >= 0 && popc32(m) < LOGE; --p)
        if (!((m >> p) & 1u)) m |= 1u << p;
    return m & all;
}
// Bits pass k transforms (those not done before it).
template <int LOGD, int LOGE, int VB>
constexpr uint32_t pass_work(int k) {
    uint32_t done = 0;
    for (int i = 0; i < k; ++i) done |= pass_bits<LOGD, LOGE, VB>(i);
    return pass_bits<LOGD, LOGE, VB>(k) & ~done;
}
CUBF_DEV uint32_t swizzle(uint32_t w) { return w ^ ((((w >> 5) ^ (w >> 8) ^ (w >> 11)) & 7u) << 2); }

template <int E, uint32_t REGS, uint32_t WORK>
CUBF_DEV void butterflies(float (&v)[E]) {
    int bit = 0;
#pragma unroll
    for (int p = 0; p < 16; ++p) {
        if (!((REGS >> p) & 1u)) continue;
        if ((WORK >> p) & 1u) {
#pragma unroll
            for (int r = 0; r < E; ++r)
                if (!(r & (1 << bit))) {
                    const float a = v[r], b = v[r | (1 << bit)];
                    v[r] = a + b;
                    v[r | (1 << bit)] = a - b;
                }
        }
        ++bit;
    }
}

template <int LOGD, int LOGE, int VB, int K, bool WRITE>
CUBF_DEV void move_row(float (&v)[1 << LOGE], float* row, int j) {
    constexpr int E = 1 << LOGE;
    constexpr uint32_t regs = pass_bits<LOGD, LOGE, VB>(K);
    constexpr Layout l = make_layout<LOGD, LOGE>(regs, K == 0);
    constexpr Offsets<E> at = make_offsets<E>(regs);
    uint32_t base = 0;
#pragma unroll
    for (int k = 0; k < LOGD - LOGE; ++k) base |= ((static_cast<uint32_t>(j) >> k) & 1u) << l.order[k];
    // the swizzle is linear over XOR, and base and at[] share no bits
    const uint32_t sb = swizzle(base);
    if constexpr (K == 0 && VB >= 2) {
#pragma unroll
        for (int r = 0; r < E; r += 4) {
            float4* q = reinterpret_cast<float4*>(row + (sb ^ swizzle(at.v[r])));
            if (WRITE) {
                *q = make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
            } else {
                const float4 f = *q;
                v[r] = f.x;
                v[r + 1] = f.y;
                v[r + 2] = f.z;
                v[r + 3] = f.w;
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < E; ++r) {
            float* q = row + (sb ^ swizzle(at.v[r]));
            if (WRITE)
                *q = v[r];
            else
                v[r] = *q;
        }
    }
}

template <int TPR>
CUBF_DEV void row_barrier() {
    if constexpr (TPR > 32)
        __syncthreads();
    else
        __syncwarp();
}

template <int LOGD, int LOGE, int VB, int TPR, int K>
CUBF_DEV void rotate_passes(float (&v)[1 << LOGE], float* row, int j) {
    constexpr int kPasses = 1 + (LOGD - LOGE + LOGE - 1) / LOGE;
    butterflies<(1 << LOGE), pass_bits<LOGD, LOGE, VB>(K), pass_work<LOGD, LOGE, VB>(K)>(v);
    if constexpr (kPasses > 1) {
        constexpr int next = K + 1 < kPasses ? K + 1 : 0;
        if constexpr (K > 0) row_barrier<TPR>();  // everyone has read the pass before
        move_row<LOGD, LOGE, VB, K, true>(v, row, j);
        row_barrier<TPR>();
        move_row<LOGD, LOGE, VB, next, false>(v, row, j);
        if constexpr (next > 0) rotate_passes<LOGD, LOGE, VB, TPR, next>(v, row, j);
    }
}

// v <- v H_D (unscaled); D = TPR EPT.  `row` holds D floats.
template <typename S>
CUBF_DEV void rotate_row(float (&v)[S::EPT], float* row, int j) {
    constexpr int loge = log2_of(S::EPT), logd = log2_of(S::TPR * S::EPT);
    rotate_passes<logd, loge, log2_of(S::VW), S::TPR, 0>(v, row, j);
    row_barrier<S::TPR>();  // the next row may write
}

// ---- forward ----------------------------------------------------------------------------------
template <typename T, typename R, typename S, bool ROTATE>
struct Forward {
    static constexpr int C = S::C, VW = S::VW;

    struct Row {
        Piece<R, VW> x[C];
        Piece<T, VW> y[C], g[C];
    };

    static CUBF_DEV void load(const BlockNormArgs& p, size_t row, int j, Row& in) {
        const R* x = static_cast<const R*>(p.x) + row * p.x_row;
        const T* y = static_cast<const T*>(p.y) + row * p.y_row;
        const T* g = static_cast<const T*>(p.gate) + row * p.gate_row;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * S::TPR + j) * VW;
            in.x[c].clear();
            in.y[c].clear();
            in.g[c].clear();
            if (at < p.dim) {
                in.x[c].load(x + at);
                if (p.y) in.y[c].load(y + at);
                if (p.gate_mode == kGateFull) in.g[c].load(g + at);
            }
        }
    }

    static CUBF_DEV void run(const BlockNormArgs& p, float* shared) {
        const int j = threadIdx.x % S::TPR, sub = threadIdx.x / S::TPR;
        float* words = shared + (ROTATE ? S::kRows * S::TPR * S::EPT : 0);
        float* row_words = shared + sub * S::TPR * S::EPT;
        const size_t stride = static_cast<size_t>(gridDim.x) * S::kRows;
        size_t row = static_cast<size_t>(blockIdx.x) * S::kRows + sub;
        const float inv_dim = 1.f / static_cast<float>(p.dim);
        Row in;
        if (row < p.rows) load(p, row, j, in);
        int slot = 0;
        for (; row < p.rows; row += stride) {
            float s[S::EPT];
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    const float y = in.y[c].get(e);
                    s[c * VW + e] = y;
                    sum = fmaf(y, y, sum);
                }
            const Row now = in;
            if (row + stride < p.rows) load(p, row + stride, j, in);
            float ry = 1.f;
            if (p.post_norm) {
                ry = rsqrtf(row_sum<S>(sum, words, slot) * inv_dim + p.eps);
                if (p.r_post && j == 0) p.r_post[row] = ry;
            }
            slot ^= 1;
            sum = 0.f;
            const size_t gate_row = p.gate_mode == kGateGroups ? row / p.rows_per_gate * p.gate_row : 0;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = (c * S::TPR + j) * VW;
                const bool in_row = at < p.dim;
                float w[VW], a[VW];
#pragma unroll
                for (int e = 0; e < VW; ++e) w[e] = ry;
                if (p.post && in_row) {
                    load_vector<T, VW>(p.post, p.post32, at, w);
#pragma unroll
                    for (int e = 0; e < VW; ++e) w[e] *= ry;
                }
                if (p.gate_mode == kGateFull) {
#pragma unroll
                    for (int e = 0; e < VW; ++e) w[e] *= activation<false>(p.act, now.g[c].get(e));
                } else if (p.gate_mode != kGateNone && in_row) {
                    load_vector<T, VW>(p.gate, p.gate32, gate_row + at, a);
#pragma unroll
                    for (int e = 0; e < VW; ++e) w[e] *= activation<false>(p.act, a[e]);
                }
#pragma unroll
                for (int e = 0; e < VW; ++e) a[e] = p.scale;
                if (p.scales && in_row) load_vector<T, VW>(p.scales, p.scales32, at, a);
                float out[VW];
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    const float x = a[e] * now.x[c].get(e);
                    const float v = p.y ? fmaf(w[e], s[c * VW + e], x) : x;
                    out[e] = v;
                    s[c * VW + e] = v;
                    sum = fmaf(v, v, sum);
                }
                if (p.residual && in_row) store_values<R, VW>(static_cast<R*>(p.residual) + row * p.dim + at, out);
            }
            if (p.normed) {
                const float rs = rsqrtf(row_sum<S>(sum, words, 2 + slot) * inv_dim + p.eps);
                if (p.r_pre && j == 0) p.r_pre[row] = rs;
                const float scale = ROTATE ? rs * p.rotate_scale : rs;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int at = (c * S::TPR + j) * VW;
                    float w[VW];
#pragma unroll
                    for (int e = 0; e < VW; ++e) w[e] = 1.f;
                    if (p.pre && at < p.dim) load_vector<T, VW>(p.pre, p.pre32, at, w);
#pragma unroll
                    for (int e = 0; e < VW; ++e) s[c * VW + e] *= scale * w[e];
                }
                if constexpr (ROTATE) rotate_row<S>(s, row_words, j);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int at = (c * S::TPR + j) * VW;
                    float out[VW];
#pragma unroll
                    for (int e = 0; e < VW; ++e) out[e] = s[c * VW + e];
                    if (at < p.dim) store_values<T, VW>(static_cast<T*>(p.normed) + row * p.dim + at, out);
                }
            }
        }
    }
};

template <typename T, typename R, typename S, bool ROTATE>
__global__ void __launch_bounds__(S::kThreads, 1) block_norm_kernel(BlockNormArgs p) {
    extern __shared__ __align__(16) float shared[];
    pdl_begin();
    Forward<T, R, S, ROTATE>::run(p, shared);
}

// ---- backward ---------------------------------------------------------------------------------
// With yn = y r(y), sn = s r(s), t = du w_pre (du rotated back first) and
// dS = ds + r(s) (t - sn mean(t sn)):
//   dx = alpha dS                dw_pre   = sum du sn        (Q)
//   dn = act(gate) dS            dalpha   = sum dS x         (Z)
//   t' = dn w_post               dy = r(y) (t' - yn mean(t' yn))
//   dgate = act'(gate) dS n      dw_post  = sum dn yn
// The sums over rows stay in registers: a thread owns its columns for every
// row of its CTA, whose rows share one gate row, so that for a gate per
// channel or per group dw_post and dgate both follow from P = sum dS yn; with
// a gate per row P = sum dn yn.  Each CTA writes its sums once and a second
// kernel adds them in a fixed order.
template <typename T, typename R, typename S, bool ROTATE>
struct Backward {
    static constexpr int C = S::C, VW = S::VW;

    // t - vn mean(t vn), the part of t that a norm lets through.  In a row of
    // one value vn^2 = 1 - eps r^2, and the difference would cancel.
    static CUBF_DEV float through_norm(const BlockNormArgs& p, float t, float vn, float mean, float r) {
        return p.dim == 1 ? t * p.eps * r * r : t - vn * mean;
    }

    struct Row {
        Piece<R, VW> x[C], ds[C];
        Piece<T, VW> y[C], g[C], du[C];
        float ry, rs;
    };

    static CUBF_DEV void load(const BlockNormArgs& p, size_t row, int j, Row& in) {
        const R* x = static_cast<const R*>(p.x) + row * p.x_row;
        const R* ds = static_cast<const R*>(p.d_residual) + row * p.d_residual_row;
        const T* y = static_cast<const T*>(p.y) + row * p.y_row;
        const T* du = static_cast<const T*>(p.d_normed) + row * p.d_normed_row;
        const T* g = static_cast<const T*>(p.gate) + row * p.gate_row;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (c * S::TPR + j) * VW;
            in.x[c].clear();
            in.y[c].clear();
            in.ds[c].clear();
            in.du[c].clear();
            in.g[c].clear();
            if (at < p.dim) {
                in.x[c].load(x + at);
                if (p.y) in.y[c].load(y + at);
                if (p.d_residual) in.ds[c].load(ds + at);
                if (p.d_normed) in.du[c].load(du + at);
                if (p.gate_mode == kGateFull) in.g[c].load(g + at);
            }
        }
        in.ry = p.post_norm ? p.r_post[row] : 1.f;
        in.rs = p.d_normed ? p.r_pre[row] : 0.f;
    }

    static CUBF_DEV void run(const BlockNormArgs& p, float* shared) {
        const int j = threadIdx.x % S::TPR, sub = threadIdx.x / S::TPR;
        float* words = shared + (ROTATE ? S::kRows * S::TPR * S::EPT : 0);
        float* row_words = shared + sub * S::TPR * S::EPT;
        const float inv_dim = 1.f / static_cast<float>(p.dim);
        // this CTA's rows: a share of one gate group's
        const size_t group = blockIdx.x / p.parts_per_group;
        const size_t share = (p.rows_per_gate + p.parts_per_group - 1) / p.parts_per_group;
        const size_t from = (blockIdx.x % p.parts_per_group) * share;
        const size_t to = from + share < p.rows_per_gate ? from + share : p.rows_per_gate;
        const size_t end = group * p.rows_per_gate + to;
        size_t row = group * p.rows_per_gate + from + sub;
        const size_t gate_row = p.gate_mode == kGateGroups ? group * p.gate_row : 0;
        float P[S::EPT], Q[S::EPT], Z[S::EPT];
#pragma unroll
        for (int k = 0; k < S::EPT; ++k) P[k] = Q[k] = Z[k] = 0.f;
        Row in;
        if (row < end) load(p, row, j, in);
        int slot = 0;
        for (; row < end; row += S::kRows) {
            const Row now = in;
            if (row + S::kRows < end) load(p, row + S::kRows, j, in);
            float d[S::EPT];   // du, then dS
            float n[S::EPT];   // act(gate) w_post, the factor of yn in s
            if (p.d_normed) {
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int e = 0; e < VW; ++e) d[c * VW + e] = now.du[c].get(e);
                if constexpr (ROTATE) {
                    rotate_row<S>(d, row_words, j);
#pragma unroll
                    for (int k = 0; k < S::EPT; ++k) d[k] *= p.rotate_scale;
                }
            } else {
#pragma unroll
                for (int k = 0; k < S::EPT; ++k) d[k] = 0.f;
            }
            float dot = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = (c * S::TPR + j) * VW;
                const bool in_row = at < p.dim;
                float w[VW], a[VW], al[VW];
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    w[e] = a[e] = 1.f;
                    al[e] = p.scale;
                }
                if (p.post && in_row) load_vector<T, VW>(p.post, p.post32, at, w);
                if (p.gate_mode == kGateFull) {
#pragma unroll
                    for (int e = 0; e < VW; ++e) a[e] = activation<false>(p.act, now.g[c].get(e));
                } else if (p.gate_mode != kGateNone && in_row) {
                    load_vector<T, VW>(p.gate, p.gate32, gate_row + at, a);
#pragma unroll
                    for (int e = 0; e < VW; ++e) a[e] = activation<false>(p.act, a[e]);
                }
                if (p.scales && in_row) load_vector<T, VW>(p.scales, p.scales32, at, al);
#pragma unroll
                for (int e = 0; e < VW; ++e) n[c * VW + e] = a[e];
                if (p.d_normed) {
                    float wp[VW];
#pragma unroll
                    for (int e = 0; e < VW; ++e) wp[e] = 1.f;
                    if (p.pre && in_row) load_vector<T, VW>(p.pre, p.pre32, at, wp);
#pragma unroll
                    for (int e = 0; e < VW; ++e) {
                        const int k = c * VW + e;
                        float s = al[e] * now.x[c].get(e);
                        if (p.y) s = fmaf(a[e] * w[e], now.y[c].get(e) * now.ry, s);
                        const float sn = s * now.rs;
                        Q[k] = fmaf(d[k], sn, Q[k]);
                        d[k] *= wp[e];
                        dot = fmaf(d[k], sn, dot);
                    }
                }
            }
            if (p.d_normed) dot = row_sum<S>(dot, words, slot) * inv_dim;
            float dot2 = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = (c * S::TPR + j) * VW;
                const bool in_row = at < p.dim;
                float w[VW], al[VW], out[VW], dg[VW];
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    w[e] = 1.f;
                    al[e] = p.scale;
                }
                if (p.post && in_row) load_vector<T, VW>(p.post, p.post32, at, w);
                if (p.scales && in_row) load_vector<T, VW>(p.scales, p.scales32, at, al);
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    const int k = c * VW + e;
                    const float x = now.x[c].get(e), yn = now.y[c].get(e) * now.ry;
                    float dS = now.ds[c].get(e);
                    if (p.d_normed) {
                        float s = al[e] * x;
                        if (p.y) s = fmaf(n[k] * w[e], yn, s);
                        dS = fmaf(now.rs, through_norm(p, d[k], s * now.rs, dot, now.rs), dS);
                    }
                    out[e] = al[e] * dS;
                    if (p.scales) Z[k] = fmaf(dS, x, Z[k]);
                    const float dn = n[k] * dS;
                    P[k] = fmaf(p.gate_mode == kGateFull ? dn : dS, yn, P[k]);
                    if (p.gate_mode == kGateFull)
                        dg[e] = dS * yn * w[e] * activation<true>(p.act, now.g[c].get(e));
                    d[k] = dn * w[e];
                    dot2 = fmaf(d[k], yn, dot2);
                }
                if (in_row) {
                    store_values<R, VW>(static_cast<R*>(p.d_x) + row * p.dim + at, out);
                    if (p.gate_mode == kGateFull)
                        store_values<T, VW>(static_cast<T*>(p.d_gate) + row * p.dim + at, dg);
                }
            }
            if (p.y) {
                if (p.post_norm) dot2 = row_sum<S>(dot2, words, 2 + slot) * inv_dim;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int at = (c * S::TPR + j) * VW;
                    float out[VW];
#pragma unroll
                    for (int e = 0; e < VW; ++e) {
                        const float yn = now.y[c].get(e) * now.ry;
                        out[e] = p.post_norm ? now.ry * through_norm(p, d[c * VW + e], yn, dot2, now.ry) : d[c * VW + e];
                    }
                    if (at < p.dim) store_values<T, VW>(static_cast<T*>(p.d_y) + row * p.dim + at, out);
                }
            }
            slot ^= 1;
        }
        // the CTA's sums; rows side by side in a CTA are added first
        float* part = p.partials + static_cast<size_t>(blockIdx.x) * 3 * p.dim;
        auto write = [&](float (&v)[S::EPT], float* dst) {
            if constexpr (S::kRows > 1) {
                __syncthreads();
#pragma unroll
                for (int k = 0; k < S::EPT; ++k) shared[(sub * S::EPT + k) * S::TPR + j] = v[k];
                __syncthreads();
                if (sub > 0) return;
#pragma unroll
                for (int k = 0; k < S::EPT; ++k)
                    for (int o = 1; o < S::kRows; ++o) v[k] += shared[(o * S::EPT + k) * S::TPR + j];
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = (c * S::TPR + j) * VW;
                float out[VW];
#pragma unroll
                for (int e = 0; e < VW; ++e) out[e] = v[c * VW + e];
                if (at < p.dim) store_values<float, VW>(dst + at, out);
            }
        };
        if (p.need_p) write(P, part);
        if (p.need_q) write(Q, part + p.dim);
        if (p.need_z) write(Z, part + 2 * static_cast<size_t>(p.dim));
    }
};

template <typename T, typename R, typename S, bool ROTATE>
__global__ void __launch_bounds__(S::kThreads, 1) block_norm_backward_kernel(BlockNormArgs p) {
    extern __shared__ __align__(16) float shared[];
    pdl_begin();
    Backward<T, R, S, ROTATE>::run(p, shared);
}

// The gradients of the per-channel vectors from the CTAs' sums: 32 columns
// per CTA, 32 slices of the parts, added in a fixed order.  blockIdx.y: 0
// d_pre, 1 d_post, 2 d_scale, 3 + g the gate row of group g.
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_sums_kernel(BlockNormArgs p, int parts) {
    __shared__ float slice[32][33];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    const unsigned what = blockIdx.y;
    void* out = what == 0 ? p.d_pre : what == 1 ? p.d_post : what == 2 ? p.d_scale : p.d_gate;
    if (!out || (what > 2 && (p.gate_mode == kGateFull || p.gate_mode == kGateNone))) return;
    const float* src = p.partials + (what == 0 ? 1 : what == 2 ? 2 : 0) * static_cast<size_t>(p.dim) + col;
    const int first = what > 2 ? static_cast<int>(what - 3) * p.parts_per_group : 0;
    const int last = what > 2 ? first + p.parts_per_group : parts;
    auto vector_at = [&](const void* v, bool is32, size_t at) {
        float f[1];
        load_vector<T, 1>(v, is32 || sizeof(T) == 4, at, f);
        return f[0];
    };
    float sum = 0.f;
    if (col < p.dim)
        for (int k = first + warp; k < last; k += 32) {
            float v = src[static_cast<size_t>(k) * 3 * p.dim];
            if (what == 1 && (p.gate_mode == kGateChannel || p.gate_mode == kGateGroups)) {
                const size_t g = p.gate_mode == kGateGroups ? static_cast<size_t>(k / p.parts_per_group) * p.gate_row : 0;
                v *= activation<false>(p.act, vector_at(p.gate, p.gate32, g + col));
            }
            sum += v;
        }
    slice[warp][lane] = sum;
    __syncthreads();
    if (warp > 0 || col >= p.dim) return;
    sum = 0.f;
    for (int k = 0; k < 32; ++k) sum += slice[k][lane];
    size_t at = col;
    bool is32 = what == 0 ? p.pre32 : what == 1 ? p.post32 : what == 2 ? p.scales32 : p.gate32;
    if (what > 2) {
        const size_t g = p.gate_mode == kGateGroups ? static_cast<size_t>(what - 3) * p.gate_row : 0;
        if (p.post) sum *= vector_at(p.post, p.post32, col);
        sum *= activation<true>(p.act, vector_at(p.gate, p.gate32, g + col));
        at += static_cast<size_t>(what - 3) * p.dim;
    }
    if (is32 || sizeof(T) == 4)
        static_cast<float*>(out)[at] = sum;
    else
        static_cast<T*>(out)[at] = Convert<T, float>::store(sum);
}

}  // namespace cubf::norm
