// block_norm.cuh -- the boundary between two blocks of a language model: the
// block's output is RMS-normed, gated and added to the scaled residual
// stream, and the sum is RMS-normed and Hadamard-rotated for the next block.
//
//   n = y r(y) w_post,  r(v) = 1/sqrt(mean(v^2) + eps)
//   s = alpha x + act(gate) n
//   u = s r(s) w_pre,   u <- u H_D / sqrt(D) where the next block is rotated
//
// Rows are independent.  TPR threads hold a row in registers (EPT values
// each, as packed fp32 pairs), so x and y are read once and s and u written
// once; the two row sums go through warp shuffles and, in rows of several
// warps, shared memory.  A CTA walks over rows and loads the next one while it
// works on this one; what depends on the channel alone is formed once.
#pragma once

#include "block_ops.hpp"
#include "common.cuh"
#include "f32x2.cuh"

namespace cubf::norm {

using f32x2::add2;
using f32x2::fma2;
using f32x2::mul2;
using f32x2::sub2;
using Pair = f32x2::P;

CUBF_DEV Pair both(float v) { return f32x2::pk(v, v); }
CUBF_DEV float2 floats(Pair p) {
    float2 f;
    f32x2::up(p, f.x, f.y);
    return f;
}
CUBF_DEV float sum_of(Pair p) {
    const float2 f = floats(p);
    return f.x + f.y;
}

// ---- memory access ----------------------------------------------------------------------------
// Thread j of a row holds chunks c = 0 .. C - 1 of VW consecutive values:
// value (c, e) is element (c TPR + j) VW + e of the row, and register c VW + e.
template <int TPR_, int EPT_, int VW_, int THREADS_ = 0>
struct Shape {
    static constexpr int TPR = TPR_, EPT = EPT_, VW = VW_, C = EPT / VW, HALF = EPT / 2;
    static constexpr int kThreads = THREADS_ > 0 ? THREADS_ : TPR == 32 ? 128 : TPR;
    static constexpr int kRows = kThreads / TPR;    // rows a CTA works on at a time
    static constexpr int kWarps = TPR / 32;
    static_assert(C * VW == EPT && TPR >= 32 && EPT >= 2, "whole chunks over whole warps");
    static_assert(TPR == 32 || kRows <= 15, "a barrier for each row of several warps");
    static CUBF_DEV int at(int c, int j) { return (c * TPR + j) * VW; }
};

// A row as loaded: EPT values, packed.  Values past the end of the row are zero.
template <typename T, typename S>
struct Values {
    static constexpr int kWords = S::EPT * static_cast<int>(sizeof(T)) / 4;
    static constexpr int kPer = S::VW * static_cast<int>(sizeof(T)) / 4;  // words of a chunk (VW > 1)
    uint32_t w[kWords];

    CUBF_DEV void clear() {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = 0;
    }
    template <bool STREAM = true>
    CUBF_DEV void load(const T* row, int j, int dim) {
        if constexpr (S::VW == 1) {
            clear();
#pragma unroll
            for (int c = 0; c < S::EPT; ++c)
                if (S::at(c, j) < dim) {
                    if constexpr (sizeof(T) == 2) {
                        const uint32_t h = __ldcs(reinterpret_cast<const unsigned short*>(row + S::at(c, j)));
                        w[c / 2] |= h << (16 * (c & 1));
                    } else {
                        w[c] = __ldcs(reinterpret_cast<const unsigned int*>(row + S::at(c, j)));
                    }
                }
        } else {
#pragma unroll
            for (int c = 0; c < S::C; ++c) {
                const bool in = S::at(c, j) < dim;
                const uint4* p = reinterpret_cast<const uint4*>(row + S::at(c, j));
#pragma unroll
                for (int k = 0; k < kPer / 4; ++k) {
                    uint4 q = make_uint4(0, 0, 0, 0);
                    if (in) q = STREAM ? __ldcs(p + k) : __ldg(p + k);
                    w[c * kPer + 4 * k] = q.x;
                    w[c * kPer + 4 * k + 1] = q.y;
                    w[c * kPer + 4 * k + 2] = q.z;
                    w[c * kPer + 4 * k + 3] = q.w;
                }
            }
        }
    }
    // registers 2 k and 2 k + 1
    CUBF_DEV Pair pair(int k) const {
        if constexpr (sizeof(T) == 4) {
            return f32x2::pk(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
        } else if constexpr (std::is_same<T, __half>::value) {
            __half2 h;
            memcpy(&h, &w[k], 4);
            const float2 f = __half22float2(h);
            return f32x2::pk(f.x, f.y);
        } else {
            return f32x2::pk(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
        }
    }
};

template <typename T>
CUBF_DEV uint32_t packed(float lo, float hi) {
    uint32_t w;
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        memcpy(&w, &h, 4);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        memcpy(&w, &h, 4);
    }
    return w;
}

// writes the row held as pairs, each rounded once
template <typename S, typename T, typename Get>
CUBF_DEV void store_row(T* row, int j, int dim, Get&& pair) {
#pragma unroll
    for (int c = 0; c < S::C; ++c) {
        if constexpr (S::VW == 1) {
            const float2 f = floats(pair(c / 2));
            if (S::at(c, j) < dim) row[S::at(c, j)] = Convert<T, float>::store(c & 1 ? f.y : f.x);
        } else {
            uint32_t w[S::VW * static_cast<int>(sizeof(T)) / 4];
#pragma unroll
            for (int k = 0; k < S::VW / 2; ++k) {
                const float2 f = floats(pair(c * (S::VW / 2) + k));
                if constexpr (sizeof(T) == 4) {
                    w[2 * k] = __float_as_uint(f.x);
                    w[2 * k + 1] = __float_as_uint(f.y);
                } else {
                    w[k] = packed<T>(f.x, f.y);
                }
            }
            if (S::at(c, j) < dim) {
                uint4* p = reinterpret_cast<uint4*>(row + S::at(c, j));
#pragma unroll
                for (int k = 0; k < S::VW * static_cast<int>(sizeof(T)) / 16; ++k)
                    __stcs(p + k, make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]));
            }
        }
    }
}

// A per-channel vector, in T or in fp32, through L1; `fill` where it is null
// and past the end of the row.
template <typename T, typename S>
CUBF_DEV void load_vector(const void* base, bool is32, int j, int dim, float fill, Pair (&v)[S::HALF]) {
#pragma unroll
    for (int k = 0; k < S::HALF; ++k) v[k] = both(fill);
    if (!base) return;
    if constexpr (S::VW == 1) {
        float f[S::EPT];
#pragma unroll
        for (int c = 0; c < S::EPT; ++c) {
            f[c] = fill;
            if (S::at(c, j) < dim)
                f[c] = is32 || sizeof(T) == 4 ? __ldg(static_cast<const float*>(base) + S::at(c, j))
                                              : Convert<T, float>::load(static_cast<const T*>(base)[S::at(c, j)]);
        }
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) v[k] = f32x2::pk(f[2 * k], f[2 * k + 1]);
    } else if (is32 || sizeof(T) == 4) {
        Values<float, S> q;
        q.template load<false>(static_cast<const float*>(base), j, dim);
#pragma unroll
        for (int k = 0; k < S::HALF; ++k)
            if (S::at(2 * k / S::VW, j) < dim) v[k] = q.pair(k);
    } else {
        Values<T, S> q;
        q.template load<false>(static_cast<const T*>(base), j, dim);
#pragma unroll
        for (int k = 0; k < S::HALF; ++k)
            if (S::at(2 * k / S::VW, j) < dim) v[k] = q.pair(k);
    }
}

CUBF_DEV float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// act(g), or its slope where SLOPE
template <bool SLOPE>
CUBF_DEV float activation(int act, float g) {
    if (act == 0) return SLOPE ? 1.f : g;
    const float s = sigmoid(g);
    if (act == 1) return SLOPE ? s * (1.f - s) : s;
    return SLOPE ? s * (1.f + g * (1.f - s)) : g * s;
}
template <bool SLOPE>
CUBF_DEV Pair activation(int act, Pair g) {
    const float2 f = floats(g);
    return f32x2::pk(activation<SLOPE>(act, f.x), activation<SLOPE>(act, f.y));
}

// ---- a row over its threads -------------------------------------------------------------------
// Rows of several warps that share a CTA with others meet on a barrier of
// their own.
template <typename S>
CUBF_DEV void row_barrier() {
    if constexpr (S::TPR == 32) {
        __syncwarp();
    } else if constexpr (S::kRows == 1) {
        __syncthreads();
    } else {
        asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / S::TPR), "n"(S::TPR) : "memory");
    }
}

// Sum over the row's threads, the same in each.  `words` is the row's own
// shared memory; `slot` (0, 1, ...) picks the words used, so that sums in turn
// need one barrier each.
template <typename S>
CUBF_DEV float row_sum(float v, float* words, int slot) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr (S::kWarps > 1) {
        float* w = words + slot * S::kWarps;
        if ((threadIdx.x & 31) == 0) w[threadIdx.x % S::TPR / 32] = v;
        row_barrier<S>();
        v = 0.f;
#pragma unroll
        for (int k = 0; k < S::kWarps; ++k) v += w[k];
    }
    return v;
}

constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

// ---- Hadamard rotation of a row ---------------------------------------------------------------
// The row's index bits are held either by a thread's registers or by the
// thread number.  Butterflies run over the register bits; then the row is
// written to shared memory and read back with other bits in registers, until
// every bit has had its turn, and at the end back in the layout of the loads.
// Four words of padding after every 2^5, 2^8 and 2^11 keep 16-byte accesses
// aligned and, with the thread bits ordered so that the 32 lanes fall into
// different banks, every access without conflicts; being linear in disjoint
// index bits, the padded address is a sum of what the thread and what the
// register contributes, so registers differ by immediate offsets.
CUBF_DEV constexpr uint32_t padded(uint32_t w) { return w + ((w >> 5) << 2) + ((w >> 8) << 2) + ((w >> 11) << 2); }
constexpr int padded_row(int dim) { return static_cast<int>(padded(static_cast<uint32_t>(dim))); }

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

// E registers as E / 2 pairs; register bit 0 lies inside a pair.
template <int E, uint32_t REGS, uint32_t WORK>
CUBF_DEV void butterflies(Pair (&v)[E / 2]) {
    int bit = 0;
#pragma unroll
    for (int p = 0; p < 16; ++p) {
        if (!((REGS >> p) & 1u)) continue;
        if ((WORK >> p) & 1u) {
            if (bit == 0) {
#pragma unroll
                for (int k = 0; k < E / 2; ++k) {
                    const float2 f = floats(v[k]);
                    v[k] = f32x2::pk(f.x + f.y, f.x - f.y);
                }
            } else {
                const int step = 1 << (bit - 1);
#pragma unroll
                for (int k = 0; k < E / 2; ++k)
                    if (!(k & step)) {
                        const Pair a = v[k], b = v[k | step];
                        v[k] = add2(a, b);
                        v[k | step] = sub2(a, b);
                    }
            }
        }
        ++bit;
    }
}

template <int LOGD, int LOGE, int VB, int K, bool WRITE>
CUBF_DEV void move_row(Pair (&v)[1 << LOGE >> 1], float* row, int j) {
    constexpr int E = 1 << LOGE;
    constexpr uint32_t regs = pass_bits<LOGD, LOGE, VB>(K);
    constexpr Layout l = make_layout<LOGD, LOGE>(regs, K == 0);
    constexpr Offsets<E> at = make_offsets<E>(regs);
    uint32_t base = 0;
#pragma unroll
    for (int k = 0; k < LOGD - LOGE; ++k) base |= ((static_cast<uint32_t>(j) >> k) & 1u) << l.order[k];
    float* const mine = row + padded(base);
    if constexpr (K == 0 && VB >= 2) {
#pragma unroll
        for (int r = 0; r < E; r += 4) {
            float4* q = reinterpret_cast<float4*>(mine + padded(at.v[r]));
            if (WRITE) {
                const float2 a = floats(v[r / 2]), b = floats(v[r / 2 + 1]);
                *q = make_float4(a.x, a.y, b.x, b.y);
            } else {
                const float4 f = *q;
                v[r / 2] = f32x2::pk(f.x, f.y);
                v[r / 2 + 1] = f32x2::pk(f.z, f.w);
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < E; r += 2) {
            float* const a = mine + padded(at.v[r]);
            float* const b = mine + padded(at.v[r + 1]);
            if (WRITE) {
                const float2 f = floats(v[r / 2]);
                *a = f.x;
                *b = f.y;
            } else {
                v[r / 2] = f32x2::pk(*a, *b);
            }
        }
    }
}

template <typename S, int K>
CUBF_DEV void rotate_passes(Pair (&v)[S::HALF], float* row, int j) {
    constexpr int LOGE = log2_of(S::EPT), LOGD = log2_of(S::TPR * S::EPT), VB = log2_of(S::VW);
    constexpr int kPasses = 1 + (LOGD - LOGE + LOGE - 1) / LOGE;
    butterflies<S::EPT, pass_bits<LOGD, LOGE, VB>(K), pass_work<LOGD, LOGE, VB>(K)>(v);
    if constexpr (kPasses > 1) {
        constexpr int next = K + 1 < kPasses ? K + 1 : 0;
        if constexpr (K > 0) row_barrier<S>();  // everyone has read the pass before
        move_row<LOGD, LOGE, VB, K, true>(v, row, j);
        row_barrier<S>();
        move_row<LOGD, LOGE, VB, next, false>(v, row, j);
        if constexpr (next > 0) rotate_passes<S, next>(v, row, j);
    }
}

// v <- v H_D (unscaled); D = TPR EPT.  `row` holds padded_row(D) floats.  The
// caller passes a row barrier (a row sum's, say) before the next rotation.
template <typename S>
CUBF_DEV void rotate_row(Pair (&v)[S::HALF], float* row, int j) {
    rotate_passes<S, 0>(v, row, j);
}

// ---- forward ----------------------------------------------------------------------------------
// Shared memory, in floats: the rotated rows, then the words of the row sums,
// then (shapes of many values a thread) the channel factors of s and u.
template <typename S, bool ROTATE>
struct ForwardPlan {
    static constexpr int kDim = S::TPR * S::EPT;
    static constexpr bool kShared = S::EPT > 16;  // factors in shared memory instead of registers
    // Rows of many values a thread are not loaded ahead: their registers go to
    // more rows at a time, whose loads overlap each other's work.
    static constexpr bool kAhead = S::EPT <= 16;
    static constexpr int kRow = ROTATE ? padded_row(kDim) : 0;
    static constexpr int kWordsAt = S::kRows * kRow;
    static constexpr int kFactorsAt = kWordsAt + S::kRows * 4 * S::kWarps;
    static constexpr int kFloats = kFactorsAt + (kShared ? 2 * kDim : 0);
    // 16-bit rows of eight values a thread fit 1024 threads an SM
    template <typename T, typename R>
    static constexpr int ctas() {
        return S::EPT == 8 && S::VW == 8 && sizeof(R) == 2 && !ROTATE && S::kThreads < 1024 ? 1024 / S::kThreads : 1;
    }
};

template <typename T, typename R, typename S, bool ROTATE>
__global__ void __launch_bounds__(S::kThreads, ForwardPlan<S, ROTATE>::template ctas<T, R>())
    block_norm_kernel(BlockNormArgs p) {
    using Plan = ForwardPlan<S, ROTATE>;
    extern __shared__ __align__(16) float shared[];
    pdl_begin();
    const int j = threadIdx.x % S::TPR, sub = threadIdx.x / S::TPR, dim = p.dim;
    float* const exchange = shared + sub * Plan::kRow;
    float* const words = shared + Plan::kWordsAt + sub * 4 * S::kWarps;
    float2* const factors = reinterpret_cast<float2*>(shared + Plan::kFactorsAt);
    const size_t stride = static_cast<size_t>(gridDim.x) * S::kRows;
    size_t row = static_cast<size_t>(blockIdx.x) * S::kRows + sub;
    const float inv_dim = 1.f / static_cast<float>(dim);

    Values<R, S> x;
    Values<T, S> y, g;
    auto load = [&](size_t at) {
        x.load(static_cast<const R*>(p.x) + at * p.x_row, j, dim);
        if (p.y) y.load(static_cast<const T*>(p.y) + at * p.y_row, j, dim);
        if (p.gate_mode == kGateFull) g.load(static_cast<const T*>(p.gate) + at * p.gate_row, j, dim);
    };
    y.clear();
    if (Plan::kAhead && row < p.rows) load(row);

    // What multiplies y r(y) in s (post_weight, and the gate where it is one
    // per channel) and s r(s) in u.
    Pair fy[Plan::kShared ? 1 : S::HALF], fu[Plan::kShared ? 1 : S::HALF];
    {
        Pair a[S::HALF], b[S::HALF];
        load_vector<T, S>(p.post, p.post32, j, dim, 1.f, a);
        if (p.gate_mode == kGateChannel) {
            load_vector<T, S>(p.gate, p.gate32, j, dim, 0.f, b);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) a[k] = mul2(a[k], activation<false>(p.act, b[k]));
        }
        load_vector<T, S>(p.pre, p.pre32, j, dim, 1.f, b);
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) {
            const Pair u = ROTATE ? mul2(b[k], both(p.rotate_scale)) : b[k];
            if constexpr (Plan::kShared) {
                if (sub == 0) {
                    factors[k * S::TPR + j] = floats(a[k]);
                    factors[(S::HALF + k) * S::TPR + j] = floats(u);
                }
            } else {
                fy[k] = a[k];
                fu[k] = u;
            }
        }
        if constexpr (Plan::kShared) __syncthreads();
    }
    auto factor = [&](int which, int k) {
        if constexpr (Plan::kShared) {
            const float2 f = factors[(which * S::HALF + k) * S::TPR + j];
            return f32x2::pk(f.x, f.y);
        } else {
            return which ? fu[k] : fy[k];
        }
    };

    for (int slot = 0; row < p.rows; row += stride, slot ^= 1) {
        if (!Plan::kAhead) load(row);
        Pair s[S::HALF];
        Pair sum = both(0.f);
        float ry = 1.f;
        if (p.post_norm) {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) sum = fma2(y.pair(k), y.pair(k), sum);
            ry = rsqrtf(row_sum<S>(sum_of(sum), words, slot) * inv_dim + p.eps);
            if (p.r_post && j == 0) p.r_post[row] = ry;
        }
        if (p.scales) {
            load_vector<T, S>(p.scales, p.scales32, j, dim, 0.f, s);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) s[k] = mul2(s[k], x.pair(k));
        } else {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) s[k] = mul2(both(p.scale), x.pair(k));
        }
        if (p.y) {
            if (p.gate_mode == kGateFull) {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k)
                    s[k] = fma2(mul2(mul2(factor(0, k), both(ry)), activation<false>(p.act, g.pair(k))), y.pair(k), s[k]);
            } else if (p.gate_mode == kGateGroups) {
                Pair a[S::HALF];
                const size_t at = row / p.rows_per_gate * p.gate_row;
                load_vector<T, S>(p.gate32 ? static_cast<const void*>(static_cast<const float*>(p.gate) + at)
                                           : static_cast<const void*>(static_cast<const T*>(p.gate) + at),
                                  p.gate32, j, dim, 0.f, a);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k)
                    s[k] = fma2(mul2(mul2(factor(0, k), both(ry)), activation<false>(p.act, a[k])), y.pair(k), s[k]);
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) s[k] = fma2(mul2(factor(0, k), both(ry)), y.pair(k), s[k]);
            }
        }
        if (Plan::kAhead && row + stride < p.rows) load(row + stride);
        if (p.residual)
            store_row<S>(static_cast<R*>(p.residual) + row * dim, j, dim, [&](int k) { return s[k]; });
        if (!p.normed) continue;
        sum = both(0.f);
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) sum = fma2(s[k], s[k], sum);
        const float rs = rsqrtf(row_sum<S>(sum_of(sum), words, 2 + slot) * inv_dim + p.eps);
        if (p.r_pre && j == 0) p.r_pre[row] = rs;
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) s[k] = mul2(s[k], mul2(factor(1, k), both(rs)));
        if constexpr (ROTATE) rotate_row<S>(s, exchange, j);
        store_row<S>(static_cast<T*>(p.normed) + row * dim, j, dim, [&](int k) { return s[k]; });
    }
}

// ---- backward ---------------------------------------------------------------------------------
// With yn = y r(y), sn = s r(s), t = du w_pre (du rotated back first) and
// dS = ds + r(s) (t - sn mean(t sn)):
//   dx = alpha dS                dw_pre   = sum du sn        (Q)
//   dn = act(gate) dS            dalpha   = sum dS x         (Z)
//   t' = dn w_post               dy = r(y) (t' - yn mean(t' yn))
//   dgate = act'(gate) dS n      dw_post  = sum dn yn
// A thread owns its columns for every row of its CTA, so the sums over rows
// stay in registers (in shared memory, by the same thread, for shapes of many
// values a thread; Z, which few calls need, always).  A CTA's rows share one
// gate row, so that for a gate per channel or per group dw_post and dgate both
// follow from P = sum dS yn; with a gate per row P = sum dn yn.  Each CTA
// writes its sums once and a second kernel adds them in a fixed order.
template <typename S, bool ROTATE>
struct BackwardPlan {
    static constexpr int kDim = S::TPR * S::EPT;
    static constexpr bool kLean = S::EPT * S::kThreads > 4096 || S::EPT > 8;  // no room for the next row in registers
    static constexpr bool kSharedSums = S::EPT > 8 && !(ROTATE && S::kThreads <= 256);
    static constexpr bool kSharedZ = !(ROTATE && kDim > 8192);  // else Z is summed in the CTA's part of the workspace
    static constexpr int kRow = ROTATE ? padded_row(kDim) : 0;
    static constexpr int kWordsAt = S::kRows * kRow;
    static constexpr int kSumsAt = kWordsAt + S::kRows * 4 * S::kWarps;   // P and Q if shared, then Z
    static constexpr int kFloats = kSumsAt + S::kRows * kDim * ((kSharedSums ? 2 : 0) + (kSharedZ ? 1 : 0));
};

// t - vn mean(t vn), the part of t that a norm lets through.  In a row of one
// value vn^2 = 1 - eps r^2, and the difference would cancel.
CUBF_DEV Pair through_norm(const BlockNormArgs& p, Pair t, Pair vn, float mean, float r) {
    return p.dim == 1 ? mul2(t, both(p.eps * r * r)) : fma2(vn, both(-mean), t);
}

template <typename T, typename R, typename S, bool ROTATE>
__global__ void __launch_bounds__(S::kThreads, 1) block_norm_backward_kernel(BlockNormArgs p) {
    using Plan = BackwardPlan<S, ROTATE>;
    extern __shared__ __align__(16) float shared[];
    pdl_begin();
    const int j = threadIdx.x % S::TPR, sub = threadIdx.x / S::TPR, dim = p.dim;
    float* const exchange = shared + sub * Plan::kRow;
    float* const words = shared + Plan::kWordsAt + sub * 4 * S::kWarps;
    // the thread's own sums: pair k at [k][thread]
    float2* const mine = reinterpret_cast<float2*>(shared + Plan::kSumsAt) + threadIdx.x;
    constexpr int kSumStride = S::HALF * S::kThreads;
    const float inv_dim = 1.f / static_cast<float>(dim);
    // this CTA's rows: a share of one gate group's
    const size_t group = blockIdx.x / p.parts_per_group;
    const size_t share = (p.rows_per_gate + p.parts_per_group - 1) / p.parts_per_group;
    const size_t from = (blockIdx.x % p.parts_per_group) * share;
    const size_t to = from + share < p.rows_per_gate ? from + share : p.rows_per_gate;
    const size_t end = group * p.rows_per_gate + to;
    size_t row = group * p.rows_per_gate + from + sub;

    struct Row {
        Values<R, S> x, ds;
        Values<T, S> y, g, du;
        float ry, rs;
    };
    auto load = [&](size_t at, Row& in) {
        in.x.load(static_cast<const R*>(p.x) + at * p.x_row, j, dim);
        if (p.y) in.y.load(static_cast<const T*>(p.y) + at * p.y_row, j, dim);
        if (p.d_residual) in.ds.load(static_cast<const R*>(p.d_residual) + at * p.d_residual_row, j, dim);
        if (p.d_normed) in.du.load(static_cast<const T*>(p.d_normed) + at * p.d_normed_row, j, dim);
        if (p.gate_mode == kGateFull) in.g.load(static_cast<const T*>(p.gate) + at * p.gate_row, j, dim);
        in.ry = p.post_norm ? p.r_post[at] : 1.f;
        in.rs = p.d_normed ? p.r_pre[at] : 0.f;
    };
    Row in;
    in.y.clear();
    in.ds.clear();
    in.du.clear();
    in.g.clear();
    if (row < end) load(row, in);

    // channel factors: w_post, act(gate) where the CTA's rows share it, and w_pre
    constexpr bool kKeep = !Plan::kLean;
    Pair kw[kKeep ? S::HALF : 1], ka[kKeep ? S::HALF : 1], kp[kKeep ? S::HALF : 1];
    const bool row_gate = p.gate_mode == kGateFull, shared_gate = p.gate_mode == kGateChannel || p.gate_mode == kGateGroups;
    auto gate_factor = [&](Pair(&a)[S::HALF]) {
        const size_t at = p.gate_mode == kGateGroups ? group * p.gate_row : 0;
        load_vector<T, S>(!shared_gate ? nullptr
                          : p.gate32   ? static_cast<const void*>(static_cast<const float*>(p.gate) + at)
                                       : static_cast<const void*>(static_cast<const T*>(p.gate) + at),
                          p.gate32, j, dim, 1.f, a);
        if (shared_gate) {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) a[k] = activation<false>(p.act, a[k]);
        }
    };
    if constexpr (kKeep) {
        load_vector<T, S>(p.post, p.post32, j, dim, 1.f, kw);
        gate_factor(ka);
        load_vector<T, S>(p.pre, p.pre32, j, dim, 1.f, kp);
    }
    Pair P[Plan::kSharedSums ? 1 : S::HALF], Q[Plan::kSharedSums ? 1 : S::HALF];
#pragma unroll
    for (int k = 0; k < (Plan::kSharedSums ? 1 : S::HALF); ++k) P[k] = Q[k] = both(0.f);
#pragma unroll
    for (int k = 0; k < S::HALF * ((Plan::kSharedSums ? 2 : 0) + (Plan::kSharedZ ? 1 : 0)); ++k)
        mine[k * S::kThreads] = make_float2(0.f, 0.f);
    float* const part = p.partials + static_cast<size_t>(blockIdx.x) * 3 * dim;
    if (!Plan::kSharedZ && p.need_z)
        store_row<S>(part + 2 * static_cast<size_t>(dim), j, dim, [&](int) { return both(0.f); });
    constexpr int kP = 0, kQ = 1, kZ = 2;
    constexpr int kPlaceZ = Plan::kSharedSums ? 2 : 0;
    auto add_sum = [&](Pair* regs, int which, int k, Pair a, Pair b) {  // += a b
        if (!Plan::kSharedSums && which != kZ) {
            regs[k] = fma2(a, b, regs[k]);
        } else {
            float2* at = mine + (which == kZ ? kPlaceZ : which) * kSumStride + k * S::kThreads;
            const float2 f = *at;
            *at = floats(fma2(a, b, f32x2::pk(f.x, f.y)));
        }
    };

    for (int slot = 0; row < end; row += S::kRows, slot ^= 1) {
        Row ahead;
        if constexpr (!Plan::kLean) {
            ahead = in;
            if (row + S::kRows < end) load(row + S::kRows, ahead);
        }
        Pair d[S::HALF];   // du, t, then t'
        Pair sn[S::HALF];  // s r(s)
        float dot = 0.f;
        if (p.d_normed) {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) d[k] = in.du.pair(k);
            if constexpr (ROTATE) {
                rotate_row<S>(d, exchange, j);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) d[k] = mul2(d[k], both(p.rotate_scale));
            }
            if (p.scales) {
                load_vector<T, S>(p.scales, p.scales32, j, dim, 0.f, sn);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(sn[k], in.x.pair(k));
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(both(p.scale), in.x.pair(k));
            }
            if (p.y) {
                Pair lw[kKeep ? 1 : S::HALF], la[kKeep ? 1 : S::HALF];
                if constexpr (!kKeep) {
                    load_vector<T, S>(p.post, p.post32, j, dim, 1.f, lw);
                    gate_factor(la);
                }
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) {
                    Pair f = kKeep ? kw[k] : lw[k];
                    f = mul2(f, row_gate ? activation<false>(p.act, in.g.pair(k)) : kKeep ? ka[k] : la[k]);
                    sn[k] = fma2(mul2(f, both(in.ry)), in.y.pair(k), sn[k]);
                }
            }
            {
                Pair lp[kKeep ? 1 : S::HALF];
                if constexpr (!kKeep) load_vector<T, S>(p.pre, p.pre32, j, dim, 1.f, lp);
                Pair sum = both(0.f);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) {
                    sn[k] = mul2(sn[k], both(in.rs));
                    if (p.need_q) add_sum(Q, kQ, k, d[k], sn[k]);
                    d[k] = mul2(d[k], kKeep ? kp[k] : lp[k]);
                    sum = fma2(d[k], sn[k], sum);
                }
                dot = row_sum<S>(sum_of(sum), words, slot) * inv_dim;
            }
            // dS
#pragma unroll
            for (int k = 0; k < S::HALF; ++k)
                d[k] = fma2(through_norm(p, d[k], sn[k], dot, in.rs), both(in.rs), in.ds.pair(k));
        } else {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) d[k] = in.ds.pair(k);
        }
        {
            if (p.scales) {
                load_vector<T, S>(p.scales, p.scales32, j, dim, 0.f, sn);
                if constexpr (Plan::kSharedZ) {
#pragma unroll
                    for (int k = 0; k < S::HALF; ++k) add_sum(nullptr, kZ, k, d[k], in.x.pair(k));
                } else {
                    float* const z = part + 2 * static_cast<size_t>(dim);
                    Values<float, S> old;
                    old.load(z, j, dim);
                    store_row<S>(z, j, dim, [&](int k) { return fma2(d[k], in.x.pair(k), old.pair(k)); });
                }
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(sn[k], d[k]);
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(both(p.scale), d[k]);
            }
            store_row<S>(static_cast<R*>(p.d_x) + row * dim, j, dim, [&](int k) { return sn[k]; });
        }
        if (p.y) {
            Pair lw[kKeep ? 1 : S::HALF], la[kKeep ? 1 : S::HALF];
            if constexpr (!kKeep) {
                load_vector<T, S>(p.post, p.post32, j, dim, 1.f, lw);
                gate_factor(la);
            }
            Pair sum = both(0.f);
            if (row_gate) {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) {
                    const Pair w = kKeep ? kw[k] : lw[k], g = in.g.pair(k);
                    const Pair yn = mul2(in.y.pair(k), both(in.ry));
                    sn[k] = mul2(mul2(mul2(d[k], yn), w), activation<true>(p.act, g));  // dgate
                    d[k] = mul2(d[k], activation<false>(p.act, g));                       // dn
                    if (p.need_p) add_sum(P, kP, k, d[k], yn);
                    d[k] = mul2(d[k], w);
                    sum = fma2(d[k], yn, sum);
                }
                store_row<S>(static_cast<T*>(p.d_gate) + row * dim, j, dim, [&](int k) { return sn[k]; });
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) {
                    const Pair yn = mul2(in.y.pair(k), both(in.ry));
                    if (p.need_p) add_sum(P, kP, k, d[k], yn);
                    d[k] = mul2(d[k], mul2(kKeep ? kw[k] : lw[k], kKeep ? ka[k] : la[k]));
                    sum = fma2(d[k], yn, sum);
                }
            }
            if (p.post_norm) {
                const float mean = row_sum<S>(sum_of(sum), words, 2 + slot) * inv_dim;
#pragma unroll
                for (int k = 0; k < S::HALF; ++k)
                    d[k] = mul2(through_norm(p, d[k], mul2(in.y.pair(k), both(in.ry)), mean, in.ry), both(in.ry));
            }
            store_row<S>(static_cast<T*>(p.d_y) + row * dim, j, dim, [&](int k) { return d[k]; });
        }
        if constexpr (Plan::kLean) {
            if (row + S::kRows < end) load(row + S::kRows, in);
        } else {
            in = ahead;
        }
    }
    // The CTA's sums; rows side by side in a CTA are added first, in shared memory.
    auto write = [&](Pair* regs, int which, float* dst) {
        const bool held = !Plan::kSharedSums && which != kZ;  // in registers
        float2* const at = mine + (which == kZ ? kPlaceZ : Plan::kSharedSums ? which : 0) * kSumStride;
        Pair v[S::HALF];
        if (held && S::kRows > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) at[k * S::kThreads] = floats(regs[k]);
        }
        if constexpr (S::kRows > 1) {
            __syncthreads();
            if (sub > 0) return;
        }
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) {
            if (held && S::kRows == 1) {
                v[k] = regs[k];
            } else {
                v[k] = both(0.f);
                for (int o = 0; o < S::kRows; ++o) {
                    const float2 f = at[k * S::kThreads + o * S::TPR];
                    v[k] = add2(v[k], f32x2::pk(f.x, f.y));
                }
            }
        }
        store_row<S>(dst, j, dim, [&](int k) { return v[k]; });
    };
    if (Plan::kSharedZ && p.need_z) write(nullptr, kZ, part + 2 * static_cast<size_t>(dim));
    if (p.need_p) write(P, kP, part);
    if (p.need_q) write(Q, kQ, part + dim);
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
        return is32 || sizeof(T) == 4 ? static_cast<const float*>(v)[at]
                                      : Convert<T, float>::load(static_cast<const T*>(v)[at]);
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
