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
// works on this one, and brings the one after towards L2; what depends on the
// channel alone is formed once.
//
// Bound by memory: 16384 x 4096 bf16 in 88 us (6.1 TB/s of the device copy's
// 6.5), with an fp32 residual and a gate per row 8192 x 4096 in 78 us (6.0).
// Rotated rows move through shared memory six times, beside 4.7 TB/s: 114 us, its
// wavefronts at 67 % and the SM's one CTA waiting on exchanges and loads in turn.
// Backward, where two row sums depend on each other: 168 us (4.8 TB/s), rotated
// 209, with the gate 148 (5.0).  Rows that are not whole vectors wait for their
// loads, one value or pair each: 16000 x 1001 in 43 and 104 us, 1002 in 26 and 49.
#pragma once

#include "block_ops.hpp"
#include "common.cuh"
#include "f32x2.cuh"
#include "gate.cuh"

namespace cubf::norm {

using f32x2::add2;
using f32x2::fma2;
using f32x2::mul2;
using f32x2::sub2;
using gate::both;
using Pair = f32x2::P;

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
    static constexpr bool kBulk = VW >= 4;          // rows are whole 16-byte vectors (see the launches)
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
                const T* from = row + S::at(c, j);
                uint32_t* to = w + c * kPer;
                if constexpr (kPer >= 4) {
#pragma unroll
                    for (int k = 0; k < kPer; k += 4) {
                        const uint4* p = reinterpret_cast<const uint4*>(from) + k / 4;
                        uint4 q = make_uint4(0, 0, 0, 0);
                        if (in) q = STREAM ? __ldcs(p) : __ldg(p);
                        to[k] = q.x;
                        to[k + 1] = q.y;
                        to[k + 2] = q.z;
                        to[k + 3] = q.w;
                    }
                } else if constexpr (kPer == 2) {
                    const uint2* p = reinterpret_cast<const uint2*>(from);
                    uint2 q = make_uint2(0, 0);
                    if (in) q = STREAM ? __ldcs(p) : __ldg(p);
                    to[0] = q.x;
                    to[1] = q.y;
                } else {
                    const unsigned int* p = reinterpret_cast<const unsigned int*>(from);
                    to[0] = 0;
                    if (in) to[0] = STREAM ? __ldcs(p) : __ldg(p);
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
            constexpr int kPer = S::VW * static_cast<int>(sizeof(T)) / 4;
            uint32_t w[kPer];
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
                T* to = row + S::at(c, j);
                if constexpr (kPer >= 4) {
#pragma unroll
                    for (int k = 0; k < kPer; k += 4)
                        __stcs(reinterpret_cast<uint4*>(to) + k / 4, make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]));
                } else if constexpr (kPer == 2) {
                    __stcs(reinterpret_cast<uint2*>(to), make_uint2(w[0], w[1]));
                } else {
                    __stcs(reinterpret_cast<unsigned int*>(to), w[0]);
                }
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

// Brings a row of `bytes` bytes towards L2: as one bulk prefetch by the row's
// first thread, which alone calls it, where rows are whole 16-byte vectors; else
// a line a thread.
template <typename S>
CUBF_DEV void prefetch_row(const void* row, uint32_t bytes, int j) {
    if constexpr (S::kBulk) {
        prefetch_l2(row, bytes);
    } else if (static_cast<uint32_t>(j) * 128 < bytes) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(row) + j * 128));
    }
}

// Beside a residual of 16 bits the gates' sigmoid is good to two units of 2^-24
// and more by |g| of them; with an fp32 residual, and in the gradients of gates
// that rows share, it is the exact one (8192 x 4096 bf16, fp32 residual, silu
// gate per row: 78 us forward and 148 backward either way; 16000 x 1001: 61 and
// 108 for 55 and 108).
template <typename R>
constexpr bool kExactGates = sizeof(R) == 4;
CUBF_DEV float short_sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }
template <bool EXACT>
CUBF_DEV Pair sigmoid(Pair g) {
    if constexpr (EXACT) {
        return gate::sigmoid(g);
    } else {
        const float2 f = floats(g);
        return f32x2::pk(short_sigmoid(f.x), short_sigmoid(f.y));
    }
}

// act(g), or its slope where SLOPE, from g and its sigmoid s
template <bool SLOPE>
CUBF_DEV float from_sigmoid(int act, float g, float s) {
    if (act == 1) return SLOPE ? s * (1.f - s) : s;
    return SLOPE ? s * (1.f + g * (1.f - s)) : g * s;
}
// act(g)
template <bool EXACT>
CUBF_DEV float activation(int act, float g) {
    if (act == 0) return g;
    return from_sigmoid<false>(act, g, EXACT ? floats(sigmoid<EXACT>(both(g))).x : short_sigmoid(g));
}
template <bool EXACT>
CUBF_DEV Pair activation(int act, Pair g) {
    const float2 f = floats(g);
    if constexpr (EXACT) {
        if (act == 0) return g;
        const float2 s = floats(sigmoid<EXACT>(g));
        return f32x2::pk(from_sigmoid<false>(act, f.x, s.x), from_sigmoid<false>(act, f.y, s.y));
    } else {
        return f32x2::pk(activation<EXACT>(act, f.x), activation<EXACT>(act, f.y));
    }
}
// act(g) and its slope from one sigmoid
template <bool EXACT, typename Act>
CUBF_DEV void activation_with_slope(Act act, Pair g, Pair& value, Pair& slope) {
    if (act == 0) {
        value = g;
        slope = both(1.f);
        return;
    }
    const Pair s = sigmoid<EXACT>(g), rest = sub2(both(1.f), s);
    if (act == 1) {
        value = s;
        slope = mul2(s, rest);
    } else {
        value = mul2(g, s);
        slope = fma2(value, rest, s);  // s + g s (1 - s)
    }
}
// body(act) with the activation a constant in it
template <typename Body>
CUBF_DEV void with_activation(int act, Body&& body) {
    if (act == 0)
        body(std::integral_constant<int, 0>());
    else if (act == 1)
        body(std::integral_constant<int, 1>());
    else
        body(std::integral_constant<int, 2>());
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
        if constexpr (S::kWarps >= 4) {
            Pair t = both(0.f);
#pragma unroll
            for (int k = 0; k < S::kWarps; k += 4) {
                const float4 q = *reinterpret_cast<const float4*>(w + k);
                t = add2(t, add2(f32x2::pk(q.x, q.y), f32x2::pk(q.z, q.w)));
            }
            v = sum_of(t);
        } else {
            v = w[0] + w[1];
        }
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

template <typename T>
CUBF_DEV uint32_t dim_bytes(int dim) {
    return static_cast<uint32_t>(dim) * static_cast<uint32_t>(sizeof(T));
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
    static constexpr uint32_t kPrefetch = kAhead ? 2 : 1;  // turns ahead that a row is brought to L2
    static constexpr int kRow = ROTATE ? padded_row(kDim) : 0;
    static constexpr int kWordsAt = S::kRows * kRow;
    static constexpr int kFactorsAt = kWordsAt + S::kRows * 4 * S::kWarps;
    static constexpr int kFloats = kFactorsAt + (kShared ? 2 * kDim : 0);
    // 16-bit rows of eight values a thread fit 1024 threads an SM
    static constexpr int kCtas = S::EPT == 8 && S::VW == 8 && !ROTATE && S::kThreads < 1024 ? 1024 / S::kThreads : 1;
};

template <typename T, typename R, typename S, bool ROTATE>
__global__ void __launch_bounds__(S::kThreads, ForwardPlan<S, ROTATE>::kCtas)
    block_norm_kernel(BlockNormArgs p) {
    using Plan = ForwardPlan<S, ROTATE>;
    extern __shared__ __align__(16) float shared[];
    pdl_begin();
    const int j = threadIdx.x % S::TPR, sub = threadIdx.x / S::TPR, dim = p.dim;
    float* const exchange = shared + sub * Plan::kRow;
    float* const words = shared + Plan::kWordsAt + sub * 4 * S::kWarps;
    float2* const factors = reinterpret_cast<float2*>(shared + Plan::kFactorsAt);
    const uint32_t stride = gridDim.x * S::kRows, rows = static_cast<uint32_t>(p.rows);
    uint32_t row = blockIdx.x * S::kRows + sub;
    const float inv_dim = 1.f / static_cast<float>(dim);

    Values<R, S> x;
    Values<T, S> y, g;
    // row `n` of a tensor: one multiply-add, its operands in constant memory
    auto at = [&](auto* base, uint32_t bytes, uint32_t n) {
        using E = std::remove_pointer_t<decltype(base)>;
        using Byte = std::conditional_t<std::is_const<E>::value, const char, char>;
        return reinterpret_cast<E*>(reinterpret_cast<Byte*>(base) + static_cast<unsigned long long>(n) * bytes);
    };
    auto load = [&](uint32_t n) {
        x.load(at(static_cast<const R*>(p.x), p.x_bytes, n), j, dim);
        if (p.y) y.load(at(static_cast<const T*>(p.y), p.y_bytes, n), j, dim);
        if (p.gate_mode == kGateFull) g.load(at(static_cast<const T*>(p.gate), p.gate_bytes, n), j, dim);
    };
    y.clear();
    if (Plan::kAhead && row < rows) load(row);

    // What multiplies y r(y) in s (post_weight, and the gate where it is one
    // per channel) and s r(s) in u.
    Pair fy[Plan::kShared ? 1 : S::HALF], fu[Plan::kShared ? 1 : S::HALF];
    {
        Pair a[S::HALF], b[S::HALF];
        load_vector<T, S>(p.post, p.post32, j, dim, 1.f, a);
        if (p.gate_mode == kGateChannel) {
            load_vector<T, S>(p.gate, p.gate32, j, dim, 0.f, b);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) a[k] = mul2(a[k], activation<kExactGates<R>>(p.act, b[k]));
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

    for (int slot = 0; row < rows; row += stride, slot ^= 1) {
        if (!Plan::kAhead) load(row);
        if ((!S::kBulk || j == 0) && row + Plan::kPrefetch * stride < rows) {  // towards L2, before it is loaded
            const uint32_t n = row + Plan::kPrefetch * stride;
            prefetch_row<S>(at(static_cast<const R*>(p.x), p.x_bytes, n), dim_bytes<R>(dim), j);
            if (p.y) prefetch_row<S>(at(static_cast<const T*>(p.y), p.y_bytes, n), dim_bytes<T>(dim), j);
            if (p.gate_mode == kGateFull) prefetch_row<S>(at(static_cast<const T*>(p.gate), p.gate_bytes, n), dim_bytes<T>(dim), j);
        }
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
                with_activation(p.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < S::HALF; ++k)
                        s[k] = fma2(mul2(mul2(factor(0, k), both(ry)), activation<kExactGates<R>>(act, g.pair(k))), y.pair(k), s[k]);
                });
            } else if (p.gate_mode == kGateGroups) {
                Pair a[S::HALF];
                const size_t from = row / static_cast<uint32_t>(p.rows_per_gate) * p.gate_row;
                load_vector<T, S>(p.gate32 ? static_cast<const void*>(static_cast<const float*>(p.gate) + from)
                                           : static_cast<const void*>(static_cast<const T*>(p.gate) + from),
                                  p.gate32, j, dim, 0.f, a);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k)
                    s[k] = fma2(mul2(mul2(factor(0, k), both(ry)), activation<kExactGates<R>>(p.act, a[k])), y.pair(k), s[k]);
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) s[k] = fma2(mul2(factor(0, k), both(ry)), y.pair(k), s[k]);
            }
        }
        if (Plan::kAhead && row + stride < rows) load(row + stride);
        if (p.residual)
            store_row<S>(at(static_cast<R*>(p.residual), dim_bytes<R>(dim), row), j, dim, [&](int k) { return s[k]; });
        if (!p.normed) continue;
        sum = both(0.f);
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) sum = fma2(s[k], s[k], sum);
        const float rs = rsqrtf(row_sum<S>(sum_of(sum), words, 2 + slot) * inv_dim + p.eps);
        if (p.r_pre && j == 0) p.r_pre[row] = rs;
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) s[k] = mul2(s[k], mul2(factor(1, k), both(rs)));
        if constexpr (ROTATE) rotate_row<S>(s, exchange, j);
        store_row<S>(at(static_cast<T*>(p.normed), dim_bytes<T>(dim), row), j, dim, [&](int k) { return s[k]; });
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
// Up to 512 threads a CTA have registers for the sums P and Q, and with eight
// values a thread for the channel factors of y r(y) and s r(s) too; else those
// lie in shared memory, or are loaded through L1 where a row does not leave
// room.  Shared memory, in floats: the rotated rows, the words of the row
// sums, the factors, the sums (with P and Q or without), and Z where needed.
template <typename S, bool ROTATE>
struct BackwardPlan {
    static constexpr int kDim = S::TPR * S::EPT;
    static constexpr bool kHeldSums = S::kThreads <= 512 && S::EPT <= 8;
    static constexpr bool kHeldFactors = kHeldSums;
    static constexpr bool kSharedFactors = !kHeldFactors && kDim <= 8192;
    static constexpr bool kSharedZ = !(ROTATE && kDim > 8192);  // else Z is summed in the CTA's part of the workspace
    static constexpr int kRow = ROTATE ? padded_row(kDim) : 0;
    static constexpr int kWordsAt = S::kRows * kRow;
    static constexpr int kFactorsAt = kWordsAt + S::kRows * 4 * S::kWarps;
    static constexpr int kSumsAt = kFactorsAt + (kSharedFactors ? 2 * kDim : 0);
    static constexpr int kSum = S::kThreads * S::EPT;
    static constexpr int kPlaces = kHeldSums ? (S::kRows > 1 ? 1 : 0) : 2;  // rows side by side add their sums there
    static constexpr int kPlaceZ = kHeldSums ? 0 : 2;
    static constexpr int floats_needed(bool z) {
        const int places = z && kSharedZ ? kPlaceZ + 1 : 0;
        return kSumsAt + kSum * (places > kPlaces ? places : kPlaces);
    }
};

// r (t - vn mean(t vn)), the part of t that a norm lets through, is taken as
// r' (t - vn m).  In a row of one value vn^2 = 1 - eps r^2, and the difference
// would cancel: there m = 0 and r' = eps r^3.
struct Through {
    float m, r;
    CUBF_DEV Through(const BlockNormArgs& p, float mean, float factor)
        : m(p.dim == 1 ? 0.f : -mean), r(p.dim == 1 ? p.eps * factor * factor * factor : factor) {}
};

template <typename T, typename R, typename S, bool ROTATE>
__global__ void __launch_bounds__(S::kThreads, 1) block_norm_backward_kernel(BlockNormArgs p) {
    using Plan = BackwardPlan<S, ROTATE>;
    extern __shared__ __align__(16) float shared[];
    pdl_begin();
    const int j = threadIdx.x % S::TPR, sub = threadIdx.x / S::TPR, dim = p.dim;
    float* const exchange = shared + sub * Plan::kRow;
    float* const words = shared + Plan::kWordsAt + sub * 4 * S::kWarps;
    float2* const factors = reinterpret_cast<float2*>(shared + Plan::kFactorsAt);
    // the thread's own sums: pair k of sum n at [n][k][thread]
    float2* const mine = reinterpret_cast<float2*>(shared + Plan::kSumsAt) + threadIdx.x;
    const float inv_dim = 1.f / static_cast<float>(dim);
    // this CTA's rows: a share of one gate group's
    const size_t group = blockIdx.x / p.parts_per_group;
    const size_t share = (p.rows_per_gate + p.parts_per_group - 1) / p.parts_per_group;
    const size_t from = (blockIdx.x % p.parts_per_group) * share;
    const size_t to = from + share < p.rows_per_gate ? from + share : p.rows_per_gate;
    const size_t end = group * p.rows_per_gate + to;
    size_t row = group * p.rows_per_gate + from + sub;

    // The row in work, and of the next one what has been loaded already: each
    // tensor's registers are loaded again as soon as they have been used.
    Values<R, S> x, ds;
    Values<T, S> y, g, du;
    float ry = 1.f, rs = 0.f, next_ry = 1.f, next_rs = 0.f;
    const bool row_gate = p.gate_mode == kGateFull;
    // row `n` of a tensor: one multiply-add, its operands in constant memory
    uint32_t n = static_cast<uint32_t>(row);
    const uint32_t last = static_cast<uint32_t>(end);
    auto at = [&](auto* base, uint32_t bytes, uint32_t ahead) {
        using E = std::remove_pointer_t<decltype(base)>;
        using Byte = std::conditional_t<std::is_const<E>::value, const char, char>;
        return reinterpret_cast<E*>(reinterpret_cast<Byte*>(base) + static_cast<unsigned long long>(n + ahead) * bytes);
    };
    auto load_du = [&](uint32_t ahead) {
        if (p.d_normed) du.load(at(static_cast<const T*>(p.d_normed), p.d_normed_bytes, ahead), j, dim);
    };
    auto load_ds = [&](uint32_t ahead) {
        if (p.d_residual) ds.load(at(static_cast<const R*>(p.d_residual), p.d_residual_bytes, ahead), j, dim);
    };
    auto load_x = [&](uint32_t ahead) { x.load(at(static_cast<const R*>(p.x), p.x_bytes, ahead), j, dim); };
    auto load_y = [&](Values<T, S>& y, Values<T, S>& g, uint32_t ahead) {
        if (p.y) y.load(at(static_cast<const T*>(p.y), p.y_bytes, ahead), j, dim);
        if (row_gate) g.load(at(static_cast<const T*>(p.gate), p.gate_bytes, ahead), j, dim);
    };
    y.clear();
    ds.clear();
    du.clear();
    if (n < last) {
        load_du(0);
        load_x(0);
        load_y(y, g, 0);
        load_ds(0);
        if (p.post_norm) ry = p.r_post[n];
        if (p.d_normed) rs = p.r_pre[n];
    }

    // channel factors: w_post times act(gate) where the CTA's rows share it, and w_pre
    auto factor_y = [&](Pair(&a)[S::HALF]) {
        load_vector<T, S>(p.post, p.post32, j, dim, 1.f, a);
        if (p.gate_mode == kGateChannel || p.gate_mode == kGateGroups) {
            const size_t at = p.gate_mode == kGateGroups ? group * p.gate_row : 0;
            Pair b[S::HALF];
            load_vector<T, S>(p.gate32 ? static_cast<const void*>(static_cast<const float*>(p.gate) + at)
                                       : static_cast<const void*>(static_cast<const T*>(p.gate) + at),
                              p.gate32, j, dim, 1.f, b);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) a[k] = mul2(a[k], activation<kExactGates<R>>(p.act, b[k]));
        }
    };
    Pair held[Plan::kHeldFactors ? 2 : 1][Plan::kHeldFactors || !Plan::kSharedFactors ? S::HALF : 1];
    if constexpr (Plan::kHeldFactors) {
        factor_y(held[0]);
        load_vector<T, S>(p.pre, p.pre32, j, dim, 1.f, held[1]);
    } else if constexpr (Plan::kSharedFactors) {
        Pair a[S::HALF];
        if (sub == 0) {
            factor_y(a);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) factors[k * S::TPR + j] = floats(a[k]);
            load_vector<T, S>(p.pre, p.pre32, j, dim, 1.f, a);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) factors[(S::HALF + k) * S::TPR + j] = floats(a[k]);
        }
        __syncthreads();
    }
    auto bring = [&](int which) {  // factors that have no place are loaded each time
        if constexpr (!Plan::kHeldFactors && !Plan::kSharedFactors) {
            if (which == 0)
                factor_y(held[0]);
            else
                load_vector<T, S>(p.pre, p.pre32, j, dim, 1.f, held[0]);
        }
    };
    auto factor = [&](int which, int k) {
        if constexpr (Plan::kSharedFactors) {
            const float2 f = factors[(which * S::HALF + k) * S::TPR + j];
            return f32x2::pk(f.x, f.y);
        } else {
            return held[Plan::kHeldFactors ? which : 0][k];
        }
    };
    constexpr int kP = 0, kQ = 1, kZ = 2;
    Pair sums[Plan::kHeldSums ? 2 : 1][Plan::kHeldSums ? S::HALF : 1];
#pragma unroll
    for (int k = 0; k < S::HALF; ++k) {
        if constexpr (Plan::kHeldSums)
            sums[kP][k] = sums[kQ][k] = both(0.f);
        else
            mine[k * S::kThreads] = mine[(S::HALF + k) * S::kThreads] = make_float2(0.f, 0.f);
        if (Plan::kSharedZ && p.need_z) mine[(Plan::kPlaceZ * S::HALF + k) * S::kThreads] = make_float2(0.f, 0.f);
    }
    float* const part = p.partials + static_cast<size_t>(blockIdx.x) * 3 * dim;
    if (!Plan::kSharedZ && p.need_z)
        store_row<S>(part + 2 * static_cast<size_t>(dim), j, dim, [&](int) { return both(0.f); });
    auto add_sum = [&](int which, int k, Pair a, Pair b) {  // += a b
        if constexpr (Plan::kHeldSums) {
            if (which != kZ) {
                sums[which][k] = fma2(a, b, sums[which][k]);
                return;
            }
        }
        float2* const at = mine + ((which == kZ ? Plan::kPlaceZ : which) * S::HALF + k) * S::kThreads;
        const float2 f = *at;
        *at = floats(fma2(a, b, f32x2::pk(f.x, f.y)));
    };

    for (int slot = 0; n < last; n += S::kRows, slot ^= 1) {
        const bool more = n + S::kRows < last;
        if ((!S::kBulk || j == 0) && n + 2 * S::kRows < last) {  // towards L2, a row before it is loaded
            constexpr uint32_t kTwo = 2 * S::kRows;
            prefetch_row<S>(at(static_cast<const R*>(p.x), p.x_bytes, kTwo), dim_bytes<R>(dim), j);
            if (p.d_residual) prefetch_row<S>(at(static_cast<const R*>(p.d_residual), p.d_residual_bytes, kTwo), dim_bytes<R>(dim), j);
            if (p.y) prefetch_row<S>(at(static_cast<const T*>(p.y), p.y_bytes, kTwo), dim_bytes<T>(dim), j);
            if (p.d_normed) prefetch_row<S>(at(static_cast<const T*>(p.d_normed), p.d_normed_bytes, kTwo), dim_bytes<T>(dim), j);
            if (row_gate) prefetch_row<S>(at(static_cast<const T*>(p.gate), p.gate_bytes, kTwo), dim_bytes<T>(dim), j);
        }
        Values<T, S> y_next, g_next;  // used first in the next row, and last in this one
        y_next.clear();
        if (more) {
            load_y(y_next, g_next, S::kRows);
            if (p.post_norm) next_ry = p.r_post[n + S::kRows];
            if (p.d_normed) next_rs = p.r_pre[n + S::kRows];
        }
        Pair d[S::HALF];   // du, t, then t'
        Pair sn[S::HALF];  // s r(s), then dx, dgate and y r(y)
        if (p.d_normed) {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) d[k] = du.pair(k);
            if (more) load_du(S::kRows);
            if constexpr (ROTATE) {
                rotate_row<S>(d, exchange, j);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) d[k] = mul2(d[k], both(p.rotate_scale));
            }
            if (p.scales) {
                load_vector<T, S>(p.scales, p.scales32, j, dim, 0.f, sn);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(sn[k], x.pair(k));
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(both(p.scale), x.pair(k));
            }
            if (p.y) {
                bring(0);
                if (row_gate) {
                    with_activation(p.act, [&](auto act) {
#pragma unroll
                        for (int k = 0; k < S::HALF; ++k)
                            sn[k] = fma2(mul2(mul2(factor(0, k), both(ry)), activation<kExactGates<R>>(act, g.pair(k))),
                                         y.pair(k), sn[k]);
                    });
                } else {
#pragma unroll
                    for (int k = 0; k < S::HALF; ++k)
                        sn[k] = fma2(mul2(factor(0, k), both(ry)), y.pair(k), sn[k]);
                }
            }
            bring(1);
            Pair sum = both(0.f);
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) {
                sn[k] = mul2(sn[k], both(rs));
                add_sum(kQ, k, d[k], sn[k]);
                d[k] = mul2(d[k], factor(1, k));
                sum = fma2(d[k], sn[k], sum);
            }
            const Through through(p, row_sum<S>(sum_of(sum), words, slot) * inv_dim, rs);
            // dS
#pragma unroll
            for (int k = 0; k < S::HALF; ++k)
                d[k] = fma2(fma2(sn[k], both(through.m), d[k]), both(through.r), ds.pair(k));
        } else {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) d[k] = ds.pair(k);
        }
        if (more) load_ds(S::kRows);
        if (p.scales) {
            load_vector<T, S>(p.scales, p.scales32, j, dim, 0.f, sn);
            if constexpr (Plan::kSharedZ) {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) add_sum(kZ, k, d[k], x.pair(k));
            } else {
                float* const z = part + 2 * static_cast<size_t>(dim);
                Values<float, S> old;
                old.load(z, j, dim);
                store_row<S>(z, j, dim, [&](int k) { return fma2(d[k], x.pair(k), old.pair(k)); });
            }
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(sn[k], d[k]);
        } else {
#pragma unroll
            for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(both(p.scale), d[k]);
        }
        if (more) load_x(S::kRows);
        store_row<S>(at(static_cast<R*>(p.d_x), dim_bytes<R>(dim), 0), j, dim, [&](int k) { return sn[k]; });
        if (p.y) {
            bring(0);
            Pair sum = both(0.f);
            if (row_gate) {
                with_activation(p.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < S::HALF; ++k) {
                        Pair value, slope;
                        activation_with_slope<kExactGates<R>>(act, g.pair(k), value, slope);
                        const Pair yn = mul2(y.pair(k), both(ry)), w = factor(0, k);
                        sn[k] = mul2(mul2(mul2(d[k], yn), w), slope);  // dgate
                        d[k] = mul2(d[k], value);                      // dn
                        add_sum(kP, k, d[k], yn);
                        d[k] = mul2(d[k], w);
                        sum = fma2(d[k], yn, sum);
                    }
                });
                store_row<S>(at(static_cast<T*>(p.d_gate), dim_bytes<T>(dim), 0), j, dim, [&](int k) { return sn[k]; });
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) sn[k] = mul2(y.pair(k), both(ry));
            } else {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k) {
                    sn[k] = mul2(y.pair(k), both(ry));
                    add_sum(kP, k, d[k], sn[k]);
                    d[k] = mul2(d[k], factor(0, k));
                    sum = fma2(d[k], sn[k], sum);
                }
            }
            if (p.post_norm) {
                const Through through(p, row_sum<S>(sum_of(sum), words, 2 + slot) * inv_dim, ry);
#pragma unroll
                for (int k = 0; k < S::HALF; ++k)
                    d[k] = mul2(fma2(sn[k], both(through.m), d[k]), both(through.r));
            }
            store_row<S>(at(static_cast<T*>(p.d_y), dim_bytes<T>(dim), 0), j, dim, [&](int k) { return d[k]; });
        }
        y = y_next;
        g = g_next;
        ry = next_ry;
        rs = next_rs;
    }
    // The CTA's sums; rows side by side in a CTA are added first, in shared memory.
    auto write = [&](int which, float* dst) {
        const bool in_registers = Plan::kHeldSums && which != kZ;
        float2* const place = mine + (which == kZ ? Plan::kPlaceZ : in_registers ? 0 : which) * S::HALF * S::kThreads;
        Pair v[S::HALF];
        if constexpr (S::kRows > 1) {
            __syncthreads();
            if (in_registers) {
#pragma unroll
                for (int k = 0; k < S::HALF; ++k)
                    place[k * S::kThreads] = floats(sums[Plan::kHeldSums ? which & 1 : 0][Plan::kHeldSums ? k : 0]);
                __syncthreads();
            }
            if (sub > 0) return;
        }
#pragma unroll
        for (int k = 0; k < S::HALF; ++k) {
            if (in_registers && S::kRows == 1) {
                v[k] = sums[Plan::kHeldSums ? which & 1 : 0][Plan::kHeldSums ? k : 0];
            } else {
                v[k] = both(0.f);
                for (int o = 0; o < S::kRows; ++o) {
                    const float2 f = place[k * S::kThreads + o * S::TPR];
                    v[k] = add2(v[k], f32x2::pk(f.x, f.y));
                }
            }
        }
        store_row<S>(dst, j, dim, [&](int k) { return v[k]; });
    };
    if (Plan::kSharedZ && p.need_z) write(kZ, part + 2 * static_cast<size_t>(dim));
    if (p.need_p) write(kP, part);
    if (p.need_q) write(kQ, part + dim);
}

// The gradients of the per-channel vectors from the CTAs' sums, added in a
// fixed order: 32 columns per CTA, four a thread, in 32 slices of the parts.
// CTAs of `what`: 0 Q -> d_pre, 1 Z -> d_scale, 2 P -> d_post, and the gate's
// gradient where one gate row serves all; 3 + g that of group g.
template <typename T>
__global__ void __launch_bounds__(256) block_norm_sums_kernel(BlockNormArgs p, int parts) {
    __shared__ float slice[32][36];
    pdl_begin();
    const unsigned blocks = static_cast<unsigned>(p.dim + 31) / 32, what = blockIdx.x / blocks;
    const int c0 = static_cast<int>(blockIdx.x % blocks) * 32;
    if ((what == 0 && !p.need_q) || (what == 1 && !p.need_z) || (what >= 2 && !p.need_p)) return;
    const int quad = threadIdx.x & 7, part = threadIdx.x >> 3;
    const int col = c0 + 4 * quad;
    const bool grouped = p.gate_mode == kGateGroups;
    auto activated = [&](float g) { return activation<true>(p.act, g); };
    auto vector_at = [&](const void* v, bool is32, size_t at) {
        return is32 || sizeof(T) == 4 ? static_cast<const float*>(v)[at]
                                      : Convert<T, float>::load(static_cast<const T*>(v)[at]);
    };
    const float* src = p.partials + (what == 0 ? 1 : what == 1 ? 2 : 0) * static_cast<size_t>(p.dim) + col;
    const int first = what > 2 ? static_cast<int>(what - 3) * p.parts_per_group : 0;
    const int last = what > 2 ? first + p.parts_per_group : parts;
    const size_t step = 3 * static_cast<size_t>(p.dim);
    const bool vec = p.dim % 4 == 0;  // the workspace is 16-byte aligned
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int k, float4& to) {
        const float* q = src + k * step;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (vec) {
            if (col < p.dim) v = __ldcg(reinterpret_cast<const float4*>(q));
        } else {
            if (col < p.dim) v.x = q[0];
            if (col + 1 < p.dim) v.y = q[1];
            if (col + 2 < p.dim) v.z = q[2];
            if (col + 3 < p.dim) v.w = q[3];
        }
        if (what == 2 && grouped) {  // d_post: each group's own gate
            const size_t g = static_cast<size_t>(k / p.parts_per_group) * p.gate_row;
            if (col < p.dim) v.x *= activated(vector_at(p.gate, p.gate32, g + col));
            if (col + 1 < p.dim) v.y *= activated(vector_at(p.gate, p.gate32, g + col + 1));
            if (col + 2 < p.dim) v.z *= activated(vector_at(p.gate, p.gate32, g + col + 2));
            if (col + 3 < p.dim) v.w *= activated(vector_at(p.gate, p.gate32, g + col + 3));
        }
        to.x += v.x;
        to.y += v.y;
        to.z += v.z;
        to.w += v.w;
    };
    float4 other = sum;
    int k = first + part;
#pragma unroll 2
    for (; k + 32 < last; k += 64) {
        add(k, sum);
        add(k + 32, other);
    }
    if (k < last) add(k, sum);
    *reinterpret_cast<float4*>(&slice[part][4 * quad]) =
        make_float4(sum.x + other.x, sum.y + other.y, sum.z + other.z, sum.w + other.w);
    __syncthreads();
    const int lane = threadIdx.x, c = c0 + lane;
    if (lane >= 32 || c >= p.dim) return;
    float total = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) total += slice[q][lane];
    auto write = [&](void* out, bool is32, size_t at, float v) {
        if (!out) return;
        if (is32 || sizeof(T) == 4)
            static_cast<float*>(out)[at] = v;
        else
            static_cast<T*>(out)[at] = Convert<T, float>::store(v);
    };
    if (what == 0) return write(p.d_pre, p.pre32, c, total);
    if (what == 1) return write(p.d_scale, p.scales32, c, total);
    const bool channel = p.gate_mode == kGateChannel;
    if (channel || what > 2) {
        const size_t row = what > 2 ? what - 3 : 0;
        const float g = vector_at(p.gate, p.gate32, row * p.gate_row + c);
        const float w = p.post ? vector_at(p.post, p.post32, c) : 1.f;
        const float slope = p.act == 0 ? 1.f : from_sigmoid<true>(p.act, g, floats(sigmoid<true>(both(g))).x);
        write(p.d_gate, p.gate32, row * p.dim + c, total * w * slope);
        if (channel) total *= activated(g);
    }
    if (what == 2) write(p.d_post, p.post32, c, total);
}

}  // namespace cubf::norm
