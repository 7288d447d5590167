// gated_scan.cuh -- the gated linear recurrence of recurrent language models,
// forward, backward and one token at a time.
//
// Per channel, along the tokens of a sequence, with gate inputs r and i,
// la = -c softplus(Lambda) sigmoid(r) and a = exp(la):
//   h_t = a_t h_{t-1} + u_t,   u_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t.
// A run of tokens is the affine map h -> A h + H (A the product of its a, H
// its last h from h = 0), and runs join by (A1, H1) . (A2, H2) =
// (A1 A2, A2 H1 + H2), so time is split three ways: a thread runs kSteps
// tokens of two channels in registers, the kWarps warps of a CTA join their
// maps through shared memory, and the CTAs of a cluster, which hold
// consecutive tiles of the same channels, join theirs through distributed
// shared memory; the cluster then walks along the sequence.  Every input is
// read once, every output written once, and no CTA waits on one outside its
// cluster.
#pragma once

#include "block_ops.hpp"
#include "common.cuh"

namespace cubf::scan {

constexpr int kSteps = 8;                  // tokens per thread and tile
constexpr int kWarps = 8;                  // warps per CTA, consecutive in time
constexpr int kTile = kSteps * kWarps;     // tokens per CTA tile
constexpr int kChannels = 64;              // channels per CTA, two per lane
static_assert(kTile == kGatedScanChunk, "the backward kernel restarts from the forward's chunk states");

// Two channels of one token as loaded: 16-bit pairs in a word, fp32 in two.
template <typename T>
struct Raw {
    using Word = uint32_t;
    static CUBF_DEV Word zero() { return 0u; }
    static CUBF_DEV Word vec(const T* p) { return __ldcs(reinterpret_cast<const unsigned int*>(p)); }
    static CUBF_DEV Word two(const T* p, bool ok0, bool ok1) {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        const uint32_t lo = ok0 ? __ldcs(q) : 0u, hi = ok1 ? __ldcs(q + 32) : 0u;
        return lo | (hi << 16);
    }
    static CUBF_DEV float2 get(Word w) {
        T v[2];
        memcpy(v, &w, 4);
        return make_float2(Convert<T, float>::load(v[0]), Convert<T, float>::load(v[1]));
    }
    static CUBF_DEV Word put(float2 f) {
        const T v[2] = {Convert<T, float>::store(f.x), Convert<T, float>::store(f.y)};
        Word w;
        memcpy(&w, v, 4);
        return w;
    }
    static CUBF_DEV void store_vec(T* p, float2 f) { __stcs(reinterpret_cast<unsigned int*>(p), put(f)); }
};
template <>
struct Raw<float> {
    using Word = float2;
    static CUBF_DEV Word zero() { return make_float2(0.f, 0.f); }
    static CUBF_DEV Word vec(const float* p) { return __ldcs(reinterpret_cast<const float2*>(p)); }
    static CUBF_DEV Word two(const float* p, bool ok0, bool ok1) {
        return make_float2(ok0 ? __ldcs(p) : 0.f, ok1 ? __ldcs(p + 32) : 0.f);
    }
    static CUBF_DEV float2 get(Word w) { return w; }
    static CUBF_DEV void store_vec(float* p, float2 f) { __stcs(reinterpret_cast<float2*>(p), f); }
};

// The lane's two channels: adjacent where every row is aligned for pair
// accesses (VEC), else 32 apart, so that scalar accesses still coalesce.
template <bool VEC>
struct Lane {
    int ch;
    bool ok0, ok1;
    CUBF_DEV Lane(int c0, int lane, int dim) {
        ch = c0 + (VEC ? 2 * lane : lane);
        ok0 = ch < dim;
        ok1 = VEC ? ok0 : ch + 32 < dim;
    }
    template <typename T>
    CUBF_DEV typename Raw<T>::Word load(const T* row) const {
        if constexpr (VEC)
            return ok0 ? Raw<T>::vec(row + ch) : Raw<T>::zero();
        else
            return Raw<T>::two(row + ch, ok0, ok1);
    }
    template <typename T>
    CUBF_DEV void store(T* row, float2 f) const {
        if constexpr (VEC) {
            if (ok0) Raw<T>::store_vec(row + ch, f);
        } else {
            if (ok0) row[ch] = Convert<T, float>::store(f.x);
            if (ok1) row[ch + 32] = Convert<T, float>::store(f.y);
        }
    }
    CUBF_DEV float2 load32(const float* row) const {
        return make_float2(ok0 ? row[ch] : 0.f, ok1 ? row[ch + (VEC ? 1 : 32)] : 0.f);
    }
    CUBF_DEV void store32(float* row, float2 f) const {
        if (ok0) row[ch] = f.x;
        if (ok1) row[ch + (VEC ? 1 : 32)] = f.y;
    }
};

CUBF_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
CUBF_DEV float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
CUBF_DEV float rsq(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f;

CUBF_DEV float sigmoid(float v) { return rcp(1.f + ex2(-kLog2e * v)); }

// c softplus(Lambda) log2(e): la in units of log2 is -rate sigmoid(r).
CUBF_DEV float softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }
CUBF_DEV float rate_of(float lambda, float exponent) { return exponent * softplus(lambda) * kLog2e; }

// 1 - a^2 = 1 - 2^(2 w) for w = log2(a) <= 0.  Near a = 1 the difference
// cancels, so for 2 la = 2 ln(2) w > -1/8 the series of -(e^z - 1) is used
// (five terms; the next is z^5/720 < 5e-8 of the sum); beyond it 1 - a^2 is
// at least 0.117, and a's rounding costs under 3e-6 of it.
CUBF_DEV float one_minus_square(float w, float a) {
    constexpr float z = 1.3862943611198906f;  // 2 ln 2
    constexpr float c1 = z, c2 = z * z / 2, c3 = z * z * z / 6, c4 = z * z * z * z / 24, c5 = z * z * z * z * z / 120;
    const float series = -w * (c1 + w * (c2 + w * (c3 + w * (c4 + w * c5))));
    return w > -0.09f ? series : 1.f - a * a;
}

// One token of one channel, from its gate inputs.
struct Coefficients {
    float sr, si;  // the gates
    float w;       // log2(a)
    float a;
    float m;       // sqrt(1 - a^2)
};
constexpr float kSmallestNormal = 1.1754944e-38f;
CUBF_DEV Coefficients coefficients(float rate, float r, float i) {
    Coefficients c;
    c.sr = sigmoid(r);
    c.si = sigmoid(i);
    c.w = -rate * c.sr;
    c.a = ex2(c.w);
    const float m2 = one_minus_square(c.w, c.a);
    // a shut gate (a = 1) keeps h as it is; NaN passes
    c.m = m2 >= kSmallestNormal ? m2 * rsq(m2) : m2;
    return c;
}

// In packed batches a run that holds a sequence's first token forgets what
// came before it whatever that was (a product with zero would keep its NaN):
// its A is the marker -0, which no product of decays (all >= +0) produces.
template <bool PACKED>
CUBF_DEV float through(float a, float h, float carry) {
    if (PACKED && __float_as_uint(a) == 0x80000000u) return h;
    return fmaf(a, carry, h);
}
template <bool PACKED>
CUBF_DEV float product(float first, float second) {
    if (PACKED && __float_as_uint(second) == 0x80000000u) return second;
    if (PACKED && __float_as_uint(first) == 0x80000000u) return first;
    return first * second;
}
CUBF_DEV float marker() { return __uint_as_float(0x80000000u); }

// Walks the sequences of a packed batch along increasing tokens.
struct Walker {
    const int* offsets;
    int last;  // sequences - 1
    int at;    // the sequence of the current token
    int start, stop;
    CUBF_DEV void init(const int* o, int sequences) {
        offsets = o;
        last = sequences - 1;
        at = 0;
        start = o[0];
        stop = o[1];
    }
    // Moves to the last sequence that starts at or before token t (doubling
    // steps, then halving: the next sequence in one comparison, far ones in
    // logarithmic time).  Offsets are read within [0, sequences] only,
    // whatever they hold.
    CUBF_DEV void seek(int t) {
        if (t < stop || at >= last) return;
        int lo = at, step = 1;
        while (lo + step <= last && offsets[lo + step] <= t) {
            lo += step;
            step <<= 1;
        }
        for (; step > 0; step >>= 1)
            if (lo + step <= last && offsets[lo + step] <= t) lo += step;
        at = lo;
        start = offsets[lo];
        stop = offsets[lo + 1];
    }
    CUBF_DEV void rewind() {
        at = 0;
        start = offsets[0];
        stop = offsets[1];
    }
};

CUBF_DEV uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
CUBF_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
CUBF_DEV void store_remote(const void* local, uint32_t rank, float4 v) {
    const uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(local));
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z),
                 "f"(v.w)
                 : "memory");
}

// {A, A, H, H} of the lane's two channels.
struct Maps {
    float4 warp[2][kWarps][32];
    float4 cta[2][kGatedScanMaxCluster][32];
};

// ---- forward -----------------------------------------------------------------------------------
template <typename T, bool PACKED, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, 2) gated_scan_kernel(GatedScanArgs p, int cluster, int tiles) {
    __shared__ Maps maps;
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const unsigned column = blockIdx.x / cluster;
    const Lane<VEC> ln(static_cast<int>(column % tiles) * kChannels, lane, p.dim);
    const size_t b = column / tiles;
    const T* x = static_cast<const T*>(p.x) + b * p.x_batch;
    const T* r = static_cast<const T*>(p.r) + b * p.r_batch;
    const T* g = static_cast<const T*>(p.i) + b * p.i_batch;
    T* out = static_cast<T*>(p.h) + b * static_cast<size_t>(p.length) * p.dim;
    const float2 lambda = ln.load32(p.decay);
    const float2 rate = make_float2(rate_of(lambda.x, p.exponent), rate_of(lambda.y, p.exponent));
    const int stride = cluster * kTile;
    int t0 = rank * kTile + warp * kSteps;

    typename Raw<T>::Word rx[kSteps], rr[kSteps], ri[kSteps];
    auto load = [&](int t) {
        const T *px = x + static_cast<size_t>(t) * p.x_token, *pr = r + static_cast<size_t>(t) * p.r_token,
                *pi = g + static_cast<size_t>(t) * p.i_token;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const bool in = t + s < p.length;
            rx[s] = in ? ln.load(px) : Raw<T>::zero();
            rr[s] = in ? ln.load(pr) : Raw<T>::zero();
            ri[s] = in ? ln.load(pi) : Raw<T>::zero();
            px += p.x_token;
            pr += p.r_token;
            pi += p.i_token;
        }
    };
    load(t0);

    Walker seq;
    if constexpr (PACKED) seq.init(p.offsets, p.sequences);
    if constexpr (PACKED) {  // sequences without tokens end where they began
        if (rank == 0)
            for (int j = warp; j < p.sequences; j += kWarps)
                if (p.offsets[j] >= p.offsets[j + 1])
                    ln.store32(p.last + static_cast<size_t>(j) * p.dim,
                               p.initial ? ln.load32(p.initial + static_cast<size_t>(j) * p.dim)
                                         : make_float2(0.f, 0.f));
    }
    float2 carry = make_float2(0.f, 0.f);  // h before the cluster's tiles
    if (!PACKED && p.initial) carry = ln.load32(p.initial + b * p.dim);

    const int rounds = (p.length + stride - 1) / stride;
    for (int round = 0; round < rounds; ++round, t0 += stride) {
        const int buf = round & 1;
        float2 a[kSteps], u[kSteps];
        float2 A = make_float2(1.f, 1.f), H = make_float2(0.f, 0.f);
        unsigned starts = 0;
        if constexpr (PACKED) seq.seek(t0);
        Walker from = seq;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (t0 + s < p.length) {
                const float2 fx = Raw<T>::get(rx[s]), fr = Raw<T>::get(rr[s]), fi = Raw<T>::get(ri[s]);
                const Coefficients c0 = coefficients(rate.x, fr.x, fi.x), c1 = coefficients(rate.y, fr.y, fi.y);
                a[s] = make_float2(c0.a, c1.a);
                u[s] = make_float2(c0.m * c0.si * fx.x, c1.m * c1.si * fx.y);
                bool first = false;
                if constexpr (PACKED) {
                    seq.seek(t0 + s);
                    first = t0 + s == seq.start;
                }
                if (PACKED && first) {
                    starts |= 1u << s;
                    if (p.initial) {
                        const float2 h0 = ln.load32(p.initial + static_cast<size_t>(seq.at) * p.dim);
                        u[s].x = fmaf(a[s].x, h0.x, u[s].x);
                        u[s].y = fmaf(a[s].y, h0.y, u[s].y);
                    }
                    A = make_float2(marker(), marker());
                    H = u[s];
                } else {
                    A.x = product<PACKED>(A.x, a[s].x);
                    A.y = product<PACKED>(A.y, a[s].y);
                    H.x = fmaf(a[s].x, H.x, u[s].x);
                    H.y = fmaf(a[s].y, H.y, u[s].y);
                }
            } else {
                a[s] = make_float2(1.f, 1.f);
                u[s] = make_float2(0.f, 0.f);
            }
        }
        if (round + 1 < rounds) load(t0 + stride);  // in flight while the maps are joined and h is written
        maps.warp[buf][warp][lane] = make_float4(A.x, A.y, H.x, H.y);
        __syncthreads();
        // the CTA's map, and the map of the warps before this one
        float2 preA = make_float2(1.f, 1.f), preH = make_float2(0.f, 0.f), totA = preA, totH = preH;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            if (k == warp) {
                preA = totA;
                preH = totH;
            }
            const float4 m = maps.warp[buf][k][lane];
            totH.x = through<PACKED>(m.x, m.z, totH.x);
            totH.y = through<PACKED>(m.y, m.w, totH.y);
            totA.x = product<PACKED>(totA.x, m.x);
            totA.y = product<PACKED>(totA.y, m.y);
        }
        float2 in = carry;  // h before this CTA's tile
        if (cluster == 1) {
            carry.x = through<PACKED>(totA.x, totH.x, carry.x);
            carry.y = through<PACKED>(totA.y, totH.y, carry.y);
        } else {
            for (int k = warp; k < cluster; k += kWarps)
                store_remote(&maps.cta[buf][rank][lane], k, make_float4(totA.x, totA.y, totH.x, totH.y));
            cluster_sync();
            for (int k = 0; k < cluster; ++k) {
                if (k == rank) in = carry;
                const float4 m = maps.cta[buf][k][lane];
                carry.x = through<PACKED>(m.x, m.z, carry.x);
                carry.y = through<PACKED>(m.y, m.w, carry.y);
            }
        }
        float2 h;
        h.x = through<PACKED>(preA.x, preH.x, in.x);
        h.y = through<PACKED>(preA.y, preH.y, in.y);
        if (p.chunk_states && warp == 0 && t0 < p.length)
            ln.store32(p.chunk_states +
                           (b * ((p.length + kTile - 1) / kTile) + static_cast<size_t>(t0 / kTile)) * p.dim,
                       h);
        T* po = out + static_cast<size_t>(t0) * p.dim;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (t0 + s < p.length) {
                if (PACKED && ((starts >> s) & 1u)) {
                    h = u[s];
                } else {
                    h.x = fmaf(a[s].x, h.x, u[s].x);
                    h.y = fmaf(a[s].y, h.y, u[s].y);
                }
                ln.store(po, h);
                if constexpr (PACKED) {
                    from.seek(t0 + s);
                    if (t0 + s + 1 == from.stop) ln.store32(p.last + static_cast<size_t>(from.at) * p.dim, h);
                }
            }
            po += p.dim;
        }
    }
    if (!PACKED && rank == 0 && warp == 0) ln.store32(p.last + b * p.dim, carry);
    if (cluster > 1) cluster_sync();  // no CTA leaves while another may still store into it
}

// ---- backward ----------------------------------------------------------------------------------
// G_t = dh_t + P_{t+1}, P_t = a_t G_t runs from the end of time by the same
// joins; h_{t-1} is run again from the chunk state the forward kept, in fp32,
// instead of read back in the outputs' type.
struct BackMaps {
    float4 warp[2][kWarps][32];  // {A, A, H, H}
    float2 back[2][kWarps][32];  // P out of the warp's tokens from P = 0 after them
    float4 cta[2][kGatedScanMaxCluster][32];
    float2 sum[kWarps][32];
};

template <typename T, bool PACKED, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, 2) gated_scan_backward_kernel(GatedScanArgs p, int cluster, int tiles) {
    __shared__ BackMaps maps;
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const unsigned column = blockIdx.x / cluster;
    const Lane<VEC> ln(static_cast<int>(column % tiles) * kChannels, lane, p.dim);
    const size_t b = column / tiles;
    const T* x = static_cast<const T*>(p.x) + b * p.x_batch;
    const T* r = static_cast<const T*>(p.r) + b * p.r_batch;
    const T* g = static_cast<const T*>(p.i) + b * p.i_batch;
    const T* dh = static_cast<const T*>(p.d_h) + b * p.dh_batch;
    const size_t out = b * static_cast<size_t>(p.length) * p.dim;
    T* dx = static_cast<T*>(p.d_x) + out;
    T* dr = static_cast<T*>(p.d_r) + out;
    T* di = static_cast<T*>(p.d_i) + out;
    const float2 lambda = ln.load32(p.decay);
    const float2 rate = make_float2(rate_of(lambda.x, p.exponent), rate_of(lambda.y, p.exponent));
    const int stride = cluster * kTile;
    const int chunks = (p.length + kTile - 1) / kTile;
    const int rounds = (p.length + stride - 1) / stride;

    if constexpr (PACKED) {  // sequences without tokens pass their gradient through
        if (p.d_initial && rank == 0)
            for (int j = warp; j < p.sequences; j += kWarps)
                if (p.offsets[j] >= p.offsets[j + 1])
                    ln.store32(p.d_initial + static_cast<size_t>(j) * p.dim,
                               p.d_last ? ln.load32(p.d_last + static_cast<size_t>(j) * p.dim)
                                        : make_float2(0.f, 0.f));
    }
    Walker seq;
    if constexpr (PACKED) seq.init(p.offsets, p.sequences);
    float2 carry = make_float2(0.f, 0.f);  // P from the tokens after the cluster's tiles
    if (!PACKED && p.d_last) carry = ln.load32(p.d_last + b * p.dim);
    float2 sum = make_float2(0.f, 0.f);    // of e, for the gradient of Lambda

    for (int round = rounds - 1; round >= 0; --round) {
        const int buf = round & 1;
        const int t0 = round * stride + rank * kTile + warp * kSteps;
        typename Raw<T>::Word rx[kSteps], rd[kSteps];
        float2 a[kSteps], m[kSteps], sr[kSteps], si[kSteps];
        {
            typename Raw<T>::Word rr[kSteps], ri[kSteps];
            const T *px = x + static_cast<size_t>(t0) * p.x_token, *pr = r + static_cast<size_t>(t0) * p.r_token,
                    *pi = g + static_cast<size_t>(t0) * p.i_token, *pd = dh + static_cast<size_t>(t0) * p.dh_token;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const bool in = t0 + s < p.length;
                rx[s] = in ? ln.load(px) : Raw<T>::zero();
                rr[s] = in ? ln.load(pr) : Raw<T>::zero();
                ri[s] = in ? ln.load(pi) : Raw<T>::zero();
                rd[s] = in ? ln.load(pd) : Raw<T>::zero();
                px += p.x_token;
                pr += p.r_token;
                pi += p.i_token;
                pd += p.dh_token;
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const float2 fr = Raw<T>::get(rr[s]), fi = Raw<T>::get(ri[s]);
                const Coefficients c0 = coefficients(rate.x, fr.x, fi.x), c1 = coefficients(rate.y, fr.y, fi.y);
                a[s] = make_float2(c0.a, c1.a);
                m[s] = make_float2(c0.m, c1.m);
                sr[s] = make_float2(c0.sr, c1.sr);
                si[s] = make_float2(c0.si, c1.si);
            }
        }
        float2 h = make_float2(0.f, 0.f);  // before the tile, from the forward
        const int chunk = round * cluster + rank;
        if (chunk < chunks) h = ln.load32(p.chunk_states + (b * chunks + chunk) * static_cast<size_t>(p.dim));

        // the maps of the warp's tokens
        unsigned starts = 0, ends = 0;
        float2 A = make_float2(1.f, 1.f), H = make_float2(0.f, 0.f);
        Walker from;
        if constexpr (PACKED) {
            seq.rewind();
            seq.seek(t0);
            from = seq;
        }
        // the token's u, with the sequence's initial state where it begins one
        auto drive = [&](int s, const Walker& w, bool first) {
            const float2 fx = Raw<T>::get(rx[s]);
            float2 u = make_float2(m[s].x * si[s].x * fx.x, m[s].y * si[s].y * fx.y);
            if (PACKED && first && p.initial) {
                const float2 h0 = ln.load32(p.initial + static_cast<size_t>(w.at) * p.dim);
                u.x = fmaf(a[s].x, h0.x, u.x);
                u.y = fmaf(a[s].y, h0.y, u.y);
            }
            return u;
        };
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (t0 + s >= p.length) continue;
            bool first = false;
            if constexpr (PACKED) {
                seq.seek(t0 + s);
                first = t0 + s == seq.start;
                if (t0 + s + 1 == seq.stop) ends |= 1u << s;
            }
            const float2 u = drive(s, seq, first);
            if (PACKED && first) {
                starts |= 1u << s;
                A = make_float2(marker(), marker());
                H = u;
            } else {
                A.x = product<PACKED>(A.x, a[s].x);
                A.y = product<PACKED>(A.y, a[s].y);
                H.x = fmaf(a[s].x, H.x, u.x);
                H.y = fmaf(a[s].y, H.y, u.y);
            }
        }
        // dh with the final states' gradients where a sequence ends
        auto arriving = [&](int s, int at) {
            float2 d = Raw<T>::get(rd[s]);
            if (PACKED && ((ends >> s) & 1u) && p.d_last) {
                const float2 l = ln.load32(p.d_last + static_cast<size_t>(at) * p.dim);
                d.x += l.x;
                d.y += l.y;
            }
            return d;
        };
        float2 R = make_float2(0.f, 0.f);
        int at = PACKED ? seq.at : 0;
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            if (t0 + s >= p.length) continue;
            const float2 d = arriving(s, at);
            R.x = a[s].x * (d.x + R.x);
            R.y = a[s].y * (d.y + R.y);
            if (PACKED && ((starts >> s) & 1u)) {
                R = make_float2(0.f, 0.f);
                // the token before belongs to the last sequence with tokens before this one
                while (at > 0 && p.offsets[at] > t0 + s - 1) --at;
            }
        }
        maps.warp[buf][warp][lane] = make_float4(A.x, A.y, H.x, H.y);
        maps.back[buf][warp][lane] = R;
        __syncthreads();
        float2 totA = make_float2(1.f, 1.f), totR = make_float2(0.f, 0.f), postA = totA, postR = totR;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            if (k >= warp) break;
            const float4 q = maps.warp[buf][k][lane];
            h.x = through<PACKED>(q.x, q.z, h.x);
            h.y = through<PACKED>(q.y, q.w, h.y);
        }
#pragma unroll
        for (int k = kWarps - 1; k >= 0; --k) {
            if (k == warp) {
                postA = totA;
                postR = totR;
            }
            const float4 q = maps.warp[buf][k][lane];
            const float2 back = maps.back[buf][k][lane];
            totR.x = through<PACKED>(q.x, back.x, totR.x);
            totR.y = through<PACKED>(q.y, back.y, totR.y);
            totA.x = product<PACKED>(totA.x, q.x);
            totA.y = product<PACKED>(totA.y, q.y);
        }
        float2 in = carry;  // P from the tokens after this CTA's tile
        if (cluster == 1) {
            carry.x = through<PACKED>(totA.x, totR.x, carry.x);
            carry.y = through<PACKED>(totA.y, totR.y, carry.y);
        } else {
            for (int k = warp; k < cluster; k += kWarps)
                store_remote(&maps.cta[buf][rank][lane], k, make_float4(totA.x, totA.y, totR.x, totR.y));
            cluster_sync();
            for (int k = cluster - 1; k >= 0; --k) {
                if (k == rank) in = carry;
                const float4 q = maps.cta[buf][k][lane];
                carry.x = through<PACKED>(q.x, q.z, carry.x);
                carry.y = through<PACKED>(q.y, q.w, carry.y);
            }
        }
        float2 P;
        P.x = through<PACKED>(postA.x, postR.x, in.x);
        P.y = through<PACKED>(postA.y, postR.y, in.y);

        // h before each token, then the gradients from the last token back
        float2 before[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            before[s] = h;
            if (t0 + s >= p.length) continue;
            const bool first = PACKED && ((starts >> s) & 1u);
            if constexpr (PACKED) {
                from.seek(t0 + s);
                if (first)
                    before[s] = p.initial ? ln.load32(p.initial + static_cast<size_t>(from.at) * p.dim)
                                          : make_float2(0.f, 0.f);
            }
            const float2 fx = Raw<T>::get(rx[s]);
            h.x = fmaf(a[s].x, before[s].x, m[s].x * si[s].x * fx.x);
            h.y = fmaf(a[s].y, before[s].y, m[s].y * si[s].y * fx.y);
        }
        at = PACKED ? seq.at : 0;
#pragma unroll
        for (int s = kSteps - 1; s >= 0; --s) {
            if (t0 + s >= p.length) continue;
            const float2 d = arriving(s, at);
            const float2 G = make_float2(d.x + P.x, d.y + P.y);
            const float2 fx = Raw<T>::get(rx[s]);
            float2 ox, orr, oi;
            auto channel = [&](float Gv, float av, float mv, float srv, float siv, float xv, float hv, float rt,
                               float& gx, float& gr, float& gi, float& total) {
                const float la = -0.6931471805599453f * rt * srv;
                const float gm = Gv * mv, gs = siv * xv;
                gx = gm * siv;
                gi = gm * gs * (1.f - siv);
                // d sqrt(1 - a^2)/d la = -a^2/m; times la it tends to 0 with la
                const float ratio = mv > 1e-18f ? -la * rcp(mv) : la;
                const float e = Gv * av * fmaf(hv, la, gs * av * ratio);
                gr = e * (1.f - srv);
                total += e;
            };
            channel(G.x, a[s].x, m[s].x, sr[s].x, si[s].x, fx.x, before[s].x, rate.x, ox.x, orr.x, oi.x, sum.x);
            channel(G.y, a[s].y, m[s].y, sr[s].y, si[s].y, fx.y, before[s].y, rate.y, ox.y, orr.y, oi.y, sum.y);
            const size_t o = static_cast<size_t>(t0 + s) * p.dim;
            ln.store(dx + o, ox);
            ln.store(dr + o, orr);
            ln.store(di + o, oi);
            P = make_float2(a[s].x * G.x, a[s].y * G.y);
            if (PACKED && ((starts >> s) & 1u)) {
                if (p.d_initial) ln.store32(p.d_initial + static_cast<size_t>(at) * p.dim, P);
                P = make_float2(0.f, 0.f);
                while (at > 0 && p.offsets[at] > t0 + s - 1) --at;
            }
        }
    }
    if (!PACKED && p.d_initial && rank == 0 && warp == 0) ln.store32(p.d_initial + b * p.dim, carry);
    maps.sum[warp][lane] = sum;
    __syncthreads();
    if (warp == 0) {
        for (int k = 1; k < kWarps; ++k) {
            sum.x += maps.sum[k][lane].x;
            sum.y += maps.sum[k][lane].y;
        }
        ln.store32(p.partials + (b * cluster + rank) * static_cast<size_t>(p.dim), sum);
    }
    if (cluster > 1) cluster_sync();
}

// dLambda = sigmoid(Lambda)/softplus(Lambda) sum e over the CTAs' partial sums
// (the ratio tends to 1 as both vanish).
__global__ void __launch_bounds__(256) gated_scan_decay_kernel(GatedScanArgs p, int parts) {
    __shared__ float slice[8][32];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ch = blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (ch < p.dim)
        for (int k = warp; k < parts; k += 8) sum += p.partials[static_cast<size_t>(k) * p.dim + ch];
    slice[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && ch < p.dim) {
        for (int k = 1; k < 8; ++k) sum += slice[k][lane];
        const float lambda = p.decay[ch];
        const float ratio = lambda < -15.f ? 1.f : 1.f / ((1.f + expf(-lambda)) * softplus(lambda));
        p.d_decay[ch] = sum * ratio;
    }
}

// ---- one token ---------------------------------------------------------------------------------
// A warp takes 64 channels of `rows` consecutive requests; a request whose
// slot lies outside the pool is padding: its output is zero and no state is
// touched.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) gated_scan_step_kernel(GatedStepArgs p, int tiles, int rows) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const unsigned task = blockIdx.x * 4 + (threadIdx.x >> 5);
    const Lane<VEC> ln(static_cast<int>(task % tiles) * kChannels, lane, p.dim);
    const size_t first = static_cast<size_t>(task / tiles) * rows;
    if (first >= p.batch) return;
    const size_t end = first + rows < p.batch ? first + rows : p.batch;
    const float2 lambda = ln.load32(p.decay);
    const float2 rate = make_float2(rate_of(lambda.x, p.exponent), rate_of(lambda.y, p.exponent));
#pragma unroll 4
    for (size_t b = first; b < end; ++b) {
        long long slot = static_cast<long long>(b);
        if (p.slots) slot = p.slots[b];
        T* h = static_cast<T*>(p.h) + b * p.dim;
        if (slot < 0 || slot >= static_cast<long long>(p.pool)) {
            ln.store(h, make_float2(0.f, 0.f));
            continue;
        }
        const float2 x = Raw<T>::get(ln.load(static_cast<const T*>(p.x) + b * p.x_row));
        const float2 r = Raw<T>::get(ln.load(static_cast<const T*>(p.r) + b * p.r_row));
        const float2 i = Raw<T>::get(ln.load(static_cast<const T*>(p.i) + b * p.i_row));
        const float2 s = ln.load32(p.state + static_cast<size_t>(slot) * p.dim);
        const Coefficients c0 = coefficients(rate.x, r.x, i.x), c1 = coefficients(rate.y, r.y, i.y);
        const float2 n = make_float2(fmaf(c0.a, s.x, c0.m * c0.si * x.x), fmaf(c1.a, s.y, c1.m * c1.si * x.y));
        ln.store(h, n);
        ln.store32(p.new_state + static_cast<size_t>(slot) * p.dim, n);
    }
}

}  // namespace cubf::scan
