// gated_delta.cuh -- the gated delta rule in chunks of 64 tokens.
//
// Per head, with a state S of K x V values:
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),  o_t = scale S_t^T q_t.
// In a chunk, with G the running sum of g, D_ij = e^{G_i - G_j} for j <= i and S the state before it:
//   M = strictly lower part of D o (k k^T),  P = scale lower part of D o (q k^T)
//   Y = v - e^G (k S),  R = (I + M beta)^-1 Y = Y - L (beta Y)  with  L = (I + M beta)^-1 M,  U = beta R
//   o = scale e^G (q S) + P U,   S' = e^{G_64} S + (e^{G_64 - G} k)^T U
// L is strictly lower and holds no beta by itself, so that the transposed system of the backward,
//   E = P^T dO + e^{G_64 - G} (k dS'),  W = E - L^T (beta E),  Z = beta W
//   dS = e^{G_64} dS' + (scale e^G q)^T dO - (e^G k)^T Z,
// takes the same L, and nothing is ever divided by beta.  From these
//   dv = Z,  dbeta = W . R,  dP = scale dO U^T,  dM = -Z U^T
//   dq = scale e^G (dO S^T) + (D o dP) k
//   dk = -e^G (Z S^T) + e^{G_64 - G} (U dS'^T) + (D o dP)^T q + (D o dM)^T k + (D o dM) k
//   dG = q . (first term of dq) + k . (first of dk) - k . (second of dk) + row sums - column sums of P o dP + M o dM,
//   dG_64 += sum of k . (second of dk) + e^{G_64} <S, dS'>,  dg = sums of dG from each token on.
//
// Four kernels.  `prepare` (a CTA per chunk and head) makes L, P and the decay
// factors.  `chain` runs along a sequence: a warp holds 16 columns of the
// state transposed, 16 x K fp32 values in registers, as accumulator fragments
// whose layout is that of the next product's A operand, so a chunk's three
// dependent products (S k, L Y, k U) need no exchange between warps and no
// shared memory but the tiles that all warps read.  The backward runs the
// forward chain again (keeping S and R of every chunk) beside the reversed
// chain, in one launch, then `gradients` (a CTA per chunk and head).
// All products are split ones (mma_split.cuh), accumulated in fp32.
#pragma once

#include <algorithm>

#include "gated_delta.hpp"
#include "mma_split.cuh"

namespace cubf::delta {

using namespace split;

constexpr int C = kDeltaChunk;
constexpr int kSquare = C * C;           // values of L or P
constexpr int kPitchC = C + 8;           // of 64-wide tiles
// Per chunk and head: e^G, e^{G_64 - G}, beta, and G as a sum of two floats
constexpr int kFactors = 5 * C;
constexpr float kLeast = -128.f;         // e^-128 is zero in fp32: a log decay below it is taken as it

template <typename T>
constexpr int kInput = std::is_same_v<T, float> ? 3 : std::is_same_v<T, __half> ? 2 : 1;  // exact pieces of an input
// Level of the products and pieces of their fp32 operands.  With 16-bit tensors 16 bits of an operand, each product's
// error 2^-16 at most and 3e-6 in the mean, stay far below one rounding of an output and below 1e-5 of the fp32 states,
// which are themselves held and added up in fp32; level 3 costs half as much again.
template <typename T>
constexpr int kLevel = std::is_same_v<T, float> ? 3 : 2;
// ... with q, k or dO as the other operand: fp16 ones bring both pieces to both of the state's.
template <typename T>
constexpr int kInputLevel = std::is_same_v<T, __nv_bfloat16> ? 2 : 3;

template <typename T>
CUBF_DEV float widen(T x) {
    return Convert<T, float>::load(x);
}
CUBF_DEV float gate_at(const HeadTensor& t, bool wide, size_t at, int type) {
    if (wide) return static_cast<const float*>(t.p)[at];
    return type == 0 ? __half2float(static_cast<const __half*>(t.p)[at])
                     : __bfloat162float(static_cast<const __nv_bfloat16*>(t.p)[at]);
}
template <typename T>
constexpr int kTypeId = std::is_same_v<T, __half> ? 0 : 1;

// ---- where things are ---------------------------------------------------------------------------
// Long sequences of few chains in segments (gated_delta_tc.cuh): of `length` chunks, 0 for none.
struct Segments {
    int length, total;
    size_t ends, d_ends, maps;           // in the workspace: states where segments end, gradients where they begin, A
};

struct Places {                          // of the workspace, in bytes from its start
    size_t factors, solve, attention, packed, values, rows, states, d_states, errors, d_writes, d_q, d_k, total;
    size_t state_piece, squares;         // bytes of a piece of a kept state, of a chunk's matrices (gated_delta_tc.cuh)
    int slots, v_pitch, v_rows;          // v_dim rounded up to 16, to 64
    Segments segments;
};

struct Span {                            // a chunk
    int sequence, chunk, first, tokens;  // first: token of the batch row
    int row;                             // batch row
};

__host__ CUBF_DEV int slot_base(const GatedDeltaArgs& a, int j, int start) {
    return a.offsets ? start / C + j : j * ((a.length + C - 1) / C);
}
// Offsets outside 0 .. length are taken as the nearest value inside.
CUBF_DEV int offset_at(const GatedDeltaArgs& a, int j) { return min(max(a.offsets[j], 0), a.length); }

// The chunk at a place; tokens = 0 where no sequence uses it.
CUBF_DEV Span span_of(const GatedDeltaArgs& a, int slot) {
    Span s{};
    if (!a.offsets) {
        const int per = (a.length + C - 1) / C;
        s.row = s.sequence = slot / per;
        s.chunk = slot % per;
        s.first = s.chunk * C;
        s.tokens = min(C, a.length - s.first);
        return s;
    }
    int low = 0, high = a.sequences;     // the last sequence whose places begin at or before `slot`
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (offset_at(a, mid) / C + mid <= slot)
            low = mid;
        else
            high = mid;
    }
    const int start = offset_at(a, low), end = offset_at(a, low + 1);
    s.sequence = low;
    s.chunk = slot - (start / C + low);
    s.first = start + s.chunk * C;
    s.tokens = s.chunk < 0 ? 0 : min(C, max(0, end - s.first));
    return s;
}

// ---- q and k of a chunk as bf16 pieces ----------------------------------------------------------
template <typename T, int KP>
CUBF_DEV const __nv_bfloat16* packed_at(const GatedDeltaArgs& a, const Places& w, int which, int slot, int head) {
    const size_t tile = (static_cast<size_t>(slot) * a.k_heads + head) * 2 + which;
    return reinterpret_cast<const __nv_bfloat16*>(static_cast<const char*>(a.workspace) + w.packed) + tile * kInput<T> * C * KP;
}
template <int NI, int KP>
CUBF_DEV void load_packed(const __nv_bfloat16* p, uint32_t tile, int tid, int threads) {
    for (int e = tid; e < NI * C * (KP / 8); e += threads) {
        const int row = e / (KP / 8), col = e % (KP / 8) * 8;  // rows of all pieces
        copy16(tile + static_cast<uint32_t>(row * (KP + 8) + col) * 2u, p + static_cast<size_t>(e) * 8, true);
    }
}
// N pieces of 64 x 64
CUBF_DEV void load_squares(const __nv_bfloat16* p, int n, uint32_t tile, int tid, int threads) {
    for (int e = tid; e < n * kSquare / 8; e += threads) {
        const int row = e / (C / 8), col = e % (C / 8) * 8;  // rows of all pieces
        copy16(tile + static_cast<uint32_t>(row * kPitchC + col) * 2u, p + static_cast<size_t>(e) * 8, true);
    }
}

template <typename T>
constexpr int kSpare = 16 / static_cast<int>(sizeof(T));  // values between rows of a tile of T
// Rows of v or dO: `width` channels from `from` on, zeros behind the last token or channel.
template <typename T>
CUBF_DEV void load_rows(const T* p, size_t row, int rows, int cols, int from, int width, bool wide, T* tile, int tid,
                        int threads) {
    constexpr int N = 16 / sizeof(T);
    const int pitch = width + kSpare<T>;
    if (wide) {
        const int per = width / N;
        for (int e = tid; e < C * per; e += threads) {
            const int r = e / per, c = e % per * N;
            const bool ok = r < rows && from + c < cols;
            copy16(smem_addr(tile + r * pitch + c), p + (ok ? r * row + from + c : 0), ok);
        }
    } else {
        for (int e = tid; e < C * width; e += threads) {
            const int r = e / width, c = e % width;
            tile[r * pitch + c] = r < rows && from + c < cols ? p[r * row + from + c] : Convert<T, float>::store(0.f);
        }
    }
}

// ---- prepare ------------------------------------------------------------------------------------
// Bounded by the substitution: 64 columns of L, a thread each, 2016 FMAs with M read as 16-byte broadcasts.
template <typename T, int KP>
struct PrepareShared {
    static constexpr int NI = kInput<T>;
    static constexpr int kTile = NI * C * (KP + 8);
    alignas(16) __nv_bfloat16 q[kTile];
    alignas(16) __nv_bfloat16 k[kTile];
    alignas(16) float m[C][C];           // M beta
    float unit[C][C + 1];                // M
    double sum[C];
    float beta[C];
};

template <typename T, int KP>
CUBF_DEV void pack_rows(const GatedDeltaArgs& a, const HeadTensor& t, const Span& s, int head, __nv_bfloat16* tile,
                        __nv_bfloat16* copy, int tid) {
    constexpr int NI = kInput<T>;
    const T* p = static_cast<const T*>(t.p) + s.row * t.batch + static_cast<size_t>(s.first) * t.token +
                 static_cast<size_t>(head) * t.head;
    for (int e = tid; e < C * KP / 2; e += 128) {
        const int row = e / (KP / 2), col = e % (KP / 2) * 2;
        float x = 0.f, y = 0.f;
        if (row < s.tokens) {
            const T* r = p + static_cast<size_t>(row) * t.token;
            if (col < a.k_dim) x = widen(r[col]);
            if (col + 1 < a.k_dim) y = widen(r[col + 1]);
        }
        uint32_t f[NI];
        pieces<NI>(x, y, f);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            *reinterpret_cast<uint32_t*>(tile + (i * C + row) * (KP + 8) + col) = f[i];
            if (copy) *reinterpret_cast<uint32_t*>(copy + (i * C + row) * KP + col) = f[i];
        }
    }
}

template <typename T, int KP>
__global__ void __launch_bounds__(128) gated_delta_prepare_kernel(GatedDeltaArgs a, Places w) {
    constexpr int NI = kInput<T>;
    using Shared = PrepareShared<T, KP>;
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& sm = *reinterpret_cast<Shared*>(raw);
    pdl_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const int group = a.heads / a.k_heads, k_head = head / group;
    const Span s = span_of(a, slot);
    if (s.tokens == 0) return;
    const size_t place = static_cast<size_t>(slot) * a.heads + head;
    char* const work = static_cast<char*>(a.workspace);

    __nv_bfloat16* copy = nullptr;
    if (head % group == 0)
        copy = reinterpret_cast<__nv_bfloat16*>(work + w.packed) +
               (static_cast<size_t>(slot) * a.k_heads + k_head) * 2 * NI * C * KP;
    pack_rows<T, KP>(a, a.q, s, k_head, sm.q, copy, tid);
    pack_rows<T, KP>(a, a.k, s, k_head, sm.k, copy ? copy + NI * C * KP : nullptr, tid);
    if (warp < 2) {  // running sums of the log decays, in 64 bits
        double sum = 0;
        float b = 0.f;
        if (tid < s.tokens) {
            const size_t token = static_cast<size_t>(s.first) + tid;
            const float g = gate_at(a.log_decay, a.log_decay32,
                                    s.row * a.log_decay.batch + token * a.log_decay.token + head * a.log_decay.head, kTypeId<T>);
            sum = g < kLeast ? kLeast : g;  // NaN stays
            b = gate_at(a.beta, a.beta32, s.row * a.beta.batch + token * a.beta.token + head * a.beta.head, kTypeId<T>);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const double other = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += other;
        }
        sm.sum[tid] = sum;
        sm.beta[tid] = b;
    }
    __syncthreads();
    if (warp == 1) sm.sum[tid] += sm.sum[31];
    __syncthreads();
    if (tid < C) {
        float* f = reinterpret_cast<float*>(work + w.factors) + place * kFactors;
        const double sum = sm.sum[tid];
        f[tid] = expf(static_cast<float>(sum));
        f[C + tid] = expf(static_cast<float>(sm.sum[C - 1] - sum));
        f[2 * C + tid] = sm.beta[tid];
        const float high = static_cast<float>(sum);
        f[3 * C + tid] = high;
        f[4 * C + tid] = static_cast<float>(sum - high);
    }

    // rows 16 warp .. + 15 of k k^T and q k^T, up to the diagonal
    const Tile<KP + 8, C*(KP + 8)> tq{smem_addr(sm.q)}, tk{smem_addr(sm.k)};
    float kk[8][4] = {}, qk[8][4] = {};
    for (int ks = 0; ks < KP / 16; ++ks) {
        uint32_t ak[NI][4], aq[NI][4];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            tk.a_rows(i, 16 * warp, 16 * ks, lane, ak[i]);
            tq.a_rows(i, 16 * warp, 16 * ks, lane, aq[i]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t <= warp) {
                uint32_t b[NI][1][4];
#pragma unroll
                for (int i = 0; i < NI; ++i) tk.b_rows(i, 16 * t, 16 * ks, lane, b[i][0]);
                products<3, NI, NI, 2>(kk + 2 * t, ak, b);
                products<3, NI, NI, 2>(qk + 2 * t, aq, b);
            }
        }
    }
    constexpr int LEVEL = kLevel<T>;
    __nv_bfloat16* attention = reinterpret_cast<__nv_bfloat16*>(work + w.attention) + place * LEVEL * kSquare;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 16 * warp + lane / 4 + 8 * h, j = 8 * t + lane % 4 * 2;
            float p[2], m[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float d = j + e <= i ? expf(static_cast<float>(sm.sum[i] - sm.sum[j + e])) : 0.f;
                p[e] = j + e <= i ? d * qk[t][2 * h + e] * a.scale : 0.f;
                m[e] = j + e < i ? d * kk[t][2 * h + e] : 0.f;
                sm.unit[i][j + e] = m[e];
                sm.m[i][j + e] = m[e] * sm.beta[j + e];
            }
            uint32_t f[LEVEL];
            pieces<LEVEL>(p[0], p[1], f);
#pragma unroll
            for (int n = 0; n < LEVEL; ++n)
                *reinterpret_cast<uint32_t*>(attention + n * kSquare + i * C + j) = f[n];
        }
    }
    __syncthreads();
    // column `tid` of L by forward substitution: l_i = M_i - sum over j < i of (M beta)_ij l_j
    if (tid >= C) return;
    float l[C];
    __nv_bfloat16* solve = reinterpret_cast<__nv_bfloat16*>(work + w.solve) + place * LEVEL * kSquare;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        float acc[4] = {sm.unit[i][tid], 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < i; j += 4) {
            const float4 m = *reinterpret_cast<const float4*>(&sm.m[i][j]);
            acc[0] = fmaf(-m.x, l[j], acc[0]);
            if (j + 1 < i) acc[1] = fmaf(-m.y, l[j + 1], acc[1]);
            if (j + 2 < i) acc[2] = fmaf(-m.z, l[j + 2], acc[2]);
            if (j + 3 < i) acc[3] = fmaf(-m.w, l[j + 3], acc[3]);
        }
        l[i] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        float rest = l[i];
#pragma unroll
        for (int n = 0; n < LEVEL; ++n) {
            const __nv_bfloat16 piece = __float2bfloat16_rn(rest);
            rest -= __bfloat162float(piece);
            solve[n * kSquare + i * C + tid] = piece;
        }
    }
}

// ---- chain --------------------------------------------------------------------------------------
// Shared memory of one chunk's tiles, for W warps (16 columns of v each).
template <typename T, int KP>
struct ChainTiles {
    static constexpr int NI = kInput<T>;
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + NI * C * (KP + 8) * 2;
    static constexpr int kSolve = kK + NI * C * (KP + 8) * 2;
    static constexpr int kAttention = kSolve + kLevel<T> * C * kPitchC * 2;
    static constexpr int kFactor = kAttention + kLevel<T> * C * kPitchC * 2;
    static constexpr int kRows = kFactor + kFactors * 4;
    static constexpr int bytes(int warps) {
        return kRows + C * (16 * warps + kSpare<T>) * static_cast<int>(sizeof(T));
    }
};

template <typename T, int KP>
CUBF_DEV void load_chunk(const GatedDeltaArgs& a, const Places& w, const HeadTensor& rows, bool wide_rows, const Span& s,
                         int slot, int head, int from, int width, unsigned char* stage, int tid, int threads) {
    using Tiles = ChainTiles<T, KP>;
    const int k_head = head / (a.heads / a.k_heads);
    const size_t place = static_cast<size_t>(slot) * a.heads + head;
    char* const work = static_cast<char*>(a.workspace);
    const uint32_t base = smem_addr(stage);
    load_packed<kInput<T>, KP>(packed_at<T, KP>(a, w, 0, slot, k_head), base + Tiles::kQ, tid, threads);
    load_packed<kInput<T>, KP>(packed_at<T, KP>(a, w, 1, slot, k_head), base + Tiles::kK, tid, threads);
    load_squares(reinterpret_cast<const __nv_bfloat16*>(work + w.solve) + place * kLevel<T> * kSquare, kLevel<T>,
                 base + Tiles::kSolve, tid, threads);
    load_squares(reinterpret_cast<const __nv_bfloat16*>(work + w.attention) + place * kLevel<T> * kSquare, kLevel<T>,
                 base + Tiles::kAttention, tid, threads);
    const float* f = reinterpret_cast<const float*>(work + w.factors) + place * kFactors;
    for (int e = tid; e < kFactors / 4; e += threads) copy16(base + Tiles::kFactor + e * 16, f + e * 4, true);
    const T* p = static_cast<const T*>(rows.p) + s.row * rows.batch + static_cast<size_t>(s.first) * rows.token +
                 static_cast<size_t>(head) * rows.head;
    load_rows<T>(p, rows.token, s.tokens, a.v_dim, from, width, wide_rows, reinterpret_cast<T*>(stage + Tiles::kRows),
                 tid, threads);
    copies_commit();
}

// A fragment of 16 columns out of two accumulator tiles; `factor` holds one factor a column.
template <int N>
CUBF_DEV void operand(const float (&a)[4], const float (&b)[4], uint32_t (&f)[N][4]) {
    fragment<N>(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], f);
}
template <int N>
CUBF_DEV void operand(const float (&a)[4], const float (&b)[4], const float* factor, float scale, int lane,
                      uint32_t (&f)[N][4]) {
    float2 lo = *reinterpret_cast<const float2*>(factor + lane % 4 * 2);
    float2 hi = *reinterpret_cast<const float2*>(factor + 8 + lane % 4 * 2);
    lo.x *= scale, lo.y *= scale, hi.x *= scale, hi.y *= scale;
    fragment<N>(a[0] * lo.x, a[1] * lo.y, a[2] * lo.x, a[3] * lo.y, b[0] * hi.x, b[1] * hi.y, b[2] * hi.x, b[3] * hi.y, f);
}

// d[0 .. N/8) += A B for a state's worth of columns: B = q or k, stored [token][channel], tokens 16 ks ..
template <int LEVEL, int NA, int NI, int KP, typename Operand>
CUBF_DEV void onto_state(float (*d)[4], const uint32_t (&a)[NA][4], const Operand& b, int ks, int lane) {
#pragma unroll
    for (int t = 0; t < KP / 32; ++t) {
        uint32_t f[NI][2][4];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            b.b_cols(i, 16 * ks, 32 * t, lane, f[i][0]);
            b.b_cols(i, 16 * ks, 32 * t + 16, lane, f[i][1]);
        }
        products<LEVEL, NA, NI, 4>(d + 4 * t, a, f);
    }
}

// State (K x V of one head, fp32) <-> the fragments of its transpose.
template <int KP>
CUBF_DEV void state_load(const float* p, int k_dim, int v_dim, int v, int lane, float (&s)[KP / 8][4]) {
#pragma unroll
    for (int t = 0; t < KP / 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = 8 * t + lane % 4 * 2 + e % 2, col = v + lane / 4 + e / 2 * 8;
            s[t][e] = p && k < k_dim && col < v_dim ? p[static_cast<size_t>(k) * v_dim + col] : 0.f;
        }
}
template <int KP>
CUBF_DEV void state_store(float* p, int k_dim, int v_dim, int v, int lane, const float (&s)[KP / 8][4]) {
#pragma unroll
    for (int t = 0; t < KP / 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = 8 * t + lane % 4 * 2 + e % 2, col = v + lane / 4 + e / 2 * 8;
            if (k < k_dim && col < v_dim) p[static_cast<size_t>(k) * v_dim + col] = s[t][e];
        }
}
// The same fragments kept for `gradients`: rows of KP values, a row for each column of v.
template <int KP>
CUBF_DEV void state_keep(float* p, int v, int lane, const float (&s)[KP / 8][4]) {
#pragma unroll
    for (int t = 0; t < KP / 8; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(p + static_cast<size_t>(v + lane / 4 + 8 * h) * KP + 8 * t + lane % 4 * 2) =
                make_float2(s[t][2 * h], s[t][2 * h + 1]);
}
// A 64-token result (transposed fragments) as fp32 rows of `pitch` values.
CUBF_DEV void rows_keep(float* p, int pitch, int v, int lane, const float (&x)[8][4]) {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            p[static_cast<size_t>(8 * t + lane % 4 * 2 + e % 2) * pitch + v + lane / 4 + e / 2 * 8] = x[t][e];
}
// The same, rounded to T, through the warp's own columns of a row tile to global rows `row` apart.
template <typename T>
CUBF_DEV void rows_store(T* p, size_t row, int rows, int cols, bool wide, T* tile, int pitch, int lane,
                         const float (&x)[8][4]) {
    __syncwarp();
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            tile[(8 * t + lane % 4 * 2 + e % 2) * pitch + lane / 4 + e / 2 * 8] = Convert<T, float>::store(x[t][e]);
    __syncwarp();
    constexpr int N = 16 / sizeof(T), PER = 16 / N;
    if (wide) {
#pragma unroll
        for (int e = lane; e < C * PER; e += 32) {
            const int r = e / PER, c = e % PER * N;
            if (r < rows && c < cols)
                *reinterpret_cast<uint4*>(p + r * row + c) = *reinterpret_cast<const uint4*>(tile + r * pitch + c);
        }
    } else {
        for (int e = lane; e < C * 16; e += 32) {
            const int r = e / 16, c = e % 16;
            if (r < rows && c < cols) p[r * row + c] = tile[r * pitch + c];
        }
    }
}

struct ChainShape {
    int slices, warps;   // CTAs along v, warps a CTA
    bool wide_v, wide_o, wide_d;
};

// One sequence of one head, 16 columns of v a warp.  KEEP: the backward's run, which keeps S before each chunk and R
// instead of writing o.
template <typename T, int KP, bool KEEP>
CUBF_DEV void forward_chain(const GatedDeltaArgs& a, const Places& w, const ChainShape& shape, int slice, int head,
                            int sequence, unsigned char* raw) {
    using Tiles = ChainTiles<T, KP>;
    constexpr int NI = Tiles::NI, LEVEL = kLevel<T>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = 32 * shape.warps;
    const int width = 16 * shape.warps, from = slice * width, v = from + 16 * warp;
    const int start = a.offsets ? offset_at(a, sequence) : 0;
    const int length = a.offsets ? max(0, offset_at(a, sequence + 1) - start) : a.length;
    const int row = a.offsets ? 0 : sequence;
    const int base = slot_base(a, sequence, start), chunks = (length + C - 1) / C;
    auto span = [&](int c) { return Span{sequence, c, start + c * C, min(C, length - c * C), row}; };
    auto load = [&](int c) {
        load_chunk<T, KP>(a, w, a.v, shape.wide_v, span(c), base + c, head, from, width,
                              raw, tid, threads);
    };
    const size_t state = (static_cast<size_t>(sequence) * a.heads + head) * a.k_dim * a.v_dim;
    float s[KP / 8][4];
    state_load<KP>(a.initial ? a.initial + state : nullptr, a.k_dim, a.v_dim, v, lane, s);
    if (chunks > 0) load(0);
    for (int c = 0; c < chunks; ++c) {
        copies_wait<0>();
        __syncthreads();
        unsigned char* const stage = raw;
        const uint32_t at = smem_addr(stage);
        const Tile<KP + 8, C*(KP + 8)> q{at + Tiles::kQ}, k{at + Tiles::kK};
        const Tile<kPitchC, C * kPitchC> solve{at + Tiles::kSolve}, attention{at + Tiles::kAttention};
        const float* f = reinterpret_cast<const float*>(stage + Tiles::kFactor);
        T* tile = reinterpret_cast<T*>(stage + Tiles::kRows) + 16 * warp;
        const int pitch = width + kSpare<T>;
        const size_t place = static_cast<size_t>(base + c) * a.heads + head;
        char* const work = static_cast<char*>(a.workspace);
        if (v < a.v_dim) {
            if (KEEP)
                state_keep<KP>(reinterpret_cast<float*>(work + w.states) + place * w.v_pitch * KP, v, lane, s);
            float x[8][4] = {}, o[8][4] = {};
#pragma unroll
            for (int ks = 0; ks < KP / 16; ++ks) {
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(s[2 * ks], s[2 * ks + 1], f3);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t b[NI][2][4];
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        k.b_rows(i, 32 * t, 16 * ks, lane, b[i][0]);
                        k.b_rows(i, 32 * t + 16, 16 * ks, lane, b[i][1]);
                    }
                    products<kInputLevel<T>, LEVEL, NI, 4>(x + 4 * t, f3, b);
                    if (!KEEP) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            q.b_rows(i, 32 * t, 16 * ks, lane, b[i][0]);
                            q.b_rows(i, 32 * t + 16, 16 * ks, lane, b[i][1]);
                        }
                        products<kInputLevel<T>, LEVEL, NI, 4>(o + 4 * t, f3, b);
                    }
                }
            }
            // Y = v - e^G (S k); o = scale e^G (S q)
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int token = 8 * t + lane % 4 * 2;
                const float2 decay = *reinterpret_cast<const float2*>(f + token);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float d = e % 2 ? decay.y : decay.x;
                    x[t][e] = fmaf(-d, x[t][e], widen(tile[(token + e % 2) * pitch + lane / 4 + e / 2 * 8]));
                    o[t][e] *= d * a.scale;
                }
            }
            // R = Y - L (beta Y), the later tokens' columns first: those are added to before they are read
#pragma unroll
            for (int ks = 3; ks >= 0; --ks) {
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(x[2 * ks], x[2 * ks + 1], f + 2 * C + 16 * ks, -1.f, lane, f3);
#pragma unroll
                for (int t = ks; t < 4; ++t) {
                    uint32_t b[LEVEL][1][4];
#pragma unroll
                    for (int i = 0; i < LEVEL; ++i) solve.b_rows(i, 16 * t, 16 * ks, lane, b[i][0]);
                    products<LEVEL, LEVEL, LEVEL, 2>(x + 2 * t, f3, b);
                }
            }
            if (KEEP)
                rows_keep(reinterpret_cast<float*>(work + w.errors) + place * C * w.v_pitch, w.v_pitch, v, lane, x);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float2 beta = *reinterpret_cast<const float2*>(f + 2 * C + 8 * t + lane % 4 * 2);
                x[t][0] *= beta.x, x[t][1] *= beta.y, x[t][2] *= beta.x, x[t][3] *= beta.y;
            }
            const float whole = f[C - 1];
#pragma unroll
            for (int t = 0; t < KP / 8; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] *= whole;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                if (!KEEP) {
                    uint32_t f2[LEVEL][4];
                    operand<LEVEL>(x[2 * ks], x[2 * ks + 1], f2);
#pragma unroll
                    for (int t = ks; t < 4; ++t) {
                        uint32_t b[LEVEL][1][4];
#pragma unroll
                        for (int i = 0; i < LEVEL; ++i) attention.b_rows(i, 16 * t, 16 * ks, lane, b[i][0]);
                        products<LEVEL, LEVEL, LEVEL, 2>(o + 2 * t, f2, b);
                    }
                }
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(x[2 * ks], x[2 * ks + 1], f + C + 16 * ks, 1.f, lane, f3);
                onto_state<kInputLevel<T>, LEVEL, NI, KP>(s, f3, k, ks, lane);
            }
            if (!KEEP) {
                const size_t token = static_cast<size_t>(row) * a.length + start + c * C;
                rows_store<T>(static_cast<T*>(a.o) + (token * a.heads + head) * a.v_dim + v,
                              static_cast<size_t>(a.heads) * a.v_dim, min(C, length - c * C), a.v_dim - v, shape.wide_o,
                              tile, pitch, lane, o);
            }
        }
        __syncthreads();
        if (c + 1 < chunks) load(c + 1);
    }
    if (!KEEP && v < a.v_dim) state_store<KP>(a.last + state, a.k_dim, a.v_dim, v, lane, s);
}

// The same sequence from its end: dS, W and dv of every chunk.
template <typename T, int KP>
CUBF_DEV void backward_chain(const GatedDeltaArgs& a, const Places& w, const ChainShape& shape, int slice, int head,
                             int sequence, unsigned char* raw) {
    using Tiles = ChainTiles<T, KP>;
    constexpr int NI = Tiles::NI, LEVEL = kLevel<T>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = 32 * shape.warps;
    const int width = 16 * shape.warps, from = slice * width, v = from + 16 * warp;
    const int start = a.offsets ? offset_at(a, sequence) : 0;
    const int length = a.offsets ? max(0, offset_at(a, sequence + 1) - start) : a.length;
    const int row = a.offsets ? 0 : sequence;
    const int base = slot_base(a, sequence, start), chunks = (length + C - 1) / C;
    auto load = [&](int c) {
        load_chunk<T, KP>(a, w, a.d_o, shape.wide_d, Span{sequence, c, start + c * C, min(C, length - c * C), row},
                                   base + c, head, from, width, raw, tid, threads);
    };
    const size_t state = (static_cast<size_t>(sequence) * a.heads + head) * a.k_dim * a.v_dim;
    float s[KP / 8][4];  // dS, transposed
    state_load<KP>(a.d_last ? a.d_last + state : nullptr, a.k_dim, a.v_dim, v, lane, s);
    if (chunks > 0) load(chunks - 1);
    for (int c = chunks - 1; c >= 0; --c) {
        copies_wait<0>();
        __syncthreads();
        unsigned char* const stage = raw;
        const uint32_t at = smem_addr(stage);
        const Tile<KP + 8, C*(KP + 8)> q{at + Tiles::kQ}, k{at + Tiles::kK};
        const Tile<kPitchC, C * kPitchC> solve{at + Tiles::kSolve}, attention{at + Tiles::kAttention};
        const float* f = reinterpret_cast<const float*>(stage + Tiles::kFactor);
        T* tile = reinterpret_cast<T*>(stage + Tiles::kRows) + 16 * warp;
        const int pitch = width + kSpare<T>;
        const size_t place = static_cast<size_t>(base + c) * a.heads + head;
        char* const work = static_cast<char*>(a.workspace);
        if (v < a.v_dim) {
            state_keep<KP>(reinterpret_cast<float*>(work + w.d_states) + place * w.v_pitch * KP, v, lane, s);
            float x[8][4] = {};
#pragma unroll
            for (int ks = 0; ks < KP / 16; ++ks) {
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(s[2 * ks], s[2 * ks + 1], f3);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t b[NI][2][4];
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        k.b_rows(i, 32 * t, 16 * ks, lane, b[i][0]);
                        k.b_rows(i, 32 * t + 16, 16 * ks, lane, b[i][1]);
                    }
                    products<kInputLevel<T>, LEVEL, NI, 4>(x + 4 * t, f3, b);
                }
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float2 tail = *reinterpret_cast<const float2*>(f + C + 8 * t + lane % 4 * 2);
                x[t][0] *= tail.x, x[t][1] *= tail.y, x[t][2] *= tail.x, x[t][3] *= tail.y;
            }
            const float whole = f[C - 1];
#pragma unroll
            for (int t = 0; t < KP / 8; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] *= whole;
            // E += P^T dO, and dO's part of dS
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                float d[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d[t][e] = widen(tile[(16 * ks + 8 * t + lane % 4 * 2 + e % 2) * pitch + lane / 4 + e / 2 * 8]);
                uint32_t exact[NI][4];
                operand<NI>(d[0], d[1], exact);
#pragma unroll
                for (int t = 0; t <= ks; ++t) {
                    uint32_t b[LEVEL][1][4];
#pragma unroll
                    for (int i = 0; i < LEVEL; ++i) attention.b_cols(i, 16 * ks, 16 * t, lane, b[i][0]);
                    products<kInputLevel<T>, NI, LEVEL, 2>(x + 2 * t, exact, b);
                }
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(d[0], d[1], f + 16 * ks, a.scale, lane, f3);
                onto_state<kInputLevel<T>, LEVEL, NI, KP>(s, f3, q, ks, lane);
            }
            // W = E - L^T (beta E), the earlier tokens' columns first
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(x[2 * ks], x[2 * ks + 1], f + 2 * C + 16 * ks, -1.f, lane, f3);
#pragma unroll
                for (int t = 0; t <= ks; ++t) {
                    uint32_t b[LEVEL][1][4];
#pragma unroll
                    for (int i = 0; i < LEVEL; ++i) solve.b_cols(i, 16 * ks, 16 * t, lane, b[i][0]);
                    products<LEVEL, LEVEL, LEVEL, 2>(x + 2 * t, f3, b);
                }
            }
            rows_keep(reinterpret_cast<float*>(work + w.d_writes) + place * C * w.v_pitch, w.v_pitch, v, lane, x);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float2 beta = *reinterpret_cast<const float2*>(f + 2 * C + 8 * t + lane % 4 * 2);
                x[t][0] *= beta.x, x[t][1] *= beta.y, x[t][2] *= beta.x, x[t][3] *= beta.y;
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                uint32_t f3[LEVEL][4];
                operand<LEVEL>(x[2 * ks], x[2 * ks + 1], f + 16 * ks, -1.f, lane, f3);
                onto_state<kInputLevel<T>, LEVEL, NI, KP>(s, f3, k, ks, lane);
            }
            const size_t token = static_cast<size_t>(row) * a.length + start + c * C;
            rows_store<T>(static_cast<T*>(a.d_v) + (token * a.heads + head) * a.v_dim + v,
                          static_cast<size_t>(a.heads) * a.v_dim, min(C, length - c * C), a.v_dim - v, shape.wide_o, tile,
                          pitch, lane, x);
        }
        __syncthreads();
        if (c > 0) load(c - 1);
    }
    if (a.d_initial && v < a.v_dim) state_store<KP>(a.d_initial + state, a.k_dim, a.v_dim, v, lane, s);
}

template <typename T, int KP>
__global__ void __launch_bounds__(256) gated_delta_forward_kernel(GatedDeltaArgs a, Places w, ChainShape shape) {
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_begin();
    const int slice = blockIdx.x % shape.slices, rest = blockIdx.x / shape.slices;
    forward_chain<T, KP, false>(a, w, shape, slice, rest % a.heads, rest / a.heads, raw);
}

// Both chains of the backward side by side: neither needs the other's results.
template <typename T, int KP>
__global__ void __launch_bounds__(256) gated_delta_chains_kernel(GatedDeltaArgs a, Places w, ChainShape shape) {
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_begin();
    const int slice = blockIdx.x / 2 % shape.slices, rest = blockIdx.x / 2 / shape.slices;
    if (blockIdx.x % 2 == 0)
        backward_chain<T, KP>(a, w, shape, slice, rest % a.heads, rest / a.heads, raw);
    else
        forward_chain<T, KP, true>(a, w, shape, slice, rest % a.heads, rest / a.heads, raw);
}

// ---- gradients ----------------------------------------------------------------------------------
// A CTA per chunk and head: 16 warps, warp (r, c) holds rows 16 r .. of the tokens and a quarter of the channels.
template <typename T, int KP>
struct GradientShared32 {
    static constexpr int NI = kInput<T>, LB = kLevel<T>, ND = NI < LB ? NI : LB;
    static constexpr int VS = 32;                    // columns of v a turn
    static constexpr int kPitchV = VS + 8;
    alignas(16) __nv_bfloat16 q[NI * C * (KP + 8)];
    alignas(16) __nv_bfloat16 k[NI * C * (KP + 8)];
    union {
        struct {
            alignas(16) __nv_bfloat16 state[LB * VS * (KP + 8)];     // S, transposed
            alignas(16) __nv_bfloat16 d_state[LB * VS * (KP + 8)];
            alignas(16) __nv_bfloat16 u[LB * C * kPitchV];
            alignas(16) __nv_bfloat16 z[LB * C * kPitchV];
            alignas(16) __nv_bfloat16 d_o[ND * C * kPitchV];
        } in;
        struct {
            alignas(16) __nv_bfloat16 d_p[LB * C * kPitchC];         // D o dP
            alignas(16) __nv_bfloat16 d_m[LB * C * kPitchC];         // D o dM
        } pairs;
    };
    float factors[kFactors];
    float sums[4][4][C];                             // partial sums of dG's terms by channel quarter or row block
    float dot[16];
    double d_sum[C], kept[2];
};

template <typename T, int KP, bool SHARED>
__global__ void __launch_bounds__(512) gated_delta_gradients_kernel(GatedDeltaArgs a, Places w) {
    using Shared = GradientShared32<T, KP>;
    constexpr int NI = Shared::NI, LB = Shared::LB, ND = Shared::ND, VS = Shared::VS, PV = Shared::kPitchV;
    constexpr int NT = KP / 32;  // tiles of 8 channels a warp
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& sm = *reinterpret_cast<Shared*>(raw);
    pdl_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rb = warp & 3, cg = warp >> 2;
    const int slot = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const int k_head = head / (a.heads / a.k_heads);
    const Span s = span_of(a, slot);
    if (s.tokens == 0) return;
    const size_t place = static_cast<size_t>(slot) * a.heads + head;
    const char* const work = static_cast<const char*>(a.workspace);
    load_packed<NI, KP>(packed_at<T, KP>(a, w, 0, slot, k_head), smem_addr(sm.q), tid, 512);
    load_packed<NI, KP>(packed_at<T, KP>(a, w, 1, slot, k_head), smem_addr(sm.k), tid, 512);
    copies_commit();
    const float* factors = reinterpret_cast<const float*>(work + w.factors) + place * kFactors;
    if (tid < kFactors) sm.factors[tid] = factors[tid];

    const float* state = reinterpret_cast<const float*>(work + w.states) + place * w.v_pitch * KP;
    const float* d_state = reinterpret_cast<const float*>(work + w.d_states) + place * w.v_pitch * KP;
    const float* errors = reinterpret_cast<const float*>(work + w.errors) + place * C * w.v_pitch;
    const float* d_writes = reinterpret_cast<const float*>(work + w.d_writes) + place * C * w.v_pitch;
    const T* d_o = static_cast<const T*>(a.d_o.p) + s.row * a.d_o.batch + static_cast<size_t>(s.first) * a.d_o.token +
                   static_cast<size_t>(head) * a.d_o.head;
    const Tile<KP + 8, C*(KP + 8)> tq{smem_addr(sm.q)}, tk{smem_addr(sm.k)};
    const Tile<KP + 8, VS*(KP + 8)> ts{smem_addr(sm.in.state)}, td{smem_addr(sm.in.d_state)};
    const Tile<PV, C * PV> tu{smem_addr(sm.in.u)}, tz{smem_addr(sm.in.z)}, to{smem_addr(sm.in.d_o)};

    float dp[2][4] = {}, dm[2][4] = {};                          // dO U^T, Z U^T: 16 x 16 at (rb, cg)
    float qs[NT][4] = {}, ks[NT][4] = {}, ku[NT][4] = {};        // dO S^T, Z S^T, U dS^T: 16 x KP / 4
    float d_beta = 0.f, dot = 0.f;                               // of token tid / 8
    __syncthreads();
    for (int from = 0; from < w.v_pitch; from += VS) {
        // states: VS rows of KP values
        for (int e = tid; e < VS * KP / 4; e += 512) {
            const int r = e / (KP / 4), c = e % (KP / 4) * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (from + r < w.v_pitch) {
                x = *reinterpret_cast<const float4*>(state + static_cast<size_t>(from + r) * KP + c);
                y = *reinterpret_cast<const float4*>(d_state + static_cast<size_t>(from + r) * KP + c);
            }
            dot += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
            uint32_t lo[LB], hi[LB];
            pieces<LB>(x.x, x.y, lo);
            pieces<LB>(x.z, x.w, hi);
#pragma unroll
            for (int i = 0; i < LB; ++i)
                *reinterpret_cast<uint2*>(sm.in.state + (i * VS + r) * (KP + 8) + c) = make_uint2(lo[i], hi[i]);
            pieces<LB>(y.x, y.y, lo);
            pieces<LB>(y.z, y.w, hi);
#pragma unroll
            for (int i = 0; i < LB; ++i)
                *reinterpret_cast<uint2*>(sm.in.d_state + (i * VS + r) * (KP + 8) + c) = make_uint2(lo[i], hi[i]);
        }
        {  // U = beta R, Z = beta W and dO: eight threads a token
            const int r = tid / 8, c = tid % 8 * 4;
            const float beta = sm.factors[2 * C + r];
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (from + c < w.v_pitch) {
                x = *reinterpret_cast<const float4*>(errors + static_cast<size_t>(r) * w.v_pitch + from + c);
                y = *reinterpret_cast<const float4*>(d_writes + static_cast<size_t>(r) * w.v_pitch + from + c);
            }
            d_beta += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
            uint32_t lo[LB], hi[LB];
            pieces<LB>(x.x * beta, x.y * beta, lo);
            pieces<LB>(x.z * beta, x.w * beta, hi);
#pragma unroll
            for (int i = 0; i < LB; ++i)
                *reinterpret_cast<uint2*>(sm.in.u + (i * C + r) * PV + c) = make_uint2(lo[i], hi[i]);
            pieces<LB>(y.x * beta, y.y * beta, lo);
            pieces<LB>(y.z * beta, y.w * beta, hi);
#pragma unroll
            for (int i = 0; i < LB; ++i)
                *reinterpret_cast<uint2*>(sm.in.z + (i * C + r) * PV + c) = make_uint2(lo[i], hi[i]);
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                d[e] = r < s.tokens && from + c + e < a.v_dim
                           ? widen(d_o[static_cast<size_t>(r) * a.d_o.token + from + c + e])
                           : 0.f;
            uint32_t dl[ND], dh[ND];
            pieces<ND>(d[0], d[1], dl);
            pieces<ND>(d[2], d[3], dh);
#pragma unroll
            for (int i = 0; i < ND; ++i)
                *reinterpret_cast<uint2*>(sm.in.d_o + (i * C + r) * PV + c) = make_uint2(dl[i], dh[i]);
        }
        __syncthreads();
#pragma unroll
        for (int step = 0; step < VS / 16; ++step) {
            uint32_t ao[ND][4], az[LB][4], au[LB][4];
#pragma unroll
            for (int i = 0; i < ND; ++i) to.a_rows(i, 16 * rb, 16 * step, lane, ao[i]);
#pragma unroll
            for (int i = 0; i < LB; ++i) {
                tz.a_rows(i, 16 * rb, 16 * step, lane, az[i]);
                tu.a_rows(i, 16 * rb, 16 * step, lane, au[i]);
            }
            if (cg <= rb) {
                uint32_t b[LB][1][4];
#pragma unroll
                for (int i = 0; i < LB; ++i) tu.b_rows(i, 16 * cg, 16 * step, lane, b[i][0]);
                products<LB, ND, LB, 2>(dp, ao, b);
                products<LB, LB, LB, 2>(dm, az, b);
            }
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                uint32_t b[LB][1][4];
                const int col = cg * (KP / 4) + 16 * t;
#pragma unroll
                for (int i = 0; i < LB; ++i) ts.b_cols(i, 16 * step, col, lane, b[i][0]);
                products<LB, ND, LB, 2>(qs + 2 * t, ao, b);
                products<LB, LB, LB, 2>(ks + 2 * t, az, b);
#pragma unroll
                for (int i = 0; i < LB; ++i) td.b_cols(i, 16 * step, col, lane, b[i][0]);
                products<LB, LB, LB, 2>(ku + 2 * t, au, b);
            }
        }
        __syncthreads();
    }
    copies_wait<0>();
    __syncthreads();
    // dbeta, and <S, dS'> of this CTA
#pragma unroll
    for (int d = 1; d < 8; d *= 2) d_beta += __shfl_xor_sync(0xffffffffu, d_beta, d);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (lane == 0) sm.dot[warp] = dot;
    const size_t gate_row = static_cast<size_t>(s.row) * a.length + s.first;
    if (tid % 8 == 0 && tid / 8 < s.tokens) {
        const size_t at = (gate_row + tid / 8) * a.heads + head;
        if (a.beta32)
            static_cast<float*>(a.d_beta)[at] = d_beta;
        else
            static_cast<T*>(a.d_beta)[at] = Convert<T, float>::store(d_beta);
    }

    // the scaled state terms and their products with q and k
    float row_sum[2] = {}, kept[2] = {};
    const int row = 16 * rb + lane / 4;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = row + 8 * h, col = cg * (KP / 4) + 8 * t + lane % 4 * 2;
            const float from_start = sm.factors[i], to_end = sm.factors[C + i];
            float2 qv = make_float2(0.f, 0.f), kv = qv;
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(sm.q + (n * C + i) * (KP + 8) + col));
                const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(sm.k + (n * C + i) * (KP + 8) + col));
                qv.x += x.x, qv.y += x.y, kv.x += y.x, kv.y += y.y;
            }
            qs[t][2 * h] *= from_start * a.scale, qs[t][2 * h + 1] *= from_start * a.scale;
            ks[t][2 * h] *= -from_start, ks[t][2 * h + 1] *= -from_start;
            ku[t][2 * h] *= to_end, ku[t][2 * h + 1] *= to_end;
            row_sum[h] += qs[t][2 * h] * qv.x + qs[t][2 * h + 1] * qv.y + ks[t][2 * h] * kv.x + ks[t][2 * h + 1] * kv.y;
            kept[h] += ku[t][2 * h] * kv.x + ku[t][2 * h + 1] * kv.y;
            ks[t][2 * h] += ku[t][2 * h], ks[t][2 * h + 1] += ku[t][2 * h + 1];
        }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
            row_sum[h] += __shfl_xor_sync(0xffffffffu, row_sum[h], d);
            kept[h] += __shfl_xor_sync(0xffffffffu, kept[h], d);
        }
    if (lane % 4 == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sm.sums[0][cg][row + 8 * h] = row_sum[h];
            sm.sums[1][cg][row + 8 * h] = kept[h];
        }

    // the pairs' terms: D o dP, D o dM and the row and column sums of P o dP + M o dM
    float row_pair[2] = {}, col_pair[2][2] = {};
    if (cg <= rb) {
        float qk[2][4] = {}, kk[2][4] = {};
        for (int step = 0; step < KP / 16; ++step) {
            uint32_t aq[NI][4], ak[NI][4], b[NI][1][4];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                tq.a_rows(i, 16 * rb, 16 * step, lane, aq[i]);
                tk.a_rows(i, 16 * rb, 16 * step, lane, ak[i]);
                tk.b_rows(i, 16 * cg, 16 * step, lane, b[i][0]);
            }
            products<LB, NI, NI, 2>(qk, aq, b);
            products<LB, NI, NI, 2>(kk, ak, b);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = row + e / 2 * 8, j = 16 * cg + 8 * t + lane % 4 * 2 + e % 2;
                // G_i - G_j of sums in two floats
                const float d = (sm.factors[3 * C + i] - sm.factors[3 * C + j]) + (sm.factors[4 * C + i] - sm.factors[4 * C + j]);
                const float decay = j <= i ? expf(d) : 0.f;
                const float p = j <= i ? decay * a.scale * dp[t][e] : 0.f, m = j < i ? -decay * dm[t][e] : 0.f;
                const float pair = (j <= i ? p * qk[t][e] : 0.f) + (j < i ? m * kk[t][e] : 0.f);
                row_pair[e / 2] += pair;
                col_pair[t][e % 2] += pair;
                dp[t][e] = p;
                dm[t][e] = m;
            }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 1; d < 4; d *= 2) row_pair[h] += __shfl_xor_sync(0xffffffffu, row_pair[h], d);
    if (lane % 4 == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) sm.sums[2][cg][row + 8 * h] = row_pair[h];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) col_pair[t][e] += __shfl_xor_sync(0xffffffffu, col_pair[t][e], d);
            if (lane < 4) sm.sums[3][rb][16 * cg + 8 * t + lane * 2 + e] = col_pair[t][e];
        }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = (row + 8 * h) * kPitchC + 16 * cg + 8 * t + lane % 4 * 2;
            uint32_t f[LB];
            pieces<LB>(dp[t][2 * h], dp[t][2 * h + 1], f);
#pragma unroll
            for (int i = 0; i < LB; ++i) *reinterpret_cast<uint32_t*>(sm.pairs.d_p + i * C * kPitchC + at) = f[i];
            pieces<LB>(dm[t][2 * h], dm[t][2 * h + 1], f);
#pragma unroll
            for (int i = 0; i < LB; ++i) *reinterpret_cast<uint32_t*>(sm.pairs.d_m + i * C * kPitchC + at) = f[i];
        }
    __syncthreads();

    const Tile<kPitchC, C * kPitchC> tp{smem_addr(sm.pairs.d_p)}, tm{smem_addr(sm.pairs.d_m)};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
        uint32_t f[LB][4];
        if (step <= rb) {  // rows rb: tokens up to their own
            uint32_t g[LB][4];
#pragma unroll
            for (int i = 0; i < LB; ++i) {
                tp.a_rows(i, 16 * rb, 16 * step, lane, f[i]);
                tm.a_rows(i, 16 * rb, 16 * step, lane, g[i]);
            }
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                uint32_t b[NI][1][4];
#pragma unroll
                for (int i = 0; i < NI; ++i) tk.b_cols(i, 16 * step, cg * (KP / 4) + 16 * t, lane, b[i][0]);
                products<LB, LB, NI, 2>(qs + 2 * t, f, b);
                products<LB, LB, NI, 2>(ks + 2 * t, g, b);
            }
        }
        if (step >= rb) {  // columns rb: tokens from their own on
            uint32_t g[LB][4];
#pragma unroll
            for (int i = 0; i < LB; ++i) {
                tp.a_cols(i, 16 * step, 16 * rb, lane, f[i]);
                tm.a_cols(i, 16 * step, 16 * rb, lane, g[i]);
            }
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                uint32_t b[NI][1][4];
#pragma unroll
                for (int i = 0; i < NI; ++i) tq.b_cols(i, 16 * step, cg * (KP / 4) + 16 * t, lane, b[i][0]);
                products<LB, LB, NI, 2>(ks + 2 * t, f, b);
#pragma unroll
                for (int i = 0; i < NI; ++i) tk.b_cols(i, 16 * step, cg * (KP / 4) + 16 * t, lane, b[i][0]);
                products<LB, LB, NI, 2>(ks + 2 * t, g, b);
            }
        }
    }
    // where heads share keys: fp32 rows for each head, summed afterwards
    using Out = std::conditional_t<SHARED, float, T>;
    const int out_heads = SHARED ? a.heads : a.k_heads, out_head = SHARED ? head : k_head;
    Out* const dq = static_cast<Out*>(SHARED ? static_cast<void*>(static_cast<char*>(a.workspace) + w.d_q) : a.d_q);
    Out* const dk = static_cast<Out*>(SHARED ? static_cast<void*>(static_cast<char*>(a.workspace) + w.d_k) : a.d_k);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = row + 8 * h, col = cg * (KP / 4) + 8 * t + lane % 4 * 2;
            if (i >= s.tokens) continue;
            const size_t at = ((gate_row + i) * out_heads + out_head) * a.k_dim + col;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (col + e < a.k_dim) {
                    dq[at + e] = Convert<Out, float>::store(qs[t][2 * h + e]);
                    dk[at + e] = Convert<Out, float>::store(ks[t][2 * h + e]);
                }
        }

    // dG and its sums from each token on, in 64 bits: the terms of a sequence's first token cancel exactly
    if (tid < C) {
        auto sum = [&](int which) {
            return static_cast<double>(sm.sums[which][0][tid]) + sm.sums[which][1][tid] + sm.sums[which][2][tid] +
                   sm.sums[which][3][tid];
        };
        const double kept_here = sum(1);
        double d = sum(0) - kept_here + sum(2) - sum(3), all = kept_here;
#pragma unroll
        for (int n = 1; n < 32; n *= 2) {
            const double other = __shfl_down_sync(0xffffffffu, d, n);
            if (lane + n < 32) d += other;
            all += __shfl_xor_sync(0xffffffffu, all, n);
        }
        sm.d_sum[tid] = d;
        if (lane == 0) sm.kept[warp] = all;
    }
    __syncthreads();
    if (tid < s.tokens) {
        double d = sm.d_sum[tid] + (tid < 32 ? sm.d_sum[32] : 0.0);
        float inner = 0.f;
#pragma unroll
        for (int n = 0; n < 16; ++n) inner += sm.dot[n];
        d += sm.kept[0] + sm.kept[1] + static_cast<double>(sm.factors[C - 1]) * inner;
        const size_t at = (gate_row + tid) * a.heads + head;
        if (a.log_decay32)
            static_cast<float*>(a.d_log_decay)[at] = static_cast<float>(d);
        else
            static_cast<T*>(a.d_log_decay)[at] = Convert<T, float>::store(static_cast<float>(d));
    }
}

// Sums the gradients of shared keys and queries over their heads.
template <typename T>
__global__ void __launch_bounds__(256) gated_delta_share_kernel(GatedDeltaArgs a, Places w, size_t values) {
    pdl_begin();
    const int group = a.heads / a.k_heads;
    const float* dq = reinterpret_cast<const float*>(static_cast<const char*>(a.workspace) + w.d_q);
    const float* dk = reinterpret_cast<const float*>(static_cast<const char*>(a.workspace) + w.d_k);
    for (size_t e = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; e < values;
         e += static_cast<size_t>(gridDim.x) * 256) {
        const size_t head = e / a.k_dim, col = e % a.k_dim;
        float x = 0.f, y = 0.f;
        for (int g = 0; g < group; ++g) {
            x += dq[(head * group + g) * a.k_dim + col];
            y += dk[(head * group + g) * a.k_dim + col];
        }
        static_cast<T*>(a.d_q)[e] = Convert<T, float>::store(x);
        static_cast<T*>(a.d_k)[e] = Convert<T, float>::store(y);
    }
}

// ---- one token ----------------------------------------------------------------------------------
// A CTA takes VW columns of a head's state: each thread one vector of VEC columns of K / 16 rows, all loaded before the
// first use.  o = scale (e^g q^T S + (q . k) u), so that both products with the old state share one reduction.
// Bounded by the state's bytes, read and written once.
template <typename T, int VEC>
__global__ void __launch_bounds__(128) gated_delta_step_kernel(GatedDeltaStepArgs a, int slices) {
    constexpr int COLS = 8 * VEC;        // a CTA's columns: 8 threads side by side, 16 rows apart
    constexpr int ROWS = kDeltaMaxDim / 16;
    __shared__ float sq[kDeltaMaxDim], sk[kDeltaMaxDim];
    __shared__ float part[4][2][COLS];
    pdl_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slice = blockIdx.x % slices;
    const size_t rest = blockIdx.x / slices;
    const int head = static_cast<int>(rest % a.heads);
    const size_t b = rest / a.heads;
    const int k_head = head / (a.heads / a.k_heads);
    const size_t slot = a.slots ? static_cast<size_t>(static_cast<long long>(a.slots[b])) : b;
    const int col = slice * COLS + tid % 8 * VEC;
    T* o = static_cast<T*>(a.o) + (b * a.heads + head) * a.v_dim;
    if (slot >= a.pool) {                // padding: a negative slot is far above the pool as an unsigned value
        if (tid < 8)
            for (int e = 0; e < VEC; ++e)
                if (col + e < a.v_dim) o[col + e] = Convert<T, float>::store(0.f);
        return;
    }
    const size_t base = (slot * a.heads + head) * static_cast<size_t>(a.k_dim) * a.v_dim;
    float s[ROWS][VEC];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int k = r * 16 + tid / 8;
        if constexpr (VEC == 4) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < a.k_dim && col < a.v_dim)
                x = *reinterpret_cast<const float4*>(a.state + base + static_cast<size_t>(k) * a.v_dim + col);
            s[r][0] = x.x, s[r][1] = x.y, s[r][2] = x.z, s[r][3] = x.w;
        } else {
            s[r][0] = k < a.k_dim && col < a.v_dim ? a.state[base + static_cast<size_t>(k) * a.v_dim + col] : 0.f;
        }
    }
    {
        const T* q = static_cast<const T*>(a.q.p) + b * a.q.batch + k_head * a.q.head;
        const T* k = static_cast<const T*>(a.k.p) + b * a.k.batch + k_head * a.k.head;
        sq[tid] = tid < a.k_dim ? widen(q[tid]) : 0.f;
        sk[tid] = tid < a.k_dim ? widen(k[tid]) : 0.f;
    }
    const float g = gate_at(a.log_decay, a.log_decay32, b * a.log_decay.batch + head * a.log_decay.head, kTypeId<T>);
    const float beta = gate_at(a.beta, a.beta32, b * a.beta.batch + head * a.beta.head, kTypeId<T>);
    const float decay = expf(g);
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        v[e] = col + e < a.v_dim ? widen(static_cast<const T*>(a.v.p)[b * a.v.batch + head * a.v.head + col + e]) : 0.f;
    __syncthreads();
    float ks[VEC] = {}, qs[VEC] = {}, qk = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const float kr = sk[r * 16 + tid / 8], qr = sq[r * 16 + tid / 8];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            s[r][e] *= decay;
            ks[e] = fmaf(kr, s[r][e], ks[e]);
            qs[e] = fmaf(qr, s[r][e], qs[e]);
        }
    }
#pragma unroll
    for (int r = 0; r < kDeltaMaxDim / 32; ++r) qk = fmaf(sq[r * 32 + lane], sk[r * 32 + lane], qk);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) qk += __shfl_xor_sync(0xffffffffu, qk, d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        ks[e] += __shfl_xor_sync(0xffffffffu, ks[e], 8);
        qs[e] += __shfl_xor_sync(0xffffffffu, qs[e], 8);
        ks[e] += __shfl_xor_sync(0xffffffffu, ks[e], 16);
        qs[e] += __shfl_xor_sync(0xffffffffu, qs[e], 16);
        if (lane < 8) {
            part[warp][0][lane * VEC + e] = ks[e];
            part[warp][1][lane * VEC + e] = qs[e];
        }
    }
    __syncthreads();
    float u[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const int c = tid % 8 * VEC + e;
        u[e] = beta * (v[e] - (part[0][0][c] + part[1][0][c] + part[2][0][c] + part[3][0][c]));
        if (tid < 8 && col + e < a.v_dim) {
            const float before = part[0][1][c] + part[1][1][c] + part[2][1][c] + part[3][1][c];
            o[col + e] = Convert<T, float>::store(a.scale * fmaf(qk, u[e], before));
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int k = r * 16 + tid / 8;
        if (k >= a.k_dim || col >= a.v_dim) continue;
        const float kr = sk[k];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[r][e] = fmaf(kr, u[e], s[r][e]);
        float* p = a.new_state + base + static_cast<size_t>(k) * a.v_dim + col;
        if constexpr (VEC == 4)
            *reinterpret_cast<float4*>(p) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
        else
            *p = s[r][0];
    }
}

}  // namespace cubf::delta
