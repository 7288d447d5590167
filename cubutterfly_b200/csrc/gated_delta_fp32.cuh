// gated_delta_fp32.cuh -- the gated delta rule for fp32 tensors (gated_delta.cuh
// has the mathematics).
//
// Four kernels.  `prepare` (a CTA per chunk and head) makes L, P and the decay
// factors.  `chain` runs along a sequence: a warp holds 16 columns of the
// state transposed, 16 x K fp32 values in registers, as accumulator fragments
// whose layout is that of the next product's A operand, so a chunk's three
// dependent products (S k, L Y, k U) need no exchange between warps and no
// shared memory but the tiles that all warps read.  The backward runs the
// forward chain again (keeping S and R of every chunk) beside the reversed
// chain, in one launch, then `gradients` (a CTA per chunk and head); where
// heads share keys, `share` adds their gradients up.
//
// Every operand is three bf16 pieces and every product six (mma_split.cuh),
// added up in fp32 (products_rounded): 1.2e-7 to 2.7e-7 of a result against 64
// bits, and 1e-6 to 5e-6 with one accumulator through all sums, which took 57
// us for 65 (257 tokens, both chains).  Three pieces of these tiles would not
// fit beside an accumulator in tensor memory, so this path stays on the
// register-fed tensor instructions, and bounded by the latency of a chunk's
// three products in one warp, 11 us a chunk of K = 64 forward.
#pragma once

#include <algorithm>

#include "gated_delta.cuh"

namespace cubf::delta {

constexpr int kPieces = 3;               // of an fp32 value
constexpr int kSquare = C * C;           // values of L or P
// Per chunk and head: e^G, e^{G_64 - G}, beta, and G as a sum of two floats
constexpr int kFactors = 5 * C;

// ---- q and k of a chunk as bf16 pieces ----------------------------------------------------------
template <int KP>
CUBF_DEV const __nv_bfloat16* packed_at(const GatedDeltaArgs& a, const Places& w, int which, int slot, int head) {
    const size_t tile = (static_cast<size_t>(slot) * a.k_heads + head) * 2 + which;
    return reinterpret_cast<const __nv_bfloat16*>(static_cast<const char*>(a.workspace) + w.packed) + tile * kPieces * C * KP;
}
template <int KP>
CUBF_DEV void load_packed(const __nv_bfloat16* p, uint32_t tile, int tid, int threads) {
    for (int e = tid; e < kPieces * C * (KP / 8); e += threads) {
        const int row = e / (KP / 8), col = e % (KP / 8) * 8;  // rows of all pieces
        copy16(tile + static_cast<uint32_t>(row * (KP + 8) + col) * 2u, p + static_cast<size_t>(e) * 8, true);
    }
}
// All pieces of 64 x 64
CUBF_DEV void load_squares(const __nv_bfloat16* p, uint32_t tile, int tid, int threads) {
    for (int e = tid; e < kPieces * kSquare / 8; e += threads) {
        const int row = e / (C / 8), col = e % (C / 8) * 8;  // rows of all pieces
        copy16(tile + static_cast<uint32_t>(row * kPitchC + col) * 2u, p + static_cast<size_t>(e) * 8, true);
    }
}

constexpr int kSpare = 4;                // values between rows of a tile
// Rows of v or dO: `width` channels from `from` on, zeros behind the last token or channel.
CUBF_DEV void load_rows(const float* p, size_t row, int rows, int cols, int from, int width, bool wide, float* tile, int tid,
                        int threads) {
    constexpr int N = 16 / sizeof(float);
    const int pitch = width + kSpare;
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
            tile[r * pitch + c] = r < rows && from + c < cols ? p[r * row + from + c] : 0.f;
        }
    }
}

// ---- prepare ------------------------------------------------------------------------------------
// Bounded by the substitution: 64 columns of L, a thread each, 2016 FMAs with M read as 16-byte broadcasts.
template <int KP>
struct PrepareShared {
    static constexpr int kTile = kPieces * C * (KP + 8);
    alignas(16) __nv_bfloat16 q[kTile];
    alignas(16) __nv_bfloat16 k[kTile];
    alignas(16) float m[C][C];           // M beta
    float unit[C][C + 1];                // M
    double sum[C];
    float beta[C];
};

template <int KP>
CUBF_DEV void pack_rows(const GatedDeltaArgs& a, const HeadTensor& t, const Span& s, int head, __nv_bfloat16* tile,
                        __nv_bfloat16* copy, int tid) {
    const float* p = static_cast<const float*>(t.p) + s.row * t.batch + static_cast<size_t>(s.first) * t.token +
                 static_cast<size_t>(head) * t.head;
    for (int e = tid; e < C * KP / 2; e += 128) {
        const int row = e / (KP / 2), col = e % (KP / 2) * 2;
        float x = 0.f, y = 0.f;
        if (row < s.tokens) {
            const float* r = p + static_cast<size_t>(row) * t.token;
            if (col < a.k_dim) x = r[col];
            if (col + 1 < a.k_dim) y = r[col + 1];
        }
        uint32_t f[kPieces];
        pieces<kPieces>(x, y, f);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            *reinterpret_cast<uint32_t*>(tile + (i * C + row) * (KP + 8) + col) = f[i];
            if (copy) *reinterpret_cast<uint32_t*>(copy + (i * C + row) * KP + col) = f[i];
        }
    }
}

template <int KP>
__global__ void __launch_bounds__(128) gated_delta_prepare_kernel(GatedDeltaArgs a, Places w) {
    using Shared = PrepareShared<KP>;
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
               (static_cast<size_t>(slot) * a.k_heads + k_head) * 2 * kPieces * C * KP;
    pack_rows<KP>(a, a.q, s, k_head, sm.q, copy, tid);
    pack_rows<KP>(a, a.k, s, k_head, sm.k, copy ? copy + kPieces * C * KP : nullptr, tid);
    if (warp < 2) {  // running sums of the log decays, in 64 bits
        double sum = 0;
        float b = 0.f;
        if (tid < s.tokens) {
            const size_t token = static_cast<size_t>(s.first) + tid;
            const float g = static_cast<const float*>(
                a.log_decay.p)[s.row * a.log_decay.batch + token * a.log_decay.token + head * a.log_decay.head];
            sum = g < kLeast ? kLeast : g;  // NaN stays
            b = static_cast<const float*>(a.beta.p)[s.row * a.beta.batch + token * a.beta.token + head * a.beta.head];
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
        uint32_t ak[kPieces][4], aq[kPieces][4];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            tk.a_rows(i, 16 * warp, 16 * ks, lane, ak[i]);
            tq.a_rows(i, 16 * warp, 16 * ks, lane, aq[i]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t <= warp) {
                uint32_t b[kPieces][1][4];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) tk.b_rows(i, 16 * t, 16 * ks, lane, b[i][0]);
                products_rounded<3, kPieces, kPieces, 2>(kk + 2 * t, ak, b);
                products_rounded<3, kPieces, kPieces, 2>(qk + 2 * t, aq, b);
            }
        }
    }
    __nv_bfloat16* attention = reinterpret_cast<__nv_bfloat16*>(work + w.attention) + place * kPieces * kSquare;
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
            uint32_t f[kPieces];
            pieces<kPieces>(p[0], p[1], f);
#pragma unroll
            for (int n = 0; n < kPieces; ++n)
                *reinterpret_cast<uint32_t*>(attention + n * kSquare + i * C + j) = f[n];
        }
    }
    __syncthreads();
    // column `tid` of L by forward substitution: l_i = M_i - sum over j < i of (M beta)_ij l_j
    if (tid >= C) return;
    float l[C];
    __nv_bfloat16* solve = reinterpret_cast<__nv_bfloat16*>(work + w.solve) + place * kPieces * kSquare;
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
        for (int n = 0; n < kPieces; ++n) {
            const __nv_bfloat16 piece = __float2bfloat16_rn(rest);
            rest -= __bfloat162float(piece);
            solve[n * kSquare + i * C + tid] = piece;
        }
    }
}

// ---- chain --------------------------------------------------------------------------------------
// Shared memory of one chunk's tiles, for W warps (16 columns of v each).
template <int KP>
struct ChainTiles {
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + kPieces * C * (KP + 8) * 2;
    static constexpr int kSolve = kK + kPieces * C * (KP + 8) * 2;
    static constexpr int kAttention = kSolve + kPieces * C * kPitchC * 2;
    static constexpr int kFactor = kAttention + kPieces * C * kPitchC * 2;
    static constexpr int kRows = kFactor + kFactors * 4;
    static constexpr int bytes(int warps) {
        return kRows + C * (16 * warps + kSpare) * static_cast<int>(sizeof(float));
    }
};

template <int KP>
CUBF_DEV void load_chunk(const GatedDeltaArgs& a, const Places& w, const HeadTensor& rows, bool wide_rows, const Span& s,
                         int slot, int head, int from, int width, unsigned char* stage, int tid, int threads) {
    using Tiles = ChainTiles<KP>;
    const int k_head = head / (a.heads / a.k_heads);
    const size_t place = static_cast<size_t>(slot) * a.heads + head;
    char* const work = static_cast<char*>(a.workspace);
    const uint32_t base = smem_addr(stage);
    load_packed<KP>(packed_at<KP>(a, w, 0, slot, k_head), base + Tiles::kQ, tid, threads);
    load_packed<KP>(packed_at<KP>(a, w, 1, slot, k_head), base + Tiles::kK, tid, threads);
    load_squares(reinterpret_cast<const __nv_bfloat16*>(work + w.solve) + place * kPieces * kSquare,
                 base + Tiles::kSolve, tid, threads);
    load_squares(reinterpret_cast<const __nv_bfloat16*>(work + w.attention) + place * kPieces * kSquare,
                 base + Tiles::kAttention, tid, threads);
    const float* f = reinterpret_cast<const float*>(work + w.factors) + place * kFactors;
    for (int e = tid; e < kFactors / 4; e += threads) copy16(base + Tiles::kFactor + e * 16, f + e * 4, true);
    const float* p = static_cast<const float*>(rows.p) + s.row * rows.batch + static_cast<size_t>(s.first) * rows.token +
                 static_cast<size_t>(head) * rows.head;
    load_rows(p, rows.token, s.tokens, a.v_dim, from, width, wide_rows, reinterpret_cast<float*>(stage + Tiles::kRows),
                 tid, threads);
    copies_commit();
}

// The same with one factor a column.
template <int N>
CUBF_DEV void operand(const float (&a)[4], const float (&b)[4], const float* factor, float scale, int lane,
                      uint32_t (&f)[N][4]) {
    float2 lo = *reinterpret_cast<const float2*>(factor + lane % 4 * 2);
    float2 hi = *reinterpret_cast<const float2*>(factor + 8 + lane % 4 * 2);
    lo.x *= scale, lo.y *= scale, hi.x *= scale, hi.y *= scale;
    fragment<N>(a[0] * lo.x, a[1] * lo.y, a[2] * lo.x, a[3] * lo.y, b[0] * hi.x, b[1] * hi.y, b[2] * hi.x, b[3] * hi.y, f);
}

// d[0 .. N/8) += A B for a state's worth of columns: B = q or k, stored [token][channel], tokens 16 ks ..
template <int KP, typename Operand>
CUBF_DEV void onto_state(float (*d)[4], const uint32_t (&a)[kPieces][4], const Operand& b, int ks, int lane) {
#pragma unroll
    for (int t = 0; t < KP / 32; ++t) {
        uint32_t f[kPieces][2][4];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            b.b_cols(i, 16 * ks, 32 * t, lane, f[i][0]);
            b.b_cols(i, 16 * ks, 32 * t + 16, lane, f[i][1]);
        }
        products_rounded<kPieces, kPieces, kPieces, 4>(d + 4 * t, a, f);
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
// The same through the warp's own columns of a row tile to global rows `row` apart.
CUBF_DEV void rows_store(float* p, size_t row, int rows, int cols, bool wide, float* tile, int pitch, int lane,
                         const float (&x)[8][4]) {
    __syncwarp();
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            tile[(8 * t + lane % 4 * 2 + e % 2) * pitch + lane / 4 + e / 2 * 8] = x[t][e];
    __syncwarp();
    constexpr int N = 16 / sizeof(float), PER = 16 / N;
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
template <int KP, bool KEEP>
CUBF_DEV void forward_chain(const GatedDeltaArgs& a, const Places& w, const ChainShape& shape, int slice, int head,
                            int sequence, unsigned char* raw) {
    using Tiles = ChainTiles<KP>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = 32 * shape.warps;
    const int width = 16 * shape.warps, from = slice * width, v = from + 16 * warp;
    const int start = a.offsets ? offset_at(a, sequence) : 0;
    const int length = a.offsets ? max(0, offset_at(a, sequence + 1) - start) : a.length;
    const int row = a.offsets ? 0 : sequence;
    const int base = slot_base(a, sequence, start), chunks = (length + C - 1) / C;
    auto span = [&](int c) { return Span{sequence, c, start + c * C, min(C, length - c * C), row}; };
    auto load = [&](int c) {
        load_chunk<KP>(a, w, a.v, shape.wide_v, span(c), base + c, head, from, width,
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
        float* tile = reinterpret_cast<float*>(stage + Tiles::kRows) + 16 * warp;
        const int pitch = width + kSpare;
        const size_t place = static_cast<size_t>(base + c) * a.heads + head;
        char* const work = static_cast<char*>(a.workspace);
        if (v < a.v_dim) {
            if (KEEP)
                state_keep<KP>(reinterpret_cast<float*>(work + w.states) + place * w.v_pitch * KP, v, lane, s);
            float x[8][4] = {}, o[8][4] = {};
#pragma unroll
            for (int ks = 0; ks < KP / 16; ++ks) {
                uint32_t f3[kPieces][4];
                operand<kPieces>(s[2 * ks], s[2 * ks + 1], f3);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t b[kPieces][2][4];
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        k.b_rows(i, 32 * t, 16 * ks, lane, b[i][0]);
                        k.b_rows(i, 32 * t + 16, 16 * ks, lane, b[i][1]);
                    }
                    products_rounded<kPieces, kPieces, kPieces, 4>(x + 4 * t, f3, b);
                    if (!KEEP) {
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            q.b_rows(i, 32 * t, 16 * ks, lane, b[i][0]);
                            q.b_rows(i, 32 * t + 16, 16 * ks, lane, b[i][1]);
                        }
                        products_rounded<kPieces, kPieces, kPieces, 4>(o + 4 * t, f3, b);
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
                    x[t][e] = fmaf(-d, x[t][e], tile[(token + e % 2) * pitch + lane / 4 + e / 2 * 8]);
                    o[t][e] *= d * a.scale;
                }
            }
            // R = Y - L (beta Y), the later tokens' columns first: those are added to before they are read
#pragma unroll
            for (int ks = 3; ks >= 0; --ks) {
                uint32_t f3[kPieces][4];
                operand<kPieces>(x[2 * ks], x[2 * ks + 1], f + 2 * C + 16 * ks, -1.f, lane, f3);
#pragma unroll
                for (int t = ks; t < 4; ++t) {
                    uint32_t b[kPieces][1][4];
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) solve.b_rows(i, 16 * t, 16 * ks, lane, b[i][0]);
                    products_rounded<kPieces, kPieces, kPieces, 2>(x + 2 * t, f3, b);
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
                    uint32_t f2[kPieces][4];
                    operand<kPieces>(x[2 * ks], x[2 * ks + 1], f2);
#pragma unroll
                    for (int t = ks; t < 4; ++t) {
                        uint32_t b[kPieces][1][4];
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) attention.b_rows(i, 16 * t, 16 * ks, lane, b[i][0]);
                        products_rounded<kPieces, kPieces, kPieces, 2>(o + 2 * t, f2, b);
                    }
                }
                uint32_t f3[kPieces][4];
                operand<kPieces>(x[2 * ks], x[2 * ks + 1], f + C + 16 * ks, 1.f, lane, f3);
                onto_state<KP>(s, f3, k, ks, lane);
            }
            if (!KEEP) {
                const size_t token = static_cast<size_t>(row) * a.length + start + c * C;
                rows_store(static_cast<float*>(a.o) + (token * a.heads + head) * a.v_dim + v,
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
template <int KP>
CUBF_DEV void backward_chain(const GatedDeltaArgs& a, const Places& w, const ChainShape& shape, int slice, int head,
                             int sequence, unsigned char* raw) {
    using Tiles = ChainTiles<KP>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = 32 * shape.warps;
    const int width = 16 * shape.warps, from = slice * width, v = from + 16 * warp;
    const int start = a.offsets ? offset_at(a, sequence) : 0;
    const int length = a.offsets ? max(0, offset_at(a, sequence + 1) - start) : a.length;
    const int row = a.offsets ? 0 : sequence;
    const int base = slot_base(a, sequence, start), chunks = (length + C - 1) / C;
    auto load = [&](int c) {
        load_chunk<KP>(a, w, a.d_o, shape.wide_d, Span{sequence, c, start + c * C, min(C, length - c * C), row},
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
        float* tile = reinterpret_cast<float*>(stage + Tiles::kRows) + 16 * warp;
        const int pitch = width + kSpare;
        const size_t place = static_cast<size_t>(base + c) * a.heads + head;
        char* const work = static_cast<char*>(a.workspace);
        if (v < a.v_dim) {
            state_keep<KP>(reinterpret_cast<float*>(work + w.d_states) + place * w.v_pitch * KP, v, lane, s);
            float x[8][4] = {};
#pragma unroll
            for (int ks = 0; ks < KP / 16; ++ks) {
                uint32_t f3[kPieces][4];
                operand<kPieces>(s[2 * ks], s[2 * ks + 1], f3);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t b[kPieces][2][4];
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        k.b_rows(i, 32 * t, 16 * ks, lane, b[i][0]);
                        k.b_rows(i, 32 * t + 16, 16 * ks, lane, b[i][1]);
                    }
                    products_rounded<kPieces, kPieces, kPieces, 4>(x + 4 * t, f3, b);
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
                        d[t][e] = tile[(16 * ks + 8 * t + lane % 4 * 2 + e % 2) * pitch + lane / 4 + e / 2 * 8];
                uint32_t exact[kPieces][4];
                operand<kPieces>(d[0], d[1], exact);
#pragma unroll
                for (int t = 0; t <= ks; ++t) {
                    uint32_t b[kPieces][1][4];
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) attention.b_cols(i, 16 * ks, 16 * t, lane, b[i][0]);
                    products_rounded<kPieces, kPieces, kPieces, 2>(x + 2 * t, exact, b);
                }
                uint32_t f3[kPieces][4];
                operand<kPieces>(d[0], d[1], f + 16 * ks, a.scale, lane, f3);
                onto_state<KP>(s, f3, q, ks, lane);
            }
            // W = E - L^T (beta E), the earlier tokens' columns first
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                uint32_t f3[kPieces][4];
                operand<kPieces>(x[2 * ks], x[2 * ks + 1], f + 2 * C + 16 * ks, -1.f, lane, f3);
#pragma unroll
                for (int t = 0; t <= ks; ++t) {
                    uint32_t b[kPieces][1][4];
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) solve.b_cols(i, 16 * ks, 16 * t, lane, b[i][0]);
                    products_rounded<kPieces, kPieces, kPieces, 2>(x + 2 * t, f3, b);
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
                uint32_t f3[kPieces][4];
                operand<kPieces>(x[2 * ks], x[2 * ks + 1], f + 16 * ks, -1.f, lane, f3);
                onto_state<KP>(s, f3, k, ks, lane);
            }
            const size_t token = static_cast<size_t>(row) * a.length + start + c * C;
            rows_store(static_cast<float*>(a.d_v) + (token * a.heads + head) * a.v_dim + v,
                          static_cast<size_t>(a.heads) * a.v_dim, min(C, length - c * C), a.v_dim - v, shape.wide_o, tile,
                          pitch, lane, x);
        }
        __syncthreads();
        if (c > 0) load(c - 1);
    }
    if (a.d_initial && v < a.v_dim) state_store<KP>(a.d_initial + state, a.k_dim, a.v_dim, v, lane, s);
}

template <int KP>
__global__ void __launch_bounds__(256) gated_delta_forward_kernel(GatedDeltaArgs a, Places w, ChainShape shape) {
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_begin();
    const int slice = blockIdx.x % shape.slices, rest = blockIdx.x / shape.slices;
    forward_chain<KP, false>(a, w, shape, slice, rest % a.heads, rest / a.heads, raw);
}

// Both chains of the backward side by side: neither needs the other's results.
template <int KP>
__global__ void __launch_bounds__(256) gated_delta_chains_kernel(GatedDeltaArgs a, Places w, ChainShape shape) {
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_begin();
    const int slice = blockIdx.x / 2 % shape.slices, rest = blockIdx.x / 2 / shape.slices;
    if (blockIdx.x % 2 == 0)
        backward_chain<KP>(a, w, shape, slice, rest % a.heads, rest / a.heads, raw);
    else
        forward_chain<KP, true>(a, w, shape, slice, rest % a.heads, rest / a.heads, raw);
}

// ---- gradients ----------------------------------------------------------------------------------
// A CTA per chunk and head: 16 warps, warp (r, c) holds rows 16 r .. of the tokens and a quarter of the channels.
template <int KP>
struct GradientsShared {
    static constexpr int VS = 32;                    // columns of v a turn
    static constexpr int kPitchV = VS + 8;
    alignas(16) __nv_bfloat16 q[kPieces * C * (KP + 8)];
    alignas(16) __nv_bfloat16 k[kPieces * C * (KP + 8)];
    union {
        struct {
            alignas(16) __nv_bfloat16 state[kPieces * VS * (KP + 8)];     // S, transposed
            alignas(16) __nv_bfloat16 d_state[kPieces * VS * (KP + 8)];
            alignas(16) __nv_bfloat16 u[kPieces * C * kPitchV];
            alignas(16) __nv_bfloat16 z[kPieces * C * kPitchV];
            alignas(16) __nv_bfloat16 d_o[kPieces * C * kPitchV];
        } in;
        struct {
            alignas(16) __nv_bfloat16 d_p[kPieces * C * kPitchC];         // D o dP
            alignas(16) __nv_bfloat16 d_m[kPieces * C * kPitchC];         // D o dM
        } pairs;
    };
    float factors[kFactors];
    float sums[4][4][C];                             // partial sums of dG's terms by channel quarter or row block
    float dot[16];
    double d_sum[C], kept[2];
};

template <int KP>
__global__ void __launch_bounds__(512) gated_delta_gradients_kernel(GatedDeltaArgs a, Places w) {
    using Shared = GradientsShared<KP>;
    constexpr int VS = Shared::VS, PV = Shared::kPitchV;
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
    load_packed<KP>(packed_at<KP>(a, w, 0, slot, k_head), smem_addr(sm.q), tid, 512);
    load_packed<KP>(packed_at<KP>(a, w, 1, slot, k_head), smem_addr(sm.k), tid, 512);
    copies_commit();
    const float* factors = reinterpret_cast<const float*>(work + w.factors) + place * kFactors;
    if (tid < kFactors) sm.factors[tid] = factors[tid];

    const float* state = reinterpret_cast<const float*>(work + w.states) + place * w.v_pitch * KP;
    const float* d_state = reinterpret_cast<const float*>(work + w.d_states) + place * w.v_pitch * KP;
    const float* errors = reinterpret_cast<const float*>(work + w.errors) + place * C * w.v_pitch;
    const float* d_writes = reinterpret_cast<const float*>(work + w.d_writes) + place * C * w.v_pitch;
    const float* d_o = static_cast<const float*>(a.d_o.p) + s.row * a.d_o.batch + static_cast<size_t>(s.first) * a.d_o.token +
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
            uint32_t lo[kPieces], hi[kPieces];
            pieces<kPieces>(x.x, x.y, lo);
            pieces<kPieces>(x.z, x.w, hi);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                *reinterpret_cast<uint2*>(sm.in.state + (i * VS + r) * (KP + 8) + c) = make_uint2(lo[i], hi[i]);
            pieces<kPieces>(y.x, y.y, lo);
            pieces<kPieces>(y.z, y.w, hi);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
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
            uint32_t lo[kPieces], hi[kPieces];
            pieces<kPieces>(x.x * beta, x.y * beta, lo);
            pieces<kPieces>(x.z * beta, x.w * beta, hi);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                *reinterpret_cast<uint2*>(sm.in.u + (i * C + r) * PV + c) = make_uint2(lo[i], hi[i]);
            pieces<kPieces>(y.x * beta, y.y * beta, lo);
            pieces<kPieces>(y.z * beta, y.w * beta, hi);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                *reinterpret_cast<uint2*>(sm.in.z + (i * C + r) * PV + c) = make_uint2(lo[i], hi[i]);
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                d[e] = r < s.tokens && from + c + e < a.v_dim
                           ? d_o[static_cast<size_t>(r) * a.d_o.token + from + c + e]
                           : 0.f;
            uint32_t dl[kPieces], dh[kPieces];
            pieces<kPieces>(d[0], d[1], dl);
            pieces<kPieces>(d[2], d[3], dh);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                *reinterpret_cast<uint2*>(sm.in.d_o + (i * C + r) * PV + c) = make_uint2(dl[i], dh[i]);
        }
        __syncthreads();
#pragma unroll
        for (int step = 0; step < VS / 16; ++step) {
            uint32_t ao[kPieces][4], az[kPieces][4], au[kPieces][4];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) to.a_rows(i, 16 * rb, 16 * step, lane, ao[i]);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                tz.a_rows(i, 16 * rb, 16 * step, lane, az[i]);
                tu.a_rows(i, 16 * rb, 16 * step, lane, au[i]);
            }
            if (cg <= rb) {
                uint32_t b[kPieces][1][4];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) tu.b_rows(i, 16 * cg, 16 * step, lane, b[i][0]);
                products_rounded<kPieces, kPieces, kPieces, 2>(dp, ao, b);
                products_rounded<kPieces, kPieces, kPieces, 2>(dm, az, b);
            }
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                uint32_t b[kPieces][1][4];
                const int col = cg * (KP / 4) + 16 * t;
#pragma unroll
                for (int i = 0; i < kPieces; ++i) ts.b_cols(i, 16 * step, col, lane, b[i][0]);
                products_rounded<kPieces, kPieces, kPieces, 2>(qs + 2 * t, ao, b);
                products_rounded<kPieces, kPieces, kPieces, 2>(ks + 2 * t, az, b);
#pragma unroll
                for (int i = 0; i < kPieces; ++i) td.b_cols(i, 16 * step, col, lane, b[i][0]);
                products_rounded<kPieces, kPieces, kPieces, 2>(ku + 2 * t, au, b);
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
        static_cast<float*>(a.d_beta)[at] = d_beta;
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
            for (int n = 0; n < kPieces; ++n) {
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
            uint32_t aq[kPieces][4], ak[kPieces][4], b[kPieces][1][4];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                tq.a_rows(i, 16 * rb, 16 * step, lane, aq[i]);
                tk.a_rows(i, 16 * rb, 16 * step, lane, ak[i]);
                tk.b_rows(i, 16 * cg, 16 * step, lane, b[i][0]);
            }
            products_rounded<kPieces, kPieces, kPieces, 2>(qk, aq, b);
            products_rounded<kPieces, kPieces, kPieces, 2>(kk, ak, b);
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
            uint32_t f[kPieces];
            pieces<kPieces>(dp[t][2 * h], dp[t][2 * h + 1], f);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) *reinterpret_cast<uint32_t*>(sm.pairs.d_p + i * C * kPitchC + at) = f[i];
            pieces<kPieces>(dm[t][2 * h], dm[t][2 * h + 1], f);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) *reinterpret_cast<uint32_t*>(sm.pairs.d_m + i * C * kPitchC + at) = f[i];
        }
    __syncthreads();

    const Tile<kPitchC, C * kPitchC> tp{smem_addr(sm.pairs.d_p)}, tm{smem_addr(sm.pairs.d_m)};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
        uint32_t f[kPieces][4];
        if (step <= rb) {  // rows rb: tokens up to their own
            uint32_t g[kPieces][4];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                tp.a_rows(i, 16 * rb, 16 * step, lane, f[i]);
                tm.a_rows(i, 16 * rb, 16 * step, lane, g[i]);
            }
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                uint32_t b[kPieces][1][4];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) tk.b_cols(i, 16 * step, cg * (KP / 4) + 16 * t, lane, b[i][0]);
                products_rounded<kPieces, kPieces, kPieces, 2>(qs + 2 * t, f, b);
                products_rounded<kPieces, kPieces, kPieces, 2>(ks + 2 * t, g, b);
            }
        }
        if (step >= rb) {  // columns rb: tokens from their own on
            uint32_t g[kPieces][4];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                tp.a_cols(i, 16 * step, 16 * rb, lane, f[i]);
                tm.a_cols(i, 16 * step, 16 * rb, lane, g[i]);
            }
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                uint32_t b[kPieces][1][4];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) tq.b_cols(i, 16 * step, cg * (KP / 4) + 16 * t, lane, b[i][0]);
                products_rounded<kPieces, kPieces, kPieces, 2>(ks + 2 * t, f, b);
#pragma unroll
                for (int i = 0; i < kPieces; ++i) tk.b_cols(i, 16 * step, cg * (KP / 4) + 16 * t, lane, b[i][0]);
                products_rounded<kPieces, kPieces, kPieces, 2>(ks + 2 * t, g, b);
            }
        }
    }
    // where heads share keys: rows for each head, summed afterwards
    const bool shared = a.heads != a.k_heads;
    float* const dq = static_cast<float*>(shared ? static_cast<void*>(static_cast<char*>(a.workspace) + w.d_q) : a.d_q);
    float* const dk = static_cast<float*>(shared ? static_cast<void*>(static_cast<char*>(a.workspace) + w.d_k) : a.d_k);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = row + 8 * h, col = cg * (KP / 4) + 8 * t + lane % 4 * 2;
            if (i >= s.tokens) continue;
            const size_t at = ((gate_row + i) * a.heads + head) * a.k_dim + col;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (col + e < a.k_dim) {
                    dq[at + e] = qs[t][2 * h + e];
                    dk[at + e] = ks[t][2 * h + e];
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
        static_cast<float*>(a.d_log_decay)[at] = static_cast<float>(d);
    }
}

// Sums the gradients of shared keys and queries over their heads.
static __global__ void __launch_bounds__(256) gated_delta_share_kernel(GatedDeltaArgs a, Places w, size_t values) {
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
        static_cast<float*>(a.d_q)[e] = x;
        static_cast<float*>(a.d_k)[e] = y;
    }
}

}  // namespace cubf::delta
