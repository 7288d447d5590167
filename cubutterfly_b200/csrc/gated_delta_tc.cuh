// gated_delta_tc.cuh -- the chains of the gated delta rule on the 5th-generation
// tensor cores, for 16-bit tensors (gated_delta.cuh has the mathematics).
//
// A CTA runs one sequence of one head.  The state is held transposed: a column
// of v is a lane of tensor memory, and a thread of the eight computing warps
// holds half of its lane's fp32 values in registers.  Every product has M = 128
// columns of v; its A operand (the state, beta Y, U) goes through tensor memory
// as two bf16 pieces, so what a product leaves in tensor memory is read,
// scaled, split and stored as the next one's operand without touching shared
// memory.  The B operands are 64-token tiles (q, k, L, P), which `prepare`
// leaves swizzled and bulk copies bring in, two chunks deep; one tile serves
// both ways round (tcgen05.cuh).  Of four more warps one issues the products and
// these copies, and three move rows of v in and of o out (16-byte pieces of
// strided rows: as work of the computing warps they cost 2600 of a chunk's 7000
// cycles, as bulk copies of a row each 8000).  All sides meet on mbarriers.
//
// A chunk is three dependent products, 16 MMAs of N = 64, 12 of 16 to 64 and 8
// of N = 128 on its critical path (bf16), with a read, a split and a store of
// 64 to 128 columns between them; that latency bounds a chain, and the CTAs of
// other chains fill the other SMs.
//
// bf16 inputs are one exact bf16 piece, fp16 ones two.  fp32 operands (states,
// L, P, beta Y, U) are taken as two pieces, within 2^-16 of themselves, and of
// two such operands the product of the second pieces is left out: a product is
// off by 2^-16 at most with one of them and by 3 x 2^-16 with two.  In the mean
// that is 2.5e-6 to 4e-6 of a final state or an initial one's gradient, which
// are themselves held and added up in fp32, and far below one rounding of a
// 16-bit output.  Third pieces of S, Y, U and L (in the columns that D, X and U
// leave free meanwhile) gave final states to 2e-7 to 8e-7, at 929 us for 609 of
// the prefill and 1189 for 1034 of training: not worth it beside 16-bit tensors;
// fp32 ones have them.
#pragma once

#include "f32x2.cuh"
#include "gated_delta.cuh"
#include "tcgen05.cuh"

namespace cubf::delta {

constexpr int kTcCompute = 256;          // threads of the computing warps
constexpr int kTcMovers = 96;            // ... and of those that move rows; between them, a warp that issues
constexpr int kTcThreads = kTcCompute + 32 + kTcMovers;
constexpr uint32_t kTcColumns = 512;     // all of tensor memory
constexpr int kQkPanel = 2 * tc::kPanel; // a panel of q's rows, then of k's
// Per chunk and head, 64 values each; the chains load the ones that they need, which lie side by side.
enum TcFactor : int {
    kTailBeta,                           // e^{G_64 - G} beta
    kDecay,                              // e^G
    kScaled,                             // scale e^G
    kTail,                               // e^{G_64 - G}
    kBeta,
    kDecayBeta,                          // e^G beta
    kSumHigh, kSumLow,                   // G / log 2 as a sum of two floats
    kTcFactors
};

template <typename T, int KP>
struct TcTiles {
    static constexpr int NI = kInput<T>;
    static constexpr int kOperand = NI * KP * 128;           // bytes of q or k
    static constexpr int kSquares = 2 * tc::kPanel;          // of a 64 x 64 matrix, two pieces
    static constexpr int kStage = 2 * kOperand + 2 * kSquares;
    // columns of tensor memory
    static constexpr uint32_t kX = 0, kO = 64, kD = 128, kS = 128 + KP, kY = 128 + 2 * KP, kU = 192 + 2 * KP;
    static constexpr int kHalf = KP / 2;                     // channels of a state a thread
};

template <typename T, int KP>
struct TcShared {
    using Tiles = TcTiles<T, KP>;
    alignas(1024) unsigned char stage[2][Tiles::kStage];
    alignas(16) T out[C * 128];                              // rows of o or dv on their way out
    alignas(16) float factors[2][5 * C];
    alignas(8) unsigned long long full[2], empty[2], ready[5], done[4], out_ready, out_free, drained;
    uint32_t base;
    int lost;                                                // a wait ran out
};

// ---- prepare ------------------------------------------------------------------------------------
// The tiles of a chunk, a CTA for each key head: q and k (and, backward, dO of its heads) swizzled, and for each head of
// its group L beta, (backward: beta L,) and P as two pieces each, beta folded into P's columns forward.  q k^T and k k^T
// stay in registers for the group.  L comes block by block of 16 rows, from the inverses of the blocks on the diagonal.
// What leaves by bulk copies is read while the next step computes, and v of the next head comes in meanwhile.
// Bounded by latency: 16384 tokens of 16 key and 32 value heads (bf16, K = V = 128) take 178 us forward, of which its own
// 0.82 GB would take 125.  A CTA waits 10000 of its 50000 cycles for q and k; prefetches of them a wave ahead gave nothing
// (190 us), four CTAs an SM instead of three 5 %, the triangles' blocks spread over the warps and lines instead of rows
// prefetched 15 %, fewer instructions to a decay 6 %.

template <typename T, int KP, bool BACKWARD>
struct TcPrepareShared {
    // P leaves before L is there; fp16's rows, transposed, need more
    static constexpr int kSquareTiles = !BACKWARD ? 2 : kInput<T> == 2 ? 6 : 4;
    static constexpr int kBelow = C - 16, kPitchBelow = kBelow + 8;
    static constexpr int kRowTile = 2 * tc::kPanel;              // 64 tokens by up to 128 columns of v
    static constexpr int kRowTiles = 1 + (BACKWARD ? kInput<T> : 0);
    static_assert(kRowTiles * kRowTile <= kSquareTiles * tc::kPanel, "transposed rows fit where L and P go");
    union {                                                      // one after another
        alignas(1024) unsigned char qk[2 * TcTiles<T, KP>::kOperand];
        alignas(1024) unsigned char rows[kRowTiles][kRowTile];   // v, and dO's pieces
        struct {
            alignas(16) float m[C][C + 4];                       // M
            alignas(16) __nv_bfloat16 scaled[2 * kBelow * kPitchBelow];  // M beta's blocks below the diagonal, two pieces
            alignas(16) __nv_bfloat16 inverse[2 * C * 24];       // of the 16 x 16 blocks of I + M beta on its diagonal
        } pairs;
    };
    union {
        alignas(1024) unsigned char columns[kRowTiles][kRowTile];
        alignas(1024) unsigned char squares[kSquareTiles][tc::kPanel];
    };
    alignas(16) float factors[kTcFactors][C];
    double ends[2];                                              // of two warps' sums of log decays
};
// As many CTAs an SM as shared memory allows, up to four: what registers leave to each.
template <typename T, int KP, bool BACKWARD>
constexpr int kPrepareCtas = sizeof(TcPrepareShared<T, KP, BACKWARD>) <= 55 * 1024 ? 4 : 3;

// 2^x with exp2f's error, but zero below 2^-126, as no decay of that size is told from none.
CUBF_DEV float exp2_flushed(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows of a tensor as NI swizzled pieces (one: the 16-bit values themselves), `width` (64 or 128) columns, zeros behind
// the last row and column.
template <typename T, int NI>
CUBF_DEV void load_swizzled(const T* p, size_t row, int rows, int cols, int width, bool wide, unsigned char* tile, int panel,
                            int tid, int threads) {
    const uint32_t base = smem_addr(tile), piece = static_cast<uint32_t>(width / 64 * panel);
    const int shift = width == 128 ? 4 : 3;          // vectors of eight a row
#pragma unroll 4
    for (int e = tid; e < C << shift; e += threads) {
        const int r = e >> shift, c = (e & ((1 << shift) - 1)) * 8;
        const bool ok = r < rows && c < cols;
        if (NI == 1 && wide) {
            copy16(base + tc::swizzled(r, c, panel), p + (ok ? r * row + c : 0), ok);
            continue;
        }
        Vec16<T> x;
        if (wide) {
            x = ok ? *reinterpret_cast<const Vec16<T>*>(p + r * row + c) : Vec16<T>{};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = ok && c + i < cols ? p[r * row + c + i] : Convert<T, float>::store(0.f);
        }
        if constexpr (NI == 1) {
            *reinterpret_cast<Vec16<T>*>(tile + tc::swizzled(r, c, panel)) = x;
        } else {
            uint32_t f[4][NI];
#pragma unroll
            for (int i = 0; i < 4; ++i) pieces<NI>(widen(x.v[2 * i]), widen(x.v[2 * i + 1]), f[i]);
#pragma unroll
            for (int n = 0; n < NI; ++n)
                *reinterpret_cast<uint4*>(tile + n * piece + tc::swizzled(r, c, panel)) =
                    make_uint4(f[0][n], f[1][n], f[2][n], f[3][n]);
        }
    }
}

// 64 swizzled rows of `width` 16-bit values, panels of 64 columns, to chunks of eight rows with a place of 16 bytes for each
// column (tcgen05.cuh).
CUBF_DEV void transpose_swizzled(const unsigned char* from, unsigned char* to, int width, int warp, int lane) {
    for (int b = warp; b < width / 8; b += 4) {          // eight columns: two times 32 rows
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t r[4];
            ldsm_t(smem_addr(from) + tc::swizzled(32 * h + lane, 8 * b), r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {                // rows 32 h + 8 i + 2 (lane % 4), + 1 of column 8 b + lane / 4
                const int col = 8 * b + lane / 4;
                *reinterpret_cast<uint32_t*>(to + ((4 * h + i) * width + col) * 16 + lane % 4 * 4) = r[i];
            }
        }
    }
}

// ldmatrix of a swizzled tile: the fragments of split::Tile's a_rows and b_rows.
CUBF_DEV void swizzled_a(uint32_t tile, int m, int k, int panel, int lane, uint32_t (&r)[4]) {
    ldsm(tile + tc::swizzled(m + ((lane >> 3) & 1) * 8 + (lane & 7), k + ((lane >> 4) << 3), panel), r);
}
CUBF_DEV void swizzled_b(uint32_t tile, int n, int k, int panel, int lane, uint32_t (&r)[4]) {
    ldsm(tile + tc::swizzled(n + ((lane >> 4) << 3) + (lane & 7), k + ((lane >> 3) & 1) * 8, panel), r);
}

template <typename T, int KP, bool BACKWARD>
__global__ void __launch_bounds__(128, kPrepareCtas<T, KP, BACKWARD>)
    gated_delta_tc_prepare_kernel(GatedDeltaArgs a, Places w, bool wide_q, bool wide_v, bool wide_d) {
    constexpr int NI = kInput<T>, kOperand = TcTiles<T, KP>::kOperand;
    using Shared = TcPrepareShared<T, KP, BACKWARD>;
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    Shared& sm = *reinterpret_cast<Shared*>(aligned_raw);
    pdl_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the blocks of a triangle that a warp takes, other ones in the CTAs beside it
    const int part = (warp + blockIdx.x + blockIdx.x / 148) & 3;
    const int slot = blockIdx.x / a.k_heads, k_head = blockIdx.x % a.k_heads;
    const int group = a.heads / a.k_heads;
    const Span s = span_of(a, slot);
    if (s.tokens == 0) return;
    char* const work = static_cast<char*>(a.workspace);
    auto row_of = [&](const HeadTensor& t, int head) {
        return static_cast<const T*>(t.p) + s.row * t.batch + static_cast<size_t>(s.first) * t.token +
               static_cast<size_t>(head) * t.head;
    };
    if (tid % C < s.tokens) {            // by lines: prefetches of whole rows queue up before the copies of q and k
        auto prefetch = [&](const T* p) {
            for (int at = tid / C * 64; at < a.v_dim; at += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + at));
        };
        for (int g = 0; g < group; ++g) {
            prefetch(row_of(a.v, k_head * group + g) + static_cast<size_t>(tid % C) * a.v.token);
            if (BACKWARD) prefetch(row_of(a.d_o, k_head * group + g) + static_cast<size_t>(tid % C) * a.d_o.token);
        }
    }
    auto gates = [&](int head, float& log_decay, float& beta) {  // of token `tid`
        log_decay = beta = 0.f;
        if (tid < s.tokens) {
            const size_t token = static_cast<size_t>(s.first) + tid;
            log_decay = gate_at(a.log_decay, a.log_decay32,
                                s.row * a.log_decay.batch + token * a.log_decay.token + head * a.log_decay.head, kTypeId<T>);
            beta = gate_at(a.beta, a.beta32, s.row * a.beta.batch + token * a.beta.token + head * a.beta.head, kTypeId<T>);
        }
    };
    float log_decay, beta;
    gates(k_head * group, log_decay, beta);
    load_swizzled<T, NI>(row_of(a.q, k_head), a.q.token, s.tokens, a.k_dim, KP, wide_q, sm.qk, kQkPanel, tid, 128);
    load_swizzled<T, NI>(row_of(a.k, k_head), a.k.token, s.tokens, a.k_dim, KP, wide_q, sm.qk + tc::kPanel, kQkPanel, tid, 128);
    copies_commit();
    copies_wait<0>();
    tc::fence_async();
    __syncthreads();
    if (tid == 0) {
        tc::bulk_store(work + w.packed + (static_cast<size_t>(slot) * a.k_heads + k_head) * 2 * kOperand, smem_addr(sm.qk),
                       2 * kOperand);
        tc::bulk_commit();
    }
    // The ten 16 x 16 blocks of k k^T and q k^T up to the diagonal, two or three a warp: the rows 1 to 3 of blocks to the warps
    // of their numbers, but for the first of row 3, which is with row 0.
    auto row_block = [&](int n) { return part == 0 ? 3 * n : part; };
    auto col_block = [&](int n) { return part == 0 ? 0 : part == 3 ? n + 1 : n; };
    const int blocks = part < 2 ? 2 : 3;
    float kk[6][4] = {}, qk[6][4] = {};
    const uint32_t tq = smem_addr(sm.qk), tk = tq + tc::kPanel;
#pragma unroll 2
    for (int ks = 0; ks < KP / 16; ++ks) {
        uint32_t ak[NI][4], aq[NI][4];
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            if (n >= blocks) break;
            if (n == 0 || part == 0) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    swizzled_a(tk + i * KP * 256, 16 * row_block(n), 16 * ks, kQkPanel, lane, ak[i]);
                    swizzled_a(tq + i * KP * 256, 16 * row_block(n), 16 * ks, kQkPanel, lane, aq[i]);
                }
            }
            uint32_t b[NI][1][4];
#pragma unroll
            for (int i = 0; i < NI; ++i) swizzled_b(tk + i * KP * 256, 16 * col_block(n), 16 * ks, kQkPanel, lane, b[i][0]);
            products<3, NI, NI, 2>(kk + 2 * n, ak, b);
            products<3, NI, NI, 2>(qk + 2 * n, aq, b);
        }
    }
    if (tid == 0) tc::bulk_read();
    __syncthreads();                     // q and k have left: their place is M's now
    // v, and dO, of a head
    auto fetch = [&](int head) {
        load_swizzled<T, 1>(row_of(a.v, head), a.v.token, s.tokens, a.v_dim, w.v_rows, wide_v, sm.rows[0], tc::kPanel, tid, 128);
        if constexpr (BACKWARD)
            load_swizzled<T, NI>(row_of(a.d_o, head), a.d_o.token, s.tokens, a.v_dim, w.v_rows, wide_d, sm.rows[1], tc::kPanel, tid,
                                 128);
        copies_commit();
    };
    fetch(k_head * group);
    for (int g = 0; g < group; ++g) {
        const int head = k_head * group + g;
        const size_t place = static_cast<size_t>(slot) * a.heads + head;
        double sum = 0;
        if (tid < C) {                   // running sums of the log decays, in 64 bits
            sum = log_decay < kLeast ? kLeast : log_decay;  // NaN stays
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const double other = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += other;
            }
            if (lane == 31) sm.ends[warp] = sum;
        }
        if (tid == 0) tc::bulk_read();   // the head before has left
        copies_wait<0>();
        __syncthreads();
        if (tid < C) {
            if (warp == 1) sum += sm.ends[0];
            const double all = sm.ends[0] + sm.ends[1];
            const double log2 = sum * 1.4426950408889634074;
            const float high = static_cast<float>(log2);
            const float from_start = expf(static_cast<float>(sum)), to_end = expf(static_cast<float>(all - sum));
            sm.factors[kTailBeta][tid] = to_end * beta;
            sm.factors[kDecay][tid] = from_start;
            sm.factors[kScaled][tid] = from_start * a.scale;
            sm.factors[kTail][tid] = to_end;
            sm.factors[kBeta][tid] = beta;
            sm.factors[kDecayBeta][tid] = from_start * beta;
            sm.factors[kSumHigh][tid] = high;
            sm.factors[kSumLow][tid] = static_cast<float>(log2 - high);
            if (g + 1 < group) gates(head + 1, log_decay, beta);
        }
        // to a row for each column
        const uint32_t tile = static_cast<uint32_t>(w.v_rows * 128);
        transpose_swizzled(sm.rows[0], sm.columns[0], w.v_rows, warp, lane);
        if (BACKWARD)
            for (int n = 0; n < NI; ++n)
                transpose_swizzled(sm.rows[1] + n * tile, sm.columns[1] + n * tile, w.v_rows, warp, lane);
        tc::fence_async();
        __syncthreads();
        if (tid == 0) {
            tc::bulk_store(work + w.values + place * tile, smem_addr(sm.columns[0]), tile);
            if (BACKWARD) tc::bulk_store(work + w.rows + place * NI * tile, smem_addr(sm.columns[1]), NI * tile);
            tc::bulk_commit();
        }
        const float *bf = sm.factors[kBeta], *gh = sm.factors[kSumHigh], *gl = sm.factors[kSumLow];
        // M and P; the blocks above the diagonal are never read
        uint32_t p[3][2][2][2];
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            if (n >= blocks) break;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int j = 16 * col_block(n) + 8 * t + lane % 4 * 2;
                const float2 high = *reinterpret_cast<const float2*>(gh + j), low = *reinterpret_cast<const float2*>(gl + j);
                const float2 b = *reinterpret_cast<const float2*>(bf + j);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = 16 * row_block(n) + lane / 4 + 8 * h;
                    const float dx = j <= i ? exp2_flushed((gh[i] - high.x) + (gl[i] - low.x)) : 0.f;
                    const float dy = j + 1 <= i ? exp2_flushed((gh[i] - high.y) + (gl[i] - low.y)) : 0.f;
                    const float mx = j < i ? dx * kk[2 * n + t][2 * h] : 0.f, my = j + 1 < i ? dy * kk[2 * n + t][2 * h + 1] : 0.f;
                    *reinterpret_cast<float2*>(&sm.pairs.m[i][j]) = make_float2(mx, my);
                    float px = j <= i ? dx * qk[2 * n + t][2 * h] * a.scale : 0.f;
                    float py = j + 1 <= i ? dy * qk[2 * n + t][2 * h + 1] * a.scale : 0.f;
                    if (!BACKWARD) px *= b.x, py *= b.y;
                    pieces<2>(px, py, p[n][t][h]);
                    if (row_block(n) == col_block(n)) continue;
                    uint32_t f[2];
                    pieces<2>(mx * b.x, my * b.y, f);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<uint32_t*>(sm.pairs.scaled + (e * Shared::kBelow + i - 16) * Shared::kPitchBelow + j) = f[e];
                }
            }
        }
        if (tid == 0) tc::bulk_read();
        __syncthreads();                 // v's columns have left
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            if (n >= blocks) break;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t to = tc::swizzled(16 * row_block(n) + lane / 4 + 8 * h, 16 * col_block(n) + 8 * t + lane % 4 * 2);
                    *reinterpret_cast<uint32_t*>(sm.squares[0] + to) = p[n][t][h][0];
                    *reinterpret_cast<uint32_t*>(sm.squares[1] + to) = p[n][t][h][1];
                }
        }
        tc::fence_async();
        __syncthreads();
        constexpr int L_TILES = BACKWARD ? 4 : 2;
        char* const matrices = work + w.solve + place * w.squares;
        if (tid == 0) {
            tc::bulk_store(matrices + L_TILES * tc::kPanel, smem_addr(sm.squares), 2 * tc::kPanel);
            tc::bulk_commit();
        }
        {   // the inverse of the warp's block on the diagonal, a lane a column, row by row
            const int col = lane & 15, base = 16 * part;
            float t[16];                 // times beta
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float acc[4] = {r == col ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < r; j += 4) {
                    const float4 m = *reinterpret_cast<const float4*>(&sm.pairs.m[base + r][base + j]);
                    acc[0] = fmaf(-m.x, t[j], acc[0]);
                    if (j + 1 < r) acc[1] = fmaf(-m.y, t[j + 1], acc[1]);
                    if (j + 2 < r) acc[2] = fmaf(-m.z, t[j + 2], acc[2]);
                    if (j + 3 < r) acc[3] = fmaf(-m.w, t[j + 3], acc[3]);
                }
                const float x = (acc[0] + acc[1]) + (acc[2] + acc[3]);
                t[r] = x * bf[base + r];
                float rest = x;
                if (lane < 16)
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const __nv_bfloat16 piece = __float2bfloat16_rn(rest);
                        rest -= __bfloat162float(piece);
                        sm.pairs.inverse[(n * C + base + r) * 24 + col] = piece;
                    }
            }
        }
        if (tid == 0) tc::bulk_read();
        __syncthreads();
        {   // 16 columns of L a warp, transposed, block by block of 16 rows: L_i = (I + M beta)_ii^-1 (M_i - sum over j < i
            // of (M beta)_ij L_j), products at level 2
            const Tile<Shared::kPitchBelow, Shared::kBelow * Shared::kPitchBelow> scaled{smem_addr(sm.pairs.scaled)};
            const Tile<24, C * 24> inverse{smem_addr(sm.pairs.inverse)};
            uint32_t done[3][2][4];      // rows of L before, negated, as operands
            const int c0 = 16 * part + lane / 4;
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                const int block = part + step;
                if (block > 3) break;
                float x[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[t][e] = sm.pairs.m[16 * block + 8 * t + lane % 4 * 2 + e % 2][c0 + e / 2 * 8];
#pragma unroll
                for (int j = 0; j < step; ++j) {
                    uint32_t b[2][1][4];
#pragma unroll
                    for (int n = 0; n < 2; ++n) scaled.b_rows(n, 16 * (block - 1), 16 * (part + j), lane, b[n][0]);
                    products<2, 2, 2, 2>(x, done[j], b);
                }
                uint32_t f[2][4], b[2][1][4];
                operand<2>(x[0], x[1], f);
#pragma unroll
                for (int n = 0; n < 2; ++n) inverse.b_rows(n, 16 * block, 0, lane, b[n][0]);
                float l[2][4] = {};
                products<2, 2, 2, 2>(l, f, b);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 16 * block + 8 * t + lane % 4 * 2 + e % 2, col = c0 + e / 2 * 8;
                        const uint32_t to = tc::swizzled(i, col);
                        const float c = l[t][e] * bf[col];
                        __nv_bfloat16 hi = __float2bfloat16_rn(c);
                        *reinterpret_cast<__nv_bfloat16*>(sm.squares[0] + to) = hi;
                        *reinterpret_cast<__nv_bfloat16*>(sm.squares[1] + to) = __float2bfloat16_rn(c - __bfloat162float(hi));
                        if (BACKWARD) {
                            const float r = l[t][e] * bf[i];
                            hi = __float2bfloat16_rn(r);
                            *reinterpret_cast<__nv_bfloat16*>(sm.squares[2] + to) = hi;
                            *reinterpret_cast<__nv_bfloat16*>(sm.squares[3] + to) = __float2bfloat16_rn(r - __bfloat162float(hi));
                        }
                        l[t][e] = -l[t][e];
                    }
                if (step < 3) operand<2>(l[0], l[1], done[step]);
            }
        }
        tc::fence_async();
        __syncthreads();
        if (tid == 0) {
            tc::bulk_store(matrices, smem_addr(sm.squares), L_TILES * tc::kPanel);
            tc::bulk_store(work + w.factors + place * sizeof(sm.factors), smem_addr(sm.factors), sizeof(sm.factors));
            tc::bulk_commit();
        }
        if (g + 1 < group) fetch(head + 1);
    }
    if (tid == 0) tc::bulk_done();
}

// One chain's place in the grid: a sequence of a head, or a segment of one.
struct Chain {
    int head, sequence, start, length, row, base, chunks;
    int index, segment, segments;        // place among all segments, number in the sequence, and how many that has
};
// Segments have places as chunks have: base(j) / length + j + s for segment s of sequence j.
CUBF_DEV int segments_of(int chunks, int length) { return max(1, (chunks + length - 1) / length); }
CUBF_DEV void locate(const GatedDeltaArgs& a, int sequence, Chain& c) {
    c.sequence = sequence;
    c.start = a.offsets ? offset_at(a, sequence) : 0;
    c.length = a.offsets ? max(0, offset_at(a, sequence + 1) - c.start) : a.length;
    c.row = a.offsets ? 0 : sequence;
    c.base = slot_base(a, sequence, c.start);
    c.chunks = (c.length + C - 1) / C;
}
CUBF_DEV int segment_base(const GatedDeltaArgs& a, const Segments& s, int sequence) {
    const int base = slot_base(a, sequence, a.offsets ? offset_at(a, sequence) : 0);
    return a.offsets ? base / s.length + sequence : sequence * segments_of((a.length + C - 1) / C, s.length);
}
// The sequence of `rank` among those of a packed batch by length, the longest first, so that no long chain starts last.  Each
// lane ranks two sequences, whose lengths go round by shuffles (read again by every lane they cost 2 us a CTA with 64
// sequences); beyond 64 their order stays.  16384 tokens with and without the order, random cuts: forward of 16 heads in 33
// sequences 223 us for 225 to 274, of 32 heads in 64 sequences 452 for 439 to 466; training of 8 heads in 33 sequences 656
// and 697 for 670 and 742, in 64 672 for 694 to 766.
CUBF_DEV int by_length(const GatedDeltaArgs& a, int rank) {
    if (a.sequences > 64) return rank;
    const int lane = threadIdx.x & 31;
    auto length = [&](int j) { return j < a.sequences ? max(0, offset_at(a, j + 1) - offset_at(a, j)) : -1; };
    const int mine[2] = {length(lane), length(lane + 32)};
    int before[2] = {0, 0};              // longer ones, and those as long that come first
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
        const int one = __shfl_sync(0xffffffffu, mine[0], j), two = __shfl_sync(0xffffffffu, mine[1], j);
        before[0] += (one > mine[0] || (one == mine[0] && j < lane)) + (two > mine[0]);
        before[1] += (one >= mine[1]) + (two > mine[1] || (two == mine[1] && j < lane));
    }
    const unsigned low = __ballot_sync(0xffffffffu, lane < a.sequences && before[0] == rank);
    const unsigned high = __ballot_sync(0xffffffffu, lane + 32 < a.sequences && before[1] == rank);
    return low ? __ffs(low) - 1 : high ? 31 + __ffs(high) : rank;
}
CUBF_DEV Chain chain_of(const GatedDeltaArgs& a, const Segments& s, int index) {
    Chain c{};
    c.head = index % a.heads;
    c.index = index / a.heads;
    c.segments = 1;
    if (s.length == 0) {
        locate(a, a.offsets ? by_length(a, c.index) : c.index, c);
        return c;
    }
    int low = 0, high = a.offsets ? a.sequences : a.batch;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (segment_base(a, s, mid) <= c.index)
            low = mid;
        else
            high = mid;
    }
    locate(a, low, c);
    c.segments = segments_of(c.chunks, s.length);
    c.segment = c.index - segment_base(a, s, low);
    const int first = c.segment * s.length;
    c.start += first * C;
    c.base += first;
    c.length = min(max(0, c.length - first * C), s.length * C);
    c.chunks = (c.length + C - 1) / C;
    return c;
}
// Places behind a sequence's last segment, and before the first sequence where that begins behind the first token.
CUBF_DEV bool no_segment(const Chain& c) { return c.segment < 0 || c.segment >= c.segments; }

constexpr uint32_t kLost = 0x7fff7fff;   // NaN as one fp32 value and as two fp16 or bf16 ones

// All roles of a CTA, from wherever they end.
CUBF_DEV void meet_all() { asm volatile("bar.sync 3, %0;" ::"n"(kTcThreads) : "memory"); }
// What the warp has in flight has ended, or another limit has passed: a copy into shared memory, all its products.
CUBF_DEV void drain_copy(unsigned long long& barrier, uint32_t phase) {
    for (int n = 0; n < kDeltaWaitLimit && !__all_sync(0xffffffffu, tc::barrier_try(smem_addr(&barrier), phase)); ++n) {}
}
CUBF_DEV void drain_products(unsigned long long& barrier) {
    if (tc::elect()) tc::commit(smem_addr(&barrier));
    __syncwarp();
    drain_copy(barrier, 0);
}

template <typename T, int KP>
struct TcChain {
    using Tiles = TcTiles<T, KP>;
    using Shared = TcShared<T, KP>;
    static constexpr int NI = Tiles::NI, H = Tiles::kHalf;

    const GatedDeltaArgs& a;
    const Places& w;
    Shared& sm;
    const Chain chain;
    const int tid, lane, warp, half, v;  // v: the thread's column
    uint32_t tmem, at;                   // tensor memory; with the warp's lanes
    int loads = 0;                       // of chunks, by the issuing warp
    bool failed;                         // a wait of this warp ran out

    CUBF_DEV TcChain(const GatedDeltaArgs& a, const Places& w, Shared& sm, const Chain& chain)
        : a(a), w(w), sm(sm), chain(chain), tid(threadIdx.x), lane(tid & 31), warp(__shfl_sync(0xffffffffu, tid >> 5, 0)),
          half(warp >> 2), v((warp & 3) * 32 + lane),
          // the swizzle acts on address bits; a chain without tokens waits for nothing
          failed(chain.chunks > 0 && ((smem_addr(&sm) & 1023u) != 0 || a.wait_limit == 0)) {
        if (tid == 0) {
            for (auto& b : sm.full) tc::barrier_init(smem_addr(&b), 1);
            for (auto& b : sm.done) tc::barrier_init(smem_addr(&b), 1);
            for (auto& b : sm.ready) tc::barrier_init(smem_addr(&b), kTcCompute / 32);
            for (auto& b : sm.empty) tc::barrier_init(smem_addr(&b), kTcCompute / 32 + 1);  // factors read, products done
            tc::barrier_init(smem_addr(&sm.out_ready), kTcCompute / 32);
            tc::barrier_init(smem_addr(&sm.out_free), kTcMovers / 32);
            tc::barrier_init(smem_addr(&sm.drained), 1);
            sm.lost = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (warp == kTcCompute / 32) tc::allocate(&sm.base, kTcColumns);
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
        tmem = __shfl_sync(0xffffffffu, sm.base, 0);
        at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    }
    // True where a wait of the CTA ran out.  Shared and tensor memory are then given back when the copies and products in
    // flight have ended (within another limit).
    CUBF_DEV bool finish() {
        tc::wait_load();
        tc::wait_store();
        if (failed && lane == 0) sm.lost = 1;
        tc::fence_before();
        meet_all();
        if (warp == kTcCompute / 32) {
            tc::fence_after();
            if (sm.lost) {
                for (int n = max(0, loads - 2); n < loads; ++n) drain_copy(sm.full[n & 1], (n >> 1) & 1);
                drain_products(sm.drained);
            }
            tc::release(tmem, kTcColumns);
        }
        return sm.lost;
    }
    CUBF_DEV char* work(size_t offset) const { return static_cast<char*>(a.workspace) + offset; }
    CUBF_DEV size_t place(int c) const { return static_cast<size_t>(chain.base + c) * a.heads + chain.head; }
    CUBF_DEV int tokens(int c) const { return min(C, chain.length - c * C); }
    CUBF_DEV size_t state_offset() const {
        return (static_cast<size_t>(chain.sequence) * a.heads + chain.head) * a.k_dim * a.v_dim;
    }
    CUBF_DEV size_t out_row(int c) const {   // of the first token of a chunk, in outputs
        return (static_cast<size_t>(chain.row) * a.length + chain.start + c * C) * a.heads + chain.head;
    }

    // The lanes of a warp go on alike, or give up alike.
    template <typename Barrier>
    CUBF_DEV void wait(Barrier& barrier, uint32_t phase) {
        uint32_t tries = 0;
        while (!failed && !__all_sync(0xffffffffu, tc::barrier_try(smem_addr(&barrier), phase))) failed = ++tries >= a.wait_limit;
        tc::fence_after();
    }
    // A computing warp's stores to tensor memory are seen by the products that the barrier lets be issued.
    CUBF_DEV void arrive(unsigned long long& barrier) const {
        tc::wait_store();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(smem_addr(&barrier));
    }

    CUBF_DEV void report(unsigned long long& barrier) const {
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(smem_addr(&barrier));
    }

    // ---- the issuing warp ----
    // A chunk's q and k, `squares` matrices from the `from`-th on, and `factors` rows of factors from `first` on.
    CUBF_DEV void load(int c, int s, int from, int squares, int first, int factors) {
        ++loads;
        const uint32_t bar = smem_addr(&sm.full[s]), dst = smem_addr(sm.stage[s]);
        const int k_head = chain.head / (a.heads / a.k_heads);
        const size_t tile = static_cast<size_t>(chain.base + c) * a.k_heads + k_head;
        if (tc::elect()) {
            tc::barrier_expect(bar, 2 * Tiles::kOperand + squares * Tiles::kSquares + factors * C * 4);
            tc::bulk_copy(dst, work(w.packed) + tile * 2 * Tiles::kOperand, 2 * Tiles::kOperand, bar);
            tc::bulk_copy(dst + 2 * Tiles::kOperand, work(w.solve) + place(c) * w.squares + from * Tiles::kSquares,
                          squares * Tiles::kSquares, bar);
            tc::bulk_copy(smem_addr(sm.factors[s]), work(w.factors) + (place(c) * kTcFactors + first) * C * 4, factors * C * 4,
                          bar);
        }
        __syncwarp();
    }
    CUBF_DEV uint32_t q(int s) const { return smem_addr(sm.stage[s]); }
    CUBF_DEV uint32_t k(int s) const { return q(s) + tc::kPanel; }
    CUBF_DEV uint32_t square(int s, int which) const { return q(s) + 2 * Tiles::kOperand + which * Tiles::kSquares; }

    // d (64 columns) = state (pieces in kS) times a tile of q or k, rows along N.
    CUBF_DEV void state_times(uint32_t d, uint32_t tile) const {
        constexpr uint32_t idesc = tc::instruction(64, false);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int s = 0; s < KP / 16; ++s)
                    tc::mma(tmem + d, tmem + Tiles::kS + i * (KP / 2) + 8 * s,
                            tc::rows_along_n(tile + j * KP * 256 + (s / 4) * kQkPanel + (s % 4) * 32), idesc, i + j + s > 0);
    }
    // d (KP columns) (+)= the pieces at `x` (64 tokens) times a tile of q or k, rows along K.
    CUBF_DEV void onto_state(uint32_t d, uint32_t x, uint32_t tile, bool add) const {
        constexpr uint32_t idesc = tc::instruction(KP, true);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    tc::mma(tmem + d, token_column(x, i, s), tc::rows_along_k(tile + j * KP * 256 + s * 2048, kQkPanel), idesc,
                            add || i + j + s > 0);
    }
    // Where tokens 16 s .. of piece i lie: a thread's half of the tokens stays in columns of its own.
    CUBF_DEV uint32_t token_column(uint32_t x, int i, int s) const { return tmem + x + 32 * (s / 2) + 16 * i + 8 * (s % 2); }
    // d (64 columns) = the two pieces at `x` times the lower triangular square M, at level 2: sum over j <= i of x_j M_ij,
    // rows along N.  The longest step comes first and covers d.
    CUBF_DEV void times_square(uint32_t d, uint32_t x, uint32_t square) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2 - i; ++j)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    tc::mma(tmem + d + 16 * s, token_column(x, i, s),
                            tc::rows_along_n(square + j * tc::kPanel + s * 2048 + s * 32), tc::instruction(64 - 16 * s, false),
                            i + j + s > 0);
    }

    // What the computing warps report: the state, Y, U and the output's first part are where a product takes them from or
    // may put its result.
    enum Ready { kStateReady, kYReady, kUReady, kOutTaken, kOutAdded };
    // What the products report: S k, L Y, k U, P U.
    enum Done { kSk, kLy, kKu, kPu };

    // The other way: sum over j >= i of x_j M_ji, rows along K; `pieces` of x, all with both of M (2) or at level 2 (1).
    template <int PIECES, bool EXACT>
    CUBF_DEV void times_transposed(uint32_t d, uint32_t x, uint32_t square) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < (EXACT ? 2 : 2 - i); ++j)
#pragma unroll
                for (int s = 3; s >= 0; --s)
                    tc::mma(tmem + d, token_column(x, i, s), tc::rows_along_k(square + j * tc::kPanel + s * 2048),
                            tc::instruction(16 * (s + 1), true), i + j + (3 - s) > 0);
    }

    template <bool KEEP>
    CUBF_DEV void load_forward(int c) {
        load(c, c & 1, 0, KEEP ? 1 : 2, kTailBeta, KEEP ? 2 : 3);
    }
    template <bool KEEP>
    CUBF_DEV void issue_forward() {
        const int chunks = chain.chunks;
        if (failed) return;
        if (chunks > 0) load_forward<KEEP>(0);
        if (chunks > 1) load_forward<KEEP>(1);
        uint32_t phase = 0;
        for (int c = 0; c < chunks && !failed; ++c, phase ^= 1) {
            const int st = c & 1;
            wait(sm.full[st], (c >> 1) & 1);
            wait(sm.ready[kStateReady], phase);
            if (failed) break;
            if (tc::elect()) {
                state_times(Tiles::kX, k(st));
                tc::commit(smem_addr(&sm.done[kSk]));
            }
            __syncwarp();
            if (!KEEP) {
                if (c > 0) wait(sm.ready[kOutAdded], phase ^ 1);
                if (failed) break;
                if (tc::elect()) state_times(Tiles::kO, q(st));
                __syncwarp();
            }
            wait(sm.ready[kYReady], phase);
            if (failed) break;
            if (tc::elect()) {
                times_square(Tiles::kX, Tiles::kY, square(st, 0));
                tc::commit(smem_addr(&sm.done[kLy]));
            }
            __syncwarp();
            if (c > 0 && c + 1 < chunks) {       // the stage that the chunk before has left
                wait(sm.empty[st ^ 1], ((c - 1) >> 1) & 1);
                if (failed) break;
                load_forward<KEEP>(c + 1);
            }
            wait(sm.ready[kUReady], phase);
            if (failed) break;
            if (tc::elect()) {
                onto_state(Tiles::kD, Tiles::kU, k(st), false);
                tc::commit(smem_addr(&sm.done[kKu]));
                if (KEEP) tc::commit(smem_addr(&sm.empty[st]));
            }
            __syncwarp();
            if (!KEEP) {
                wait(sm.ready[kOutTaken], phase);
                if (failed) break;
                if (tc::elect()) {
                    times_square(Tiles::kO, Tiles::kY, square(st, 1));
                    tc::commit(smem_addr(&sm.done[kPu]));
                    tc::commit(smem_addr(&sm.empty[st]));
                }
                __syncwarp();
            }
        }
    }

    // The backward's stage: q, k, beta L, P and the factors from kDecay on.
    CUBF_DEV void issue_backward() {
        const int chunks = chain.chunks;
        auto bring = [&](int n) { load(chunks - 1 - n, n & 1, 1, 2, kDecay, 5); };
        if (failed) return;
        if (chunks > 0) bring(0);
        if (chunks > 1) bring(1);
        uint32_t phase = 0;
        for (int n = 0; n < chunks && !failed; ++n, phase ^= 1) {
            const int st = n & 1;
            wait(sm.full[st], (n >> 1) & 1);
            wait(sm.ready[kStateReady], phase);
            if (failed) break;
            if (tc::elect()) {
                state_times(Tiles::kX, k(st));
                times_transposed<NI, true>(Tiles::kO, Tiles::kY, square(st, 1));
                tc::commit(smem_addr(&sm.done[kSk]));
                onto_state(Tiles::kD, Tiles::kU, q(st), false);
            }
            __syncwarp();
            wait(sm.ready[kYReady], phase);
            if (failed) break;
            if (tc::elect()) {
                times_transposed<2, false>(Tiles::kX, Tiles::kO, square(st, 0));
                tc::commit(smem_addr(&sm.done[kLy]));
            }
            __syncwarp();
            if (n > 0 && n + 1 < chunks) {
                wait(sm.empty[st ^ 1], ((n - 1) >> 1) & 1);
                if (failed) break;
                bring(n + 1);
            }
            wait(sm.ready[kUReady], phase);
            if (failed) break;
            if (tc::elect()) {
                onto_state(Tiles::kD, Tiles::kO, k(st), true);
                tc::commit(smem_addr(&sm.done[kKu]));
                tc::commit(smem_addr(&sm.empty[st]));
            }
            __syncwarp();
        }
    }

    // ---- the moving warps ----
    // 16 threads a row of 128 columns, six rows at a time; addresses advance by constants, since these warps share the
    // schedulers and instruction caches with the computing ones.  Every barrier is one of a ring: none can complete a
    // second time before its waiter has gone on.
    CUBF_DEV void store_tile(T* out, int c, bool wide) const {
        constexpr int SIDE = kTcMovers / 16, TURNS = (C + SIDE - 1) / SIDE;
        T* p = out + out_row(c) * a.v_dim;
        const size_t step = static_cast<size_t>(a.heads) * a.v_dim;
        const int n = tokens(c), first = tid - kTcCompute - 32;
        if (wide) {
            const int row = first / 16, col = first % 16 * 8, valid = col < a.v_dim ? n - row : 0;
            const T* from = sm.out + row * 128 + col;
            T* to = p + row * step + col;
#pragma unroll
            for (int i = 0; i < TURNS; ++i) {
                if (SIDE * i < valid) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from + i * SIDE * 128);
                to += SIDE * step;
            }
        } else {
            for (int e = first; e < n * 128; e += kTcMovers) {
                const int r = e / 128, col = e % 128;
                if (col < a.v_dim) p[r * step + col] = sm.out[e];
            }
        }
        report(sm.out_free);
    }
    CUBF_DEV void move_out(T* out, bool reversed, bool wide) {
        for (int n = 0; n < chain.chunks && !failed; ++n) {
            wait(sm.out_ready, n & 1);
            if (!failed) store_tile(out, reversed ? chain.chunks - 1 - n : n, wide);
        }
    }

    // ---- the computing warps ----
    // Values go in pairs: y, o and the state are packed fp32 pairs of neighbouring tokens or channels.
    using P = f32x2::P;
    static CUBF_DEV float2 widen2(uint32_t x) {
        if constexpr (std::is_same_v<T, __half>)
            return __half22float2(*reinterpret_cast<const __half2*>(&x));
        else
            return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
    static CUBF_DEV void pieces_of(P x, uint32_t& hi, uint32_t& lo) {
        float a, b;
        f32x2::up(x, a, b);
        hi = pack(a, b);
        f32x2::up(f32x2::sub2(x, f32x2::pk(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u))), a, b);
        lo = pack(a, b);
    }
    // Factors of the thread's tokens 4 g .. 4 g + 3.
    CUBF_DEV void factors_of(const float* f, int g, P& a, P& b) const {
        const float4 x = *reinterpret_cast<const float4*>(f + 32 * half + 4 * g);
        a = f32x2::pk(x.x, x.y), b = f32x2::pk(x.z, x.w);
    }
    // Where the thread's 32 tokens of a transposed tile (v or dO, R or W) lie, 16-byte chunk g of four.
    CUBF_DEV uint32_t token_chunk(int g) const {
        return static_cast<uint32_t>(((4 * half + g) * w.v_rows + v) * 16);
    }
    template <int N>
    CUBF_DEV void fetch(size_t region, int c, uint4 (&r)[N][4]) const {
        const char* p = work(region) + place(c) * N * w.v_rows * 128;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                r[n][g] = v < w.v_rows ? *reinterpret_cast<const uint4*>(p + n * w.v_rows * 128 + token_chunk(g))
                                       : make_uint4(0, 0, 0, 0);
    }
    static CUBF_DEV uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }
    // Two pieces of 32 tokens kept for the gradients.
    CUBF_DEV void keep_tokens(size_t region, int c, const P (&y)[16]) const {
        if (v < w.v_rows) {
            char* p = work(region) + place(c) * 2 * w.v_rows * 128;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pieces_of(y[4 * g + i], hi[i], lo[i]);
                *reinterpret_cast<uint4*>(p + token_chunk(g)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(p + w.v_rows * 128 + token_chunk(g)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        __syncwarp();
    }
    // 32 columns of tensor memory from `x` on, the thread's half.
    CUBF_DEV void get_tokens(uint32_t x, P (&y)[16]) const {
        uint32_t r[32];
        tc::load<32>(at + x + 32 * half, r);
        tc::wait_load();
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = f32x2::pk(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    }
    // Two pieces of the thread's 32 tokens to tensor memory, as the operand at `x`, times a factor a token.
    CUBF_DEV void put_tokens(uint32_t x, const P (&y)[16]) const {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pieces_of(y[i], hi[i], lo[i]);
        tc::store<16>(at + x + 32 * half, hi);
        tc::store<16>(at + x + 32 * half + 16, lo);
    }
    CUBF_DEV void put_tokens(uint32_t x, const P (&y)[16], const float* factor) const {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            P a, b;
            factors_of(factor, g, a, b);
            pieces_of(f32x2::mul2(y[2 * g], a), hi[2 * g], lo[2 * g]);
            pieces_of(f32x2::mul2(y[2 * g + 1], b), hi[2 * g + 1], lo[2 * g + 1]);
        }
        tc::store<16>(at + x + 32 * half, hi);
        tc::store<16>(at + x + 32 * half + 16, lo);
    }
    // The state's pieces, its thread's half, as an operand and (keep) for the gradients.
    CUBF_DEV void put_state(const P (&s)[H / 2], char* keep) const {
#pragma unroll
        for (int n = 0; n < H / 32; ++n) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) pieces_of(s[16 * n + i], hi[i], lo[i]);
            const uint32_t column = half * (H / 2) + 16 * n;
            tc::store<16>(at + Tiles::kS + column, hi);
            tc::store<16>(at + Tiles::kS + KP / 2 + column, lo);
            if (keep && v < w.v_rows) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint32_t to = kept(v, half * H + 32 * n + 8 * g);
                    *reinterpret_cast<uint4*>(keep + to) = make_uint4(hi[4 * g], hi[4 * g + 1], hi[4 * g + 2], hi[4 * g + 3]);
                    *reinterpret_cast<uint4*>(keep + to + w.state_piece) =
                        make_uint4(lo[4 * g], lo[4 * g + 1], lo[4 * g + 2], lo[4 * g + 3]);
                }
            }
            __syncwarp();
        }
    }
    // Byte of (column of v, channel) in a kept state's piece: chunks of eight channels.
    CUBF_DEV uint32_t kept(int row, int col) const { return static_cast<uint32_t>(((col >> 3) * w.v_rows + row) * 16); }
    // A state (null: zero), and where to, a row of `columns` values a channel.
    CUBF_DEV void state_in(const float* p, P (&s)[H / 2]) const {
#pragma unroll
        for (int i = 0; i < H / 2; ++i) {
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = half * H + 2 * i + e;
                x[e] = p && k < a.k_dim && v < a.v_dim ? p[static_cast<size_t>(k) * a.v_dim + v] : 0.f;
            }
            s[i] = f32x2::pk(x[0], x[1]);
        }
    }
    CUBF_DEV void state_out(float* p, int columns, const P (&s)[H / 2]) const {
#pragma unroll
        for (int i = 0; i < H / 2; ++i) {
            float x[2];
            f32x2::up(s[i], x[0], x[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = half * H + 2 * i + e;
                if (k < a.k_dim && v < columns)
                    p[static_cast<size_t>(k) * columns + v] = x[e];
            }
        }
    }
    CUBF_DEV float* end_of(size_t region, int index) const {
        return reinterpret_cast<float*>(work(region)) + (static_cast<size_t>(index) * a.heads + chain.head) * a.k_dim * a.v_dim;
    }
    CUBF_DEV float* map_of(int index) const {
        return reinterpret_cast<float*>(work(w.segments.maps)) + (static_cast<size_t>(index) * a.heads + chain.head) * KP * KP;
    }
    // S = whole S + what the products left in kD
    CUBF_DEV void state_add(float whole, P (&s)[H / 2]) const {
        uint32_t d[H];
#pragma unroll
        for (int n = 0; n < H / 32; ++n) tc::load<32>(at + Tiles::kD + half * H + 32 * n, d + 32 * n);
        tc::wait_load();
        const P w2 = f32x2::pk(whole, whole);
#pragma unroll
        for (int i = 0; i < H / 2; ++i)
            s[i] = f32x2::fma2(w2, s[i], f32x2::pk(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])));
    }
    CUBF_DEV void put_out(const P (&x)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float a, b;
            f32x2::up(x[i], a, b);
            sm.out[(32 * half + 2 * i) * 128 + v] = Convert<T, float>::store(a);
            sm.out[(32 * half + 2 * i + 1) * 128 + v] = Convert<T, float>::store(b);
        }
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(smem_addr(&sm.out_ready));
    }
    // Results of a forward run: o and the final state, or, the backward's, the state before each chunk and R, or the state
    // at the end of a segment alone, from the one before it (kEnd) or as the map of a segment (kMap: from the identity,
    // with v = 0).
    enum Mode { kOut, kKeep, kEnd, kMap };
    template <int MODE>
    CUBF_DEV void compute_forward() {
        constexpr bool OUT = MODE == kOut, KEEP = MODE == kKeep;
        P s[H / 2], y[16], x[16], o[16];
        if (MODE == kMap) {
#pragma unroll
            for (int i = 0; i < H / 2; ++i)
                s[i] = f32x2::pk(half * H + 2 * i == v && v < a.k_dim ? 1.f : 0.f, half * H + 2 * i + 1 == v && v < a.k_dim ? 1.f : 0.f);
        } else if (chain.segment == 0) {
            state_in(a.initial ? a.initial + state_offset() : nullptr, s);
        } else {
            state_in(MODE == kEnd ? nullptr : end_of(w.segments.ends, chain.index - 1), s);
        }
        const int chunks = chain.chunks;
        auto add_out = [&](int c) {          // the last part of a chunk's o
            wait(sm.done[kPu], c & 1);
            get_tokens(Tiles::kO, x);
            if (c + 1 < chunks) arrive(sm.ready[kOutAdded]);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = f32x2::add2(o[i], x[i]);
        };
        auto move_out = [&](int c) {
            if (c > 0) wait(sm.out_free, (c - 1) & 1);
            put_out(o);
        };
        uint4 rows[1][4];
        if (chunks > 0) {
            if (MODE != kMap) fetch<1>(w.values, 0, rows);
            put_state(s, KEEP ? work(w.states) + place(0) * 2 * w.state_piece : nullptr);
            arrive(sm.ready[kStateReady]);
        }
        uint32_t phase = 0;
        for (int c = 0; c < chunks && !failed; ++c, phase ^= 1) {
            const float* f = sm.factors[c & 1];
            // while the state meets k
            if (OUT && c > 0) add_out(c - 1);
            wait(sm.full[c & 1], (c >> 1) & 1);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 two = MODE == kMap ? make_float2(0.f, 0.f) : widen2(word(rows[0][i / 4], i % 4));
                y[i] = f32x2::pk(two.x, two.y);
            }
            if (MODE != kMap && c + 1 < chunks) fetch<1>(w.values, c + 1, rows);
            wait(sm.done[kSk], phase);
            get_tokens(Tiles::kX, x);
#pragma unroll
            for (int g = 0; g < 8; ++g) {    // Y = v - e^G (S k)
                P a, b;
                factors_of(f + (kDecay - kTailBeta) * C, g, a, b);
                y[2 * g] = f32x2::sub2(y[2 * g], f32x2::mul2(a, x[2 * g]));
                y[2 * g + 1] = f32x2::sub2(y[2 * g + 1], f32x2::mul2(b, x[2 * g + 1]));
            }
            put_tokens(Tiles::kY, y);
            arrive(sm.ready[kYReady]);
            if (OUT && c > 0) move_out(c - 1);  // while Y meets L
            wait(sm.done[kLy], phase);
            get_tokens(Tiles::kX, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = f32x2::sub2(y[i], x[i]);  // R = Y - (L beta) Y
            put_tokens(Tiles::kU, y, f);
            arrive(sm.ready[kUReady]);
            // while U meets k
            if (KEEP) {
                keep_tokens(w.errors, c, y);
            } else if (OUT) {
                put_tokens(Tiles::kY, y);
                get_tokens(Tiles::kO, x);
                arrive(sm.ready[kOutTaken]);
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    P a, b;
                    factors_of(f + (kScaled - kTailBeta) * C, g, a, b);
                    o[2 * g] = f32x2::mul2(a, x[2 * g]);
                    o[2 * g + 1] = f32x2::mul2(b, x[2 * g + 1]);
                }
            }
            const float whole = f[(kDecay - kTailBeta) * C + C - 1];
            report(sm.empty[c & 1]);
            wait(sm.done[kKu], phase);
            state_add(whole, s);
            put_state(s, KEEP && c + 1 < chunks ? work(w.states) + place(c + 1) * 2 * w.state_piece : nullptr);
            if (c + 1 < chunks) arrive(sm.ready[kStateReady]);
        }
        if (OUT) {
            if (chunks > 0 && !failed) {
                add_out(chunks - 1);
                move_out(chunks - 1);
            }
            if (chain.segment + 1 == chain.segments) state_out(a.last + state_offset(), a.v_dim, s);
        }
        if (MODE == kEnd) state_out(end_of(w.segments.ends, chain.index), a.v_dim, s);
        if (MODE == kMap) state_out(map_of(chain.index), KP, s);
    }

    // The sequence from its end: dS, W and dv of every chunk, or (END) dS where a segment begins alone.
    template <bool END>
    CUBF_DEV void compute_backward() {
        P s[H / 2], y[16], x[16], o[16];
        if (chain.segment + 1 == chain.segments)
            state_in(a.d_last ? a.d_last + state_offset() : nullptr, s);
        else
            state_in(END ? nullptr : end_of(w.segments.d_ends, chain.index + 1), s);
        const int chunks = chain.chunks;
        uint4 rows[NI][4];
        auto put_rows = [&] {                // dO, exactly
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                uint32_t r[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = word(rows[n][i / 4], i % 4);
                tc::store<16>(at + Tiles::kY + 32 * half + 16 * n, r);
            }
        };
        auto put_scaled = [&](const float* f) {  // scale e^G dO
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float2 two = make_float2(0.f, 0.f);
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const uint32_t r = word(rows[n][i / 4], i % 4);
                    two.x += __uint_as_float(r << 16);
                    two.y += __uint_as_float(r & 0xffff0000u);
                }
                x[i] = f32x2::pk(two.x, two.y);
            }
            put_tokens(Tiles::kU, x, f + (kScaled - kDecay) * C);
        };
        auto kept_at = [&](int n) -> char* { return END ? nullptr : work(w.d_states) + place(chunks - 1 - n) * 2 * w.state_piece; };
        if (chunks > 0) {
            fetch<NI>(w.rows, chunks - 1, rows);
            put_state(s, kept_at(0));
            put_rows();
            wait(sm.full[0], 0);
            put_scaled(sm.factors[0]);
            arrive(sm.ready[kStateReady]);
        }
        uint32_t phase = 0;
        for (int n = 0; n < chunks && !failed; ++n, phase ^= 1) {
            const int c = chunks - 1 - n;
            const float* f = sm.factors[n & 1];
            if (c > 0) fetch<NI>(w.rows, c - 1, rows);
            wait(sm.full[n & 1], (n >> 1) & 1);
            wait(sm.done[kSk], phase);
            get_tokens(Tiles::kX, x);
            get_tokens(Tiles::kO, y);
#pragma unroll
            for (int g = 0; g < 8; ++g) {    // E = e^{G_64 - G} (dS k) + P^T dO
                P a, b;
                factors_of(f + (kTail - kDecay) * C, g, a, b);
                y[2 * g] = f32x2::fma2(a, x[2 * g], y[2 * g]);
                y[2 * g + 1] = f32x2::fma2(b, x[2 * g + 1], y[2 * g + 1]);
            }
            put_tokens(Tiles::kO, y);
            arrive(sm.ready[kYReady]);
            wait(sm.done[kLy], phase);
            get_tokens(Tiles::kX, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) {   // W = E - (beta L)^T E
                y[i] = f32x2::sub2(y[i], x[i]);
                x[i] = f32x2::mul2(y[i], f32x2::pk(-1.f, -1.f));
            }
            put_tokens(Tiles::kO, x, f + (kDecayBeta - kDecay) * C);
            arrive(sm.ready[kUReady]);
            // while Z meets k
            if (!END) {
                keep_tokens(w.d_writes, c, y);
#pragma unroll
                for (int g = 0; g < 8; ++g) {    // dv = beta W
                    P a, b;
                    factors_of(f + (kBeta - kDecay) * C, g, a, b);
                    o[2 * g] = f32x2::mul2(a, y[2 * g]);
                    o[2 * g + 1] = f32x2::mul2(b, y[2 * g + 1]);
                }
                if (n > 0) wait(sm.out_free, (n - 1) & 1);
                put_out(o);
            }
            const float whole = f[C - 1];
            report(sm.empty[n & 1]);
            if (c > 0) put_rows();
            wait(sm.done[kKu], phase);
            state_add(whole, s);
            if (c > 0) {
                put_state(s, kept_at(n + 1));
                wait(sm.full[(n + 1) & 1], ((n + 1) >> 1) & 1);
                put_scaled(sm.factors[(n + 1) & 1]);
                arrive(sm.ready[kStateReady]);
            }
        }
        if (END)
            state_out(end_of(w.segments.d_ends, chain.index), a.v_dim, s);
        else if (chain.segment == 0 && a.d_initial)
            state_out(a.d_initial + state_offset(), a.v_dim, s);
    }

    // ---- where a wait ran out ----
    // NaN in all that the chain leaves, by the computing warps when every role has ended: its rows of o or dv, its states,
    // and what other kernels go by, so that nothing that comes of it passes for a result: the ends and maps of segments,
    // R (of which dq, dk and the gates' gradients come) and W (dk and the gates').
    CUBF_DEV void lose(void* p, size_t words) const {
        for (size_t e = tid; e < words; e += kTcCompute) static_cast<uint32_t*>(p)[e] = kLost;
    }
    CUBF_DEV void lose_rows(T* out) const {
        const size_t step = static_cast<size_t>(a.heads) * a.v_dim, values = static_cast<size_t>(chain.length) * a.v_dim;
        uint16_t* const p = reinterpret_cast<uint16_t*>(out + out_row(0) * a.v_dim);
        for (size_t e = tid; e < values; e += kTcCompute) p[e / a.v_dim * step + e % a.v_dim] = kLost & 0xffff;
    }
    CUBF_DEV void lose_kept(size_t region) const {
        for (int c = 0; c < chain.chunks; ++c) lose(work(region) + place(c) * 2 * w.v_rows * 128, 2 * w.v_rows * 32);
    }
    template <int MODE>
    CUBF_DEV void lose_forward() const {
        const size_t state = static_cast<size_t>(a.k_dim) * a.v_dim;
        if (MODE == kOut) {
            lose_rows(static_cast<T*>(a.o));
            if (chain.segment + 1 == chain.segments) lose(a.last + state_offset(), state);
        }
        if (MODE == kKeep) lose_kept(w.errors);
        if (MODE == kEnd) lose(end_of(w.segments.ends, chain.index), state);
        if (MODE == kMap) lose(map_of(chain.index), KP * KP);
    }
    template <bool END>
    CUBF_DEV void lose_backward() const {
        const size_t state = static_cast<size_t>(a.k_dim) * a.v_dim;
        if (END) return lose(end_of(w.segments.d_ends, chain.index), state);
        lose_rows(static_cast<T*>(a.d_v));
        lose_kept(w.d_writes);
        if (chain.segment == 0 && a.d_initial) lose(a.d_initial + state_offset(), state);
    }
};

// 224 registers for a computing thread, 56 for the others: 256 x 224 + 128 x 56 = 384 x 168, what the CTA starts with.
template <int N>
CUBF_DEV void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
CUBF_DEV void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// A chunk takes 2.4 us of its chain (K = V = 128, bf16), tensor pipe 41 % busy: 32 heads of 16384 tokens 622 us in one piece,
// 229 in three segments whose ends took 193 (1.9 to 2.2 us a chunk without outputs) and their joins 10 to 27.
template <typename T, int KP>
__global__ void __launch_bounds__(kTcThreads, 1) gated_delta_tc_forward_kernel(GatedDeltaArgs a, Places w, bool wide) {
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    pdl_begin();
    using Run = TcChain<T, KP>;
    const Chain chain = chain_of(a, w.segments, blockIdx.x);
    if (no_segment(chain)) return;
    Run run(a, w, *reinterpret_cast<TcShared<T, KP>*>(aligned_raw), chain);
    if (run.warp >= kTcCompute / 32) {
        fewer_registers<56>();
        if (run.warp == kTcCompute / 32)
            run.template issue_forward<false>();
        else
            run.move_out(static_cast<T*>(a.o), false, wide);
        run.finish();
    } else {
        more_registers<224>();
        run.template compute_forward<Run::kOut>();
        if (run.finish()) run.template lose_forward<Run::kOut>();
    }
}

// Both chains of the backward side by side: neither needs the other's results.  (One kind after the other is no faster for
// training's 128 + 128 chains on 148 SMs, 420 us against 433, and slower for packed sequences, 587 against 350, both measured
// before the chains' later steps; the 256 chains of 32 chunks take 296 now, two rounds of 4.5 us a chunk, 2.5 TB/s of writes.)
template <typename T, int KP>
__global__ void __launch_bounds__(kTcThreads, 1) gated_delta_tc_chains_kernel(GatedDeltaArgs a, Places w, bool wide) {
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    pdl_begin();
    using Run = TcChain<T, KP>;
    const Chain chain = chain_of(a, w.segments, blockIdx.x / 2);
    if (no_segment(chain)) return;
    Run run(a, w, *reinterpret_cast<TcShared<T, KP>*>(aligned_raw), chain);
    const bool reversed = blockIdx.x % 2 == 0;
    if (run.warp >= kTcCompute / 32) {
        fewer_registers<56>();
        if (run.warp == kTcCompute / 32) {
            if (reversed)
                run.issue_backward();
            else
                run.template issue_forward<true>();
        } else if (reversed) {
            run.move_out(static_cast<T*>(a.d_v), true, wide);
        }
        run.finish();
    } else {
        more_registers<224>();
        if (reversed)
            run.template compute_backward<false>();
        else
            run.template compute_forward<Run::kKeep>();
        if (!run.finish()) return;
        if (reversed)
            run.template lose_backward<false>();
        else
            run.template lose_forward<Run::kKeep>();
    }
}

// ---- segments -----------------------------------------------------------------------------------
// A chunk takes a chain from one state to the next by a map that is the same for all columns of v: S' = A S + D.  Where
// chains are few and long they are cut into segments that run side by side, twice: first each for its D (from a state of
// zero) and its A (from the identity, v = 0); then, from the states that those give, for its results.  Backward the map
// is A transposed.  The first segment starts from the true state and needs no A, the last needs nothing of the first run.
// That doubles the work and more, and is worth it where SMs would idle.
template <typename T, int KP>
__global__ void __launch_bounds__(kTcThreads, 1) gated_delta_tc_ends_kernel(GatedDeltaArgs a, Places w, int kinds) {
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    pdl_begin();
    using Run = TcChain<T, KP>;
    const int kind = blockIdx.x % kinds;                        // D, A and, backward, the reversed chain's D
    const Chain chain = chain_of(a, w.segments, blockIdx.x / kinds);
    const bool first = chain.segment == 0, last = chain.segment + 1 == chain.segments;
    if (no_segment(chain) || (kind == 2 ? first : last) || (kind == 1 && first)) return;
    Run run(a, w, *reinterpret_cast<TcShared<T, KP>*>(aligned_raw), chain);
    if (run.warp >= kTcCompute / 32) {
        fewer_registers<56>();
        if (run.warp == kTcCompute / 32) {
            if (kind == 2)
                run.issue_backward();
            else
                run.template issue_forward<true>();
        }
        run.finish();
    } else {
        more_registers<224>();
        if (kind == 0)
            run.template compute_forward<Run::kEnd>();
        else if (kind == 1)
            run.template compute_forward<Run::kMap>();
        else
            run.template compute_backward<true>();
        if (!run.finish()) return;
        if (kind == 0)
            run.template lose_forward<Run::kEnd>();
        else if (kind == 1)
            run.template lose_forward<Run::kMap>();
        else
            run.template lose_backward<true>();
    }
}

// The states where segments end, one after another, in place of the D's: a CTA takes 8 columns of a chain's state, a thread
// four columns of a row; fp32 throughout.  The next map and D are on their way in registers while one map is used.  Odd CTAs of the
// backward go through the gradients from the end.
constexpr int kJoinColumns = 8;
template <int KP>
struct JoinShared {
    alignas(16) float map[2][KP][KP + 4];
    alignas(16) float state[2][KP][kJoinColumns];
};
template <int KP>
__global__ void __launch_bounds__(2 * KP) gated_delta_join_kernel(GatedDeltaArgs a, Places w, int slices, bool backward) {
    extern __shared__ __align__(16) unsigned char raw[];
    JoinShared<KP>& sm = *reinterpret_cast<JoinShared<KP>*>(raw);
    pdl_begin();
    const int row = threadIdx.x % KP, part = threadIdx.x / KP * 4;
    int index = blockIdx.x;
    const bool reversed = backward && index % 2;
    if (backward) index /= 2;
    const int from = index % slices * kJoinColumns, head = index / slices % a.heads, sequence = index / slices / a.heads;
    Chain c{};
    locate(a, sequence, c);
    const int segments = segments_of(c.chunks, w.segments.length), base = segment_base(a, w.segments, sequence);
    if (segments < 3) return;
    char* const work = static_cast<char*>(a.workspace);
    float* const ends = reinterpret_cast<float*>(work + (reversed ? w.segments.d_ends : w.segments.ends));
    auto place = [&](int s) { return static_cast<size_t>(base + s) * a.heads + head; };
    auto row_at = [&](int s) { return ends + (place(s) * a.k_dim + row) * a.v_dim + from + part; };
    auto segment = [&](int n) { return reversed ? segments - 1 - n : n; };
    constexpr int VECTORS = KP / 8;              // of a map, a thread
    float4 next[VECTORS];
    float x[4];
    const bool own = row < a.k_dim;
    auto fetch = [&](int s) {
        const float4* m = reinterpret_cast<const float4*>(work + w.segments.maps) + place(s) * (KP * KP / 4);
#pragma unroll
        for (int e = 0; e < VECTORS; ++e) {
            const int at = threadIdx.x + e * 2 * KP;
            next[e] = at < a.k_dim * (KP / 4) ? m[at] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    auto read = [&](int s) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = own && from + part + e < a.v_dim ? row_at(s)[e] : 0.f;
    };
    read(segment(0));
    *reinterpret_cast<float4*>(&sm.state[0][row][part]) = make_float4(x[0], x[1], x[2], x[3]);
    fetch(segment(1));
    read(segment(1));
    for (int n = 1; n + 1 < segments; ++n) {
        const int now = (n - 1) & 1;
        float (*const map)[KP + 4] = sm.map[now];
#pragma unroll
        for (int e = 0; e < VECTORS; ++e) {
            const int at = threadIdx.x + e * 2 * KP;
            *reinterpret_cast<float4*>(&map[at / (KP / 4)][at % (KP / 4) * 4]) = next[e];
        }
        float sum[4] = {x[0], x[1], x[2], x[3]};
        if (n + 2 < segments) fetch(segment(n + 1)), read(segment(n + 1));
        __syncthreads();  // all have this map and state, and are past the ones that the next step writes over
#pragma unroll 4
        for (int k = 0; k < KP; k += 4) {
            float f[4];
            if (reversed) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = map[k + e][row];
            } else {
                const float4 y = *reinterpret_cast<const float4*>(&map[row][k]);
                f[0] = y.x, f[1] = y.y, f[2] = y.z, f[3] = y.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 y = *reinterpret_cast<const float4*>(&sm.state[now][k + e][part]);
                sum[0] = fmaf(f[e], y.x, sum[0]), sum[1] = fmaf(f[e], y.y, sum[1]);
                sum[2] = fmaf(f[e], y.z, sum[2]), sum[3] = fmaf(f[e], y.w, sum[3]);
            }
        }
        *reinterpret_cast<float4*>(&sm.state[now ^ 1][row][part]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (own && from + part + e < a.v_dim) row_at(segment(n))[e] = sum[e];
    }
}

// ---- gradients ----------------------------------------------------------------------------------
// A CTA per chunk and key head, the heads of its group one after another.  Products have M = 128: two operands of 64
// tokens on top of one another, q's side (lanes 0 to 63) and k's (64 to 127), so that a thread's lane is a token and
// the sums along channels and along the pairs' rows are its own:
//   [q; k] k^T      [dO; W] R^T      [dO; W] S^T      [.; R] dS^T
// then, with the pairs' coefficients Cq = D o dP and Cm = D o dM written as one tile of 128 rows,
//   [Cq; Cm] k      and, the tile turned,  [.; Cq^T q + Cm^T k].
// What has to come is the kept S and dS, 64 KB each, R and W, 32 KB each, and the tiles of q, k and dO per chunk and head;
// they fill shared memory, so a head's steps are one after another and their latency bounds it.  8 sequences of 2048 tokens,
// 16 heads (bf16, K = V = 128): 330 to 336 us, where the bytes alone take 145; 353 without the next head's prefetch to L2, and 490
// with 168 registers a thread (1 KB spilled) instead of 224 and all 32 columns of the pairs at once.
constexpr int kGradientThreads = kTcThreads;  // three warps only leave their registers to the computing ones

template <typename T, int KP>
struct GradientShared {
    static constexpr int NI = kInput<T>;
    static constexpr int kPiece = KP / 64 * 128 * 128;           // of a state
    static constexpr int kBuffers = NI == 1 ? 2 : 1;             // pieces of states in shared memory
    static constexpr int kTile = 128 * 128;                      // a piece of dO, R or W (128 columns of v by 64 tokens)
    alignas(1024) unsigned char qk[2 * TcTiles<T, KP>::kOperand];
    // dO, W, R and then the second pieces of (fp16) dO, W, R, one after another: two neighbours are one operand
    alignas(1024) unsigned char tiles[4 + NI][kTile];
    alignas(1024) unsigned char state[kBuffers][kPiece];
    alignas(1024) unsigned char pairs[NI == 1 ? 2 : 1][NI == 1 ? kTile : 16];  // pieces of Cq and Cm
    alignas(16) float factors[kTcFactors][C];
    float row[2][2][C], kept[2][C], column[4][C], dot[8], beta[C];
    double d_sum[C], all[2];
    alignas(8) unsigned long long full, state_full[kBuffers], state_empty[kBuffers], done[4], ready, free, drained;
    uint32_t base;
    int lost;                                                    // a wait ran out
    // With fp16 the pairs take dO's place, or with few columns of v the end of the tiles, which those do not reach.
    CUBF_DEV unsigned char* pair_tile(int n, int v_rows) { return NI == 1 ? pairs[n] : v_rows == 128 ? tiles[3 * n] : tiles[4 + n]; }
};

// Sums over the warp's lanes of 32 values a thread; lane l keeps that of value l.
CUBF_DEV float lane_sums(float (&x)[32], int lane) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < d; ++i) {
            const bool upper = lane & d;
            const float send = upper ? x[i] : x[i + d], keep = upper ? x[i + d] : x[i];
            x[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
        }
    return x[0];
}

template <typename T, int KP>
struct Gradients {
    using Shared = GradientShared<T, KP>;
    static constexpr int NI = Shared::NI, H = KP / 2, kOperand = TcTiles<T, KP>::kOperand;
    static constexpr uint32_t kQS = 0, kKU = KP, kPM = 2 * KP, kQK = 2 * KP + 64, kPairs = 2 * KP + 128, kTurned = kPM;
    enum Done { kPairsDone, kQsDone, kStatesDone, kAllDone };

    const GatedDeltaArgs& a;
    const Places& w;
    Shared& sm;
    const Span s;
    const int slot, k_head, group;
    const int tid, lane, warp;
    uint32_t tmem;
    bool failed = false;
    int head_loads = 0, state_loads = 0; // by the issuing warp

    template <typename Barrier>
    CUBF_DEV void wait(Barrier& barrier, uint32_t phase) {
        uint32_t tries = 0;
        while (!failed && !__all_sync(0xffffffffu, tc::barrier_try(smem_addr(&barrier), phase))) failed = ++tries >= a.wait_limit;
        tc::fence_after();
    }
    // As a chain's.
    CUBF_DEV bool finish() {
        tc::wait_load();
        if (failed && lane == 0) sm.lost = 1;
        tc::fence_before();
        meet_all();
        if (warp == kTcCompute / 32) {
            tc::fence_after();
            if (sm.lost) {
                if (head_loads > 0) drain_copy(sm.full, (head_loads - 1) & 1);
                for (int n = max(0, state_loads - Shared::kBuffers); n < state_loads; ++n)
                    drain_copy(sm.state_full[n % Shared::kBuffers], n / Shared::kBuffers & 1);
                drain_products(sm.drained);
            }
            tc::release(tmem, kTcColumns);
        }
        return sm.lost;
    }
    CUBF_DEV void lose() const {
        const size_t first = static_cast<size_t>(s.row) * a.length + s.first;
        for (int e = tid; e < s.tokens * a.k_dim; e += kTcCompute) {
            const size_t at = ((first + e / a.k_dim) * a.k_heads + k_head) * a.k_dim + e % a.k_dim;
            static_cast<uint16_t*>(a.d_q)[at] = static_cast<uint16_t*>(a.d_k)[at] = kLost & 0xffff;
        }
        for (int e = tid; e < s.tokens * group; e += kTcCompute) {
            const size_t at = (first + e / group) * a.heads + k_head * group + e % group;
            auto lose = [&](void* p, bool wide) {
                if (wide)
                    static_cast<uint32_t*>(p)[at] = kLost;
                else
                    static_cast<uint16_t*>(p)[at] = kLost & 0xffff;
            };
            lose(a.d_log_decay, a.log_decay32);
            lose(a.d_beta, a.beta32);
        }
    }
    CUBF_DEV void report(unsigned long long& barrier) const {
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(smem_addr(&barrier));
    }
    CUBF_DEV char* work(size_t offset) const { return static_cast<char*>(a.workspace) + offset; }
    CUBF_DEV size_t place(int g) const { return static_cast<size_t>(slot) * a.heads + k_head * group + g; }

    // ---- the issuing warp ----
    CUBF_DEV void load_state(int g, int n) {                     // n: S, then dS, two pieces each
        ++state_loads;
        const int b = n % Shared::kBuffers;
        const uint32_t bytes = static_cast<uint32_t>(w.state_piece);
        const char* from = work(n < 2 ? w.states : w.d_states) + (place(g) * 2 + n % 2) * w.state_piece;
        if (tc::elect()) {
            tc::barrier_expect(smem_addr(&sm.state_full[b]), bytes);
            tc::bulk_copy(smem_addr(sm.state[b]), from, bytes, smem_addr(&sm.state_full[b]));
        }
        __syncwarp();
    }
    CUBF_DEV void load_head(int g) {
        ++head_loads;
        const uint32_t bar = smem_addr(&sm.full), tile = static_cast<uint32_t>(w.v_rows * 128);
        if (tc::elect()) {
            tc::barrier_expect(bar, (g == 0 ? 2 * kOperand : 0) + (NI + 4) * tile + sizeof(sm.factors));
            if (g == 0)
                tc::bulk_copy(smem_addr(sm.qk), work(w.packed) + (static_cast<size_t>(slot) * a.k_heads + k_head) * 2 * kOperand,
                              2 * kOperand, bar);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                if (n < NI) tc::bulk_copy(stack(n), work(w.rows) + (place(g) * NI + n) * tile, tile, bar);
                tc::bulk_copy(stack(n) + tile, work(w.d_writes) + (place(g) * 2 + n) * tile, tile, bar);
                tc::bulk_copy(stack(n) + 2 * tile, work(w.errors) + (place(g) * 2 + n) * tile, tile, bar);
            }
            tc::bulk_copy(smem_addr(sm.factors), work(w.factors) + place(g) * sizeof(sm.factors), sizeof(sm.factors), bar);
        }
        __syncwarp();
    }
    // What the next head reads, or the first one of the CTA a resident wave later, to L2 while this head computes.
    CUBF_DEV void prefetch_next(int g) const {
        const unsigned next = blockIdx.x + 148;
        const uint32_t tile = static_cast<uint32_t>(w.v_rows * 128), states = 2 * static_cast<uint32_t>(w.state_piece);
        if (g + 1 == group && next >= gridDim.x) return;
        const size_t at = g + 1 < group ? place(g + 1) : static_cast<size_t>(next) * group;
        if (tc::elect()) {
            if (g + 1 == group) prefetch_l2(work(w.packed) + static_cast<size_t>(next) * 2 * kOperand, 2 * kOperand);
            prefetch_l2(work(w.rows) + at * NI * tile, NI * tile);
            prefetch_l2(work(w.d_writes) + at * 2 * tile, 2 * tile);
            prefetch_l2(work(w.errors) + at * 2 * tile, 2 * tile);
            prefetch_l2(work(w.states) + at * states, states);
            prefetch_l2(work(w.d_states) + at * states, states);
        }
        __syncwarp();
    }
    // Where piece n of [dO; W; R] begins; with bf16 dO has one piece, and what lies before W's second is not of use.
    CUBF_DEV uint32_t stack(int n) const {
        return smem_addr(sm.tiles) + static_cast<uint32_t>(n * (NI + 1) * w.v_rows * 128);
    }
    // d (n columns) (+)= two neighbouring tiles from `a` on times b over v.
    CUBF_DEV void over_v(uint32_t d, uint32_t a, uint32_t b, int n, bool add, bool only_lower) const {
        const uint32_t idesc = tc::instruction(n, true, true), chunk = static_cast<uint32_t>(w.v_rows * 16);
        for (int s = 0; s < w.v_rows / 16; ++s)
            tc::mma_shared(tmem + d, tc::chunks_along_k(a + s * 256, chunk), tc::chunks_along_k(b + s * 256, chunk), idesc,
                           add || s > 0, only_lower);
    }
    // [dO; W] b, with both pieces of the first.
    CUBF_DEV void stacked(uint32_t d, uint32_t b, int n, bool add) const {
        over_v(d, stack(0), b, n, add, false);
        over_v(d, stack(1), b, n, true, NI == 1);
    }
    CUBF_DEV void issue() {
        const uint32_t qk = smem_addr(sm.qk);
        const uint32_t tile = static_cast<uint32_t>(w.v_rows * 128);
        for (int g = 0; g < group && !failed; ++g) {
            const uint32_t phase = g & 1;
            if (g > 0) wait(sm.free, phase ^ 1);                 // the head before is done with shared memory
            if (failed) break;
            load_head(g);
            auto use = [&](int n) { return static_cast<uint32_t>(g * (4 / Shared::kBuffers) + n / Shared::kBuffers); };
            auto bring = [&](int n) {
                if (use(n) > 0) wait(sm.state_empty[n % Shared::kBuffers], (use(n) - 1) & 1);
                if (!failed) load_state(g, n);
            };
            for (int n = 0; n < Shared::kBuffers; ++n) bring(n);
            wait(sm.full, phase);
            if (failed) break;
            prefetch_next(g);
            if (tc::elect()) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j)
#pragma unroll
                        for (int s = 0; s < KP / 16; ++s) {
                            const uint32_t step = (s / 4) * kQkPanel + (s % 4) * 32;
                            tc::mma_shared(tmem + kQK, tc::rows_along_n(qk + i * KP * 256 + step),
                                           tc::rows_along_n(qk + tc::kPanel + j * KP * 256 + step), tc::instruction(64, false),
                                           i + j + s > 0);
                        }
                stacked(kPM, stack(0) + 2 * tile, 64, false);
                over_v(kPM, stack(0), stack(1) + 2 * tile, 64, true, false);
                tc::commit(smem_addr(&sm.done[kPairsDone]));
            }
            __syncwarp();
            for (int n = 0; n < 4; ++n) {
                const int b = n % Shared::kBuffers;
                wait(sm.state_full[b], use(n) & 1);
                if (failed) break;
                if (tc::elect()) {
                    const uint32_t state = smem_addr(sm.state[b]);
                    if (n == 0) stacked(kQS, state, KP, false);
                    if (n == 1) {
                        if (NI == 2)
                            stacked(kQS, state, KP, true);
                        else
                            over_v(kQS, stack(0), state, KP, true, false);
                        tc::commit(smem_addr(&sm.done[kQsDone]));
                    }
                    if (n == 2) {
                        over_v(kKU, stack(0) + tile, state, KP, false, false);
                        over_v(kKU, stack(1) + tile, state, KP, true, false);
                    }
                    if (n == 3) {
                        over_v(kKU, stack(0) + tile, state, KP, true, false);
                        tc::commit(smem_addr(&sm.done[kStatesDone]));
                    }
                    tc::commit(smem_addr(&sm.state_empty[b]));
                }
                __syncwarp();
                if (n + Shared::kBuffers < 4) bring(n + Shared::kBuffers);
            }
            wait(sm.ready, phase);                               // Cq and Cm are written, dP and q k^T read
            if (failed) break;
            if (tc::elect()) {
                constexpr uint32_t idesc = tc::instruction(KP, true), turned = tc::instruction(KP, true, true);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) {
                        const uint32_t c = smem_addr(sm.pair_tile(i, w.v_rows));
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            tc::mma_shared(tmem + kPairs, tc::rows_along_n(c + s * 32),
                                           tc::rows_along_k(qk + tc::kPanel + j * KP * 256 + s * 2048, kQkPanel), idesc,
                                           i + j + s > 0);
#pragma unroll
                        for (int s = 0; s < 8; ++s)              // lanes below 64 hold nothing of use
                            tc::mma_shared(tmem + kTurned, tc::rows_along_k(qk, c + s * 2048 - qk),
                                           tc::rows_along_k(qk + j * KP * 256 + s * 2048, kQkPanel), turned, i + j + s > 0);
                    }
                tc::commit(smem_addr(&sm.done[kAllDone]));
            }
            __syncwarp();
        }
    }

    // ---- the computing warps ----
    CUBF_DEV void compute() {
        const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, i = row & 63;
        const bool key = quarter >= 2;
        const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        float total[H];
#pragma unroll
        for (int n = 0; n < H; ++n) total[n] = 0.f;
        const size_t gate_row = static_cast<size_t>(s.row) * a.length + s.first;
        for (int g = 0; g < group; ++g) {
            const uint32_t phase = g & 1;
            const int head = k_head * group + g;
            wait(sm.full, phase);
            // the pairs' place is dO's with fp16, whose pieces of states come one at a time: all of those go first
            uint4 states[2][kShare];
            take_states(g, states);
            if (NI == 2) inner(g, states);
            wait(sm.done[kPairsDone], phase);
            {
                const float high = sm.factors[kSumHigh][i], low = sm.factors[kSumLow][i];
                const float scale = key ? -sm.factors[kBeta][i] : a.scale;
                if (NI == 2) wait(sm.done[kQsDone], phase);      // dO's place is free
                float pair[32], sum = 0.f;
#pragma unroll
                for (int part = 0; part < 2; ++part) {           // 16 columns at a time: all 32 would not stay in registers
                    const int from = 32 * half + 16 * part;
                    uint32_t x[16], kk[16];
                    tc::load<16>(at + kPM + from, x);
                    tc::load<16>(at + kQK + from, kk);
                    tc::wait_load();
                    if (key && i / 16 == 2 * half + part) {
                        float d = 0.f;                           // dbeta = W . R of the token itself
#pragma unroll
                        for (int j = 0; j < 16; ++j) d = j == i % 16 ? __uint_as_float(x[j]) : d;
                        sm.beta[i] = d;
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float c[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) c[e] = pair[16 * part + 8 * q + e] = 0.f;
                        if ((quarter & 1) == 1 || half == 0) {   // the others are all behind their row
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const int first = from + 8 * q + 4 * r;
                                const float4 h = *reinterpret_cast<const float4*>(&sm.factors[kSumHigh][first]);
                                const float4 l = *reinterpret_cast<const float4*>(&sm.factors[kSumLow][first]);
                                const float4 b = *reinterpret_cast<const float4*>(&sm.factors[kBeta][first]);
                                const float hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w}, bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int j = 8 * q + 4 * r + e, at_j = from + j;
                                    const bool in = key ? at_j < i : at_j <= i;
                                    const float d = exp2_flushed((high - hs[e]) + (low - ls[e])) * scale * bs[e] * __uint_as_float(x[j]);
                                    c[4 * r + e] = in ? d : 0.f;
                                    pair[16 * part + j] = in ? d * __uint_as_float(kk[j]) : 0.f;
                                    sum += pair[16 * part + j];
                                }
                            }
                        }
                        uint32_t f[4][2];
#pragma unroll
                        for (int e = 0; e < 4; ++e) pieces<2>(c[2 * e], c[2 * e + 1], f[e]);
                        const uint32_t to = row * 128 + (((4 * half + 2 * part + q) ^ (row & 7)) << 4);
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            *reinterpret_cast<uint4*>(sm.pair_tile(n, w.v_rows) + to) = make_uint4(f[0][n], f[1][n], f[2][n], f[3][n]);
                    }
                }
                sm.row[half][key][i] = sum;
                tc::fence_async();
                tc::fence_before();
                report(sm.ready);
                sm.column[quarter][32 * half + lane] = lane_sums(pair, lane);
            }
            if (NI == 1) inner(g, states);       // while the products with the states run
            // the states' terms, scaled, and their products with q and k
            wait(sm.done[kStatesDone], phase);
            float sum = 0.f, kept = 0.f;
            const float scale = key ? -sm.factors[kDecayBeta][i] : sm.factors[kScaled][i];
            const float tail = sm.factors[kTailBeta][i];
#pragma unroll
            for (int n = 0; n < H / 32; ++n) {
                const int channel = half * H + 32 * n;
                uint32_t x[32];
                float qk[32];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) qk[8 * q + e] = 0.f;
#pragma unroll
                    for (int p = 0; p < NI; ++p) {
                        const uint4 y = *reinterpret_cast<const uint4*>(sm.qk + p * KP * 256 + tc::swizzled(row, channel + 8 * q, kQkPanel));
                        const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            qk[8 * q + 2 * e] += __uint_as_float(z[e] << 16);
                            qk[8 * q + 2 * e + 1] += __uint_as_float(z[e] & 0xffff0000u);
                        }
                    }
                }
                tc::load<32>(at + kQS + channel, x);
                tc::wait_load();
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float y = scale * __uint_as_float(x[e]);
                    sum = fmaf(y, qk[e], sum);
                    total[32 * n + e] += y;
                }
                if (key) {
                    tc::load<32>(at + kKU + channel, x);
                    tc::wait_load();
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float y = tail * __uint_as_float(x[e]);
                        kept = fmaf(y, qk[e], kept);
                        total[32 * n + e] += y;
                    }
                }
                __syncwarp();
            }
            sm.row[half][key][i] += sum;
            if (key) sm.kept[half][i] = kept;
            meet();
            if (warp < 2) gates(head, gate_row);                 // while the last products run
            wait(sm.done[kAllDone], phase);
#pragma unroll
            for (int n = 0; n < H / 32; ++n) {
                uint32_t x[32];
                tc::load<32>(at + kPairs + half * H + 32 * n, x);
                tc::wait_load();
#pragma unroll
                for (int e = 0; e < 32; ++e) total[32 * n + e] += __uint_as_float(x[e]);
                if (key) {
                    tc::load<32>(at + kTurned + half * H + 32 * n, x);
                    tc::wait_load();
#pragma unroll
                    for (int e = 0; e < 32; ++e) total[32 * n + e] += __uint_as_float(x[e]);
                }
                __syncwarp();
            }
            tc::fence_before();
            if (g + 1 < group) meet();                           // the sums are read
            report(sm.free);
        }
        if (i < s.tokens) {
            T* out = static_cast<T*>(key ? a.d_k : a.d_q) + ((gate_row + i) * a.k_heads + k_head) * a.k_dim;
            const int first = half * H;
            const bool wide = a.k_dim % 8 == 0 && (reinterpret_cast<uintptr_t>(key ? a.d_k : a.d_q) & 15u) == 0;
#pragma unroll
            for (int n = 0; n < H; n += 8) {
                Vec16<T> x;
#pragma unroll
                for (int e = 0; e < 8; ++e) x.v[e] = Convert<T, float>::store(total[n + e]);
                if (wide) {
                    if (first + n < a.k_dim) *reinterpret_cast<Vec16<T>*>(out + first + n) = x;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (first + n + e < a.k_dim) out[first + n + e] = x.v[e];
                }
            }
        }
    }
    // <S, dS> of the thread's share, as the pieces come by: S's are kept until dS's are there.
    static constexpr int kShare = Shared::kPiece / 16 / kTcCompute;  // 16-byte chunks
    CUBF_DEV uint4 share(int g, int n, int p) const {
        const int e = tid + p * kTcCompute;
        return e * 16 < static_cast<int>(w.state_piece)
                   ? *reinterpret_cast<const uint4*>(sm.state[n % Shared::kBuffers] + e * 16)
                   : make_uint4(0, 0, 0, 0);
    }
    CUBF_DEV uint32_t use_of(int g, int n) const { return static_cast<uint32_t>(g * (4 / Shared::kBuffers) + n / Shared::kBuffers); }
    CUBF_DEV void take_states(int g, uint4 (&x)[2][kShare]) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            wait(sm.state_full[n % Shared::kBuffers], use_of(g, n) & 1);
#pragma unroll
            for (int p = 0; p < kShare; ++p) x[n][p] = share(g, n, p);
            report(sm.state_empty[n % Shared::kBuffers]);
        }
    }
    CUBF_DEV void inner(int g, const uint4 (&x)[2][kShare]) {
        float dot = 0.f;
#pragma unroll
        for (int n = 2; n < 4; ++n) {
            wait(sm.state_full[n % Shared::kBuffers], use_of(g, n) & 1);
#pragma unroll
            for (int p = 0; p < kShare; ++p) {
                const uint4 y = share(g, n, p);
                dot += product(x[0][p].x, x[1][p].x, y.x) + product(x[0][p].y, x[1][p].y, y.y) +
                       product(x[0][p].z, x[1][p].z, y.z) + product(x[0][p].w, x[1][p].w, y.w);
            }
            report(sm.state_empty[n % Shared::kBuffers]);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (lane == 0) sm.dot[warp] = dot;
    }
    // (x0 + x1) y over a pair of values
    static CUBF_DEV float product(uint32_t x0, uint32_t x1, uint32_t y) {
        const float a = __uint_as_float(x0 << 16) + __uint_as_float(x1 << 16);
        const float b = __uint_as_float(x0 & 0xffff0000u) + __uint_as_float(x1 & 0xffff0000u);
        return fmaf(a, __uint_as_float(y << 16), b * __uint_as_float(y & 0xffff0000u));
    }
    // The computing warps meet; for that they all run through every head, whatever became of a wait.
    CUBF_DEV void meet() const { asm volatile("bar.sync 1, %0;" ::"n"(kTcCompute) : "memory"); }
    // dG and its sums from each token on, in 64 bits: the terms of a sequence's first token cancel exactly.
    CUBF_DEV void gates(int head, size_t gate_row) {             // two warps
        const double kept = static_cast<double>(sm.kept[0][tid]) + sm.kept[1][tid];
        double d = static_cast<double>(sm.row[0][0][tid]) + sm.row[1][0][tid] + sm.row[0][1][tid] + sm.row[1][1][tid] - kept -
                   (static_cast<double>(sm.column[0][tid]) + sm.column[1][tid] + sm.column[2][tid] + sm.column[3][tid]);
        double all = kept;
#pragma unroll
        for (int n = 1; n < 32; n *= 2) {
            const double other = __shfl_down_sync(0xffffffffu, d, n);
            if (lane + n < 32) d += other;
            all += __shfl_xor_sync(0xffffffffu, all, n);
        }
        sm.d_sum[tid] = d;
        if (lane == 0) sm.all[warp] = all;
        asm volatile("bar.sync 2, 64;" ::: "memory");
        if (tid < s.tokens) {
            double d = sm.d_sum[tid] + (tid < 32 ? sm.d_sum[32] : 0.0);
            float inner = 0.f;
#pragma unroll
            for (int n = 0; n < 8; ++n) inner += sm.dot[n];
            d += sm.all[0] + sm.all[1] + static_cast<double>(sm.factors[kDecay][C - 1]) * inner;
            const float d_log = static_cast<float>(d);
            const size_t at = (gate_row + tid) * a.heads + head;
            if (a.log_decay32)
                static_cast<float*>(a.d_log_decay)[at] = d_log;
            else
                static_cast<T*>(a.d_log_decay)[at] = Convert<T, float>::store(d_log);
            if (a.beta32)
                static_cast<float*>(a.d_beta)[at] = sm.beta[tid];
            else
                static_cast<T*>(a.d_beta)[at] = Convert<T, float>::store(sm.beta[tid]);
        }
        __syncwarp();
    }
};

template <typename T, int KP>
__global__ void __launch_bounds__(kGradientThreads, 1) gated_delta_tc_gradients_kernel(GatedDeltaArgs a, Places w) {
    using Shared = GradientShared<T, KP>;
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    Shared& sm = *reinterpret_cast<Shared*>(aligned_raw);
    pdl_begin();
    const int slot = blockIdx.x / a.k_heads, k_head = blockIdx.x % a.k_heads;
    const Span s = span_of(a, slot);
    if (s.tokens == 0) return;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid == 0) {
        tc::barrier_init(smem_addr(&sm.full), 1);
        for (auto& b : sm.state_full) tc::barrier_init(smem_addr(&b), 1);
        for (auto& b : sm.state_empty) tc::barrier_init(smem_addr(&b), kTcCompute / 32 + 1);
        for (auto& b : sm.done) tc::barrier_init(smem_addr(&b), 1);
        tc::barrier_init(smem_addr(&sm.ready), kTcCompute / 32);
        tc::barrier_init(smem_addr(&sm.free), kTcCompute / 32);
        tc::barrier_init(smem_addr(&sm.drained), 1);
        sm.lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTcCompute / 32) tc::allocate(&sm.base, kTcColumns);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    Gradients<T, KP> run{a, w, sm, s, slot, k_head, a.heads / a.k_heads, tid, tid & 31, warp, __shfl_sync(0xffffffffu, sm.base, 0),
                         (smem_addr(&sm) & 1023u) != 0 || a.wait_limit == 0};
    if (warp >= kTcCompute / 32) {
        fewer_registers<56>();
        if (warp == kTcCompute / 32) run.issue();
        run.finish();
    } else {
        more_registers<224>();
        run.compute();
        if (run.finish()) run.lose();
    }
}

}  // namespace cubf::delta
