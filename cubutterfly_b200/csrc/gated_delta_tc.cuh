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
#pragma once

#include "f32x2.cuh"
#include "gated_delta.cuh"
#include "tcgen05.cuh"

namespace cubf::delta {

constexpr int kTcCompute = 256;          // threads of the computing warps
constexpr int kTcMovers = 96;            // ... and of those that move rows; between them, a warp that issues
constexpr int kTcThreads = kTcCompute + 32 + kTcMovers;
constexpr uint32_t kTcColumns = 512;     // all of tensor memory
// Per chunk and head, 64 values each; the chains load the ones that they need, which lie side by side.
enum TcFactor : int {
    kTailBeta,                           // e^{G_64 - G} beta
    kDecay,                              // e^G
    kScaled,                             // scale e^G
    kTail,                               // e^{G_64 - G}
    kBeta,
    kDecayBeta,                          // e^G beta
    kSumHigh, kSumLow,                   // G as a sum of two floats
    kTcFactors
};

template <typename T, int KP>
struct TcTiles {
    static constexpr int NI = kInput<T>;
    static constexpr int kOperand = NI * KP * 128;           // bytes of q or k
    static constexpr int kSquares = 2 * tc::kPanel;          // of L beta or P beta, two pieces
    static constexpr int kStage = 2 * kOperand + 2 * kSquares;
    // columns of tensor memory
    static constexpr uint32_t kX = 0, kO = 64, kD = 128, kS = 128 + KP, kY = 128 + 2 * KP, kU = 192 + 2 * KP;
    static constexpr int kHalf = KP / 2;                     // channels of a state a thread
};

template <typename T, int KP>
struct TcShared {
    using Tiles = TcTiles<T, KP>;
    alignas(1024) unsigned char stage[2][Tiles::kStage];
    alignas(16) T rows[C * 128];                             // v of a chunk
    alignas(16) T out[C * 128];                              // o of a chunk
    alignas(16) float factors[2][3 * C];                     // kTailBeta, kDecay, kScaled
    alignas(8) unsigned long long full[2], empty[2], ready[5], done[4], rows_full, rows_empty, out_ready, out_free;
    uint32_t base;
};

// ---- prepare ------------------------------------------------------------------------------------
// The tiles of a chunk, a CTA for each key head: q and k (and, backward, dO of its heads) swizzled, and for each head of
// its group L beta, (backward: beta L,) and P as two pieces each, beta folded into P's columns forward.  q k^T and k k^T
// stay in registers for the group.  L is solved column by column, two threads a column.

template <typename T, int KP, bool BACKWARD>
struct TcPrepareShared {
    static constexpr int kOperand = TcTiles<T, KP>::kOperand;
    static constexpr int kSquareTiles = BACKWARD ? 6 : 4;
    static constexpr int kRows = kInput<T> * 2 * tc::kPanel;     // dO: up to 128 columns
    union {
        struct {
            alignas(1024) unsigned char q[kOperand];
            alignas(1024) unsigned char k[kOperand];
        } in;
        struct {
            alignas(1024) float m[C][C];     // M beta
            alignas(1024) float unit[C][C];  // M
        } pairs;
    };
    alignas(1024) unsigned char squares[kSquareTiles][tc::kPanel];
    alignas(1024) unsigned char rows[BACKWARD ? kRows : 16];
    double sum[C];
    alignas(16) float factors[kTcFactors][C];
};

// Rows of a tensor as swizzled pieces, `width` (64 or 128) columns, zeros behind the last row and column.
template <typename T>
CUBF_DEV void load_swizzled(const T* p, size_t row, int rows, int cols, int width, bool wide, unsigned char* tile, int tid,
                            int threads) {
    constexpr int NI = kInput<T>;
    const uint32_t base = smem_addr(tile), piece = static_cast<uint32_t>(width / 64 * tc::kPanel);
    const int per = width / 8;
#pragma unroll 4
    for (int e = tid; e < C * per; e += threads) {
        const int r = e / per, c = e % per * 8;
        const bool ok = r < rows && c < cols;
        if (NI == 1 && wide) {
            copy16(base + tc::swizzled(r, c), p + (ok ? r * row + c : 0), ok);
            continue;
        }
        float x[8];
        if (wide) {
            Vec16<T> v{};
            if (ok) v = *reinterpret_cast<const Vec16<T>*>(p + r * row + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = widen(v.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = ok && c + i < cols ? widen(p[r * row + c + i]) : 0.f;
        }
        uint32_t f[4][NI];
#pragma unroll
        for (int i = 0; i < 4; ++i) pieces<NI>(x[2 * i], x[2 * i + 1], f[i]);
#pragma unroll
        for (int n = 0; n < NI; ++n)
            *reinterpret_cast<uint4*>(tile + n * piece + tc::swizzled(r, c)) = make_uint4(f[0][n], f[1][n], f[2][n], f[3][n]);
    }
}

// ldmatrix of a swizzled tile: the fragments of split::Tile's a_rows and b_rows.
CUBF_DEV void swizzled_a(uint32_t tile, int m, int k, int lane, uint32_t (&r)[4]) {
    ldsm(tile + tc::swizzled(m + ((lane >> 3) & 1) * 8 + (lane & 7), k + ((lane >> 4) << 3)), r);
}
CUBF_DEV void swizzled_b(uint32_t tile, int n, int k, int lane, uint32_t (&r)[4]) {
    ldsm(tile + tc::swizzled(n + ((lane >> 4) << 3) + (lane & 7), k + ((lane >> 3) & 1) * 8), r);
}

template <typename T, int KP, bool BACKWARD>
__global__ void __launch_bounds__(128) gated_delta_tc_prepare_kernel(GatedDeltaArgs a, Places w, bool wide_q, bool wide_d) {
    constexpr int NI = kInput<T>, kOperand = TcTiles<T, KP>::kOperand;
    using Shared = TcPrepareShared<T, KP, BACKWARD>;
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    Shared& sm = *reinterpret_cast<Shared*>(aligned_raw);
    pdl_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = blockIdx.x / a.k_heads, k_head = blockIdx.x % a.k_heads;
    const int group = a.heads / a.k_heads;
    const Span s = span_of(a, slot);
    if (s.tokens == 0) return;
    char* const work = static_cast<char*>(a.workspace);
    auto row_of = [&](const HeadTensor& t, int head) {
        return static_cast<const T*>(t.p) + s.row * t.batch + static_cast<size_t>(s.first) * t.token +
               static_cast<size_t>(head) * t.head;
    };
    load_swizzled<T>(row_of(a.q, k_head), a.q.token, s.tokens, a.k_dim, KP, wide_q, sm.in.q, tid, 128);
    load_swizzled<T>(row_of(a.k, k_head), a.k.token, s.tokens, a.k_dim, KP, wide_q, sm.in.k, tid, 128);
    copies_commit();
    copies_wait<0>();
    tc::fence_async();
    __syncthreads();
    if (tid == 0) {
        char* to = work + w.packed + (static_cast<size_t>(slot) * a.k_heads + k_head) * 2 * kOperand;
        tc::bulk_store(to, smem_addr(sm.in.q), kOperand);
        tc::bulk_store(to + kOperand, smem_addr(sm.in.k), kOperand);
        tc::bulk_commit();
    }
    // rows 16 warp .. + 15 of k k^T and q k^T, up to the diagonal
    float kk[8][4] = {}, qk[8][4] = {};
    const uint32_t tq = smem_addr(sm.in.q), tk = smem_addr(sm.in.k);
    for (int ks = 0; ks < KP / 16; ++ks) {
        uint32_t ak[NI][4], aq[NI][4];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            swizzled_a(tk + i * KP * 128, 16 * warp, 16 * ks, lane, ak[i]);
            swizzled_a(tq + i * KP * 128, 16 * warp, 16 * ks, lane, aq[i]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t <= warp) {
                uint32_t b[NI][1][4];
#pragma unroll
                for (int i = 0; i < NI; ++i) swizzled_b(tk + i * KP * 128, 16 * t, 16 * ks, lane, b[i][0]);
                products<3, NI, NI, 2>(kk + 2 * t, ak, b);
                products<3, NI, NI, 2>(qk + 2 * t, aq, b);
            }
        }
    }
    if (tid == 0) tc::bulk_read();
    __syncthreads();                     // q and k have left: their place is M's now
    for (int g = 0; g < group; ++g) {
        const int head = k_head * group + g;
        const size_t place = static_cast<size_t>(slot) * a.heads + head;
        if (BACKWARD) {
            const int width = w.v_rows;
            load_swizzled<T>(row_of(a.d_o, head), a.d_o.token, s.tokens, a.v_dim, width, wide_d, sm.rows, tid, 128);
            copies_commit();
        }
        double sum = 0;
        float beta = 0.f;
        if (tid < C) {                   // running sums of the log decays, in 64 bits
            if (tid < s.tokens) {
                const size_t token = static_cast<size_t>(s.first) + tid;
                const float d = gate_at(a.log_decay, a.log_decay32,
                                        s.row * a.log_decay.batch + token * a.log_decay.token + head * a.log_decay.head,
                                        kTypeId<T>);
                sum = d < kLeast ? kLeast : d;  // NaN stays
                beta = gate_at(a.beta, a.beta32, s.row * a.beta.batch + token * a.beta.token + head * a.beta.head, kTypeId<T>);
            }
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const double other = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += other;
            }
            sm.sum[tid] = sum;
        }
        __syncthreads();
        if (tid < C) {
            if (warp == 1) sum += sm.sum[31];
            const double all = sm.sum[31] + sm.sum[63];
            const float high = static_cast<float>(sum), from_start = expf(high), to_end = expf(static_cast<float>(all - sum));
            sm.factors[kTailBeta][tid] = to_end * beta;
            sm.factors[kDecay][tid] = from_start;
            sm.factors[kScaled][tid] = from_start * a.scale;
            sm.factors[kTail][tid] = to_end;
            sm.factors[kBeta][tid] = beta;
            sm.factors[kDecayBeta][tid] = from_start * beta;
            sm.factors[kSumHigh][tid] = high;
            sm.factors[kSumLow][tid] = static_cast<float>(sum - high);
        }
        __syncthreads();
        const float *bf = sm.factors[kBeta], *gh = sm.factors[kSumHigh], *gl = sm.factors[kSumLow];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 16 * warp + lane / 4 + 8 * h, j = 8 * t + lane % 4 * 2;
                float p[2], m[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float d = j + e <= i ? expf((gh[i] - gh[j + e]) + (gl[i] - gl[j + e])) : 0.f;
                    p[e] = j + e <= i ? d * qk[t][2 * h + e] * a.scale : 0.f;
                    m[e] = j + e < i ? d * kk[t][2 * h + e] : 0.f;
                    if (!BACKWARD) p[e] *= bf[j + e];
                }
                *reinterpret_cast<float2*>(&sm.pairs.unit[i][j]) = make_float2(m[0], m[1]);
                *reinterpret_cast<float2*>(&sm.pairs.m[i][j]) = make_float2(m[0] * bf[j], m[1] * bf[j + 1]);
                uint32_t f[2];
                pieces<2>(p[0], p[1], f);
                constexpr int at = BACKWARD ? 4 : 2;
                *reinterpret_cast<uint32_t*>(sm.squares[at] + tc::swizzled(i, j)) = f[0];
                *reinterpret_cast<uint32_t*>(sm.squares[at + 1] + tc::swizzled(i, j)) = f[1];
            }
        }
        __syncthreads();
        // column tid / 2 of L by forward substitution: l_i = M_i - sum over j < i of (M beta)_ij l_j, every other four
        // values of j a thread
        {
            const int col = tid / 2, part = tid % 2;
            const float beta_col = bf[col];
            float l[C / 2] = {};         // the thread's own l_j; what is not known yet meets zeros of M
#pragma unroll
            for (int i = 0; i < C; ++i) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < i; j += 8) {
                    const float4 m = *reinterpret_cast<const float4*>(&sm.pairs.m[i][j + 4 * part]);
                    acc[0] = fmaf(-m.x, l[j / 2], acc[0]);
                    acc[1] = fmaf(-m.y, l[j / 2 + 1], acc[1]);
                    acc[2] = fmaf(-m.z, l[j / 2 + 2], acc[2]);
                    acc[3] = fmaf(-m.w, l[j / 2 + 3], acc[3]);
                }
                float x = (acc[0] + acc[1]) + (acc[2] + acc[3]);
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += sm.pairs.unit[i][col];
                if (i / 4 % 2 == part) l[i / 8 * 4 + i % 4] = x;
                if (i % 2 == part) {
                    const float c = x * beta_col;
                    __nv_bfloat16 hi = __float2bfloat16_rn(c);
                    const uint32_t to = tc::swizzled(i, col);
                    *reinterpret_cast<__nv_bfloat16*>(sm.squares[0] + to) = hi;
                    *reinterpret_cast<__nv_bfloat16*>(sm.squares[1] + to) = __float2bfloat16_rn(c - __bfloat162float(hi));
                    if (BACKWARD) {
                        const float r = x * bf[i];
                        hi = __float2bfloat16_rn(r);
                        *reinterpret_cast<__nv_bfloat16*>(sm.squares[2] + to) = hi;
                        *reinterpret_cast<__nv_bfloat16*>(sm.squares[3] + to) = __float2bfloat16_rn(r - __bfloat162float(hi));
                    }
                }
            }
        }
        if (BACKWARD) copies_wait<0>();
        tc::fence_async();
        __syncthreads();
        if (tid == 0) {
            tc::bulk_store(work + w.solve + place * sizeof(sm.squares), smem_addr(sm.squares), sizeof(sm.squares));
            tc::bulk_store(work + w.factors + place * sizeof(sm.factors), smem_addr(sm.factors), sizeof(sm.factors));
            if (BACKWARD) {
                const uint32_t bytes = static_cast<uint32_t>(NI * w.v_rows * 128);
                tc::bulk_store(work + w.rows + place * bytes, smem_addr(sm.rows), bytes);
            }
            tc::bulk_commit();
            if (g + 1 < group)
                tc::bulk_read();
            else
                tc::bulk_done();
        }
        __syncthreads();
    }
}

// One chain's place in the grid.
struct Chain {
    int head, sequence, start, length, row, base, chunks;
};
CUBF_DEV Chain chain_of(const GatedDeltaArgs& a, int index) {
    Chain c;
    c.head = index % a.heads;
    c.sequence = index / a.heads;
    c.start = a.offsets ? offset_at(a, c.sequence) : 0;
    c.length = a.offsets ? max(0, offset_at(a, c.sequence + 1) - c.start) : a.length;
    c.row = a.offsets ? 0 : c.sequence;
    c.base = slot_base(a, c.sequence, c.start);
    c.chunks = (c.length + C - 1) / C;
    return c;
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
    bool failed;

    CUBF_DEV TcChain(const GatedDeltaArgs& a, const Places& w, Shared& sm, const Chain& chain)
        : a(a), w(w), sm(sm), chain(chain), tid(threadIdx.x), lane(tid & 31), warp(__shfl_sync(0xffffffffu, tid >> 5, 0)),
          half(warp >> 2), v((warp & 3) * 32 + lane),
          failed((smem_addr(&sm) & 1023u) != 0) {  // the swizzle acts on address bits
        if (tid == 0) {
            for (auto& b : sm.full) tc::barrier_init(smem_addr(&b), 1);
            for (auto& b : sm.done) tc::barrier_init(smem_addr(&b), 1);
            for (auto& b : sm.ready) tc::barrier_init(smem_addr(&b), kTcCompute / 32);
            for (auto& b : sm.empty) tc::barrier_init(smem_addr(&b), kTcCompute / 32 + 1);  // factors read, products done
            tc::barrier_init(smem_addr(&sm.rows_full), kTcMovers);
            tc::barrier_init(smem_addr(&sm.rows_empty), kTcCompute / 32);
            tc::barrier_init(smem_addr(&sm.out_ready), kTcCompute / 32);
            tc::barrier_init(smem_addr(&sm.out_free), kTcMovers / 32);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (warp == kTcCompute / 32) tc::allocate(&sm.base, kTcColumns);
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
        tmem = __shfl_sync(0xffffffffu, sm.base, 0);
        at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    }
    // Also where a wait ran out: what was in flight had another such limit's time to end.
    CUBF_DEV void finish() {
        tc::fence_before();
        __syncthreads();
        if (warp == kTcCompute / 32) {
            tc::fence_after();
            tc::release(tmem, kTcColumns);
        }
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

    template <typename Barrier>
    CUBF_DEV void wait(Barrier& barrier, uint32_t phase) {
        failed = failed || !tc::barrier_wait(smem_addr(&barrier), phase);
        __syncwarp();
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
    CUBF_DEV void load(int c, int s) const {
        const uint32_t bar = smem_addr(&sm.full[s]), dst = smem_addr(sm.stage[s]);
        const int k_head = chain.head / (a.heads / a.k_heads);
        const size_t tile = static_cast<size_t>(chain.base + c) * a.k_heads + k_head;
        if (tc::elect()) {
            tc::barrier_expect(bar, Tiles::kStage + sizeof(sm.factors[s]));
            tc::bulk_copy(dst, work(w.packed) + tile * 2 * Tiles::kOperand, 2 * Tiles::kOperand, bar);
            tc::bulk_copy(dst + 2 * Tiles::kOperand, work(w.solve) + place(c) * 2 * Tiles::kSquares, 2 * Tiles::kSquares, bar);
            tc::bulk_copy(smem_addr(sm.factors[s]), work(w.factors) + place(c) * kTcFactors * C * 4, sizeof(sm.factors[s]), bar);
        }
        __syncwarp();
    }
    CUBF_DEV uint32_t q(int s) const { return smem_addr(sm.stage[s]); }
    CUBF_DEV uint32_t k(int s) const { return q(s) + Tiles::kOperand; }
    CUBF_DEV uint32_t solve(int s) const { return q(s) + 2 * Tiles::kOperand; }
    CUBF_DEV uint32_t attention(int s) const { return solve(s) + Tiles::kSquares; }

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
                            tc::rows_along_n(tile + j * KP * 128 + (s / 4) * tc::kPanel + (s % 4) * 32), idesc, i + j + s > 0);
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
                    tc::mma(tmem + d, token_column(x, i, s), tc::rows_along_k(tile + j * KP * 128 + s * 2048), idesc,
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

    template <bool KEEP>
    CUBF_DEV void issue_forward() {
        const int chunks = chain.chunks;
        if (chunks > 0) load(0, 0);
        if (chunks > 1) load(1, 1);
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
                times_square(Tiles::kX, Tiles::kY, solve(st));
                tc::commit(smem_addr(&sm.done[kLy]));
            }
            __syncwarp();
            if (c > 0 && c + 1 < chunks) {       // the stage that the chunk before has left
                wait(sm.empty[st ^ 1], ((c - 1) >> 1) & 1);
                if (failed) break;
                load(c + 1, st ^ 1);
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
                    times_square(Tiles::kO, Tiles::kY, attention(st));
                    tc::commit(smem_addr(&sm.done[kPu]));
                    tc::commit(smem_addr(&sm.empty[st]));
                }
                __syncwarp();
            }
        }
    }

    // ---- the moving warps ----
    // 16 threads a row of 128 columns, six rows at a time; addresses advance by constants, since these warps share the
    // schedulers and instruction caches with the computing ones.
    static constexpr int kSide = kTcMovers / 16, kTurns = (C + kSide - 1) / kSide;
    CUBF_DEV void load_tile(const HeadTensor& t, int c, bool wide) const {
        const int n = tokens(c), first = tid - kTcCompute - 32;
        const T* p = static_cast<const T*>(t.p) + chain.row * t.batch + (static_cast<size_t>(chain.start) + c * C) * t.token +
                     static_cast<size_t>(chain.head) * t.head;
        if (wide) {
            const int row = first / 16, col = first % 16 * 8;
            const T* q = p + (col < a.v_dim ? row * t.token + col : 0);
            const size_t step = col < a.v_dim ? kSide * t.token : 0;
            const uint32_t to = smem_addr(sm.rows + row * 128 + col);
            const int valid = col < a.v_dim ? n - row : 0;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const bool ok = kSide * i < valid;
                if (kSide * i + row < C) copy16(to + i * kSide * 256, ok ? q : p, ok);
                q += step;
            }
        } else {
            for (int e = first; e < C * 128; e += kTcMovers) {
                const int r = e / 128, col = e % 128;
                sm.rows[e] = r < n && col < a.v_dim ? p[r * t.token + col] : Convert<T, float>::store(0.f);
            }
        }
        // arrives when the thread's copies have; its plain stores before are released with it
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&sm.rows_full)) : "memory");
        __syncwarp();
    }
    CUBF_DEV void store_tile(T* out, int c, bool wide) const {
        T* p = out + out_row(c) * a.v_dim;
        const size_t step = static_cast<size_t>(a.heads) * a.v_dim;
        const int n = tokens(c), first = tid - kTcCompute - 32;
        if (wide) {
            const int row = first / 16, col = first % 16 * 8, valid = col < a.v_dim ? n - row : 0;
            const T* from = sm.out + row * 128 + col;
            T* to = p + row * step + col;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                if (kSide * i < valid) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from + i * kSide * 128);
                to += kSide * step;
            }
        } else {
            for (int e = first; e < n * 128; e += kTcMovers) {
                const int r = e / 128, col = e % 128;
                if (col < a.v_dim) p[r * step + col] = sm.out[e];
            }
        }
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(smem_addr(&sm.out_free));
    }
    // Rows come in once those before were read, the output leaves.  Every barrier here is one of a ring: none can complete
    // a second time before its waiter has gone on.
    template <bool KEEP>
    CUBF_DEV void move_forward(bool wide_v, bool wide_o) {
        const int chunks = chain.chunks;
        for (int c = 0; c < chunks && !failed; ++c) {
            if (c > 0) wait(sm.rows_empty, (c - 1) & 1);
            if (!failed) load_tile(a.v, c, wide_v);
            if (!KEEP && c > 1) {
                wait(sm.out_ready, c & 1);
                if (!failed) store_tile(static_cast<T*>(a.o), c - 2, wide_o);
            }
        }
        if (!KEEP)
            for (int c = max(0, chunks - 2); c < chunks && !failed; ++c) {
                wait(sm.out_ready, c & 1);
                if (!failed) store_tile(static_cast<T*>(a.o), c, wide_o);
            }
        copies_wait<0>();
    }

    // ---- the computing warps ----
    // Values go in pairs: y, o and the state are packed fp32 pairs of neighbouring tokens or channels.
    using P = f32x2::P;
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
            if (keep && v < w.v_pitch) {
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
    // Byte of (column of v, channel) in a kept state's piece: panels of 64 channels, a row for each column of v.
    CUBF_DEV uint32_t kept(int row, int col) const {
        return static_cast<uint32_t>((col >> 6) * (w.v_rows * 128) + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4));
    }
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
    // NaN where a wait ran out.
    CUBF_DEV void state_out(float* p, const P (&s)[H / 2]) const {
#pragma unroll
        for (int i = 0; i < H / 2; ++i) {
            float x[2];
            f32x2::up(s[i], x[0], x[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = half * H + 2 * i + e;
                if (k < a.k_dim && v < a.v_dim)
                    p[static_cast<size_t>(k) * a.v_dim + v] = failed ? __int_as_float(0x7fffffff) : x[e];
            }
        }
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
    CUBF_DEV void rows_keep(size_t region, int c, const P (&x)[16]) const {
        if (v < w.v_pitch) {
            float* p = reinterpret_cast<float*>(work(region)) + (place(c) * C + 32 * half) * w.v_pitch + v;
#pragma unroll
            for (int i = 0; i < 16; ++i) f32x2::up(x[i], p[2 * i * w.v_pitch], p[(2 * i + 1) * w.v_pitch]);
        }
        __syncwarp();
    }

    // KEEP: the backward's run, which keeps the state before each chunk and R in place of writing o.
    template <bool KEEP>
    CUBF_DEV void compute_forward() {
        P s[H / 2], y[16], x[16], o[16];
        state_in(a.initial ? a.initial + state_offset() : nullptr, s);
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
        if (chunks > 0) {
            put_state(s, KEEP ? work(w.states) + place(0) * 2 * w.state_piece : nullptr);
            arrive(sm.ready[kStateReady]);
        }
        uint32_t phase = 0;
        for (int c = 0; c < chunks && !failed; ++c, phase ^= 1) {
            const float* f = sm.factors[c & 1];
            // while the state meets k
            if (!KEEP && c > 0) add_out(c - 1);
            wait(sm.full[c & 1], (c >> 1) & 1);
            wait(sm.rows_full, phase);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                y[i] = f32x2::pk(widen(sm.rows[(32 * half + 2 * i) * 128 + v]), widen(sm.rows[(32 * half + 2 * i + 1) * 128 + v]));
            report(sm.rows_empty);
            wait(sm.done[kSk], phase);
            get_tokens(Tiles::kX, x);
#pragma unroll
            for (int g = 0; g < 8; ++g) {    // Y = v - e^G (S k)
                P a, b;
                factors_of(f + kDecay * C, g, a, b);
                y[2 * g] = f32x2::sub2(y[2 * g], f32x2::mul2(a, x[2 * g]));
                y[2 * g + 1] = f32x2::sub2(y[2 * g + 1], f32x2::mul2(b, x[2 * g + 1]));
            }
            put_tokens(Tiles::kY, y);
            arrive(sm.ready[kYReady]);
            if (!KEEP && c > 0) move_out(c - 1);  // while Y meets L
            wait(sm.done[kLy], phase);
            get_tokens(Tiles::kX, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = f32x2::sub2(y[i], x[i]);  // R = Y - (L beta) Y
            put_tokens(Tiles::kU, y, f + kTailBeta * C);
            arrive(sm.ready[kUReady]);
            // while U meets k
            if (KEEP) {
                rows_keep(w.errors, c, y);
            } else {
                put_tokens(Tiles::kY, y);
                get_tokens(Tiles::kO, x);
                arrive(sm.ready[kOutTaken]);
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    P a, b;
                    factors_of(f + kScaled * C, g, a, b);
                    o[2 * g] = f32x2::mul2(a, x[2 * g]);
                    o[2 * g + 1] = f32x2::mul2(b, x[2 * g + 1]);
                }
            }
            const float whole = f[kDecay * C + C - 1];
            report(sm.empty[c & 1]);
            wait(sm.done[kKu], phase);
            state_add(whole, s);
            put_state(s, KEEP && c + 1 < chunks ? work(w.states) + place(c + 1) * 2 * w.state_piece : nullptr);
            if (c + 1 < chunks) arrive(sm.ready[kStateReady]);
        }
        if (!KEEP) {
            if (chunks > 0 && !failed) {
                add_out(chunks - 1);
                move_out(chunks - 1);
            }
            state_out(a.last + state_offset(), s);
        }
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

template <typename T, int KP>
__global__ void __launch_bounds__(kTcThreads, 1) gated_delta_tc_forward_kernel(GatedDeltaArgs a, Places w, bool wide_v, bool wide_o) {
    extern __shared__ __align__(1024) unsigned char aligned_raw[];
    pdl_begin();
    TcChain<T, KP> run(a, w, *reinterpret_cast<TcShared<T, KP>*>(aligned_raw), chain_of(a, blockIdx.x));
    if (run.warp >= kTcCompute / 32) {
        fewer_registers<56>();
        if (run.warp == kTcCompute / 32)
            run.template issue_forward<false>();
        else
            run.template move_forward<false>(wide_v, wide_o);
    } else {
        more_registers<224>();
        run.template compute_forward<false>();
    }
    run.finish();
}

}  // namespace cubf::delta
