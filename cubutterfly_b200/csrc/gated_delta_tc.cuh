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

#include "gated_delta.cuh"
#include "tcgen05.cuh"

namespace cubf::delta {

constexpr int kTcCompute = 256;          // threads of the computing warps
constexpr int kTcMovers = 96;            // ... and of those that move rows; between them, a warp that issues
constexpr int kTcThreads = kTcCompute + 32 + kTcMovers;
constexpr uint32_t kTcColumns = 512;     // all of tensor memory

template <typename T, int KP>
struct TcTiles {
    static constexpr int NI = kInput<T>;
    static constexpr int kOperand = NI * KP * 128;           // bytes of q or k
    static constexpr int kSquares = 2 * tc::kPanel;          // of L or P, two pieces
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
    alignas(16) float factors[2][kFactors];
    alignas(8) unsigned long long full[2], ready[4], done[4], rows_full, out_ready, out_free;
    uint32_t base;
};

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
            tc::barrier_init(smem_addr(&sm.rows_full), kTcMovers);
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

    // ---- the issuing warp ----
    CUBF_DEV void load(int c, int s) const {
        const uint32_t bar = smem_addr(&sm.full[s]), dst = smem_addr(sm.stage[s]);
        const int k_head = chain.head / (a.heads / a.k_heads);
        const size_t tile = static_cast<size_t>(chain.base + c) * a.k_heads + k_head;
        if (tc::elect()) {
            tc::barrier_expect(bar, Tiles::kStage + kFactors * 4);
            tc::bulk_copy(dst, work(w.packed) + tile * 2 * Tiles::kOperand, 2 * Tiles::kOperand, bar);
            tc::bulk_copy(dst + 2 * Tiles::kOperand, work(w.solve) + place(c) * Tiles::kSquares, Tiles::kSquares, bar);
            tc::bulk_copy(dst + 2 * Tiles::kOperand + Tiles::kSquares, work(w.attention) + place(c) * Tiles::kSquares,
                          Tiles::kSquares, bar);
            tc::bulk_copy(smem_addr(sm.factors[s]), work(w.factors) + place(c) * kFactors * 4, kFactors * 4, bar);
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

    template <bool KEEP>
    CUBF_DEV void issue_forward() {
        const int chunks = chain.chunks;
        if (chunks > 0) load(0, 0);
        uint32_t phase = 0;
        for (int c = 0; c < chunks && !failed; ++c, phase ^= 1) {
            const int st = c & 1;
            wait(sm.ready[0], phase);
            wait(sm.full[st], (c >> 1) & 1);
            if (failed) break;
            if (tc::elect()) {
                state_times(Tiles::kX, k(st));
                tc::commit(smem_addr(&sm.done[0]));
                if (!KEEP) state_times(Tiles::kO, q(st));
            }
            __syncwarp();
            // the other stage is free: its chunk's last products are done, its factors read
            if (c > 0) wait(sm.done[KEEP ? 2 : 3], phase ^ 1);
            if (failed) break;
            if (c + 1 < chunks) load(c + 1, st ^ 1);
            wait(sm.ready[1], phase);
            if (failed) break;
            if (tc::elect()) {
                times_square(Tiles::kX, Tiles::kY, solve(st));
                tc::commit(smem_addr(&sm.done[1]));
            }
            __syncwarp();
            wait(sm.ready[2], phase);
            if (failed) break;
            if (tc::elect()) {
                onto_state(Tiles::kD, Tiles::kU, k(st), false);
                tc::commit(smem_addr(&sm.done[2]));
            }
            __syncwarp();
            if (KEEP) continue;
            wait(sm.ready[3], phase);
            if (failed) break;
            if (tc::elect()) {
                times_square(Tiles::kX, Tiles::kY, attention(st));
                tc::commit(smem_addr(&sm.done[3]));
            }
            __syncwarp();
        }
    }

    // ---- the moving warps ----
    CUBF_DEV void load_tile(const HeadTensor& t, int c, bool wide) const {
        const T* p = static_cast<const T*>(t.p) + chain.row * t.batch + (static_cast<size_t>(chain.start) + c * C) * t.token +
                     static_cast<size_t>(chain.head) * t.head;
        const int n = tokens(c), first = tid - kTcCompute - 32;
        constexpr int N = 16 / sizeof(T);
        if (wide) {
            for (int e = first; e < C * 128 / N; e += kTcMovers) {
                const int r = e / (128 / N), col = e % (128 / N) * N;
                const bool ok = r < n && col < a.v_dim;
                copy16(smem_addr(sm.rows + r * 128 + col), p + (ok ? r * t.token + col : 0), ok);
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
        constexpr int N = 16 / sizeof(T);
        if (wide) {
            for (int e = first; e < n * (128 / N); e += kTcMovers) {
                const int r = e / (128 / N), col = e % (128 / N) * N;
                if (col < a.v_dim)
                    *reinterpret_cast<uint4*>(p + r * step + col) = *reinterpret_cast<const uint4*>(sm.out + r * 128 + col);
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
    // Rows of chunk c come in once those before were read, the output before leaves.
    template <bool KEEP>
    CUBF_DEV void move_forward(bool wide_v, bool wide_o) {
        for (int c = 0; c < chain.chunks && !failed; ++c) {
            if (c > 0) wait(sm.ready[1], (c - 1) & 1);
            if (!failed) load_tile(a.v, c, wide_v);
            if (!KEEP && c > 0) {
                wait(sm.out_ready, (c - 1) & 1);
                if (!failed) store_tile(static_cast<T*>(a.o), c - 1, wide_o);
            }
        }
        if (!KEEP && chain.chunks > 0) {
            wait(sm.out_ready, (chain.chunks - 1) & 1);
            if (!failed) store_tile(static_cast<T*>(a.o), chain.chunks - 1, wide_o);
        }
        copies_wait<0>();
    }

    // ---- the computing warps ----
    // Two pieces of the thread's 32 tokens to tensor memory, as the operand at `x`, times a factor a token.
    CUBF_DEV void put_tokens(uint32_t x, const float (&y)[32], const float* factor) const {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            const float4 m = factor ? *reinterpret_cast<const float4*>(factor + 32 * half + 4 * g) : make_float4(1, 1, 1, 1);
            uint32_t p[2];
            pieces<2>(y[4 * g] * m.x, y[4 * g + 1] * m.y, p);
            hi[2 * g] = p[0], lo[2 * g] = p[1];
            pieces<2>(y[4 * g + 2] * m.z, y[4 * g + 3] * m.w, p);
            hi[2 * g + 1] = p[0], lo[2 * g + 1] = p[1];
        }
        tc::store<16>(at + x + 32 * half, hi);
        tc::store<16>(at + x + 32 * half + 16, lo);
    }
    // The state's pieces, its thread's half, as an operand and (keep) for the gradients.
    CUBF_DEV void put_state(const float (&s)[H], char* keep) const {
#pragma unroll
        for (int n = 0; n < H / 32; ++n) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                uint32_t p[2];
                pieces<2>(s[32 * n + 2 * i], s[32 * n + 2 * i + 1], p);
                hi[i] = p[0], lo[i] = p[1];
            }
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
    CUBF_DEV void state_in(const float* p, float (&s)[H]) const {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int k = half * H + i;
            s[i] = p && k < a.k_dim && v < a.v_dim ? p[static_cast<size_t>(k) * a.v_dim + v] : 0.f;
        }
    }
    CUBF_DEV void state_out(float* p, const float (&s)[H]) const {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int k = half * H + i;
            if (k < a.k_dim && v < a.v_dim) p[static_cast<size_t>(k) * a.v_dim + v] = failed ? __int_as_float(0x7fffffff) : s[i];
        }
    }
    // S = whole S + what the products left in kD
    CUBF_DEV void state_add(float whole, float (&s)[H]) const {
        uint32_t d[H];
#pragma unroll
        for (int n = 0; n < H / 32; ++n) tc::load<32>(at + Tiles::kD + half * H + 32 * n, d + 32 * n);
        tc::wait_load();
#pragma unroll
        for (int i = 0; i < H; ++i) s[i] = fmaf(whole, s[i], __uint_as_float(d[i]));
    }
    CUBF_DEV void put_out(const float (&x)[32]) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sm.out[(32 * half + i) * 128 + v] = Convert<T, float>::store(x[i]);
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(smem_addr(&sm.out_ready));
    }
    CUBF_DEV void rows_keep(size_t region, int c, const float (&x)[32]) const {
        if (v < w.v_pitch) {
            float* p = reinterpret_cast<float*>(work(region)) + (place(c) * C + 32 * half) * w.v_pitch + v;
#pragma unroll
            for (int i = 0; i < 32; ++i) p[i * w.v_pitch] = x[i];
        }
        __syncwarp();
    }

    // KEEP: the backward's run, which keeps the state before each chunk and R in place of writing o.
    template <bool KEEP>
    CUBF_DEV void compute_forward() {
        float s[H], o[32];
        state_in(a.initial ? a.initial + state_offset() : nullptr, s);
        const int chunks = chain.chunks;
        if (chunks > 0) {
            put_state(s, KEEP ? work(w.states) + place(0) * 2 * w.state_piece : nullptr);
            arrive(sm.ready[0]);
        }
        uint32_t phase = 0;
        for (int c = 0; c < chunks && !failed; ++c, phase ^= 1) {
            const int st = c & 1;
            const float* f = sm.factors[st];
            // while the state meets k and q: the last chunk's o leaves, this one's v is read
            if (!KEEP && c > 0) {
                if (c > 1) wait(sm.out_free, phase);
                put_out(o);
            }
            wait(sm.rows_full, phase);
            float y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = widen(sm.rows[(32 * half + i) * 128 + v]);
            wait(sm.full[st], (c >> 1) & 1);
            wait(sm.done[0], phase);
            {
                uint32_t x[32];
                tc::load<32>(at + Tiles::kX + 32 * half, x);
                tc::wait_load();
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float4 d = *reinterpret_cast<const float4*>(f + 32 * half + 4 * g);
                    y[4 * g] = fmaf(-d.x, __uint_as_float(x[4 * g]), y[4 * g]);
                    y[4 * g + 1] = fmaf(-d.y, __uint_as_float(x[4 * g + 1]), y[4 * g + 1]);
                    y[4 * g + 2] = fmaf(-d.z, __uint_as_float(x[4 * g + 2]), y[4 * g + 2]);
                    y[4 * g + 3] = fmaf(-d.w, __uint_as_float(x[4 * g + 3]), y[4 * g + 3]);
                }
            }
            put_tokens(Tiles::kY, y, f + 2 * C);
            arrive(sm.ready[1]);
            wait(sm.done[1], phase);
            {
                uint32_t x[32];
                tc::load<32>(at + Tiles::kX + 32 * half, x);
                tc::wait_load();
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] -= __uint_as_float(x[i]);
            }
            if (KEEP) rows_keep(w.errors, c, y);
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const float4 beta = *reinterpret_cast<const float4*>(f + 2 * C + 32 * half + 4 * g);
                y[4 * g] *= beta.x, y[4 * g + 1] *= beta.y, y[4 * g + 2] *= beta.z, y[4 * g + 3] *= beta.w;
            }
            put_tokens(Tiles::kU, y, f + C);
            arrive(sm.ready[2]);
            if (!KEEP) {
                put_tokens(Tiles::kY, y, nullptr);
                arrive(sm.ready[3]);
                // q's part of o is there since the products with L
                uint32_t x[32];
                tc::load<32>(at + Tiles::kO + 32 * half, x);
                tc::wait_load();
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float4 d = *reinterpret_cast<const float4*>(f + 32 * half + 4 * g);
                    o[4 * g] = d.x * a.scale * __uint_as_float(x[4 * g]);
                    o[4 * g + 1] = d.y * a.scale * __uint_as_float(x[4 * g + 1]);
                    o[4 * g + 2] = d.z * a.scale * __uint_as_float(x[4 * g + 2]);
                    o[4 * g + 3] = d.w * a.scale * __uint_as_float(x[4 * g + 3]);
                }
            }
            const float whole = f[C - 1];
            wait(sm.done[2], phase);
            state_add(whole, s);
            put_state(s, KEEP && c + 1 < chunks ? work(w.states) + place(c + 1) * 2 * w.state_piece : nullptr);
            if (!KEEP) {
                wait(sm.done[3], phase);
                uint32_t x[32];
                tc::load<32>(at + Tiles::kX + 32 * half, x);
                tc::wait_load();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] += __uint_as_float(x[i]);
            }
            if (c + 1 < chunks) arrive(sm.ready[0]);
        }
        if (!KEEP) {
            if (chunks > 1) wait(sm.out_free, chunks & 1);
            if (chunks > 0) put_out(o);
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
