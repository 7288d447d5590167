// gated_scan.cuh -- the gated linear recurrence of recurrent language models,
// forward, backward and one token at a time.
//
// Per channel, along the tokens of a sequence, with gate inputs r and i,
// la = -c softplus(Lambda) sigmoid(r) and a = exp(la):
//   h_t = a_t h_{t-1} + u_t,   u_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t.
// A run of tokens is the affine map h -> A h + H (A the product of its a, H
// its last h from h = 0), and runs join by (A1, H1) . (A2, H2) =
// (A1 A2, A2 H1 + H2).  A thread runs STEPS tokens of two channels in
// registers; GROUPS groups of lanes hold consecutive runs of the same
// channels and join them by shuffles; the state then goes from warp to warp
// of a CTA, and from its last warp to the first one's next tile, one fused
// multiply-add a warp.  Every input is read once, every output written once,
// and no CTA waits on another.
//
// What bounds it is latency: 8 to 16 warps fit an SM beside their registers and
// the rows copied ahead, and none of its units is near its limit (8 x 1024 x 2048
// bf16: 53 % of the issue slots, 49 % of the FMA pipe and 55 % of the special
// functions forward, 61, 49 and 42 % backward).  A warp's chain is as long as its
// instructions are many, so the two channels of a lane are computed as packed
// fp32 pairs, and a is formed on the FMA pipe.  That makes 31 instructions and
// four special functions an element forward, 58 and five backward: 16384 x 4096
// bf16 in 114 us (4.7 TB/s) and 246 us backward, 8 x 2048 x 2048 in 60 and 102 us
// (4.5 and 4.6 TB/s); fp32, with half the elements a byte, 4 x 4096 x 1024 in 47
// and 88 us (5.7 and 5.3 TB/s).
#pragma once

#include "block_ops.hpp"
#include "common.cuh"
#include "f32x2.cuh"
#include "gate.cuh"

namespace cubf::scan {

using f32x2::add2;
using f32x2::fma2;
using f32x2::mul2;
using f32x2::sub2;
using gate::both;
using gate::each;
using gate::ex2;
using gate::kLn2;
using gate::kLog2e;
using gate::max_nan;
using gate::rcp;
using Pair = f32x2::P;

constexpr int kWarps = 8;                  // warps per CTA, consecutive in time
constexpr int kWarpChannels = 64;          // channels times lane groups of a warp: two channels per lane
// Tokens per thread and tile: as many as two CTAs' registers and shared
// memory allow.  Forward rows that are not 16-byte aligned take more of the
// latter.  With 8 and 16 tokens, bf16: 6 x 3602 x 974 92, 107 us; 16384 x 2050 120,
// 150; 32730 x 425 223, 257; 8 x 2048 x 2050 96, 97.  Only long even rows on fewer
// CTAs than SMs, of one or two lane groups, gain: 16384 x 4098 233, 217 and 4 x
// 4096 x 2050 120, 117 (but 2048 x 4098 36, 37, and four groups, as 16384 x 2050).
template <typename T, int PIECE>
constexpr int kForwardSteps = sizeof(T) == 2 && PIECE == 16 ? 16 : 8;
constexpr int kBackwardSteps = 8;
static_assert(kGatedScanChunk == 2 * kBackwardSteps && kGatedScanChunk % kForwardSteps<__half, 16> == 0,
              "chunks begin where a forward warp and every other backward warp do");

CUBF_DEV Pair pair(float2 v) { return f32x2::pk(v.x, v.y); }
CUBF_DEV float2 floats(Pair p) {
    float2 f;
    f32x2::up(p, f.x, f.y);
    return f;
}

// ---- access to two channels of a token --------------------------------------------------------
// 16-bit pairs come in a word, fp32 pairs in two.
template <typename T>
struct Raw {
    using Word = uint32_t;
    static CUBF_DEV Word zero() { return 0u; }
    static CUBF_DEV Word lowest() { return std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u; }  // -inf
    static CUBF_DEV Word vec(const T* p) { return __ldcs(reinterpret_cast<const unsigned int*>(p)); }
    static CUBF_DEV Pair get(Word w) {
        if constexpr (std::is_same<T, __half>::value) {
            __half2 h;
            memcpy(&h, &w, 4);
            return pair(__half22float2(h));
        } else {
            return f32x2::pk(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        }
    }
    static CUBF_DEV Word word_of(float2 f) {
        uint32_t w;
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __float22half2_rn(f);
            memcpy(&w, &h, 4);
        } else {
            const __nv_bfloat162 h = __float22bfloat162_rn(f);
            memcpy(&w, &h, 4);
        }
        return w;
    }
    static CUBF_DEV void store_vec(T* p, float2 f) { __stcs(reinterpret_cast<unsigned int*>(p), word_of(f)); }
};
template <>
struct Raw<float> {
    using Word = float2;
    static CUBF_DEV Word zero() { return make_float2(0.f, 0.f); }
    static CUBF_DEV Word lowest() { return make_float2(-INFINITY, -INFINITY); }
    static CUBF_DEV Word vec(const float* p) { return __ldcs(reinterpret_cast<const float2*>(p)); }
    static CUBF_DEV Pair get(Word w) { return pair(w); }
    static CUBF_DEV Word word_of(float2 f) { return f; }
    static CUBF_DEV void store_vec(float* p, float2 f) { __stcs(reinterpret_cast<float2*>(p), f); }
};

// The lane's two channels of a row, which are adjacent.  Lanes of a group are
// adjacent; groups hold consecutive runs of tokens.
template <int GROUPS>
struct Lane {
    static constexpr int kLanes = 32 / GROUPS;
    int ch;
    bool ok0, ok1;
    CUBF_DEV Lane(int c0, int lane, int dim) {
        ch = c0 + 2 * (lane % kLanes);
        ok0 = ch < dim;
        ok1 = ch + 1 < dim;
    }
    CUBF_DEV Pair load32(const float* row) const {
        return f32x2::pk(ok0 ? row[ch] : 0.f, ok1 ? row[ch + 1] : 0.f);
    }
    CUBF_DEV void store32(float* row, Pair p) const {
        const float2 f = floats(p);
        if (ok0) row[ch] = f.x;
        if (ok1) row[ch + 1] = f.y;
    }
    // rows of T, pair by pair where they are aligned for it
    template <bool PAIRS, typename T>
    CUBF_DEV Pair load(const T* row) const {
        if constexpr (PAIRS)
            return Raw<T>::get(ok0 ? Raw<T>::vec(row + ch) : Raw<T>::zero());
        else
            return f32x2::pk(ok0 ? Convert<T, float>::load(row[ch]) : 0.f, ok1 ? Convert<T, float>::load(row[ch + 1]) : 0.f);
    }
    template <bool PAIRS, typename T>
    CUBF_DEV void store(T* row, Pair p) const {
        const float2 f = floats(p);
        if constexpr (PAIRS) {
            if (ok0) Raw<T>::store_vec(row + ch, f);
        } else {
            if (ok0) row[ch] = Convert<T, float>::store(f.x);
            if (ok1) row[ch + 1] = Convert<T, float>::store(f.y);
        }
    }
};

// The rows of a warp's tokens: N tensors of GROUPS x STEPS tokens x CHANNELS
// channels.  A warp copies its own rows into its own shared memory (no barrier
// beyond the warp's), STAGES tiles deep: the copies of a later tile are in
// flight while this one is worked on, and hold no registers.  Token g STEPS + s
// lies at row s GROUPS + g, so that the lanes of all groups read adjacent
// words.  Results take the place of words that have been read and leave the
// same way: stored from registers, each pair would cost as many instructions in
// addresses as its arithmetic.  Rows are copied in 16-byte pieces (ShiftedRows:
// where they are not aligned for that).  Channels past the end are zero; tokens
// past the end are what `close` says.
template <typename T, int N, int STEPS_, int STAGES_, int GROUPS>
struct Rows {
    static constexpr int STEPS = STEPS_, STAGES = STAGES_, TOKENS = STEPS * GROUPS;
    static constexpr int kChannels = kWarpChannels / GROUPS;
    static constexpr int kRowBytes = kChannels * static_cast<int>(sizeof(T));
    static constexpr int kTensorBytes = TOKENS * kRowBytes;
    static constexpr int kBytes = N * kTensorBytes;
    static constexpr int kPerRow = kRowBytes / 16;     // pieces of a row
    static constexpr int kRowsPer = 32 / kPerRow;      // rows a warp copies at a time
    static constexpr int kCopies = TOKENS / kRowsPer;  // rows a lane copies of a tensor
    using Word = typename Raw<T>::Word;
    const T* base[N];
    size_t stride[N];
    const T* next[N];     // this lane's first piece of the tile fetched next
    unsigned char* mine;  // this warp's stages
    int lane, c0, length, dim;

    CUBF_DEV int column() const { return c0 + lane % kPerRow * (16 / static_cast<int>(sizeof(T))); }
    // where this lane's piece of the k-th rows lies: what follows from the lane, and from k
    CUBF_DEV int piece_place() const {
        const int r = lane / kPerRow;
        return (r % STEPS * GROUPS + r / STEPS) * kRowBytes + lane % kPerRow * 16;
    }
    static constexpr int row_place(int k) {
        return (k * kRowsPer % STEPS * GROUPS + k * kRowsPer / STEPS) * kRowBytes;
    }

    CUBF_DEV void init(unsigned char* shared, int lane_, int c0_, int length_, int dim_, int first) {
        mine = shared;
        lane = lane_;
        c0 = c0_;
        length = length_;
        dim = dim_;
#pragma unroll
        for (int n = 0; n < N; ++n)
            next[n] = base[n] + static_cast<ptrdiff_t>(first + lane / kPerRow) * static_cast<ptrdiff_t>(stride[n]) +
                      column();
    }
    CUBF_DEV Word* word(int stage, int n, int s) const {  // of the lane's own token s
        return reinterpret_cast<Word*>(mine + stage * kBytes + n * kTensorBytes + s * GROUPS * kRowBytes) + lane;
    }
    // starts the copies of tokens [t, t + TOKENS), closes their group, and
    // moves on by `advance` tokens
    CUBF_DEV void fetch(int stage, int t, int advance) {
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(mine + stage * kBytes)) + piece_place();
        if (t >= 0 && t + TOKENS <= length && c0 + kChannels <= dim) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const T* src = next[n];
#pragma unroll
                for (int k = 0; k < kCopies; ++k) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + n * kTensorBytes + row_place(k)),
                                 "l"(src)
                                 : "memory");
                    src += kRowsPer * stride[n];
                }
            }
        } else if (t < length && t + TOKENS > 0) {
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < kCopies; ++k) {
                    const int at = t + lane / kPerRow + k * kRowsPer;
                    const bool in = at >= 0 && at < length && column() < dim;
                    const T* src = in ? base[n] + static_cast<size_t>(at) * stride[n] + column() : base[n];
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + n * kTensorBytes +
                                                                                      row_place(k)),
                                 "l"(src), "r"(in ? 16 : 0)
                                 : "memory");
                }
        } else {
            // nothing of the sequence: zeros, so that no stale word is computed with
            for (int k = 0; k < kBytes / 512; ++k)
                *reinterpret_cast<uint4*>(mine + stage * kBytes + lane * 16 + k * 512) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
        for (int n = 0; n < N; ++n) next[n] += static_cast<ptrdiff_t>(advance) * static_cast<ptrdiff_t>(stride[n]);
    }
    // waits for the oldest of STAGES groups
    CUBF_DEV void arrive() const {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
    }
    CUBF_DEV void begin(int) const {}  // the lane's run
    // The lane's token s.
    CUBF_DEV Pair get(int stage, int n, int s) const { return Raw<T>::get(*word(stage, n, s)); }
    // gives the lane's tokens past the end, its run beginning at t, the value
    // `tail` (the copies leave zeros there)
    CUBF_DEV void close(int stage, int n, int t, Word tail) const {
        if (t + STEPS <= length) return;
        for (int s = 0; s < STEPS; ++s)
            if (t + s >= length) *word(stage, n, s) = tail;
    }
    // A result of the lane's token s, into the place of tensor n's word.
    CUBF_DEV void put(int stage, int n, int s, Pair v) const { *word(stage, n, s) = Raw<T>::word_of(floats(v)); }
    // writes the tile put in tensor n's place, the warp's tokens from t, out to rows of `dim` channels
    CUBF_DEV void flush(int stage, int n, T* out, int t) const {
        const unsigned char* src = mine + stage * kBytes + n * kTensorBytes + piece_place();
        const int row = t + lane / kPerRow, col = column();
        T* dst = out + static_cast<size_t>(row) * dim + col;
        const bool whole = t + TOKENS <= length && c0 + kChannels <= dim;
#pragma unroll
        for (int k = 0; k < kCopies; ++k) {
            if (whole || (row + k * kRowsPer < length && col < dim))
                __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<const uint4*>(src + row_place(k)));
            dst += static_cast<size_t>(kRowsPer) * dim;
        }
    }
};

// The same for rows that are not 16-byte aligned: the aligned 16-byte pieces
// over a row's channels are copied, one more than the row has, and lie in
// shared memory as they do in memory; the row's address modulo 16, its shift,
// says where in them its values are.  Results go to the bytes that the lane's own
// values came from.  Whole pieces of them leave as such, the first and last,
// which the row shares with its neighbours, unit by unit.  Channels past the
// end hold what lies there; no result of theirs is kept.
// 2 x 8501 x 3947 fp16: 304 us forward, 633 backward; loaded value by value into
// registers 635 and 1921.  2 x 8500 x 3946: 239 and 416; copied in 4-byte pieces
// 356 and 477.
// PIECE is what shifts are multiples of: 4, or 2 where a pair of 16-bit values
// may straddle two words.
template <typename T, int N, int STEPS_, int STAGES_, int GROUPS, int PIECE>
struct ShiftedRows {
    static_assert(PIECE == 4 || (PIECE == 2 && sizeof(T) == 2), "rows are aligned for their values");
    static constexpr int STEPS = STEPS_, STAGES = STAGES_, TOKENS = STEPS * GROUPS;
    static constexpr int kChannels = kWarpChannels / GROUPS;
    static constexpr int kLanes = 32 / GROUPS;
    static constexpr int kSize = static_cast<int>(sizeof(T));
    static constexpr int kSpan = kSize * kChannels;  // bytes of a row's channels
    static constexpr int kRowBytes = kSpan + 16;
    static constexpr int kTensorBytes = TOKENS * kRowBytes;
    static constexpr int kBytes = N * kTensorBytes;
    static constexpr int kPieces = kSpan / 16;
    static constexpr int kRowsPer = 32 / kPieces;  // rows a warp copies at a time
    static constexpr int kCopies = TOKENS / kRowsPer;
    static constexpr int kEdge = 16 / PIECE;  // units of a shifted row outside its whole pieces
    using Word = typename Raw<T>::Word;
    using Unit = std::conditional_t<PIECE == 2, unsigned short, unsigned int>;
    const T* base[N];
    size_t stride[N];
    unsigned char* mine;  // this warp's stages
    int lane, c0, length, dim;
    int token;  // where the lane's run begins

    CUBF_DEV void init(unsigned char* shared, int lane_, int c0_, int length_, int dim_, int) {
        mine = shared;
        lane = lane_;
        c0 = c0_;
        length = length_;
        dim = dim_;
    }
    CUBF_DEV void begin(int t0) { token = t0; }
    static CUBF_DEV int place_of(int row) { return (row % STEPS * GROUPS + row / STEPS) * kRowBytes; }
    CUBF_DEV unsigned char* tensor(int stage, int n) const { return mine + stage * kBytes + n * kTensorBytes; }
    CUBF_DEV uintptr_t row_address(int n, int t) const {
        return reinterpret_cast<uintptr_t>(base[n] + static_cast<size_t>(t) * stride[n] + c0);
    }
    CUBF_DEV uint32_t shift_of(int n, int t) const {
        return (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base[n])) +
                kSize * (static_cast<uint32_t>(t) * static_cast<uint32_t>(stride[n]) + static_cast<uint32_t>(c0))) &
               15u;
    }
    // the lane's pair of its token s
    CUBF_DEV unsigned char* own(int stage, int n, int s) const {
        return tensor(stage, n) + (s * GROUPS + lane / kLanes) * kRowBytes + 2 * kSize * (lane % kLanes) +
               shift_of(n, token + s);
    }
    static CUBF_DEV void copy(uint32_t to, uintptr_t from) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    }
    CUBF_DEV void fetch(int stage, int t, int) {
        const int bytes = kSize * (dim - c0 < kChannels ? dim - c0 : kChannels);
        // Pieces reach over the row's ends: not in the first and last rows, where
        // that may be outside the tensor (rows below 16 bytes: the first and last 16).
        const int apart = dim * kSize >= 16 ? 1 : 16;
        if (t >= apart && t + TOKENS + apart <= length) {
            const int piece = lane % kPieces * 16;
            const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(tensor(stage, 0)));
#pragma unroll
            for (int n = 0; n < N; ++n) {
                uintptr_t src = row_address(n, t + lane / kPieces);
#pragma unroll
                for (int k = 0; k < kCopies; ++k) {
                    if (piece < static_cast<int>(src & 15) + bytes)
                        copy(dst + n * kTensorBytes + place_of(k * kRowsPer + lane / kPieces) + piece,
                             (src & ~static_cast<uintptr_t>(15)) + piece);
                    src += kSize * kRowsPer * stride[n];
                }
#pragma unroll
                for (int row = lane; row < TOKENS; row += 32) {
                    const uintptr_t last = row_address(n, t + row);
                    if (kSpan < static_cast<int>(last & 15) + bytes)
                        copy(dst + n * kTensorBytes + place_of(row) + kSpan,
                             (last & ~static_cast<uintptr_t>(15)) + kSpan);
                }
            }
        } else {
#pragma unroll 1
            for (int e = lane; e < N * TOKENS * (kPieces + 1); e += 32) {
                const int piece = e % (kPieces + 1) * 16, row = e / (kPieces + 1) % TOKENS;
                const int n = e / (kPieces + 1) / TOKENS, at = t + row;
                const T* origin = base[0];
                size_t apart_by = stride[0];
#pragma unroll
                for (int m = 1; m < N; ++m)
                    if (n == m) {
                        origin = base[m];
                        apart_by = stride[m];
                    }
                unsigned char* to = tensor(stage, 0) + n * kTensorBytes + place_of(row) + piece;
                const bool in = at >= 0 && at < length;
                const uintptr_t src = reinterpret_cast<uintptr_t>(origin + (in ? at * apart_by : 0) + c0);
                const uintptr_t from = (src & ~static_cast<uintptr_t>(15)) + piece;
                const uintptr_t lo = reinterpret_cast<uintptr_t>(origin);
                const uintptr_t hi = reinterpret_cast<uintptr_t>(origin + static_cast<size_t>(length - 1) * apart_by + dim);
                if (in && from >= lo && from + 16 <= hi) {
                    copy(static_cast<uint32_t>(__cvta_generic_to_shared(to)), from);
                } else {
                    for (int j = 0; j < 16; j += PIECE) {
                        const uintptr_t unit = from + j;
                        *reinterpret_cast<Unit*>(to + j) =
                            in && unit >= lo && unit < hi ? *reinterpret_cast<const Unit*>(unit) : static_cast<Unit>(0);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    CUBF_DEV void arrive() const {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
    }
    CUBF_DEV Pair get(int stage, int n, int s) const {
        if constexpr (kSize == 4) {
            const float* f = reinterpret_cast<const float*>(own(stage, n, s));
            return f32x2::pk(f[0], f[1]);
        } else if constexpr (PIECE == 2) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(own(stage, n, s));
            const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
            return Raw<T>::get(__funnelshift_r(w[0], w[1], static_cast<uint32_t>(at & 2) * 8));
        } else {
            return Raw<T>::get(*reinterpret_cast<const Word*>(own(stage, n, s)));
        }
    }
    CUBF_DEV void write(int stage, int n, int s, Word w) const {
        unsigned char* to = own(stage, n, s);
        if constexpr (kSize == 4) {
            reinterpret_cast<float*>(to)[0] = w.x;
            reinterpret_cast<float*>(to)[1] = w.y;
        } else if constexpr (PIECE == 2) {
            reinterpret_cast<Unit*>(to)[0] = static_cast<Unit>(w);
            reinterpret_cast<Unit*>(to)[1] = static_cast<Unit>(w >> 16);
        } else {
            *reinterpret_cast<Word*>(to) = w;
        }
    }
    CUBF_DEV void close(int stage, int n, int t, Word tail) const {
        if (t + STEPS <= length) return;
        for (int s = 0; s < STEPS; ++s)
            if (t + s >= length) write(stage, n, s, tail);
    }
    CUBF_DEV void put(int stage, int n, int s, Pair v) const { write(stage, n, s, Raw<T>::word_of(floats(v))); }
    CUBF_DEV void flush(int stage, int n, T* out, int t) const {
        const uint32_t differ = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(out)) -
                                static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base[n]));
        const bool same = ((differ | kSize * (static_cast<uint32_t>(dim) - static_cast<uint32_t>(stride[n]))) & 15u) == 0;
        if (same && c0 + kChannels <= dim) {  // out's rows have the shifts that its values lie at
            const int piece = lane % kPieces * 16;
            const unsigned char* from = tensor(stage, n);
            uintptr_t to = reinterpret_cast<uintptr_t>(out + static_cast<size_t>(t + lane / kPieces) * dim + c0);
#pragma unroll
            for (int k = 0; k < kCopies; ++k) {
                const int row = k * kRowsPer + lane / kPieces;
                if ((piece > 0 || (to & 15) == 0) && t + row < length)
                    __stcs(reinterpret_cast<uint4*>((to & ~static_cast<uintptr_t>(15)) + piece),
                           *reinterpret_cast<const uint4*>(from + place_of(row) + piece));
                to += kSize * static_cast<size_t>(kRowsPer) * dim;
            }
#pragma unroll 4
            for (int e = lane; e < TOKENS * kEdge; e += 32) {
                const int row = e / kEdge;
                const uintptr_t first = reinterpret_cast<uintptr_t>(out + static_cast<size_t>(t + row) * dim + c0);
                const int shift = static_cast<int>(first & 15);
                int at = shift + e % kEdge * PIECE;
                if (at >= 16) at += kSpan - 16;
                if (shift && t + row < length)
                    *reinterpret_cast<Unit*>(first - shift + at) =
                        *reinterpret_cast<const Unit*>(from + place_of(row) + at);
            }
        } else {
            const int ch = c0 + 2 * (lane % kLanes);
#pragma unroll 1
            for (int s = 0; s < STEPS; ++s)
                if (token + s < length) {
                    const T* from = reinterpret_cast<const T*>(own(stage, n, s));
                    T* to = out + static_cast<size_t>(token + s) * dim + ch;
                    if (ch < dim) to[0] = from[0];
                    if (ch + 1 < dim) to[1] = from[1];
                }
        }
    }
};
template <typename T, int N, int STEPS, int STAGES, int GROUPS, int PIECE>
using RowsOf = std::conditional_t<PIECE == 16, Rows<T, N, STEPS, STAGES, GROUPS>,
                                  ShiftedRows<T, N, STEPS, STAGES, GROUPS, PIECE == 16 ? 4 : PIECE>>;

// ---- the arithmetic of a token ----------------------------------------------------------------
CUBF_DEV float rsq(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Gates of 16 bits, rounded by 2^-9 or 2^-12 of themselves, take the sigmoid by
// 2^(-v log2 e) with the product as rounded, off by |v| 2^-24; fp32 calls, which
// are bound by memory, the exact one (4 x 4096 x 1024: 47.0 us forward and 88
// backward for 45.6 and 87; 10007 x 1000 packed: 55 and 128 for 52 and 127).
template <typename T>
constexpr bool kExactGates = sizeof(T) == 4;
CUBF_DEV Pair exp_minus(Pair v) {
    return each(mul2(v, both(-kLog2e)), [](float x) { return ex2(x); });
}
template <typename T>
CUBF_DEV Pair sigmoid(Pair v) {
    if constexpr (kExactGates<T>) return gate::sigmoid(v);
    return each(add2(exp_minus(v), both(1.f)), [](float x) { return rcp(x); });
}

// c softplus(Lambda) log2(e): la in units of log2 is -rate sigmoid(r).  Kept
// finite, so that a shut gate, such as the tokens past the end, makes a = 1 for
// an infinite rate too.
CUBF_DEV float softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }
CUBF_DEV Pair rates(Pair lambda, float exponent) {
    return each(lambda, [&](float v) {
        const float rate = exponent * softplus(v) * kLog2e;
        return rate > 1e30f ? 1e30f : rate;  // not fminf: NaN stays
    });
}

// a = 2^w and 1 - a^2 for w = log2(a) <= 0.  A recurrence forgets over
// 1/(1 - a) tokens and multiplies by a every time, so a has to be rounded
// without a bias and 1 - a must not cancel.  With w = n + f, n the nearest
// integer and |f| <= 1/2, t = 2^f - 1 = f P(f) comes from a polynomial (the
// Chebyshev-node least-squares fit of (2^f - 1)/f of degree five, weighted to
// equal ripples: 2.1e-8 relative with its coefficients in fp32, 6.5e-9 of 2^f),
// s = 2^n is put together from n's bits, and
//   a = s + s t,   1 - a = (1 - s) - s t,   1 - a^2 = (1 - a)(1 + a);
// for n = 0 the second is -t itself.  For w below -126.5 n's bits are those of
// zero, and a is zero: what is forgotten leaves no gradient either, whatever la.
CUBF_DEV void decay(Pair w, Pair& a, Pair& m2) {
    const Pair magic = both(12582912.f + 127.f);  // 1.5 2^23: n + 127 lands in the low bits
    w = each(w, [](float x) { return max_nan(x, -127.f); });
    const Pair r = add2(w, magic);
    const Pair f = sub2(w, sub2(r, magic));
    Pair t = fma2(f, both(0.00015403512f), both(0.0013390735f));
    t = fma2(f, t, both(0.0096182376f));
    t = fma2(f, t, both(0.055503573f));
    t = fma2(f, t, both(0.24022649f));
    t = fma2(f, t, both(0.69314718f));
    const Pair s = each(r, [](float x) { return __uint_as_float(__float_as_uint(x) << 23); });
    const Pair st = mul2(s, mul2(f, t));
    a = add2(s, st);
    const Pair q = sub2(sub2(both(1.f), s), st);
    m2 = fma2(q, a, q);
}
// 1/sqrt(1 - a^2); where a = 1 (a gate that is shut) finite, so that its
// products with 1 - a^2 = 0 and log a = 0 vanish as their limits do.
CUBF_DEV Pair inverse_root(Pair m2) {
    return each(add2(m2, both(1e-37f)), [](float x) { return rsq(x); });
}

// sqrt(1 - a^2) sigmoid(i) x from 1 - a^2.  In 16-bit calls with Q = 1 + e^-i,
// sqrt(m2)/Q = m2/sqrt(m2 Q^2), one special-function instruction for root and
// quotient.  Q^2 may reach infinity there, for i below -44, where the factor
// (below 1e-19) is taken as zero.
template <typename T>
CUBF_DEV Pair drive(Pair m2, Pair i, Pair x) {
    if constexpr (kExactGates<T>) {
        return mul2(mul2(mul2(m2, inverse_root(m2)), sigmoid<T>(i)), x);
    } else {
        const Pair q = add2(exp_minus(i), both(1.f));
        const Pair root = each(mul2(add2(m2, both(1e-37f)), mul2(q, q)), [](float v) { return rsq(v); });
        return mul2(mul2(m2, root), x);
    }
}

// ---- joining runs -----------------------------------------------------------------------------
// In packed batches a run that holds a sequence's first token forgets what
// came before it whatever that was (a product with zero would keep its NaN):
// its A is the marker -0 in both channels, which no product of decays (all
// >= +0) produces.
constexpr Pair kMarker = 0x8000000080000000ULL;
CUBF_DEV bool marked(Pair a) { return static_cast<uint32_t>(a) == 0x80000000u; }

template <bool PACKED>
CUBF_DEV Pair through(Pair a, Pair h, Pair carry) {
    if (PACKED && marked(a)) return h;
    return fma2(a, carry, h);
}
template <bool PACKED>
CUBF_DEV Pair product(Pair first, Pair second) {
    if (PACKED && (marked(first) || marked(second))) return kMarker;
    return mul2(first, second);
}

// Walks the sequences of a packed batch along increasing tokens.
struct Walker {
    const int* offsets;
    int last;  // sequences - 1
    int at;    // the sequence of the current token
    int start, stop;
    CUBF_DEV void init(const int* o, int sequences) {
        offsets = o;
        last = sequences - 1;
        rewind();
    }
    CUBF_DEV void rewind() {
        at = 0;
        start = offsets[0];
        stop = offsets[1];
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
};

// Which tokens of a run [t, t + n) are their sequence's first and last (bit s:
// token t + s), and the sequences of its first and last token.
struct Marks {
    unsigned starts = 0, ends = 0;
    int first = 0, last = 0;

    CUBF_DEV bool none() const { return (starts | ends) == 0; }
    // `seq` moves to the run's last token
    CUBF_DEV void find(Walker& seq, int t, int n, int length) {
        seq.seek(t);
        first = last = seq.at;
        n = n < length - t ? n : length - t;
        if (n <= 0) return;
        if (seq.start >= t && seq.start < t + n) starts = 1u << (seq.start - t);
        while (seq.stop <= t + n) {
            if (seq.stop > t) ends |= 1u << (seq.stop - 1 - t);
            if (seq.stop == t + n || seq.at >= seq.last) break;
            seq.seek(seq.stop);
            if (seq.start < t || seq.start >= t + n) break;  // offsets that do not ascend
            starts |= 1u << (seq.start - t);
            last = seq.at;
        }
    }
};
// The next sequence after `at` that has tokens, and the one before.
CUBF_DEV int following(const int* offsets, int sequences, int at) {
    for (++at; at + 1 < sequences && offsets[at + 1] <= offsets[at];) ++at;
    return at < sequences ? at : sequences - 1;
}
CUBF_DEV int preceding(const int* offsets, int at) {
    for (--at; at > 0 && offsets[at + 1] <= offsets[at];) --at;
    return at > 0 ? at : 0;
}

// Hand-over from one warp to another on a named barrier that counts both
// warps: the giver's shared-memory writes before give() are seen after take().
// A giver comes back to a barrier only after what it gave has come round, so a
// barrier never holds two hand-overs.
CUBF_DEV void give(int barrier) { asm volatile("bar.arrive %0, 64;" ::"r"(barrier) : "memory"); }
CUBF_DEV void take(int barrier) { asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory"); }

// The affine map of a run, and of the runs of the lane groups before (or with
// REVERSE after) this lane's own, and of all of them.
template <int GROUPS, bool PACKED, bool REVERSE>
struct Joined {
    Pair before_a, before_h, a, h;

    static CUBF_DEV Pair from(Pair v, int lane) {
        return __shfl_sync(0xffffffffu, v, lane);
    }
    CUBF_DEV void join(Pair run_a, Pair run_h, int lane) {
        a = run_a;
        h = run_h;
        before_a = both(1.f);
        before_h = both(0.f);
        if constexpr (GROUPS > 1) {
            constexpr int kLanes = 32 / GROUPS;
            const int group = REVERSE ? GROUPS - 1 - lane / kLanes : lane / kLanes;
#pragma unroll
            for (int d = 1; d < GROUPS; d *= 2) {  // inclusive over the groups
                const int src = (lane + (REVERSE ? d : -d) * kLanes) & 31;
                const Pair pa = from(a, src), ph = from(h, src);
                if (group >= d) {
                    h = through<PACKED>(a, h, ph);
                    a = product<PACKED>(pa, a);
                }
            }
            const int src = (lane + (REVERSE ? 1 : -1) * kLanes) & 31;
            const Pair pa = from(a, src), ph = from(h, src);
            if (group > 0) {
                before_a = pa;
                before_h = ph;
            }
            const int last = lane % kLanes + (REVERSE ? 0 : (GROUPS - 1) * kLanes);
            a = from(a, last);
            h = from(h, last);
        }
    }
};

// ---- forward ----------------------------------------------------------------------------------
template <typename T, int GROUPS, int PIECE>
using ForwardRows = RowsOf<T, 3, kForwardSteps<T, PIECE>, 2, GROUPS, PIECE>;

template <typename T, bool PACKED, int GROUPS, int PIECE>
__global__ void __launch_bounds__(kWarps * 32, 2) gated_scan_kernel(GatedScanArgs p, int tiles) {
    using Tile = ForwardRows<T, GROUPS, PIECE>;
    constexpr int kSteps = Tile::STEPS, stride = Tile::TOKENS * kWarps;  // tokens a CTA takes a round
    extern __shared__ __align__(16) unsigned char staged[];
    __shared__ Pair handed[kWarps][32];  // h before the warp's tokens
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int group = lane / (32 / GROUPS);
    const int c0 = static_cast<int>(blockIdx.x % tiles) * Tile::kChannels;
    const Lane<GROUPS> ln(c0, lane, p.dim);
    const size_t b = blockIdx.x / tiles;
    int w0 = warp * Tile::TOKENS;  // the warp's first token; the lane's run begins at t0
    Tile rows{{static_cast<const T*>(p.x) + b * p.x_batch, static_cast<const T*>(p.r) + b * p.r_batch,
               static_cast<const T*>(p.i) + b * p.i_batch},
              {p.x_token, p.r_token, p.i_token}};
    rows.init(staged + warp * Tile::STAGES * Tile::kBytes, lane, c0, p.length, p.dim, w0);
#pragma unroll
    for (int k = 0; k < Tile::STAGES; ++k) rows.fetch(k, w0 + k * stride, stride);
    T* out = static_cast<T*>(p.h) + b * static_cast<size_t>(p.length) * p.dim;
    const Pair rate = mul2(rates(ln.load32(p.decay), p.exponent), both(-1.f));
    float* chunk_states = nullptr;
    if (p.chunk_states)
        chunk_states = p.chunk_states +
                       b * static_cast<size_t>((p.length + kGatedScanChunk - 1) / kGatedScanChunk) * p.dim;

    Walker seq;
    if constexpr (PACKED) {
        seq.init(p.offsets, p.sequences);
        if (group == 0)  // sequences without tokens end where they began
            for (int j = warp; j < p.sequences; j += kWarps)
                if (p.offsets[j] >= p.offsets[j + 1])
                    ln.store32(p.last + static_cast<size_t>(j) * p.dim,
                               p.initial ? ln.load32(p.initial + static_cast<size_t>(j) * p.dim) : both(0.f));
    }
    Pair carry = both(0.f);  // h before the sequence, in the end after it
    if (!PACKED && p.initial) carry = ln.load32(p.initial + b * p.dim);

    const int rounds = (p.length + stride - 1) / stride;
    for (int round = 0; round < rounds; ++round, w0 += stride) {
        const int buf = round & 1, t0 = w0 + group * kSteps;
        // Tokens past the end are a shut gate (r = -inf: a = 1) over x = 0:
        // the identity map.
        Pair a[kSteps], u[kSteps];
        rows.arrive();
        rows.begin(t0);
        rows.close(buf, 1, t0, Raw<T>::lowest());
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            Pair m2;
            decay(mul2(rate, sigmoid<T>(rows.get(buf, 1, s))), a[s], m2);
            u[s] = drive<T>(m2, rows.get(buf, 2, s), rows.get(buf, 0, s));
        }
        Marks marks;
        if constexpr (PACKED) {
            marks.find(seq, t0, kSteps, p.length);
            if (marks.starts && p.initial) {  // the initial states enter with the first tokens
                int at = marks.starts & 1u ? marks.first : following(p.offsets, p.sequences, marks.first);
                for (unsigned left = marks.starts; left; left &= left - 1) {
                    const Pair h0 = ln.load32(p.initial + static_cast<size_t>(at) * p.dim);
                    const int token = __ffs(left) - 1;
#pragma unroll
                    for (int s = 0; s < kSteps; ++s)
                        if (s == token) u[s] = fma2(a[s], h0, u[s]);
                    at = following(p.offsets, p.sequences, at);
                }
            }
        }
        // One way for the whole warp: two in turn would take as long as both.
        const bool plain = !PACKED || __all_sync(0xffffffffu, marks.none());
        Pair A = both(1.f), H = both(0.f);
        if (plain) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                A = mul2(A, a[s]);
                H = fma2(a[s], H, u[s]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                A = mul2(A, a[s]);
                H = (marks.starts >> s) & 1u ? u[s] : fma2(a[s], H, u[s]);
            }
            if (marks.starts) A = kMarker;
        }
        // The state goes from warp to warp, and from the last one to the first
        // one's next tile; no barrier holds all warps, so they drift apart and
        // one's loads, gates and stores overlap another's.
        Joined<GROUPS, PACKED, false> runs;
        runs.join(A, H, lane);
        Pair h = carry;
        if (warp > 0 || round > 0) {
            take(1 + warp);
            h = handed[warp][lane];
        }
        const Pair next = through<PACKED>(runs.a, runs.h, h);
        if (warp + 1 < kWarps || round + 1 < rounds) {
            const int to = (warp + 1) % kWarps;
            handed[to][lane] = next;
            give(1 + to);
        } else {
            carry = next;
        }
        if (GROUPS > 1 && group > 0) h = through<PACKED>(runs.before_a, runs.before_h, h);  // before the lane's run
        if (chunk_states && t0 % kGatedScanChunk == 0 && t0 < p.length)
            ln.store32(chunk_states + static_cast<size_t>(t0 / kGatedScanChunk) * p.dim, h);
        if (plain) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                h = fma2(a[s], h, u[s]);
                rows.put(buf, 0, s, h);
            }
        } else {
            int at = marks.first;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                h = (marks.starts >> s) & 1u ? u[s] : fma2(a[s], h, u[s]);
                rows.put(buf, 0, s, h);
                if ((marks.ends >> s) & 1u) {
                    ln.store32(p.last + static_cast<size_t>(at) * p.dim, h);
                    at = following(p.offsets, p.sequences, at);
                }
            }
        }
        __syncwarp();
        rows.flush(buf, 0, out, w0);
        __syncwarp();  // the tile has been read
        rows.fetch(buf, w0 + Tile::STAGES * stride, stride);
    }
    if (!PACKED && warp == kWarps - 1 && group == 0) ln.store32(p.last + b * p.dim, carry);
}

// ---- backward ----------------------------------------------------------------------------------
// G_t = dh_t + P_{t+1}, P_t = a_t G_t runs from the end of time by the same
// joins; h_{t-1} is run again from the chunk state the forward kept, in fp32,
// instead of read back in the outputs' type.  With m = sqrt(1 - a^2),
// v = m sigmoid(i) and e = dL/d(la) la (d m/d la = -a^2/m):
//   dx = G v                  di = dx x (1 - sigmoid(i))
//   e  = a G la (h_{t-1} - sigmoid(i) x a/m)
//   dr = e (1 - sigmoid(r))   dLambda = sum e sigmoid(Lambda)/softplus(Lambda)
// A thread keeps a, v, 1/m and sigmoid(r) of its tokens and gets sigmoid(i)
// back as v/m, which leaves room for two CTAs per SM.
template <typename T, int GROUPS, int PIECE>
using BackwardRows = RowsOf<T, 4, kBackwardSteps, sizeof(T) == 2 ? 2 : 1, GROUPS, PIECE>;

template <typename T, bool PACKED, int GROUPS, int PIECE>
__global__ void __launch_bounds__(kWarps * 32, 2) gated_scan_backward_kernel(GatedScanArgs p, int tiles) {
    using Tile = BackwardRows<T, GROUPS, PIECE>;
    constexpr int kSteps = Tile::STEPS, stride = Tile::TOKENS * kWarps;  // tokens a CTA takes a round
    extern __shared__ __align__(16) unsigned char staged[];
    __shared__ Pair handed[kWarps][32];  // P from the tokens after the warp's
    __shared__ Pair middle[kWarps][32];  // h before the warp's tokens, where the warp before has it
    __shared__ Pair sums[kWarps][32];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int group = lane / (32 / GROUPS);
    const int c0 = static_cast<int>(blockIdx.x % tiles) * Tile::kChannels;
    const Lane<GROUPS> ln(c0, lane, p.dim);
    const size_t b = blockIdx.x / tiles;
    const int rounds = (p.length + stride - 1) / stride;
    int w0 = (rounds - 1) * stride + warp * Tile::TOKENS;  // the warp's first token; the lane's run begins at t0
    Tile rows{{static_cast<const T*>(p.x) + b * p.x_batch, static_cast<const T*>(p.r) + b * p.r_batch,
               static_cast<const T*>(p.i) + b * p.i_batch, static_cast<const T*>(p.d_h) + b * p.dh_batch},
              {p.x_token, p.r_token, p.i_token, p.dh_token}};
    rows.init(staged + warp * Tile::STAGES * Tile::kBytes, lane, c0, p.length, p.dim, w0);
#pragma unroll
    for (int k = 0; k < Tile::STAGES; ++k) rows.fetch(k, w0 - k * stride, -stride);
    const size_t out = b * static_cast<size_t>(p.length) * p.dim;
    T* dx = static_cast<T*>(p.d_x) + out;
    T* dr = static_cast<T*>(p.d_r) + out;
    T* di = static_cast<T*>(p.d_i) + out;
    const Pair rate = mul2(rates(ln.load32(p.decay), p.exponent), both(-1.f));
    const Pair rate_e = mul2(rate, both(kLn2));  // of la itself
    const float* chunk_states =
        p.chunk_states + b * static_cast<size_t>((p.length + kGatedScanChunk - 1) / kGatedScanChunk) * p.dim;

    Walker seq;
    if constexpr (PACKED) {
        seq.init(p.offsets, p.sequences);
        if (p.d_initial && group == 0)  // sequences without tokens pass their gradient through
            for (int j = warp; j < p.sequences; j += kWarps)
                if (p.offsets[j] >= p.offsets[j + 1])
                    ln.store32(p.d_initial + static_cast<size_t>(j) * p.dim,
                               p.d_last ? ln.load32(p.d_last + static_cast<size_t>(j) * p.dim) : both(0.f));
    }
    Pair carry = both(0.f);  // P from after the sequence, in the end from all of it
    if (!PACKED && p.d_last) carry = ln.load32(p.d_last + b * p.dim);
    Pair sum = both(0.f);    // of e

    for (int round = 0; round < rounds; ++round, w0 -= stride) {  // from the end of time
        const int stage = Tile::STAGES == 2 ? round & 1 : 0, t0 = w0 + group * kSteps;
        // before the run: from the forward, or (below) from the run before in its chunk
        Pair h = both(0.f);
        const bool second = (GROUPS > 1 ? group : warp) % 2;
        if (!second && t0 < p.length)
            h = ln.load32(chunk_states + static_cast<size_t>(t0 / kGatedScanChunk) * p.dim);
        // x and dh are read where they are used, from shared memory
        Pair a[kSteps], v[kSteps], im[kSteps], sr[kSteps];
        rows.arrive();
        rows.begin(t0);
        rows.close(stage, 1, t0, Raw<T>::lowest());
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            Pair m2;
            sr[s] = sigmoid<T>(rows.get(stage, 1, s));
            decay(mul2(rate, sr[s]), a[s], m2);
            im[s] = inverse_root(m2);
            v[s] = mul2(mul2(m2, im[s]), sigmoid<T>(rows.get(stage, 2, s)));
        }
        auto x_of = [&](int s) { return rows.get(stage, 0, s); };
        auto dh_of = [&](int s) { return rows.get(stage, 3, s); };

        // the maps of the run, forward and backward
        Pair A = both(1.f), H = both(0.f), R = both(0.f);
        Marks marks;
        if constexpr (PACKED) {
            if (t0 < seq.start) seq.rewind();
            marks.find(seq, t0, kSteps, p.length);
        }
        const bool plain = !PACKED || __all_sync(0xffffffffu, marks.none());  // one way for the whole warp
        // h before a sequence's first token, and the final state's gradient at its last
        auto initial_of = [&](int at) {
            return p.initial ? ln.load32(p.initial + static_cast<size_t>(at) * p.dim) : both(0.f);
        };
        auto last_of = [&](int at) {
            return p.d_last ? ln.load32(p.d_last + static_cast<size_t>(at) * p.dim) : both(0.f);
        };
        if (plain) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                A = mul2(A, a[s]);
                H = fma2(a[s], H, mul2(v[s], x_of(s)));
            }
#pragma unroll
            for (int s = kSteps - 1; s >= 0; --s) R = mul2(a[s], add2(dh_of(s), R));
        } else {
            int at = marks.first;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                if ((marks.starts >> s) & 1u) {
                    if (s > 0) at = following(p.offsets, p.sequences, at);
                    H = initial_of(at);
                }
                A = mul2(A, a[s]);
                H = fma2(a[s], H, mul2(v[s], x_of(s)));
            }
            if (marks.starts) A = kMarker;
            at = marks.last;
#pragma unroll
            for (int s = kSteps - 1; s >= 0; --s) {
                Pair d = dh_of(s);
                if ((marks.ends >> s) & 1u) d = add2(d, last_of(at));
                R = mul2(a[s], add2(d, R));
                if ((marks.starts >> s) & 1u) {
                    R = both(0.f);
                    at = preceding(p.offsets, at);
                }
            }
        }
        // h from the run before, within a chunk
        const Pair middle_h = through<PACKED>(A, H, h);
        if constexpr (GROUPS > 1) {
            const Pair before = __shfl_sync(0xffffffffu, middle_h, (lane - 32 / GROUPS) & 31);
            if (second) h = before;
        } else if (!second) {
            middle[warp + 1][lane] = middle_h;
            give(1 + kWarps + warp / 2);
        } else {
            take(1 + kWarps + warp / 2);
            h = middle[warp][lane];
        }
        // P from warp to warp, as the forward's state, from the end of time
        Joined<GROUPS, PACKED, true> runs;
        runs.join(A, R, lane);
        Pair P = carry;
        if (warp + 1 < kWarps || round > 0) {
            take(1 + warp);
            P = handed[warp][lane];
        }
        const Pair next = through<PACKED>(runs.a, runs.h, P);
        if (warp > 0 || round + 1 < rounds) {
            const int to = (warp + kWarps - 1) % kWarps;
            handed[to][lane] = next;
            give(1 + to);
        } else {
            carry = next;
        }
        if (GROUPS > 1 && group + 1 < GROUPS) P = through<PACKED>(runs.before_a, runs.before_h, P);

        // h before each token, then the gradients from the last token back
        Pair before[kSteps];
        auto gradients = [&](int s, Pair d) {
            const Pair fx = x_of(s);
            const Pair G = add2(d, P);
            const Pair gx = mul2(G, v[s]), si = mul2(v[s], im[s]);
            const Pair gi = mul2(mul2(gx, fx), sub2(both(1.f), si));
            P = mul2(a[s], G);
            const Pair e = mul2(mul2(P, mul2(rate_e, sr[s])), sub2(before[s], mul2(mul2(mul2(si, fx), a[s]), im[s])));
            rows.put(stage, 0, s, gx);
            rows.put(stage, 1, s, mul2(e, sub2(both(1.f), sr[s])));
            rows.put(stage, 2, s, gi);
            return e;
        };
        if (plain) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                before[s] = h;
                h = fma2(a[s], h, mul2(v[s], x_of(s)));
            }
            const bool whole = t0 + kSteps <= p.length;
#pragma unroll
            for (int s = kSteps - 1; s >= 0; --s) {
                const Pair e = gradients(s, dh_of(s));
                if (whole || t0 + s < p.length) sum = add2(sum, e);
            }
        } else {
            int at = marks.first;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                if ((marks.starts >> s) & 1u) {
                    if (s > 0) at = following(p.offsets, p.sequences, at);
                    h = initial_of(at);
                }
                before[s] = h;
                h = fma2(a[s], h, mul2(v[s], x_of(s)));
            }
            at = marks.last;
#pragma unroll
            for (int s = kSteps - 1; s >= 0; --s) {
                Pair d = dh_of(s);
                if ((marks.ends >> s) & 1u) d = add2(d, last_of(at));
                const Pair e = gradients(s, d);
                if (t0 + s < p.length) sum = add2(sum, e);
                if ((marks.starts >> s) & 1u) {
                    if (p.d_initial) ln.store32(p.d_initial + static_cast<size_t>(at) * p.dim, P);
                    P = both(0.f);
                    at = preceding(p.offsets, at);
                }
            }
        }
        __syncwarp();
        rows.flush(stage, 0, dx, w0);
        rows.flush(stage, 1, dr, w0);
        rows.flush(stage, 2, di, w0);
        __syncwarp();  // the tile has been read
        rows.fetch(stage, w0 - Tile::STAGES * stride, -stride);
    }
    if (!PACKED && p.d_initial && warp == 0 && group == 0) ln.store32(p.d_initial + b * p.dim, carry);
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && group == 0) {
        sum = both(0.f);
        for (int k = 0; k < kWarps; ++k)
            for (int q = 0; q < GROUPS; ++q) sum = add2(sum, sums[k][lane + q * (32 / GROUPS)]);
        ln.store32(p.partials + b * static_cast<size_t>(p.dim), sum);
    }
}

// dLambda = sigmoid(Lambda)/softplus(Lambda) sum e over the CTAs' partial sums
// (the ratio tends to 1 as both vanish).
template <typename T>
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
constexpr int kStepRows = 4;
// PAIRS, WIDE: pairs of channels of the rows, of the fp32 states are aligned.
template <typename T, bool PAIRS, bool WIDE>
__global__ void __launch_bounds__(128) gated_scan_step_kernel(GatedStepArgs p, int tiles, int rows) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const unsigned task = blockIdx.x * 4 + (threadIdx.x >> 5);
    const Lane<1> ln(static_cast<int>(task % tiles) * kWarpChannels, lane, p.dim);
    const size_t first = static_cast<size_t>(task / tiles) * rows;
    if (first >= p.batch) return;
    const size_t end = first + rows < p.batch ? first + rows : p.batch;
    const Pair rate = mul2(rates(ln.load32(p.decay), p.exponent), both(-1.f));
    // kStepRows requests at a time, all their loads before the arithmetic of the first
    for (size_t b0 = first; b0 < end; b0 += kStepRows) {
        long long slot[kStepRows];
        Pair x[kStepRows], r[kStepRows], i[kStepRows], state[kStepRows];
#pragma unroll
        for (int k = 0; k < kStepRows; ++k) {
            const size_t b = b0 + k < end ? b0 + k : end - 1;
            slot[k] = p.slots ? p.slots[b] : static_cast<long long>(b);
            x[k] = ln.template load<PAIRS>(static_cast<const T*>(p.x) + b * p.x_row);
            r[k] = ln.template load<PAIRS>(static_cast<const T*>(p.r) + b * p.r_row);
            i[k] = ln.template load<PAIRS>(static_cast<const T*>(p.i) + b * p.i_row);
        }
#pragma unroll
        for (int k = 0; k < kStepRows; ++k) {
            const bool in = slot[k] >= 0 && slot[k] < static_cast<long long>(p.pool);
            if (!in) slot[k] = -1;
            state[k] = in ? ln.template load<WIDE>(p.state + static_cast<size_t>(slot[k]) * p.dim) : both(0.f);
        }
#pragma unroll
        for (int k = 0; k < kStepRows; ++k) {
            if (b0 + k >= end) break;
            Pair a, m2;
            decay(mul2(rate, sigmoid<T>(r[k])), a, m2);
            const Pair n = fma2(a, state[k], drive<T>(m2, i[k], x[k]));
            ln.template store<PAIRS>(static_cast<T*>(p.h) + (b0 + k) * p.dim, slot[k] < 0 ? both(0.f) : n);
            if (slot[k] >= 0) ln.template store<WIDE>(p.new_state + static_cast<size_t>(slot[k]) * p.dim, n);
        }
    }
}

}  // namespace cubf::scan
