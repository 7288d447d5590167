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
// 16-bit tensors: gated_delta_tc.cuh; fp32 ones: gated_delta_fp32.cuh.  Here: what both use, and the kernel of one token.
#pragma once

#include "gated_delta.hpp"
#include "mma_split.cuh"

namespace cubf::delta {

using namespace split;

constexpr int C = kDeltaChunk;
constexpr int kPitchC = C + 8;           // of 64-wide tiles
constexpr float kLeast = -128.f;         // e^-128 is zero in fp32: a log decay below it is taken as it

template <typename T>
constexpr int kInput = std::is_same_v<T, __half> ? 2 : 1;  // bf16 pieces that hold a 16-bit input exactly
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

// A fragment of 16 columns out of two accumulator tiles.
template <int N>
CUBF_DEV void operand(const float (&a)[4], const float (&b)[4], uint32_t (&f)[N][4]) {
    fragment<N>(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], f);
}

// ---- tokens of no sequence ----------------------------------------------------------------------
// Before the first offset of a packed batch and behind the last one: their outputs or gradients are zero, as a padded
// batch's other rows are.  (Left as they were allocated they could be NaN, which a zero gradient does not mask.)
template <typename T>
__global__ void __launch_bounds__(256) gated_delta_rest_kernel(GatedDeltaArgs a, bool backward) {
    pdl_begin();
    const size_t first = static_cast<size_t>(offset_at(a, 0)), last = static_cast<size_t>(offset_at(a, a.sequences));
    auto zero = [&](void* p, size_t width) {             // 16-bit units a token
        auto* const x = static_cast<uint16_t*>(p);
        const size_t step = static_cast<size_t>(gridDim.x) * 256, from = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
        for (size_t e = from; e < first * width; e += step) x[e] = 0;
        for (size_t e = last * width + from; e < a.length * width; e += step) x[e] = 0;
    };
    constexpr size_t units = sizeof(T) / 2;
    const size_t values = a.heads * a.v_dim * units, keys = a.k_heads * a.k_dim * units;
    if (!backward) return zero(a.o, values);
    zero(a.d_q, keys);
    zero(a.d_k, keys);
    zero(a.d_v, values);
    zero(a.d_log_decay, a.heads * (a.log_decay32 ? 2 : 1));
    zero(a.d_beta, a.heads * (a.beta32 ? 2 : 1));
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
