// mma_split.cuh -- fp32 products on the bf16 tensor pipe, operands split into
// bf16 pieces.
//
// A value x is held as x0 + x1 + x2, each piece the bf16 nearest to what the
// pieces before it left: two pieces are within 2^-16 of it, three within 2^-24
// (half a step of bf16, 2^-8, a piece).  bf16 inputs are one piece, fp16 ones
// two (11 bits), both exactly; fp32 values three.  A product of level L adds
// the piece products a_i b_j with i + j < L: what is left out is below 2^-8L of
// the product, so level 3 is an fp32 product and level 2 keeps 16 bits.  One
// m16n8k16 does 2048 multiply-adds, so a level-3 product with an exact bf16
// operand runs at a third of the bf16 rate, 2.7 times that of fp32 FMAs.
#pragma once

#include "common.cuh"

namespace cubf::split {

CUBF_DEV uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

CUBF_DEV uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Pieces of the pair (x, y), x in the low half.
template <int N>
CUBF_DEV void pieces(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = pack(x, y);
        if (i + 1 < N) {
            x -= __uint_as_float(p[i] << 16);
            y -= __uint_as_float(p[i] & 0xffff0000u);
        }
    }
}

// 16 x 16 A fragment out of four pairs (rows r and r + 8 of columns c, c + 1 and c + 8, c + 9).
template <int N>
CUBF_DEV void fragment(float a0, float a1, float b0, float b1, float c0, float c1, float d0, float d1,
                       uint32_t (&f)[N][4]) {
    uint32_t p[N];
    pieces<N>(a0, a1, p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i][0] = p[i];
    pieces<N>(b0, b1, p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i][1] = p[i];
    pieces<N>(c0, c1, p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i][2] = p[i];
    pieces<N>(d0, d1, p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i][3] = p[i];
}

CUBF_DEV void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

CUBF_DEV void ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
CUBF_DEV void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// A tile of bf16 pieces in shared memory: PITCH values a row, STEP values a piece.  Rows are 16 bytes times an odd
// number apart, so that the eight rows of an ldmatrix lie in different banks.
template <int PITCH, int STEP>
struct Tile {
    static_assert(PITCH % 16 == 8, "rows in different banks");
    uint32_t base;
    CUBF_DEV uint32_t at(int piece, int row, int col) const {
        return base + static_cast<uint32_t>(piece * STEP + row * PITCH + col) * 2u;
    }
    // B fragments (two registers each) of the tiles n .. n + 7 and n + 8 .. n + 15, rows k .. k + 15 of the product
    CUBF_DEV void b_rows(int piece, int n, int k, int lane, uint32_t (&r)[4]) const {  // stored [n][k]
        ldsm(at(piece, n + ((lane >> 4) << 3) + (lane & 7), k + ((lane >> 3) & 1) * 8), r);
    }
    CUBF_DEV void b_cols(int piece, int k, int n, int lane, uint32_t (&r)[4]) const {  // stored [k][n]
        ldsm_t(at(piece, k + ((lane >> 3) & 1) * 8 + (lane & 7), n + ((lane >> 4) << 3)), r);
    }
    // A fragment of rows m .. m + 15 and columns k .. k + 15
    CUBF_DEV void a_rows(int piece, int m, int k, int lane, uint32_t (&r)[4]) const {  // stored [m][k]
        ldsm(at(piece, m + ((lane >> 3) & 1) * 8 + (lane & 7), k + ((lane >> 4) << 3)), r);
    }
    CUBF_DEV void a_cols(int piece, int k, int m, int lane, uint32_t (&r)[4]) const {  // stored [k][m]
        ldsm_t(at(piece, k + ((lane >> 4) << 3) + (lane & 7), m + ((lane >> 3) & 1) * 8), r);
    }
};

// d[t] += A B[t] over the piece products of a level, for NT tiles side by side: products outermost, so that NT
// independent accumulators stand between two uses of one.
template <int LEVEL, int NA, int NB, int NT>
CUBF_DEV void products(float (*d)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][NT / 2][4]) {
    static_assert(NT % 2 == 0, "tiles come in pairs");
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (i + j < LEVEL) {
#pragma unroll
                for (int t = 0; t < NT; ++t) mma(d[t], a[i], b[j][t / 2][(t & 1) * 2], b[j][t / 2][(t & 1) * 2 + 1]);
            }
}

// The same in full fp32: the tensor pipe cuts a sum's last bits at every step, always towards zero, so that an accumulator
// that runs through all piece products of a long sum loses 2^-24 of itself at each.  Here the products of 16 terms are added
// up by themselves, the smallest first, and go to the accumulator by an addition that rounds to nearest.
template <int LEVEL, int NA, int NB, int NT>
CUBF_DEV void products_rounded(float (*d)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][NT / 2][4]) {
    float sum[NT][4] = {};
#pragma unroll
    for (int size = LEVEL - 1; size >= 0; --size)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = size - i;
            if (j < 0 || j >= NB) continue;
#pragma unroll
            for (int t = 0; t < NT; ++t) mma(sum[t], a[i], b[j][t / 2][(t & 1) * 2], b[j][t / 2][(t & 1) * 2 + 1]);
        }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[t][e] += sum[t][e];
}

CUBF_DEV void copy16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
CUBF_DEV void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
CUBF_DEV void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

}  // namespace cubf::split
