// tcgen05.cuh -- the 5th-generation tensor cores for kernels whose operands
// are 64-row bf16 tiles: descriptors, MMA with the A operand in tensor memory,
// tensor-memory loads and stores, bulk copies and bounded waits.
//
// A tile is panels of 64 rows x 64 values in the canonical 128-byte-swizzled
// form: row r is 128 bytes at 128 r, its 16-byte chunk c stored at chunk
// c ^ (r % 8).  The same bytes are an operand either way round:
//   rows along N, values along K (K-major): K steps of 16 are 32 bytes apart;
//   rows along K, values along N (MN-major): K steps of 16 are 2048 bytes apart.
#pragma once

#include "common.cuh"
#include "mma_split.cuh"

namespace cubf::tc {

using split::smem_addr;

constexpr int kPanel = 8192;             // bytes of 64 x 64 values

// Byte offset of (row, col) in a tile of panels `panel` bytes apart.
CUBF_DEV uint32_t swizzled(int row, int col, int panel = kPanel) {
    return static_cast<uint32_t>((col >> 6) * panel + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2);
}

// Start, leading and stride byte offsets in 16-byte units, version 1, 128-byte swizzle.
CUBF_DEV uint64_t descriptor(uint32_t addr, uint32_t leading) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((leading >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
CUBF_DEV uint64_t rows_along_n(uint32_t addr) { return descriptor(addr, 16); }
CUBF_DEV uint64_t rows_along_k(uint32_t addr, uint32_t panel = kPanel) { return descriptor(addr, panel); }

// The other form of a tile, written and read by threads that hold a row of it each: chunks of eight values along N (or M),
// `chunk` bytes apart, each with the rows along K 16 bytes apart and not swizzled, so that a warp's 16-byte accesses to one
// chunk are side by side.  K steps of 16 are 256 bytes apart.
CUBF_DEV uint64_t chunks_along_k(uint32_t addr, uint32_t chunk) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 16) |
           (static_cast<uint64_t>((chunk >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}

// fp32 accumulators, bf16 operands, M = 128; A K-major (tensor memory) unless `a_mn`, B K-major unless `b_mn`.
constexpr uint32_t instruction(int n, bool b_mn, bool a_mn = false, int m = 128) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// D (tensor memory) (+)= A (tensor memory) B (shared memory), K = 16
CUBF_DEV void mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// The same with A in shared memory; rows 0 to 63 of D stay as they are with `upper`.
CUBF_DEV void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, bool upper = false) {
    const uint32_t off = upper ? 0xffffffffu : 0u;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %6, %6}, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(off), "r"(0u)
        : "memory");
}
CUBF_DEV void commit(uint32_t barrier) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
}
CUBF_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
CUBF_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
CUBF_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// N consecutive columns of the thread's lane, N = 16 or 32.
template <int N>
CUBF_DEV void load(uint32_t addr, uint32_t* r) {
    if constexpr (N == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(addr));
    } else {
        static_assert(N == 32, "16 or 32 columns");
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
              "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
              "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(addr));
    }
}
template <int N>
CUBF_DEV void store(uint32_t addr, const uint32_t* r) {
    static_assert(N == 16, "16 columns");
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}
CUBF_DEV void wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
CUBF_DEV void wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

CUBF_DEV void barrier_init(uint32_t barrier, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(arrivals) : "memory");
}
CUBF_DEV void barrier_arrive(uint32_t barrier) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory");
}
// One lane of a converged warp.
CUBF_DEV bool elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
CUBF_DEV void barrier_expect(uint32_t barrier, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
// A phase has ended: within some 8 us, or at once.
CUBF_DEV bool barrier_try(uint32_t barrier, uint32_t phase) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, P1;\n\t}"
        : "=r"(done)
        : "r"(barrier), "r"(phase)
        : "memory");
    return done != 0;
}
// `bytes` (a multiple of 16, both addresses 16-byte aligned) to shared memory, counted by a barrier.
CUBF_DEV void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(barrier)
                 : "memory");
}

// The same the other way; a thread's copies are done with shared memory after bulk_read.
CUBF_DEV void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
CUBF_DEV void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
CUBF_DEV void bulk_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
CUBF_DEV void bulk_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

CUBF_DEV void allocate(uint32_t* where, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
CUBF_DEV void release(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

}  // namespace cubf::tc
