// pk_umma.cuh -- sm_100a building blocks shared by libparakeet_cuda's tensor-memory
// kernels (pk_encproj.cu: the enc-proj GEMM; pk_bulk.cu: the step loop for large
// live batches; pk_mx4.cu, pk_fp8.cu: the 4-bit and 8-bit products): mbarrier waits bounded in time, tcgen05.mma operand descriptors
// for 128-byte-swizzled K-major f16 tiles, the kind::f16 instruction descriptor,
// MMA issue / commit and 2-D TMA tile loads.
#pragma once

#include "pk_internal.h"

#include <cuda.h>

namespace pk {
namespace {

__device__ __forceinline__ unsigned smem_u32(const void * p) { return (unsigned) __cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(unsigned long long * b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_u32(b)), "r"(count) : "memory");
}

__device__ __forceinline__ bool mbar_test(unsigned long long * b, unsigned parity) {
    unsigned done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done) : "r"(smem_u32(b)), "r"(parity) : "memory");
    return done != 0;
}

// The same, acquiring at cluster scope what the other block's threads released.
__device__ __forceinline__ bool mbar_test_cluster(unsigned long long * b, unsigned parity) {
    unsigned done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done) : "r"(smem_u32(b)), "r"(parity) : "memory");
    return done != 0;
}

// Bounded wait on one phase of an mbarrier; false (and *err set) on timeout.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(unsigned long long * b, unsigned parity, long long timeout_ns, int * err) {
    unsigned long long t0 = 0;
    for (unsigned it = 0;; ++it) {
        if (CLUSTER ? mbar_test_cluster(b, parity) : mbar_test(b, parity)) return true;
        if (*reinterpret_cast<volatile int *>(err) != 0) return false;
        if ((it & 255u) == 0u) {
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (it == 0) t0 = now;
            else if ((long long) (now - t0) > timeout_ns) { atomicExch(err, 1); return false; }
        }
    }
}

__device__ __forceinline__ void mbar_arrive(unsigned long long * b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(b)) : "memory");
}

// K-major operand tile of `rows` x 128 bytes (64 f16 or 128 int8) in the 128-byte swizzle layout:
// 8-row atoms of 1024 bytes, row r at byte r * 128, 16-byte chunk c stored at
// chunk c ^ (r & 7).
__device__ __forceinline__ unsigned long long umma_desc_sw128(unsigned saddr) {
    unsigned long long d = 0;
    d |= (unsigned long long) ((saddr >> 4) & 0x3FFFu);          // start address
    d |= (unsigned long long) 1u << 16;                           // leading byte offset (unused for SW128 K-major)
    d |= (unsigned long long) (1024u >> 4) << 32;                 // stride byte offset: next 8-row atom
    d |= (unsigned long long) 1u << 46;                           // descriptor version (tcgen05)
    d |= (unsigned long long) 2u << 61;                           // layout: 128-byte swizzle
    return d;
}

// kind::f16 instruction descriptor: f32 accumulator, f16 A and B, both K-major.
__host__ __device__ constexpr unsigned umma_idesc_f16(int m, int n) {
    return (1u << 4)                          // D format f32
         | (0u << 7) | (0u << 10)             // A, B format f16
         | ((unsigned) (n >> 3) << 17)        // N / 8
         | ((unsigned) (m >> 4) << 24);       // M / 16
}

__device__ __forceinline__ void umma_f16(unsigned tmem_d, unsigned long long adesc, unsigned long long bdesc,
                                         unsigned idesc, unsigned accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                 :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// kind::i8 instruction descriptor: s32 accumulator, signed 8-bit A and B, both K-major.
__host__ __device__ constexpr unsigned umma_idesc_s8(int m, int n) {
    return (2u << 4)                          // D format s32
         | (1u << 7) | (1u << 10)             // A, B format signed 8-bit
         | ((unsigned) (n >> 3) << 17)        // N / 8
         | ((unsigned) (m >> 4) << 24);       // M / 16
}

// One kind::i8 MMA (K = 32 bytes of each operand row).
__device__ __forceinline__ void umma_i8(unsigned tmem_d, unsigned long long adesc, unsigned long long bdesc,
                                        unsigned idesc, unsigned accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }"
                 :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// kind::mxf4 instruction descriptor: f32 accumulator, e2m1 A and B, both K-major, e8m0 scales, one
// per 32 values; `id` (0 or 2) names the first of the two scale bytes that a K = 64 product reads of
// each row's 4-byte scale word.
__host__ __device__ constexpr unsigned umma_idesc_mxf4(int m, int n, int id) {
    return ((unsigned) id << 4)               // B scale id
         | (1u << 7) | (1u << 10)             // A, B format e2m1
         | ((unsigned) (n >> 3) << 17)        // N / 8
         | (1u << 23)                         // e8m0 scales
         | ((unsigned) (m >> 7) << 27)        // M / 128
         | ((unsigned) id << 29);             // A scale id
}

// One block-scaled product of 64 values of K (32 bytes of each operand row); sfa, sfb: tensor-memory
// addresses of the rows' scale words (row r in lane r % 32, column r / 32). PAIR: over a pair of blocks
// (M = 256), issued by the pair's first block, each block's operand and scale rows at the same places
// of its own shared and tensor memory.
template <bool PAIR>
__device__ __forceinline__ void umma_mxf4(unsigned tmem_d, unsigned long long adesc, unsigned long long bdesc, unsigned idesc,
                                          unsigned sfa, unsigned sfb, unsigned accumulate) {
    if (PAIR)
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p; }"
                     :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p; }"
                     :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}

// kind::mxf8f6f4 instruction descriptor: f32 accumulator, e4m3 A and B, both K-major, e8m0 scales; `id` (0 to 3)
// names the byte of each row's 4-byte scale word that a K = 32 product reads.
__host__ __device__ constexpr unsigned umma_idesc_mxf8(int m, int n, int id) {
    return ((unsigned) id << 4)               // B scale id
         | (0u << 7) | (0u << 10)             // A, B format e4m3
         | ((unsigned) (n >> 3) << 17)        // N / 8
         | (1u << 23)                         // e8m0 scales
         | ((unsigned) (m >> 7) << 27)        // M / 128
         | ((unsigned) id << 29);             // A scale id
}

// One block-scaled product of 32 values of K (32 bytes of each operand row); scales and PAIR as above.
template <bool PAIR>
__device__ __forceinline__ void umma_mxf8(unsigned tmem_d, unsigned long long adesc, unsigned long long bdesc, unsigned idesc,
                                          unsigned sfa, unsigned sfb, unsigned accumulate) {
    if (PAIR)
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p; }"
                     :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p; }"
                     :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}

// 512 bytes of scale words (32 rows of 16 bytes) from shared memory to four tensor-memory columns,
// the same for each of the four lane quarters. Ordered before products that the same thread issues.
template <bool PAIR>
__device__ __forceinline__ void umma_copy_scales(unsigned tmem, unsigned long long desc) {
    if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc) : "memory");
}
// Their descriptor: no swizzle, the next 8 rows of 16 bytes 128 bytes on.
__device__ __forceinline__ unsigned long long scale_desc(unsigned saddr) {
    return (unsigned long long) ((saddr >> 4) & 0x3FFFu) | (unsigned long long) (128u >> 4) << 32 | (unsigned long long) 1u << 46;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile("{ .reg .pred q; elect.sync _|q, 0xFFFFFFFF; selp.u32 %0, 1, 0, q; }" : "=r"(p));
    return p != 0;
}

// Arrives on the barrier at this place of both blocks once the pair's products so far are done.
__device__ __forceinline__ void umma_commit_pair(unsigned long long * b) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(smem_u32(b)), "h"((unsigned short) 3) : "memory");
}

// Address in the cluster's window of what lies at this place of its block `rank`.
__device__ __forceinline__ unsigned mbar_at(unsigned long long * b, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(b)), "r"(rank));
    return r;
}
// Arrives there, releasing at cluster scope.
__device__ __forceinline__ void mbar_arrive_at(unsigned long long * b, unsigned rank) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(mbar_at(b, rank)) : "memory");
}

// The same without releasing anything: for a thread that has read tensor memory (tcgen05.wait::ld) and tells so. Releasing
// would first wait for its global stores.
__device__ __forceinline__ void mbar_arrive_at_relaxed(unsigned long long * b, unsigned rank) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" :: "r"(mbar_at(b, rank)) : "memory");
}

__device__ __forceinline__ void umma_commit(unsigned long long * b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 :: "r"(smem_u32(b)) : "memory");
}

__device__ __forceinline__ void tma_load_2d(void * dst, const CUtensorMap * map, int x, int y, unsigned long long * bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}

// The same for a block of a pair: the bytes arrive on a barrier of either block (`bar`: its address in
// the cluster's window, see mbar_at).
__device__ __forceinline__ void tma_load_2d_pair(void * dst, const CUtensorMap * map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Untiled copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) to shared memory.
__device__ __forceinline__ void bulk_load(void * dst, const void * src, unsigned bytes, unsigned long long * bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void mbar_expect(unsigned long long * b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(smem_u32(b)), "r"(bytes) : "memory");
}

// Counts `bytes` as arrived on the barrier's phase, in place of a copy that was expected and never issued.
__device__ __forceinline__ void mbar_complete(unsigned long long * b, unsigned bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" :: "r"(smem_u32(b)), "r"(bytes) : "memory");
}

// 16 columns of this warp's 32 tensor-memory lanes (issue only; tcgen05.wait::ld before use).
__device__ __forceinline__ void tmem_load16(unsigned taddr, unsigned * v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr));
}

// 32 columns of this warp's 32 tensor-memory lanes (issue only; tcgen05.wait::ld before use).
__device__ __forceinline__ void tmem_load32(unsigned taddr, unsigned * v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
                   "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
                   "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(taddr));
}

}  // namespace
}  // namespace pk
