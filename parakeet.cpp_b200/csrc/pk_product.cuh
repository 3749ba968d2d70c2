// pk_product.cuh -- what the products of quantised rows share (pk_mx4.cu, pk_fp8.cu): waits with a bound that
// report to a layer's error word, the meeting of a cluster's blocks, and launches.
#pragma once

#include "pk_ops.cuh"
#include "pk_umma.cuh"

#include <utility>

namespace pk {

cudaError_t encode_2d(void * map, CUtensorMapDataType type, size_t esize, const void * base, long long rows, long long cols,
                      int box_rows, int box_cols, CUtensorMapSwizzle swz);   // pk_encproj.cu
cudaError_t encode_2d_strided(void * map, CUtensorMapDataType type, const void * base, long long rows, long long cols,
                              long long stride, int box_rows, int box_cols, CUtensorMapSwizzle swz);

namespace {

constexpr long long kWaitNs = 2000000000LL;             // bound on every device-side wait, unless a layer sets another

// An allocation of tensor memory waits, without a bound, until an SM's 512 columns have room, and nothing but shared
// memory, registers and threads keeps blocks off an SM. Blocks of a cluster hold their columns while they wait for the
// cluster's others to have theirs, so two clusters that each held what the other waits for would never end. Shared memory
// rules that out: a block of a cluster that takes half of the columns asks for kClusterSmem at least, so that two fit an SM,
// not three, and none beside a block that takes all columns. (The blocks of pk_bulk.cu, which take all and wait for their grid,
// have 193 KB. Blocks without a cluster hold columns too, and wait for nobody.)
constexpr size_t kSmSmem = 228 * 1024, kBlockSmem = 1024;      // of an SM; what each block takes beside its own
constexpr size_t kClusterSmem = 76 * 1024;
constexpr bool sharing_ruled_out(size_t a, size_t b) { return a + b + 2 * kBlockSmem > kSmSmem; }
static_assert(3 * (kClusterSmem + kBlockSmem) > kSmSmem, "no three blocks of half the columns");

// Of a product's waits: their bound, where to tell that one ran out, and (a test's) that the first block, or a
// pair's second, loads nothing, so that its waits run out.
struct Waits {
    long long ns;
    int * err;
    int stall;
};

// What a layer knows of its products' waits.
struct LayerWaits {
    int * err = nullptr;                // host memory that the device sees: a wait of a product ran out
    int * err_dev = nullptr;
    long long timeouts = 0;             // times that it was found so
    int unreported = 0;                 // and no product's call has said so yet
    long long wait_ns = kWaitNs;
    int stall = 0;                      // the next product's, see Waits
};

inline void notice_timeout(LayerWaits & w) {
    if (!take_error(w.err)) return;
    __atomic_fetch_add(&w.timeouts, 1, __ATOMIC_ACQ_REL);
    __atomic_store_n(&w.unreported, 1, __ATOMIC_RELEASE);
}

inline pk_status set_wait_option(LayerWaits & w, const char * fn, int32_t option, int64_t value) {
    switch (option) {
        case PK_OPT_TIMEOUT_US:
            if (value <= 0 || value > INT64_MAX / 1000) return op_fail(PK_ERR_INVALID, fn, "timeout must be > 0");
            __atomic_store_n(&w.wait_ns, (long long) value * 1000, __ATOMIC_RELAXED);
            return PK_OK;
        case PK_OPT_TEST_STALL:
            __atomic_store_n(&w.stall, value != 0 ? 1 : 0, __ATOMIC_RELAXED);
            return PK_OK;
        default:
            return op_fail(PK_ERR_INVALID, fn, "a layer has PK_OPT_TIMEOUT_US and PK_OPT_TEST_STALL");
    }
}

// The wait of a whole warp, of one mind about its outcome.
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(unsigned long long * b, unsigned parity, long long ns, int * err) {
    return __all_sync(0xFFFFFFFFu, mbar_wait<CLUSTER>(b, parity, ns, err));
}

// Wait with a bound and nothing else to end it: for copies in flight before an early exit.
__device__ __forceinline__ void mbar_drain(unsigned long long * b, unsigned parity) {
    unsigned long long t0, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    now = t0;
    while (!mbar_test(b, parity) && (long long) (now - t0) <= kWaitNs) asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
}

__device__ __forceinline__ void put_at(unsigned * p, unsigned rank, unsigned v) {   // to the same place of block `rank`
    asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %0, %1; st.shared::cluster.u32 [a], %2; }"
                 :: "r"(smem_u32(p)), "r"(rank), "r"(v) : "memory");
}

__device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Raises a kernel's limit of shared memory, once per device (`set`: the devices done).
template <class F> cudaError_t allow_smem(F kernel, size_t bytes, int device, unsigned long long & set) {
    if (__atomic_load_n(&set, __ATOMIC_RELAXED) >> device & 1) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) bytes);
    if (e == cudaSuccess) __atomic_fetch_or(&set, 1ull << device, __ATOMIC_RELAXED);
    return e;
}

// Launch of a product behind the quantisation of its rows, which lets it start before it has ended.
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, A &&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

}  // namespace
}  // namespace pk
