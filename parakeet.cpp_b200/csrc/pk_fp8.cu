// pk_fp8.cu -- 8-bit floating point with a scale for each block of 128: quantisation of rows, the values
// back, and the product of quantised rows with a weight matrix quantised in blocks of 128 x 128.
//
// Values are held as e4m3 codes (three bits of fraction, largest magnitude 448, smallest 2^-9) and a scale
// byte B per block (e8m0), value = code * 2^(B - 127). The exponent is the smallest, not below -127, by which
// the block's largest magnitude a comes to at most 448 = 1.75 * 2^8: nothing saturates, and as scales are
// powers of two every scaling is exact and codes are a's own bits rounded once. With f the exponent field of
// a: B = f - 8, one more where a's fraction is above 1.75, so B = max(((bits of a) + 2^21 - 1 >> 23) - 8, 0),
// exactly, subnormals included. (Scales of any value would use the top binade in full, which gains nothing
// where codes are floating point themselves, and could not be applied inside the tensor cores.)

#include "pk_product.cuh"
#include "pk_rows.cuh"

#include <algorithm>
#include <new>

namespace pk {
namespace {

constexpr int kBlock = 128;

__host__ __device__ inline int blocks_of(int K) { return (K + kBlock - 1) / kBlock; }
__host__ __device__ inline int row_bytes(int K) { return (K + 15) / 16 * 16; }   // of a row of codes

// Scales in the layout of the product: atoms of 128 rows by 4 blocks (K = 512), 512 bytes; row r, block b at
// byte (r % 32) * 16 + (r / 32) * 4 + b: a word holds the four blocks of one row. `quads` atoms per 128 rows.
__host__ __device__ inline int quads_of(int K) { return (K + 4 * kBlock - 1) / (4 * kBlock); }
__device__ __forceinline__ size_t scale_at(long long row, int blk, int quads) {
    return ((size_t) (row >> 7) * quads + (blk >> 2)) * 512 + (size_t) ((row & 31) * 16 + ((row >> 5) & 3) * 4 + (blk & 3));
}

// Scale byte of a block from the bits of its largest magnitude; 255 (NaN) for Inf or NaN.
__device__ __forceinline__ unsigned scale_byte(unsigned amax_bits) {
    if (amax_bits >= 0x7F800000u) return 255u;
    const unsigned f = (amax_bits + 0x1FFFFFu) >> 23;
    return f > 8u ? f - 8u : 0u;                     // at most 247
}
// 2^(127 - B), for B up to 247, and 2^(B - 127).
__device__ __forceinline__ float scale_inv(unsigned b) { return __uint_as_float((254u - b) << 23); }
__device__ __forceinline__ float scale_val(unsigned b) {
    return __uint_as_float(b == 255u ? 0x7FC00000u : b == 0u ? 0x00400000u : b << 23);
}

// Four e4m3 codes, nearest, ties to the even one.
__device__ __forceinline__ unsigned cvt_e4m3x4(float a, float b, float c, float d) {
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (unsigned) lo | (unsigned) hi << 16;
}

// Eight codes and their block's scale byte; 2^lg neighbouring lanes hold a block's part of the row.
template <int LG> __device__ __forceinline__ unsigned block_max(unsigned m, int lg) {
#pragma unroll
    for (int o = 0; o < 4; ++o)
        if (LG > o || (LG < 0 && lg > o)) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1 << o));
    return m;
}
template <int LG> __device__ __forceinline__ uint2 quantize8(const Eight<float> & v, int lg, unsigned & sb) {
    sb = scale_byte(block_max<LG>(amax_bits(v), lg));
    if (sb == 255u) return make_uint2(0u, 0u);
    const float s = scale_inv(sb);
    return make_uint2(cvt_e4m3x4(v.e[0] * s, v.e[1] * s, v.e[2] * s, v.e[3] * s),
                      cvt_e4m3x4(v.e[4] * s, v.e[5] * s, v.e[6] * s, v.e[7] * s));
}
template <int LG> __device__ __forceinline__ uint2 quantize8(const Eight<__nv_bfloat16> & v, int lg, unsigned & sb) {
    const unsigned both = word_of(amax_pair<__nv_bfloat162>(v));
    sb = scale_byte(block_max<LG>(max(both << 16, both & 0xFFFF0000u), lg));
    if (sb == 255u) return make_uint2(0u, 0u);
    const float s = scale_inv(sb);
    const unsigned * w = reinterpret_cast<const unsigned *>(v.e);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16) * s;
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u) * s;
    }
    return make_uint2(cvt_e4m3x4(f[0], f[1], f[2], f[3]), cvt_e4m3x4(f[4], f[5], f[6], f[7]));
}
template <int LG> __device__ __forceinline__ uint2 quantize8(const Eight<__half> & v, int lg, unsigned & sb) {
    const __half2 m = amax_pair<__half2>(v);
    sb = scale_byte(block_max<LG>(__float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))), lg));
    if (sb == 255u) return make_uint2(0u, 0u);
    const float s = scale_inv(sb);
    const unsigned * w = reinterpret_cast<const unsigned *>(v.e);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(pair_of<__half2>(w[i]));
        f[2 * i] = x.x * s;
        f[2 * i + 1] = x.y * s;
    }
    return make_uint2(cvt_e4m3x4(f[0], f[1], f[2], f[3]), cvt_e4m3x4(f[4], f[5], f[6], f[7]));
}

// A warp's 256 values of a row, two blocks: eight per lane. Where a row goes on, the next 256 follow in the
// same warp, gridDim.y segments further on; several loads are in flight before the first is used. SHORT, for rows
// of up to 256 values: 2^gs lanes a row, and the next rows instead of the next segments.
// ATOMS: scales in the product's layout. Bound: HBM from f32 (66044 x 1024: 44 us, 270 MB read), instructions from half precision
// (66043 x 1000 bf16: 37 us for 132 MB read and 66 written, of which the codes stay in L2).
template <class T, bool VEC, bool ATOMS, bool SHORT>
__global__ void __launch_bounds__(kQThreads) fp8_quantize_kernel(const T * __restrict__ x, long long rows, int K, long long ldx, int gs,
                                                                 unsigned char * __restrict__ codes,
                                                                 unsigned char * __restrict__ scales) {
    constexpr int UN = sizeof(T) == 4 ? 2 : 4;
    const int lane = threadIdx.x & 31;
    // the product may set itself up while the last blocks work; it waits for all of them before it loads
    if (ATOMS) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int segs = (K + 255) >> 8, nb = blocks_of(K), quads = quads_of(K), ldc = row_bytes(K);
    long long row = (long long) blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5);
    long long stride = (long long) gridDim.x * (kQThreads / 32);
    if constexpr (SHORT) {
        const int sub = lane & ((1 << gs) - 1), blk = sub >> 4;
        row = (row << (5 - gs)) + (lane >> gs);
        stride <<= 5 - gs;
        for (; __any_sync(0xFFFFFFFFu, row < rows); row += UN * stride) {
            Eight<T> v[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const bool on = row + u * stride < rows;
                v[u] = load8<T, VEC>(x + (on ? (row + u * stride) * ldx : 0), on ? sub * 8 : 256, on ? K : 0);
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const long long r = row + u * stride;
                unsigned sb;
                const uint2 q = quantize8<-1>(v[u], min(gs, 4), sb);
                if (r >= rows) continue;
                if (sub * 8 < ldc) *reinterpret_cast<uint2 *>(codes + (size_t) r * ldc + sub * 8) = q;
                if ((sub & 15) == 0 && blk < nb) scales[ATOMS ? scale_at(r, blk, quads) : (size_t) r * nb + blk] = (unsigned char) sb;
            }
        }
    } else {
        for (; row < rows; row += stride) {
            const T * xr = x + row * ldx;
            unsigned char * cr = codes + (size_t) row * ldc + lane * 8;
            for (int s0 = blockIdx.y; s0 < segs; s0 += UN * (int) gridDim.y) {
                Eight<T> v[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int seg = s0 + u * (int) gridDim.y;
                    v[u] = load8<T, VEC>(xr, seg < segs ? seg * 256 + lane * 8 : K, K);
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int seg = s0 + u * (int) gridDim.y;
                    if (seg >= segs) break;
                    const int blk = seg * 2 + (lane >> 4);
                    unsigned sb;
                    const uint2 q = quantize8<4>(v[u], 4, sb);
                    if (seg * 256 + lane * 8 < ldc) *reinterpret_cast<uint2 *>(cr + (size_t) seg * 256) = q;
                    if ((lane & 15) == 0 && blk < nb) scales[ATOMS ? scale_at(row, blk, quads) : (size_t) row * nb + blk] = (unsigned char) sb;
                }
            }
        }
    }
}

// Eight codes' values. A code is exact in f16; code 127 is NaN.
template <class T> __device__ __forceinline__ void codes_to_values(uint2 q, unsigned b, Eight<T> & o) {
    const float s = scale_val(b);
    const unsigned w[2] = {q.x, q.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned h;
        const unsigned short c = (unsigned short) (w[i >> 1] >> (16 * (i & 1)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
        const float2 f = __half22float2(pair_of<__half2>(h));
        o.e[2 * i] = from_f32<T>(f.x * s);
        o.e[2 * i + 1] = from_f32<T>(f.y * s);
    }
}

// The value of each code, eight a lane, rows and lanes as in the quantisation. Bound: HBM, writing y (66043 x 1000 bf16: 35 us).
template <class T, bool VEC, bool SHORT>
__global__ void __launch_bounds__(kQThreads) fp8_dequantize_kernel(const unsigned char * __restrict__ codes,
                                                                   const unsigned char * __restrict__ scales, long long rows,
                                                                   int K, T * __restrict__ y, long long ldy, int gs) {
    constexpr int UN = 4;
    const int lane = threadIdx.x & 31;
    const int segs = (K + 255) >> 8, nb = blocks_of(K), ldc = row_bytes(K);
    long long row = (long long) blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5);
    long long stride = (long long) gridDim.x * (kQThreads / 32);
    if constexpr (SHORT) {
        const int sub = lane & ((1 << gs) - 1);
        row = (row << (5 - gs)) + (lane >> gs);
        stride <<= 5 - gs;
        for (; __any_sync(0xFFFFFFFFu, row < rows); row += UN * stride) {
            uint2 q[UN];
            unsigned char b[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const long long r = row + u * stride;
                const bool in = r < rows && sub * 8 < K;
                q[u] = in ? __ldcs(reinterpret_cast<const uint2 *>(codes + (size_t) r * ldc + sub * 8)) : make_uint2(0u, 0u);
                b[u] = in ? __ldcs(scales + (size_t) r * nb + (sub >> 4)) : (unsigned char) 0;
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const long long r = row + u * stride;
                Eight<T> o;
                codes_to_values(q[u], b[u], o);
                store8<T, VEC>(y + (r < rows ? r * ldy : 0), sub * 8, K, o, sub, 1 << gs, r < rows);
            }
        }
    } else {
        for (; row < rows; row += stride) {
            const unsigned char * cr = codes + (size_t) row * ldc + lane * 8, * sr = scales + (size_t) row * nb + (lane >> 4);
            for (int s0 = blockIdx.y; s0 < segs; s0 += UN * (int) gridDim.y) {
                uint2 q[UN];
                unsigned char b[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int seg = s0 + u * (int) gridDim.y;
                    const bool in = seg < segs && seg * 256 + lane * 8 < K;
                    q[u] = in ? __ldcs(reinterpret_cast<const uint2 *>(cr + (size_t) seg * 256)) : make_uint2(0u, 0u);
                    b[u] = in ? __ldcs(sr + seg * 2) : (unsigned char) 0;
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int seg = s0 + u * (int) gridDim.y;
                    if (seg >= segs) break;
                    Eight<T> o;
                    codes_to_values(q[u], b[u], o);
                    store8<T, VEC>(y + row * ldy, seg * 256 + lane * 8, K, o, lane, 32, true);
                }
            }
        }
    }
}

// Weights, once per layer: a block of threads takes 128 rows x 128 values, a warp every eighth row.
template <class T>
__global__ void __launch_bounds__(256) fp8_weight_kernel(const T * __restrict__ w, int N, int K, unsigned char * __restrict__ codes,
                                                         unsigned char * __restrict__ scales) {
    __shared__ unsigned amax;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blk = blockIdx.x;
    const int c = blk * kBlock + lane * 4, ldc = row_bytes(K);
    const long long n0 = (long long) blockIdx.y * kBlock;
    if (threadIdx.x == 0) amax = 0;
    __syncthreads();
    float v[16][4];
    unsigned m = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long n = n0 + r * 8 + warp;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[r][j] = n < N && c + j < K ? to_f32(w[n * K + c + j]) : 0.0f;
            m = max(m, __float_as_uint(fabsf(v[r][j])));     // infinities and NaN are the largest
        }
    }
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (lane == 0) atomicMax(&amax, m);
    __syncthreads();
    const unsigned sb = scale_byte(amax);
    const float s = scale_inv(sb);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long n = n0 + r * 8 + warp;
        if (n >= N || c >= ldc) continue;
        *reinterpret_cast<unsigned *>(codes + (size_t) n * ldc + c) =
            sb == 255u ? 0u : cvt_e4m3x4(v[r][0] * s, v[r][1] * s, v[r][2] * s, v[r][3] * s);
    }
    if (threadIdx.x < kBlock) scales[scale_at(n0 + threadIdx.x, blk, quads_of(K))] = (unsigned char) sb;
}

// ---- product on the tensor cores ------------------------------------------------
//
// tcgen05.mma kind::mxf8f6f4 with block scales: 32 values of K a product, accumulator in tensor memory. The
// weights are operand A: an output n is a tensor-memory lane, a row m of x a column. So a warp that empties
// 32 lanes of a column has 32 neighbouring values of y's row m, and stores them as they come, whatever y's
// alignment, without shared memory; and few rows of x are few columns, not a tile of 128. A stage is 128 values
// of K, one block and one 128-byte swizzled row: its four products share one scale byte per row, the one that
// the stage's place among four blocks names; scale words are copied to tensor memory every fourth stage.
constexpr int kTN = 128;                                // weight rows of a block
constexpr unsigned kTileBytes = kTN * 128u;
constexpr unsigned kAtom = 512;

// The four products of a stage, by one elected lane (the whole warp runs the loop around it, so that addresses
// and descriptors stay in uniform registers), and before them, where `scales`, the copies of the quad's scales:
// one atom of weights at columns `cs`, XA of x behind it. `shift`: columns to the tile's first row of x in them.
template <bool PAIR>
__device__ __forceinline__ void issue_stage(unsigned d, unsigned w, unsigned x, int bm, unsigned sw, unsigned sx, int xa, unsigned cs,
                                            unsigned shift, int id, bool scales, bool fresh) {
    const unsigned long long dw = umma_desc_sw128(w), dx = umma_desc_sw128(x);
    if (scales) {
        umma_copy_scales<PAIR>(cs, scale_desc(sw));
        umma_copy_scales<PAIR>(cs + 4, scale_desc(sx));
        if (xa > 1) umma_copy_scales<PAIR>(cs + 8, scale_desc(sx + kAtom));
    }
    const unsigned idesc = umma_idesc_mxf8(PAIR ? 2 * kTN : kTN, bm, id);
#pragma unroll
    for (unsigned j = 0; j < 4; ++j)                     // 32 bytes along the swizzled rows
        umma_mxf8<PAIR>(d, dw + 2 * j, dx + 2 * j, idesc, cs, cs + 4 + shift, j > 0 || !fresh ? 1u : 0u);
}

// One value of y.
template <class T> __device__ __forceinline__ void put(T * y, float v) { *y = from_f32<T>(v); }

// ---- many rows: pairs of blocks ---------------------------------------------------
//
// Two blocks of a cluster (cta_group::2) take 256 outputs by `bm` rows: each holds its 128 weight rows and half
// of the rows of x, and the products read the other half from the other SM. At bm = 256 a stage is 32 KB for 512
// cycles of products, at 128 24 KB for 256: the L2 gives an SM some 50 bytes a cycle, so wide tiles pay. Warp 0
// loads, warp 1 of the first block issues, warps from 4 on empty the accumulators, of which there are two. Two of
// 256 columns and the scales' 32 are more than there is: they overlap by 32 columns, which are emptied first.
// Both blocks' loads arrive on the first one's barriers. Measured, replayed from a graph, quantisation included: 8192 x 4096 by
// 8192 bf16 212 us (64 to 192 columns: 540, 295, 242), of which the product 190, 2.9 PFLOP/s, its operands at some 45 bytes a
// cycle and SM from L2; 66044 x 1024 by 640 f32 110 us, the product 65 of them, for 169 MB of y and 411 MB of operands from L2;
// with sixteen epilogue warps in place of eight the same within 1 %.
constexpr int kPStages = 6;
constexpr int kPEpi = 8;                                 // warps of the epilogue
constexpr int kPThreads = 32 * (4 + kPEpi);
constexpr unsigned kPStage = 2 * kTileBytes;
constexpr unsigned kPQuad = 3 * kAtom;
constexpr unsigned kScaleCol = 480;                      // tensor-memory columns of the scales: 12, and 12 from 496 on
struct PairSmem {
    unsigned long long full[kPStages], empty[kPStages], quad_empty[2], acc_full[2], acc_empty[2], done;
    unsigned tmem;
    int err;
    unsigned loads;              // stages that this block's loader issued
    unsigned its_loads;          // the other block's, and whether a wait of its ran out
    int its_err;
};
constexpr size_t kPSmem = 1024 + (size_t) kPStages * kPStage + 2 * kPQuad + sizeof(PairSmem);
static_assert(sharing_ruled_out(kPSmem, kPSmem) && sharing_ruled_out(kPSmem, kClusterSmem), "it takes all of the tensor memory");

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap xsmap, long long M, int K, int bm,
                const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap wsmap, int N,
                const float * __restrict__ bias, T * __restrict__ y, long long ldy, const Waits w) {
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char * ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t) 1023);
    unsigned char * quad = ring + kPStages * kPStage;
    PairSmem & S = *reinterpret_cast<PairSmem *>(quad + 2 * kPQuad);
    const int warp = __shfl_sync(0xFFFFFFFFu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned rank = blockIdx.x & 1u;
    const int nb = blocks_of(K), nt = (N + 2 * kTN - 1) / (2 * kTN), xa = bm > 128 ? 2 : 1;
    const long long tiles = ((M + bm - 1) / bm) * nt, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const unsigned stage_bytes = kTileBytes + (unsigned) bm * 64u, quad_bytes = (unsigned) (1 + xa) * kAtom;
    const bool lap = 2 * bm > (int) kScaleCol;
    const unsigned second = kScaleCol - (unsigned) bm;   // first column of the second accumulator

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPStages; ++s) {
            mbar_init(&S.full[s], 1);                     // used in the first block
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.quad_empty[b], 1);
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 2 * kPEpi);
        }
        mbar_init(&S.done, 1);
        S.err = 0;
        S.loads = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&S.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_meet();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = __shfl_sync(0xFFFFFFFFu, S.tmem, 0);

    if (warp == 0) {
        if (lane == 0) {
            unsigned it = 0, qi = 0;
            bool ok = true;
            asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' codes and scales are there
            for (long long t = w.stall && blockIdx.x == 1 ? tiles : first; t < tiles && ok; t += step) {
                const int tm = (int) (t / nt), tn = (int) (t % nt);
                for (int kb = 0; kb < nb; ++kb, ++it) {
                    const int s = (int) (it % kPStages);
                    const bool fresh = (kb & 3) == 0;
                    if (!mbar_wait(&S.empty[s], ((it / kPStages) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                    if (fresh && !mbar_wait(&S.quad_empty[qi & 1u], ((qi >> 1) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                    unsigned char * a = ring + s * kPStage, * b = a + kTileBytes;
                    // rows past M or N, and their scales, read as zeros
                    const unsigned bar = mbar_at(&S.full[s], 0);
                    if (rank == 0) mbar_expect(&S.full[s], 2u * (stage_bytes + (fresh ? quad_bytes : 0u)));
                    tma_load_2d_pair(a, &wmap, kb * 128, (tn * 2 + (int) rank) * kTN, bar);
                    tma_load_2d_pair(b, &xmap, kb * 128, tm * bm + (int) rank * (bm / 2), bar);
                    if (fresh) {
                        unsigned char * q = quad + (qi & 1u) * kPQuad;
                        tma_load_2d_pair(q, &wsmap, (kb >> 2) * 128, tn * 2 + (int) rank, bar);
                        tma_load_2d_pair(q + kAtom, &xsmap, (kb >> 2) * 128, (tm * bm) >> 7, bar);
                        ++qi;
                    }
                }
            }
            S.loads = it;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            unsigned tile = 0, s = 0, ph = 0, qi = 0;
            bool ok = true;
            for (long long t = first; t < tiles && ok; t += step, ++tile) {
                const unsigned buf = tile & 1u, shift = (unsigned) ((t / nt * bm) & 127) >> 5;
                // two before is empty; where the accumulators overlap, so is the one before in what they share
                const unsigned before = lap ? tile - 1u : tile - 2u;
                if ((lap ? tile > 0 : tile > 1) && !warp_wait<true>(&S.acc_empty[before & 1u], (before >> 1) & 1u, w.ns, &S.err)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < nb; ++kb) {
                    if (!warp_wait<true>(&S.full[s], ph, w.ns, &S.err)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned a = smem_u32(ring) + s * kPStage, q = smem_u32(quad) + (qi & 1u) * kPQuad;
                    const bool last = (kb & 3) == 3 || kb == nb - 1;
                    if (elect_one()) {
                        issue_stage<true>(tmem + (buf ? second : 0u), a, a + kTileBytes, bm, q, q + kAtom, xa,
                                          tmem + kScaleCol + (qi & 1u) * 16u, shift, kb & 3, (kb & 3) == 0, kb == 0);
                        umma_commit_pair(&S.empty[s]);
                        if (last) umma_commit_pair(&S.quad_empty[qi & 1u]);
                        if (kb == nb - 1) umma_commit_pair(&S.acc_full[buf]);
                    }
                    __syncwarp();
                    if (last) ++qi;
                    if (++s == kPStages) { s = 0; ph ^= 1u; }
                }
            }
            // no product in flight when the blocks end
            if (elect_one()) umma_commit_pair(&S.done);
            mbar_drain(&S.done, 0u);
        }
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2, chunks = bm / 32;
        unsigned tile = 0;
        for (long long t = first; t < tiles; t += step, ++tile) {
            const unsigned buf = tile & 1u;
            const long long n = ((t % nt) * 2 + rank) * kTN + q * 32 + lane, m0 = t / nt * bm;
            const float bv = bias && n < N ? __ldg(bias + n) : 0.0f;
            if (!warp_wait(&S.acc_full[buf], (tile >> 1) & 1u, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned acc = tmem + (buf ? second : 0u) + ((unsigned) (q * 32) << 16);
            for (int i = half; i < chunks; i += 2) {
                const int c = (buf ? i : chunks - 1 - i) * 32;   // what the accumulators share comes first
                unsigned v[32];
                tmem_load32(acc + c, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (lap ? i == half : i + 2 >= chunks) {         // what the next products wait for is read
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    if (lane == 0) mbar_arrive_at_relaxed(&S.acc_empty[buf], 0);
                }
                if (n < N) {
                    T * o = y + (m0 + c) * ldy + n;
                    const int rows = (int) max(0LL, min(32LL, M - m0 - c));
                    if (rows == 32) {
#pragma unroll
                        for (int r = 0; r < 32; ++r, o += ldy) put(o, __uint_as_float(v[r]) + bv);
                    } else {
#pragma unroll
                        for (int r = 0; r < 32; ++r, o += ldy)
                            if (r < rows) put(o, __uint_as_float(v[r]) + bv);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        put_at(&S.its_loads, rank ^ 1u, S.loads);
        put_at(reinterpret_cast<unsigned *>(&S.its_err), rank ^ 1u, (unsigned) S.err);
    }
    cluster_meet();                                       // the other's memory and barriers are used no more
    if (threadIdx.x == 0) mbar_drain(&S.done, 0u);        // the second block's too: its arrival comes from the first's products
    // Where no wait ran out every stage was multiplied, so its loads have come. Otherwise one block may have issued
    // stages that the other has not (as many as there are, at most: a stage is free again once both blocks' was
    // multiplied). The first block, whose barriers count both blocks' bytes, sets the counts right and waits for
    // what was issued.
    if (S.err | S.its_err) {
        if (rank == 0 && threadIdx.x == 0) {
            const unsigned least = min(S.loads, S.its_loads), most = max(S.loads, S.its_loads);
            for (unsigned j = least; j < most; ++j) {
                const unsigned bytes = stage_bytes + ((j % (unsigned) nb & 3u) == 0u ? quad_bytes : 0u);
                if (S.loads < most) mbar_expect(&S.full[j % kPStages], bytes);
                else mbar_complete(&S.full[j % kPStages], bytes);
            }
            for (unsigned j = most > kPStages ? most - kPStages : 0; j < most; ++j) mbar_drain(&S.full[j % kPStages], (j / kPStages) & 1u);
        }
        cluster_meet();
    }
    if (warp == 2) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
    if (threadIdx.x == 0 && S.err != 0) atomicExch_system(w.err, 1);
}

// ---- few rows: K over the blocks of a cluster --------------------------------------
//
// With few rows the weights are nearly all of the bytes and there are fewer tiles than SMs, so the S blocks of a
// cluster each take a stretch of K of one tile of 128 outputs by `bm` rows, hand each other their sums through
// distributed shared memory, and add them in the blocks' order, each for its share of the rows. FUSED: every
// block quantises its stretch of the rows for itself, into the products' layout in its shared memory, while its
// first weights are on their way: one launch. Otherwise codes and scales come from the row kernel.
constexpr int kSWarps = 12;                              // warps that quantise; the first four empty the accumulator
constexpr int kSThreads = 32 * (4 + kSWarps);
constexpr int kSMaxStages = 8;
constexpr unsigned kSCols = 256;                         // tensor memory: accumulator of up to 128, scales from 128 on
struct SplitSmem {
    unsigned long long full[kSMaxStages], empty[kSMaxStages], quad_empty[2], x_full, acc_full, done;
    unsigned tmem;
    int err;
};

struct SplitPlan {
    int bm, split, stages;
    size_t smem;
};

template <class TX, class TY, bool VEC, bool FUSED>
__global__ void __launch_bounds__(kSThreads)
fp8_split_kernel(const TX * __restrict__ x, long long ldx, long long M, int K, const __grid_constant__ CUtensorMap xmap,
                 const unsigned char * __restrict__ xscale, const __grid_constant__ CUtensorMap wmap,
                 const unsigned char * __restrict__ wscale, int N, const float * __restrict__ bias, TY * __restrict__ y, long long ldy,
                 const SplitPlan p, const Waits w) {
    extern __shared__ __align__(1024) unsigned char raw[];
    const int warp = __shfl_sync(0xFFFFFFFFu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = (int) (blockIdx.x % (unsigned) p.split), nb = blocks_of(K), quads = quads_of(K);
    const long long tile = blockIdx.x / (unsigned) p.split, mt = (M + p.bm - 1) / p.bm;
    const int tn = (int) (tile / mt);
    const long long m0 = tile % mt * p.bm;
    const int kb0 = (int) ((long long) nb * rank / p.split), kb1 = (int) ((long long) nb * (rank + 1) / p.split);
    const int most = (nb + p.split - 1) / p.split;       // blocks of K at most
    const unsigned xbytes = (unsigned) p.bm * 128u, stage = kTileBytes + (FUSED ? 0u : xbytes);
    unsigned char * ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t) 1023);
    unsigned char * xs = ring + p.stages * stage;        // FUSED: the rows' codes, then all their scales
    unsigned char * xss = xs + (FUSED ? (size_t) most * xbytes : 0);
    unsigned char * quad = xss + (FUSED ? (size_t) (most / 4 + 2) * kAtom : 0);
    float * sums = reinterpret_cast<float *>(quad + 4 * kAtom);
    SplitSmem & S = *reinterpret_cast<SplitSmem *>(sums + (p.split > 1 ? p.bm * kTN : 0));

    if (threadIdx.x == 0) {
        for (int s = 0; s < kSMaxStages; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        mbar_init(&S.quad_empty[0], 1);
        mbar_init(&S.quad_empty[1], 1);
        mbar_init(&S.x_full, kSWarps);
        mbar_init(&S.acc_full, 1);
        mbar_init(&S.done, 1);
        S.err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&S.tmem)), "r"(kSCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = __shfl_sync(0xFFFFFFFFu, S.tmem, 0);

    if (warp == 0) {
        if (lane == 0) {
            // weights do not wait for the row kernel; rows do. `behind` stages have their weights under way only.
            unsigned it = 0, qi = 0, behind = 0;
            bool ok = true;
            auto rows_of = [&](int kb, unsigned s) {
                if constexpr (!FUSED) tma_load_2d(ring + s * stage + kTileBytes, &xmap, kb * 128, (int) m0, &S.full[s]);
            };
            auto row_scales = [&](int kb, unsigned s, unsigned slot) {
                if constexpr (!FUSED)
                    bulk_load(quad + slot * 2 * kAtom + kAtom, xscale + ((size_t) (m0 >> 7) * quads + (kb >> 2)) * kAtom, kAtom, &S.full[s]);
            };
            const int end = w.stall && blockIdx.x == 0 ? kb0 : kb1;
            for (int kb = kb0; kb < end; ++kb, ++it) {
                const unsigned s = it % (unsigned) p.stages;
                const bool fresh = kb == kb0 || (kb & 3) == 0;
                if (!FUSED && (it == (unsigned) p.stages || (fresh && qi == 2)) && it == behind) {
                    // the ring, or the scales' two places, are full: now the rows
                    asm volatile("griddepcontrol.wait;" ::: "memory");
                    unsigned k2 = 0;
                    for (unsigned j = 0; j < behind; ++j) {
                        const int kk = kb0 + (int) j;
                        rows_of(kk, j);
                        if (j == 0 || (kk & 3) == 0) row_scales(kk, j, k2++);
                    }
                    behind = 0;
                }
                const bool ahead = !FUSED && it == behind;
                if (!mbar_wait(&S.empty[s], ((it / (unsigned) p.stages) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                if (fresh && !mbar_wait(&S.quad_empty[qi & 1u], ((qi >> 1) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                mbar_expect(&S.full[s], stage + (fresh ? (FUSED ? kAtom : 2 * kAtom) : 0u));
                tma_load_2d(ring + s * stage, &wmap, kb * 128, tn * kTN, &S.full[s]);
                if (fresh) bulk_load(quad + (qi & 1u) * 2 * kAtom, wscale + ((size_t) tn * quads + (kb >> 2)) * kAtom, kAtom, &S.full[s]);
                if (ahead) {
                    ++behind;
                } else {
                    rows_of(kb, s);
                    if (fresh) row_scales(kb, s, qi & 1u);
                }
                if (fresh) ++qi;
            }
            if (!FUSED && behind == it && it > 0) {      // the whole stretch fits the ring
                asm volatile("griddepcontrol.wait;" ::: "memory");
                unsigned k2 = 0;
                for (unsigned j = 0; j < behind; ++j) {
                    const int kk = kb0 + (int) j;
                    rows_of(kk, j);
                    if (j == 0 || (kk & 3) == 0) row_scales(kk, j, k2++);
                }
            }
            (void) ok;
            // nothing in flight when the block ends, however the others ended
            for (unsigned j = it > (unsigned) p.stages ? it - (unsigned) p.stages : 0; j < it; ++j)
                mbar_drain(&S.full[j % (unsigned) p.stages], (j / (unsigned) p.stages) & 1u);
        }
    } else if (warp == 1) {
        unsigned s = 0, ph = 0, qi = 0;
        const unsigned shift = (unsigned) (m0 & 127) >> 5;
        bool ok = !FUSED || warp_wait(&S.x_full, 0u, w.ns, &S.err);
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
            if (!warp_wait(&S.full[s], ph, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned a = smem_u32(ring) + s * stage, q = smem_u32(quad) + (qi & 1u) * 2 * kAtom;
            const bool fresh = kb == kb0 || (kb & 3) == 0, last = (kb & 3) == 3 || kb == kb1 - 1;
            if (elect_one()) {
                const unsigned xa = FUSED ? smem_u32(xs) + (unsigned) (kb - kb0) * xbytes : a + kTileBytes;
                const unsigned sx = FUSED ? smem_u32(xss) + (unsigned) ((kb >> 2) - (kb0 >> 2)) * kAtom : q + kAtom;
                issue_stage<false>(tmem, a, xa, p.bm, q, sx, 1, tmem + 128 + (qi & 1u) * 8u, shift, kb & 3, fresh, kb == kb0);
                umma_commit(&S.empty[s]);
                if (last) umma_commit(&S.quad_empty[qi & 1u]);
                if (kb == kb1 - 1) umma_commit(&S.acc_full);
            }
            __syncwarp();
            if (last) ++qi;
            if (++s == (unsigned) p.stages) { s = 0; ph ^= 1u; }
        }
        if (elect_one()) umma_commit(&S.done);           // no product in flight either
        mbar_drain(&S.done, 0u);
    } else if (FUSED && warp >= 4) {
        // the rows past M keep what is there: their columns of the accumulator are not stored
        const int c0 = kb0 * kBlock, end = min(K, kb1 * kBlock), segs = (kb1 - kb0 + 1) >> 1;
        for (int i = warp - 4; i < (int) M * segs; i += kSWarps) {
            const int r = i / segs, seg = i - r * segs, kb = seg * 2 + (lane >> 4);
            unsigned sb;
            const uint2 q = quantize8<4>(load8<TX, VEC>(x + r * ldx, c0 + seg * 256 + lane * 8, end), 4, sb);
            if (kb >= kb1 - kb0) continue;
            // 128-byte swizzle: 16-byte piece c of row r at piece c ^ (r % 8)
            *reinterpret_cast<uint2 *>(xs + (unsigned) kb * xbytes + (unsigned) r * 128u + ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8) = q;
            if ((lane & 15) == 0)
                xss[(((kb0 + kb) >> 2) - (kb0 >> 2)) * kAtom + (r & 31) * 16 + (r >> 5) * 4 + ((kb0 + kb) & 3)] = (unsigned char) sb;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.x_full);
    }
    if (p.split > 1) cluster_meet();                     // every block of the cluster runs: their memory may be written
    const int rows = (int) min((long long) p.bm, M - m0);
    if (warp >= 4 && warp < 8) {
        const int q = warp & 3;
        const long long n = (long long) tn * kTN + q * 32 + lane;
        if (warp_wait(&S.acc_full, 0u, w.ns, &S.err)) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned acc = tmem + ((unsigned) (q * 32) << 16);
            const float bv = bias && n < N ? __ldg(bias + n) : 0.0f;
            const int lg = 31 - __clz(p.bm / p.split);   // of the rows that a block of the cluster adds up, a power of two
            for (int c = 0; c < rows; c += 16) {
                unsigned v[16];
                tmem_load16(acc + c, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (p.split == 1) {
                    if (n < N) {
                        TY * o = y + (m0 + c) * ldy + n;
#pragma unroll
                        for (int r = 0; r < 16; ++r, o += ldy)
                            if (c + r < rows) put(o, __uint_as_float(v[r]) + bv);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (c + r >= rows) break;
                        const int owner = (c + r) >> lg, place = (rank << lg) + c + r - (owner << lg);
                        unsigned at;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(sums + place * kTN + q * 32 + lane)), "r"(owner));
                        asm volatile("st.shared::cluster.u32 [%0], %1;" :: "r"(at), "r"(v[r]) : "memory");
                    }
                }
            }
        }
    }
    if (p.split > 1) {
        cluster_meet();                                  // all sums are there
        const int each = p.bm / p.split;
        for (int i = threadIdx.x; i < each * kTN; i += kSThreads) {
            const int r = rank * each + i / kTN;
            const long long n = (long long) tn * kTN + i % kTN;
            if (r >= rows || n >= N) continue;
            float v = sums[i];
            for (int b = 1; b < p.split; ++b) v += sums[(size_t) b * each * kTN + i];
            put(y + (m0 + r) * ldy + n, v + (bias ? __ldg(bias + n) : 0.0f));
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 2) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(kSCols) : "memory");
    }
    if (threadIdx.x == 0 && S.err != 0) atomicExch_system(w.err, 1);
}

template <bool ATOMS>
cudaError_t launch_quantize(const void * x, int type, long long rows, int K, long long ldx, unsigned char * codes,
                            unsigned char * scales, cudaStream_t s) {
    if (rows <= 0) return cudaSuccess;
    const bool vec = aligned_to(x, 16) && (ldx * elem_size(type)) % 16 == 0;
    const int gs = row_lanes(K);
    const dim3 g = row_blocks(rows, K);
#define PK_Q2(T, V, S) launch_on(fp8_quantize_kernel<T, V, ATOMS, S>, g, kQThreads, 0, s, static_cast<const T *>(x), rows, K, ldx, gs, codes, scales)
#define PK_Q(T) \
    (K <= 256 ? (vec ? PK_Q2(T, true, true) : PK_Q2(T, false, true)) : vec ? PK_Q2(T, true, false) : PK_Q2(T, false, false))
    return type == PK_GGML_F32 ? PK_Q(float) : type == PK_GGML_F16 ? PK_Q(__half) : PK_Q(__nv_bfloat16);
#undef PK_Q
#undef PK_Q2
}

constexpr int64_t kMaxDim = 1 << 20;        // K, N
constexpr int64_t kMaxRows = 0x7FFFFFFF;
constexpr size_t kSmemCap = 227 * 1024;

}  // namespace
}  // namespace pk

struct pk_fp8 : pk::LayerWaits {
    int device = 0;
    int N = 0, K = 0, nb = 0, quads = 0;
    unsigned char * codes = nullptr;    // [N][row_bytes(K)]; owns the memory of all three
    unsigned char * scales = nullptr;   // atoms, every row of a block with the same byte
    float * bias = nullptr;             // or null
    alignas(64) CUtensorMap map;        // codes in boxes of 128 rows and 128 bytes
    alignas(64) CUtensorMap smap;       // scales in boxes of one atom
};

namespace pk {
namespace {

// Scale atoms as rows of words, one row for 128 rows of values; a box is one quad's atoms of `rows` such rows.
cudaError_t map_scales(CUtensorMap * map, const unsigned char * scales, long long atom_rows, int quads, int rows) {
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, scales, atom_rows, (long long) quads * 128, rows, 128, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct Call {
    const pk_fp8 * w;
    Waits waits;
    const void * x;
    long long ldx, M;
    void * y;
    long long ldy;
    cudaStream_t s;
};

// The cluster kernel's shared memory beside its ring, and whether the rest holds at least two stages.
bool fit_split(SplitPlan & p, int K, bool fused) {
    const int nb = blocks_of(K), most = (nb + p.split - 1) / p.split;
    const size_t x = (size_t) p.bm * 128, stage = kTileBytes + (fused ? 0 : x);
    const size_t rest = 1024 + 4 * kAtom + (fused ? most * x + (size_t) (most / 4 + 2) * kAtom : 0) +
                        (p.split > 1 ? (size_t) p.bm * kTN * 4 : 0) + sizeof(SplitSmem);
    if (rest + std::min(most, 2) * stage > kSmemCap) return false;
    p.stages = (int) std::min<size_t>({(size_t) kSMaxStages, (size_t) most, (kSmemCap - rest) / stage});
    p.smem = rest + p.stages * stage;
    if (p.split > 1) p.smem = std::max(p.smem, kClusterSmem);    // with half of the tensor memory, see there
    return true;
}

// The most blocks of K a tile is parted over: up to eight, while there are SMs for all tiles' blocks. (Sixteen clusters of eight
// do not run at once all the same: see plan_split.)
int split_of(long long tiles, int nb) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= 148 && s * 2 <= nb) s *= 2;
    return s;
}

// Rows that the cluster kernel quantises itself, none of its blocks more than these values. Replayed from a graph, this way and in
// two launches, the second in pairs of blocks: a row of 640 by 8198 6.5 us and 6.9, of 1024 by 1024 5.7 and 7.5, of 2048 by 8198
// 9.0 and 9.8; 16 rows of 1024 by 1024 6.7 and 7.7, of 640 by 8198 8.0 and 7.0; 32 of 2048 by 1024 8.0 and 9.8, of 1024 by 1024 7.8
// and 7.6, of 640 by 8198 10.2 and 7.2. So it is sooner for few rows and for long ones; from some 16 rows on of a wide layer it
// is not, from a program's calls either (one row of 640 by 8198 8.2 us and 8.3, 32 12.3 and 8.3).
constexpr long long kFusedRows = 32, kFusedValues = 32768;
bool plan_fused(const pk_fp8 * w, long long M, SplitPlan & p) {
    if (M > kFusedRows) return false;
    p.bm = M <= 16 ? 16 : 32;
    p.split = split_of((w->N + kTN - 1) / kTN, w->nb);
    if (M * std::min(w->K, (w->nb + p.split - 1) / p.split * kBlock) > kFusedValues) return false;
    return fit_split(p, w->K, true);
}

// Few tiles and a long K, codes from the row kernel. Replayed from a graph, this way and in pairs of blocks, 64 rows: by 1024
// outputs, K of 1024 9.4 us and 7.8, 2048 10.0 and 10.0, 2560 10.7 and 11.2, 3328 11.4 and 12.8, 4096 11.5 and 14.3, 8192 13.9 and
// 23.1; by 4096, K of 2560 12.3 and 11.4, 3328 13.6 and 12.9, 4096 14.3 and 14.5, 8192 17.9 and 23.4. 128 rows by 1024: 2560 13.3 and
// 11.3, 3328 14.1 and 13.1, 4096 14.1 and 14.5. By 2048 outputs, which ask for 16 clusters of eight blocks, not all of them run at
// once and pairs are sooner (K of 4096: 20.1 and 14.3), up to K of some 8192 (25.3 and 23.2).
bool plan_split(const pk_fp8 * w, long long M, SplitPlan & p) {
    const long long nt = (w->N + kTN - 1) / kTN;
    if (M > 128 || w->nb < 26) return false;
    p.bm = M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const long long tiles = nt * ((M + p.bm - 1) / p.bm);
    if (tiles > 148) return false;
    p.split = split_of(tiles, w->nb);
    return fit_split(p, w->K, false);
}

template <class TX, class TY, bool VEC, bool FUSED>
cudaError_t launch_split_as(const Call & c, const SplitPlan & p, const CUtensorMap & xmap, const unsigned char * xs) {
    auto kernel = fp8_split_kernel<TX, TY, VEC, FUSED>;
    static unsigned long long set;
    const cudaError_t e = allow_smem(kernel, kSmemCap, c.w->device, set);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long) ((c.w->N + kTN - 1) / kTN) * ((c.M + p.bm - 1) / p.bm);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    cfg.gridDim = dim3((unsigned) (tiles * p.split));
    cfg.blockDim = dim3(kSThreads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = c.s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned) p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = FUSED ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<const TX *>(c.x), c.ldx, c.M, c.w->K, xmap, xs, c.w->map, (const unsigned char *) c.w->scales, c.w->N,
                              (const float *) c.w->bias, static_cast<TY *>(c.y), c.ldy, p, c.waits);
}

template <class TX, class TY> cudaError_t launch_fused_xy(const Call & c, const SplitPlan & p) {
    CUtensorMap none{};
    return aligned_to(c.x, 16) && c.ldx * sizeof(TX) % 16 == 0 ? launch_split_as<TX, TY, true, true>(c, p, none, nullptr)
                                                              : launch_split_as<TX, TY, false, true>(c, p, none, nullptr);
}
template <class TX> cudaError_t launch_fused(const Call & c, const SplitPlan & p, int y_type) {
    return y_type == PK_GGML_F32 ? launch_fused_xy<TX, float>(c, p)
           : y_type == PK_GGML_F16 ? launch_fused_xy<TX, __half>(c, p) : launch_fused_xy<TX, __nv_bfloat16>(c, p);
}

// Rows of a pair's tile: fewest rounds of tiles over the pairs, a round costed by the bytes that a block loads.
int pair_rows(long long M, int N) {
    int best = 256;
    long long least = INT64_MAX;
    for (const int bm : {256, 192, 128, 64}) {
        const long long tiles = (M + bm - 1) / bm * ((N + 2 * kTN - 1) / (2 * kTN)), cost = (tiles + 73) / 74 * (kTN + bm / 2);
        if (cost < least) { least = cost; best = bm; }
    }
    return best;
}

template <class T> cudaError_t launch_product(const Call & c, const unsigned char * xc, const unsigned char * xs) {
    alignas(64) CUtensorMap xmap, xsmap;
    SplitPlan p;
    const bool split = plan_split(c.w, c.M, p);
    const int bm = split ? p.bm : pair_rows(c.M, c.w->N);
    cudaError_t e = encode_2d(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xc, c.M, row_bytes(c.w->K), split ? bm : bm / 2, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (e != cudaSuccess) return e;
    if (split) return launch_split_as<float, T, true, false>(c, p, xmap, xs);
    e = map_scales(&xsmap, xs, (c.M + 127) / 128, c.w->quads, bm > 128 ? 2 : 1);
    if (e != cudaSuccess) return e;
    auto kernel = fp8_pair_kernel<T>;
    static unsigned long long set;
    e = allow_smem(kernel, kPSmem, c.w->device, set);
    if (e != cudaSuccess) return e;
    const long long tiles = (c.M + bm - 1) / bm * ((c.w->N + 2 * kTN - 1) / (2 * kTN));
    return launch_after(kernel, (unsigned) (2 * std::min<long long>(tiles, 74)), kPThreads, kPSmem, c.s, xmap, xsmap, c.M, c.w->K, bm, c.w->map,
                        c.w->smap, c.w->N, (const float *) c.w->bias, static_cast<T *>(c.y), c.ldy, c.waits);
}

}  // namespace

void fp8_dims(const pk_fp8 * w, int * device, int * N, int * K) {
    if (device) *device = w->device;
    if (N) *N = w->N;
    if (K) *K = w->K;
}

}  // namespace pk

namespace {

using namespace pk;

// What quantize and dequantize refuse alike.
pk_status check_rows(const char * fn, int device, int type, int64_t rows, int64_t cols, int64_t stride, const void * a, int a_align,
                     const void * codes, const void * scales) {
    if (elem_size(type) == 0) return op_fail(PK_ERR_INVALID, fn, "element type must be F32, F16 or BF16");
    if (rows < 0 || rows > kMaxRows || cols < 1 || cols > kMaxDim || stride < cols || stride > (INT64_MAX >> 34))
        return op_fail(PK_ERR_INVALID, fn, "rows must be in [0, 2^31), cols in [1, 2^20], row_stride >= cols");
    if (rows > 0 && (!a || !codes || !scales)) return op_fail(PK_ERR_INVALID, fn, "null pointer");
    if (!aligned_to(a, (size_t) a_align)) return op_fail(PK_ERR_INVALID, fn, "rows must be aligned to their element");
    if (!aligned_to(codes, 8)) return op_fail(PK_ERR_INVALID, fn, "codes must be 8-byte aligned");
    if (!device_ok(device)) return op_fail(PK_ERR_NO_DEVICE, fn, "no sm_100 device with that index");
    return PK_OK;
}

size_t ws_codes(const pk_fp8 * w, int64_t rows) { return ((size_t) rows * row_bytes(w->K) + 255) / 256 * 256; }

}  // namespace

extern "C" PK_API pk_status pk_fp8_quantize(int device, const void * x, int32_t x_type, int64_t rows, int64_t cols,
                                            int64_t row_stride, uint8_t * codes, uint8_t * scales, void * stream) {
    const char * fn = "pk_fp8_quantize";
    const pk_status st = check_rows(fn, device, x_type, rows, cols, row_stride, x, elem_size(x_type), codes, scales);
    if (st != PK_OK || rows == 0) return st;
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    const cudaError_t e = launch_quantize<false>(x, x_type, rows, (int) cols, row_stride, codes, scales, (cudaStream_t) stream);
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}

extern "C" PK_API pk_status pk_fp8_dequantize(int device, const uint8_t * codes, const uint8_t * scales, int64_t rows, int64_t cols,
                                              void * y, int32_t y_type, int64_t row_stride, void * stream) {
    const char * fn = "pk_fp8_dequantize";
    const pk_status st = check_rows(fn, device, y_type, rows, cols, row_stride, y, elem_size(y_type), codes, scales);
    if (st != PK_OK || rows == 0) return st;
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    const bool vec = aligned_to(y, 16) && (row_stride * elem_size(y_type)) % 16 == 0;
    const dim3 g = row_blocks(rows, cols);
    const int gs = row_lanes(cols);
    cudaStream_t s = (cudaStream_t) stream;
#define PK_D2(T, V, S) launch_on(fp8_dequantize_kernel<T, V, S>, g, kQThreads, 0, s, codes, scales, rows, (int) cols, static_cast<T *>(y), row_stride, gs)
#define PK_D(T) \
    (cols <= 256 ? (vec ? PK_D2(T, true, true) : PK_D2(T, false, true)) : vec ? PK_D2(T, true, false) : PK_D2(T, false, false))
    const cudaError_t e = y_type == PK_GGML_F32 ? PK_D(float) : y_type == PK_GGML_F16 ? PK_D(__half) : PK_D(__nv_bfloat16);
#undef PK_D
#undef PK_D2
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}

extern "C" PK_API void pk_fp8_destroy(pk_fp8 * w) {
    if (!w) return;
    DeviceScope dev(w->device);
    cudaDeviceSynchronize();
    cudaFree(w->codes);
    if (w->err) give_error_word(w->err);
    delete w;
}

extern "C" PK_API pk_status pk_fp8_create(int device, const pk_tensor * weight, int32_t on_device, const float * bias, pk_fp8 ** out) {
    const char * fn = "pk_fp8_create";
    if (!out) return op_fail(PK_ERR_INVALID, fn, "null output");
    *out = nullptr;
    if (!weight || !weight->data) return op_fail(PK_ERR_INVALID, fn, "null weight");
    const int64_t K = weight->ne0, N = weight->ne1;
    if (K < 1 || K > kMaxDim || N < 1 || N > kMaxDim) return op_fail(PK_ERR_MODEL, fn, "weight dimensions must be in [1, 2^20]");
    const int type = weight->type;
    const bool q8 = type == PK_GGML_Q8_0;
    if (!q8 && elem_size(type) == 0) return op_fail(PK_ERR_MODEL, fn, "weight type must be F32, F16, BF16 or Q8_0");
    if (q8 && K % 32 != 0) return op_fail(PK_ERR_MODEL, fn, "ne0 of a block type must be a multiple of 32");
    const uint64_t want = q8 ? (uint64_t) N * (K / 32) * 34 : (uint64_t) N * K * elem_size(type);
    if (weight->nbytes != want) return op_fail(PK_ERR_MODEL, fn, "weight nbytes does not match its type and shape");
    if (on_device && (!aligned_to(weight->data, q8 ? 2 : (size_t) elem_size(type)) || (bias && !aligned_to(bias, 4))))
        return op_fail(PK_ERR_INVALID, fn, "device weight and bias must be aligned to their element");
    if (!device_ok(device)) return op_fail(PK_ERR_NO_DEVICE, fn, "no sm_100 device with that index");
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    pk_fp8 * w = new (std::nothrow) pk_fp8();
    if (!w) return op_fail(PK_ERR_OOM, fn, "host memory");
    w->device = device;
    w->N = (int) N;
    w->K = (int) K;
    w->nb = blocks_of((int) K);
    w->quads = quads_of((int) K);
    const int64_t nt = (N + kTN - 1) / kTN;
    const size_t code_bytes = ((size_t) N * row_bytes((int) K) + 511) / 512 * 512, scale_bytes = (size_t) nt * w->quads * kAtom;
    void * raw = nullptr;    // a host weight's copy
    void * f32 = nullptr;    // q8_0 blocks dequantised
    const cudaStream_t s = cudaStreamPerThread;
    cudaError_t e = on_device ? cudaDeviceSynchronize() : cudaSuccess;
    if (e == cudaSuccess) e = cudaMalloc(&w->codes, code_bytes + scale_bytes + (bias ? (size_t) N * 4 : 0));
    if (e == cudaSuccess) {
        w->scales = w->codes + code_bytes;
        if (bias) w->bias = reinterpret_cast<float *>(w->scales + scale_bytes);
        e = cudaMemsetAsync(w->scales, 0, scale_bytes, s);
    }
    const void * src = weight->data;
    if (e == cudaSuccess && !on_device) {
        e = cudaMalloc(&raw, want);
        if (e == cudaSuccess) e = cudaMemcpyAsync(raw, weight->data, want, cudaMemcpyHostToDevice, s);
        src = raw;
    }
    if (e == cudaSuccess && q8) {
        e = cudaMalloc(&f32, (size_t) N * K * 4);
        if (e == cudaSuccess) e = launch_dequant(src, type, K, N, static_cast<float *>(f32), s);
        src = f32;
    }
    if (e == cudaSuccess) {
        const dim3 g((unsigned) w->nb, (unsigned) nt);
#define PK_W(T) launch_on(fp8_weight_kernel<T>, g, 256, 0, s, static_cast<const T *>(src), w->N, w->K, w->codes, w->scales)
        e = q8 || type == PK_GGML_F32 ? PK_W(float) : type == PK_GGML_F16 ? PK_W(__half) : PK_W(__nv_bfloat16);
#undef PK_W
    }
    if (e == cudaSuccess && bias)
        e = cudaMemcpyAsync(w->bias, bias, (size_t) N * 4, on_device ? cudaMemcpyDeviceToDevice : cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) w->err = take_error_word(e);
    if (e == cudaSuccess) e = cudaHostGetDevicePointer(reinterpret_cast<void **>(&w->err_dev), w->err, 0);
    if (e == cudaSuccess)
        e = encode_2d(&w->map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w->codes, N, row_bytes((int) K), kTN, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (e == cudaSuccess) e = map_scales(&w->smap, w->scales, nt, w->quads, 1);
    const cudaError_t e2 = cudaStreamSynchronize(s);
    if (e == cudaSuccess) e = e2;
    cudaFree(raw);
    cudaFree(f32);
    if (e != cudaSuccess) {
        pk_fp8_destroy(w);
        return op_cuda_fail(e, fn);
    }
    *out = w;
    return PK_OK;
}

extern "C" PK_API pk_status pk_fp8_set_option(pk_fp8 * w, int32_t option, int64_t value) {
    const char * fn = "pk_fp8_set_option";
    return w ? set_wait_option(*w, fn, option, value) : op_fail(PK_ERR_INVALID, fn, "null layer");
}

extern "C" PK_API int64_t pk_fp8_workspace(const pk_fp8 * w, int64_t rows) {
    if (!w) return -1;
    SplitPlan p;
    if (rows <= 0 || plan_fused(w, rows, p)) return 0;
    return (int64_t) (ws_codes(w, rows) + (size_t) ((rows + 127) / 128) * w->quads * kAtom);
}

// A product that reports to the error word `err_dev` (the device's address of it); null: to the layer's, whose
// unreported timeouts it then tells of instead of running.
pk_status pk::fp8_linear(pk_fp8 * w, const char * fn, const void * x, int32_t x_type, int64_t rows, int64_t x_stride, void * y,
                         int32_t y_type, int64_t y_stride, void * workspace, int64_t workspace_bytes, void * stream, int * err_dev) {
    if (!w) return op_fail(PK_ERR_INVALID, fn, "null layer");
    if (elem_size(x_type) == 0 || elem_size(y_type) == 0) return op_fail(PK_ERR_INVALID, fn, "element types must be F32, F16 or BF16");
    if (rows < 0 || rows > kMaxRows) return op_fail(PK_ERR_INVALID, fn, "rows must be in [0, 2^31)");
    if (x_stride < w->K || y_stride < w->N || x_stride > (INT64_MAX >> 34) || y_stride > (INT64_MAX >> 34))
        return op_fail(PK_ERR_INVALID, fn, "x_stride must be at least K and y_stride at least N");
    if (rows == 0) return PK_OK;
    const int64_t need = pk_fp8_workspace(w, rows);
    if (!x || !y || (need > 0 && !workspace)) return op_fail(PK_ERR_INVALID, fn, "null pointer");
    if (!aligned_to(x, (size_t) elem_size(x_type)) || !aligned_to(y, (size_t) elem_size(y_type)))
        return op_fail(PK_ERR_INVALID, fn, "x and y must be aligned to their element");
    if (!aligned_to(workspace, 256)) return op_fail(PK_ERR_INVALID, fn, "workspace must be 256-byte aligned");
    if (workspace_bytes < need)
        return op_fail(PK_ERR_INVALID, fn, "workspace_bytes is below pk_fp8_workspace(w, rows)");
    if (!err_dev) {
        notice_timeout(*w);
        if (__atomic_exchange_n(&w->unreported, 0, __ATOMIC_ACQ_REL))
            return op_fail(PK_ERR_TIMEOUT, fn, "a device-side wait of an earlier call ran out; this call did not run");
        err_dev = w->err_dev;
    }
    DeviceScope dev(w->device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    cudaStream_t s = (cudaStream_t) stream;
    unsigned char * xc = static_cast<unsigned char *>(workspace);
    unsigned char * xs = xc + ws_codes(w, rows);
    const Waits waits{__atomic_load_n(&w->wait_ns, __ATOMIC_RELAXED), err_dev, __atomic_exchange_n(&w->stall, 0, __ATOMIC_RELAXED)};
    const Call c{w, waits, x, x_stride, rows, y, y_stride, s};
    cudaError_t e;
    SplitPlan p;
    if (plan_fused(w, rows, p)) {
        e = x_type == PK_GGML_F32 ? launch_fused<float>(c, p, y_type)
            : x_type == PK_GGML_F16 ? launch_fused<__half>(c, p, y_type) : launch_fused<__nv_bfloat16>(c, p, y_type);
    } else {
        e = launch_quantize<true>(x, x_type, rows, w->K, x_stride, xc, xs, s);
        if (e == cudaSuccess)
            e = y_type == PK_GGML_F32 ? launch_product<float>(c, xc, xs)
                : y_type == PK_GGML_F16 ? launch_product<__half>(c, xc, xs) : launch_product<__nv_bfloat16>(c, xc, xs);
    }
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}

extern "C" PK_API pk_status pk_fp8_linear(pk_fp8 * w, const void * x, int32_t x_type, int64_t rows, int64_t x_stride, void * y,
                                          int32_t y_type, int64_t y_stride, void * workspace, int64_t workspace_bytes,
                                          void * stream) {
    return pk::fp8_linear(w, "pk_fp8_linear", x, x_type, rows, x_stride, y, y_type, y_stride, workspace, workspace_bytes, stream, nullptr);
}

extern "C" PK_API int64_t pk_fp8_timeouts(pk_fp8 * w) {
    if (!w) return -1;
    notice_timeout(*w);
    return __atomic_load_n(&w->timeouts, __ATOMIC_ACQUIRE);
}
