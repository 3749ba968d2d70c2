// pk_mx4.cu -- 4-bit microscaled floating point: quantisation of rows, the values back,
// and the product of quantised rows with a quantised weight matrix.
//
// A block of 32 values of a row is held as 32 e2m1 codes (sign, two exponent bits, one
// mantissa bit: magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6) and one e8m0 scale byte B, value =
// code * 2^(B - 127). With a = max |x| of the block, B - 127 = max(floor(log2 a) - 2, -127):
// the top code's exponent is 2, so a / 2^(B - 127) lies in [4, 8) and what exceeds 6 saturates.
// floor(log2 a) is a's exponent field, so B = max(field - 2, 0), exactly, subnormals included;
// x / 2^(B - 127) is an exact f32 product with 2^(127 - B) and the code its nearest value, ties
// to the even code.

#include "pk_product.cuh"
#include "pk_rows.cuh"

#include <algorithm>
#include <mutex>
#include <new>
#include <vector>

namespace pk {
namespace {

// Scales in the layout of the product: 128-row atoms of 4 blocks (K = 128) each, 512 bytes; row r,
// block b at byte (r % 32) * 16 + (r / 32) * 4 + b: 32 rows of four words, a word = the four
// blocks of one row. `chunks` atoms per 128 rows, an even number: stages are two atoms deep.
__host__ __device__ inline int scale_chunks(int K) { return 2 * ((K + 255) / 256); }
__device__ __forceinline__ size_t scale_at(long long row, int blk, int chunks) {
    return ((size_t) (row >> 7) * chunks + (blk >> 2)) * 512 + (size_t) ((row & 31) * 16 + ((row >> 5) & 3) * 4 + (blk & 3));
}

// Scale byte of a block from the bits of its largest magnitude; 255 (NaN) for Inf or NaN.
__device__ __forceinline__ unsigned scale_byte(unsigned amax_bits) {
    const unsigned field = amax_bits >> 23;
    return field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
}

// 2^(127 - B) and 2^(B - 127).
__device__ __forceinline__ float scale_inv(unsigned b) { return __uint_as_float((254u - b) << 23); }
__device__ __forceinline__ float scale_val(unsigned b) {
    return __uint_as_float(b == 255u ? 0x7FC00000u : b == 0u ? 0x00400000u : b << 23);
}

// Two e2m1 codes, lo in bits 0-3 and hi in bits 4-7: nearest, ties to even, saturating.
__device__ __forceinline__ unsigned cvt_e2m1x2(float lo, float hi) {
    unsigned r;
    asm("{ .reg .b8 t; cvt.rn.satfinite.e2m1x2.f32 t, %1, %2; cvt.u32.u8 %0, t; }" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Eight codes and their block's scale byte; four neighbouring lanes hold a block.
__device__ __forceinline__ unsigned join_codes(const unsigned * c) {
    return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
__device__ __forceinline__ unsigned quantize8(const Eight<float> & v, unsigned & sb) {
    unsigned m = amax_bits(v);
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    sb = scale_byte(m);
    const float inv = scale_inv(sb);                 // garbage for byte 255, whose codes are dropped
    unsigned c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = cvt_e2m1x2(v.e[2 * i] * inv, v.e[2 * i + 1] * inv);
    const unsigned q = join_codes(c);
    return sb == 255u ? 0u : q;
}
__device__ __forceinline__ unsigned quantize8(const Eight<__nv_bfloat16> & v, unsigned & sb) {
    using T2 = __nv_bfloat162;
    T2 m = amax_pair<T2>(v);
    m = __hmax2_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = __hmax2_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    const unsigned both = word_of(m);
    sb = scale_byte(max(both << 16, both & 0xFFFF0000u));
    // the product with a power of two is exact in bf16 too, what underflows being far below a half code
    const unsigned inv = (254u - sb) << 7;
    const T2 inv2 = pair_of<T2>(inv << 16 | inv);
    const unsigned * w = reinterpret_cast<const unsigned *>(v.e);
    unsigned c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned x = word_of(__hmul2(pair_of<T2>(w[i]), inv2));
        c[i] = cvt_e2m1x2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
    }
    const unsigned q = join_codes(c);
    return sb == 255u ? 0u : q;
}
__device__ __forceinline__ unsigned quantize8(const Eight<__half> & v, unsigned & sb) {
    using T2 = __half2;
    T2 m = amax_pair<T2>(v);
    m = __hmax2_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = __hmax2_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    sb = scale_byte(__float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))));
    const float inv = scale_inv(sb);
    const unsigned * w = reinterpret_cast<const unsigned *>(v.e);
    unsigned c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(pair_of<T2>(w[i]));
        c[i] = cvt_e2m1x2(x.x * inv, x.y * inv);
    }
    const unsigned q = join_codes(c);
    return sb == 255u ? 0u : q;
}

// The scale bytes of a warp's eight blocks (each in four lanes) as two words of four, in lanes 0 and 16.
__device__ __forceinline__ unsigned scale_word(unsigned sb) {
    unsigned w = sb | __shfl_down_sync(0xFFFFFFFFu, sb, 4) << 8;
    w |= __shfl_down_sync(0xFFFFFFFFu, w, 8) << 16;
    return w;
}

// A warp's 256 values of a row: eight per lane. Where a row goes on, the next 256 follow in the same
// warp, gridDim.y segments further on; several loads are in flight before the first is used. SHORT, for
// rows of up to 256 values: 2^gs lanes a row, and the next rows instead of the next segments (483966 rows of
// 49 bf16: 24 us, a warp a row 114).
// ATOMS: scales in the product's layout, zeros for the blocks past K that its stages read.
// Bound: HBM from f32 (66044 x 1024: 44 us, of which the 270 MB read are 6.1 TB/s; the 36 MB written stay in
// L2), instructions from half precision (66043 x 1000 bf16: 32 us for 132 MB read and 35 written).
template <class T, bool VEC, bool ATOMS, bool SHORT>
__global__ void __launch_bounds__(kQThreads) mx4_quantize_kernel(const T * __restrict__ x, long long rows, int K, long long ldx, int gs,
                                                                 unsigned char * __restrict__ codes,
                                                                 unsigned char * __restrict__ scales) {
    constexpr int UN = sizeof(T) == 4 ? 2 : 4;
    const int lane = threadIdx.x & 31;
    // the product may set itself up while the last blocks work; it waits for all of them before it loads
    if (ATOMS) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int segs = (K + 255) >> 8, nb = (K + 31) >> 5, chunks = scale_chunks(K);
    long long row = (long long) blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5);
    long long stride = (long long) gridDim.x * (kQThreads / 32);
    if constexpr (SHORT) {
        const int sub = lane & ((1 << gs) - 1), blk = sub >> 2;
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
                const unsigned q = quantize8(v[u], sb);
                if (r < rows && blk < nb) *reinterpret_cast<unsigned *>(codes + (size_t) r * nb * 16 + sub * 4) = q;
                if (ATOMS) {
                    // two words a row: with fewer lanes than blocks in them, other rows' bytes are zeros here
                    const unsigned word = scale_word(sb);
                    if (gs == 5) {
                        if (r < rows && (lane & 15) == 0) *reinterpret_cast<unsigned *>(scales + scale_at(r, blk, chunks)) = word;
                    } else if (r < rows && sub < 2) {
                        *reinterpret_cast<unsigned *>(scales + scale_at(r, sub * 4, chunks)) =
                            sub == 0 ? word & (0xFFFFFFFFu >> (32 - 8 * nb)) : 0u;
                    }
                } else if (r < rows && (lane & 3) == 0 && blk < nb) {
                    scales[(size_t) r * nb + blk] = (unsigned char) sb;
                }
            }
        }
    } else {
        for (; row < rows; row += stride) {
            const T * xr = x + row * ldx;
            unsigned char * cr = codes + (size_t) row * nb * 16 + lane * 4;
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
                    const int blk = seg * 8 + (lane >> 2);
                    unsigned sb;
                    const unsigned q = quantize8(v[u], sb);
                    if (blk < nb) *reinterpret_cast<unsigned *>(cr + (size_t) seg * 128) = q;
                    if (ATOMS) {
                        const unsigned word = scale_word(sb);
                        if ((lane & 15) == 0) *reinterpret_cast<unsigned *>(scales + scale_at(row, blk, chunks)) = word;
                    } else if ((lane & 3) == 0 && blk < nb) {
                        scales[(size_t) row * nb + blk] = (unsigned char) sb;
                    }
                }
            }
        }
    }
}

// Eight codes as bf16 bit patterns, two a word: 0, 0x3F00, 0x3F80, 0x3FC0, 0x4000, 0x4040, 0x4080,
// 0x40C0 and the sign. Four codes' low and high bytes are each one byte permutation.
__device__ __forceinline__ void codes_to_bf16(unsigned q, unsigned * w) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned c = (q >> (16 * h)) & 0xFFFFu, sel = c & 0x7777u;
        const unsigned lo = __byte_perm(0xC0800000u, 0xC0804000u, sel), hi = __byte_perm(0x3F3F3F00u, 0x40404040u, sel);
        const unsigned sign = (c & 0x8u) << 4 | (c & 0x80u) << 8 | (c & 0x800u) << 12 | (c & 0x8000u) << 16;
        w[2 * h] = __byte_perm(lo, hi | sign, 0x5140);
        w[2 * h + 1] = __byte_perm(lo, hi | sign, 0x7362);
    }
}

// Eight codes' values. In bf16 the product with the scale, a power of two, is exact (subnormals are
// bf16's as they are f32's), or infinite as the rounded value is.
template <class T> __device__ __forceinline__ void codes_to_values(unsigned q, unsigned b, Eight<T> & o) {
    unsigned w[4];
    codes_to_bf16(q, w);
    const float s = scale_val(b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o.e[2 * i] = from_f32<T>(__uint_as_float(w[i] << 16) * s);
        o.e[2 * i + 1] = from_f32<T>(__uint_as_float(w[i] & 0xFFFF0000u) * s);
    }
}
template <> __device__ __forceinline__ void codes_to_values(unsigned q, unsigned b, Eight<__nv_bfloat16> & o) {
    unsigned w[4];
    codes_to_bf16(q, w);
    const unsigned s = b == 255u ? 0x7FC0u : b == 0u ? 0x0040u : b << 7;
    const __nv_bfloat162 s2 = pair_of<__nv_bfloat162>(s << 16 | s);
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<unsigned *>(o.e)[i] = word_of(__hmul2(pair_of<__nv_bfloat162>(w[i]), s2));
}

// The value of each code, eight a lane, rows and lanes as in the quantisation. Bound: HBM, writing y
// (66043 x 1000 bf16: 34 us for 35 MB read, mostly from L2, and 132 written).
template <class T, bool VEC, bool SHORT>
__global__ void __launch_bounds__(kQThreads) mx4_dequantize_kernel(const unsigned char * __restrict__ codes,
                                                                   const unsigned char * __restrict__ scales, long long rows,
                                                                   int K, T * __restrict__ y, long long ldy, int gs) {
    constexpr int UN = 4;
    const int lane = threadIdx.x & 31;
    const int segs = (K + 255) >> 8, nb = (K + 31) >> 5;
    long long row = (long long) blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5);
    long long stride = (long long) gridDim.x * (kQThreads / 32);
    if constexpr (SHORT) {
        const int sub = lane & ((1 << gs) - 1);
        row = (row << (5 - gs)) + (lane >> gs);
        stride <<= 5 - gs;
        for (; __any_sync(0xFFFFFFFFu, row < rows); row += UN * stride) {
            unsigned q[UN];
            unsigned char b[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const long long r = row + u * stride;
                const bool in = r < rows && sub * 8 < K;
                q[u] = in ? __ldcs(reinterpret_cast<const unsigned *>(codes + (size_t) r * nb * 16 + sub * 4)) : 0u;
                b[u] = in ? __ldcs(scales + (size_t) r * nb + (sub >> 2)) : (unsigned char) 0;
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
            const unsigned char * cr = codes + (size_t) row * nb * 16 + lane * 4, * sr = scales + (size_t) row * nb + (lane >> 2);
            for (int s0 = blockIdx.y; s0 < segs; s0 += UN * (int) gridDim.y) {
                unsigned q[UN];
                unsigned char b[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int seg = s0 + u * (int) gridDim.y;
                    const bool in = seg * 256 + lane * 8 < K;
                    q[u] = in ? __ldcs(reinterpret_cast<const unsigned *>(cr + (size_t) seg * 128)) : 0u;
                    b[u] = in ? __ldcs(sr + seg * 8) : (unsigned char) 0;
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

// GGUF MXFP4 blocks (17 bytes: the scale byte, then 16 bytes whose low halves are values 0-15 and
// high halves values 16-31) to codes in value order and scale atoms. One thread per block.
__global__ void __launch_bounds__(kQThreads) mx4_repack_kernel(const unsigned char * __restrict__ src, long long rows, int nb,
                                                               unsigned char * __restrict__ codes,
                                                               unsigned char * __restrict__ scales) {
    const long long i = (long long) blockIdx.x * kQThreads + threadIdx.x;
    if (i >= rows * nb) return;
    const long long row = i / nb;
    const int blk = (int) (i - row * nb);
    const unsigned char * b = src + i * 17;
    unsigned char * c = codes + i * 16;
    const int chunks = scale_chunks(nb * 32);
    scales[scale_at(row, blk, chunks)] = b[0];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned lo = b[1 + 2 * j], hi = b[2 + 2 * j];
        c[j] = (unsigned char) ((lo & 15u) | (hi & 15u) << 4);
        c[8 + j] = (unsigned char) (lo >> 4 | (hi & 0xF0u));
    }
}

// ---- product on the tensor cores ------------------------------------------------
//
// tcgen05.mma kind::mxf4 with block scales: 64 values of K a product, accumulator in tensor memory.
// One persistent CTA an SM walks over 128 x BN tiles of y. Warp 0 loads (codes by TMA, 256 values =
// one 128-byte swizzled row a stage; scale atoms by bulk copies), warp 1 copies the stage's scales to
// tensor memory and issues its four products, warps from 4 on empty the accumulator, of which there are
// two, so that a tile's epilogue runs under the next tile's products. Each stage has tensor-memory
// columns of its own for its scales: they are free when the stage is.
constexpr int kTM = 128;
template <bool BOX> constexpr int tc_stages() { return BOX ? 5 : 4; }
// Warps of the epilogue, for each 32 rows two where TMA stores y and four where the warps do (layers replayed
// from a graph, quantisation included: 16391 x 1024 by 1025 34.9 us, with two 36.8; 66044 x 1024 by 640, by TMA,
// 90.4 us, with four, whose staging costs a stage of the ring, 94.4).
template <bool BOX> constexpr int epi_warps() { return BOX ? 8 : 16; }
template <bool BOX> constexpr int tc_threads() { return 32 * (4 + epi_warps<BOX>()); }
constexpr unsigned kScaleA = 1024;                      // two atoms of 128 rows
constexpr unsigned kScaleCols = 16;                     // tensor-memory columns of a stage's scales: 8 + 8

struct TcSmem {
    unsigned long long full[5], empty[5], acc_full[2], acc_empty[2], done;
    unsigned tmem;
    int err;
};

// The four products of a stage of 256 values and the copies of their scales (columns ca: 8 for x, then
// NA per chunk for the weights), by one elected lane. The whole warp runs the loop around it, so that
// addresses and descriptors stay in uniform registers: with one lane in the loop a stage took as long
// to issue as 2.5 stages take to multiply.
template <int BN, bool PAIR>
__device__ __forceinline__ void issue_stage(unsigned d, unsigned a, unsigned b, unsigned sa, unsigned sb, unsigned ca, unsigned shift,
                                            bool fresh) {
    constexpr unsigned NA = BN > 128 ? 8 : 4;
    const unsigned cb = ca + 8;
    const unsigned long long da = umma_desc_sw128(a), db = umma_desc_sw128(b), dsa = scale_desc(sa), dsb = scale_desc(sb);
#pragma unroll
    for (unsigned c = 0; c < 2; ++c) {                    // an atom of 512 bytes is 32 in a descriptor's units
        umma_copy_scales<PAIR>(ca + c * 4, dsa + c * 32);
        umma_copy_scales<PAIR>(cb + c * NA, dsb + c * 32);
        if (BN > 128) umma_copy_scales<PAIR>(cb + c * NA + 4, dsb + 64 + c * 32);
    }
#pragma unroll
    for (unsigned j = 0; j < 4; ++j)                      // 32 bytes along the swizzled rows
        umma_mxf4<PAIR>(d, da + 2 * j, db + 2 * j, umma_idesc_mxf4(PAIR ? 2 * kTM : kTM, BN, 2 * (j & 1)), ca + (j >> 1) * 4,
                        cb + (j >> 1) * NA + shift, j > 0 || !fresh ? 1u : 0u);
}

template <int BN> constexpr unsigned tc_stage_bytes() { return kTM * 128u + BN * 128u + 2 * kScaleA; }
constexpr unsigned kOutBytes = 4096;                    // an epilogue warp's 32 staged rows of 128 bytes
template <int BN, bool BOX> constexpr size_t tc_smem_bytes() {
    return 1024 + (size_t) tc_stages<BOX>() * tc_stage_bytes<BN>() + epi_warps<BOX>() * kOutBytes + sizeof(TcSmem);
}

// A warp's 32 rows of an accumulator to y, 128 bytes of them in every STEP (the `half`-th), through shared
// memory. BOX: staged as the 128-byte swizzle has it and stored by TMA, which leaves out what lies past
// M or N; otherwise by the warp, a row's values together.
template <class T> constexpr int store_cols() { return 128 / (int) sizeof(T); }

__device__ __forceinline__ void box_store(const CUtensorMap * map, int n, long long m, const void * src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                 :: "l"(map), "r"(n), "r"((int) m), "r"(smem_u32(src)) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <class T, int BN, bool BOX, int STEP>
__device__ __forceinline__ void store_tile(unsigned acc, unsigned char * st, int half, int lane, long long m0, int rows, int n0, int N,
                                           const float * __restrict__ bias, T * __restrict__ y, long long ldy, const CUtensorMap * ymap) {
    if constexpr (BOX) {
        constexpr int COLS = store_cols<T>(), PARTS = COLS / 32;
#pragma unroll 1
        for (int c = half * COLS; c < BN && n0 + c < N; c += STEP * COLS) {
            if (rows <= 0) break;
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
#pragma unroll
            for (int h = 0; h < PARTS; ++h) {
                unsigned v[32];
                tmem_load32(acc + c + h * 32, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (bias) {                              // padded to whole tiles
                    const float4 * b4 = reinterpret_cast<const float4 *>(bias + n0 + c + h * 32);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 b = __ldg(b4 + i);
                        v[4 * i] = __float_as_uint(__uint_as_float(v[4 * i]) + b.x);
                        v[4 * i + 1] = __float_as_uint(__uint_as_float(v[4 * i + 1]) + b.y);
                        v[4 * i + 2] = __float_as_uint(__uint_as_float(v[4 * i + 2]) + b.z);
                        v[4 * i + 3] = __float_as_uint(__uint_as_float(v[4 * i + 3]) + b.w);
                    }
                }
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4 *>(st + lane * 128 + ((i ^ (lane & 7)) << 4)) =
                            make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        T e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(__uint_as_float(v[8 * i + j]));
                        *reinterpret_cast<uint4 *>(st + lane * 128 + (((h * 4 + i) ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4 *>(e);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) box_store(ymap, n0 + c, m0, st);
        }
    } else {
        float * sf = reinterpret_cast<float *>(st);      // value i of row r at place i ^ r of the row
#pragma unroll 1
        for (int c = half * 32; c < BN && n0 + c < N; c += STEP * 32) {
            unsigned v[32];
            tmem_load32(acc + c, v);
            const int n = n0 + c + lane;
            const float bv = bias && n < N ? __ldg(bias + n) : 0.0f;
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 32; ++i) sf[lane * 32 + (i ^ lane)] = __uint_as_float(v[i]);
            __syncwarp();
            if (n < N) {
                T * o = y + m0 * ldy + n;
                if (rows == 32) {
#pragma unroll
                    for (int r = 0; r < 32; ++r, o += ldy) *o = from_f32<T>(sf[r * 32 + (lane ^ r)] + bv);
                } else {
                    for (int r = 0; r < rows; ++r, o += ldy) *o = from_f32<T>(sf[r * 32 + (lane ^ r)] + bv);
                }
            }
            __syncwarp();
        }
    }
}

template <class T, int BN, bool BOX>
__global__ void __launch_bounds__(tc_threads<BOX>(), 1)
mx4_tc_kernel(const __grid_constant__ CUtensorMap amap, const unsigned char * __restrict__ ascale, long long M, int K,
              const __grid_constant__ CUtensorMap wmap, const unsigned char * __restrict__ wscale, int N,
              const float * __restrict__ bias, T * __restrict__ y, long long ldy, const __grid_constant__ CUtensorMap ymap, const Waits w) {
    constexpr int STAGES = tc_stages<BOX>(), EPI = epi_warps<BOX>();
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char * ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t) 1023);
    unsigned char * out = reinterpret_cast<unsigned char *>(ring + STAGES * tc_stage_bytes<BN>());
    TcSmem & S = *reinterpret_cast<TcSmem *>(out + EPI * kOutBytes);
    const int warp = __shfl_sync(0xFFFFFFFFu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int chunks = scale_chunks(K), nks = chunks / 2, nt = (N + BN - 1) / BN;
    const long long tiles = ((M + kTM - 1) / kTM) * nt;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], EPI);
        }
        mbar_init(&S.done, 1);
        S.err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&S.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = __shfl_sync(0xFFFFFFFFu, S.tmem, 0);

    if (warp == 0) {
        if (lane == 0) {
            unsigned it = 0;
            bool ok = true;
            asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' codes and scales are there
            for (long long t = w.stall && blockIdx.x == 0 ? tiles : blockIdx.x; t < tiles && ok; t += gridDim.x) {
                const int m = (int) (t / nt), n0 = (int) (t % nt) * BN;
                const unsigned char * as = ascale + (size_t) m * chunks * 512;
                const unsigned char * bs = wscale + (size_t) (n0 >> 7) * chunks * 512;
                for (int ks = 0; ks < nks; ++ks, ++it) {
                    const int s = (int) (it % STAGES);
                    if (!mbar_wait(&S.empty[s], ((it / STAGES) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                    unsigned char * a = ring + s * tc_stage_bytes<BN>(), * b = a + kTM * 128, * sa = b + BN * 128;
                    mbar_expect(&S.full[s], tc_stage_bytes<BN>());
                    tma_load_2d(a, &amap, ks * 128, m * kTM, &S.full[s]);
                    tma_load_2d(b, &wmap, ks * 128, n0, &S.full[s]);
                    bulk_load(sa, as + (size_t) ks * 1024, 1024, &S.full[s]);
                    bulk_load(sa + kScaleA, bs + (size_t) ks * 1024, 1024, &S.full[s]);
                }
            }
            // nothing in flight when the block ends, however the others ended
            for (unsigned j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_drain(&S.full[j % STAGES], (j / STAGES) & 1u);
        }
    } else if (warp == 1) {
        unsigned tile = 0, s = 0, ph = 0;
        bool ok = true;
        for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++tile) {
            const unsigned buf = tile & 1u, shift = (unsigned) ((int) (t % nt) * BN & 127) >> 5;
            if (!warp_wait(&S.acc_empty[buf], ((tile >> 1) & 1u) ^ 1u, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int ks = 0; ks < nks; ++ks) {
                if (!warp_wait(&S.full[s], ph, w.ns, &S.err)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned a = smem_u32(ring) + s * tc_stage_bytes<BN>(), b = a + kTM * 128u, sa = b + BN * 128u;
                if (elect_one()) {
                    issue_stage<BN, false>(tmem + buf * BN, a, b, sa, sa + kScaleA, tmem + 2 * BN + s * kScaleCols, shift, ks == 0);
                    umma_commit(&S.empty[s]);
                    if (ks == nks - 1) umma_commit(&S.acc_full[buf]);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
        }
        if (elect_one()) umma_commit(&S.done);           // no product in flight either
        mbar_drain(&S.done, 0u);
    } else if (warp >= 4) {
        const int q = warp & 3;                          // this warp's tensor-memory lanes: rows 32 q ..
        const int half = (warp - 4) >> 2;                // its columns: every other 32
        unsigned char * st = out + (warp - 4) * kOutBytes;
        unsigned tile = 0;
        for (long long t = blockIdx.x; t < tiles; t += gridDim.x, ++tile) {
            const long long m0 = (t / nt) * kTM + q * 32;
            const int n0 = (int) (t % nt) * BN;
            const unsigned buf = tile & 1u;
            if (!warp_wait(&S.acc_full[buf], (tile >> 1) & 1u, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int rows = (int) max(0LL, min(32LL, M - m0));
            store_tile<T, BN, BOX, EPI / 4>(tmem + buf * BN + ((unsigned) (q * 32) << 16), st, half, lane, m0, rows, n0, N, bias, y, ldy, &ymap);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) mbar_arrive(&S.acc_empty[buf]);
        }
        if (BOX && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 2) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
    if (threadIdx.x == 0 && S.err != 0) atomicExch_system(w.err, 1);
}

// ---- many rows: pairs of blocks ---------------------------------------------------
//
// With single blocks' tiles a stage of 128 x 192 x 256 products reads 44 KB, which the L2 gives an SM in
// twice the time that the products take. Two blocks of a cluster together take 256 rows (cta_group::2): each holds
// its 128 rows' codes and half of the tile's weights, and the products read the other half from the
// other SM, so a stage is 31 KB. The pair's first block issues, and both blocks' loads arrive on its
// barrier. The scales of all BN weight rows are loaded by both, each for its own tensor memory.
constexpr int kPStages = 5;
constexpr unsigned kScaleB = 2048;                      // two atoms of each of two times 128 weight rows
constexpr unsigned kPScaleCols = 24;
template <int BN> constexpr unsigned pair_stage() { return kTM * 128u + BN / 2 * 128u + kScaleA + kScaleB; }
// bytes that one block loads a stage
template <int BN> constexpr unsigned pair_bytes() { return kTM * 128u + BN / 2 * 128u + kScaleA + (BN > 128 ? 2048u : 1024u); }
struct PairSmem {
    unsigned long long full[kPStages], empty[kPStages], acc_full[2], acc_empty[2], done;
    unsigned tmem;
    int err;
    unsigned loads;              // stages that this block's loader issued
    unsigned its_loads;          // the other block's, and whether a wait of its ran out
    int its_err;
};
template <int BN, bool BOX> constexpr size_t pair_smem() {
    return 1024 + (size_t) kPStages * pair_stage<BN>() + epi_warps<BOX>() * kOutBytes + sizeof(PairSmem);
}
static_assert(sharing_ruled_out(pair_smem<128, true>(), pair_smem<128, true>()) && sharing_ruled_out(pair_smem<128, true>(), kClusterSmem),
              "it takes all of the tensor memory");

template <class T, int BN, bool BOX>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(tc_threads<BOX>(), 1)
mx4_pair_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap asmap, long long M, int K,
                const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap wsmap, int N,
                const float * __restrict__ bias, T * __restrict__ y, long long ldy, const __grid_constant__ CUtensorMap ymap, const Waits w) {
    constexpr int EPI = epi_warps<BOX>();
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char * ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t) 1023);
    unsigned char * out = ring + kPStages * pair_stage<BN>();
    PairSmem & S = *reinterpret_cast<PairSmem *>(out + EPI * kOutBytes);
    const int warp = __shfl_sync(0xFFFFFFFFu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned rank = blockIdx.x & 1u;
    const int nks = scale_chunks(K) / 2, nt = (N + BN - 1) / BN;
    const long long tiles = ((M + 2 * kTM - 1) / (2 * kTM)) * nt, first = blockIdx.x >> 1, step = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPStages; ++s) {
            mbar_init(&S.full[s], 1);                     // used in the first block
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 2 * EPI);
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
            unsigned it = 0;
            bool ok = true;
            asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' codes and scales are there
            for (long long t = w.stall && blockIdx.x == 1 ? tiles : first; t < tiles && ok; t += step) {
                const int m = (int) (t / nt) * 2 + (int) rank, n0 = (int) (t % nt) * BN;
                for (int ks = 0; ks < nks; ++ks, ++it) {
                    const int s = (int) (it % kPStages);
                    if (!mbar_wait(&S.empty[s], ((it / kPStages) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                    unsigned char * a = ring + s * pair_stage<BN>(), * b = a + kTM * 128, * sa = b + BN / 2 * 128;
                    // rows past M or N, and their scales, read as zeros
                    const unsigned bar = mbar_at(&S.full[s], 0);
                    if (rank == 0) mbar_expect(&S.full[s], 2u * pair_bytes<BN>());
                    tma_load_2d_pair(a, &amap, ks * 128, m * kTM, bar);
                    tma_load_2d_pair(b, &wmap, ks * 128, n0 + (int) rank * (BN / 2), bar);
                    tma_load_2d_pair(sa, &asmap, ks * 256, m, bar);
                    tma_load_2d_pair(sa + kScaleA, &wsmap, ks * 256, n0 >> 7, bar);
                }
            }
            S.loads = it;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            unsigned tile = 0, s = 0, ph = 0;
            bool ok = true;
            for (long long t = first; t < tiles && ok; t += step, ++tile) {
                const unsigned buf = tile & 1u, shift = (unsigned) ((int) (t % nt) * BN & 127) >> 5;
                if (!warp_wait<true>(&S.acc_empty[buf], ((tile >> 1) & 1u) ^ 1u, w.ns, &S.err)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int ks = 0; ks < nks; ++ks) {
                    if (!warp_wait<true>(&S.full[s], ph, w.ns, &S.err)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned a = smem_u32(ring) + s * pair_stage<BN>(), b = a + kTM * 128u, sa = b + BN / 2 * 128u;
                    if (elect_one()) {
                        issue_stage<BN, true>(tmem + buf * BN, a, b, sa, sa + kScaleA, tmem + 2 * 192 + s * kPScaleCols, shift, ks == 0);
                        umma_commit_pair(&S.empty[s]);
                        if (ks == nks - 1) umma_commit_pair(&S.acc_full[buf]);
                    }
                    __syncwarp();
                    if (++s == kPStages) { s = 0; ph ^= 1u; }
                }
            }
            // no product in flight when the blocks end
            if (elect_one()) umma_commit_pair(&S.done);
            mbar_drain(&S.done, 0u);
        }
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2;
        unsigned char * st = out + (warp - 4) * kOutBytes;
        unsigned tile = 0;
        for (long long t = first; t < tiles; t += step, ++tile) {
            const long long m0 = ((t / nt) * 2 + rank) * kTM + q * 32;
            const int n0 = (int) (t % nt) * BN;
            const unsigned buf = tile & 1u;
            if (!warp_wait(&S.acc_full[buf], (tile >> 1) & 1u, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int rows = (int) max(0LL, min(32LL, M - m0));
            store_tile<T, BN, BOX, EPI / 4>(tmem + buf * BN + ((unsigned) (q * 32) << 16), st, half, lane, m0, rows, n0, N, bias, y, ldy, &ymap);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) mbar_arrive_at(&S.acc_empty[buf], 0);
        }
        if (BOX && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
    // stages that the other has not (five at most: a stage is free again once both blocks' was multiplied). The
    // first block, whose barriers count both blocks' bytes, sets the counts right and waits for what was issued.
    if (S.err | S.its_err) {
        if (rank == 0 && threadIdx.x == 0) {
            const unsigned least = min(S.loads, S.its_loads), most = max(S.loads, S.its_loads);
            for (unsigned j = least; j < most; ++j) {
                if (S.loads < most) mbar_expect(&S.full[j % kPStages], pair_bytes<BN>());
                else mbar_complete(&S.full[j % kPStages], pair_bytes<BN>());
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

// ---- few rows: quantisation and product in one kernel -----------------------------
//
// With few rows the time is that of launches and of single loads, and the weights are nearly all
// of the bytes: every block quantises the rows for itself, into the products' layout in its shared
// memory, while the first weights are on their way, and takes its share of the tiles of 64 outputs.
// One launch: 9.0 us for 1 x 640 by 8198 called from Python, 12.6 us with a kernel for each. Replayed from
// a graph 5.2 and 6.6 us for 1 x 1024, 6.4 and 6.8 for 16, 7.8 and 7.0 for 32; 8.5 and 8.2 for 16 x 2048,
// 10.8 and 8.6 for 32: hence the bound on the values of x. Not so
// for more rows: at 64 the rows' loads, again in every block, take longer than the second launch
// (called from Python 14.3 us against 11.4), and at 66044 keeping the codes on the SM took a seventh longer
// than two kernels, sixteen warps of one block being too few to keep x streaming.
constexpr int kFewRows = 32;
constexpr int kFewK = 2048;                             // the rows' codes stay in shared memory
constexpr int kFewX = 32768;                            // every block quantises all of x
constexpr int kFewN = 64;
constexpr int kFewStages = 4;
constexpr int kFewQuant = 16;                           // quantising warps
constexpr int kFewThreads = 32 * (4 + kFewQuant + 8);
constexpr unsigned kFewSeg = kTM * 128u + kScaleA;      // codes and scales of 256 values of K
constexpr unsigned kFewStage = kFewN * 128u + 1024u;

struct FewSmem {
    unsigned long long full[kFewStages], empty[kFewStages], a_full, acc_full[2], acc_empty[2], done;
    unsigned tmem;
    int err;
};
constexpr size_t few_smem(int nks) { return 1024 + (size_t) nks * kFewSeg + kFewStages * kFewStage + 2 * kOutBytes + sizeof(FewSmem); }

template <class TX, class TY, bool VEC>
__global__ void __launch_bounds__(kFewThreads, 1)
mx4_few_kernel(const TX * __restrict__ x, long long ldx, int M, int K, const __grid_constant__ CUtensorMap wmap,
               const unsigned char * __restrict__ wscale, int N, const float * __restrict__ bias, TY * __restrict__ y, long long ldy,
               const Waits w) {
    extern __shared__ __align__(1024) unsigned char raw[];
    const int chunks = scale_chunks(K), nks = chunks / 2, nt = (N + kFewN - 1) / kFewN;
    unsigned char * a = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t) 1023);
    unsigned char * sa = a + (size_t) nks * kTM * 128;    // the rows' scales follow their codes
    unsigned char * ring = sa + nks * kScaleA;
    unsigned char * out = ring + kFewStages * kFewStage;
    FewSmem & S = *reinterpret_cast<FewSmem *>(out + 2 * kOutBytes);
    const int warp = __shfl_sync(0xFFFFFFFFu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kFewStages; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        mbar_init(&S.a_full, kFewQuant);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 2);
        }
        mbar_init(&S.done, 1);
        S.err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&S.tmem)), "r"(256u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = __shfl_sync(0xFFFFFFFFu, S.tmem, 0);

    if (warp == 0) {
        if (lane == 0) {
            unsigned it = 0;
            bool ok = true;
            for (int t = w.stall && blockIdx.x == 0 ? nt : blockIdx.x; t < nt && ok; t += gridDim.x) {
                const int n0 = t * kFewN;
                const unsigned char * bs = wscale + (size_t) (n0 >> 7) * chunks * 512;
                for (int ks = 0; ks < nks; ++ks, ++it) {
                    const int s = (int) (it % kFewStages);
                    if (!mbar_wait(&S.empty[s], ((it / kFewStages) & 1u) ^ 1u, w.ns, &S.err)) { ok = false; break; }
                    unsigned char * b = ring + s * kFewStage;
                    mbar_expect(&S.full[s], kFewStage);
                    tma_load_2d(b, &wmap, ks * 128, n0, &S.full[s]);
                    bulk_load(b + kFewN * 128, bs + (size_t) ks * 1024, 1024, &S.full[s]);
                }
            }
            for (unsigned j = it > kFewStages ? it - kFewStages : 0; j < it; ++j) mbar_drain(&S.full[j % kFewStages], (j / kFewStages) & 1u);
        }
    } else if (warp == 1) {
        unsigned tile = 0, s = 0, ph = 0;
        bool ok = warp_wait(&S.a_full, 0u, w.ns, &S.err);
        for (int t = blockIdx.x; t < nt && ok; t += gridDim.x, ++tile) {
            const unsigned buf = tile & 1u, shift = (unsigned) ((t * kFewN) & 127) >> 5;
            if (!warp_wait(&S.acc_empty[buf], ((tile >> 1) & 1u) ^ 1u, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int ks = 0; ks < nks; ++ks) {
                if (!warp_wait(&S.full[s], ph, w.ns, &S.err)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned kb = smem_u32(ring) + s * kFewStage;
                if (elect_one()) {
                    issue_stage<kFewN, false>(tmem + buf * kFewN, smem_u32(a) + (unsigned) ks * kTM * 128u, kb,
                                              smem_u32(sa) + (unsigned) ks * kScaleA, kb + kFewN * 128u, tmem + 2 * kFewN + s * 16u, shift, ks == 0);
                    umma_commit(&S.empty[s]);
                    if (ks == nks - 1) umma_commit(&S.acc_full[buf]);
                }
                __syncwarp();
                if (++s == kFewStages) { s = 0; ph ^= 1u; }
            }
        }
        if (elect_one()) umma_commit(&S.done);
        mbar_drain(&S.done, 0u);
    } else if (warp >= 4 && warp < 4 + kFewQuant) {
        // the rows past M keep what is there: their part of the accumulator is not stored
        constexpr int UN = 4;
        for (int r = warp - 4; r < M; r += kFewQuant) {
            const TX * xr = x + r * ldx;
            for (int s0 = 0; s0 < nks; s0 += UN) {
                Eight<TX> v[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) v[u] = load8<TX, VEC>(xr, s0 + u < nks ? (s0 + u) * 256 + lane * 8 : K, K);
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int seg = s0 + u;
                    if (seg >= nks) break;
                    unsigned sb;
                    const unsigned q = quantize8(v[u], sb);
                    // 128-byte swizzle: 16-byte piece c of row r at piece c ^ (r % 8)
                    *reinterpret_cast<unsigned *>(a + (unsigned) (seg * kTM * 128 + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)) = q;
                    const unsigned word = scale_word(sb);
                    if ((lane & 15) == 0)
                        *reinterpret_cast<unsigned *>(sa + (unsigned) (seg * kScaleA + (lane >> 4) * 512 + (r & 31) * 16 + (r >> 5) * 4)) = word;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.a_full);
    } else if (warp >= 4 + kFewQuant && (warp & 3) == 0) {
        // rows 0 to 31 are the tensor-memory lanes of the warps whose number is a multiple of four
        const int half = (warp - 4 - kFewQuant) >> 2;
        unsigned tile = 0;
        for (int t = blockIdx.x; t < nt; t += gridDim.x, ++tile) {
            const unsigned buf = tile & 1u;
            if (!warp_wait(&S.acc_full[buf], (tile >> 1) & 1u, w.ns, &S.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            store_tile<TY, kFewN, false, 2>(tmem + buf * kFewN, out + half * kOutBytes, half, lane, 0, M, t * kFewN, N, bias, y, ldy, nullptr);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) mbar_arrive(&S.acc_empty[buf]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 2) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(256u) : "memory");
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
#define PK_Q2(T, V, S) launch_on(mx4_quantize_kernel<T, V, ATOMS, S>, g, kQThreads, 0, s, static_cast<const T *>(x), rows, K, ldx, gs, codes, scales)
#define PK_Q(T) \
    (K <= 256 ? (vec ? PK_Q2(T, true, true) : PK_Q2(T, false, true)) : vec ? PK_Q2(T, true, false) : PK_Q2(T, false, false))
    return type == PK_GGML_F32 ? PK_Q(float) : type == PK_GGML_F16 ? PK_Q(__half) : PK_Q(__nv_bfloat16);
#undef PK_Q
#undef PK_Q2
}

// Host-visible error words of the layers and of pk_ctc handles, from pages that stay: creating one pays for
// no pinned allocation of its own.
std::mutex error_lock;
std::vector<int *> free_words;

constexpr int64_t kMaxDim = 1 << 20;        // K, N
constexpr int64_t kMaxRows = 0x7FFFFFFF;

}  // namespace

void give_error_word(int * w) {
    std::lock_guard<std::mutex> g(error_lock);
    free_words.push_back(w);
}

int * take_error_word(cudaError_t & e) {
    std::lock_guard<std::mutex> g(error_lock);
    if (free_words.empty()) {
        static size_t words;
        try {
            free_words.reserve(words + 1024);       // giving back never allocates
        } catch (const std::bad_alloc &) {
            e = cudaErrorMemoryAllocation;
            return nullptr;
        }
        void * page = nullptr;
        e = cudaHostAlloc(&page, 4096, cudaHostAllocMapped | cudaHostAllocPortable);
        if (e != cudaSuccess) return nullptr;
        words += 1024;
        for (int i = 0; i < 1024; ++i) free_words.push_back(static_cast<int *>(page) + i);
    }
    int * w = free_words.back();
    free_words.pop_back();
    *w = 0;
    return w;
}

// Whether a wait of a finished product that reports to `w` ran out (asked once).
bool take_error(int * w) { return __atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL) != 0; }

}  // namespace pk

struct pk_mx4 : pk::LayerWaits {
    int device = 0;
    int N = 0, K = 0, nb = 0, chunks = 0;
    unsigned char * codes = nullptr;    // [N][16 nb]; owns the memory of all three
    unsigned char * scales = nullptr;   // atoms
    float * bias = nullptr;             // padded to whole tiles, or null
    alignas(64) CUtensorMap map[3];     // codes in boxes of kBox[i] rows
    alignas(64) CUtensorMap smap[2];    // scales: the two atoms of a stage of 128 rows, of 256 rows
};

namespace pk {
namespace {

constexpr int kBox[3] = {64, 128, 96};   // the last: half of a pair's 192

// Scale atoms as rows of words, one row for 128 rows of values; a box is a stage's two atoms of `rows`
// such rows.
cudaError_t map_scales(CUtensorMap * map, const unsigned char * scales, long long atom_rows, int chunks, int rows) {
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, scales, atom_rows, (long long) chunks * 128, rows, 256, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// y as boxes of 32 rows and 128 bytes; false where TMA cannot store it: rows not 16-byte aligned, or
// not whole 16 bytes long (a store then also writes what follows a row's last value, up to 16 bytes).
bool map_y(CUtensorMap * map, void * y, int type, long long M, int N, long long ldy, cudaError_t & e) {
    const int es = elem_size(type);
    if (!aligned_to(y, 16) || ldy * es % 16 != 0 || (long long) N * es % 16 != 0) return false;
    e = encode_2d_strided(map, type == PK_GGML_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                               : type == PK_GGML_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          y, M, N, ldy * es, 32, 128 / es, CU_TENSOR_MAP_SWIZZLE_128B);
    return true;
}

struct Call {
    const pk_mx4 * w;
    Waits waits;
    const void * x;
    long long ldx, M;
    void * y;
    long long ldy;
    cudaStream_t s;
};

template <class T, int BN, bool BOX>
cudaError_t launch_tc_as(const Call & c, const CUtensorMap & amap, const unsigned char * xs, const CUtensorMap & wmap, const CUtensorMap & ymap) {
    auto kernel = mx4_tc_kernel<T, BN, BOX>;
    static unsigned long long set;
    const size_t smem = tc_smem_bytes<BN, BOX>();
    const cudaError_t e = allow_smem(kernel, smem, c.w->device, set);
    if (e != cudaSuccess) return e;
    const long long tiles = (c.M + kTM - 1) / kTM * ((c.w->N + BN - 1) / BN);
    return launch_after(kernel, (unsigned) std::min<long long>(tiles, 148), tc_threads<BOX>(), smem, c.s,
        amap, xs, c.M, c.w->K, wmap, c.w->scales, c.w->N, c.w->bias, static_cast<T *>(c.y), c.ldy, ymap, c.waits);
}

template <class T, int BN, bool BOX>
cudaError_t launch_pair_as(const Call & c, const CUtensorMap & amap, const unsigned char * xs, const CUtensorMap & ymap) {
    alignas(64) CUtensorMap asmap;
    cudaError_t e = map_scales(&asmap, xs, (c.M + kTM - 1) / kTM, c.w->chunks, 1);
    if (e != cudaSuccess) return e;
    auto kernel = mx4_pair_kernel<T, BN, BOX>;
    static unsigned long long set;
    const size_t smem = pair_smem<BN, BOX>();
    e = allow_smem(kernel, smem, c.w->device, set);
    if (e != cudaSuccess) return e;
    const long long tiles = (c.M + 2 * kTM - 1) / (2 * kTM) * ((c.w->N + BN - 1) / BN);
    return launch_after(kernel, (unsigned) (2 * std::min<long long>(tiles, 74)), tc_threads<BOX>(), smem, c.s,
        amap, asmap, c.M, c.w->K, c.w->map[BN > 128 ? 2 : 0], c.w->smap[BN > 128 ? 1 : 0], c.w->N, c.w->bias, static_cast<T *>(c.y), c.ldy, ymap, c.waits);
}

template <class TX, class TY, bool VEC>
cudaError_t launch_few_as(const Call & c) {
    auto kernel = mx4_few_kernel<TX, TY, VEC>;
    static unsigned long long set;
    const cudaError_t e = allow_smem(kernel, few_smem(kFewK / 256), c.w->device, set);
    if (e != cudaSuccess) return e;
    const int grid = std::min((c.w->N + kFewN - 1) / kFewN, 148);
    return launch_on(kernel, dim3(grid), kFewThreads, few_smem(c.w->chunks / 2), c.s, static_cast<const TX *>(c.x), c.ldx, (int) c.M, c.w->K,
                     c.w->map[0], c.w->scales, c.w->N, c.w->bias, static_cast<TY *>(c.y), c.ldy, c.waits);
}

template <class TX, class TY> cudaError_t launch_few_xy(const Call & c) {
    return aligned_to(c.x, 16) && c.ldx * sizeof(TX) % 16 == 0 ? launch_few_as<TX, TY, true>(c) : launch_few_as<TX, TY, false>(c);
}

template <class TX> cudaError_t launch_few(const Call & c, int y_type) {
    return y_type == PK_GGML_F32 ? launch_few_xy<TX, float>(c)
           : y_type == PK_GGML_F16 ? launch_few_xy<TX, __half>(c) : launch_few_xy<TX, __nv_bfloat16>(c);
}

bool few(const pk_mx4 * w, int64_t rows) { return rows <= kFewRows && w->K <= kFewK && rows * w->K <= kFewX; }

// Tile width of the single blocks: fewest rounds of tiles over the SMs, a round costed by the rows that
// a tile loads. (192, with fewer loads a product, was slower where K is short: by 3 % for 66044 x 1024 by 640, by
// 7 % for 16391 x 1024 by 1025; where K is long the pairs are faster.)
bool narrow_tiles(long long M, int N) {
    auto cost = [&](int bn) { return ((M + kTM - 1) / kTM * ((N + bn - 1) / bn) + 147) / 148 * (kTM + bn); };
    return cost(64) < cost(128);
}

template <class T> cudaError_t launch_product(const Call & c, int y_type, const unsigned char * xc, const unsigned char * xs) {
    alignas(64) CUtensorMap amap, ymap{};
    cudaError_t e = encode_2d(&amap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xc, c.M, (long long) c.w->nb * 16, kTM, 128,
                              CU_TENSOR_MAP_SWIZZLE_128B);
    if (e != cudaSuccess) return e;
    const bool box = map_y(&ymap, c.y, y_type, c.M, c.w->N, c.ldy, e);
    if (e != cudaSuccess) return e;
    // Pairs where there are tiles for all of them and K is long. Layers replayed from a graph, pairs and single
    // blocks, at K = 1024, 1536, 1792, 2048 and 4096: 16391 rows by 1025 42 us and 35, 48 and 45, 50 and 50, 52 and
    // 54, 83 and 91; 66044 by 640 98 and 91, 128 and 127, 145 and 147, 159 and 165, 286 and 304. With more work for
    // each load pairs gain earlier (8192 by 8192 at 1024: 53 and 62, at 512: 47 and 41), with few tiles never (2600
    // by 1300, 1.6 rounds of pairs, at 4096: 24.3 and 23.4); the rule is set by the first two.
    if (c.w->K > 1536 && (c.M + 2 * kTM - 1) / (2 * kTM) * ((c.w->N + 127) / 128) >= 74) {
        const long long mp = (c.M + 2 * kTM - 1) / (2 * kTM);
        const long long r128 = (mp * ((c.w->N + 127) / 128) + 73) / 74 * (kTM + 64), r192 = (mp * ((c.w->N + 191) / 192) + 73) / 74 * (kTM + 96);
        if (r192 <= r128) return box ? launch_pair_as<T, 192, true>(c, amap, xs, ymap) : launch_pair_as<T, 192, false>(c, amap, xs, ymap);
        return box ? launch_pair_as<T, 128, true>(c, amap, xs, ymap) : launch_pair_as<T, 128, false>(c, amap, xs, ymap);
    }
    if (narrow_tiles(c.M, c.w->N))
        return box ? launch_tc_as<T, 64, true>(c, amap, xs, c.w->map[0], ymap) : launch_tc_as<T, 64, false>(c, amap, xs, c.w->map[0], ymap);
    return box ? launch_tc_as<T, 128, true>(c, amap, xs, c.w->map[1], ymap) : launch_tc_as<T, 128, false>(c, amap, xs, c.w->map[1], ymap);
}

}  // namespace
}  // namespace pk

namespace pk {

void mx4_dims(const pk_mx4 * w, int * device, int * N, int * K) {
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
    if (!aligned_to(codes, 4)) return op_fail(PK_ERR_INVALID, fn, "codes must be 4-byte aligned");
    if (!device_ok(device)) return op_fail(PK_ERR_NO_DEVICE, fn, "no sm_100 device with that index");
    return PK_OK;
}

}  // namespace

extern "C" PK_API pk_status pk_mx4_quantize(int device, const void * x, int32_t x_type, int64_t rows, int64_t cols,
                                            int64_t row_stride, uint8_t * codes, uint8_t * scales, void * stream) {
    const char * fn = "pk_mx4_quantize";
    const pk_status st = check_rows(fn, device, x_type, rows, cols, row_stride, x, elem_size(x_type), codes, scales);
    if (st != PK_OK || rows == 0) return st;
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    const cudaError_t e = launch_quantize<false>(x, x_type, rows, (int) cols, row_stride, codes, scales, (cudaStream_t) stream);
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}

extern "C" PK_API pk_status pk_mx4_dequantize(int device, const uint8_t * codes, const uint8_t * scales, int64_t rows, int64_t cols,
                                              void * y, int32_t y_type, int64_t row_stride, void * stream) {
    const char * fn = "pk_mx4_dequantize";
    const pk_status st = check_rows(fn, device, y_type, rows, cols, row_stride, y, elem_size(y_type), codes, scales);
    if (st != PK_OK || rows == 0) return st;
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    const bool vec = aligned_to(y, 16) && (row_stride * elem_size(y_type)) % 16 == 0;
    const dim3 g = row_blocks(rows, cols);
    const int gs = row_lanes(cols);
    cudaStream_t s = (cudaStream_t) stream;
#define PK_D2(T, V, S) launch_on(mx4_dequantize_kernel<T, V, S>, g, kQThreads, 0, s, codes, scales, rows, (int) cols, static_cast<T *>(y), row_stride, gs)
#define PK_D(T) \
    (cols <= 256 ? (vec ? PK_D2(T, true, true) : PK_D2(T, false, true)) : vec ? PK_D2(T, true, false) : PK_D2(T, false, false))
    const cudaError_t e = y_type == PK_GGML_F32 ? PK_D(float) : y_type == PK_GGML_F16 ? PK_D(__half) : PK_D(__nv_bfloat16);
#undef PK_D
#undef PK_D2
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}

extern "C" PK_API void pk_mx4_destroy(pk_mx4 * w) {
    if (!w) return;
    DeviceScope dev(w->device);
    cudaDeviceSynchronize();
    cudaFree(w->codes);
    if (w->err) give_error_word(w->err);
    delete w;
}

extern "C" PK_API pk_status pk_mx4_create(int device, const pk_tensor * weight, int32_t on_device, const float * bias, pk_mx4 ** out) {
    const char * fn = "pk_mx4_create";
    if (!out) return op_fail(PK_ERR_INVALID, fn, "null output");
    *out = nullptr;
    if (!weight || !weight->data) return op_fail(PK_ERR_INVALID, fn, "null weight");
    const int64_t K = weight->ne0, N = weight->ne1;
    if (K < 1 || K > kMaxDim || N < 1 || N > kMaxDim) return op_fail(PK_ERR_MODEL, fn, "weight dimensions must be in [1, 2^20]");
    const int type = weight->type;
    const bool blocks = type == PK_GGML_Q8_0 || type == PK_GGML_MXFP4;
    if (!blocks && elem_size(type) == 0) return op_fail(PK_ERR_MODEL, fn, "weight type must be F32, F16, BF16, Q8_0 or MXFP4");
    if (blocks && K % 32 != 0) return op_fail(PK_ERR_MODEL, fn, "ne0 of a block type must be a multiple of 32");
    const uint64_t want = blocks ? (uint64_t) N * (K / 32) * (type == PK_GGML_Q8_0 ? 34 : 17) : (uint64_t) N * K * elem_size(type);
    if (weight->nbytes != want) return op_fail(PK_ERR_MODEL, fn, "weight nbytes does not match its type and shape");
    const size_t w_align = type == PK_GGML_MXFP4 ? 1 : type == PK_GGML_Q8_0 ? 2 : (size_t) elem_size(type);
    if (on_device && (!aligned_to(weight->data, w_align) || (bias && !aligned_to(bias, 4))))
        return op_fail(PK_ERR_INVALID, fn, "device weight and bias must be aligned to their element");
    if (!device_ok(device)) return op_fail(PK_ERR_NO_DEVICE, fn, "no sm_100 device with that index");
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    pk_mx4 * w = new (std::nothrow) pk_mx4();
    if (!w) return op_fail(PK_ERR_OOM, fn, "host memory");
    w->device = device;
    w->N = (int) N;
    w->K = (int) K;
    w->nb = (int) ((K + 31) / 32);
    w->chunks = scale_chunks((int) K);
    const size_t code_bytes = ((size_t) N * w->nb * 16 + 511) / 512 * 512, scale_bytes = (size_t) ((N + 127) / 128) * w->chunks * 512;
    void * raw = nullptr;    // a host weight's copy
    void * f32 = nullptr;    // q8_0 blocks dequantised
    const cudaStream_t s = cudaStreamPerThread;
    cudaError_t e = on_device ? cudaDeviceSynchronize() : cudaSuccess;
    if (e == cudaSuccess) e = cudaMalloc(&w->codes, code_bytes + scale_bytes + (bias ? (size_t) (N + 255) / 64 * 64 * 4 : 0));
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
    if (e == cudaSuccess && type == PK_GGML_MXFP4) {
        const long long n = N * (long long) w->nb;
        e = launch_on(mx4_repack_kernel, dim3((unsigned) ((n + kQThreads - 1) / kQThreads)), kQThreads, 0, s,
                      static_cast<const unsigned char *>(src), N, w->nb, w->codes, w->scales);
    } else if (e == cudaSuccess && type == PK_GGML_Q8_0) {
        e = cudaMalloc(&f32, (size_t) N * K * 4);
        if (e == cudaSuccess) e = launch_dequant(src, type, K, N, static_cast<float *>(f32), s);
        if (e == cudaSuccess) e = launch_quantize<true>(f32, PK_GGML_F32, N, (int) K, K, w->codes, w->scales, s);
    } else if (e == cudaSuccess) {
        e = launch_quantize<true>(src, type, N, (int) K, K, w->codes, w->scales, s);
    }
    if (e == cudaSuccess && bias)
        e = cudaMemcpyAsync(w->bias, bias, (size_t) N * 4, on_device ? cudaMemcpyDeviceToDevice : cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) w->err = take_error_word(e);
    if (e == cudaSuccess) e = cudaHostGetDevicePointer(reinterpret_cast<void **>(&w->err_dev), w->err, 0);
    for (int i = 0; i < 3 && e == cudaSuccess; ++i)
        e = encode_2d(&w->map[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w->codes, N, (long long) w->nb * 16, kBox[i], 128,
                      CU_TENSOR_MAP_SWIZZLE_128B);
    for (int i = 0; i < 2 && e == cudaSuccess; ++i) e = map_scales(&w->smap[i], w->scales, (N + 127) / 128, w->chunks, i + 1);
    const cudaError_t e2 = cudaStreamSynchronize(s);
    if (e == cudaSuccess) e = e2;
    cudaFree(raw);
    cudaFree(f32);
    if (e != cudaSuccess) {
        pk_mx4_destroy(w);
        return op_cuda_fail(e, fn);
    }
    *out = w;
    return PK_OK;
}

extern "C" PK_API pk_status pk_mx4_set_option(pk_mx4 * w, int32_t option, int64_t value) {
    const char * fn = "pk_mx4_set_option";
    return w ? set_wait_option(*w, fn, option, value) : op_fail(PK_ERR_INVALID, fn, "null layer");
}

namespace {

size_t ws_codes(const pk_mx4 * w, int64_t rows) { return ((size_t) rows * w->nb * 16 + 255) / 256 * 256; }

}  // namespace

extern "C" PK_API int64_t pk_mx4_workspace(const pk_mx4 * w, int64_t rows) {
    if (!w) return -1;
    if (rows <= 0 || few(w, rows)) return 0;
    return (int64_t) (ws_codes(w, rows) + (size_t) ((rows + 127) / 128) * w->chunks * 512);
}

// A product that reports to the error word `err_dev` (the device's address of it); null: to the layer's, whose
// unreported timeouts it then tells of instead of running.
pk_status pk::mx4_linear(pk_mx4 * w, const char * fn, const void * x, int32_t x_type, int64_t rows, int64_t x_stride, void * y,
                         int32_t y_type, int64_t y_stride, void * workspace, int64_t workspace_bytes, void * stream, int * err_dev) {
    if (!w) return op_fail(PK_ERR_INVALID, fn, "null layer");
    if (elem_size(x_type) == 0 || elem_size(y_type) == 0) return op_fail(PK_ERR_INVALID, fn, "element types must be F32, F16 or BF16");
    if (rows < 0 || rows > kMaxRows) return op_fail(PK_ERR_INVALID, fn, "rows must be in [0, 2^31)");
    if (x_stride < w->K || y_stride < w->N || x_stride > (INT64_MAX >> 34) || y_stride > (INT64_MAX >> 34))
        return op_fail(PK_ERR_INVALID, fn, "x_stride must be at least K and y_stride at least N");
    if (rows == 0) return PK_OK;
    const int64_t need = pk_mx4_workspace(w, rows);
    if (!x || !y || (need > 0 && !workspace)) return op_fail(PK_ERR_INVALID, fn, "null pointer");
    if (!aligned_to(x, (size_t) elem_size(x_type)) || !aligned_to(y, (size_t) elem_size(y_type)))
        return op_fail(PK_ERR_INVALID, fn, "x and y must be aligned to their element");
    if (!aligned_to(workspace, 256)) return op_fail(PK_ERR_INVALID, fn, "workspace must be 256-byte aligned");
    if (workspace_bytes < need)
        return op_fail(PK_ERR_INVALID, fn, "workspace_bytes is below pk_mx4_workspace(w, rows)");
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
    if (few(w, rows)) {
        e = x_type == PK_GGML_F32 ? launch_few<float>(c, y_type)
            : x_type == PK_GGML_F16 ? launch_few<__half>(c, y_type) : launch_few<__nv_bfloat16>(c, y_type);
    } else {
        e = launch_quantize<true>(x, x_type, rows, w->K, x_stride, xc, xs, s);
        if (e == cudaSuccess)
            e = y_type == PK_GGML_F32 ? launch_product<float>(c, y_type, xc, xs)
                : y_type == PK_GGML_F16 ? launch_product<__half>(c, y_type, xc, xs) : launch_product<__nv_bfloat16>(c, y_type, xc, xs);
    }
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}

extern "C" PK_API pk_status pk_mx4_linear(pk_mx4 * w, const void * x, int32_t x_type, int64_t rows, int64_t x_stride, void * y,
                                          int32_t y_type, int64_t y_stride, void * workspace, int64_t workspace_bytes,
                                          void * stream) {
    return pk::mx4_linear(w, "pk_mx4_linear", x, x_type, rows, x_stride, y, y_type, y_stride, workspace, workspace_bytes, stream, nullptr);
}

extern "C" PK_API int64_t pk_mx4_timeouts(pk_mx4 * w) {
    if (!w) return -1;
    notice_timeout(*w);
    return __atomic_load_n(&w->timeouts, __ATOMIC_ACQUIRE);
}
