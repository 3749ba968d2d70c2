// pk_rows.cuh -- rows of f32, f16 or bf16 as the quantisers read and write them (pk_mx4.cu: blocks of 32
// in 4 bits; pk_fp8.cu: blocks of 128 in 8): eight elements a lane, aligned or not, and largest magnitudes.
#pragma once

#include "pk_ops.cuh"

#include <algorithm>

namespace pk {
namespace {

constexpr int kQThreads = 256;

// Eight consecutive elements of a row, as loaded.
template <class T> struct alignas(16) Eight { T e[8]; };

// The four values from column c of a row on, zeros for what is not in the row. 16-byte aligned.
__device__ __forceinline__ void four_of(const float * __restrict__ row, int c, int K, unsigned * w) {
    if (c >= 0 && c + 4 <= K) {
        const uint4 q = __ldg(reinterpret_cast<const uint4 *>(row + c));
        w[0] = q.x;
        w[1] = q.y;
        w[2] = q.z;
        w[3] = q.w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 0;
    if (c >= K) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (c + i < 0 || c + i >= K) continue;
        w[i] = __float_as_uint(__ldg(row + c + i));
    }
}

// Words from byte `off` (below 16, whole elements) of N + 4 words on, N of them, to the front.
template <int N, int ES>
__device__ __forceinline__ void shift_words(unsigned * w, int off) {
#pragma unroll
    for (int i = 0; i < N + 2; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < N + 1; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
    if constexpr (ES == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
    }
}

// Eight elements of a row from column c (a multiple of eight) on, zeros from column K on. VEC: rows are
// 16-byte aligned. Otherwise f32 loads the aligned 16 bytes around and shifts them into place (66043 x 1000:
// 62 us, element by element 74); half precision goes by elements, whose second to eighth load hits the first
// one's lines (49 us; the other way 66, for the row ends' sake).
template <class T, bool VEC>
__device__ __forceinline__ Eight<T> load8(const T * __restrict__ row, int c, int K) {
    Eight<T> v;
    if constexpr (!VEC && sizeof(T) == 4) {
        const int off = (int) (reinterpret_cast<uintptr_t>(row) & 15), at = c - off / 4;
        unsigned w[12];
        four_of(row, at, K, w);
        four_of(row, at + 4, K, w + 4);
        four_of(row, at + 8, off ? K : 0, w + 8);
        shift_words<8, 4>(w, off);
#pragma unroll
        for (int i = 0; i < 8; ++i) v.e[i] = __uint_as_float(w[i]);
    } else if (VEC && c + 8 <= K) {
#pragma unroll
        for (int i = 0; i < (int) sizeof(T) / 2; ++i)
            reinterpret_cast<uint4 *>(v.e)[i] = __ldcs(reinterpret_cast<const uint4 *>(row + c) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.e[i] = from_f32<T>(0.0f);
        if (c < K) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < K) v.e[i] = row[c + i];
        }
    }
    return v;
}

// The other way: a group of `lanes` neighbouring lanes, this one the sub-th, has eight elements each from
// column c on; what lies before column K is stored. The whole warp calls. `on`: this lane's row is there.
// Not VEC: each lane stores the aligned 16 bytes that its neighbour's elements begin, what the ends of a row
// or of the warp's piece of it cut by elements (66043 x 1000 bf16: 67 us, by elements throughout 175).
template <class T, bool VEC>
__device__ __forceinline__ void store8(T * __restrict__ row, int c, int K, const Eight<T> & o, int sub, int lanes, bool on) {
    if constexpr (VEC) {
        if (!on) return;
        if (c + 8 <= K) {
#pragma unroll
            for (int i = 0; i < (int) sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(row + c)[i] = reinterpret_cast<const uint4 *>(o.e)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < K) row[c + i] = o.e[i];
        }
    } else {
        constexpr int ES = (int) sizeof(T), N = 2 * ES, PER = 16 / ES;
        const unsigned * own = reinterpret_cast<const unsigned *>(o.e);
        const int off = (int) (reinterpret_cast<uintptr_t>(row) & 15), bytes = K * ES;
        unsigned w[N + 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xFFFFFFFFu, own[N - 4 + i], 1);
#pragma unroll
        for (int i = 0; i < N; ++i) w[4 + i] = own[i];
        if (!on) return;
        shift_words<N, ES>(w, (16 - off) & 15);
        char * at = reinterpret_cast<char *>(row);
        const int from = sub == 0 ? c * ES : 0;          // what lies before is another warp's
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            if (off == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i + j] = own[i + j];
            }
            const int b = c * ES - off + 4 * i;
            if (b >= from && b + 16 <= bytes) {
                *reinterpret_cast<uint4 *>(at + b) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            } else if (b < bytes) {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int e = b + j * ES;
                    if (e < from || e >= bytes) continue;
                    if constexpr (ES == 4) *reinterpret_cast<unsigned *>(at + e) = w[i + j];
                    else *reinterpret_cast<unsigned short *>(at + e) = (unsigned short) (w[i + (j >> 1)] >> (16 * (j & 1)));
                }
            }
        }
        if (sub == lanes - 1) {                          // the end of the last lane's elements has no lane behind it
#pragma unroll
            for (int j = 1; j < 8; ++j)
                if ((8 - j) * ES <= off && c + j < K) row[c + j] = o.e[j];
        }
    }
}

// Largest magnitude of three; a NaN if one is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
    return m;
}

// Bits of the largest magnitude (as f32; Inf < NaN as integers, in each type).
__device__ __forceinline__ unsigned amax_bits(const Eight<float> & v) {
    const float m = max3_abs(max3_abs(v.e[0], v.e[1], v.e[2]), max3_abs(v.e[3], v.e[4], v.e[5]), max3_abs(v.e[6], v.e[7], 0.0f));
    return __float_as_uint(m);
}
// In half precision two at a time; the larger of the two halves is taken once four lanes have theirs.
template <class T2> __device__ __forceinline__ T2 pair_of(unsigned w) { return *reinterpret_cast<const T2 *>(&w); }
template <class T2> __device__ __forceinline__ unsigned word_of(T2 p) { return *reinterpret_cast<const unsigned *>(&p); }
template <class T2, class T>
__device__ __forceinline__ T2 amax_pair(const Eight<T> & v) {
    const unsigned * w = reinterpret_cast<const unsigned *>(v.e);
    return __hmax2_nan(__hmax2_nan(__habs2(pair_of<T2>(w[0])), __habs2(pair_of<T2>(w[1]))),
                       __hmax2_nan(__habs2(pair_of<T2>(w[2])), __habs2(pair_of<T2>(w[3]))));
}

// Lanes of a row, as a power of two.
inline int row_lanes(long long K) { return K <= 32 ? 2 : K <= 64 ? 3 : K <= 128 ? 4 : 5; }

// Launch of a row kernel: a warp for 32 lanes' rows, up to a few waves; with few rows a warp for each 256 values.
inline dim3 row_blocks(long long rows, long long K) {
    const long long per = (kQThreads / 32) << (5 - row_lanes(K)), x = std::min<long long>((rows + per - 1) / per, 148LL * 32);
    const long long segs = (K + 255) / 256;
    return dim3((unsigned) x, (unsigned) std::max<long long>(1, std::min<long long>(segs, 148 * 8 / x)));
}

}  // namespace
}  // namespace pk
