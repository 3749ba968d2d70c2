// pk_sample.cu -- one token per row of logits: temperature, top-k, top-p and min-p, and a draw
// by a given random number.
//
// The three filters each keep a prefix of the same order (larger logit first, among equal ones
// the lower index), so together they keep the shortest of the three: everything above one logit
// and the first few, by index, of those equal to it. No sort is needed, only that logit.
//
// Weights w = exp((l - max) / T) are held as integers, round(w * 2^43): their sums are exact
// whatever their order, so the cut and the draw do not depend on how a row is split over
// threads. A token is lost only below 2^-44 of the largest weight, and 2^19 tokens of weight
// one stay below 2^63. The exponential is taken in f64: with f32's error of 2^-23 of each
// weight the running sum would move by as much as one token in a thousand rows needs to become
// another.

#include "pk_ops.cuh"

#include <algorithm>
#include <math_constants.h>

namespace pk {
namespace {

using u64 = unsigned long long;

constexpr int kSThreads = 512;
constexpr double kOne = 8796093022208.0;   // 2^43

// Order-preserving key of a logit; NaN as -infinity, -0 as +0.
__device__ __forceinline__ unsigned key_of(float l) {
    if (l != l) l = -CUDART_INF_F;
    const unsigned b = __float_as_uint(l + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
constexpr unsigned kNone = 0x007FFFFFu;    // key of -infinity

struct Row {
    float top;        // largest logit
    float temp;
    double lmin;      // log of min_p, -infinity when off
};

// (l - max) / T; 0 at the maximum itself, infinite or not.
__device__ __forceinline__ double scaled(float l, const Row & r) {
    return l == r.top ? 0.0 : ((double) l - (double) r.top) / (double) r.temp;
}
// 0 for what min-p drops
__device__ __forceinline__ u64 weight(float l, const Row & r) {
    const double a = scaled(l, r);
    return a >= r.lmin ? (u64) __double2ull_rn(exp(a) * kOne) : 0ull;
}

template <class V> struct BlockScratch {
    V warp[kSThreads / 32];
    V total;
};

template <class V>
__device__ V block_sum(V v, BlockScratch<V> & s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (lane == 0) s.warp[warp] = v;
    __syncthreads();
    V t = 0;
#pragma unroll
    for (int i = 0; i < kSThreads / 32; ++i) t += s.warp[i];
    return t;
}

// Exclusive scan over the block's threads; total in `total`.
template <class V>
__device__ V block_exclusive(V v, V & total, BlockScratch<V> & s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s.warp[warp] = x;
    __syncthreads();
    V before = 0, t = 0;
#pragma unroll
    for (int i = 0; i < kSThreads / 32; ++i) {
        if (i < warp) before += s.warp[i];
        t += s.warp[i];
    }
    total = t;
    return before + x - v;
}

// One CTA per row. The cut is found by bisection over the 32 bits of the key.
template <class T>
__global__ void __launch_bounds__(kSThreads) sample_kernel(pk_sample_args a) {
    __shared__ BlockScratch<u64> s64;
    __shared__ BlockScratch<int> s32;
    __shared__ unsigned s_key[kSThreads / 32];
    __shared__ int s_found;
    const int V = a.vocab, tid = threadIdx.x;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T * l = static_cast<const T *>(a.logits) + row * a.row_stride;
        unsigned best = 0;
        for (int i = tid; i < V; i += kSThreads) best = max(best, key_of(to_f32(l[i])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
        __syncthreads();
        if ((tid & 31) == 0) s_key[tid >> 5] = best;
        if (tid == 0) s_found = 0x7FFFFFFF;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSThreads / 32; ++i) best = max(best, s_key[i]);
        if (best == kNone) {
            if (tid == 0) {
                a.tokens[row] = -1;
                if (a.logprobs) a.logprobs[row] = -CUDART_INF_F;
            }
            continue;
        }
        Row r;
        r.top = of_key(best);
        r.temp = a.temperatures ? a.temperatures[row] : a.temperature;
        int k = a.top_ks ? a.top_ks[row] : a.top_k;
        const float p = a.top_ps ? a.top_ps[row] : a.top_p;
        const float m = a.min_ps ? a.min_ps[row] : a.min_p;
        float u = a.uniforms[row];
        if (!(r.temp > 0.0f)) {
            int first = 0x7FFFFFFF;
            for (int i = tid; i < V && first == 0x7FFFFFFF; i += kSThreads)
                if (key_of(to_f32(l[i])) == best) first = i;
            atomicMin(&s_found, first);
            __syncthreads();
            if (tid == 0) {
                a.tokens[row] = s_found;
                if (a.logprobs) a.logprobs[row] = 0.0f;
            }
            continue;
        }
        r.lmin = m > 0.0f ? log((double) fminf(m, 1.0f)) : -CUDART_INF;
        if (k <= 0 || k > V) k = V;
        // cut: kept = key > ck, or key == ck and one of the first `ties` of that key
        unsigned ck = kNone;
        long long ties = V;
        if (k < V) {
            unsigned lo = kNone, hi = best;   // largest key with at least k tokens at or above it
            while (lo < hi) {
                const unsigned mid = lo + (hi - lo) / 2 + 1;
                int n = 0;
                for (int i = tid; i < V; i += kSThreads) n += key_of(to_f32(l[i])) >= mid;
                if (block_sum(n, s32) >= k) lo = mid; else hi = mid - 1;
            }
            int n = 0;
            for (int i = tid; i < V; i += kSThreads) n += key_of(to_f32(l[i])) > lo;
            ck = lo;
            ties = k - block_sum(n, s32);
        }
        if (!(p >= 1.0f)) {
            // weights without min-p, which goes by the largest and not by the sum
            Row all = r;
            all.lmin = -CUDART_INF;
            u64 w = 0;
            for (int i = tid; i < V; i += kSThreads) {
                const float x = to_f32(l[i]);
                if (key_of(x) > ck) w += weight(x, all);
            }
            const u64 at_cut = ck > kNone ? weight(of_key(ck), all) : 0ull;
            const u64 sum = block_sum(w, s64) + (ck > kNone ? at_cut * (u64) ties : 0ull);
            const u64 need = max((u64) ceil(p > 0.0f ? (double) p * (double) sum : 0.0), 1ull);
            unsigned lo = ck, hi = best;      // largest key with that weight at or above it
            while (lo < hi) {
                const unsigned mid = lo + (hi - lo) / 2 + 1;
                u64 x = 0;
                for (int i = tid; i < V; i += kSThreads) {
                    const float v = to_f32(l[i]);
                    if (key_of(v) >= mid) x += weight(v, all);
                }
                if (block_sum(x, s64) >= need) lo = mid; else hi = mid - 1;
            }
            u64 x = 0;
            for (int i = tid; i < V; i += kSThreads) {
                const float v = to_f32(l[i]);
                if (key_of(v) > lo) x += weight(v, all);
            }
            const u64 above = block_sum(x, s64), each = weight(of_key(lo), all);
            long long want = each > 0 && need > above ? (long long) ((need - above + each - 1) / each) : ties;
            if (lo == ck) want = min(want, ties);
            ck = lo;
            ties = want;
        }
        // which index is the last tie kept, and the kept total
        u64 total = 0;
        long long seen = 0;

        for (int c = 0; c < V; c += kSThreads) {
            const int i = c + tid;
            const float v = i < V ? to_f32(l[i]) : -CUDART_INF_F;
            const unsigned key = key_of(v);
            int n = 0;
            const int pos = block_exclusive(key == ck && i < V ? 1 : 0, n, s32);
            const bool keep = i < V && key > kNone && (key > ck || (key == ck && seen + pos < ties));
            if (keep) total += weight(v, r);
            seen += n;
        }
        total = block_sum(total, s64);
        u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
        const u64 t = min((u64) ((double) u * (double) total), total - 1);
        u64 run = 0;
        seen = 0;
        for (int c = 0; c < V; c += kSThreads) {
            const int i = c + tid;
            const float v = i < V ? to_f32(l[i]) : -CUDART_INF_F;
            const unsigned key = key_of(v);
            int n = 0;
            const int pos = block_exclusive(key == ck && i < V ? 1 : 0, n, s32);
            const bool keep = i < V && key > kNone && (key > ck || (key == ck && seen + pos < ties));
            const u64 w = keep ? weight(v, r) : 0ull;
            u64 sum = 0;
            const u64 before = run + block_exclusive(w, sum, s64);
            if (before <= t && t < before + w) {
                a.tokens[row] = i;
                if (a.logprobs) a.logprobs[row] = (float) (scaled(v, r) - log((double) total / kOne));
            }
            seen += n;
            run += sum;
            if (run > t) break;
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace pk

extern "C" PK_API pk_status pk_sample(int device, const pk_sample_args * a, void * stream) {
    using namespace pk;
    const char * fn = "pk_sample";
    if (!a) return op_fail(PK_ERR_INVALID, fn, "null arguments");
    const int es = elem_size(a->logits_type);
    if (es == 0) return op_fail(PK_ERR_INVALID, fn, "logits_type must be F32, F16 or BF16");
    if (a->vocab < 1 || a->vocab > PK_SAMPLE_MAX_VOCAB) return op_fail(PK_ERR_INVALID, fn, "vocab must be in [1, PK_SAMPLE_MAX_VOCAB]");
    if (a->rows < 0 || a->rows > 0x7FFFFFFF || a->row_stride < a->vocab || a->row_stride > (INT64_MAX >> 34))
        return op_fail(PK_ERR_INVALID, fn, "rows must be in [0, 2^31) and row_stride at least vocab");
    if (a->rows > 0 && (!a->logits || !a->uniforms || !a->tokens)) return op_fail(PK_ERR_INVALID, fn, "null pointer");
    if (!aligned_to(a->logits, (size_t) es)) return op_fail(PK_ERR_INVALID, fn, "logits must be aligned to their element");
    for (const void * q : {(const void *) a->uniforms, (const void *) a->tokens, (const void *) a->logprobs,
                           (const void *) a->temperatures, (const void *) a->top_ks, (const void *) a->top_ps,
                           (const void *) a->min_ps})
        if (!aligned_to(q, 4)) return op_fail(PK_ERR_INVALID, fn, "row arrays must be 4-byte aligned");
    if (!device_ok(device)) return op_fail(PK_ERR_NO_DEVICE, fn, "no sm_100 device with that index");
    if (a->rows == 0) return PK_OK;
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    const unsigned g = (unsigned) std::min<int64_t>(a->rows, 148 * 4);
    cudaStream_t s = (cudaStream_t) stream;
    if (a->logits_type == PK_GGML_F32) sample_kernel<float><<<g, kSThreads, 0, s>>>(*a);
    else if (a->logits_type == PK_GGML_F16) sample_kernel<__half><<<g, kSThreads, 0, s>>>(*a);
    else sample_kernel<__nv_bfloat16><<<g, kSThreads, 0, s>>>(*a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}
