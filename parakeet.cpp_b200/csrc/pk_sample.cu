// pk_sample.cu -- one token per row of logits: temperature, top-k, top-p and min-p, and a draw
// by a given random number.
//
// The three filters each keep a prefix of the same order (larger logit first, among equal ones
// the lower index), so together they keep the shortest of the three: everything above one logit,
// the cut, and the first few, by index, of those equal to it. No sort is needed, only the cut.
//
// Weights w = exp((l - max) / T) are held as integers, round(w * 2^43): their sums are exact
// whatever their order, so the cut and the draw do not depend on how a row is split over threads
// and no atomic's order shows. A token is lost only below 2^-44 of the largest weight, and 2^19
// tokens of weight one stay below 2^63. The exponential is a polynomial in f64, off by 2^-44 at
// most: with f32's 2^-22 the running sum would pass the random number at another token in one of
// a few hundred rows, since a row has as many borders as tokens.
//
// A team of threads (a warp, a block, or a cluster of blocks) holds one row in shared memory:
//  1. load, largest and smallest logit;
//  2. with top-k or top-p, the cut: a histogram over the range that can matter (31 T below the
//     top: weights below are zero), linear in the logit, of counts or of weights; the bin in which
//     the running sum passes what is asked; its tokens, if few, ranked against each other, else a
//     histogram of that bin, and so on;
//  3. each thread the sum over a run of consecutive indices, a scan of those sums, and the run that
//     the random number falls in searched by a warp.

#include "pk_ops.cuh"

#include <algorithm>
#include <cooperative_groups.h>
#include <math_constants.h>

namespace pk {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr double kOne = 8796093022208.0;   // 2^43
constexpr float kMaxF = 3.402823466e+38f;
constexpr int kList = 128;                 // tokens that are ranked against each other
constexpr int kMaxCluster = 8;

// 2^x * 2^43 rounded to an integer, for -50 <= x <= 0: x = n + r with |r| <= 1/2, 2^r = 1 + r q(r),
// q interpolating (2^r - 1) / r at the nine Chebyshev nodes of [-1/2, 1/2] (relative error of 2^r
// below 2^-44.6; exactly 1 at r = 0). `x` comes as d * c, reduced with fused products.
__device__ __forceinline__ u64 exp2_fixed(double d, double c) {
    const double magic = 6755399441055744.0;            // 1.5 * 2^52: the sum's low word is round(x)
    const double y = fma(d, c, magic);
    const double r = fma(d, c, magic - y);
    double q = 1.0203121045191294e-07;
    q = fma(q, r, 1.3255224877814737e-06);
    q = fma(q, r, 1.5252686846287112e-05);
    q = fma(q, r, 0.00015403455852457495);
    q = fma(q, r, 0.0013333558179043266);
    q = fma(q, r, 0.009618129159402555);
    q = fma(q, r, 0.055504108664760424);
    q = fma(q, r, 0.2402265069581299);
    q = fma(q, r, 0.6931471805599453);
    q = fma(q, r, 1.0);
    const double w = __hiloint2double(__double2hiint(q) + ((__double2loint(y) + 43) << 20), __double2loint(q));
    return (u64) __double_as_longlong(w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // 2^52 holds the integer
}

struct Row {
    double top;       // largest logit; the largest number in a row that holds +infinity
    double c;         // log2(e) / T
    float base;       // logits below have weight zero
};

__device__ __forceinline__ u64 weight(float v, const Row & r) {
    return v >= r.base ? exp2_fixed((double) fminf(v, kMaxF) - r.top, r.c) : 0ull;
}

template <class V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

struct Pair { float v; int i; };

// What the blocks of a cluster tell each other, in each one's shared memory.
struct Xchg {
    u64 a;
    u64 b;
    float hi, lo;
};

template <int NT> constexpr int bins_of() { return NT == 32 ? 256 : 1024; }

template <int NT>
struct TeamSmem {
    u64 wscan[NT / 32 + 1];
    u64 found_before;
    Xchg x[2];
    float whi[NT / 32], wlo[NT / 32];
    int found_thread, found_ties;
    int listed;                              // tokens put on the list
    float cut;
    u64 cut_ties;
};
template <int NT>
struct TeamBins {
    unsigned lo[bins_of<NT>()], hi[bins_of<NT>()];     // sums of weights, or counts in lo
    Pair list[kList];
    Pair all[kList];
};

// The threads of one row. CL: several blocks of a cluster, each with a slice of the row.
template <int NT, bool CL>
struct Team {
    int tid, rank, blocks;
    unsigned phase = 0;
    TeamSmem<NT> * s;

    __device__ __forceinline__ void sync() const {
        if (NT == 32) __syncwarp(); else __syncthreads();
    }
    // Every block's slot written before it is complete; the other slot is free again after it.
    __device__ __forceinline__ void meet() { cg::this_cluster().sync(); }

    __device__ u64 block_sum(u64 v) {
        v = warp_sum(v);
        if (NT == 32) return v;
        sync();
        if ((tid & 31) == 0) s->wscan[tid >> 5] = v;
        sync();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) t += s->wscan[i];
        return t;
    }
    __device__ u64 sum(u64 v) {
        u64 t = block_sum(v);
        if (CL) {
            Xchg & x = s->x[phase];
            if (tid == 0) x.a = t;
            meet();
            t = 0;
            for (int b = 0; b < blocks; ++b) t += cg::this_cluster().map_shared_rank(&x, b)->a;
            phase ^= 1;
        }
        return t;
    }
    // Sum over the threads before this one (blocks before included); the sum of all in `total`.
    __device__ u64 scan(u64 v, u64 & total) {
        u64 x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xFFFFFFFFu, x, o);
            if ((tid & 31) >= o) x += y;
        }
        u64 before = x - v, t;
        if (NT == 32) {
            t = __shfl_sync(0xFFFFFFFFu, x, 31);
        } else {
            sync();
            if ((tid & 31) == 31) s->wscan[tid >> 5] = x;
            sync();
            t = 0;
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) {
                if (i < (tid >> 5)) before += s->wscan[i];
                t += s->wscan[i];
            }
        }
        if (CL) {
            Xchg & x2 = s->x[phase];
            if (tid == 0) x2.a = t;
            meet();
            t = 0;
            for (int b = 0; b < blocks; ++b) {
                const u64 o = cg::this_cluster().map_shared_rank(&x2, b)->a;
                if (b < rank) before += o;
                t += o;
            }
            phase ^= 1;
        }
        total = t;
        return before;
    }
    // Largest of hi, smallest of lo, over the team.
    __device__ void range(float & hi, float & lo) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
            lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        }
        if (NT > 32) {
            sync();
            if ((tid & 31) == 0) { s->whi[tid >> 5] = hi; s->wlo[tid >> 5] = lo; }
            sync();
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) { hi = fmaxf(hi, s->whi[i]); lo = fminf(lo, s->wlo[i]); }
        }
        if (CL) {
            Xchg & x = s->x[phase];
            if (tid == 0) { x.hi = hi; x.lo = lo; }
            meet();
            for (int b = 0; b < blocks; ++b) {
                const Xchg * o = cg::this_cluster().map_shared_rank(&x, b);
                hi = fmaxf(hi, o->hi);
                lo = fminf(lo, o->lo);
            }
            phase ^= 1;
        }
    }
};

// The slice of a row that this block holds: shared memory, or the logits themselves where a slice
// is larger than that.
template <class T>
struct Slice {
    const float * sm;
    const T * gl;
    int n;
    __device__ __forceinline__ float operator()(int i) const { return sm ? sm[i] : to_f32(gl[i]); }
};

template <class T, int NT>
__device__ __forceinline__ void load_slice(const T * __restrict__ g, int n, float * sm, int tid) {
    constexpr int W = 16 / (int) sizeof(T);
    const int head = min(n, (int) ((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / (int) sizeof(T));
    const int vecs = (n - head) / W;
    // sm is placed so that its element `head` is 16-byte aligned
    if constexpr (sizeof(T) == 4) {
        for (int i = tid; i < vecs; i += NT) {
            const unsigned d = (unsigned) __cvta_generic_to_shared(sm + head + i * 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(d), "l"(g + head + i * 4) : "memory");
        }
        for (int i = tid; i < head; i += NT) sm[i] = to_f32(g[i]);
        for (int i = head + vecs * W + tid; i < n; i += NT) sm[i] = to_f32(g[i]);
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
#pragma unroll 4
        for (int i = tid; i < vecs; i += NT) {
            const uint4 q = *reinterpret_cast<const uint4 *>(g + head + i * W);
            const unsigned w[4] = {q.x, q.y, q.z, q.w};
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                T e[2];
                *reinterpret_cast<unsigned *>(e) = w[j];
                f[2 * j] = to_f32(e[0]);
                f[2 * j + 1] = to_f32(e[1]);
            }
            float4 * d = reinterpret_cast<float4 *>(sm + head + i * W);
            d[0] = make_float4(f[0], f[1], f[2], f[3]);
            d[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
        for (int i = tid; i < head; i += NT) sm[i] = to_f32(g[i]);
        for (int i = head + vecs * W + tid; i < n; i += NT) sm[i] = to_f32(g[i]);
    }
}

// The cut at which the running sum over falling logits reaches `need` >= 1, among logits of
// [lo, hi], which hold that much: counts of tokens, or (WEIGHTS) their weights. Everything above the
// returned logit is kept, and `ties` of those equal to it.
template <bool WEIGHTS, class T, int NT, bool CL>
__device__ float find_cut(Team<NT, CL> & team, TeamBins<NT> * B, const Slice<T> & l, const Row & row, float hi, float lo, u64 need,
                          u64 & ties) {
    constexpr int NB = bins_of<NT>(), PER = NB / NT;
    TeamSmem<NT> * s = team.s;
    u64 above = 0;
    for (;;) {
        if (!(hi > lo)) {                       // one value left
            const u64 each = WEIGHTS ? weight(hi, row) : 1ull;
            ties = (need - above + each - 1) / max(each, 1ull);
            return hi;
        }
        for (int b = team.tid; b < NB; b += NT) { B->lo[b] = 0; if (WEIGHTS) B->hi[b] = 0; }
        if (team.tid == 0) { s->listed = 0; }
        team.sync();
        // Falling logits in rising bins: each operation is monotone, `hi` falls in bin 0 and `lo` in the
        // last (0 * inf, a NaN, is 0 as an integer), so every level parts the two and takes a range
        // 1 / NB as wide: 28 levels for NB = 1024 at the very most. Halves where the difference could
        // overflow; not otherwise, since half of the smallest number is zero.
        const float half = fmaxf(fabsf(hi), fabsf(lo)) > 1e37f ? 0.5f : 1.0f;
        const float top = half * hi, inv = (float) NB / (top - half * lo);
        auto bin_of = [&](float v) { return min(NB - 1, (int) ((top - half * v) * inv)); };
        for (int i = team.tid; i < l.n; i += NT) {
            const float v = l(i);
            if (v <= hi && v >= lo) {
                const int b = bin_of(v);
                if (WEIGHTS) {
                    const u64 w = weight(v, row);
                    const unsigned wl = (unsigned) w, old = atomicAdd(&B->lo[b], wl);
                    const unsigned up = (unsigned) (w >> 32) + (old + wl < old ? 1u : 0u);
                    if (up) atomicAdd(&B->hi[b], up);
                } else {
                    atomicAdd(&B->lo[b], 1u);
                }
            }
        }
        if (CL) team.meet();
        team.sync();
        // each thread PER consecutive bins
        u64 mine[PER], sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int b = team.tid * PER + j;
            u64 w = 0;
            if (CL) {
                for (int q = 0; q < team.blocks; ++q) {
                    const TeamBins<NT> * o = cg::this_cluster().map_shared_rank(B, q);
                    w += (WEIGHTS ? (u64) o->hi[b] << 32 : 0ull) + o->lo[b];
                }
            } else {
                w = (WEIGHTS ? (u64) B->hi[b] << 32 : 0ull) + B->lo[b];
            }
            mine[j] = w;
            sum += w;
        }
        // the scan over this block's threads alone: the bins are the cluster's already
        u64 total;
        Team<NT, false> block{team.tid, 0, 1, 0, s};
        u64 before = above + block.scan(sum, total);
        if (before < need && need <= before + sum) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (before < need && need <= before + mine[j]) {
                    s->found_thread = team.tid * PER + j;
                    s->found_before = before;
                }
                before += mine[j];
            }
        }
        team.sync();
        const int bin = s->found_thread;
        above = s->found_before;
        // the tokens of that bin: listed if they fit, and their range
        float bhi = -CUDART_INF_F, blo = CUDART_INF_F;
        for (int i = team.tid; i < l.n; i += NT) {
            const float v = l(i);
            if (v <= hi && v >= lo && bin_of(v) == bin) {
                bhi = fmaxf(bhi, v);
                blo = fminf(blo, v);
                const int at = atomicAdd(&s->listed, 1);
                if (at < kList) B->list[at] = Pair{v, i};
            }
        }
        team.range(bhi, blo);
        team.sync();
        hi = bhi;
        lo = blo;
        int n = s->listed;
        const Pair * list = B->list;
        team.sync();                            // read by all before it is set back
        if (CL) {
            Xchg & x = s->x[team.phase];
            if (team.tid == 0) x.a = (u64) n;
            team.meet();
            int base = 0;
            n = 0;
            for (int q = 0; q < team.blocks; ++q) n += (int) cg::this_cluster().map_shared_rank(&x, q)->a;
            if (n <= kList) {
                for (int q = 0; q < team.blocks; ++q) {
                    const int c = (int) cg::this_cluster().map_shared_rank(&x, q)->a;
                    const TeamBins<NT> * o = cg::this_cluster().map_shared_rank(B, q);
                    for (int i = team.tid; i < c; i += NT) B->all[base + i] = o->list[i];
                    base += c;
                }
                list = B->all;
            }
            team.phase ^= 1;
            team.meet();                        // nobody lists anew while another still reads
            team.sync();
        }
        if (n <= kList) {
            for (int j = team.tid; j < n; j += NT) {
                const float v = list[j].v;
                u64 over = above, same = 0;
                for (int i = 0; i < n; ++i) {
                    const float o = list[i].v;
                    const u64 w = WEIGHTS ? (o >= v ? weight(o, row) : 0ull) : 1ull;
                    if (o > v) over += w;
                    else if (o == v) same += w;
                }
                if (over < need && need <= over + same) {
                    const u64 each = WEIGHTS ? weight(v, row) : 1ull;
                    s->cut = v;
                    s->cut_ties = (need - over + each - 1) / each;
                }
            }
            team.sync();
            ties = s->cut_ties;
            const float v = s->cut;
            team.sync();
            return v;
        }
    }
}

template <class T, int NT, bool FILTERS, bool CL>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT)
sample_kernel(pk_sample_args a, int slice, int teams, int row_floats) {
    extern __shared__ __align__(16) unsigned char raw[];
    const int t_in = NT == 32 ? (int) threadIdx.x >> 5 : 0;      // team within the block
    Team<NT, CL> team;
    team.tid = NT == 32 ? (int) threadIdx.x & 31 : (int) threadIdx.x;
    team.blocks = CL ? (int) cg::this_cluster().num_blocks() : 1;
    team.rank = CL ? (int) cg::this_cluster().block_rank() : 0;
    team.s = reinterpret_cast<TeamSmem<NT> *>(raw) + t_in;
    TeamBins<NT> * bins = reinterpret_cast<TeamBins<NT> *>(reinterpret_cast<TeamSmem<NT> *>(raw) + teams) + t_in;
    float * rows_at = FILTERS ? reinterpret_cast<float *>(reinterpret_cast<TeamBins<NT> *>(reinterpret_cast<TeamSmem<NT> *>(raw) + teams) + teams)
                              : reinterpret_cast<float *>(reinterpret_cast<TeamSmem<NT> *>(raw) + teams);
    rows_at = reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(rows_at) + 15) & ~(uintptr_t) 15) + (size_t) t_in * row_floats;
    const long long row = CL ? (long long) (blockIdx.x / team.blocks) : (long long) blockIdx.x * teams + t_in;
    if (NT == 32 && row >= a.rows) return;                       // warps by themselves: nothing to meet
    const int s0 = min(team.rank * slice, a.vocab);
    Slice<T> l;
    l.n = min(slice, a.vocab - s0);
    l.gl = static_cast<const T *>(a.logits) + row * a.row_stride + s0;
    l.sm = nullptr;
    if (row_floats > 0) {
        // element i in the slice at the same place of its 16 bytes (in f32) as the logits have
        const int skew = (int) ((reinterpret_cast<uintptr_t>(l.gl) & 15) / sizeof(T)) & 3;
        float * sm = rows_at + skew;
        load_slice<T, NT>(l.gl, l.n, sm, team.tid);
        team.sync();
        l.sm = sm;
    }
    float hi = -CUDART_INF_F, lo = CUDART_INF_F;                 // fmaxf and fminf pass over NaN
    for (int i = team.tid; i < l.n; i += NT) {
        const float v = l(i);
        hi = fmaxf(hi, v);
        if (v > -CUDART_INF_F) lo = fminf(lo, v);
    }
    team.range(hi, lo);
    const bool writer = team.tid == 0 && team.rank == 0;
    const float temp = a.temperatures ? a.temperatures[row] : a.temperature;
    if (hi == -CUDART_INF_F || !(temp > 0.0f)) {
        // nothing to draw, or the first index of the largest
        u64 first = ~0ull;
        if (hi > -CUDART_INF_F)
            for (int i = team.tid; i < l.n && first == ~0ull; i += NT)
                if (l(i) == hi) first = (u64) (s0 + i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xFFFFFFFFu, first, o));
        if (NT > 32) {
            team.sync();
            if ((team.tid & 31) == 0) team.s->wscan[team.tid >> 5] = first;
            team.sync();
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) first = min(first, team.s->wscan[i]);
        }
        if (CL) {
            Xchg & x = team.s->x[team.phase];
            if (team.tid == 0) x.a = first;
            team.meet();
            for (int b = 0; b < team.blocks; ++b) first = min(first, cg::this_cluster().map_shared_rank(&x, b)->a);
            team.meet();
        }
        if (writer) {
            a.tokens[row] = hi == -CUDART_INF_F ? -1 : (int) first;
            if (a.logprobs) a.logprobs[row] = hi == -CUDART_INF_F ? -CUDART_INF_F : 0.0f;
        }
        return;
    }
    Row r;
    const bool inf = hi == CUDART_INF_F;
    r.top = (double) fminf(hi, kMaxF);
    r.c = 1.4426950408889634074 / (double) temp;                 // 0 for an infinite T
    // below 2^-44 of the largest: 31 T is more than 44 ln 2 = 30.5 T; rounded up, so that what is
    // not below lies within the exponential's range
    r.base = inf ? hi : fmaxf(__double2float_ru(r.top - 31.0 * (double) temp), -kMaxF);
    float least = r.base;                                        // kept: >= least, and what the cut says
    float cut = -CUDART_INF_F;
    u64 ties = ~0ull;
    if (FILTERS) {
        const float m = a.min_ps ? a.min_ps[row] : a.min_p;
        const float p = a.top_ps ? a.top_ps[row] : a.top_p;
        const int k = a.top_ks ? a.top_ks[row] : a.top_k;
        if (m >= 1.0f) least = hi;
        else if (m > 0.0f && !inf) least = fmaxf(least, __double2float_ru(r.top + (double) temp * log((double) m)));
        const float low = fmaxf(r.base, lo);                     // the range that can have weight
        if (k > 0 && k < a.vocab) {
            u64 n = 0;
            for (int i = team.tid; i < l.n; i += NT) n += l(i) >= low ? 1u : 0u;
            if (team.sum(n) > (u64) k) cut = find_cut<false>(team, bins, l, r, hi, low, (u64) k, ties);
        }
        if (!(p >= 1.0f)) {
            u64 w = 0;
            for (int i = team.tid; i < l.n; i += NT) {
                const float v = l(i);
                if (v > cut) w += weight(v, r);
            }
            w = team.sum(w);
            const u64 at_cut = cut > -CUDART_INF_F ? weight(cut, r) * ties : 0ull;
            const u64 need = max((u64) ceil(p > 0.0f ? (double) p * (double) (w + at_cut) : 0.0), 1ull);
            if (need > w) {
                // the cut stays, with fewer ties
                if (cut > -CUDART_INF_F) ties = min(ties, (need - w + weight(cut, r) - 1) / max(weight(cut, r), 1ull));
            } else {
                // above the cut of k: from the next number on
                float from = low;
                if (cut > -CUDART_INF_F) {
                    const float up = cut == 0.0f ? 1.401298464e-45f
                                                 : __int_as_float(__float_as_int(cut) + (cut > 0.0f ? 1 : -1));
                    from = fmaxf(low, up);
                }
                cut = find_cut<true>(team, bins, l, r, hi, from, need, ties);
            }
        }
    }
    // runs of consecutive indices; an odd length keeps their first elements in different banks
    const int len = ((l.n + NT - 1) / NT) | 1;
    const int i0 = min(team.tid * len, l.n), i1 = min(i0 + len, l.n);
    // equal logits at the cut, where not all of them are kept, go by index
    u64 tie0 = 0;
    bool partial = false;
    if (FILTERS && cut > -CUDART_INF_F) {
        u64 n = 0, all = 0;
        for (int i = i0; i < i1; ++i) n += l(i) == cut ? 1u : 0u;
        tie0 = team.scan(n, all);
        partial = ties < all;
    }
    u64 sum = 0, seen = tie0;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
        const float v = l(i);
        if (v >= least) {
            if (FILTERS) {
                bool keep = v >= cut;
                if (partial && v == cut) keep = seen++ < ties;
                if (keep) sum += weight(v, r);
            } else {
                sum += weight(v, r);
            }
        }
    }
    u64 total = 0;
    const u64 before = team.scan(sum, total);
    float u = a.uniforms[row];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    const u64 t = min((u64) ((double) u * (double) total), total - 1);
    if (team.tid == 0) team.s->found_thread = -1;
    team.sync();
    if (before <= t && t < before + sum) {
        team.s->found_thread = team.tid;
        team.s->found_before = before;
        team.s->found_ties = (int) min(tie0, (u64) 0x7FFFFFFF);
    }
    team.sync();
    const int who = team.s->found_thread;
    if (who >= 0 && team.tid < 32) {
        u64 run = team.s->found_before;
        u64 tie = (u64) team.s->found_ties;
        const int b = who * len, e = min(b + len, l.n);
        for (int c = b; c < e; c += 32) {
            const int i = c + team.tid;
            const float v = i < e ? l(i) : -CUDART_INF_F;
            u64 w = 0;
            if (v >= least && v >= cut) w = weight(v, r);
            if (FILTERS && partial) {
                const unsigned eq = __ballot_sync(0xFFFFFFFFu, i < e && v == cut);
                if (v == cut && tie + __popc(eq & ((1u << team.tid) - 1u)) >= ties) w = 0;
                tie += __popc(eq);
            }
            u64 x = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (team.tid >= o) x += y;
            }
            if (w > 0 && run + x - w <= t && t < run + x) {
                a.tokens[row] = s0 + i;
                if (a.logprobs) {
                    const double scaled = v == hi ? 0.0 : ((double) v - (double) hi) / (double) temp;
                    a.logprobs[row] = (float) (scaled - log((double) total / kOne));
                }
            }
            run += __shfl_sync(0xFFFFFFFFu, x, 31);
        }
    }
    if (CL) team.meet();                                         // a block's memory stays while others may read it
}

constexpr size_t kSmemCap = 220 * 1024;

template <class T, int NT, bool FILTERS, bool CL>
cudaError_t launch(const pk_sample_args & a, int blocks, cudaStream_t s) {
    const int teams = NT == 32 ? 8 : 1;
    // slices of whole 16 bytes, so that every slice is aligned as its row is
    const int slice = CL ? ((a.vocab + blocks - 1) / blocks + 31) / 32 * 32 : a.vocab;
    const size_t fixed = teams * (sizeof(TeamSmem<NT>) + (FILTERS ? sizeof(TeamBins<NT>) : 0)) + 16;
    int row_floats = (slice + 4 + 3) / 4 * 4;
    size_t smem = fixed + (size_t) teams * row_floats * 4;
    if (smem > kSmemCap) {                                       // read from the logits each time
        row_floats = 0;
        smem = fixed;
    }
    auto kernel = sample_kernel<T, NT, FILTERS, CL>;
    static unsigned long long set;                               // devices on which the limit is raised
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (!(__atomic_load_n(&set, __ATOMIC_RELAXED) >> device & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) kSmemCap);
        if (e != cudaSuccess) return e;
        __atomic_fetch_or(&set, 1ull << device, __ATOMIC_RELAXED);
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.gridDim = dim3((unsigned) (CL ? a.rows * blocks : (a.rows + teams - 1) / teams));
    cfg.blockDim = dim3(NT == 32 ? 256 : NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    if (CL) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned) blocks;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, a, slice, teams, row_floats);
}

template <class T, bool FILTERS>
cudaError_t dispatch(const pk_sample_args & a, cudaStream_t s) {
    if (a.vocab <= 1280 && a.rows >= 512) return launch<T, 32, FILTERS, false>(a, 1, s);
    if (a.vocab <= 2048) return launch<T, 128, FILTERS, false>(a, 1, s);
    int blocks = 1;
    while (blocks < kMaxCluster && a.rows * blocks * 2 <= 148 && a.vocab / (blocks * 2) >= 1024) blocks *= 2;
    while (blocks < kMaxCluster && (size_t) (a.vocab / blocks) * 4 > 200 * 1024) blocks *= 2;
    if (blocks > 1) return launch<T, 512, FILTERS, true>(a, blocks, s);
    return launch<T, 512, FILTERS, false>(a, 1, s);
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
    cudaStream_t s = (cudaStream_t) stream;
    // nothing to cut: neither an array of settings nor a setting that cuts
    const bool filters = a->top_ks || a->top_ps || a->min_ps || (a->top_k > 0 && a->top_k < a->vocab) || !(a->top_p >= 1.0f) ||
                         a->min_p > 0.0f;
    cudaError_t e;
#define PK_S(T) e = filters ? dispatch<T, true>(*a, s) : dispatch<T, false>(*a, s)
    if (a->logits_type == PK_GGML_F32) PK_S(float);
    else if (a->logits_type == PK_GGML_F16) PK_S(__half);
    else PK_S(__nv_bfloat16);
#undef PK_S
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}
