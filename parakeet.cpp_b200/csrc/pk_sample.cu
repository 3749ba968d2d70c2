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
// tokens of weight one stay below 2^63. The exponential is taken in f64, to 2^-42 of itself: with
// f32's 2^-22 the running sum would pass the random number at another token in one of a few hundred
// rows, since a row has as many borders as tokens.
//
// Rows of up to 2048 logits with nothing cut, as a CTC path has them by the ten thousand, are summed in
// f32 first: four instructions a token for weight and sum instead of twenty. That settles the token unless
// the random number lies within a proven bound of a border (one or two rows in a hundred), and those rows go
// on to the f64 sums, so the token is the same; the log-probability then has f32's sum, 2^-18 off at most
// (see draw_f32). 66044 rows of 1025 take 67 us replayed from a graph, 865 warp instructions a row, 26 for
// every 32 logits: most of them stage the row, find its maximum and scan.
//
// A team of threads (a warp, a block, or a cluster of blocks) holds one row in shared memory:
//  1. load, largest and smallest logit;
//  2. with top-k or top-p, a histogram over the range that can matter, linear in the logit, of
//     counts or of weights, and the bin in which the running sum reaches what is asked. If few
//     tokens lie in that bin and above, they are listed, ranked against each other, cut and drawn
//     from: done. Else the cut is found inside the bin: its tokens ranked if few, or a histogram of
//     that bin alone, and so on;
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
constexpr int kList = 128;                 // tokens that are ranked against each other
constexpr int kMaxCluster = 8;
constexpr unsigned kFull = 0xFFFFFFFFu;

// 2^(j / 32), j = 0 .. 31, the first with its last bit set (see weight_onto).
__device__ const double kExp2[32] = {
    0x1.0000000000001p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

struct Row {
    double top;       // largest logit
    double c;         // 32 log2(e) / T
    float base;       // logits below have weight zero (and lie outside the exponential's range)
};

// Weight of a logit v >= base. 2^x * 2^43 for x = (v - top) c / 32 >= -45: 32 x = n + t, n whole,
// |t| <= 1/2; 2^(n / 32) from the table's entry n % 32 and n / 32 added to its exponent, 2^(t / 32)
// = 1 + t q(t) with q cubic, interpolating at the four Chebyshev nodes of [-1/2, 1/2] (off by
// 2^-42.5 at most; exactly 1 at t = 0). Adding a number of [2^52, 2^53) rounds the product to an
// integer in the low bits. A product halfway between two integers would go to the one that makes the
// sum so far even, and sums would depend on their order. None is halfway: a table entry's lowest bit is at
// 2^-46 or below (1 is held as 1 + 2^-52 for that), the polynomial's at 2^0 or below, so that of their
// product times 2^43 is at 2^-3 or below; 1 still rounds to 2^43. `entry(n)` gives 2^43 * table[n % 32] with n % 32 taken off the exponent
// field's place 15 bits up, where all of n is added. All callers share these operations.
template <class F>
__device__ __forceinline__ double weight_onto(float v, const Row & r, double onto, F entry) {
    const double magic = 6755399441055744.0;            // 1.5 * 2^52: the sum's low word is the nearest integer
    const double d = (double) v - r.top;
    const double y = fma(d, r.c, magic);
    const double t = fma(d, r.c, magic - y);
    double q = 9.172598566078425e-09;
    q = fma(q, t, 1.6938609067364243e-06);
    q = fma(q, t, 0.00023459619820112603);
    q = fma(q, t, 0.021660849392187844);
    q = fma(q, t, 1.0);
    const int n = __double2loint(y);
    const double e = entry(n);
    return fma(q, __hiloint2double(__double2hiint(e) + (n << 15), __double2loint(e)), onto);
}
constexpr double kZero = 4503599627370496.0;             // 2^52
__device__ __forceinline__ u64 whole(double onto) { return (u64) __double_as_longlong(onto) - 0x4330000000000000ull; }
__device__ __forceinline__ double table_entry(int j) {
    const double e = kExp2[j] * kOne;
    return __hiloint2double(__double2hiint(e) - (j << 15), __double2loint(e));
}
// The table across a warp's lanes: every lane calls, and drops what it gets for v < base. A shuffle
// takes n modulo 32.
__device__ __forceinline__ double weight_warp(float v, const Row & r, double mine, double onto = kZero) {
    return weight_onto(v, r, onto, [&](int n) { return __shfl_sync(kFull, mine, n); });
}
// Any thread by itself.
__device__ __forceinline__ u64 weight_one(float v, const Row & r) {
    return v >= r.base ? whole(weight_onto(v, r, kZero, [](int n) { return table_entry(n & 31); })) : 0ull;
}

template <class V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
template <class V> __device__ __forceinline__ V warp_scan(V x, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

struct Pair { float v; int i; };

// What the blocks of a cluster tell each other, in each one's shared memory.
struct Xchg {
    u64 a;
    float hi, lo;
};

template <int NT> constexpr int bins_of() { return NT == 32 ? 256 : 1024; }

template <int NT> constexpr int sets_of() { return NT == 1024 ? 2 : 1; }   // clusters are of 1024 threads

template <int NT>
struct TeamSmem {
    u64 wscan[NT / 32 + 1];
    u64 found_before, found_sum;
    Xchg x[2];
    float whi[NT / 32], wlo[NT / 32];
    int found, found_ties;
    int listed;                              // tokens put on the list
    float cut;
    int cut_partial;
    u64 cut_ties;
};
template <int NT>
struct TeamBins {
    // sums of weights, in two halves, or counts in x; in a cluster levels take turns with two sets, so that
    // one may be cleared while other blocks still read the other
    uint2 sum[sets_of<NT>()][bins_of<NT>()];
    Pair list[kList];
    Pair all[kList];                                   // of all blocks of a cluster
    u64 w[kList];
};

// The threads of one row. CL: several blocks of a cluster, each with a slice of the row.
template <int NT, bool CL>
struct Team {
    int tid, rank, blocks;
    unsigned phase;
    TeamSmem<NT> * s;
    double mine;                             // this lane's entry of the exponential's table
    unsigned level = 0;                      // levels of bins so far

    __device__ __forceinline__ int lane() const { return tid & 31; }
    __device__ __forceinline__ void sync() const {
        if (NT == 32) __syncwarp(); else __syncthreads();
    }
    // Every block's slot written before it is complete, what was read before it may be overwritten.
    __device__ __forceinline__ void meet() const { cg::this_cluster().sync(); }

    // All blocks' slots, asked for before the first is used: f(block, slot) in turn.
    template <class F> __device__ __forceinline__ void hear(const Xchg & mine, F f) const {
        Xchg o[kMaxCluster];
#pragma unroll
        for (int b = 0; b < kMaxCluster; ++b) o[b] = *cg::this_cluster().map_shared_rank(const_cast<Xchg *>(&mine), b < blocks ? b : 0);
#pragma unroll
        for (int b = 0; b < kMaxCluster; ++b)
            if (b < blocks) f(b, o[b]);
    }

    __device__ u64 sum(u64 v) {
        v = warp_sum(v);
        if (NT > 32) {
            sync();
            if (lane() == 0) s->wscan[tid >> 5] = v;
            sync();
            v = s->wscan[lane() & (NT / 32 - 1)];
#pragma unroll
            for (int o = NT / 64; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        }
        if (CL) {
            Xchg & x = s->x[phase];
            if (tid == 0) x.a = v;
            meet();
            v = 0;
            hear(x, [&](int, const Xchg & o) { v += o.a; });
            phase ^= 1;
        }
        return v;
    }
    // Sum over the threads before this one (blocks before included); the sum of all in `total`.
    __device__ u64 scan(u64 v, u64 & total) {
        const u64 x = warp_scan(v, lane());
        u64 before = x - v, t;
        if (NT == 32) {
            t = __shfl_sync(kFull, x, 31);
        } else {
            sync();
            if (lane() == 31) s->wscan[tid >> 5] = x;
            sync();
            u64 w = s->wscan[lane() & (NT / 32 - 1)];
#pragma unroll
            for (int o = 1; o < NT / 32; o <<= 1) {
                const u64 y = __shfl_up_sync(kFull, w, o, NT / 32);
                if ((lane() & (NT / 32 - 1)) >= o) w += y;
            }
            t = __shfl_sync(kFull, w, NT / 32 - 1);
            w = __shfl_sync(kFull, w, max((tid >> 5) - 1, 0));
            if (tid >= 32) before += w;
        }
        if (CL) {
            Xchg & o = s->x[phase];
            if (tid == 0) o.a = t;
            meet();
            t = 0;
            hear(o, [&](int b, const Xchg & w) {
                if (b < rank) before += w.a;
                t += w.a;
            });
            phase ^= 1;
        }
        total = t;
        return before;
    }
    // Largest of hi, smallest of lo, over the block, over the team.
    template <bool LO = true>
    __device__ __forceinline__ void block_range(float & hi, float & lo) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
            if (LO) lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
        }
        if (NT > 32) {
            sync();
            if (lane() == 0) { s->whi[tid >> 5] = hi; s->wlo[tid >> 5] = lo; }
            sync();
            hi = s->whi[lane() & (NT / 32 - 1)];
            lo = s->wlo[lane() & (NT / 32 - 1)];
#pragma unroll
            for (int o = NT / 64; o > 0; o >>= 1) {
                hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
                lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
            }
        }
    }
    template <bool LO = true>
    __device__ __forceinline__ void range(float & hi, float & lo) {
        block_range<LO>(hi, lo);
        if (CL) {
            Xchg & x = s->x[phase];
            if (tid == 0) { x.hi = hi; x.lo = lo; }
            meet();
            hear(x, [&](int, const Xchg & o) {
                hi = fmaxf(hi, o.hi);
                lo = fminf(lo, o.lo);
            });
            phase ^= 1;
        }
    }
};

// Consecutive elements of a thread: an odd number, whose first ones lie in different banks.
template <int NT> __host__ __device__ __forceinline__ int run_of(int n) { return ((n + NT - 1) / NT) | 1; }

// The slice of a row that this block holds. RES: in shared memory, `skew` elements after a 16-byte
// boundary, as in global memory, -infinity before it and after it up to `pad` elements: whole 16 bytes
// and whole runs. Otherwise, for slices larger than that, the logits are read again and again. `inf`: the row's maximum is
// +infinity, whose logits count as 0 and all others as -infinity.
template <class T, bool RES>
struct Slice {
    float * sm;
    const T * gl;
    int n, skew, pad;
    bool inf;
    __device__ __forceinline__ float operator()(int i) const {
        if (RES) return sm[skew + i];
        const float v = to_f32(gl[i]);
        return inf ? (v == CUDART_INF_F ? 0.0f : -CUDART_INF_F) : v;
    }
    // f(four values, index of the first in the slice) over all quads, -infinities around the slice's
    // elements, a whole warp at a time
    template <int NT, class F>
    __device__ __forceinline__ void quads(int tid, F f) const {
        const int n4 = RES ? (skew + n + 3) >> 2 : (n + 3) >> 2;
#pragma unroll 2
        for (int q = tid & ~31; q < n4; q += NT) {
            const int i = q + (tid & 31);
            float4 v = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
            if constexpr (RES) {
                if (i < n4) v = reinterpret_cast<const float4 *>(sm)[i];
            } else {
                if (4 * i < n) v.x = (*this)(4 * i);
                if (4 * i + 1 < n) v.y = (*this)(4 * i + 1);
                if (4 * i + 2 < n) v.z = (*this)(4 * i + 2);
                if (4 * i + 3 < n) v.w = (*this)(4 * i + 3);
            }
            f(v, 4 * i - (RES ? skew : 0));
        }
    }
    // f(value, index in the slice), the same way
    template <int NT, class F>
    __device__ __forceinline__ void each(int tid, F f) const {
        quads<NT>(tid, [&](float4 v, int e) {
            f(v.x, e);
            f(v.y, e + 1);
            f(v.z, e + 2);
            f(v.w, e + 3);
        });
    }
};

template <class T, int NT>
__device__ __forceinline__ void load_slice(const Slice<T, true> & l, int tid) {
    constexpr int W = 16 / (int) sizeof(T);
    const T * g = l.gl;
    const int n = l.n;
    const int head = min(n, (int) ((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / (int) sizeof(T));
    const int vecs = (n - head) / W;
    float * sm = l.sm + l.skew;                          // its element `head` is 16-byte aligned
    if constexpr (sizeof(T) == 4) {
        for (int i = tid; i < vecs; i += NT) {
            const unsigned d = (unsigned) __cvta_generic_to_shared(sm + head + i * 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(d), "l"(g + head + i * 4) : "memory");
        }
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
    }
    if (tid < 16) {                                      // fewer than W at either end
        const int i = tid < 8 ? tid : head + vecs * W + tid - 8;
        if (tid < 8 ? i < head : i < n) sm[i] = to_f32(g[i]);
    }
    if (tid < l.skew) l.sm[tid] = -CUDART_INF_F;
    for (int i = n + tid; i < l.pad; i += NT) sm[i] = -CUDART_INF_F;
    if constexpr (sizeof(T) == 4) asm volatile("cp.async.wait_all;" ::: "memory");
}

// A range of logits parted evenly into bins. Bins rise as the logit falls: each operation of bin_of is
// monotone, `hi` lies in bin 0 and `lo` in the last (0 * inf, a NaN, is 0 as an integer), so a level
// parts the two and leaves a range 1 / NB as wide: 28 levels for NB = 1024 at the very most.
struct Level {
    float hi, lo, top, inv, half;
    int bin;
    u64 above, with;      // sums over what lies above the bin, and over that and the bin
    __device__ __forceinline__ void range(float h, float l, int nb) {
        hi = h;
        lo = l;
        // halves where the difference could overflow; not otherwise, since half of the smallest number is zero
        half = fmaxf(fabsf(h), fabsf(l)) > 1e37f ? 0.5f : 1.0f;
        top = half * h;
        inv = (float) nb / (top - half * l);
    }
    template <int NB> __device__ __forceinline__ int bin_of(float v) const { return min(NB - 1, (int) ((top - half * v) * inv)); }
    __device__ __forceinline__ bool holds(float v) const { return v <= hi && v >= lo; }
};

// What top-p asks for: a share of the weights of [from, hi] (those below the level's range are summed
// without a bin) and of `lump`.
struct Share {
    double p;
    float from;
    u64 lump;
};

// Bins the level's range and finds the bin in which the running sum over falling logits (from L.above
// on) reaches `need` >= 1: of counts, or (WEIGHTS) of weights. With `share`, need is worked out from
// it first. False: the range does not hold that much; L.with is then what it and its tail hold.
template <bool WEIGHTS, class T, int NT, bool CL, bool RES>
__device__ bool find_bin(Team<NT, CL> & team, TeamBins<NT> * B, const Slice<T, RES> & l, const Row & row, Level & L, u64 & need,
                         const Share * share) {
    constexpr int NB = bins_of<NT>(), PER = NB / NT;
    TeamSmem<NT> * s = team.s;
    const unsigned set = CL ? team.level++ & 1u : 0u;
    uint2 * bins = B->sum[set];
    for (int b = team.tid; b < NB; b += NT) {
        bins[b] = make_uint2(0, 0);
    }
    if (team.tid == 0) { s->found = -1; s->listed = 0; }
    team.sync();
    u64 rest = 0;
    const float from = share ? share->from : L.lo;
    l.template each<NT>(team.tid, [&](float v, int) {
        if (WEIGHTS) {
            const bool any = v <= L.hi && v >= from;
            if (!__any_sync(kFull, any)) return;
            const u64 w = whole(weight_warp(v, row, team.mine));
            if (any) {
                if (v >= L.lo) {
                    const int b = L.bin_of<NB>(v);
                    const unsigned wl = (unsigned) w, old = atomicAdd(&bins[b].x, wl);
                    const unsigned up = (unsigned) (w >> 32) + (old + wl < old ? 1u : 0u);
                    if (up) atomicAdd(&bins[b].y, up);
                } else {
                    rest += w;
                }
            }
        } else if (L.holds(v)) {
            atomicAdd(&bins[L.bin_of<NB>(v)].x, 1u);
        }
    });
    if (WEIGHTS && share) rest = team.sum(rest);                 // in a cluster, all bins are complete after it
    else if (CL) team.meet();
    team.sync();
    u64 mine[PER], sum = 0;                                      // PER consecutive bins a thread
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int b = team.tid * PER + j;
        u64 w = 0;
        if (CL) {
            // all blocks' words are asked for before the first is used
            uint2 r[kMaxCluster];
#pragma unroll
            for (int q = 0; q < kMaxCluster; ++q) r[q] = cg::this_cluster().map_shared_rank(B, q < team.blocks ? q : 0)->sum[set][b];
#pragma unroll
            for (int q = 0; q < kMaxCluster; ++q)
                if (q < team.blocks) w += ((u64) r[q].y << 32) + r[q].x;
        } else {
            w = ((u64) bins[b].y << 32) + bins[b].x;
        }
        mine[j] = w;
        sum += w;
    }
    u64 total;
    Team<NT, false> block{team.tid, 0, 1, 0, s, 0.0};            // the bins are the cluster's already
    u64 before = L.above + block.scan(sum, total);
    total += L.above + rest;
    if (WEIGHTS && share) need = max((u64) ceil(share->p * (double) (total + share->lump)), 1ull);
    if (before < need && need <= before + sum) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (before < need && need <= before + mine[j]) {
                s->found = team.tid * PER + j;
                s->found_before = before;
                s->found_sum = before + mine[j];
            }
            before += mine[j];
        }
    }
    team.sync();
    L.bin = s->found;
    if (L.bin < 0) {
        L.with = total;
        return false;
    }
    L.above = s->found_before;
    L.with = s->found_sum;
    return true;
}

// Puts the slice's elements that `want` names on the list, and joins the lists of a cluster's blocks.
// The number of them; past kList the list is not complete and not to be used. RANGE: also their largest
// and smallest value; with `few` false nothing is listed, as there are more than kList.
template <bool RANGE, class T, int NT, bool CL, bool RES, class F>
__device__ int gather(Team<NT, CL> & team, TeamBins<NT> * B, const Slice<T, RES> & l, int s0, const Pair *& list, F want, bool few,
                      float & hi, float & lo) {
    TeamSmem<NT> * s = team.s;
    if (RANGE) {
        hi = -CUDART_INF_F;
        lo = CUDART_INF_F;
    }
    l.template quads<NT>(team.tid, [&](float4 v, int i) {
        const bool a = want(v.x), b = want(v.y), c = want(v.z), d = want(v.w);
        if (!(a || b || c || d)) return;
        if (RANGE) {
            const float inf = CUDART_INF_F;
            hi = fmaxf(fmaxf(hi, fmaxf(a ? v.x : -inf, b ? v.y : -inf)), fmaxf(c ? v.z : -inf, d ? v.w : -inf));
            lo = fminf(fminf(lo, fminf(a ? v.x : inf, b ? v.y : inf)), fminf(c ? v.z : inf, d ? v.w : inf));
            if (!few) return;
        }
        int at = atomicAdd(&s->listed, (int) a + (int) b + (int) c + (int) d);
        if (a && at < kList) B->list[at] = Pair{v.x, s0 + i};
        at += a;
        if (b && at < kList) B->list[at] = Pair{v.y, s0 + i + 1};
        at += b;
        if (c && at < kList) B->list[at] = Pair{v.z, s0 + i + 2};
        at += c;
        if (d && at < kList) B->list[at] = Pair{v.w, s0 + i + 3};
    });
    team.sync();
    int n = few ? s->listed : kList + 1;
    list = B->list;
    if (RANGE && (CL || n > kList)) team.block_range(hi, lo);
    if (CL) {
        Xchg & x = s->x[team.phase];
        if (team.tid == 0) {
            x.a = (u64) n;
            x.hi = hi;
            x.lo = lo;
        }
        team.meet();
        n = 0;
        // entry tid of the joint list is entry tid - start of block `from`'s
        int from = 0, start = 0;
        team.hear(x, [&](int q, const Xchg & o) {
            if (n <= team.tid) {
                from = q;
                start = n;
            }
            n += (int) o.a;
            if (RANGE) {
                hi = fmaxf(hi, o.hi);
                lo = fminf(lo, o.lo);
            }
        });
        if (n <= kList) {
            if (team.tid < n) B->all[team.tid] = cg::this_cluster().map_shared_rank(B, from)->list[team.tid - start];
            list = B->all;
            team.phase ^= 1;
            team.meet();                        // nobody lists anew while another still reads
        } else {
            team.phase ^= 1;
        }
    }
    team.sync();
    if (team.tid == 0) s->listed = 0;           // read by all: the next list starts empty
    team.sync();
    return n;
}

// For each token of a list of n: f(token, sum of g(token, other token) over the list), a few
// neighbouring threads sharing a token's sum. Entries behind the list count for nothing.
template <int NT> constexpr int sharers() { return NT >= 8 * kList ? 8 : NT >= 4 * kList ? 4 : NT >= 2 * kList ? 2 : 1; }
template <int NT, class V, class G, class F>
__device__ __forceinline__ void over_list(int tid, int n, G g, F f) {
    constexpr int SH = sharers<NT>(), PER = (kList * SH + NT - 1) / NT;
    const int padded = min(kList, (n + 4 * SH - 1) / (4 * SH) * (4 * SH));
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int j = (tid + q * NT) / SH;
        V sum{};
#pragma unroll 4
        for (int i = tid % SH; i < padded; i += SH) g(sum, j, i);
#pragma unroll
        for (int o = 1; o < SH; o <<= 1) sum.add(sum.across(o));
        if (j < n && tid % SH == 0) f(j, sum, q);
    }
}
struct Rank {                                   // tokens before one in the order, and their weight
    u64 w = 0;
    int n = 0;
    __device__ __forceinline__ void add(const Rank & o) { w += o.w; n += o.n; }
    __device__ __forceinline__ Rank across(int o) const {
        Rank r;
        r.w = __shfl_xor_sync(kFull, w, o);
        r.n = __shfl_xor_sync(kFull, n, o);
        return r;
    }
};
struct Around {                                 // weight above a logit, and at it
    u64 over = 0, same = 0;
    __device__ __forceinline__ void add(const Around & o) { over += o.over; same += o.same; }
    __device__ __forceinline__ Around across(int o) const {
        Around r;
        r.over = __shfl_xor_sync(kFull, over, o);
        r.same = __shfl_xor_sync(kFull, same, o);
        return r;
    }
};

// Weights of the list's tokens (1: `ones`), nothing behind them.
template <int NT>
__device__ __forceinline__ void weigh_list(int tid, TeamBins<NT> * B, const Pair * list, int n, const Row & r, bool ones) {
    for (int j = tid; j < kList; j += NT) B->w[j] = j < n ? (ones ? 1ull : weight_one(list[j].v, r)) : 0ull;
}

// The cut inside the bin that find_bin found: everything above the returned logit is kept, and
// `ties` of those equal to it, which may be all (`partial` false).
template <bool WEIGHTS, class T, int NT, bool CL, bool RES>
__device__ float find_cut(Team<NT, CL> & team, TeamBins<NT> * B, const Slice<T, RES> & l, const Row & row, Level L, u64 need,
                          u64 & ties, bool & partial) {
    constexpr int NB = bins_of<NT>();
    TeamSmem<NT> * s = team.s;
    for (;;) {
        // at least this many tokens are in the bin, as none is heavier than its upper edge
        const float edge = fminf(L.hi, L.hi - (L.hi - L.lo) * (((float) L.bin - 0.01f) / (float) NB));
        const u64 most = WEIGHTS ? max(weight_one(edge, row), 1ull) : 1ull;
        const Pair * list;
        float hi, lo;
        const int n = gather<true, T, NT, CL, RES>(team, B, l, 0, list, [&](float v) { return L.holds(v) && L.bin_of<NB>(v) == L.bin; },
                                                   L.with - L.above <= (u64) kList * most, hi, lo);
        if (n <= kList) {
            weigh_list<NT>(team.tid, B, list, n, row, !WEIGHTS);
            team.sync();
            over_list<NT, Around>(team.tid, n,
                [&](Around & a, int j, int i) {
                    const float o = list[i].v, v = list[j].v;
                    if (o > v) a.over += B->w[i];
                    if (o == v) a.same += B->w[i];
                },
                [&](int j, const Around & a, int) {
                    const u64 over = L.above + a.over;
                    if (over < need && need <= over + a.same) {  // threads with equal logits write the same
                        s->cut = list[j].v;
                        s->cut_ties = (need - over + B->w[j] - 1) / B->w[j];
                        s->cut_partial = s->cut_ties * B->w[j] < a.same;
                    }
                });
            team.sync();
            ties = s->cut_ties;
            partial = s->cut_partial != 0;
            const float v = s->cut;
            team.sync();
            return v;
        }
        if (!(hi > lo)) {                       // one value
            const u64 each = WEIGHTS ? weight_one(hi, row) : 1ull;
            ties = (need - L.above + each - 1) / max(each, 1ull);
            partial = true;
            return hi;
        }
        L.range(hi, lo, NB);
        find_bin<WEIGHTS, T, NT, CL, RES>(team, B, l, row, L, need, nullptr);
    }
}

__device__ __forceinline__ void write_token(const pk_sample_args & a, long long row, int token, float v, float hi, double inv_t, u64 total) {
    a.tokens[row] = token;
    if (a.logprobs) a.logprobs[row] = (float) ((v == hi ? 0.0 : ((double) v - (double) hi) * inv_t) - log((double) total * (1.0 / kOne)));
}

__device__ __forceinline__ u64 place_of(float u, u64 total) {
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    return min((u64) ((double) u * (double) total), total - 1);
}

// All tokens that may be kept are on the list: of the first k of them those before which less than
// `need` lies (0: the share p of the k tokens' weight), of these those that reach `least`; the draw.
template <int NT, bool CL>
__device__ void draw_listed(Team<NT, CL> & team, TeamBins<NT> * B, const Pair * list, int n, const pk_sample_args & a, long long row,
                            const Row & r, float hi, double inv_t, int k, float p, u64 need, float least) {
    weigh_list<NT>(team.tid, B, list, n, r, false);
    team.sync();
    constexpr int PER = (kList * sharers<NT>() + NT - 1) / NT;   // tokens of a thread
    Rank rank[PER];
    u64 sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) rank[q].n = kList;
    over_list<NT, Rank>(team.tid, n,
        [&](Rank & a, int j, int i) {
            const Pair me = list[j], o = list[i];
            if (i < n && (o.v > me.v || (o.v == me.v && o.i < me.i))) { a.w += B->w[i]; ++a.n; }
        },
        [&](int j, const Rank & a, int q) {
            rank[q] = a;
            if (a.n < k) sum += B->w[j];
        });
    Team<NT, false> block{team.tid, 0, 1, 0, team.s, 0.0};
    if (need == 0) {
        sum = block.sum(sum);
        need = p >= 1.0f ? ~0ull : max((u64) ceil(p > 0.0f ? (double) p * (double) sum : 0.0), 1ull);
    }
    team.sync();
    u64 kept = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int j = (team.tid + q * NT) / sharers<NT>();
        if (j < n && team.tid % sharers<NT>() == 0) {
            const bool keep = rank[q].n < k && rank[q].w < need && list[j].v >= least;
            if (!keep) B->w[j] = 0;
            else kept += B->w[j];
        }
    }
    const u64 total = block.sum(kept);
    team.sync();
    const u64 t = place_of(a.uniforms[row], total);
    over_list<NT, Rank>(team.tid, n,
        [&](Rank & a, int j, int i) { if (list[i].i < list[j].i) a.w += B->w[i]; },
        [&](int j, const Rank & before, int) {
            const u64 w = B->w[j];
            if (before.w <= t && t < before.w + w && team.rank == 0) write_token(a, row, list[j].i, list[j].v, hi, inv_t, total);
        });
}

// A warp's row by f32 sums; false where they cannot tell the token.
//
// w^ = ex2(x^), x^ = fma(v, c, -k) with c = fl(log2(e) / T) and k = fl(hi c). What k is off by is the same
// for all tokens and drops out (of the log-probability it is taken again). c is off by 3 2^-24, the sum
// by 2^-24 of itself, so x^ by 4 2^-24 |x|, and ex2.approx by 2^-21 of its result at most:
// |w^ - w| <= w 2^-24 (8 + 2.78 |x|). With p = w / S and S >= 1, the sum of p |x| is the entropy of p
// less log2 S, so at most log2 V: any sum of w^ over tokens is within S 2^-24 (8 + 2.78 log2 V) <=
// 39 S 2^-24 of that of w, for V <= 2048. A run's terms (65 at most) go to four accumulators, 17 additions
// each and two more: 19 S 2^-24. The runs are added in f64. Together below 2^-18 S = E for every prefix and for
// S, so u S is off by as much: the token is settled if the border before it and the one behind are each
// more than 2 E (2.5 E, against what is left) from u S.
struct Row32 {
    float inv_t, c, k, hi;
    bool fine;            // no product is NaN or far from what the bound assumes
    __device__ __forceinline__ Row32(float top, float temp) {
        inv_t = 1.0f / temp;
        c = 1.4426950408889634f * inv_t;
        k = top * c;
        hi = top;
        fine = c > 1e-30f && c < 1e30f && fabsf(k) < 1e6f;
    }
    __device__ __forceinline__ float weight(float v) const {     // 0 for -infinity; a NaN ends in the sum
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf(v, c, -k)));
        return w;
    }
    __device__ __forceinline__ float logprob(float v, double total) const {
        const double off = (double) k - (double) hi * (double) c;   // every weight is 2^-off of what it should be
        return (float) ((double) (v - hi) * (double) inv_t - 0.6931471805599453 * off - (double) logf((float) total));
    }
};

template <class T, bool RES>
__device__ __forceinline__ bool draw_f32(const Slice<T, RES> & l, int len, int lane, float hi, float temp, float u, const pk_sample_args & a,
                                         long long row) {
    const Row32 r(hi, temp);
    if (!r.fine) return false;
    const int i0 = lane * len;
    float part[4] = {};
    int j = 0;
    for (; j + 4 <= len; j += 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q) part[q] += r.weight(l(i0 + j + q));
    }
    for (; j < len; ++j) part[0] += r.weight(l(i0 + j));
    const double sum = (double) ((part[0] + part[1]) + (part[2] + part[3]));
    const double upto = warp_scan(sum, lane), total = __shfl_sync(kFull, upto, 31);
    if (!(total < 1e30)) return false;
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    const double t = (double) u * total, margin = total * 0x1.4p-17;
    // the run that holds t: the first whose end is past it
    const unsigned past = __ballot_sync(kFull, upto > t);
    if (past == 0) return false;
    const int who = __ffs((int) past) - 1;
    double run = __shfl_sync(kFull, upto - sum, who);
    const int e = min((who + 1) * len, l.n);
    for (int b = who * len; b < e; b += 32) {
        const int i = b + lane;
        const float v = i < e ? l(i) : -CUDART_INF_F, w = r.weight(v);
        const double end = run + warp_scan((double) w, lane);
        const unsigned beyond = __ballot_sync(kFull, end > t);
        if (beyond != 0) {
            const bool mine = lane == __ffs((int) beyond) - 1;
            const bool sure = mine && i < e && end - t > margin && (t - (end - (double) w) > margin);
            if (sure) {
                a.tokens[row] = i;
                if (a.logprobs) a.logprobs[row] = r.logprob(v, total);
            }
            return __any_sync(kFull, sure);
        }
        run = __shfl_sync(kFull, end, 31);
    }
    return false;
}

// Top-p by f32 sums, for a block's row with nothing cut by k: what they can tell, with bounds as above.
//
// One pass sums all weights and counts the tokens of each bin. A bin's weight lies between its count times
// the weights at its two edges, so the bins in which the sum over falling logits may reach the share p
// are known; a second pass sums what lies above them and lists their tokens, and the cut is read from
// the list's ranks. A third pass draws. For V <= 16384, and at most 64 logits a thread, a sum of f32 weights is off by less than
// S 2^-24 (8 + 2.78 * 14 + 19) < 70 2^-24 S = E (19: the additions of a thread's quarter); sums are
// joined as integers of 2^-40. A step that a sum within 2.5 E of its border decides is left to the f64
// sums (some 3 rows in 100 of 8193 logits).
enum { kNothing = 0, kCut = 1, kDrawn = 2 };
constexpr double kOff = 70.0 * 0x1p-24;
constexpr double kFix = 1099511627776.0;        // 2^40

template <class T, int NT>
__device__ int nucleus_f32(Team<NT, false> & team, TeamBins<NT> * B, const Slice<T, true> & l, int len, float hi, float low, float temp,
                           float least, float p, float u, const pk_sample_args & a, long long row, float & cut, u64 & ties, bool & partial) {
    constexpr int NB = bins_of<NT>(), PER = NB / NT;
    TeamSmem<NT> * s = team.s;
    const Row32 r(hi, temp);
    if (!(r.fine && p > 0.0f)) return kNothing;
    // tokens of less than (1 - p) / V of the largest weight cannot be at the cut, see below
    const float tail = 0.5f * (1.0f - p) / (float) a.vocab;
    const float from = fmaxf(low, hi + 0.6931f * log2f(fmaxf(tail, 1e-13f)) * temp * 1.001f);
    if (!(from < hi)) return kNothing;
    Level L;
    L.range(hi, from, NB);
    if (L.half != 1.0f || !(L.inv < 1e30f)) return kNothing;
    uint2 * bins = B->sum[0];
    for (int b = team.tid; b < NB; b += NT) bins[b].x = 0;
    if (team.tid == 0) { s->found = NB - 1; s->found_ties = NB - 1; s->listed = 0; }
    team.sync();
    float part[4] = {};
    l.template quads<NT>(team.tid, [&](float4 v, int) {
        auto one = [&](float x, float & sum) {
            sum += r.weight(x);
            if (x >= from) atomicAdd(&bins[L.bin_of<NB>(x)].x, 1u);
        };
        one(v.x, part[0]);
        one(v.y, part[1]);
        one(v.z, part[2]);
        one(v.w, part[3]);
    });
    auto fixed = [](float w) { return (u64) __double2ull_rn((double) w * kFix); };
    const float mine = (part[0] + part[1]) + (part[2] + part[3]);
    // A thread's at most 64 weights of at most 2^(2^-24 |k|) < 1.05 each stay below 128; a NaN shows in the sum that
    // it enters. What such a thread gives instead is more than all threads' honest sums (NT 68 2^40) together, and
    // less than would wrap if every thread gave it.
    constexpr u64 kBad = 1ull << 55;
    static_assert(NT <= 256, "honest sums below kBad, NT times kBad below 2^64");
    const u64 total = team.sum(mine < 128.0f ? fixed(mine) : kBad);
    if (total >= kBad) return kNothing;
    const double S = (double) total, E = S * kOff;
    // bounds of what the bins hold, and the first that may and the first that must reach the share
    const float width = (hi - from) / (float) NB;
    // in units of 2^-29 of the sum, rounded outwards, the upper bound in the high word
    const float unit = (float) (kFix * 536870912.0 / S);
    u64 bound[PER], sum_bound = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int b = team.tid * PER + j;
        const float n = (float) bins[b].x * unit;
        // the edges moved out by more than bin_of's rounding
        const float up = n * r.weight(hi - ((float) b - 0.01f) * width) * 1.0001f, down = n * r.weight(hi - ((float) b + 1.01f) * width) * 0.9999f;
        bound[j] = n > 0.0f ? (u64) (__float2uint_ru(fminf(up, 1e9f))) << 32 | __float2uint_rd(fminf(down, 1e9f)) : 0ull;
        sum_bound += bound[j];
    }
    u64 all;
    u64 before = team.scan(sum_bound, all);
    const unsigned need_lo = (unsigned) max(1.0, (double) p * 536870912.0 * (1.0 - kOff)), need_hi = (unsigned) ((double) p * 536870912.0 * (1.0 + kOff)) + 2;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const u64 upto = before + bound[j];
        if ((unsigned) (before >> 32) < need_lo && need_lo <= (unsigned) (upto >> 32)) s->found = team.tid * PER + j;
        if ((unsigned) before < need_hi && need_hi <= (unsigned) upto) s->found_ties = team.tid * PER + j;
        before = upto;
    }
    team.sync();
    const int b1 = s->found, b2 = s->found_ties;
    // down to `sure` a token lies above those bins, down to `reach` it goes on the list
    const float reach = fmaxf(from, hi - ((float) b2 + 1.01f) * width), sure = hi - ((float) b1 - 0.02f) * width;
    float above[4] = {};
    l.template quads<NT>(team.tid, [&](float4 v, int i) {
        const float top4 = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        if (!__any_sync(kFull, top4 >= reach)) return;
        auto one = [&](float x, float & sum) {
            const float w = r.weight(x);
            if (x >= sure) sum += w;
            return x >= reach && x < sure;
        };
        const bool bx = one(v.x, above[0]), by = one(v.y, above[1]), bz = one(v.z, above[2]), bw = one(v.w, above[3]);
        if (bx || by || bz || bw) {
            int n = atomicAdd(&s->listed, (int) bx + (int) by + (int) bz + (int) bw);
            if (bx && n < kList) B->list[n] = Pair{v.x, i};
            n += bx;
            if (by && n < kList) B->list[n] = Pair{v.y, i + 1};
            n += by;
            if (bz && n < kList) B->list[n] = Pair{v.z, i + 2};
            n += bz;
            if (bw && n < kList) B->list[n] = Pair{v.w, i + 3};
        }
    });
    const u64 over0 = team.sum(fixed((above[0] + above[1]) + (above[2] + above[3])));
    team.sync();
    const int n = s->listed;
    if (team.tid == 0) s->found = kNothing;
    team.sync();
    if (team.tid == 0) s->listed = 0;
    if (n > kList) return kNothing;
    for (int j = team.tid; j < kList; j += NT) B->w[j] = j < n ? max(fixed(r.weight(B->list[j].v)), 1ull) : 0ull;
    team.sync();
    const double want = (double) p * S, margin = 2.5 * E;
    over_list<NT, Around>(team.tid, n,
        [&](Around & x, int j, int i) {
            const float o = B->list[i].v, v = B->list[j].v;
            if (o > v) x.over += B->w[i];
            if (o == v) x.same += B->w[i];
        },
        [&](int j, const Around & x, int) {
            const u64 w = B->w[j], over = over0 + x.over;
            if ((double) over < want && want <= (double) (over + x.same)) {
                const u64 t = (u64) ceil((want - (double) over) / (double) w);
                // without its last tie the sum falls short, with it it does not, whatever f32 is off by
                if (t >= 1 && t * w <= x.same && (double) (over + (t - 1) * w) + margin < want && (double) (over + t * w) - margin > want) {
                    s->cut = B->list[j].v;
                    s->cut_ties = t;
                    s->cut_partial = t * w < x.same;
                    s->found = kCut;
                }
            }
        });
    team.sync();
    const int state = s->found;
    if (state == kCut) {
        cut = s->cut;
        ties = s->cut_ties;
        partial = s->cut_partial != 0;
    }
    team.sync();
    if (state != kCut || partial) return state;
    // the draw, over runs of consecutive indices
    const float keep = fmaxf(least, cut);
    const int i0 = team.tid * len;
    float run[4] = {};
    int j = 0;
    auto kept = [&](int i) {
        const float v = l(i);
        return v >= keep ? r.weight(v) : 0.0f;
    };
    for (; j + 4 <= len; j += 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q) run[q] += kept(i0 + j + q);
    }
    for (; j < len; ++j) run[0] += kept(i0 + j);
    const u64 sum = fixed((run[0] + run[1]) + (run[2] + run[3]));
    u64 S2 = 0;
    before = team.scan(sum, S2);
    const u64 t = place_of(u, S2), edge = (u64) ((double) S2 * (2.5 * kOff)) + 1;
    if (team.tid == 0) s->found = -1;
    team.sync();
    if (before <= t && t < before + sum) {
        s->found = team.tid;
        s->found_before = before;
    }
    team.sync();
    const int who = s->found;
    team.sync();
    if (team.tid == 0) s->found = kCut;
    team.sync();
    if (who >= 0 && team.tid < 32) {
        const int e = min((who + 1) * len, l.n);
        u64 at = s->found_before;
        for (int b = who * len; b < e; b += 32) {
            const int i = b + team.tid;
            const u64 w = i < e ? fixed(kept(i)) : 0ull;
            const u64 end = at + warp_scan(w, team.tid);
            if (end - w <= t && t < end && end - t > edge && t - (end - w) >= edge) {
                a.tokens[row] = i;
                if (a.logprobs) a.logprobs[row] = r.logprob(l(i), (double) S2 * (1.0 / kFix));
                s->found = kDrawn;
            }
            at = __shfl_sync(kFull, end, 31);
            if (at > t) break;
        }
    }
    team.sync();
    const int done = s->found;
    team.sync();
    return done;
}

template <class T, int NT, bool FILTERS, bool CL, bool RES>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT, NT == 32 ? (FILTERS ? 4 : 5) : 1024 / NT)
sample_kernel(pk_sample_args a, int slice, int teams, int row_floats) {
    extern __shared__ __align__(16) unsigned char raw[];
    const int t_in = NT == 32 ? (int) threadIdx.x >> 5 : 0;      // team within the block
    Team<NT, CL> team;
    team.tid = NT == 32 ? (int) threadIdx.x & 31 : (int) threadIdx.x;
    team.blocks = CL ? (int) cg::this_cluster().num_blocks() : 1;
    team.rank = CL ? (int) cg::this_cluster().block_rank() : 0;
    team.phase = 0;
    const long long row = CL ? (long long) (blockIdx.x / team.blocks) : (long long) blockIdx.x * teams + t_in;
    if (NT == 32 && row >= a.rows) return;                       // warps by themselves: nothing to meet
    float * rows_at = reinterpret_cast<float *>(raw);
    TeamSmem<NT> * state = reinterpret_cast<TeamSmem<NT> *>(rows_at + (size_t) teams * row_floats);
    team.s = state + t_in;
    TeamBins<NT> * bins = reinterpret_cast<TeamBins<NT> *>(state + teams) + t_in;
    team.mine = table_entry(team.lane());
    const int s0 = min(team.rank * slice, a.vocab);
    Slice<T, RES> l;
    l.n = min(slice, a.vocab - s0);
    l.gl = static_cast<const T *>(a.logits) + row * a.row_stride + s0;
    l.sm = rows_at + (size_t) t_in * row_floats;
    l.skew = RES ? (int) ((reinterpret_cast<uintptr_t>(l.gl) & 15) / sizeof(T)) & 3 : 0;
    l.inf = false;
    const int len = run_of<NT>(l.n);
    l.pad = max(((l.skew + l.n + 3) & ~3) - l.skew, NT * len);
    if constexpr (RES) {
        load_slice<T, NT>(l, team.tid);
        team.sync();
    }
    const float temp_f = a.temperatures ? a.temperatures[row] : a.temperature;
    const double temp = (double) temp_f;
    float hi = -CUDART_INF_F, lo = CUDART_INF_F;                 // fmaxf and fminf pass over NaN
    l.template each<NT>(team.tid, [&](float v, int) {
        hi = fmaxf(hi, v);
        if (FILTERS && v > -CUDART_INF_F) lo = fminf(lo, v);
    });
    team.template range<FILTERS>(hi, lo);
    if (hi == -CUDART_INF_F || !(temp_f > 0.0f)) {
        // nothing to draw, or the first index of the largest
        u64 first = ~0ull;
        if (hi > -CUDART_INF_F)
            for (int i = team.tid; i < l.n && first == ~0ull; i += NT)
                if (l(i) == hi) first = (u64) (s0 + i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(kFull, first, o));
        if (NT > 32) {
            team.sync();
            if (team.lane() == 0) team.s->wscan[team.tid >> 5] = first;
            team.sync();
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) first = min(first, team.s->wscan[i]);
        }
        if (CL) {
            Xchg & x = team.s->x[team.phase];
            if (team.tid == 0) x.a = first;
            team.meet();
            team.hear(x, [&](int, const Xchg & o) { first = min(first, o.a); });
            team.meet();
        }
        if (team.tid == 0 && team.rank == 0) {
            a.tokens[row] = hi == -CUDART_INF_F ? -1 : (int) first;
            if (a.logprobs) a.logprobs[row] = hi == -CUDART_INF_F ? -CUDART_INF_F : 0.0f;
        }
        return;
    }
    if (hi == CUDART_INF_F) {                                    // zeros where it is +infinity, nothing elsewhere
        if constexpr (RES) {
            team.sync();
            for (int i = team.tid; i < l.n; i += NT) l.sm[l.skew + i] = l.sm[l.skew + i] == CUDART_INF_F ? 0.0f : -CUDART_INF_F;
            team.sync();
        }
        l.inf = true;
        hi = lo = 0.0f;
    }
    if constexpr (!FILTERS && NT == 32)
        if (draw_f32<T, RES>(l, len, team.tid, hi, temp_f, a.uniforms[row], a, row)) return;
    Row r;
    r.top = (double) hi;
    const double inv_t = 1.0 / temp;                             // 0 for an infinite T
    r.c = 46.166241308446828384 * inv_t;                         // 32 log2(e) / T
    // below 2^-44 of the largest: 31 T is more than 44 ln 2 = 30.5 T; rounded up, so that what is
    // not below lies within the exponential's range
    r.base = fmaxf(__double2float_ru(r.top - 31.0 * temp), -3.402823466e+38f);
    float least = r.base;                                        // kept: >= least, and what the cut says
    float cut = -CUDART_INF_F;
    u64 ties = ~0ull;
    bool partial = false;
    if constexpr (FILTERS) {
        constexpr int NB = bins_of<NT>();
        const float m = a.min_ps ? a.min_ps[row] : a.min_p;
        const float p = a.top_ps ? a.top_ps[row] : a.top_p;
        const int k = a.top_ks ? a.top_ks[row] : a.top_k;
        if (m >= 1.0f) least = hi;
        else if (m > 0.0f) least = fmaxf(least, __double2float_ru(r.top + temp * log((double) m)));
        const float low = fmaxf(r.base, lo);                     // the range that can have weight
        Level L;
        u64 need = 0;
        if (k > 0 && k < a.vocab) {
            // with p off, what min-p drops need not be counted
            L.range(hi, p >= 1.0f ? fmaxf(low, least) : low, NB);
            L.above = 0;
            need = (u64) k;
            if (find_bin<false, T, NT, CL, RES>(team, bins, l, r, L, need, nullptr)) {
                if (L.with <= (u64) kList) {
                    const Pair * list;
                    float h, w;
                    const int n = gather<false, T, NT, CL, RES>(team, bins, l, s0, list,
                        [&](float v) { return L.holds(v) && L.bin_of<NB>(v) <= L.bin; }, true, h, w);
                    draw_listed<NT, CL>(team, bins, list, n, a, row, r, hi, inv_t, k, p, 0, least);
                    return;
                }
                cut = find_cut<false, T, NT, CL, RES>(team, bins, l, r, L, need, ties, partial);
            }
        }
        int known = kNothing;
        // With many rows; a single one is sooner through the f64 sums, which take fewer steps one after another
        // (64 rows of 8193, each with its own settings: 16 us against 19).
        if constexpr (RES && !CL && (NT == 128 || NT == 256)) {
            if (!(p >= 1.0f) && !(cut > -CUDART_INF_F) && a.vocab <= 64 * NT) {
                known = nucleus_f32<T, NT>(team, bins, l, len, hi, low, temp_f, least, p, a.uniforms[row], a, row, cut, ties, partial);
                if (known == kDrawn) return;
            }
        }
        if (!(p >= 1.0f) && known == kNothing) {
            Share share;
            share.p = p > 0.0f ? (double) p : 0.0;
            share.from = low;
            share.lump = 0;
            u64 each = 0;
            if (cut > -CUDART_INF_F) {
                // above the cut of k, from the next number on; equal logits there count as many as are kept
                const float up = cut == 0.0f ? 1.401298464e-45f : __int_as_float(__float_as_int(cut) + (cut > 0.0f ? 1 : -1));
                share.from = fmaxf(low, up);
                each = weight_one(cut, r);
                share.lump = each * ties;
            }
            // Tokens of less than (1 - p) / V of the largest weight cannot be at the cut of p, all of them
            // together being less than the share 1 - p: no bins for them (half of that, against rounding).
            const double tail = 0.5 * (1.0 - share.p) / (double) a.vocab;
            float from = share.from;
            if (tail > 0x1p-40) from = fmaxf(from, __double2float_rd(r.top + temp * log(tail)));
            L.with = 0;
            bool found = false;
            if (share.from <= hi) {
                L.range(hi, from, NB);
                L.above = 0;
                found = find_bin<true, T, NT, CL, RES>(team, bins, l, r, L, need, &share);
            } else {
                need = max((u64) ceil(share.p * (double) share.lump), 1ull);
            }
            if (found) {
                // Few enough to be listed? None is lighter than the bin's lower edge. With more than some 32
                // the list's ranks cost more than the sums below.
                const float edge = fmaxf(from, hi - (hi - from) * ((float) (L.bin + 1) / (float) NB));
                if ((double) L.with <= 32.0 * (double) max(weight_one(edge, r), 1ull)) {
                    const Pair * list;
                    float h, w;
                    const int n = gather<false, T, NT, CL, RES>(team, bins, l, s0, list,
                        [&](float v) { return L.holds(v) && L.bin_of<NB>(v) <= L.bin; }, true, h, w);
                    if (n <= kList) {
                        draw_listed<NT, CL>(team, bins, list, n, a, row, r, hi, inv_t, kList, p, need, least);
                        return;
                    }
                }
                cut = find_cut<true, T, NT, CL, RES>(team, bins, l, r, L, need, ties, partial);
            } else if (each > 0) {
                // the cut of k, with fewer ties
                const u64 fewer = (need - L.with + each - 1) / each;
                if (fewer < ties) { ties = fewer; partial = true; }
            }
        }
    }
    const int i0 = RES ? team.tid * len : min(team.tid * len, l.n), i1 = RES ? i0 + len : min(i0 + len, l.n);
    // a run has fewer than 2^9 elements, so its sum stays below 2^53 and is whole
    double onto = kZero;
    const float from = fmaxf(least, cut);
    unsigned equal = 0;
#pragma unroll 4
    for (int j = 0; j < len; ++j) {
        const float v = RES || i0 + j < i1 ? l(i0 + j) : -CUDART_INF_F;
        bool keep = v >= from;
        if (FILTERS) {
            if (partial && v == cut) {
                ++equal;
                keep = false;
            }
            if (!__any_sync(kFull, keep)) continue;
        }
        const double w = weight_warp(v, r, team.mine, onto);
        if (keep) onto = w;
    }
    u64 sum = whole(onto), tie0 = 0;
    if (FILTERS && partial) {
        // equal logits at the cut, not all of which are kept, go by index
        u64 all;
        tie0 = team.scan((u64) equal, all);
        if (cut >= least && tie0 < ties) sum += min((u64) equal, ties - tie0) * weight_one(cut, r);
    }
    u64 total = 0;
    const u64 before = team.scan(sum, total);
    const u64 t = place_of(a.uniforms[row], total);
    if (team.tid == 0) team.s->found = -1;
    team.sync();
    if (before <= t && t < before + sum) {
        team.s->found = team.tid;
        team.s->found_before = before;
        team.s->found_ties = (int) tie0;
    }
    team.sync();
    const int who = team.s->found;
    if (who >= 0 && team.tid < 32) {
        // the run again, 32 elements at a time
        const int e = min((who + 1) * len, l.n);
        u64 run = team.s->found_before, tie = FILTERS ? (u64) team.s->found_ties : 0ull;
        for (int c = who * len; c < e; c += 32) {
            const int i = c + team.tid;
            const float v = i < e ? l(i) : -CUDART_INF_F;
            bool keep = v >= from;
            if (FILTERS && partial) {
                const unsigned eq = __ballot_sync(kFull, v == cut);
                if (v == cut) keep = keep && tie + __popc(eq & ((1u << team.tid) - 1u)) < ties;
                tie += __popc(eq);
            }
            u64 w = whole(weight_warp(v, r, team.mine));
            if (!keep) w = 0;
            const u64 x = run + warp_scan(w, team.tid);
            if (x - w <= t && t < x) write_token(a, row, s0 + i, v, hi, inv_t, total);
            run = __shfl_sync(kFull, x, 31);
            if (run > t) break;
        }
    }
    if (CL) team.meet();                                         // a block's memory stays while others may read it
}

constexpr size_t kSmemCap = 220 * 1024;

template <class T, int NT, bool FILTERS, bool CL, bool RES>
cudaError_t launch(const pk_sample_args & a, int blocks, int slice, int row_floats, size_t smem, cudaStream_t s) {
    const int teams = NT == 32 ? 8 : 1;
    auto kernel = sample_kernel<T, NT, FILTERS, CL, RES>;
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

// Shared memory of a block: the teams' rows, then their state, then their bins.
template <int NT, bool FILTERS>
size_t team_bytes(int slice, int & row_floats) {
    row_floats = (std::max(slice, NT * run_of<NT>(slice)) + 3 + 3) / 4 * 4;
    return (NT == 32 ? 8 : 1) * ((size_t) row_floats * 4 + sizeof(TeamSmem<NT>) + (FILTERS ? sizeof(TeamBins<NT>) : 0));
}

template <class T, bool FILTERS, int NT>
cudaError_t launch_block(const pk_sample_args & a, cudaStream_t s) {
    int row_floats;
    const size_t smem = team_bytes<NT, FILTERS>(a.vocab, row_floats);
    return launch<T, NT, FILTERS, false, true>(a, 1, a.vocab, row_floats, smem, s);
}

template <class T, bool FILTERS>
cudaError_t launch_cluster(const pk_sample_args & a, int blocks, cudaStream_t s) {
    // slices of whole 16 bytes, so that every slice is aligned as its row is
    const int slice = ((a.vocab + blocks - 1) / blocks + 31) / 32 * 32;
    int row_floats;
    const size_t smem = team_bytes<1024, FILTERS>(slice, row_floats);
    if (smem <= kSmemCap) return launch<T, 1024, FILTERS, true, true>(a, blocks, slice, row_floats, smem, s);
    return launch<T, 1024, FILTERS, true, false>(a, blocks, slice, 0, smem - (size_t) row_floats * 4, s);
}

template <class T, bool FILTERS>
cudaError_t dispatch(const pk_sample_args & a, cudaStream_t s) {
    // All figures here: replayed from a graph, peaked logits (spread 2.5 and a few likely tokens), p = 0.9.
    // A row a warp, in blocks of eight, from one block an SM on with nothing cut (1500 rows of 600: 5.8 us, with
    // a block of 128 a row 7.2; 700 rows: 5.4 and 4.3; 20000 rows of 2048: 45 and 85) and from 20 rows an SM on
    // with filters, if three such blocks and their bins fit an SM (6000 rows of 1025, top-p: 54 us and 62, 1500
    // rows with k = 64: 53 and 35; 6000 rows of 1150: 70 and 64).
    if (FILTERS ? a.vocab <= 1056 && a.rows >= 20 * 148 : a.vocab <= 2048 && a.rows >= 8 * 148) return launch_block<T, FILTERS, 32>(a, s);
    // Few rows of a large vocabulary over clusters. A cluster's barriers cost more than they save below (one
    // row with top-p, in one block of 512 and in a cluster of eight: of 8193 14 us and 23, of 20000 24 us
    // and 23, of 50000 48 us and 25).
    int blocks = 1;
    if (a.vocab > 16384)
        while (blocks < kMaxCluster && a.rows * blocks * 2 <= 148) blocks *= 2;
    while (blocks < kMaxCluster && (size_t) (a.vocab / blocks) * 4 > 200 * 1024) blocks *= 2;
    if (blocks > 1) return launch_cluster<T, FILTERS>(a, blocks, s);
    // Otherwise a row a block, of as many threads as let every row have its block at once (450 rows of 4097,
    // top-p, in blocks of 128, 256 and 512: 27 us, 22, 26; 296 rows: 26, 20, 15), though of at least 256 for
    // up to 2048 logits (one row of 1600: 6.7 us, of 512 8.2). Past that the fewest threads that a row's length
    // leaves busy: 128 up to 5120 (4096 rows of 4097: 90 us, 100, 172), 256 up to 16384 (4096 rows of 8193:
    // 219 us, 160, 242), 512.
    const bool wave512 = a.rows <= 2 * 148 && a.vocab > 2048, wave256 = a.rows <= 4 * 148;
    if (a.vocab > 16384 || wave512) return launch_block<T, FILTERS, 512>(a, s);
    if (a.vocab > 5120 || wave256) return launch_block<T, FILTERS, 256>(a, s);
    return launch_block<T, FILTERS, 128>(a, s);
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
