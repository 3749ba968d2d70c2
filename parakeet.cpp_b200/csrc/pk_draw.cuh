// pk_draw.cuh -- rows of logits as weights (pk_sample.cu: drawing from them; pk_verify.cu: two of them against each
// other): a row in the shared memory of a team of threads, its largest logit, its cuts by top-k and top-p, and
// exponentials as integers. The head of pk_sample.cu says how they work together.
#pragma once

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

// The threads of one row. CL: several blocks of a cluster, each with a slice of the row. NM: one of several teams of a
// block, which meet at barriers of their own.
template <int NT, bool CL, bool NM = false>
struct Team {
    int tid, rank, blocks;
    unsigned phase;
    TeamSmem<NT> * s;
    double mine;                             // this lane's entry of the exponential's table
    unsigned level = 0;                      // levels of bins so far
    int bar = 0;                             // its barrier

    // This block's threads by themselves.
    __device__ __forceinline__ Team<NT, false, NM> alone() const { return Team<NT, false, NM>{tid, 0, 1, 0, s, 0.0, 0, bar}; }
    __device__ __forceinline__ int lane() const { return tid & 31; }
    __device__ __forceinline__ void sync() const {
        if (NT == 32) __syncwarp();
        else if (NM) asm volatile("barrier.sync %0, %1;" :: "r"(bar), "n"(NT) : "memory");
        else __syncthreads();
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
template <bool WEIGHTS, class T, int NT, bool CL, bool RES, bool NM>
__device__ bool find_bin(Team<NT, CL, NM> & team, TeamBins<NT> * B, const Slice<T, RES> & l, const Row & row, Level & L, u64 & need,
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
    auto block = team.alone();            // the bins are the cluster's already
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
template <bool RANGE, class T, int NT, bool CL, bool RES, bool NM, class F>
__device__ int gather(Team<NT, CL, NM> & team, TeamBins<NT> * B, const Slice<T, RES> & l, int s0, const Pair *& list, F want, bool few,
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
template <bool WEIGHTS, class T, int NT, bool CL, bool RES, bool NM>
__device__ float find_cut(Team<NT, CL, NM> & team, TeamBins<NT> * B, const Slice<T, RES> & l, const Row & row, Level L, u64 need,
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

__device__ __forceinline__ u64 place_of(float u, u64 total) {
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    return min((u64) ((double) u * (double) total), total - 1);
}

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

template <class T, int NT, bool NM>
__device__ int nucleus_cut(Team<NT, false, NM> & team, TeamBins<NT> * B, const Slice<T, true> & l, float hi, float low, float temp,
                           float p, int vocab, float & cut, u64 & ties, bool & partial, double & kept) {
    constexpr int NB = bins_of<NT>(), PER = NB / NT;
    TeamSmem<NT> * s = team.s;
    const Row32 r(hi, temp);
    if (!(r.fine && p > 0.0f)) return kNothing;
    // tokens of less than (1 - p) / V of the largest weight cannot be at the cut, see below
    const float tail = 0.5f * (1.0f - p) / (float) vocab;
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
                    s->found_sum = over + t * w;
                    s->found = kCut;
                }
            }
        });
    team.sync();
    const int state = s->found;
    if (state == kCut) {
        kept = (double) s->found_sum * (1.0 / kFix);
        cut = s->cut;
        ties = s->cut_ties;
        partial = s->cut_partial != 0;
    }
    team.sync();
    return state;
}

// Where top-p goes by f32 sums.
template <int NT, bool CL, bool RES> constexpr bool nucleus_fits() { return RES && !CL && (NT == 128 || NT == 256); }

// What the filters leave of a row with largest logit hi and smallest lo: all logits from `least` on (given: what can
// have weight; min-p raises it) that are above `cut`, or equal to it and among the first `ties` (`partial`: which are
// not all). True where the answer was had on the way: from `listed`, called with a list of all tokens that may be kept
// (of the first so many of them those before which less than `need` lies, or, where that is 0, the share of their
// weight), or from `sure`, which is asked once the cut is known without f64 sums, and told the weight from the cut on
// as f32 sums have it. `s0`: index of the slice's first.
template <class T, int NT, bool CL, bool RES, bool NM, class Listed, class Sure>
__device__ bool cut_row(Team<NT, CL, NM> & team, TeamBins<NT> * bins, const Slice<T, RES> & l, int s0, const Row & r, float hi, float lo, float temp_f,
                        int vocab, int k, float p, float m, float & least, float & cut, u64 & ties, bool & partial, Listed listed, Sure sure) {
    const double temp = (double) temp_f;
    constexpr int NB = bins_of<NT>();
    if (m >= 1.0f) least = hi;
    else if (m > 0.0f) least = fmaxf(least, __double2float_ru(r.top + temp * log((double) m)));
    const float low = fmaxf(r.base, lo);                     // the range that can have weight
    Level L;
    u64 need = 0;
    if (k > 0 && k < vocab) {
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
                listed(list, n, k, p, 0);
                return true;
            }
            cut = find_cut<false, T, NT, CL, RES>(team, bins, l, r, L, need, ties, partial);
        }
    }
    int known = kNothing;
    // With many rows; a single one is sooner through the f64 sums, which take fewer steps one after another
    // (64 rows of 8193, each with its own settings: 16 us against 19).
    if constexpr (nucleus_fits<NT, CL, RES>()) {
        if (!(p >= 1.0f) && !(cut > -CUDART_INF_F) && vocab <= 64 * NT) {
            double kept = 0.0;
            known = nucleus_cut<T, NT>(team, bins, l, hi, low, temp_f, p, vocab, cut, ties, partial, kept);
            if (known == kCut && !partial && sure(kept)) return true;
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
        const double tail = 0.5 * (1.0 - share.p) / (double) vocab;
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
                    listed(list, n, kList, p, need);
                    return true;
                }
            }
            cut = find_cut<true, T, NT, CL, RES>(team, bins, l, r, L, need, ties, partial);
        } else if (each > 0) {
            // the cut of k, with fewer ties
            const u64 fewer = (need - L.with + each - 1) / each;
            if (fewer < ties) { ties = fewer; partial = true; }
        }
    }
    return false;
}

constexpr size_t kSmemCap = 220 * 1024;

// Shared memory of a block: the teams' rows, then their state, then their bins.
template <int NT, bool FILTERS>
size_t team_bytes(int slice, int & row_floats) {
    row_floats = (std::max(slice, NT * run_of<NT>(slice)) + 3 + 3) / 4 * 4;
    return (NT == 32 ? 8 : 1) * ((size_t) row_floats * 4 + sizeof(TeamSmem<NT>) + (FILTERS ? sizeof(TeamBins<NT>) : 0));
}

}  // namespace
}  // namespace pk
