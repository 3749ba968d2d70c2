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

#include "pk_draw.cuh"

namespace pk {
namespace {

__device__ __forceinline__ void write_token(const pk_sample_args & a, long long row, int token, float v, float hi, double inv_t, u64 total) {
    a.tokens[row] = token;
    if (a.logprobs) a.logprobs[row] = (float) ((v == hi ? 0.0 : ((double) v - (double) hi) * inv_t) - log((double) total * (1.0 / kOne)));
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
    auto block = team.alone();
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

// The draw over runs of consecutive indices, by f32 sums too, where no ties are parted.
template <class T, int NT>
__device__ int nucleus_draw(Team<NT, false> & team, const Slice<T, true> & l, int len, float hi, float temp, float least, float cut, float u,
                            const pk_sample_args & a, long long row) {
    TeamSmem<NT> * s = team.s;
    const Row32 r(hi, temp);
    auto fixed = [](float w) { return (u64) __double2ull_rn((double) w * kFix); };
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
    const u64 before = team.scan(sum, S2);
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
        const float m = a.min_ps ? a.min_ps[row] : a.min_p;
        const float p = a.top_ps ? a.top_ps[row] : a.top_p;
        const int k = a.top_ks ? a.top_ks[row] : a.top_k;
        const bool done = cut_row<T, NT, CL, RES>(team, bins, l, s0, r, hi, lo, temp_f, a.vocab, k, p, m, least, cut, ties, partial,
            [&](const Pair * list, int n, int first, float share, u64 need) {
                draw_listed<NT, CL>(team, bins, list, n, a, row, r, hi, inv_t, first, share, need, least);
            },
            [&](double) {
                if constexpr (nucleus_fits<NT, CL, RES>())
                    return nucleus_draw<T, NT>(team, l, len, hi, temp_f, least, cut, a.uniforms[row], a, row) == kDrawn;
                return false;
            });
        if (done) return;
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
