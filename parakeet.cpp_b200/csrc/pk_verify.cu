// pk_verify.cu -- verification of drafted tokens: the longest run of a sequence's drafts that given random
// numbers accept, and the token behind it, so that what comes out is distributed as if the target had drawn it.
//
// p and q are the distributions that pk_sample draws from, of the target's and the draft's row of a position with
// the sequence's settings. A draft d is accepted when u q(d) < p(d). At the first that is not, the token is drawn
// from max(p - q, 0), and behind the last draft from p.
//
// Vocabularies whose two rows fit a block's shared memory take one kernel: a block (a warp for short rows) goes over
// a sequence's positions and stops at the first rejection, whose rows it then holds; what lies behind is never read.
// With few sequences the blocks of a cluster share the positions out and tell each other the outcomes. The two rows
// of a position go to two teams of threads. Without filters a draft is first tested in one pass over its rows. Otherwise
// what a test needs of a row is its largest logit, its cut, the sum of its weights and the draft's weight. Sums, of tests
// and of draws, go by f32 with a proven bound, and by pk_sample's whole numbers, exact whatever their order, where that
// leaves the answer open.
//
// Longer rows take two kernels, see below.
//
// Measured (calls among others, Python's included): 1024 sequences of four drafts by 8193 f32 logits, temperature alone, 105 us,
// of which the rows up to the first rejections are 192 MB, 29 us; most of the rest is the latency of a block's steps, two blocks
// of 512 threads an SM. 256 of eight by 8193 bf16, top-p and min-p, 132 to 144 us for some 1830 rows: the cuts of two rows a position,
// chains of block-wide steps with 44 % of the warps that an SM can hold, one position after the other. It is not what cutting
// rows takes: pk_sample cuts as many, and draws from all of them, in 71 us. One of four, top-k and top-p, 22 us, the chain of a
// cut, an exchange and a draw over all logits; pk_sample takes 9 us for a row with these settings, replayed from a graph.

#include "pk_draw.cuh"

#include <type_traits>

namespace pk {
namespace {

// What the test and the draw need of a row.
struct RowStat {
    double drafted;       // weight of the draft, relative to the largest; 0 if it is cut
    u64 total;            // of the weights kept, times 2^43; 0: no logit above -infinity
    float hi;             // largest logit (0 where it is +infinity)
    float from, cut;      // kept: at least `from`, which is not below `cut`, and above `cut` or up to index `last`
    int last;
    int flags;
};
// The largest is +infinity; the first of the largest alone is kept; the total is off by kOff of itself at most.
enum { kInf = 1, kGreedy = 2, kNear = 4 };
constexpr int kAny = 0x7FFFFFFF;

__device__ __forceinline__ int drafts_of(const pk_verify_args & a, long long seq) {
    return a.n_drafts ? max(0, min(a.n_drafts[seq], a.max_drafts)) : a.max_drafts;
}
__device__ __forceinline__ float temperature_of(const pk_verify_args & a, long long seq) { return a.temperatures ? a.temperatures[seq] : a.temperature; }
__device__ __forceinline__ float number_of(float u) { return u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f; }

// A logit as a row's statistics see it.
__device__ __forceinline__ float seen(float v, int flags) {
    return flags & kInf ? (v == CUDART_INF_F ? 0.0f : -CUDART_INF_F) : v;
}

// A row's weights, times 2^43 and whole: weight_warp's, as its numbers are needed there.
__device__ __forceinline__ Row row_of(float hi, double temp) {
    Row r;
    r.top = (double) hi;
    r.c = 46.166241308446828384 * (1.0 / temp);                  // 32 log2(e) / T, as pk_sample has it
    // below 2^-44 of the largest, see pk_sample.cu
    r.base = fmaxf(__double2float_ru(r.top - 31.0 * temp), -3.402823466e+38f);
    return r;
}

// Weight of a draft with logit v: what min-p asks for and the cut it is subject to, not `base`.
__device__ __forceinline__ double draft_weight(float v, int draft, const RowStat & st, const Row & r, double temp, float m) {
    const float floor = fmaxf(!(m > 0.0f) ? -CUDART_INF_F : m >= 1.0f ? st.hi : __double2float_ru(r.top + temp * log((double) m)), -3.402823466e+38f);
    if (!(v >= floor && (v > st.cut || (v == st.cut && draft <= st.last)))) return 0.0;
    if (v == st.hi) return 1.0;                                  // the table's first entry is one and a bit
    // pk_sample's weight as it is before it is rounded, to 2^-42 of itself
    if (v >= r.base) return weight_onto(v, r, 0.0, [](int n) { return table_entry(n & 31); }) * (1.0 / kOne);
    return exp(((double) v - r.top) / temp);
}

// The tokens before a draft of logit v, in the order that top-k goes by. Where fewer than k logits can have weight cut_row cuts
// nothing; of what lies below them nothing is drawn, but a draft there has its own probability, and is cut by its rank.
template <class T, int NT, bool CL, bool RES, bool NM>
__device__ __forceinline__ u64 rank_of(Team<NT, CL, NM> & team, const Slice<T, RES> & l, int s0, int draft, float v) {
    unsigned before = 0;
    l.template each<NT>(team.tid, [&](float x, int i) { before += x > v || (x == v && s0 + i < draft) ? 1u : 0u; });
    return team.sum((u64) before);
}

// A team's list holds all that may be kept, of the first `first` those before which less than `need` lies (0: the share
// of their weight), of these those from `least` on: the sum of what is kept, and the last of it in the order, told by the
// thread that has it to f(logit, index, sum).
template <int NT, bool CL, bool NM, class F>
__device__ void keep_listed(Team<NT, CL, NM> & team, TeamBins<NT> * bins, const Pair * list, int count, const Row & r, int first, float share, u64 need,
                            float least, F f) {
    weigh_list<NT>(team.tid, bins, list, count, r, false);
    team.sync();
    constexpr int SH = sharers<NT>(), PER = (kList * SH + NT - 1) / NT;
    Rank rank[PER];
    u64 sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) rank[q].n = kList;
    over_list<NT, Rank>(team.tid, count,
        [&](Rank & b, int j, int i) {
            const Pair me = list[j], o = list[i];
            if (i < count && (o.v > me.v || (o.v == me.v && o.i < me.i))) { b.w += bins->w[i]; ++b.n; }
        },
        [&](int j, const Rank & b, int q) {
            rank[q] = b;
            if (b.n < first) sum += bins->w[j];
        });
    auto block = team.alone();
    if (need == 0) {
        sum = block.sum(sum);
        need = share >= 1.0f ? ~0ull : max((u64) ceil(share > 0.0f ? (double) share * (double) sum : 0.0), 1ull);
    }
    // the weights stay below 2^51 in all, their number below 2^8: one sum
    u64 kept = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int j = (team.tid + q * NT) / SH;
        if (j < count && team.tid % SH == 0 && rank[q].n < first && rank[q].w < need && list[j].v >= least) kept += bins->w[j] + (1ull << 52);
    }
    kept = block.sum(kept);
    const int all = (int) (kept >> 52);
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        const int j = (team.tid + q * NT) / SH;
        if (j < count && team.tid % SH == 0 && rank[q].n == all - 1) f(list[j].v, list[j].i, kept & ((1ull << 52) - 1));
    }
}

constexpr double kShare = 1125899906842624.0;           // 2^50: probabilities as integers, whose sums f64 holds
constexpr double kMagic = 6755399441055744.0;           // 1.5 * 2^52: what is added to it is rounded to an integer
constexpr double kFine = 68719476736.0;                 // 2^36: f32 sums as integers

// What f32's weights of a row, all 2^-off of what they should be, are to be multiplied by: |off| is below 2^-4 (k is
// below 10^6 and rounded once), where four terms tell 2^off to 2^-28.
__device__ __forceinline__ double scale_of(const Row32 & f, float hi) {
    const double x = 0.6931471805599453 * ((double) f.k - (double) hi * (double) f.c);
    return 1.0 + x * (1.0 + x * (0.5 + x * (1.0 / 6.0 + x * (1.0 / 24.0))));
}

// A row's total, times 2^43, from the sum of its f32 weights. Where nearly all of it is the largest's, by what that alone gives: a
// row that leaves nothing else has exactly one. Either way the sum is off by less than kOff of itself: by the additions' 19 2^-24
// and a little of the rest, below 2^-20, in the first case.
__device__ __forceinline__ u64 total_of(double sum, const Row32 & f, float hi) {
    const double own = (double) f.weight(hi);
    return (u64) ((sum - own < 0x1p-20 * own ? sum / own : sum * scale_of(f, hi)) * kOne);
}

// Log-probability of the token with logit v: log() of a number below 2^16 in f32 is off by a unit, 2^-20, at most.
__device__ __forceinline__ float logprob_of(float v, const RowStat & p, double heat) {
    return fminf((float) ((v == p.hi ? 0.0 : ((double) v - (double) p.hi) / heat) - (double) logf((float) ((double) p.total * (1.0 / kOne)))), 0.0f);
}

// The rows that a block's shared memory holds, one of so many logits or two of half as many, and the longest that a warp and
// teams of 128 and 256 threads are given; the rest go to 512.
constexpr int kResident = 176 * 1024 / 4, kWarpMost = 1056, k128Most = 6144, k256Most = 16384;
constexpr int logits_each(int logits, int threads) { return ((logits + 6) / 4 + threads - 1) / threads * 4; }   // of a thread, in quads

// The sum of a resident row's weights that are kept. A thread's are at most 92 of 2^43, below 2^50 in all, so its sum is whole.
static_assert(logits_each(kWarpMost, 32) <= 92 && logits_each(k128Most, 128) <= 92 && logits_each(k256Most, 256) <= 92 &&
              logits_each(kResident, 512) <= 92, "a thread's logits");
template <class T, int NT, bool NM>
__device__ u64 exact_sum(Team<NT, false, NM> & team, const Slice<T, true> & l, const Row & r, float from, float cut, int last) {
    double onto = kZero;
    l.template quads<NT>(team.tid, [&](float4 v, int i) {
        bool keep[4] = {v.x >= from, v.y >= from, v.z >= from, v.w >= from};
        if (last != kAny) {
            keep[0] = keep[0] && (v.x > cut || i <= last);
            keep[1] = keep[1] && (v.y > cut || i + 1 <= last);
            keep[2] = keep[2] && (v.z > cut || i + 2 <= last);
            keep[3] = keep[3] && (v.w > cut || i + 3 <= last);
        }
        if (!__any_sync(kFull, keep[0] || keep[1] || keep[2] || keep[3])) return;
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const double w = weight_warp(x[q], r, team.mine, onto);
            if (keep[q]) onto = w;
        }
    });
    return team.sum(whole(onto));
}

// Statistics of a resident row into `st` (shared memory), by its team; complete once the team has met.
template <class T, int NT, bool FILTERS, bool NM>
__device__ void row_stat(Team<NT, false, NM> & team, TeamBins<NT> * bins, Slice<T, true> l, const pk_verify_args & a, long long seq, int draft,
                         RowStat * st) {
    const float temp_f = temperature_of(a, seq);
    const double temp = (double) temp_f;
    float hi = -CUDART_INF_F, lo = CUDART_INF_F;                 // fmaxf and fminf pass over NaN
    l.template each<NT>(team.tid, [&](float v, int) {
        hi = fmaxf(hi, v);
        if (FILTERS && v > -CUDART_INF_F) lo = fminf(lo, v);
    });
    team.template range<FILTERS>(hi, lo);
    const bool one = team.tid == 0;
    const int flags = hi == CUDART_INF_F ? kInf : 0;
    if (hi == -CUDART_INF_F || !(temp_f > 0.0f)) {
        // nothing to draw, or the first index of the largest
        u64 first = ~0ull;
        if (hi > -CUDART_INF_F)
            for (int i = team.tid; i < l.n && first == ~0ull; i += NT)
                if (l(i) == hi) first = (u64) i;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(kFull, first, o));
        if (NT > 32) {
            team.sync();
            if (team.lane() == 0) team.s->wscan[team.tid >> 5] = first;
            team.sync();
#pragma unroll
            for (int i = 0; i < NT / 32; ++i) first = min(first, team.s->wscan[i]);
        }
        if (one) {
            st->flags = flags | kGreedy;
            st->hi = st->from = st->cut = flags & kInf ? 0.0f : hi;
            st->last = (int) min(first, (u64) kAny);
            st->total = first == ~0ull ? 0ull : (u64) kOne;
            st->drafted = first != ~0ull && draft == (int) first ? 1.0 : 0.0;
        }
    }
    if (flags & kInf) {                                          // zeros where it is +infinity, nothing elsewhere
        team.sync();
        for (int i = team.tid; i < l.n; i += NT) l.sm[l.skew + i] = seen(l.sm[l.skew + i], kInf);
        team.sync();
        hi = lo = 0.0f;
    }
    if (hi == -CUDART_INF_F || !(temp_f > 0.0f)) return;
    const Row r = row_of(hi, temp);
    float least = r.base;                                        // kept: >= least, and what the cut says
    float cut = -CUDART_INF_F;
    u64 ties = ~0ull;
    bool partial = false;
    const float m = a.min_ps ? a.min_ps[seq] : a.min_p;
    auto leave = [&](float from, float cut_at, int last, u64 sum, int more) {
        st->flags = flags | more;
        st->hi = hi;
        st->from = from;
        st->cut = cut_at;
        st->last = last;
        st->total = sum;
        st->drafted = draft >= 0 && draft < l.n ? draft_weight(l(draft), draft, *st, r, temp, m) : 0.0;
    };
    if constexpr (FILTERS) {
        const float p = a.top_ps ? a.top_ps[seq] : a.top_p;
        const int k = a.top_ks ? a.top_ks[seq] : a.top_k;
        const bool done = cut_row<T, NT, false, true>(team, bins, l, 0, r, hi, lo, temp_f, a.vocab, k, p, m, least, cut, ties, partial,
            [&](const Pair * list, int count, int first, float share, u64 need) {
                keep_listed(team, bins, list, count, r, first, share, need, least,
                            [&](float v, int i, u64 sum) { leave(v, v, i, sum, 0); });
            },
            [&](double kept) {
                if (!(cut >= least)) return false;               // min-p drops more
                if (one) leave(cut, cut, kAny, total_of(kept, Row32(hi, temp_f), hi), kNear);
                return true;
            });
        if (done) return;
    }
    const float from = fmaxf(least, cut);
    int last = kAny;
    if (FILTERS && partial && cut >= least) {
        // equal logits at the cut, not all of which are kept, go by index: the last of them that is
        const int len = run_of<NT>(l.n), i0 = team.tid * len;
        unsigned equal = 0;
        for (int j = 0; j < len; ++j) equal += l(i0 + j) == cut ? 1u : 0u;
        u64 all;
        const u64 before = team.scan((u64) equal, all);
        if (one) team.s->found = kAny;
        team.sync();
        if (before < ties && ties <= before + equal) {
            int i = i0;
            for (u64 left = ties - before;; ++i)
                if (l(i) == cut && --left == 0) break;
            team.s->found = i;
        }
        team.sync();
        last = team.s->found;
    }
    // The sum by f32, as nucleus_cut takes it: off by kOff of itself at most for up to 64 logits a thread.
    if (l.n <= 64 * NT && last == kAny) {
        const Row32 f(hi, temp_f);
        if (f.fine) {
            float part[4] = {};
            l.template quads<NT>(team.tid, [&](float4 v, int) {
                // a NaN is not kept; nothing of what has no weight counts
                part[0] += !FILTERS || v.x >= from ? f.weight(v.x) : 0.0f;
                part[1] += !FILTERS || v.y >= from ? f.weight(v.y) : 0.0f;
                part[2] += !FILTERS || v.z >= from ? f.weight(v.z) : 0.0f;
                part[3] += !FILTERS || v.w >= from ? f.weight(v.w) : 0.0f;
            });
            const float mine = (part[0] + part[1]) + (part[2] + part[3]);
            // a thread's at most 68 weights stay below 128, all threads' below 2^52; a NaN gives more than that
            constexpr u64 kBad = 1ull << 54;
            static_assert(NT <= 512, "honest sums below kBad, NT times kBad below 2^64");
            const u64 sum = team.sum(mine < 128.0f ? __double2ull_rn((double) mine * kFine) : kBad);
            if (sum < kBad) {
                if (one) leave(from, cut, last, total_of((double) sum * (1.0 / kFine), f, hi), kNear);
                return;
            }
        }
    }
    const u64 sum = exact_sum<T, NT>(team, l, r, from, cut, last);
    if (one) leave(from, cut, last, sum, 0);
}

// The exact sum of a row whose statistics have f32's; complete once the team has met.
template <class T, int NT, bool NM>
__device__ void settle(Team<NT, false, NM> & team, const Slice<T, true> & l, double temp, RowStat * st) {
    if (!(st->flags & kNear)) return;
    const u64 sum = exact_sum<T, NT>(team, l, row_of(st->hi, temp), st->from, st->cut, st->last);
    if (team.tid == 0) {
        st->total = sum;
        st->flags &= ~kNear;
    }
}

enum { kAll, kLess, kWithout };                          // draws: from p, from what p has more than q, from p without the draft

// The draw by f32 weights, where they can tell the token; false where they cannot. The group's threads come together on
// entry.
//
// With w^ off by 2^-24 (8 + 2.78 |x|) of itself and sums by kOff, see pk_sample.cu, a probability p^ = w^ / S^ is
// off by 2^-24 (8 + 2.78 |x| + 70 + 2) of itself, and over all tokens by 2^-24 (8 + 41 + 72) = 121 2^-24 at most (V <= 22528).
// max(p - q, 0) is off by no more than both, 242 2^-24 in any sum over tokens; the subtraction, 1 more, and a thread's
// additions, 19. So sums are off by E = 262 2^-24 (in units of p's sum: 70 2^-24 where q has no part), u times the total by as
// much, and a token is settled if t is more than 2 E from its borders (2.5 E, against what else is rounded).
template <class T, int G>
__device__ bool draw_near(Team<G, false> & group, const Slice<T, true> & pl, const Slice<T, true> & ql, const RowStat * st, int mode, int draft,
                          float temp, float u, int32_t * token, float * logprob) {
    const RowStat & p = st[0], & q = st[1];
    const int len = run_of<G>(pl.n);
    if (len > 64 || (p.flags & kGreedy) || p.last != kAny || (mode == kLess && ((q.flags & kGreedy) || q.last != kAny))) return false;
    const Row32 pr(p.hi, temp), qr(mode == kLess ? q.hi : 0.0f, temp);
    if (!pr.fine || !qr.fine) return false;
    constexpr double kUnit = 274877906944.0;             // 2^38
    const float sp = mode == kLess ? (float) (scale_of(pr, p.hi) * kOne / (double) p.total) : 1.0f;
    const float sq = mode == kLess ? (float) (scale_of(qr, q.hi) * kOne / (double) q.total) : 0.0f;
    const float p_from = p.from, q_from = q.from;
    auto weigh = [&](int i) {
        const float x = pl(i);
        float w = x >= p_from ? pr.weight(x) : 0.0f;
        if (mode == kLess) {
            const float y = ql(i);
            const float less = y >= q_from ? qr.weight(y) * sq : 0.0f;
            w = fmaxf(fmaf(w, sp, -less), 0.0f);
        }
        if (mode == kWithout && i == draft) w = 0.0f;
        return w;
    };
    const int i0 = group.tid * len;
    float part[4] = {};
    int j = 0;
    for (; j + 4 <= len; j += 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) part[k] += weigh(i0 + j + k);
    }
    for (; j < len; ++j) part[0] += weigh(i0 + j);
    const float mine = (part[0] + part[1]) + (part[2] + part[3]);
    const u64 sum = __double2ull_rn((double) fminf(mine, 128.0f) * kUnit);
    u64 total;
    const u64 before = group.scan(sum, total);
    const double t = (double) number_of(u) * (double) total;
    const double edge = mode == kLess ? 2.5 * 262.0 * 0x1p-24 * kUnit
                                      : 2.5 * kOff * ((double) p.total * (1.0 / kOne) / scale_of(pr, p.hi)) * kUnit;
    if (group.tid == 0) group.s->found = -1;
    group.sync();
    if ((double) before <= t && t < (double) (before + sum)) {
        group.s->found = group.tid;
        group.s->found_before = before;
    }
    group.sync();
    const int who = group.s->found;
    group.sync();
    if (group.tid == 0) group.s->found = 0;
    group.sync();
    if (who >= 0 && group.tid < 32) {
        const int e = min((who + 1) * len, pl.n);
        u64 run = group.s->found_before;
        for (int c = who * len; c < e; c += 32) {
            const int i = c + group.tid;
            const u64 w = i < e ? __double2ull_rn((double) weigh(i) * kUnit) : 0ull;
            const u64 upto = run + warp_scan(w, group.tid);
            if ((double) upto - t > edge && t - (double) (upto - w) > edge) {
                *token = i;
                if (logprob) *logprob = logprob_of(pl(i), p, (double) temp);
                group.s->found = 1;
            }
            run = __shfl_sync(kFull, upto, 31);
            if ((double) run > t) break;
        }
    }
    group.sync();
    const bool done = group.s->found != 0;
    group.sync();
    return done;
}

// ---- the test of a draft where nothing is cut ---------------------------------------
//
// 1 / p(d) is the sum of exp((l_i - l_d) / T): one pass over the row as it comes from memory, without the largest logit
// and without shared memory. As in pk_sample.cu a weight w^ of a logit x = log2 w away is off by 2^-24 (8 + 2.78 |x|)
// of itself; with p = w / S, the sum of p |x| is at most the entropy and |log2 p(d)|, 15.5 + 24 for S < 2^24, and the
// additions of a thread's quarter are 46 at most; the draft's own weight, by which the sum is divided, is off by 8:
// 172 2^-24 together. What it leaves open, and rows with NaN or infinities that matter, are left to the row's statistics.
constexpr double kQuick = 180.0 * 0x1p-24;

// A thread's part of the sum.
template <class T, int NT>
__device__ __forceinline__ float quick_part(const T * __restrict__ g, int n, int tid, float c, float k) {
    constexpr int W = 16 / (int) sizeof(T);
    auto weight = [&](float v) {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf(v, c, -k)));
        return w;
    };
    const int head = min(n, (int) ((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / (int) sizeof(T)), vecs = (n - head) / W;
    float part[4] = {};
    const uint4 * at = reinterpret_cast<const uint4 *>(g + head);
    auto add = [&](const uint4 & q) {
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
                part[j] += weight(__uint_as_float(w[j]));
            } else {
                T e[2];
                *reinterpret_cast<unsigned *>(e) = w[j];
                part[j] += weight(to_f32(e[0]));
                part[j] += weight(to_f32(e[1]));
            }
        }
    };
    int i = tid;
    for (; i + 7 * NT < vecs; i += 8 * NT) {
        uint4 q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = __ldg(at + i + j * NT);
#pragma unroll
        for (int j = 0; j < 8; ++j) add(q[j]);
    }
    for (; i < vecs; i += NT) add(__ldg(at + i));
    if (tid < 16) {                                      // fewer than W at either end
        const int e = tid < 8 ? tid : head + vecs * W + tid - 8;
        if (tid < 8 ? e < head : e < n) part[0] += weight(to_f32(g[e]));
    }
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// 1 / p(d) of a row by its team; no number, or 2^24 and more, where it does not tell.
template <class T, int NT, bool NM>
__device__ double quick_sum(Team<NT, false, NM> & team, const T * row, int n, int draft, float temp) {
    const float c = 1.4426950408889634f * (1.0f / temp), v = to_f32(row[draft]), k = v * c;
    const bool fine = c > 1e-30f && c < 1e30f && fabsf(k) < 1e6f;   // the same for all
    double sum = 0.0;
    if (fine) sum = (double) quick_part<T, NT>(row, n, team.tid, c, k);
    sum = warp_sum(sum);
    if (NT > 32) {
        team.sync();
        if (team.lane() == 0) team.s->wscan[team.tid >> 5] = (u64) __double_as_longlong(sum);
        team.sync();
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) sum += __longlong_as_double((long long) team.s->wscan[i]);
    }
    float own;                                           // the draft's own weight: one, but for the rounding of k
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(own) : "f"(fmaf(v, c, -k)));
    return fine ? sum / (double) own : __longlong_as_double(0x7FF8000000000000ll);
}

template <int NT, bool DUAL> constexpr int group_of() { return DUAL ? 2 * NT : NT; }
struct SeqSums { double quick[2]; };                    // of the test where nothing is cut
struct NoSums {};
template <int NT, bool DUAL, bool FILTERS> struct SeqSmem : std::conditional_t<FILTERS, NoSums, SeqSums> {
    TeamSmem<NT> team[DUAL ? 2 : 1];
    TeamSmem<group_of<NT, DUAL>()> group;
    RowStat st[2];
    int code[2];
};
template <int NT, bool DUAL> struct SeqBins { TeamBins<NT> bins[DUAL ? 2 : 1]; };
constexpr int kSeqGroups = 8;                            // sequences of a block where each has a warp

// DUAL: the target's row and the draft's go to a team of NT threads each, otherwise to one team, one after the other.
template <class T, int NT, bool DUAL, bool FILTERS>
__global__ void __launch_bounds__(NT == 32 ? 256 : group_of<NT, DUAL>(), NT == 32 ? 4 : 1024 / group_of<NT, DUAL>())
verify_sequence_kernel(const pk_verify_args a, int rows_each, int row_floats) {
    constexpr int G = group_of<NT, DUAL>(), GROUPS = NT == 32 ? kSeqGroups : 1;
    // rows of whole 16 bytes (row_floats is a multiple of four), the states and the bins behind them
    static_assert(alignof(SeqSmem<NT, DUAL, FILTERS>) <= 8 && sizeof(SeqSmem<NT, DUAL, FILTERS>) % 8 == 0 && alignof(SeqBins<NT, DUAL>) <= 8 &&
                  sizeof(SeqBins<NT, DUAL>) % 8 == 0, "what follows the rows is aligned");
    extern __shared__ __align__(16) unsigned char raw[];
    const int g = NT == 32 ? (int) threadIdx.x >> 5 : 0;
    const int blocks = NT == 32 ? 1 : (int) cg::this_cluster().num_blocks(), rank = NT == 32 ? 0 : (int) cg::this_cluster().block_rank();
    const long long seq = NT == 32 ? (long long) blockIdx.x * GROUPS + g : (long long) (blockIdx.x / blocks);
    if (NT == 32 && seq >= a.sequences) return;                  // warps by themselves: nothing to meet
    float * rows_at = reinterpret_cast<float *>(raw) + (size_t) g * rows_each * row_floats;
    auto * states = reinterpret_cast<SeqSmem<NT, DUAL, FILTERS> *>(reinterpret_cast<float *>(raw) + (size_t) GROUPS * rows_each * row_floats);
    SeqSmem<NT, DUAL, FILTERS> & S = states[g];
    SeqBins<NT, DUAL> * B = reinterpret_cast<SeqBins<NT, DUAL> *>(states + GROUPS) + g;
    Team<G, false> group;
    group.tid = NT == 32 ? (int) threadIdx.x & 31 : (int) threadIdx.x;
    group.blocks = 1;
    group.rank = 0;
    group.phase = 0;
    group.s = &S.group;
    const int own = DUAL ? group.tid / NT : 0;                   // this thread's row
    Team<NT, false, DUAL> team;
    team.tid = DUAL ? group.tid % NT : group.tid;
    team.blocks = 1;
    team.rank = 0;
    team.phase = 0;
    team.s = &S.team[own];
    team.bar = 1 + own;
    team.mine = table_entry(team.lane());
    group.mine = team.mine;

    const int d = a.max_drafts, n = drafts_of(a, seq), v = a.vocab;
    const int32_t * drafts = a.drafts + seq * d;
    const float * u = a.uniforms + seq * (d + 1);
    int32_t * tokens = a.tokens + seq * (d + 1);
    float * logprobs = a.logprobs ? a.logprobs + seq * (d + 1) : nullptr;
    const float temp_f = temperature_of(a, seq);
    const double temp = (double) temp_f;
    const int g_len = run_of<G>(v), t_len = run_of<NT>(v);
    Slice<T, true> rows[2];
    auto slice = [&](int which, int pos) {
        Slice<T, true> & l = rows[which];
        l.gl = which == 0 ? static_cast<const T *>(a.logits) + (seq * (d + 1) + pos) * a.row_stride
                          : static_cast<const T *>(a.draft_logits) + (seq * d + pos) * a.draft_stride;
        l.n = v;
        l.sm = rows_at + which * row_floats;
        l.skew = (int) ((reinterpret_cast<uintptr_t>(l.gl) & 15) / sizeof(T)) & 3;
        l.inf = false;
        l.pad = max(((l.skew + v + 3) & ~3) - l.skew, max(NT * t_len, G * g_len));
    };
    enum { kAccepted, kRejected, kEnd };
    for (int base = 0, round = 0;; base += blocks, ++round) {
        const int pos = base + rank;
        const bool two = a.draft_logits && pos < n;
        int code = kAccepted, draft = -1;
        float quick_log = CUDART_INF_F;
        if (pos <= n) {
            if (pos < n) draft = drafts[pos];
            slice(0, pos);
            if (two) slice(1, pos);
            bool open = true;                                    // whether the draft stands
            if constexpr (!FILTERS) {
                if (pos < n && draft >= 0 && draft < v && temp_f > 0.0f) {
                    if (!DUAL || own == 0 || two) {
                        for (int i = 0; i < (DUAL || !two ? 1 : 2); ++i) {
                            const int which = DUAL ? own : i;
                            const double sum = quick_sum<T, NT>(team, rows[which].gl, v, draft, temp_f);
                            if (team.tid == 0) S.quick[which] = sum;
                        }
                    }
                    group.sync();
                    // u q(d) < p(d) by more than the sums are off by, twice
                    const double p = S.quick[0], q = two ? S.quick[1] : 1.0;
                    open = !(p < 0x1p24 && q < 0x1p24 && (double) number_of(u[pos]) * p * (1.0 + 4.0 * kQuick) < q);
                    if (!open && logprobs && group.tid == 0) quick_log = fminf(-logf((float) p), 0.0f);
                    group.sync();
                }
            }
            if (open) {
                if (!DUAL || own == 0 || two) {
                    const int end = DUAL || !two ? 1 : 2;
                    for (int i = 0; i < end; ++i) load_slice<T, NT>(rows[DUAL ? own : i], team.tid);
                    team.sync();
                    for (int i = 0; i < end; ++i) {
                        const int which = DUAL ? own : i;
                        row_stat<T, NT, FILTERS>(team, &B->bins[own], rows[which], a, seq, draft, &S.st[which]);
                        if (end > 1) team.sync();
                    }
                }
                group.sync();
                if constexpr (FILTERS) {
                    // see rank_of; the statistics are not changed before all threads have looked
                    const int k = a.top_ks ? a.top_ks[seq] : a.top_k;
                    auto low = [&](const RowStat & st) { return !(st.flags & kGreedy) && !(st.cut > -CUDART_INF_F) && st.drafted > 0.0 && st.drafted < 0x1p-44; };
                    if (k > 0 && k < v && (low(S.st[0]) || (two && low(S.st[1])))) {
                        group.sync();
                        if (!DUAL || own == 0 || two)
                            for (int i = 0; i < (DUAL || !two ? 1 : 2); ++i) {
                                const int which = DUAL ? own : i;
                                const u64 rank = rank_of(team, rows[which], 0, draft, rows[which](draft));
                                if (team.tid == 0 && rank >= (u64) k && low(S.st[which])) S.st[which].drafted = 0.0;
                            }
                        group.sync();
                    }
                }
            }
            if (!open) {
                code = kAccepted;
            } else if (pos == n) {
                code = kEnd;
            } else {
                // u q(d) < p(d), as u w_q(d) P < w_p(d) Q; f32 sums may leave it open
                const bool inside = draft >= 0 && draft < v;
                const double x = (double) number_of(u[pos]);
                auto sides = [&](double & l, double & r) {
                    const RowStat & p = S.st[0], & q = S.st[1];
                    l = two ? x * q.drafted * (double) p.total : inside ? x * (double) p.total * (1.0 / kOne) : 0.0;
                    r = two ? p.drafted * (double) q.total : p.drafted;
                    // no logit in the draft's row: its tokens have no probability
                    if (two && q.total == 0) { l = 0.0; r = p.drafted; }
                    if (p.total == 0) r = 0.0;
                };
                double l, r;
                sides(l, r);
                const int near = (S.st[0].flags | (two ? S.st[1].flags : 0)) & kNear;
                if (near && fmax(l, r) > 0.0 && fabs(l - r) <= 5.0 * kOff * fmax(l, r)) {
                    group.sync();
                    if (!DUAL || own == 0 || two)
                        for (int i = 0; i < (DUAL || !two ? 1 : 2); ++i) settle<T, NT>(team, rows[DUAL ? own : i], temp, &S.st[DUAL ? own : i]);
                    group.sync();
                    sides(l, r);
                }
                code = l < r ? kAccepted : kRejected;
            }
        }
        int first = code != kAccepted ? 0 : -1;                  // of the blocks, the first that did not accept
        if (NT > 32 && blocks > 1) {
            if (group.tid == 0) S.code[round & 1] = code;
            cg::this_cluster().sync();
            int its = kAccepted;
            if (group.lane() < blocks) its = *cg::this_cluster().map_shared_rank(&S.code[round & 1], group.lane());
            const unsigned not_accepted = __ballot_sync(kFull, its != kAccepted);
            first = not_accepted ? __ffs((int) not_accepted) - 1 : -1;
        }
        if (code == kAccepted && pos < n && (first < 0 || rank < first) && group.tid == 0) {
            tokens[pos] = draft;
            if (logprobs)
                logprobs[pos] = !FILTERS && quick_log < CUDART_INF_F ? quick_log : logprob_of(rows[0](draft), S.st[0], S.st[0].flags & kGreedy ? 1.0 : temp);
        }
        if (first < 0) {
            group.sync();                                        // the rows' memory is read
            continue;
        }
        // a block's codes stay while others may read them
        __syncwarp();
        if (NT > 32 && blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (rank == first) {
            for (int j = pos + 1 + group.tid; j <= d; j += G) {
                tokens[j] = -1;
                if (logprobs) logprobs[j] = -CUDART_INF_F;
            }
            if (group.tid == 0) a.accepted[seq] = pos;
            int mode = kAll;
            if (code == kRejected) mode = two ? (S.st[1].total ? kLess : kAll) : a.draft_logits ? kAll : kWithout;
            const double heat = S.st[0].flags & kGreedy ? 1.0 : temp;
            if (S.st[0].total == 0) {                            // nothing to draw from
                if (group.tid == 0) {
                    tokens[pos] = -1;
                    if (logprobs) logprobs[pos] = -CUDART_INF_F;
                }
            } else if (!draw_near<T, G>(group, rows[0], rows[1], S.st, mode, draft, temp_f, u[d], tokens + pos, logprobs ? logprobs + pos : nullptr)) {
                if (mode == kLess) {
                    for (int i = 0; i < (DUAL ? 1 : 2); ++i) settle<T, NT>(team, rows[DUAL ? own : i], temp, &S.st[DUAL ? own : i]);
                }
                if (group.tid == 0) S.group.found = -1;
                group.sync();
                const RowStat p = S.st[0], q = S.st[1];
                const Row pr = row_of(p.hi, heat), qr = row_of(mode == kLess ? q.hi : 0.0f, heat);
                const double sp = kShare / (double) p.total, sq = mode == kLess ? kShare / (double) q.total : 0.0;
                // what token i weighs in the draw, a whole number; the whole warp calls
                const bool p_cut = p.last != kAny, q_cut = q.last != kAny;
                auto weigh = [&](int i, bool in) -> double {
                    const float x = in ? rows[0](i) : -CUDART_INF_F;
                    bool keep = x >= p.from;
                    if (p_cut) keep = keep && (x > p.cut || i <= p.last);
                    if (mode == kWithout) keep = keep && i != draft;
                    if (FILTERS && !__any_sync(kFull, keep)) return 0.0;
                    double w = weight_warp(x, pr, team.mine) - kZero;
                    if (mode == kLess) {
                        const float y = in ? rows[1](i) : -CUDART_INF_F;
                        bool less = y >= q.from;
                        if (q_cut) less = less && (y > q.cut || i <= q.last);
                        const double z = weight_warp(y, qr, team.mine) - kZero;
                        // the two products rounded alike: equal rows leave nothing
                        w = __dmul_rn(w, sp) - (less ? __dmul_rn(z, sq) : 0.0);
                        w = (w + kMagic) - kMagic;
                        keep = keep && w > 0.0;
                    }
                    return keep ? w : 0.0;
                };
                const int i0 = group.tid * g_len;
                u64 total = 0, before = 0, sum = 0;
                for (;;) {
                    // a thread's run: fewer than 2^9 weights of 2^43 at most, or shares of 2^50 in all
                    double run = 0.0;
#pragma unroll 4
                    for (int j = 0; j < g_len; ++j) run += weigh(i0 + j, i0 + j < v);
                    sum = (u64) run;
                    before = group.scan(sum, total);
                    if (total > 0 || mode == kAll) break;
                    mode = kAll;                                 // q has all that p has: only a draft that q never draws ends here
                }
                const u64 t = place_of(u[d], total);
                if (before <= t && t < before + sum) {
                    S.group.found = group.tid;
                    S.group.found_before = before;
                }
                group.sync();
                const int who = S.group.found;
                if (who >= 0 && group.tid < 32) {
                    // the run again, 32 elements at a time
                    const int e = min((who + 1) * g_len, v);
                    u64 run = S.group.found_before;
                    for (int c = who * g_len; c < e; c += 32) {
                        const int i = c + group.tid;
                        const u64 w = (u64) weigh(i, i < e), upto = run + warp_scan(w, group.tid);
                        if (upto - w <= t && t < upto) {
                            const float x = rows[0](i);
                            tokens[pos] = i;
                            if (logprobs) logprobs[pos] = logprob_of(x, p, heat);
                        }
                        run = __shfl_sync(kFull, upto, 31);
                        if (run > t) break;
                    }
                }
            }
        }
        if (NT > 32 && blocks > 1) {
            __syncwarp();
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
        return;
    }
}

template <class T, int NT, bool DUAL, bool FILTERS>
cudaError_t launch_sequences(const pk_verify_args & a, int blocks, cudaStream_t s) {
    constexpr int G = group_of<NT, DUAL>(), GROUPS = NT == 32 ? kSeqGroups : 1;
    const int rows_each = a.draft_logits ? 2 : 1;
    const int row_floats = (std::max({a.vocab, NT * run_of<NT>(a.vocab), G * run_of<G>(a.vocab)}) + 3 + 3) / 4 * 4;
    const size_t smem = GROUPS * ((size_t) rows_each * row_floats * 4 + sizeof(SeqSmem<NT, DUAL, FILTERS>) + (FILTERS ? sizeof(SeqBins<NT, DUAL>) : 0));
    auto kernel = verify_sequence_kernel<T, NT, DUAL, FILTERS>;
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
    cfg.gridDim = dim3((unsigned) (NT == 32 ? (a.sequences + GROUPS - 1) / GROUPS : a.sequences * blocks));
    cfg.blockDim = dim3(NT == 32 ? 32 * GROUPS : G);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    if (NT > 32) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned) blocks;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, a, rows_each, row_floats);
}

// Whether the kernel above can hold a position's rows: beside them there are up to 2048 logits' room in front of and
// behind each, and 25 KB of the teams'.
bool resident(int vocab, bool two) { return vocab <= (two ? kResident / 2 : kResident); }

template <class T, bool FILTERS, int NT> cudaError_t sequences_block(const pk_verify_args & a, cudaStream_t s) {
    // The blocks of a cluster share the positions out while there is room for them (four drafts by 8193, temperature alone, 64
    // sequences in clusters of 4, 2 and 1: 25.5 us, 25.9, 26.9; of 5, which no longer all run at once, 29.8). With filters a
    // position takes longer and more blocks than there is room for still pay (64 sequences, settings mixed: of 5 37.6 us, of 4
    // 41.1, of 1 85; 256 of eight drafts, top-p: of 2 120 us, of 1 136; 300: 155 and 159).
    const long long room = 148 * std::max(1, 1024 / (2 * NT)), share = (FILTERS ? room * 7 / 4 : room) / std::max<long long>(1, a.sequences);
    const int blocks = (int) std::max<long long>(1, std::min<long long>({FILTERS ? kMaxCluster : 4, (long long) a.max_drafts + 1, share}));
    if (a.draft_logits) return launch_sequences<T, NT, true, FILTERS>(a, blocks, s);
    return launch_sequences<T, NT <= 256 ? 2 * NT : NT, false, FILTERS>(a, blocks, s);
}

// Replayed from a graph, four drafts a sequence. A warp per sequence for many short rows (by 1025, a warp and two teams of 128
// threads: 2000 sequences, temperature alone, 45 us and 50; top-k 173 and 199; min-p 48 and 65; by 300 27 and 46, 142 and 200, 35
// and 63. But top-p 203 and 143, and of 592 sequences, where it begins, 41 and 20, so that the teams would be sooner up to some
// 1500). Otherwise two teams of 128 for short rows (128 and 256: 400 by 4000, temperature alone, 29 us and 36, by 6100 39 and 45,
// by 8193 46 and 54, but 64 by 8193 29 and 25; top-p, 400 by 2040 63 and 70, by 4000 104 and 93), of 512 for long ones (256 and
// 512: temperature alone, 300 by 12000 49 us and 68, by 16000 76 and 79, by 19000 94 and 90; top-p, 64 by 8193 55 and 62, by
// 12000 97 and 71, 300 by 12000 169 and 175, by 16000 235 and 212) and for few with filters (8 by 8193, top-p: 34 us and 25), of
// 256 in between.
template <class T, bool FILTERS> cudaError_t sequences_dispatch(const pk_verify_args & a, cudaStream_t s) {
    if (a.vocab <= kWarpMost && a.sequences >= 4 * 148) return launch_sequences<T, 32, false, FILTERS>(a, 1, s);
    if (a.vocab <= (FILTERS ? 2048 : k128Most)) return sequences_block<T, FILTERS, 128>(a, s);
    if (FILTERS ? a.vocab > 12288 || a.sequences * (a.max_drafts + 1) <= 148 : a.vocab > k256Most) return sequences_block<T, FILTERS, 512>(a, s);
    return sequences_block<T, FILTERS, 256>(a, s);
}

// ---- long rows ---------------------------------------------------------------------
//
// Two kernels (4 sequences of eight looked-up drafts by 131072 bf16: 27 us, two launches and the draw's passes over one row,
// 16,384 logits a block; of two models 61; with top-p 117 and 154, with top-k 61 and 90; 32 of four by 50000 f32, two models, 49,
// with top-p 125). The first takes a block or cluster per row, all rows at once, and leaves what the test needs of it; with filters
// as pk_sample does. The second takes a block or cluster per sequence: it tests all drafts at once and draws from the one row, or
// two, that the first rejection names, reading them again. But at T <= 0 without filters the first tells nothing, and the second
// settles the positions one after the other, two passes over each row of theirs: 4 sequences of eight looked-up drafts by 131072
// bf16 take 36 us where the first is rejected, 129 where all are accepted, of two models 61 and 211.

struct Plan {
    pk_verify_args a;
    RowStat * stats;      // [sequences][max_drafts + 1] of the target, [sequences][max_drafts] of the draft
};

template <class T, int NT, bool CL, bool RES>
__global__ void __launch_bounds__(NT, 1024 / NT) verify_rows_kernel(const Plan plan, int slice, int row_floats) {
    extern __shared__ __align__(16) unsigned char raw[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const pk_verify_args & a = plan.a;
    Team<NT, CL> team;
    team.tid = (int) threadIdx.x;
    team.blocks = CL ? (int) cg::this_cluster().num_blocks() : 1;
    team.rank = CL ? (int) cg::this_cluster().block_rank() : 0;
    team.phase = 0;
    const long long id = (long long) (blockIdx.x / team.blocks);
    const long long targets = a.sequences * (a.max_drafts + 1);
    const bool target = id < targets;
    const long long at = target ? id : id - targets;
    const int per = target ? a.max_drafts + 1 : a.max_drafts;
    if (id >= targets + (a.draft_logits ? a.sequences * a.max_drafts : 0)) return;
    const long long seq = at / per;
    const int pos = (int) (at - seq * per), n = drafts_of(a, seq);
    if (target ? pos > n : pos >= n) return;                     // behind the last draft
    float * rows_at = reinterpret_cast<float *>(raw);
    team.s = reinterpret_cast<TeamSmem<NT> *>(rows_at + row_floats);
    TeamBins<NT> * bins = reinterpret_cast<TeamBins<NT> *>(team.s + 1);
    team.mine = table_entry(team.lane());
    const int s0 = min(team.rank * slice, a.vocab);
    const T * row_at = target ? static_cast<const T *>(a.logits) + at * a.row_stride : static_cast<const T *>(a.draft_logits) + at * a.draft_stride;
    Slice<T, RES> l;
    l.n = min(slice, a.vocab - s0);
    l.gl = row_at + s0;
    l.sm = rows_at;
    l.skew = RES ? (int) ((reinterpret_cast<uintptr_t>(l.gl) & 15) / sizeof(T)) & 3 : 0;
    l.inf = false;
    const int len = run_of<NT>(l.n);
    l.pad = max(((l.skew + l.n + 3) & ~3) - l.skew, NT * len);
    if constexpr (RES) {
        load_slice<T, NT>(l, team.tid);
        team.sync();
    }
    const float temp_f = temperature_of(a, seq);
    const double temp = (double) temp_f;
    float hi = -CUDART_INF_F, lo = CUDART_INF_F;                 // fmaxf and fminf pass over NaN
    l.template each<NT>(team.tid, [&](float v, int) {
        hi = fmaxf(hi, v);
        if (v > -CUDART_INF_F) lo = fminf(lo, v);
    });
    team.template range<true>(hi, lo);
    RowStat * out = plan.stats + id;
    const int draft = pos < n ? a.drafts[seq * a.max_drafts + pos] : -1;
    const bool one = team.tid == 0 && team.rank == 0;
    RowStat st;
    st.drafted = 0.0;
    st.flags = hi == CUDART_INF_F ? kInf : 0;
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
        if (one) {
            st.flags |= kGreedy;
            st.hi = st.from = st.cut = st.flags & kInf ? 0.0f : hi;
            st.last = (int) min(first, (u64) kAny);
            st.total = first == ~0ull ? 0ull : (u64) kOne;
            st.drafted = first != ~0ull && draft == (int) first ? 1.0 : 0.0;
            *out = st;
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
    const Row r = row_of(hi, temp);
    float least = r.base;                                        // kept: >= least, and what the cut says
    float cut = -CUDART_INF_F;
    u64 ties = ~0ull, total = 0;
    bool partial = false;
    const float m = a.min_ps ? a.min_ps[seq] : a.min_p;
    const bool inside = draft >= 0 && draft < a.vocab;
    bool beyond = false;                                         // the draft is not among the first k
    auto leave = [&](float from, float cut_at, int last, u64 sum) {
        st.hi = hi;
        st.from = from;
        st.cut = cut_at;
        st.last = last;
        st.total = sum;
        if (inside && !beyond) st.drafted = draft_weight(seen(to_f32(row_at[draft]), st.flags), draft, st, r, temp, m);
        *out = st;
    };
    const float p = a.top_ps ? a.top_ps[seq] : a.top_p;
    const int k = a.top_ks ? a.top_ks[seq] : a.top_k;
    const bool done = cut_row<T, NT, CL, RES>(team, bins, l, s0, r, hi, lo, temp_f, a.vocab, k, p, m, least, cut, ties, partial,
        [&](const Pair * list, int count, int first, float share, u64 need) {
            keep_listed(team, bins, list, count, r, first, share, need, least,
                        [&](float v, int i, u64 sum) { if (team.rank == 0) leave(v, v, i, sum); });
        },
        [](double) { return false; });
    if (done) {
        if (CL) team.meet();
        return;
    }
    if (inside && k > 0 && k < a.vocab && !(cut > -CUDART_INF_F)) {
        const float v = seen(to_f32(row_at[draft]), st.flags);
        if (v < r.base && v > -CUDART_INF_F) beyond = rank_of(team, l, s0, draft, v) >= (u64) k;   // the same for all threads
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
        if (partial && v == cut) {
            ++equal;
            keep = false;
        }
        if (!__any_sync(kFull, keep)) continue;
        const double w = weight_warp(v, r, team.mine, onto);
        if (keep) onto = w;
    }
    u64 sum = whole(onto);
    bool mine = false;                                           // the last of the ties that are kept is in this run
    u64 before = 0;
    if (partial) {
        u64 all;
        before = team.scan((u64) equal, all);
        if (cut >= least && before < ties) sum += min((u64) equal, ties - before) * weight_one(cut, r);
        mine = before < ties && ties <= before + equal;
    }
    total = team.sum(sum);
    if (partial) {
        if (mine) {
            int i = i0;
            for (u64 left = ties - before; i < i1; ++i)
                if (l(i) == cut && --left == 0) break;
            leave(from, cut, s0 + i, total);
        }
    } else if (one) {
        leave(from, cut, kAny, total);
    }
    if (CL) team.meet();                                         // a block's memory stays while others may read it
}

// ---- the drafts' test and the draw ------------------------------------------------

// A row as the draw reads it.
template <class T> struct DrawRow {
    const T * at;
    Row r;
    float from, cut;
    int last, flags;
    __device__ __forceinline__ void set(const T * row, const RowStat & s, float temp) {
        at = row;
        flags = s.flags;
        from = s.from;
        cut = s.cut;
        last = s.last;
        r = row_of(s.hi, flags & kGreedy ? 1.0 : (double) temp);
    }
    // Whether token i is kept, its logit as `seen` has it.
    __device__ __forceinline__ bool keeps(float v, int i) const { return v >= from && (v > cut || i <= last); }
    // Weight of token i with logit v (times 2^43, a whole number); the whole warp calls.
    __device__ __forceinline__ double weight(float v, int i, double mine) const {
        v = seen(v, flags);
        const bool keep = keeps(v, i);
        const double w = weight_warp(keep ? v : (float) r.top, r, mine) - kZero;
        return keep ? w : 0.0;
    }
};

constexpr int kDrawThreads = 512;
constexpr int kDrawWarps = kDrawThreads / 32;

// Without filters the test takes 1 / p(d) by f32, see quick_part: a block or cluster per row and draft, the sum to
// `drafted` of the row's place.
template <class T, bool CL>
__global__ void __launch_bounds__(kDrawThreads) verify_sums_kernel(const Plan plan) {
    const pk_verify_args & a = plan.a;
    __shared__ float sums[kDrawWarps];
    __shared__ float its;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x;
    const int blocks = CL ? (int) cg::this_cluster().num_blocks() : 1, rank = CL ? (int) cg::this_cluster().block_rank() : 0;
    const long long id = blockIdx.x / blocks, drafts = a.sequences * a.max_drafts;
    const long long at = id < drafts ? id : id - drafts, seq = at / a.max_drafts;
    const int pos = (int) (at - seq * a.max_drafts), draft = a.drafts[at], v = a.vocab;
    if (pos >= drafts_of(a, seq)) return;                        // behind the last draft
    const T * row = id < drafts ? static_cast<const T *>(a.logits) + (seq * (a.max_drafts + 1) + pos) * a.row_stride
                                : static_cast<const T *>(a.draft_logits) + at * a.draft_stride;
    const float temp_f = temperature_of(a, seq), c = 1.4426950408889634f * (1.0f / temp_f);
    const bool inside = draft >= 0 && draft < v;
    const float l = inside ? to_f32(row[draft]) : CUDART_NAN_F, k = l * c;
    const bool fine = temp_f > 0.0f && c > 1e-30f && c < 1e30f && fabsf(k) < 1e6f;    // the same for all
    const int slice = ((v + blocks - 1) / blocks + 31) & ~31, s0 = min(rank * slice, v);
    float sum = fine ? quick_part<T, kDrawThreads>(row + s0, min(slice, v - s0), tid, c, k) : 0.0f;
    sum = warp_sum(sum);
    if ((tid & 31) == 0) sums[tid >> 5] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kDrawWarps; ++i) sum += sums[i];
    if (CL) {
        if (tid == 0) its = sum;
        cg::this_cluster().sync();
        sum = 0.0f;
        for (int b = 0; b < blocks; ++b) sum += *cg::this_cluster().map_shared_rank(&its, b);
        cg::this_cluster().sync();                               // its memory stays while others read it
    }
    float own;                                                   // the draft's own weight: one, but for the rounding of k
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(own) : "f"(fmaf(l, c, -k)));
    const long long place = id < drafts ? seq * (a.max_drafts + 1) + pos : a.sequences * (a.max_drafts + 1) + at;
    if (tid == 0 && rank == 0) plan.stats[place].drafted = fine ? (double) (sum / own) : (double) CUDART_NAN_F;
}

// FILTERS: the rows' statistics are there. Otherwise the test's sums are, and what else is needed of the few rows that
// it leaves open, or that are drawn from, is found here.
template <class T, bool CL, bool FILTERS>
__global__ void __launch_bounds__(kDrawThreads) verify_draw_kernel(const Plan plan) {
    const pk_verify_args & a = plan.a;
    __shared__ u64 sums[kDrawWarps];
    __shared__ u64 exchange[2];
    __shared__ int s_first, s_warp;
    __shared__ u64 s_before;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = CL ? (int) cg::this_cluster().num_blocks() : 1, rank = CL ? (int) cg::this_cluster().block_rank() : 0;
    const long long seq = blockIdx.x / blocks;
    const int d = a.max_drafts, n = drafts_of(a, seq), v = a.vocab;
    unsigned phase = 0;                                  // the exchanges take turns
    if (tid == 0) s_first = n;
    const double mine = table_entry(lane);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    const RowStat * ps = plan.stats + seq * (d + 1), * qs = plan.stats + a.sequences * (d + 1) + seq * d;
    const int32_t * drafts = a.drafts + seq * d;
    const float * u = a.uniforms + seq * (d + 1);
    const float temp = temperature_of(a, seq);
    auto target_row = [&](int j) { return static_cast<const T *>(a.logits) + (seq * (d + 1) + j) * a.row_stride; };
    auto draft_row = [&](int j) { return static_cast<const T *>(a.draft_logits) + (seq * d + j) * a.draft_stride; };
    // over all threads of all blocks
    auto join_all = [&](u64 x, auto join) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x = join(x, __shfl_xor_sync(kFull, x, o));
        __syncthreads();
        if (lane == 0) sums[warp] = x;
        __syncthreads();
        x = sums[0];
#pragma unroll
        for (int i = 1; i < kDrawWarps; ++i) x = join(x, sums[i]);
        if (CL) {
            if (tid == 0) exchange[phase] = x;
            cg::this_cluster().sync();
            for (int b = 0; b < blocks; ++b) x = b == 0 ? *cg::this_cluster().map_shared_rank(&exchange[phase], 0)
                                                        : join(x, *cg::this_cluster().map_shared_rank(&exchange[phase], b));
            phase ^= 1;
        }
        return x;
    };
    const int all = kDrawThreads * blocks, me = rank * kDrawThreads + tid;
    // a row's statistics by whole numbers, where nothing is cut; the same for every thread. Without `sum` the total is only
    // known to be more than nothing.
    auto stat_of = [&](const T * row, int draft, bool with_sum) {
        RowStat st;
        st.drafted = 0.0;
        st.last = kAny;
        float hi = -CUDART_INF_F;                        // fmaxf passes over NaN
#pragma unroll 8
        for (int i = me; i < v; i += all) hi = fmaxf(hi, to_f32(row[i]));
        hi = __uint_as_float((unsigned) join_all((u64) __float_as_uint(hi), [](u64 x, u64 y) {
            return (u64) __float_as_uint(fmaxf(__uint_as_float((unsigned) x), __uint_as_float((unsigned) y)));
        }));
        st.flags = hi == CUDART_INF_F ? kInf : 0;
        if (hi == -CUDART_INF_F || !(temp > 0.0f)) {
            u64 first = (u64) kAny;                      // nothing to draw, or the first index of the largest
            if (hi > -CUDART_INF_F)
                for (int i = me; i < v && first == (u64) kAny; i += all)
                    if (to_f32(row[i]) == hi) first = (u64) i;
            first = join_all(first, [](u64 x, u64 y) { return min(x, y); });
            st.flags |= kGreedy;
            st.hi = st.from = st.cut = st.flags & kInf ? 0.0f : hi;
            st.last = (int) first;
            st.total = first == (u64) kAny ? 0ull : (u64) kOne;
            if (first != (u64) kAny && draft == (int) first) st.drafted = 1.0;
            return st;
        }
        if (st.flags & kInf) hi = 0.0f;
        const Row r = row_of(hi, (double) temp);
        st.hi = hi;
        st.from = r.base;
        st.cut = -CUDART_INF_F;
        st.total = 1;
        if (!with_sum) return st;
        u64 sum = 0;
        for (int i = me; i - lane < v; i += 8 * all) {   // eight loads on their way
            float x[8];
            double onto = kZero;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = i + j * all < v ? seen(to_f32(row[i + j * all]), st.flags) : -CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double w = weight_warp(x[j], r, mine, onto);
                if (x[j] >= r.base) onto = w;
            }
            sum += whole(onto);
        }
        st.total = join_all(sum, [](u64 x, u64 y) { return x + y; });
        if (draft >= 0 && draft < v) st.drafted = draft_weight(seen(to_f32(row[draft]), st.flags), draft, st, r, (double) temp, 0.0f);
        return st;
    };
    auto less = [&](const RowStat & p, const RowStat * q, int j) {   // u q(d) < p(d)
        const double pd = p.total ? p.drafted / ((double) p.total * (1.0 / kOne)) : 0.0;
        const double qd = q ? (q->total ? q->drafted / ((double) q->total * (1.0 / kOne)) : 0.0) : drafts[j] >= 0 && drafts[j] < v ? 1.0 : 0.0;
        return (double) number_of(u[j]) * qd < pd;
    };
    // the test's answer: 1 accepted, -1 rejected, 0 open; the sums' errors as for quick_part, of slices over 512 threads
    auto told = [&](int j) {
        const double sp = ps[j].drafted, sq = a.draft_logits ? qs[j].drafted : 1.0;
        if (!(sp < 0x1p24 && sq < 0x1p24)) return 0;
        const double edge = 0x1p-23 * (double) (16.0f + 2.78f * (2.0f * log2f((float) v) + log2f((float) sp) + log2f((float) sq)) +
                                                2.0f * ((float) v * (1.0f / (4.0f * kDrawThreads)) + 24.0f + 9.0f));
        const double l = (double) number_of(u[j]) * sp;
        return l * (1.0 + edge) < sq ? 1 : l > sq * (1.0 + edge) ? -1 : 0;
    };
    auto logprob_at = [&](int j, float x) { if (a.logprobs) a.logprobs[seq * (d + 1) + j] = fminf(x, 0.0f); };
    RowStat p, q;
    int first = 0;
    for (;;) {
        // the first from `first` on that is not accepted
        for (int j = first + tid; j < n; j += kDrawThreads)
            if (FILTERS ? !less(ps[j], a.draft_logits ? qs + j : nullptr, j) : told(j) < 1) atomicMin(&s_first, j);
        __syncthreads();
        const int until = s_first;
        if (rank == 0) {
            for (int j = first + tid; j < until; j += kDrawThreads) {
                a.tokens[seq * (d + 1) + j] = drafts[j];
                logprob_at(j, FILTERS ? (float) (log(ps[j].drafted) - log((double) ps[j].total * (1.0 / kOne))) : -logf((float) ps[j].drafted));
            }
        }
        first = until;
        if (FILTERS) {
            p = ps[first];
            if (first < n && a.draft_logits) q = qs[first];
            break;
        }
        const bool rejected = first < n && told(first) < 0;
        p = stat_of(target_row(first), first < n ? drafts[first] : -1, first < n && (a.draft_logits || !rejected));
        if (first == n) break;
        if (a.draft_logits) q = stat_of(draft_row(first), drafts[first], true);
        if (rejected || !less(p, a.draft_logits ? &q : nullptr, first)) break;
        if (rank == 0 && tid == 0) {
            a.tokens[seq * (d + 1) + first] = drafts[first];
            logprob_at(first, (float) (log(p.drafted) - log((double) p.total * (1.0 / kOne))));
        }
        ++first;
        __syncthreads();
        if (tid == 0) s_first = n;
        __syncthreads();
    }
    if (rank == 0) {
        for (int j = first + 1 + tid; j <= d; j += kDrawThreads) {
            a.tokens[seq * (d + 1) + j] = -1;
            logprob_at(j, -CUDART_INF_F);
        }
        if (tid == 0) a.accepted[seq] = first;
    }
    if (p.total == 0) {                                  // nothing to draw from
        if (rank == 0 && tid == 0) {
            a.tokens[seq * (d + 1) + first] = -1;
            logprob_at(first, -CUDART_INF_F);
        }
        if (CL && !FILTERS) cg::this_cluster().sync();   // exchanges are read
        return;
    }
    DrawRow<T> pr, qr;
    pr.set(target_row(first), p, temp);
    int mode = kAll, out = -1;
    double sp = 0.0, sq = 0.0;
    if (first < n) {
        if (a.draft_logits) {
            if (q.total) {
                mode = kLess;
                qr.set(draft_row(first), q, temp);
                sp = kShare / (double) p.total;
                sq = kShare / (double) q.total;
            }
        } else {
            out = drafts[first];
            mode = kWithout;
        }
    }
    // what token i, of logits x and y in the two rows, weighs in the draw, a whole number; the whole warp calls
    auto weigh = [&](int i, float x, float y) {
        double w = pr.weight(x, i, mine);
        if (mode == kLess) {
            // the two products rounded alike: equal rows leave nothing
            w = fmax((__dmul_rn(w, sp) - __dmul_rn(qr.weight(y, i, mine), sq) + kMagic) - kMagic, 0.0);
        }
        return mode == kWithout && i == out ? 0.0 : w;
    };
    auto target_at = [&](int i, int end) { return i < end ? to_f32(pr.at[i]) : -CUDART_INF_F; };
    auto draft_at = [&](int i, int end) { return mode == kLess && i < end ? to_f32(qr.at[i]) : -CUDART_INF_F; };
    auto stretch = [&](int begin, int end) {             // its sum, over a warp: eight loads of each row on their way
        u64 s = 0;
        for (int b = begin; b < end; b += 256) {
            const int i = b + lane;
            float x[8], y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = target_at(i + 32 * j, end);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = draft_at(i + 32 * j, end);
            double run = 0.0;                            // eight weights of 2^43, or shares of 2^50 in all
#pragma unroll
            for (int j = 0; j < 8; ++j) run += weigh(i + 32 * j, x[j], y[j]);
            s += (u64) run;
        }
        return warp_sum(s);
    };
    const int part = ((v + kDrawWarps * blocks - 1) / (kDrawWarps * blocks) + 31) & ~31;
    const int begin = min((rank * kDrawWarps + warp) * part, v), end = min(begin + part, v);
    u64 total = 0, before = 0;
    for (;;) {
        const u64 s = stretch(begin, end);
        __syncthreads();
        if (lane == 0) sums[warp] = s;
        __syncthreads();
        u64 own = 0;
        before = 0;
#pragma unroll
        for (int i = 0; i < kDrawWarps; ++i) {
            if (i < warp) before += sums[i];
            own += sums[i];
        }
        total = own;
        if (CL) {
            if (tid == 0) exchange[phase] = own;
            cg::this_cluster().sync();
            total = 0;
            for (int b = 0; b < blocks; ++b) {
                const u64 o = *cg::this_cluster().map_shared_rank(&exchange[phase], b);
                if (b < rank) before += o;
                total += o;
            }
            phase ^= 1;
        }
        if (total > 0 || mode == kAll) break;
        mode = kAll;                                     // q has all that p has: only a draft that q never draws ends here
    }
    const u64 t = place_of(u[d], total);
    u64 whole_row = p.total;
    if (!FILTERS && mode != kLess) {
        // the row's weights: those of the draw, and the draft's, which the draw leaves out, if the row keeps it (a greedy row keeps
        // the first of its largest alone)
        whole_row = total;
        if (mode == kWithout && out >= 0 && out < v) {
            const float l = seen(to_f32(pr.at[out]), pr.flags);
            if (pr.keeps(l, out)) whole_row += weight_one(l, pr.r);
        }
    }
    if (tid == 0) s_warp = -1;
    __syncthreads();
    if (lane == 0 && before <= t && t < before + sums[warp]) {
        s_warp = warp;
        s_before = before;
    }
    if (CL) cg::this_cluster().sync();                   // exchanges are read
    __syncthreads();
    const int who = s_warp;
    if (who < 0) return;                                 // another block's
    before = s_before;
    // the stretch parted over the warps again, then searched
    const int b0 = min((rank * kDrawWarps + who) * part, v), e0 = min(b0 + part, v);
    const int sub = ((part + kDrawWarps - 1) / kDrawWarps + 31) & ~31;
    const int b1 = min(b0 + warp * sub, e0), e1 = min(b1 + sub, e0);
    __syncthreads();
    const u64 s = stretch(b1, e1);
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    for (int i = 0; i < warp; ++i) before += sums[i];
    if (!(before <= t && t < before + s)) return;
    for (int i = b1; i < e1; i += 32) {
        const u64 w = (u64) weigh(i + lane, target_at(i + lane, e1), draft_at(i + lane, e1));
        const u64 x = before + warp_scan(w, lane);
        if (x - w <= t && t < x) {
            const float l = seen(to_f32(pr.at[i + lane]), pr.flags);
            a.tokens[seq * (d + 1) + first] = i + lane;
            const double tt = pr.flags & kGreedy ? 1.0 : (double) temp;
            logprob_at(first, (float) ((l == p.hi ? 0.0 : ((double) l - (double) p.hi) / tt) - log((double) whole_row * (1.0 / kOne))));
        }
        before = __shfl_sync(kFull, x, 31);
        if (before > t) break;
    }
}

// ---- launches -----------------------------------------------------------------------

template <class T, int NT, bool CL, bool RES>
cudaError_t launch_rows(const Plan & p, long long rows, int blocks, int slice, int row_floats, size_t smem, cudaStream_t s) {
    auto kernel = verify_rows_kernel<T, NT, CL, RES>;
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
    cfg.gridDim = dim3((unsigned) (rows * blocks));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    if (CL) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned) blocks;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, p, slice, row_floats);
}

template <class T>
cudaError_t rows_cluster(const Plan & p, long long rows, int blocks, cudaStream_t s) {
    // slices of whole 16 bytes, so that every slice is aligned as its row is
    const int slice = ((p.a.vocab + blocks - 1) / blocks + 31) / 32 * 32;
    int row_floats;
    const size_t smem = team_bytes<1024, true>(slice, row_floats);
    if (smem <= kSmemCap) return launch_rows<T, 1024, true, true>(p, rows, blocks, slice, row_floats, smem, s);
    return launch_rows<T, 1024, true, false>(p, rows, blocks, slice, 0, smem - (size_t) row_floats * 4, s);
}

// Blocks by rows and vocabulary as in pk_sample.
template <class T>
cudaError_t rows_dispatch(const Plan & p, cudaStream_t s) {
    const int v = p.a.vocab;
    const long long rows = p.a.sequences * (p.a.max_drafts + 1) + (p.a.draft_logits ? p.a.sequences * p.a.max_drafts : 0);
    int blocks = 1;
    while (blocks < kMaxCluster && rows * blocks * 2 <= 148) blocks *= 2;
    while (blocks < kMaxCluster && (size_t) (v / blocks) * 4 > 200 * 1024) blocks *= 2;
    if (blocks > 1) return rows_cluster<T>(p, rows, blocks, s);
    int row_floats;
    const size_t smem = team_bytes<512, true>(v, row_floats);
    return launch_rows<T, 512, false, true>(p, rows, 1, v, row_floats, smem, s);
}

template <class T, bool CL, bool FILTERS>
cudaError_t launch_draw(const Plan & p, int blocks, bool behind, cudaStream_t s) {   // behind: a kernel that lets it start
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    cfg.gridDim = dim3((unsigned) (p.a.sequences * blocks));
    cfg.blockDim = dim3(kDrawThreads);
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned) blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = behind ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, verify_draw_kernel<T, CL, FILTERS>, p);
}

template <class T> cudaError_t launch_sums(const Plan & p, cudaStream_t s) {
    const long long rows = p.a.sequences * p.a.max_drafts * (p.a.draft_logits ? 2 : 1);
    int blocks = 1;
    while (blocks < kMaxCluster && rows * blocks * 2 <= 2 * 148) blocks *= 2;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.gridDim = dim3((unsigned) (rows * blocks));
    cfg.blockDim = dim3(kDrawThreads);
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned) blocks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = blocks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, blocks > 1 ? verify_sums_kernel<T, true> : verify_sums_kernel<T, false>, p);
}

template <class T, bool FILTERS> cudaError_t long_rows(const Plan & p, cudaStream_t s) {
    cudaError_t e;
    const bool rows = FILTERS || p.a.max_drafts > 0;             // the draw's own rows need no test
    if constexpr (FILTERS) e = rows_dispatch<T>(p, s);
    else e = rows ? launch_sums<T>(p, s) : cudaSuccess;
    if (e != cudaSuccess) return e;
    int blocks = 1;
    while (blocks < kMaxCluster && p.a.sequences * blocks * 2 <= 148) blocks *= 2;
    return blocks > 1 ? launch_draw<T, true, FILTERS>(p, blocks, rows, s) : launch_draw<T, false, FILTERS>(p, 1, rows, s);
}

template <class T> cudaError_t dispatch(const Plan & p, bool filters, cudaStream_t s) {
    if (resident(p.a.vocab, p.a.draft_logits != nullptr)) return filters ? sequences_dispatch<T, true>(p.a, s) : sequences_dispatch<T, false>(p.a, s);
    return filters ? long_rows<T, true>(p, s) : long_rows<T, false>(p, s);
}

// Rows of a call, -1 for sizes that are refused.
int64_t rows_of(int64_t sequences, int32_t max_drafts, int32_t vocab) {
    if (sequences < 0 || max_drafts < 0 || max_drafts > PK_VERIFY_MAX_DRAFTS || vocab < 1 || vocab > PK_SAMPLE_MAX_VOCAB) return -1;
    if (sequences > 0x7FFFFFFFll / kMaxCluster / (2 * max_drafts + 1)) return -1;
    return sequences * (2 * max_drafts + 1);
}

}  // namespace
}  // namespace pk

extern "C" PK_API int64_t pk_verify_workspace(int64_t sequences, int32_t max_drafts, int32_t vocab) {
    const int64_t rows = pk::rows_of(sequences, max_drafts, vocab);
    return rows < 0 ? -1 : pk::resident(vocab, true) ? 0 : rows * (int64_t) sizeof(pk::RowStat);
}

extern "C" PK_API pk_status pk_verify(int device, const pk_verify_args * a, void * stream) {
    using namespace pk;
    const char * fn = "pk_verify";
    if (!a) return op_fail(PK_ERR_INVALID, fn, "null arguments");
    const int es = elem_size(a->logits_type);
    if (es == 0) return op_fail(PK_ERR_INVALID, fn, "logits_type must be F32, F16 or BF16");
    if (a->vocab < 1 || a->vocab > PK_SAMPLE_MAX_VOCAB) return op_fail(PK_ERR_INVALID, fn, "vocab must be in [1, PK_SAMPLE_MAX_VOCAB]");
    const int64_t rows = rows_of(a->sequences, a->max_drafts, a->vocab);
    if (rows < 0)
        return op_fail(PK_ERR_INVALID, fn, "max_drafts must be in [0, PK_VERIFY_MAX_DRAFTS], sequences times 2 max_drafts + 1 in [0, 2^28)");
    if (a->row_stride < a->vocab || a->row_stride > (INT64_MAX >> 34) ||
        (a->draft_logits && (a->draft_stride < a->vocab || a->draft_stride > (INT64_MAX >> 34))))
        return op_fail(PK_ERR_INVALID, fn, "row_stride and draft_stride must be at least vocab");
    if (a->sequences > 0 && (!a->logits || !a->uniforms || !a->tokens || !a->accepted || (a->max_drafts > 0 && !a->drafts)))
        return op_fail(PK_ERR_INVALID, fn, "null pointer");
    if (!aligned_to(a->logits, (size_t) es) || !aligned_to(a->draft_logits, (size_t) es))
        return op_fail(PK_ERR_INVALID, fn, "logits must be aligned to their element");
    for (const void * q : {(const void *) a->drafts, (const void *) a->n_drafts, (const void *) a->uniforms, (const void *) a->tokens,
                           (const void *) a->accepted, (const void *) a->logprobs, (const void *) a->temperatures,
                           (const void *) a->top_ks, (const void *) a->top_ps, (const void *) a->min_ps})
        if (!aligned_to(q, 4)) return op_fail(PK_ERR_INVALID, fn, "arrays must be 4-byte aligned");
    if (!aligned_to(a->workspace, 8)) return op_fail(PK_ERR_INVALID, fn, "workspace must be 8-byte aligned");
    if (a->sequences > 0 && !resident(a->vocab, a->draft_logits && a->max_drafts > 0) &&
        (!a->workspace || a->workspace_bytes < rows * (int64_t) sizeof(RowStat)))
        return op_fail(PK_ERR_INVALID, fn, "workspace is null or workspace_bytes below pk_verify_workspace()");
    if (!device_ok(device)) return op_fail(PK_ERR_NO_DEVICE, fn, "no sm_100 device with that index");
    if (a->sequences == 0) return PK_OK;
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return op_cuda_fail(dev.err, fn);
    Plan p{*a, static_cast<RowStat *>(a->workspace)};
    if (a->max_drafts == 0) p.a.draft_logits = nullptr;
    // nothing to cut: neither an array of settings nor a setting that cuts
    const bool filters = a->top_ks || a->top_ps || a->min_ps || (a->top_k > 0 && a->top_k < a->vocab) || !(a->top_p >= 1.0f) ||
                         a->min_p > 0.0f;
    cudaStream_t s = (cudaStream_t) stream;
    const cudaError_t e = a->logits_type == PK_GGML_F32 ? dispatch<float>(p, filters, s)
                          : a->logits_type == PK_GGML_F16 ? dispatch<__half>(p, filters, s) : dispatch<__nv_bfloat16>(p, filters, s);
    return e == cudaSuccess ? PK_OK : op_cuda_fail(e, fn);
}
