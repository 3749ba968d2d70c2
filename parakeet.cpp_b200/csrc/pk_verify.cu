// pk_verify.cu -- verification of drafted tokens: the longest run of a sequence's drafts that given random
// numbers accept, and the token behind it, so that what comes out is distributed as if the target had drawn it.
//
// p and q are the distributions that pk_sample draws from, of the target's and the draft's row of a position with
// the sequence's settings. A draft d is accepted when u q(d) < p(d). At the first that is not, the token is drawn
// from max(p - q, 0), and behind the last draft from p.
//
// Two kernels. The first takes a team of threads per row, as pk_sample does, and leaves of each row what the
// second needs: its largest logit, its cut, the sum of its weights and the draft's weight. The second takes a block
// (or cluster) per sequence: it tests all drafts at once and draws from the one row, or two, that the first
// rejection names, reading them again. Weights are pk_sample's integers, so sums are exact whatever their order;
// the weights of the tested tokens alone are f64 exponentials that nothing cuts off.

#include "pk_draw.cuh"

namespace pk {
namespace {

// What the draw needs of a row.
struct RowStat {
    double drafted;       // weight of the draft, relative to the largest; 0 if it is cut
    u64 total;            // of the weights kept; 0: no logit above -infinity
    float hi;             // largest logit (0 where it is +infinity)
    float from, cut;      // kept: at least `from`, and above `cut` or equal to it up to index `last`
    int last;
    int flags;
};
enum { kInf = 1, kGreedy = 2 };   // the largest is +infinity; the first of the largest alone is kept

struct Plan {
    pk_verify_args a;
    RowStat * stats;      // [sequences][max_drafts + 1] of the target, [sequences][max_drafts] of the draft
};

__device__ __forceinline__ int drafts_of(const pk_verify_args & a, long long seq) {
    return a.n_drafts ? max(0, min(a.n_drafts[seq], a.max_drafts)) : a.max_drafts;
}
__device__ __forceinline__ float temperature_of(const pk_verify_args & a, long long seq) { return a.temperatures ? a.temperatures[seq] : a.temperature; }

// A logit as a row's statistics see it.
__device__ __forceinline__ float seen(float v, int flags) {
    return flags & kInf ? (v == CUDART_INF_F ? 0.0f : -CUDART_INF_F) : v;
}

template <class T, int NT, bool FILTERS, bool CL, bool RES>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT, NT == 32 ? (FILTERS ? 4 : 5) : 1024 / NT)
verify_rows_kernel(const Plan plan, int slice, int teams, int row_floats) {
    extern __shared__ __align__(16) unsigned char raw[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const pk_verify_args & a = plan.a;
    const int t_in = NT == 32 ? (int) threadIdx.x >> 5 : 0;      // team within the block
    Team<NT, CL> team;
    team.tid = NT == 32 ? (int) threadIdx.x & 31 : (int) threadIdx.x;
    team.blocks = CL ? (int) cg::this_cluster().num_blocks() : 1;
    team.rank = CL ? (int) cg::this_cluster().block_rank() : 0;
    team.phase = 0;
    const long long id = CL ? (long long) (blockIdx.x / team.blocks) : (long long) blockIdx.x * teams + t_in;
    const long long targets = a.sequences * (a.max_drafts + 1);
    const bool target = id < targets;
    const long long at = target ? id : id - targets;
    const int per = target ? a.max_drafts + 1 : a.max_drafts;
    if (id >= targets + (a.draft_logits ? a.sequences * a.max_drafts : 0)) return;
    const long long seq = at / per;
    const int pos = (int) (at - seq * per), n = drafts_of(a, seq);
    if (target ? pos > n : pos >= n) return;                     // behind the last draft
    float * rows_at = reinterpret_cast<float *>(raw);
    TeamSmem<NT> * state = reinterpret_cast<TeamSmem<NT> *>(rows_at + (size_t) teams * row_floats);
    team.s = state + t_in;
    TeamBins<NT> * bins = reinterpret_cast<TeamBins<NT> *>(state + teams) + t_in;
    team.mine = table_entry(team.lane());
    const int s0 = min(team.rank * slice, a.vocab);
    const T * row_at = target ? static_cast<const T *>(a.logits) + at * a.row_stride : static_cast<const T *>(a.draft_logits) + at * a.draft_stride;
    Slice<T, RES> l;
    l.n = min(slice, a.vocab - s0);
    l.gl = row_at + s0;
    l.sm = rows_at + (size_t) t_in * row_floats;
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
        if (FILTERS && v > -CUDART_INF_F) lo = fminf(lo, v);
    });
    team.template range<FILTERS>(hi, lo);
    RowStat * out = plan.stats + id;
    const int draft = pos < n ? a.drafts[seq * a.max_drafts + pos] : -1;
    const bool one = team.tid == 0 && team.rank == 0;
    RowStat st;
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
            st.last = (int) min(first, (u64) 0x7FFFFFFF);
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
    Row r;
    r.top = (double) hi;
    r.c = 46.166241308446828384 / temp;                          // 32 log2(e) / T
    r.base = fmaxf(__double2float_ru(r.top - 31.0 * temp), -3.402823466e+38f);
    float least = r.base;                                        // kept: >= least, and what the cut says
    float cut = -CUDART_INF_F;
    u64 ties = ~0ull, total = 0;
    bool partial = false;
    const float m = a.min_ps ? a.min_ps[seq] : a.min_p;
    // The draft's weight is not subject to `base`; what min-p asks for and the cut it is.
    auto leave = [&](float from, float cut_at, int last, u64 sum) {
        st.hi = hi;
        st.from = from;
        st.cut = cut_at;
        st.last = last;
        st.total = sum;
        st.drafted = 0.0;
        if (draft >= 0 && draft < a.vocab) {
            const float v = seen(to_f32(row_at[draft]), st.flags);
            const float floor = fmaxf(!(m > 0.0f) ? -CUDART_INF_F : m >= 1.0f ? hi : __double2float_ru(r.top + temp * log((double) m)), -3.402823466e+38f);
            if (v >= floor && (v > cut_at || (v == cut_at && draft <= last))) st.drafted = v == hi ? 1.0 : exp(((double) v - r.top) / temp);
        }
        *out = st;
    };
    if constexpr (FILTERS) {
        const float p = a.top_ps ? a.top_ps[seq] : a.top_p;
        const int k = a.top_ks ? a.top_ks[seq] : a.top_k;
        const bool done = cut_row<T, NT, CL, RES>(team, bins, l, s0, r, hi, lo, temp_f, a.vocab, k, p, m, least, cut, ties, partial,
            [&](const Pair * list, int count, int first, float share, u64 need) {
                // all that may be kept is on the list: the sum of what is, and the last of it in the order
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
                Team<NT, false> block{team.tid, 0, 1, 0, team.s, 0.0};
                if (need == 0) {
                    sum = block.sum(sum);
                    need = share >= 1.0f ? ~0ull : max((u64) ceil(share > 0.0f ? (double) share * (double) sum : 0.0), 1ull);
                }
                u64 kept = 0;
                int tokens = 0;
#pragma unroll
                for (int q = 0; q < PER; ++q) {
                    const int j = (team.tid + q * NT) / SH;
                    if (j < count && team.tid % SH == 0 && rank[q].n < first && rank[q].w < need && list[j].v >= least) {
                        kept += bins->w[j];
                        ++tokens;
                    }
                }
                kept = block.sum(kept);
                const int all = (int) block.sum((u64) tokens);
#pragma unroll
                for (int q = 0; q < PER; ++q) {
                    const int j = (team.tid + q * NT) / SH;
                    if (j < count && team.tid % SH == 0 && rank[q].n == all - 1 && team.rank == 0) leave(least, list[j].v, list[j].i, kept);
                }
            },
            [] { return false; });
        if (done) {
            if (CL) team.meet();
            return;
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
    u64 sum = whole(onto);
    bool mine = false;                                           // the last of the ties that are kept is in this run
    u64 before = 0;
    if (FILTERS && partial) {
        u64 all;
        before = team.scan((u64) equal, all);
        if (cut >= least && before < ties) sum += min((u64) equal, ties - before) * weight_one(cut, r);
        mine = before < ties && ties <= before + equal;
    }
    total = team.sum(sum);
    if (FILTERS && partial) {
        if (mine) {
            int i = i0;
            for (u64 left = ties - before; i < i1; ++i)
                if (l(i) == cut && --left == 0) break;
            leave(from, cut, s0 + i, total);
        }
    } else if (one) {
        leave(from, cut, 0x7FFFFFFF, total);
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
        r.top = (double) s.hi;
        r.c = 46.166241308446828384 / (flags & kGreedy ? 1.0 : (double) temp);
        r.base = s.from;
    }
    // Weight of token i with logit v (times 2^43, a whole number); the whole warp calls.
    __device__ __forceinline__ double weight(float v, int i, double mine) const {
        v = seen(v, flags);
        const bool keep = v >= from && (v > cut || (v == cut && i <= last));
        const double w = weight_warp(keep ? v : (float) r.top, r, mine) - kZero;
        return keep ? w : 0.0;
    }
};

constexpr int kDrawThreads = 512;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr double kShare = 1152921504606846976.0;        // 2^60: probabilities as integers

template <class T, bool CL>
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
    if (tid == 0) s_first = n;
    const double mine = table_entry(lane);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    const RowStat * ps = plan.stats + seq * (d + 1), * qs = plan.stats + a.sequences * (d + 1) + seq * d;
    const int32_t * drafts = a.drafts + seq * d;
    const float * u = a.uniforms + seq * (d + 1);
    for (int j = tid; j < n; j += kDrawThreads) {
        const double pd = ps[j].total ? ps[j].drafted / ((double) ps[j].total * (1.0 / kOne)) : 0.0;
        double qd;
        if (a.draft_logits) qd = qs[j].total ? qs[j].drafted / ((double) qs[j].total * (1.0 / kOne)) : 0.0;
        else qd = drafts[j] >= 0 && drafts[j] < v ? 1.0 : 0.0;
        const float x = u[j] > 0.0f ? fminf(u[j], 0x1.fffffep-1f) : 0.0f;
        if (!((double) x * qd < pd)) atomicMin(&s_first, j);
    }
    __syncthreads();
    const int first = s_first;
    const float temp = temperature_of(a, seq);
    if (rank == 0) {
        for (int j = tid; j <= d; j += kDrawThreads) {
            if (j == first) continue;
            const bool ok = j < first;
            a.tokens[seq * (d + 1) + j] = ok ? drafts[j] : -1;
            if (a.logprobs)
                a.logprobs[seq * (d + 1) + j] = ok ? (float) (log(ps[j].drafted) - log((double) ps[j].total * (1.0 / kOne))) : -CUDART_INF_F;
        }
        if (tid == 0) a.accepted[seq] = first;
    }
    const RowStat p = ps[first];
    if (p.total == 0) {                                  // nothing to draw from
        if (rank == 0 && tid == 0) {
            a.tokens[seq * (d + 1) + first] = -1;
            if (a.logprobs) a.logprobs[seq * (d + 1) + first] = -CUDART_INF_F;
        }
        return;
    }
    DrawRow<T> pr, qr;
    pr.set(static_cast<const T *>(a.logits) + (seq * (d + 1) + first) * a.row_stride, p, temp);
    enum { kAll, kLess, kWithout };                      // from p, from what p has more than q, from p without the draft
    int mode = kAll, out = -1;
    double sp = 0.0, sq = 0.0;
    if (first < n) {
        if (a.draft_logits) {
            const RowStat q = qs[first];
            if (q.total) {
                mode = kLess;
                qr.set(static_cast<const T *>(a.draft_logits) + (seq * d + first) * a.draft_stride, q, temp);
                sp = kShare / (double) p.total;
                sq = kShare / (double) q.total;
            }
        } else {
            out = drafts[first];
            mode = kWithout;
        }
    }
    // what token i weighs in the draw; the whole warp calls, lanes past `end` for nothing
    auto weigh = [&](int i, int end) -> u64 {
        const bool in = i < end;
        double w = pr.weight(in ? to_f32(pr.at[i]) : -CUDART_INF_F, i, mine);
        if (mode == kLess) {
            // the two products rounded alike: equal rows leave nothing
            const double less = qr.weight(in ? to_f32(qr.at[i]) : -CUDART_INF_F, i, mine);
            w = fmax(__dmul_rn(w, sp) - __dmul_rn(less, sq), 0.0);
        }
        if (mode == kWithout && i == out) w = 0.0;
        return in ? __double2ull_rn(w) : 0ull;
    };
    auto stretch = [&](int begin, int end) {             // its sum, over a warp
        u64 s = 0;
#pragma unroll 4
        for (int i = begin; i < end; i += 32) s += weigh(i + lane, end);
        return warp_sum(s);
    };
    const int part = ((v + kDrawWarps * blocks - 1) / (kDrawWarps * blocks) + 31) & ~31;
    const int begin = min((rank * kDrawWarps + warp) * part, v), end = min(begin + part, v);
    u64 total = 0, before = 0;
    for (int phase = 0;; ++phase) {
        const u64 s = stretch(begin, end);
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
        }
        if (total > 0 || mode == kAll) break;
        mode = kAll;                                     // q has all that p has: only a draft that q never draws ends here
        __syncthreads();
    }
    const u64 t = place_of(u[d], total);
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
        const u64 w = weigh(i + lane, e1);
        const u64 x = before + warp_scan(w, lane);
        if (x - w <= t && t < x) {
            const float l = seen(to_f32(pr.at[i + lane]), pr.flags);
            a.tokens[seq * (d + 1) + first] = i + lane;
            const double tt = pr.flags & kGreedy ? 1.0 : (double) temp;
            if (a.logprobs)
                a.logprobs[seq * (d + 1) + first] =
                    (float) ((l == p.hi ? 0.0 : ((double) l - (double) p.hi) / tt) - log((double) p.total * (1.0 / kOne)));
        }
        before = __shfl_sync(kFull, x, 31);
        if (before > t) break;
    }
}

// ---- launches -----------------------------------------------------------------------

template <class T, int NT, bool FILTERS, bool CL, bool RES>
cudaError_t launch_rows(const Plan & p, long long rows, int blocks, int slice, int row_floats, size_t smem, cudaStream_t s) {
    const int teams = NT == 32 ? 8 : 1;
    auto kernel = verify_rows_kernel<T, NT, FILTERS, CL, RES>;
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
    cfg.gridDim = dim3((unsigned) (CL ? rows * blocks : (rows + teams - 1) / teams));
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
    return cudaLaunchKernelEx(&cfg, kernel, p, slice, teams, row_floats);
}

template <class T, bool FILTERS, int NT>
cudaError_t rows_block(const Plan & p, long long rows, cudaStream_t s) {
    int row_floats;
    const size_t smem = team_bytes<NT, FILTERS>(p.a.vocab, row_floats);
    return launch_rows<T, NT, FILTERS, false, true>(p, rows, 1, p.a.vocab, row_floats, smem, s);
}

template <class T, bool FILTERS>
cudaError_t rows_cluster(const Plan & p, long long rows, int blocks, cudaStream_t s) {
    // slices of whole 16 bytes, so that every slice is aligned as its row is
    const int slice = ((p.a.vocab + blocks - 1) / blocks + 31) / 32 * 32;
    int row_floats;
    const size_t smem = team_bytes<1024, FILTERS>(slice, row_floats);
    if (smem <= kSmemCap) return launch_rows<T, 1024, FILTERS, true, true>(p, rows, blocks, slice, row_floats, smem, s);
    return launch_rows<T, 1024, FILTERS, true, false>(p, rows, blocks, slice, 0, smem - (size_t) row_floats * 4, s);
}

// Teams by rows and vocabulary as in pk_sample, whose figures hold here too: most of a row's time is the same.
template <class T, bool FILTERS>
cudaError_t rows_dispatch(const Plan & p, cudaStream_t s) {
    const int v = p.a.vocab;
    const long long rows = p.a.sequences * (p.a.max_drafts + 1) + (p.a.draft_logits ? p.a.sequences * p.a.max_drafts : 0);
    if (FILTERS ? v <= 1056 && rows >= 20 * 148 : v <= 2048 && rows >= 8 * 148) return rows_block<T, FILTERS, 32>(p, rows, s);
    int blocks = 1;
    if (v > 16384)
        while (blocks < kMaxCluster && rows * blocks * 2 <= 148) blocks *= 2;
    while (blocks < kMaxCluster && (size_t) (v / blocks) * 4 > 200 * 1024) blocks *= 2;
    if (blocks > 1) return rows_cluster<T, FILTERS>(p, rows, blocks, s);
    const bool wave512 = rows <= 2 * 148 && v > 2048, wave256 = rows <= 4 * 148;
    if (v > 16384 || wave512) return rows_block<T, FILTERS, 512>(p, rows, s);
    if (v > 5120 || wave256) return rows_block<T, FILTERS, 256>(p, rows, s);
    return rows_block<T, FILTERS, 128>(p, rows, s);
}

template <class T, bool CL>
cudaError_t launch_draw(const Plan & p, int blocks, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    cfg.gridDim = dim3((unsigned) (p.a.sequences * blocks));
    cfg.blockDim = dim3(kDrawThreads);
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned) blocks;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CL ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, verify_draw_kernel<T, CL>, p);
}

template <class T> cudaError_t dispatch(const Plan & p, bool filters, cudaStream_t s) {
    const cudaError_t e = filters ? rows_dispatch<T, true>(p, s) : rows_dispatch<T, false>(p, s);
    if (e != cudaSuccess) return e;
    int blocks = 1;
    if (p.a.vocab > 16384)
        while (blocks < kMaxCluster && p.a.sequences * blocks * 2 <= 148) blocks *= 2;
    return blocks > 1 ? launch_draw<T, true>(p, blocks, s) : launch_draw<T, false>(p, 1, s);
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
    return rows < 0 ? -1 : rows * (int64_t) sizeof(pk::RowStat);
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
    if (a->sequences > 0 && (!a->logits || !a->uniforms || !a->tokens || !a->accepted || !a->workspace || (a->max_drafts > 0 && !a->drafts)))
        return op_fail(PK_ERR_INVALID, fn, "null pointer");
    if (!aligned_to(a->logits, (size_t) es) || !aligned_to(a->draft_logits, (size_t) es))
        return op_fail(PK_ERR_INVALID, fn, "logits must be aligned to their element");
    for (const void * q : {(const void *) a->drafts, (const void *) a->n_drafts, (const void *) a->uniforms, (const void *) a->tokens,
                           (const void *) a->accepted, (const void *) a->logprobs, (const void *) a->temperatures,
                           (const void *) a->top_ks, (const void *) a->top_ps, (const void *) a->min_ps})
        if (!aligned_to(q, 4)) return op_fail(PK_ERR_INVALID, fn, "arrays must be 4-byte aligned");
    if (!aligned_to(a->workspace, 8)) return op_fail(PK_ERR_INVALID, fn, "workspace must be 8-byte aligned");
    if (a->workspace_bytes < rows * (int64_t) sizeof(RowStat))
        return op_fail(PK_ERR_INVALID, fn, "workspace_bytes is below pk_verify_workspace()");
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
