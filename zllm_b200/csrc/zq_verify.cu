// Verification of drafted tokens: the walk down a drafted tree from given random numbers, and the token behind its end.
//
// With p the target's distribution at the walk's row and q the draft's, child c of token t is kept if u_c q(t) < p(t); else p becomes
// max(p - q, 0) / Z and the next child is tried.  Kept or drawn, tokens are then distributed as the target alone would draw them.
//
// The token drawn at the end is a whole number that a random number picks among a vocabulary's running sums, most of which lie closer
// together than f32 tells apart (two f32 sums of 128 000 weights disagree about one pick in a hundred): the weights of that pick and their sums
// are f64, exact to 2e-12 (of the lightest tokens: in f32, see Weights).  A child's test has one border only; while none was rejected at a row, its sums are f32 inside a thread.
//
// Only rows on the walk are read, so the work is latency more than bytes: a cluster of CTAs per sequence shares a row (each CTA a
// run of the vocabulary) and walks in step: all CTAs exchange their sums through distributed shared memory, one barrier each time, and come to
// the same decision.  A row is read once for its largest logit and sum (f32); where the walk ends, once more (from L2) for f64 weights,
// kept as one sum per segment of tokens.  The pick looks for its CTA, then its segment, then its token, and evaluates one segment again.
//
// What rejections of drawn children leave has a closed form: after k of them p is (p - m q)+ / Z with m = 1 at first and m + Z after each, Z the
// sum of (p - m q)+.  So a rejection is one pass, in f32 for the test of the next child and, for those of the last row only, in f64.
#include <cooperative_groups.h>

#include "zq_draft.cuh"

namespace zq {

namespace cg = cooperative_groups;

// 1024 threads of an SM in four CTAs: each pass waits for memory and for chains of dependent operations more than for issue slots (with 512 threads of
// twice the tokens at a time 64 sequences of 128 003 tokens took 235 us, so 170).
constexpr int kVerifyThreads = 256, kVerifyCtas = 4, kVerifyWarps = kVerifyThreads / 32, kMaxCluster = 16, kSegment = 256;  // tokens that a warp takes at a time and whose sum is kept
constexpr float kHeavy = -18.f;  // weights above 2^kHeavy of the largest are evaluated in f64

struct VerifyArgs {
    const uint8_t *logits, *draft;
    const int32_t *tokens, *parents, *lens;
    const float *accept_u, *sample_u, *temperature;
    int32_t *path, *accepted, *token;
    int64_t vocab;
    int rows, shared_parents, segments;  // segments of a CTA
    uint32_t *status;
};

// A row's largest logit (NaN if the row holds one), its first place, and the sum of its weights relative to it.
struct RowPart {
    float top;
    int32_t at;
    double sum;
};

struct VerifyShared {
    RowPart part[2][2][kMaxCluster];  // [exchanges in turn][target, draft]: what the CTAs of the cluster tell each other
    RowPart warp_part[2][kVerifyWarps];
    int32_t gone[kMaxDraftRows];      // rejected tokens at this row (chosen children)
    int32_t parent[kMaxDraftRows], token[kMaxDraftRows];
    float u[kMaxDraftRows];
    float2 list[kVerifyWarps][kSegment];
};

template <class T> __device__ __forceinline__ float logit(const T *row, int64_t v) {
    if constexpr (sizeof(T) == 4) return row[v];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(row[v]);
    else return __bfloat162float(row[v]);
}

// The eight values of a row from place v on; places outside [0, vocab) give -infinity.  v is a multiple of 8 less the row's
// distance from a 16-byte boundary, so that whole vectors are aligned (wide).
template <class T> struct Eight {
    static constexpr int kPer = 16 / sizeof(T);
    uint4 w[8 / kPer];
    __device__ __forceinline__ void load(const T *row, int64_t v, int64_t vocab, bool wide) {
        if (wide && v >= 0 && v + 8 <= vocab) {
#pragma unroll
            for (int j = 0; j < 8 / kPer; ++j) w[j] = *reinterpret_cast<const uint4 *>(row + v + j * kPer);
        } else {
            T x[8];
            const float low = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (v + e >= 0 && v + e < vocab) x[e] = row[v + e];
                else if constexpr (sizeof(T) == 4) x[e] = low;
                else if constexpr (std::is_same<T, __half>::value) x[e] = __float2half_rn(low);
                else x[e] = __float2bfloat16_rn(low);
            }
            memcpy(w, x, sizeof(x));
        }
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        T t[8];
        memcpy(t, w, sizeof(t));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = logit(t, e);
    }
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ double warp_sum(double x) {
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// 2^((l - top) c) to 2e-12 of itself: 2^(n + j / 32 + r), |r| <= 1 / 64, with 2^(j / 32) from lane j of the warp and a Taylor sum of degree 4 for
// 2^r; 11 f64 operations.  Below `low` (2^-900 of the largest) it is 0.  All lanes of the warp call it.
//
// light(): the same in f32, the argument to twice f32's bits, off by 2^-21 of the weight.  Of weights below 2^-18 of the largest that is
// 2^-39 each, and of either sign: 128 000 of them move a running sum by less than 1e-9 of a border's usual distance.
struct Weights {
    double c, top;
    float low, c_hi, c_lo, top32, least;
    __device__ void set(double scale, float largest) {
        c = scale;
        top = (double)largest;
        low = fmaxf((float)(top - 900.0 / c), -3.4028235e38f);
        top32 = largest;
        c_hi = (float)fmin(scale, 1e30);
        c_lo = (float)(fmin(scale, 1e30) - (double)c_hi);
        least = fmaxf(-200.f / c_hi, -3.4028235e38f);
    }
    __device__ __forceinline__ bool heavy(float l) const { return (l - top32) * c_hi > kHeavy; }
    __device__ __forceinline__ float light(float l) const {
        const float d = fmaxf(l - top32, least), y = d * c_hi;
        float w = ex2(y);
        w = fmaf(w * 0.69314718f, fmaf(d, c_lo, fmaf(d, c_hi, -y)), w);
        return l == -INFINITY ? 0.f : w;
    }
    __device__ __forceinline__ double operator()(float l, double root) const {
        constexpr double kMagic = 6755399441055744.0 / 32;  // 1.5 * 2^52 / 32: adding it leaves the number of 32nds in the low bits
        const bool none = !(l >= low);
        const double y = none ? 0.0 : ((double)l - top) * c;
        const double t = y + kMagic;
        const int k = __double2loint(t);
        const double r = y - (t - kMagic);
        double s = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);
        s = fma(r, s, 2.402265069591007e-1);
        s = fma(r, s, 6.931471805599453e-1);
        s = fma(r, s, 1.0);
        s *= __shfl_sync(0xffffffffu, root, k & 31);
        s = __hiloint2double(__double2hiint(s) + ((k >> 5) << 20), __double2loint(s));
        return none ? 0.0 : s;
    }
};

// The sum over a lane's tokens of `value` in f64 where a weight is heavy and of `light` elsewhere.  Few tokens are heavy: the warp lists them
// and takes 32 at a time.
template <class Heavy, class Value, class Light> __device__ __forceinline__ double lane_sum(float2 *list, const float (&l)[8], const float (&ql)[8], Heavy heavy, Value value, Light light) {
    const int lane = threadIdx.x & 31;
    unsigned heavies = 0;
    float some = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float w = light(l[e], ql[e]);
        const bool h = heavy(l[e], ql[e]);
        if (h) heavies |= 1u << e;
        some += h ? 0.f : w;
    }
    double t = (double)some;
    const int mine = __popc(heavies);
    int incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (total == 0) return t;
    int at = incl - mine;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (heavies >> e & 1) list[at++] = make_float2(l[e], ql[e]);
    __syncwarp();
    for (int i = lane; i - lane < total; i += 32) {
        const float2 x = list[min(i, total - 1)];
        const double v = value(x.x, x.y);
        if (i < total) t += v;
    }
    __syncwarp();
    return t;
}

template <class T> __global__ void __launch_bounds__(kVerifyThreads, kVerifyCtas) verify_draft_kernel(const VerifyArgs a) {
    pdl_launch_dependents();
    extern __shared__ double s_seg[];  // sums of this CTA's segments
    __shared__ VerifyShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), seq = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const double root = exp2(lane / 32.0);
    pdl_wait_prior_grid();
    const int n = draft_len(a.lens, seq, a.rows, a.status);
    const size_t row0 = (size_t)seq * a.rows;
    const float heat = a.temperature[seq];
    for (int i = tid; i < n; i += kVerifyThreads) {
        s.parent[i] = a.parents[(a.shared_parents ? 0 : row0) + i];
        s.token[i] = a.tokens[row0 + i];
        s.u[i] = a.accept_u[row0 + i];
    }
    __syncthreads();
    const bool greedy = heat == 0.f, drawn = a.draft != nullptr && !greedy;
    const double scale = 1.4426950408889634074 / (greedy ? 1.0 : (double)heat);
    const float scale32 = (float)fmin(scale, 1e30);
    const int64_t first = (int64_t)rank * a.segments, last = first + a.segments;
    int parity = 0, node = 0, count = 0, token = -1;
    bool bad = n > 0 && !(heat >= 0.f && heat < INFINITY);

    const T *row = nullptr, *qrow = nullptr;
    int64_t shift = 0;
    bool wide = false, q_wide = false;
    Weights pw, qw;
    double p_inv = 0, q_inv = 0;  // 1 / sum of weights
    double m = 0, rest = 1;         // drawn children: p is (p - m q)+ / rest
    int n_gone = 0;

    // Joins (largest, place, sum) of the lanes of a warp; a NaN stays.
    auto join_lanes = [&](RowPart p) {
        RowPart m = p;
        for (int o = 16; o > 0; o >>= 1) {
            const float top = __shfl_xor_sync(0xffffffffu, m.top, o);
            const int32_t at = __shfl_xor_sync(0xffffffffu, m.at, o);
            if (isnan(top) || top > m.top || (top == m.top && at < m.at)) {
                m.top = top;
                m.at = at;
            }
        }
        m.sum = warp_sum(p.top == -INFINITY ? 0.0 : p.sum * (double)exp2f((p.top - m.top) * scale32));
        return m;
    };
    // Every CTA gets every CTA's part: the warps' parts are joined by the first warp, which stores the result into all CTAs.
    auto exchange = [&](bool both, bool sums_only) {
        parity ^= 1;
        __syncthreads();
        if (warp < (both ? 2 : 1)) {
            RowPart p = lane < kVerifyWarps ? s.warp_part[warp][lane] : RowPart{-INFINITY, 0x7fffffff, 0.0};
            if (sums_only) p.sum = warp_sum(p.sum);
            else p = join_lanes(p);
            if (lane < ctas) cluster.map_shared_rank(&s, lane)->part[parity][warp][rank] = p;
        }
        cluster.sync();
    };
    // Largest logit, its place and 1 / sum of a row from all CTAs' parts.
    auto joined = [&](int which, Weights &w, double &inv, int32_t &at) {
        const RowPart p = join_lanes(lane < ctas ? s.part[parity][which][lane] : RowPart{-INFINITY, 0x7fffffff, 0.0});
        at = p.at;
        inv = 1.0 / p.sum;
        w.set(scale, p.top);
        return isfinite(p.top);
    };
    auto total_of = [&](int which) { return warp_sum(lane < ctas ? s.part[parity][which][lane].sum : 0.0); };
    auto place = [&](int64_t g) { return g * kSegment + lane * 8 - shift; };
    auto load = [&](const T *r, bool w, int64_t g, float (&l)[8]) {
        Eight<T> x;
        x.load(r, place(g), a.vocab, w);
        x.get(l);
    };
    // The largest logit and the sum of weights of this CTA's run of a row, in f32 inside a thread.  A NaN makes the sum one.
    struct Run {
        float top = -INFINITY, sum = 0.f;
        int32_t at = 0x7fffffff;
    };
    auto take = [&](Run &run, const float (&l)[8], int64_t g) {
        float most = l[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) most = fmaxf(most, l[e]);
        if (most > run.top) {
            run.sum *= ex2((run.top - most) * scale32);
            run.top = most;
            int e0 = 7;
#pragma unroll
            for (int e = 7; e >= 0; --e)
                if (l[e] == most) e0 = e;
            run.at = (int32_t)(place(g) + e0);
        }
        const float base = run.top == -INFINITY ? 0.f : run.top;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[e & 3] += ex2((l[e] - base) * scale32);
        run.sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    };
    auto scan = [&](bool both) {
        Run p, q;
        for (int64_t g = first + warp; g < last; g += kVerifyWarps) {
            Eight<T> x, y;
            x.load(row, place(g), a.vocab, wide);
            if (both) y.load(qrow, place(g), a.vocab, q_wide);
            float l[8];
            x.get(l);
            take(p, l, g);
            if (both) {
                y.get(l);
                take(q, l, g);
            }
        }
        const RowPart jp = join_lanes({isnan(p.sum) ? NAN : p.top, p.at, (double)p.sum});
        if (lane == 0) s.warp_part[0][warp] = jp;
        if (both) {
            const RowPart jq = join_lanes({isnan(q.sum) ? NAN : q.top, q.at, (double)q.sum});
            if (lane == 0) s.warp_part[1][warp] = jq;
        }
    };
    // What is left of p at a token, times `rest`.  All lanes call it.
    auto left = [&](float l, float ql, bool two) {
        const double p = pw(l, root) * p_inv;
        return two ? fmax(p - m * (qw(ql, root) * q_inv), 0.0) : p;
    };
    // Sum of a row's weights (its largest logit is known).
    auto precise_sum = [&](const T *r, bool w, const Weights &weight, int which) {
        double mine = 0;
        for (int64_t g = first + warp; g < last; g += kVerifyWarps) {
            float l[8];
            load(r, w, g, l);
            mine += lane_sum(s.list[warp], l, l, [&](float v, float) { return weight.heavy(v); }, [&](float v, float) { return weight(v, root); }, [&](float v, float) { return weight.light(v); });
        }
        mine = warp_sum(mine);
        if (lane == 0) s.warp_part[which][warp] = {0.f, 0, mine};
    };
    // Takes the rejected tokens out of a lane's tokens of segment g.
    auto drop_gone = [&](float (&l)[8], int64_t g) {
        for (int i0 = 0; i0 < n_gone; i0 += 32) {
            const int64_t d = i0 + lane < n_gone ? s.gone[i0 + lane] - (g * kSegment - shift) : -1;
            unsigned hits = __ballot_sync(0xffffffffu, d >= 0 && d < kSegment);
            while (hits) {
                const int at = __shfl_sync(0xffffffffu, (int)d, __ffs(hits) - 1);
                hits &= hits - 1;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at == lane * 8 + e) l[e] = -INFINITY;
            }
        }
    };
    // The sums of the segments of what is left, times `rest`; of all of them, over the cluster.
    auto fill_segments = [&](bool two) {
        double mine = 0;
        const float p32 = (float)p_inv, mq32 = (float)(m * q_inv);
        for (int64_t g = first + warp; g < last; g += kVerifyWarps) {
            float l[8];
            double t;
            load(row, wide, g, l);
            if (two) {
                float ql[8];
                load(qrow, q_wide, g, ql);
                t = lane_sum(s.list[warp], l, ql, [&](float v, float w) { return pw.heavy(v) || qw.heavy(w); }, [&](float v, float w) { return left(v, w, true); },
                             [&](float v, float w) { return fmaxf(fmaf(-mq32, qw.light(w), p32 * pw.light(v)), 0.f); });
            } else {
                drop_gone(l, g);
                t = lane_sum(s.list[warp], l, l, [&](float v, float) { return pw.heavy(v); }, [&](float v, float) { return left(v, v, false); }, [&](float v, float) { return p32 * pw.light(v); });
            }
            t = warp_sum(t);
            if (lane == 0) s_seg[g - first] = t;
            mine += t;
        }
        if (lane == 0) s.warp_part[0][warp] = {0.f, 0, mine};
        exchange(false, true);
        return total_of(0);
    };
    // The sum of what a rejection leaves, in f32 inside a thread.
    auto light_rest = [&] {
        float mine = 0.f;
        const float p32 = (float)p_inv, mq32 = (float)(m * q_inv);
        for (int64_t g = first + warp; g < last; g += kVerifyWarps) {
            float l[8], ql[8];
            load(row, wide, g, l);
            load(qrow, q_wide, g, ql);
#pragma unroll
            for (int e = 0; e < 8; ++e) mine += fmaxf(fmaf(-mq32, ex2((ql[e] - qw.top32) * scale32), p32 * ex2((l[e] - pw.top32) * scale32)), 0.f);
        }
        const double t = warp_sum((double)mine);
        if (lane == 0) s.warp_part[0][warp] = {0.f, 0, t};
        exchange(false, true);
        return total_of(0);
    };

    if (n > 0 && !bad) {
        count = 1;
        if (rank == 0 && tid == 0) a.path[row0] = 0;
        while (true) {
            row = reinterpret_cast<const T *>(a.logits) + (row0 + node) * a.vocab;
            shift = (int64_t)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
            wide = true;
            n_gone = 0;
            m = 0;
            rest = 1;
            bool child = false;
            for (int j = node + 1; j < n && !child; ++j) child = s.parent[j] == node;
            const bool use_q = drawn && child;
            if (use_q) {
                qrow = reinterpret_cast<const T *>(a.draft) + (row0 + node) * a.vocab;
                q_wide = ((reinterpret_cast<uintptr_t>(qrow) ^ reinterpret_cast<uintptr_t>(row)) & 15) == 0;
            }
            scan(use_q);
            exchange(use_q, false);
            int32_t best, unused;
            bad = !joined(0, pw, p_inv, best);
            if (use_q) bad |= !joined(1, qw, q_inv, unused);
            if (bad) break;

            int next = -1;
            int rejected = 0;  // drawn children
            double gone = 0;   // what the rejected chosen children had of p
            for (int j = node + 1; j < n; ++j) {
                if (s.parent[j] != node) continue;
                const int t = s.token[j];
                if (t < 0 || t >= a.vocab) {
                    if (tid == 0 && rank == 0) atomicMax(a.status, (uint32_t)kStatusBadIndex);
                    continue;
                }
                if (greedy) {
                    if (t == best) next = j;
                    if (next >= 0) break;
                    continue;
                }
                const double u = (double)s.u[j];
                const float l = logit(row, t);
                if (drawn) {
                    const float ql = logit(qrow, t);
                    if (u * qw(ql, root) * q_inv * rest < left(l, ql, true)) {
                        next = j;
                        break;
                    }
                    const double before = m;
                    m += rest;
                    const double sum = light_rest();
                    if (sum > 0) rest = sum;
                    else m = before;  // nothing left: p stays as it was
                    ++rejected;
                } else {
                    bool again = false;
                    for (int i = 0; i < n_gone; ++i) again |= s.gone[i] == t;
                    const double chance = again ? 0.0 : pw(l, root) * p_inv;
                    if (u < chance / (1.0 - gone)) {
                        next = j;
                        break;
                    }
                    if (!again && 1.0 - gone - chance > 0) {
                        __syncthreads();
                        if (tid == 0) s.gone[n_gone] = t;
                        gone += chance;
                        ++n_gone;
                        __syncthreads();
                    }
                }
            }
            if (next >= 0) {
                if (rank == 0 && tid == 0) a.path[row0 + count] = next;
                ++count;
                node = next;
                continue;
            }
            if (greedy) {
                token = best;
                break;
            }
            // ---- nobody kept: a token from what is left
            bool filled = false;
            if (rejected) {  // the rejections once more, in f64
                precise_sum(row, wide, pw, 0);
                precise_sum(qrow, q_wide, qw, 1);
                exchange(true, true);
                p_inv = 1.0 / total_of(0);
                q_inv = 1.0 / total_of(1);
                m = 0;
                rest = 1;
                for (int i = 0; i < rejected; ++i) {
                    const double before = m;
                    m += rest;
                    const double sum = fill_segments(true);
                    filled = sum > 0;
                    if (!filled) {  // and so it would be for the others
                        m = before;
                        break;
                    }
                    rest = sum;
                }
            }
            if (!filled) fill_segments(m > 0);
            double total = 0, before = 0, upto = 0;
            int owner = -1, some = 0;
            for (int i = 0; i < ctas; ++i) total += s.part[parity][0][i].sum;
            const double target = (double)a.sample_u[seq] * total;
            for (int i = 0; i < ctas; ++i) {
                const double part = s.part[parity][0][i].sum;
                if (part > 0) some = i;
                if (owner < 0 && upto + part > target) {
                    owner = i;
                    before = upto;
                }
                upto += part;
            }
            if (owner < 0) {  // the target is the total, to rounding
                owner = some;
                before = upto - s.part[parity][0][some].sum;
            }
            if (owner == rank && warp == 0) {
                double at = before;
                int64_t found = -1, likely = 0;
                for (int64_t g0 = 0; g0 < a.segments && found < 0; g0 += 32) {
                    const double x = g0 + lane < a.segments ? s_seg[g0 + lane] : 0.0;
                    double incl = x;
                    for (int o = 1; o < 32; o <<= 1) {
                        const double up = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += up;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, x > 0 && at + incl > target), any = __ballot_sync(0xffffffffu, x > 0);
                    if (any) likely = g0 + 31 - __clz(any);
                    if (over) {
                        const int l = __ffs(over) - 1;
                        found = g0 + l;
                        at += __shfl_sync(0xffffffffu, incl - x, l);
                    } else {
                        at += __shfl_sync(0xffffffffu, incl, 31);
                    }
                }
                const bool end = found < 0;
                if (end) found = likely;
                float l[8], ql[8];
                load(row, wide, first + found, l);
                if (m > 0) load(qrow, q_wide, first + found, ql);
                drop_gone(l, first + found);
                double x[8], t = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = left(l[e], ql[e], m > 0);
                    t += x[e];
                }
                double incl = t;
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += up;
                }
                double run = at + incl - t;
                int hit = -1, seen = -1;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    run += x[e];
                    if (x[e] > 0) seen = e;
                    if (hit < 0 && !end && x[e] > 0 && run > target) hit = e;
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, seen >= 0);
                if (lane == (hits ? __ffs(hits) - 1 : any ? 31 - __clz(any) : 0)) a.token[seq] = (int32_t)(place(first + found) + (hits ? hit : seen));
            }
            token = -2;  // written by its owner
            break;
        }
    }
    if (bad && rank == 0 && tid == 0) atomicMax(a.status, (uint32_t)kStatusBadIndex);
    if (rank == 0) {
        if (tid == 0) {
            a.accepted[seq] = count;
            if (token != -2) a.token[seq] = bad ? -1 : token;
        }
        for (int i = count + tid; i < a.rows; i += kVerifyThreads) a.path[row0 + i] = -1;
    }
    cluster.sync();  // no CTA leaves while another may still write into its shared memory
}

template <class T> static int launch_verify(zq_ctx *ctx, VerifyArgs &a, int cluster, size_t batch, size_t smem, zq_error *err) {
    ZQ_CUDA_CHECK(cudaFuncSetAttribute(verify_draft_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), err);
    ZQ_CUDA_CHECK(cudaFuncSetAttribute(verify_draft_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), err);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * cluster));
    cfg.blockDim = dim3(kVerifyThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->disable_pdl ? 1 : 2;
    ZQ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_draft_kernel<T>, a), err);
    ctx->launches++;
    return ZQ_OK;
}

}  // namespace zq

using namespace zq;

extern "C" int zq_verify_draft(zq_ctx *ctx, const void *dev_logits, const void *dev_draft_logits, int dtype, size_t batch, size_t rows, size_t vocab, const int32_t *dev_tokens, const int32_t *dev_parents, int parents_shared, const float *dev_accept_u,
                               const float *dev_sample_u, const float *dev_temperature, const int32_t *dev_draft_lens, int32_t *dev_path, int32_t *dev_accepted, int32_t *dev_token, zq_error *err) {
    if (!ctx || !dev_logits || !dev_tokens || !dev_parents || !dev_accept_u || !dev_sample_u || !dev_temperature || !dev_path || !dev_accepted || !dev_token) return set_error(err, ZQ_ERR_ARG, "zq_verify_draft: null argument");
    if (dtype != ZQ_F32 && dtype != ZQ_F16 && dtype != ZQ_BF16) return set_error(err, ZQ_ERR_ARG, "zq_verify_draft: unknown dtype %d", dtype);
    if (batch == 0 || batch > 65535 || rows == 0 || rows > kMaxDraftRows) return set_error(err, ZQ_ERR_SHAPE, "zq_verify_draft: %zu sequences of %zu rows (1..65535, 1..%d)", batch, rows, kMaxDraftRows);
    if (vocab == 0 || vocab > (size_t(1) << 22)) return set_error(err, ZQ_ERR_SHAPE, "zq_verify_draft: a vocabulary of %zu (up to 2^22)", vocab);
    if ((reinterpret_cast<uintptr_t>(dev_logits) | reinterpret_cast<uintptr_t>(dev_draft_logits)) & (dtype_size(dtype) - 1)) return set_error(err, ZQ_ERR_ARG, "zq_verify_draft: logits are not aligned to their type");
    int rc = use_device(ctx, err);
    if (rc) return rc;
    // CTAs of a sequence: several for each SM, so that the sequences that walk longest have the SMs of the others at the end; at least eight segments each
    int cluster = kMaxCluster;
    while (cluster > 1 && (batch * cluster > kVerifyCtas * (size_t)ctx->sm_count || vocab < (size_t)cluster * 8 * kSegment)) cluster /= 2;
    VerifyArgs a = {};
    a.logits = static_cast<const uint8_t *>(dev_logits);
    a.draft = static_cast<const uint8_t *>(dev_draft_logits);
    a.tokens = dev_tokens;
    a.parents = dev_parents;
    a.lens = dev_draft_lens;
    a.accept_u = dev_accept_u;
    a.sample_u = dev_sample_u;
    a.temperature = dev_temperature;
    a.path = dev_path;
    a.accepted = dev_accepted;
    a.token = dev_token;
    a.vocab = (int64_t)vocab;
    a.rows = (int)rows;
    a.shared_parents = parents_shared;
    a.status = ctx->status_dev;
    const size_t segments = (vocab + 7 + kSegment - 1) / kSegment;  // a row may begin up to seven values behind a boundary
    a.segments = (int)((segments + cluster - 1) / cluster);
    const size_t smem = a.segments * sizeof(double);
    return dtype == ZQ_F32 ? launch_verify<float>(ctx, a, cluster, batch, smem, err) : dtype == ZQ_F16 ? launch_verify<__half>(ctx, a, cluster, batch, smem, err) : launch_verify<__nv_bfloat16>(ctx, a, cluster, batch, smem, err);
}
