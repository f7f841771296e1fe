// Verification of drafted tokens: the walk down a drafted tree from given random numbers, and the token behind its end.
//
// With p the target's distribution at the walk's row and q the draft's, child c of token t is kept if u_c q(t) < p(t); else p becomes
// max(p - q, 0) / Z and the next child is tried.  Kept or drawn, tokens are then distributed as the target alone would draw them.
//
// The token drawn at the end is a whole number that a random number picks among a vocabulary's running sums, most of which lie closer
// together than f32 tells apart (two f32 sums of 128 000 weights disagree about one pick in a hundred): the weights of that pick and their sums
// are f64, exact to 2e-12 (of the lightest tokens: in f32, see Weights).  A child's test has one border only: its sums are f32 inside a thread, and a test that lies
// within their error of its border, some one in ten thousand, is decided by the f64 pass, as is whether a rejection left anything.
//
// Only rows on the walk are read, so the work is latency more than bytes: a cluster of CTAs per sequence shares a row (each CTA a
// run of the vocabulary) and walks in step: all CTAs exchange their sums through distributed shared memory, one barrier each time, and come to
// the same decision.  A row is read once for its largest logit and sum (f32); where the walk ends, once more (from L2) for f64 weights,
// kept as one sum per segment of tokens.  The pick looks for its CTA, then its segment, then its token, and evaluates one segment again.
//
// What rejections of drawn children leave has a closed form: after k of them p is (p - m_k q)+ / Z_k with m_1 = 1 and m_(k+1) = m_k + Z_k, Z_k the
// sum of (p - m_k q)+.  For the test of the next child Z_k is summed in f32.  Where the walk ends, one pass finds it in f64, for two rejections at a
// time, although each m_k hangs on the Z before it: the pass sums at the m that f32 gave, along with the q of the tokens that count, which is
// the sum's slope, and the sums are moved to the exact m afterwards (it lies 1e-7 away, so that what the line leaves out is 1e-14).
#include <cooperative_groups.h>

#include "zq_draft.cuh"

namespace zq {

namespace cg = cooperative_groups;

// 1024 threads of an SM in four CTAs: each pass waits for memory and for chains of dependent operations more than for issue slots (64 sequences of 13 rows of 128 003
// tokens, drawn, took 150 us; with 768 threads 214, with 512 of twice the registers 179; with the tests next to a border in f64 152, 137 to 171 by the draw; the kernels of drawn
// children spill 500 to 660 bytes a thread at 64 registers, in the f64 passes above all).
constexpr int kVerifyThreads = 256, kVerifyCtas = 4, kVerifyWarps = kVerifyThreads / 32, kMaxCluster = 16, kAhead = 2, kSegment = 256;  // tokens that a warp takes at a time and whose sum is kept
constexpr float kHeavy = -18.f;  // weights above 2^kHeavy of the largest are evaluated in f64
constexpr int kSums = 6;         // sums of a pass over both rows: of p, of q; at two m: of what is left, its slope

struct VerifyArgs {
    const uint8_t *logits, *draft;
    const int32_t *tokens, *parents, *lens;
    const float *accept_u, *sample_u, *temperature;
    int32_t *path, *accepted, *token;
    int vocab, rows, shared_parents, segments;  // segments of a CTA
    float border;  // how far f32's sums may be off, relative to themselves (first_error)
    uint32_t *status;
};

// What the f32 sums of a row, and of what a rejection leaves, are off by, at most: ex2.approx by 2^-22, its argument, of up to 100, by three roundings, 100 x 3 x
// 2^-24 ln 2 = 2^-16.3, and a thread adds four weights of a segment to each of two sums, half a step each. With p, q, the factors m and the sums Z
// off by that much (m and Z of the k-th rejection by 2 (k + 1) as much: m + Z moves by no more than m does), both sides of a child's test differ from the exact ones by less than this times (2 k + 2) q + p.
static float first_error(int segments) { return 1.f / (1 << 15) + (float)segments / (1 << 25); }

// A row's largest logit (NaN if the row holds one; where its place is not asked for, one that is not far below), its first place, and the sum of its weights
// relative to it.
struct RowPart {
    float top;
    int32_t at;
    double sum;
};

struct VerifyShared {
    // what the CTAs of the cluster tell each other, in two sets of places in turn
    RowPart part[2][2][kMaxCluster];  // [..][target, draft]
    double sums[2][kSums][kMaxCluster];
    RowPart warp_part[2][kVerifyWarps];
    double warp_sums[kSums][kVerifyWarps];
    double m[kMaxDraftRows];          // of the rejections at this row (drawn children)
    int32_t gone[kMaxDraftRows];      // rejected tokens at this row (chosen children)
    int32_t parent[kMaxDraftRows], token[kMaxDraftRows];
    float u[kMaxDraftRows];
    double roots[32];
    alignas(16) float2 list[kVerifyWarps][kSegment];
};
constexpr size_t kSegmentBytes = (227 << 10) - (sizeof(VerifyShared) + 1023) / 1024 * 1024;  // room for the sums of a CTA's segments

template <class T> __device__ __forceinline__ float logit(const T *row, int v) {
    if constexpr (sizeof(T) == 4) return row[v];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(row[v]);
    else return __bfloat162float(row[v]);
}

// The eight values of a row from place v on; places outside [0, vocab) give -infinity.  v is a multiple of 8 less the row's
// distance from a 16-byte boundary, so that whole vectors are aligned (wide).
template <class T> struct Eight {
    static constexpr int kPer = 16 / sizeof(T);
    uint4 w[8 / kPer];
    __device__ __forceinline__ void load(const T *row, int v, int vocab, bool wide) {
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

__device__ __forceinline__ double warp_sum(double x) {
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// 2^((l - top) c) to 2e-12 of itself: 2^(n + j / 32 + r), |r| <= 1 / 64, with 2^(j / 32) from a table and a Taylor sum of degree 4 for
// 2^r (Tang's table-driven method); 11 f64 operations.  Below `low` (2^-900 of the largest) it is 0.
//
// light(): the same in f32, the argument to twice f32's bits, off by 2^-21 of the weight.  Of weights below 2^-18 of the largest that is
// 2^-39 each, and of either sign: 128 000 of them move a running sum by less than 1e-9 of the largest weight, a ten-thousandth of the usual distance between borders.
struct Weights {
    double c, top;
    float low, c_hi, c_lo, top32, least;
    __device__ void scale_by(double scale) {
        c = scale;
        c_hi = (float)fmin(scale, 1e30);
        c_lo = (float)(fmin(scale, 1e30) - (double)c_hi);
        least = fmaxf(-200.f / c_hi, -3.4028235e38f);
    }
    __device__ void relative_to(float largest, double gap) {  // gap: 900 / c
        top = (double)largest;
        low = fmaxf((float)(top - gap), -3.4028235e38f);
        top32 = largest;
    }
    __device__ __forceinline__ bool heavy(float l, float from) const { return (l - top32) * c_hi > from; }
    __device__ __forceinline__ float light(float l) const {
        const float d = fmaxf(l - top32, least), y = d * c_hi;
        float w = ex2(y);
        w = fmaf(w * 0.69314718f, fmaf(d, c_lo, fmaf(d, c_hi, -y)), w);
        return l == -INFINITY ? 0.f : w;
    }
    __device__ __forceinline__ double operator()(float l, const double *roots) const {
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
        s *= roots[k & 31];
        s = __hiloint2double(__double2hiint(s) + ((k >> 5) << 20), __double2loint(s));
        return none ? 0.0 : s;
    }
};

// Puts a lane's heavy tokens (bits of its eight) into the warp's list; returns how many there are.  Few are heavy, and the warp takes 32 of the list at a time.
__device__ __forceinline__ int list_heavy(float2 *list, const float (&l)[8], const float (&ql)[8], unsigned heavies) {
    const int lane = threadIdx.x & 31, mine = __popc(heavies);
    int incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (total) {
        int at = incl - mine;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (heavies >> e & 1) list[at++] = make_float2(l[e], ql[e]);
        __syncwarp();
    }
    return total;
}

// Joins (largest, place, sum) of the lanes of each half of a warp; a NaN stays.
__device__ __noinline__ RowPart join_halves(RowPart p, float scale32) {
    RowPart m = p;
    for (int o = 8; o > 0; o >>= 1) {
        const float top = __shfl_xor_sync(0xffffffffu, m.top, o);
        const int32_t at = __shfl_xor_sync(0xffffffffu, m.at, o);
        if (isnan(top) || top > m.top || (top == m.top && at < m.at)) {
            m.top = top;
            m.at = at;
        }
    }
    m.sum = p.top == -INFINITY ? 0.0 : p.sum * (double)exp2f((p.top - m.top) * scale32);
    for (int o = 8; o > 0; o >>= 1) m.sum += __shfl_xor_sync(0xffffffffu, m.sum, o);
    return m;
}
// Every CTA gets every CTA's part of both rows: half a warp joins the warps' parts of a row and stores the result into all CTAs.
__device__ __noinline__ void exchange_rows(VerifyShared &s, int parity, bool both, float scale32) {
    cg::cluster_group cluster = cg::this_cluster();
    const int which = threadIdx.x >> 4, i = threadIdx.x & 15;
    static_assert(kVerifyWarps <= 16 && kMaxCluster <= 16, "half a warp");
    __syncthreads();
    if (threadIdx.x < 32) {
        const RowPart p = join_halves(i < kVerifyWarps && (both || !which) ? s.warp_part[which][i] : RowPart{-INFINITY, 0x7fffffff, 0.0}, scale32);
        if (i < (int)cluster.num_blocks()) cluster.map_shared_rank(&s, i)->part[parity][which][cluster.block_rank()] = p;
    }
    cluster.sync();
}
__device__ __noinline__ void exchange_sums(VerifyShared &s, int parity, int n) {
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    static_assert(kSums <= kVerifyWarps, "a warp each");
    __syncthreads();
    if (warp < n) {
        const double sum = warp_sum(lane < kVerifyWarps ? s.warp_sums[warp][lane] : 0.0);
        if (lane < (int)cluster.num_blocks()) cluster.map_shared_rank(&s, lane)->sums[parity][warp][cluster.block_rank()] = sum;
    }
    cluster.sync();
}

// DRAWN: children were drawn from the draft's distributions. (A constant: with a condition of the launch in its place, nvcc 12.9 compiled what follows the children's loop as if
// they had been chosen, whatever the condition was.)
template <class T, bool DRAWN> __global__ void __launch_bounds__(kVerifyThreads, kVerifyCtas) verify_draft_kernel(const VerifyArgs a) {
    pdl_launch_dependents();
    extern __shared__ double s_seg[];  // sums of this CTA's segments, then their slopes
    __shared__ VerifyShared s;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();  // this CTA runs: peers wait for it before they store into this CTA
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), seq = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 32) s.roots[tid] = exp2(tid / 32.0);
    const double *root = s.roots;
    pdl_wait_prior_grid();
    const int n = draft_len(a.lens, seq, a.rows, a.status);
    const size_t row0 = (size_t)seq * a.rows;
    const float heat = a.temperature[seq];
    for (int i = tid; i < n; i += kVerifyThreads) {
        const int up = a.parents[(a.shared_parents ? 0 : row0) + i];
        if (rank == 0 && (up < -1 || up >= i)) atomicMax(a.status, (uint32_t)kStatusBadIndex);  // such a row hangs below none: it is never tried
        s.parent[i] = up;
        s.token[i] = a.tokens[row0 + i];
        s.u[i] = a.accept_u[row0 + i];
    }
    __syncthreads();
    cluster.barrier_wait();  // all CTAs run, and have done so since before the tables were read
    const bool greedy = heat == 0.f;
    const double scale = 1.4426950408889634074 / (greedy ? 1.0 : (double)heat);
    const float scale32 = (float)fmin(scale, 1e30);
    const int first = rank * a.segments, last = first + a.segments;
    constexpr int kNowhere = 1 << 22;  // a segment behind every row's end
    int parity = 0, node = 0, count = 0, token = -1;
    bool bad = n > 0 && !(heat >= 0.f && heat < INFINITY);

    const T *row = nullptr, *qrow = nullptr;
    int shift = 0;
    bool q_wide = false;
    Weights pw, qw;
    const double gap = 900.0 / scale;
    pw.scale_by(scale);
    qw.scale_by(scale);
    double p_inv = 0, q_inv = 0;  // 1 / sum of weights
    int n_gone = 0;

    // Largest logit, its place and 1 / sum of the rows from all CTAs' parts; false where one is no distribution.
    auto joined = [&](bool both, int32_t &at) {
        const int i = lane & 15;
        const RowPart p = join_halves(i < ctas ? s.part[parity][lane >> 4][i] : RowPart{-INFINITY, 0x7fffffff, 0.0}, scale32);
        const double inv = 1.0 / p.sum;
        const float p_top = __shfl_sync(0xffffffffu, p.top, 0), q_top = __shfl_sync(0xffffffffu, p.top, 16);
        at = __shfl_sync(0xffffffffu, p.at, 0);
        p_inv = __shfl_sync(0xffffffffu, inv, 0);
        q_inv = __shfl_sync(0xffffffffu, inv, 16);
        pw.relative_to(p_top, gap);
        if (both) qw.relative_to(q_top, gap);
        return isfinite(p_top) && (!both || isfinite(q_top));
    };
    // The next row from `from` on that hangs below the walk's row, -1 where there is none.
    auto child_from = [&](int from) {
        for (int j0 = from; j0 < n; j0 += 32) {
            const unsigned hits = __ballot_sync(0xffffffffu, j0 + lane < n && s.parent[j0 + lane] == node);
            if (hits) return j0 + __ffs(hits) - 1;
        }
        return -1;
    };
    auto total_of = [&](int which) { return warp_sum(lane < ctas ? s.sums[parity][which][lane] : 0.0); };
    auto place = [&](int g) { return g * kSegment + lane * 8 - shift; };
    auto load = [&](const T *r, bool w, int g, float (&l)[8]) {
        Eight<T> x;
        x.load(r, place(g), a.vocab, w);
        x.get(l);
    };
    // A large logit, its place where it is asked for (greedy), and the sum of weights relative to it, of this CTA's run of the target's row and of the draft's, in f32 inside
    // a thread.  They are relative to the largest logit of the warp's first segment; where that is none, or is so far from the others that the sum leaves f32's
    // range, and where the place is asked for, the warp takes its run with a running maximum.  A NaN makes that sum one.
    const uint64_t scale2 = twice(scale32);
    auto weigh = [&](const Eight<T> &x, uint64_t base2, uint64_t (&sums)[2]) {
        float l[8];
        x.get(l);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float lo, hi;
            unpair64(mul2(add2(pair64(__float_as_uint(l[e]), __float_as_uint(l[e + 1])), base2), scale2), lo, hi);
            sums[e >> 1 & 1] = add2(sums[e >> 1 & 1], pair64(__float_as_uint(ex2(lo)), __float_as_uint(ex2(hi))));
        }
    };
    auto most_of = [&](const Eight<T> &x) {
        float l[8], m;
        x.get(l);
        m = l[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) m = fmaxf(m, l[e]);
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
    };
    auto scan = [&](bool both) {
        float top[2] = {-INFINITY, -INFINITY};
        double sum[2] = {0, 0};
        if (!greedy) {
            uint64_t ps[2] = {0, 0}, qs[2] = {0, 0}, p_base = 0, q_base = 0;
            for (int g = first + warp; g < last; g += kAhead * kVerifyWarps) {
                Eight<T> x[kAhead], y[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int v = place(g + k * kVerifyWarps < last ? g + k * kVerifyWarps : kNowhere);
                    x[k].load(row, v, a.vocab, true);
                    if (both) y[k].load(qrow, v, a.vocab, q_wide);
                }
                if (g == first + warp) {
                    top[0] = most_of(x[0]);
                    p_base = twice(-top[0]);
                    if (both) {
                        top[1] = most_of(y[0]);
                        q_base = twice(-top[1]);
                    }
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    weigh(x[k], p_base, ps);
                    if (both) weigh(y[k], q_base, qs);
                }
            }
            float lo, hi;
            unpair64(add2(ps[0], ps[1]), lo, hi);
            sum[0] = warp_sum((double)(lo + hi));
            unpair64(add2(qs[0], qs[1]), lo, hi);
            if (both) sum[1] = warp_sum((double)(lo + hi));
        }
#pragma unroll 1
        for (int which = 0; which < (both ? 2 : 1); ++which) {
            const float t = which ? top[1] : top[0];
            const double all = which ? sum[1] : sum[0];
            RowPart p{t, 0x7fffffff, all};  // of a warp without tokens: no logit, no sum
            if (!(isfinite(t) && all >= 0.5 && all < 1e30) && (first + warp) * kSegment - shift < a.vocab) {
                float run = -INFINITY, some = 0.f;
                int32_t at = 0x7fffffff;
#pragma unroll 1
                for (int g = first + warp; g < last; g += kVerifyWarps) {
                    float l[8];
                    load(which ? qrow : row, which ? q_wide : true, g, l);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (l[e] > run) {
                            some *= ex2((run - l[e]) * scale32);
                            run = l[e];
                            at = place(g) + e;
                        }
                        some += ex2((l[e] - (run == -INFINITY ? 0.f : run)) * scale32);
                    }
                }
                p = join_halves({isnan(some) ? NAN : run, at, (double)some}, scale32);
                // the two halves
                const float other = __shfl_xor_sync(0xffffffffu, p.top, 16);
                const int32_t other_at = __shfl_xor_sync(0xffffffffu, p.at, 16);
                const double other_sum = __shfl_xor_sync(0xffffffffu, p.sum, 16);
                const float larger = isnan(p.top) || isnan(other) ? NAN : fmaxf(p.top, other);
                p.sum = (p.top == -INFINITY ? 0.0 : p.sum * (double)exp2f((p.top - larger) * scale32)) + (other == -INFINITY ? 0.0 : other_sum * (double)exp2f((other - larger) * scale32));
                if (other > p.top || (other == p.top && other_at < p.at)) p.at = other_at;
                p.top = larger;
            }
            if (lane == 0) s.warp_part[which][warp] = p;
        }
    };
    // Takes the rejected tokens out of a lane's tokens of segment g.
    auto drop_gone = [&](float (&l)[8], int g) {
        for (int i0 = 0; i0 < n_gone; i0 += 32) {
            const int d = i0 + lane < n_gone ? s.gone[i0 + lane] - (g * kSegment - shift) : -1;
            unsigned hits = __ballot_sync(0xffffffffu, d >= 0 && d < kSegment);
            while (hits) {
                const int at = __shfl_sync(0xffffffffu, d, __ffs(hits) - 1);
                hits &= hits - 1;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at == lane * 8 + e) l[e] = -INFINITY;
            }
        }
    };
    // Sums of the segments of the target's weights, without rejected tokens.
    auto row_segments = [&](float from) {
        double mine = 0;
#pragma unroll 1
        for (int g = first + warp; g < last; g += kVerifyWarps) {
            float l[8], some = 0.f;
            load(row, true, g, l);
            drop_gone(l, g);
            unsigned heavies = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool h = pw.heavy(l[e], from);
                if (h) heavies |= 1u << e;
                some += h ? 0.f : pw.light(l[e]);
            }
            const int total = list_heavy(s.list[warp], l, l, heavies);
            double t = (double)some;
#pragma unroll 4
            for (int i = lane; i - lane < total; i += 32) {
                const double w = pw(s.list[warp][min(i, total - 1)].x, root);
                t += i < total ? w : 0.0;
            }
            t = warp_sum(t);
            if (lane == 0) {
                s_seg[g - first] = t;
                s_seg[a.segments + g - first] = 0;
            }
            mine += t;
            __syncwarp();
        }
        if (lane == 0) s.warp_sums[0][warp] = mine;
        exchange_sums(s, parity ^= 1, 1);
    };
    // Sums over both rows: of p's weights and q's, and at factors c0 and c1 of (p - c q)+ and of the q in it, at c1 kept for every segment.
    auto both_segments = [&](double c0, double c1, float from) {
        const float f0 = (float)c0, f1 = (float)c1;
        double all[kSums] = {0, 0, 0, 0, 0, 0};
#pragma unroll 1
        for (int g = first + warp; g < last; g += kVerifyWarps) {
            float l[8], ql[8], some[kSums] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            load(row, true, g, l);
            load(qrow, q_wide, g, ql);
            unsigned heavies = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool h = pw.heavy(l[e], from) || qw.heavy(ql[e], from);
                if (h) heavies |= 1u << e;
                const float p = h ? 0.f : pw.light(l[e]), q = h ? 0.f : qw.light(ql[e]), r0 = fmaf(-f0, q, p), r1 = fmaf(-f1, q, p);
                some[0] += p;
                some[1] += q;
                some[2] += fmaxf(r0, 0.f);
                some[3] += r0 > 0.f ? q : 0.f;
                some[4] += fmaxf(r1, 0.f);
                some[5] += r1 > 0.f ? q : 0.f;
            }
            const int total = list_heavy(s.list[warp], l, ql, heavies);
            double left = (double)some[4], slope = (double)some[5];
            all[0] += (double)some[0];
            all[1] += (double)some[1];
            all[2] += (double)some[2];
            all[3] += (double)some[3];
#pragma unroll 2
            for (int i = lane; i - lane < total; i += 32) {
                const float2 x = s.list[warp][min(i, total - 1)];
                const bool in = i < total;
                const double p = pw(x.x, root), q = qw(x.y, root), wp = in ? p : 0.0, wq = in ? q : 0.0, r0 = wp - c0 * wq, r1 = wp - c1 * wq;
                all[0] += wp;
                all[1] += wq;
                all[2] += fmax(r0, 0.0);
                all[3] += r0 > 0 ? wq : 0.0;
                left += fmax(r1, 0.0);
                slope += r1 > 0 ? wq : 0.0;
            }
            all[4] += left;
            all[5] += slope;
            left = warp_sum(left);
            slope = warp_sum(slope);
            if (lane == 0) {
                s_seg[g - first] = left;
                s_seg[a.segments + g - first] = slope;
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < kSums; ++i) {
            all[i] = warp_sum(all[i]);
            if (lane == 0) s.warp_sums[i][warp] = all[i];
        }
        exchange_sums(s, parity ^= 1, kSums);
    };
    // The sum of (p - m q)+, in f32 inside a thread.
    auto light_rest = [&](double m) {
        const float p32 = (float)p_inv, mq32 = (float)(m * q_inv);
        float some[2] = {0.f, 0.f};
        for (int g = first + warp; g < last; g += 2 * kVerifyWarps) {
            Eight<T> x[2], y[2];
            const int other = g + kVerifyWarps < last ? g + kVerifyWarps : kNowhere;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                x[k].load(row, place(k ? other : g), a.vocab, true);
                y[k].load(qrow, place(k ? other : g), a.vocab, q_wide);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float l[8], ql[8];
                x[k].get(l);
                y[k].get(ql);
#pragma unroll
                for (int e = 0; e < 8; ++e) some[e & 1] += fmaxf(fmaf(-mq32, ex2((ql[e] - qw.top32) * scale32), p32 * ex2((l[e] - pw.top32) * scale32)), 0.f);
            }
        }
        const double t = warp_sum((double)(some[0] + some[1]));
        if (lane == 0) s.warp_sums[0][warp] = t;
        exchange_sums(s, parity ^= 1, 1);
        return total_of(0);
    };

    auto note = [&](auto &list, int at, auto value) {
        __syncthreads();
        if (tid == 0) list[at] = value;
        __syncthreads();
    };

    if (n > 0 && !bad) {
        count = 1;
        if (rank == 0 && tid == 0) a.path[row0] = 0;
        while (true) {
            row = reinterpret_cast<const T *>(a.logits) + (row0 + node) * a.vocab;
            shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
            n_gone = 0;
            const int child = child_from(node + 1);
            const bool use_q = DRAWN && !greedy && child >= 0;
            if (use_q) {
                qrow = reinterpret_cast<const T *>(a.draft) + (row0 + node) * a.vocab;
                q_wide = ((reinterpret_cast<uintptr_t>(qrow) ^ reinterpret_cast<uintptr_t>(row)) & 15) == 0;
            }
            if (child >= 0 && !greedy) {  // the first child's logits come while the rows are summed
                const int t = s.token[child];
                if (t >= 0 && t < a.vocab) {
                    asm volatile("prefetch.global.L1 [%0];" ::"l"(row + t));
                    if (use_q) asm volatile("prefetch.global.L1 [%0];" ::"l"(qrow + t));
                }
            }
            scan(use_q);
            exchange_rows(s, parity ^= 1, use_q, scale32);
            int32_t best;
            bad = !joined(use_q, best);
            if (bad) break;
            int sum_at = 0;              // place of the segments' sum among the last pass's sums

            // ---- its children, in f32's sums until one is kept, none is left, or one lies within these sums' error of a border; then in 64 bits
            int next = -1;
            int rejected = 0;         // drawn children that left something: p is (p - m q)+ / rest
            double m = 0, rest = 1;
            double gone = 0;          // what the rejected chosen children had of p
            double factor = 0, off = 0;  // what is left: w_p - factor w_q; off: the exact factor less the one that the segments are taken at
            bool seen = false;        // child j has failed its test in 64 bits
            for (int j = child;;) {
                enum { kToken, kChild, kRest } ask = kToken;  // what the sums in 64 bits are for
                for (; j >= 0; j = child_from(j + 1)) {
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
                    const double u = (double)s.u[j], p = pw(logit(row, t), root) * p_inv;
                    if constexpr (DRAWN) {
                        if (!seen) {
                            const double q = qw(logit(qrow, t), root) * q_inv, bound = u * q * rest, of = p - m * q;
                            if (p > 0 && fabs(bound - of) <= (double)a.border * ((2 * rejected + 2) * q + p)) {
                                ask = kChild;
                                break;
                            }
                            if (bound < fmax(of, 0.0)) {
                                next = j;
                                break;
                            }
                        }
                        seen = false;
                        m += rest;
                        rest = light_rest(m);
                        note(s.m, rejected++, m);
                        if (!(rest > (double)a.border * (rejected + 1))) {
                            ask = kRest;
                            break;
                        }
                    } else {
                        bool again = false;
                        for (int i = 0; i < n_gone; ++i) again |= s.gone[i] == t;
                        if (again) continue;  // nothing of it is left
                        const double bound = u * (1.0 - gone), near = (double)a.border * (p + gone);
                        const bool close = p > 0 && (fabs(bound - p) <= near || (!(bound < p) && 1.0 - gone - p <= near));
                        if (!close && bound < p) {
                            next = j;
                            break;
                        }
                        note(s.gone, n_gone++, t);
                        if (close) {
                            ask = kChild;
                            break;
                        }
                        gone += p;
                    }
                }
                if (next >= 0 || greedy) break;

                // ---- the sums in 64 bits; where little is left, of the lightest tokens too
                const float from = ask == kRest || (DRAWN ? rest : 1.0 - gone) < 1.0 / 64 ? -INFINITY : kHeavy;
                const bool both = DRAWN && (rejected || ask != kToken);
                double m_before = 0, rest_before = 1;  // the last rejection
                factor = off = 0;
                if (both) {
                    // where little is left, p and q are near each other and many terms change sign on a step of m: once more from the m of the first time
                    for (int times = from < kHeavy && rejected ? 2 : 1; times > 0; --times) {
                        m = 0;
                        rest = 1;
                        double sum_p = 0, ratio = 0;
                        for (int i = 0; i == 0 || i < rejected; i += 2) {
                            // factors for weights: m times (sum of w_p) / (sum of w_q), as f32 gave them; one rejection counts twice
                            const double by = q_inv / p_inv, c0 = i < rejected ? s.m[i] * by : 0.0, c1 = i + 1 < rejected ? s.m[i + 1] * by : c0;
                            both_segments(c0, c1, from);
                            sum_p = total_of(0);
                            ratio = sum_p / total_of(1);
#pragma unroll 1
                            for (int k = 0; k < 2 && i + k < rejected; ++k) {
                                m_before = m;
                                rest_before = rest;
                                m += rest;
                                factor = m * ratio;
                                off = factor - (k ? c1 : c0);
                                rest = (total_of(2 + 2 * k) - off * total_of(3 + 2 * k)) / sum_p;
                                note(s.m, i + k, m);
                            }
                        }
                        p_inv = 1.0 / sum_p;
                        q_inv = ratio * p_inv;
                    }
                } else {
                    row_segments(from);
                }
                if (ask == kToken) {
                    sum_at = both ? 4 : 0;
                    break;
                }
                if (ask == kRest) {
                    if (!(rest > 0)) {  // nothing: p stays as it was
                        --rejected;
                        m = m_before;
                        rest = rest_before;
                    }
                    j = child_from(j + 1);
                    continue;
                }
                const double u = (double)s.u[j], w = pw(logit(row, s.token[j]), root);
                bool yes;
                if constexpr (DRAWN) {
                    const double p = w * p_inv, q = qw(logit(qrow, s.token[j]), root) * q_inv;
                    yes = u * q * rest < fmax(p - m * q, 0.0);
                    seen = !yes;
                } else {
                    const double others = total_of(0);  // u (w + others) < w, also where w is all there is
                    yes = u * others < (1.0 - u) * w;
                    if (!yes) {
                        if (others > 0) gone += w * p_inv;
                        else --n_gone;  // nothing left: p stays as it was
                        j = child_from(j + 1);
                    }
                }
                if (yes) {
                    next = j;
                    break;
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

            // ---- nobody kept: a token from what is left, weights w_p - factor w_q where that is positive
            // a lane has a CTA's part; before: of the CTAs in front
            double part = 0;
            if (lane < ctas) part = sum_at ? fmax(s.sums[parity][4][lane] - off * s.sums[parity][5][lane], 0.0) : s.sums[parity][0][lane];
            double upto = part;
            for (int o = 1; o < 16; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            const double target = (double)a.sample_u[seq] * __shfl_sync(0xffffffffu, upto, ctas - 1);
            const unsigned over_here = __ballot_sync(0xffffffffu, lane < ctas && part > 0 && upto > target), some = __ballot_sync(0xffffffffu, part > 0);
            // where none is over, the target is the total, to rounding
            const int owner = over_here ? __ffs(over_here) - 1 : some ? 31 - __clz(some) : 0;
            const double before = __shfl_sync(0xffffffffu, upto - part, owner);
            if (owner == rank && warp == 0) {
                // the segment, 32 at a time
                double at = before;
                int found = -1, likely = 0;
                for (int g0 = 0; g0 < a.segments && found < 0; g0 += 32) {
                    const double x = g0 + lane < a.segments ? fmax(s_seg[g0 + lane] - off * s_seg[a.segments + g0 + lane], 0.0) : 0.0;
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
                // its tokens, by way of the list: a lane's eight weights one after the other
                float l[8], ql[8];
                load(row, true, first + found, l);
                drop_gone(l, first + found);
                if (factor > 0) load(qrow, q_wide, first + found, ql);
#pragma unroll
                for (int e = 0; e < 8; ++e) s.list[0][lane * 8 + e] = make_float2(l[e], factor > 0 ? ql[e] : 0.f);
                double t = 0, *weight = reinterpret_cast<double *>(s.list[0]) + lane * 8;
#pragma unroll 4
                for (int e = 0; e < 8; ++e) {
                    const float2 v = s.list[0][lane * 8 + e];
                    double x = pw(v.x, root);
                    if (factor > 0) x = fmax(x - factor * qw(v.y, root), 0.0);
                    weight[e] = x;
                    t += x;
                }
                double incl = t;
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += up;
                }
                double run = at + incl - t;
                int hit = -1, last_one = -1;
#pragma unroll 1
                for (int e = 0; e < 8; ++e) {
                    const double x = weight[e];
                    run += x;
                    if (x > 0) last_one = e;
                    if (hit < 0 && !end && x > 0 && run > target) hit = e;
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, last_one >= 0);
                if (hits | any) {
                    if (lane == (hits ? __ffs(hits) - 1 : 31 - __clz(any))) a.token[seq] = place(first + found) + (hits ? hit : last_one);
                } else {  // the segment's sum was rounding, and so is the choice: its likeliest token
                    load(row, true, first + found, l);
                    drop_gone(l, first + found);
                    RowPart p{-INFINITY, 0x7fffffff, 0.0};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (l[e] > p.top) p.top = l[e], p.at = place(first + found) + e;
                    for (int o = 16; o > 0; o >>= 1) {
                        const float top = __shfl_xor_sync(0xffffffffu, p.top, o);
                        const int32_t at = __shfl_xor_sync(0xffffffffu, p.at, o);
                        if (top > p.top || (top == p.top && at < p.at)) p.top = top, p.at = at;
                    }
                    if (lane == 0) {
                        if (p.top == -INFINITY) atomicMax(a.status, (uint32_t)kStatusBadIndex);
                        a.token[seq] = p.top == -INFINITY ? -1 : p.at;
                    }
                }
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

template <class T, bool DRAWN> static int launch_verify(zq_ctx *ctx, VerifyArgs &a, int cluster, size_t batch, size_t smem, zq_error *err) {
    ZQ_CUDA_CHECK(cudaFuncSetAttribute(verify_draft_kernel<T, DRAWN>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), err);
    // the same value every time: calls of other threads set it too
    ZQ_CUDA_CHECK(cudaFuncSetAttribute(verify_draft_kernel<T, DRAWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSegmentBytes), err);
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
    ZQ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_draft_kernel<T, DRAWN>, a), err);
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
    a.vocab = (int)vocab;
    a.rows = (int)rows;
    a.shared_parents = parents_shared;
    a.status = ctx->status_dev;
    const size_t segments = (vocab + 7 + kSegment - 1) / kSegment;  // a row may begin up to seven values behind a boundary
    auto bytes = [&](int ctas) { return 2 * ((segments + ctas - 1) / ctas) * sizeof(double); };
    while (bytes(cluster) > kSegmentBytes) cluster *= 2;  // some 3 million tokens a CTA
    static_assert(2 * ((((size_t(1) << 22) + 7) / kSegment + 1) / 2 + 1) * sizeof(double) <= kSegmentBytes, "two CTAs hold the largest vocabulary");
    a.segments = (int)((segments + cluster - 1) / cluster);
    a.border = first_error(a.segments);
    const size_t smem = bytes(cluster);
    if (a.draft) return dtype == ZQ_F32 ? launch_verify<float, true>(ctx, a, cluster, batch, smem, err) : dtype == ZQ_F16 ? launch_verify<__half, true>(ctx, a, cluster, batch, smem, err) : launch_verify<__nv_bfloat16, true>(ctx, a, cluster, batch, smem, err);
    return dtype == ZQ_F32 ? launch_verify<float, false>(ctx, a, cluster, batch, smem, err) : dtype == ZQ_F16 ? launch_verify<__half, false>(ctx, a, cluster, batch, smem, err) : launch_verify<__nv_bfloat16, false>(ctx, a, cluster, batch, smem, err);
}
