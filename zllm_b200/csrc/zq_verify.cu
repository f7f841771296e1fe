// Verification of drafted tokens: the walk down a drafted tree from given random numbers, and the token behind its end.
//
// With p the target's distribution at the walk's row and q the draft's, child c of token t is kept if u_c q(t) < p(t); else p becomes
// max(p - q, 0) / Z and the next child is tried.  Kept or drawn, tokens are then distributed as the target alone would draw them.
//
// The token drawn at the end is a whole number that a random number picks among a vocabulary's running sums, most of which lie closer
// together than f32 tells apart (two f32 sums of 128 000 weights disagree about one pick in a hundred): weights and sums are f64.
//
// Only rows on the walk are read, so the work is latency more than bytes: a cluster of CTAs per sequence shares a row (each CTA a
// run of the vocabulary) and walks in step.  Each CTA takes its own largest logit, then its weights relative to that, kept as one sum per
// segment of 256 tokens; the CTAs exchange two numbers per row through distributed shared memory and all come to the same
// decision.  The pick looks for its CTA, then its segment, then its token, and evaluates one segment again.
#include <cooperative_groups.h>

#include "zq_draft.cuh"

namespace zq {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 1024, kVerifyWarps = kVerifyThreads / 32, kSegment = 256, kMaxCluster = 16;

struct VerifyArgs {
    const uint8_t *logits, *draft;
    const int32_t *tokens, *parents, *lens;
    const float *accept_u, *sample_u, *temperature;
    int32_t *path, *accepted, *token;
    int64_t vocab;
    int rows, shared_parents, segments;  // segments of a CTA
    uint32_t *status;
};

// What the CTAs of a cluster tell each other about a row.
struct RowPart {
    float top;    // largest logit of the CTA's run (NaN if it holds one)
    int32_t at;   // its first place, greedy
    double sum;   // of the weights relative to `top`
};

struct VerifyShared {
    RowPart part[2][2][kMaxCluster];  // [exchange parity][target, draft]
    double z[kMaxDraftRows];          // normalisers of the rejections at this row (drawn children)
    int32_t gone[kMaxDraftRows];      // rejected tokens at this row (chosen children)
    double red[kVerifyWarps];
    float red_top[kVerifyWarps];
    int32_t red_at[kVerifyWarps];
    int32_t pick;
};

template <class T> __device__ __forceinline__ float logit(const T *row, int64_t v) {
    if constexpr (sizeof(T) == 4) return row[v];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(row[v]);
    else return __bfloat162float(row[v]);
}

// The eight values of a row from place v on; places outside [0, vocab) give -infinity.  v is a multiple of 8 less the row's
// distance from a 16-byte boundary, so that whole vectors are aligned.
template <class T> __device__ __forceinline__ void eight(const T *row, int64_t v, int64_t vocab, bool wide, float (&x)[8]) {
    if (wide && v >= 0 && v + 8 <= vocab) {
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8 / kPer; ++j) {
            const uint4 w = *reinterpret_cast<const uint4 *>(row + v + j * kPer);
            const T *t = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[j * kPer + e] = logit(t, e);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v + e >= 0 && v + e < vocab ? logit(row, v + e) : -INFINITY;
    }
}

template <class T> struct Walk {
    const VerifyArgs &a;
    VerifyShared &s;
    double *seg;  // sums of this CTA's segments
    const T *row, *qrow;
    double inv_t, p_top, p_inv, q_top, q_inv;  // 1 / temperature; largest logit and 1 / sum of the row's weights
    int64_t shift, first, last;                // the row's distance from its boundary; this CTA's segments
    int n_gone, n_z;
    bool wide, q_wide, drawn;

    __device__ double weight(float l, double top) const { return l == -INFINITY ? 0.0 : exp(((double)l - top) * inv_t); }
    // What is left at the row of token v, up to a factor: z[0..n) have been divided by, one more subtraction with `open`.
    __device__ double left(float l, float ql, int n, bool open) const {
        double r = weight(l, p_top) * p_inv;
        if (n == 0 && !open) return r;
        const double q = weight(ql, q_top) * q_inv;
        for (int i = 0; i < n; ++i) r = fmax(r - q, 0.0) / s.z[i];
        return open ? fmax(r - q, 0.0) : r;
    }
    __device__ bool is_gone(int64_t v) const {
        for (int i = 0; i < n_gone; ++i)
            if (s.gone[i] == v) return true;
        return false;
    }
    // Values of lane `lane` of segment g.
    __device__ int64_t place(int64_t g, int lane) const { return g * kSegment + lane * 8 - shift; }
    __device__ void lane_weights(int64_t g, int lane, int n, bool open, double (&w)[8]) const {
        float x[8], y[8];
        const int64_t v = place(g, lane);
        eight(row, v, a.vocab, wide, x);
        if (drawn && (n || open)) eight(qrow, v, a.vocab, q_wide, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e] = n_gone && is_gone(v + e) ? 0.0 : left(x[e], drawn && (n || open) ? y[e] : 0.f, n, open);
        }
    }
    __device__ double block_sum(double x) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        __syncthreads();
        if (lane == 0) s.red[warp] = x;
        __syncthreads();
        double t = 0;
        for (int w = 0; w < kVerifyWarps; ++w) t += s.red[w];
        return t;
    }
};

template <class T> __global__ void __launch_bounds__(kVerifyThreads, 1) verify_draft_kernel(const VerifyArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    extern __shared__ double s_seg[];
    __shared__ VerifyShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), seq = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = draft_len(a.lens, seq, a.rows, a.status);
    const size_t row0 = (size_t)seq * a.rows;
    const int32_t *parents = a.parents + (a.shared_parents ? 0 : row0);
    const float heat = a.temperature[seq];
    const bool greedy = heat == 0.f;
    Walk<T> w{a, s, s_seg};
    w.inv_t = greedy ? 1.0 : 1.0 / (double)heat;
    w.first = (int64_t)rank * a.segments;
    w.last = w.first + a.segments;
    w.drawn = a.draft != nullptr && !greedy;
    int parity = 0, node = 0, count = 0, token = -1;
    bool bad = n > 0 && !(heat >= 0.f && heat < INFINITY);

    // Largest logit (and its first place) of this CTA's run of a row.
    auto find_top = [&](const T *row, int64_t shift, bool wide, float &top, int32_t &at) {
        float m = -INFINITY;
        int32_t where = 0x7fffffff;
        bool nan = false;
        for (int64_t g = w.first + warp; g < w.last; g += kVerifyWarps) {
            float x[8];
            const int64_t v = g * kSegment + lane * 8 - shift;
            eight(row, v, a.vocab, wide, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                nan |= isnan(x[e]);
                if (x[e] > m) {
                    m = x[e];
                    where = (int32_t)(v + e);
                }
            }
        }
        if (nan) m = NAN;
        for (int o = 16; o > 0; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m, o);
            const int32_t ow = __shfl_xor_sync(0xffffffffu, where, o);
            if (isnan(om) || om > m || (om == m && ow < where)) {
                m = om;
                where = ow;
            }
        }
        __syncthreads();
        if (lane == 0) {
            s.red_top[warp] = m;
            s.red_at[warp] = where;
        }
        __syncthreads();
        m = s.red_top[0];
        where = s.red_at[0];
        for (int i = 1; i < kVerifyWarps; ++i) {
            const float om = s.red_top[i];
            const int32_t ow = s.red_at[i];
            if (isnan(om) || om > m || (om == m && ow < where)) {
                m = om;
                where = ow;
            }
        }
        top = m;
        at = where;
    };
    // Sums of this CTA's segments of what is left at the row; their sum.
    auto fill_segments = [&](int n_z, bool open) {
        double mine = 0;
        for (int64_t g = w.first + warp; g < w.last; g += kVerifyWarps) {
            double x[8], t = 0;
            w.lane_weights(g, lane, n_z, open, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) t += x[e];
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) {
                s_seg[g - w.first] = t;
                mine += t;
            }
        }
        return w.block_sum(lane == 0 ? mine : 0.0);
    };
    // Every CTA gets every CTA's part; one barrier, two sets of places in turn.
    auto exchange = [&](const RowPart &p, const RowPart &q) {
        parity ^= 1;
        if (tid < ctas) {
            VerifyShared *other = cluster.map_shared_rank(&s, tid);
            other->part[parity][0][rank] = p;
            other->part[parity][1][rank] = q;
        }
        cluster.sync();
    };
    // Largest logit and 1 / sum of a row from all CTAs' parts.
    auto joined = [&](int which, double &top, double &inv, int32_t &at) {
        float m = -INFINITY;
        at = 0x7fffffff;
        for (int i = 0; i < ctas; ++i) {
            const RowPart &p = s.part[parity][which][i];
            if (isnan(p.top) || p.top > m) {
                m = p.top;
                at = p.at;
            }
            if (isnan(m)) break;
        }
        top = m;
        double sum = 0;
        for (int i = 0; i < ctas; ++i) sum += s.part[parity][which][i].sum * w.weight(s.part[parity][which][i].top, top);
        inv = 1.0 / sum;
        return isfinite(m);
    };
    auto local_sum = [&](const T *row, int64_t shift, bool wide, float top, bool keep) {
        double mine = 0;
        for (int64_t g = w.first + warp; g < w.last; g += kVerifyWarps) {
            float x[8];
            eight(row, g * kSegment + lane * 8 - shift, a.vocab, wide, x);
            double t = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) t += w.weight(x[e], top);
            if (keep) {
                for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
                if (lane == 0) s_seg[g - w.first] = t;
                if (lane) t = 0;
            }
            mine += t;
        }
        return w.block_sum(mine);
    };

    if (n > 0 && !bad) {
        count = 1;
        if (rank == 0 && tid == 0) a.path[row0] = 0;
        while (true) {
            // ---- the row of the target, and of the draft where it has children
            w.row = reinterpret_cast<const T *>(a.logits) + (row0 + node) * a.vocab;
            w.shift = (int64_t)((reinterpret_cast<uintptr_t>(w.row) & 15) / sizeof(T));
            w.wide = (reinterpret_cast<uintptr_t>(w.row) & (sizeof(T) - 1)) == 0;
            w.n_gone = w.n_z = 0;
            bool child = false;
            for (int j = node + 1; j < n && !child; ++j) child = parents[j] == node;
            RowPart p{-INFINITY, 0, 0}, q{-INFINITY, 0, 0};
            find_top(w.row, w.shift, w.wide, p.top, p.at);
            if (!greedy && p.top < INFINITY) p.sum = local_sum(w.row, w.shift, w.wide, p.top, true);
            const bool use_q = w.drawn && child;
            if (use_q) {
                w.qrow = reinterpret_cast<const T *>(a.draft) + (row0 + node) * a.vocab;
                w.q_wide = ((reinterpret_cast<uintptr_t>(w.qrow) ^ reinterpret_cast<uintptr_t>(w.row)) & 15) == 0;
                find_top(w.qrow, w.shift, w.q_wide, q.top, q.at);
                if (q.top < INFINITY) q.sum = local_sum(w.qrow, w.shift, w.q_wide, q.top, false);
            }
            exchange(p, q);
            int32_t best, unused;
            bad = !joined(0, w.p_top, w.p_inv, best);
            if (use_q) bad |= !joined(1, w.q_top, w.q_inv, unused);
            if (bad) break;

            // ---- its children
            int next = -1;
            bool stale = false;        // s_seg holds something else than what is left
            double gone = 0;           // chosen children: what the rejected ones had of p
            for (int j = node + 1; j < n; ++j) {
                if (parents[j] != node) continue;
                const int t = a.tokens[row0 + j];
                if (t < 0 || t >= a.vocab) {
                    if (tid == 0 && rank == 0) atomicMax(a.status, (uint32_t)kStatusBadIndex);
                    continue;
                }
                if (greedy) {
                    if (t == best) next = j;
                    if (next >= 0) break;
                    continue;
                }
                const double u = (double)a.accept_u[row0 + j];
                const float l = logit(w.row, t);
                if (w.drawn) {
                    const float ql = logit(w.qrow, t);
                    if (u * w.weight(ql, w.q_top) * w.q_inv < w.left(l, ql, w.n_z, false)) {
                        next = j;
                        break;
                    }
                    const double mine = fill_segments(w.n_z, true);
                    RowPart z{0, 0, mine};
                    exchange(z, z);
                    double sum = 0;
                    for (int i = 0; i < ctas; ++i) sum += s.part[parity][0][i].sum;
                    stale = !(sum > 0);
                    if (sum > 0) {
                        if (tid == 0) s.z[w.n_z] = sum;
                        ++w.n_z;
                    }
                    __syncthreads();
                } else {
                    const double chance = w.is_gone(t) ? 0.0 : w.weight(l, w.p_top) * w.p_inv;
                    if (u < chance / (1.0 - gone)) {
                        next = j;
                        break;
                    }
                    __syncthreads();
                    if (tid == 0) s.gone[w.n_gone] = t;
                    if (1.0 - gone - chance > 0) {
                        gone += chance;
                        ++w.n_gone;
                    }
                    __syncthreads();
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
            __syncthreads();
            if (stale) fill_segments(w.n_z, false);  // the last rejection left nothing, and p as it was before
            double scale = 1.0;  // of the CTA's segments
            if (!stale && w.n_z) {
                scale = 1.0 / s.z[w.n_z - 1];
            } else if (!stale) {     // those of p are relative to the CTA's own largest logit
                scale = w.weight(p.top, w.p_top) * w.p_inv;
                for (int i = warp; i < w.n_gone; i += kVerifyWarps) {  // without the rejected tokens
                    const int64_t g = (s.gone[i] + w.shift) / kSegment;
                    if (g >= w.first && g < w.last) {
                        double x[8], t = 0;
                        w.lane_weights(g, lane, 0, false, x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) t += x[e];
                        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
                        if (lane == 0) s_seg[g - w.first] = scale > 0 ? t / scale : 0.0;
                    }
                }
            }
            __syncthreads();
            double mine = 0;
            for (int64_t g = tid; g < a.segments; g += kVerifyThreads) mine += s_seg[g];
            mine = w.block_sum(mine) * scale;
            RowPart z{0, 0, mine};
            exchange(z, z);
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
                // the segment, 32 at a time
                double at = before;
                int64_t found = -1, likely = 0;
                for (int64_t g0 = 0; g0 < a.segments && found < 0; g0 += 32) {
                    const double x = g0 + lane < a.segments ? s_seg[g0 + lane] * scale : 0.0;
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
                double x[8], t = 0;
                w.lane_weights(w.first + found, lane, w.n_z, false, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) t += x[e];
                double incl = t;
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += up;
                }
                const unsigned over = __ballot_sync(0xffffffffu, !end && t > 0 && at + incl > target), any = __ballot_sync(0xffffffffu, t > 0);
                const int l = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
                if (lane == l) {
                    double run = at + incl - t;
                    int pick = -1, last_seen = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        run += x[e];
                        if (x[e] > 0) last_seen = e;
                        if (pick < 0 && over && x[e] > 0 && run > target) pick = e;
                    }
                    a.token[seq] = (int32_t)(w.place(w.first + found, lane) + (pick < 0 ? last_seen : pick));
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
    // CTAs of a sequence: all SMs at work, at least 16 segments each
    int cluster = kMaxCluster;
    while (cluster > 1 && (batch * cluster > (size_t)ctx->sm_count || vocab < (size_t)cluster * 16 * kSegment)) cluster /= 2;
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
