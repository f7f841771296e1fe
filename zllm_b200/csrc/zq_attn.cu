// Attention of drafted rows over a paged cache.
//
//     out_i = sum_j w_ij v_j / sum_j w_ij,   w_ij = exp(scale q_i k_j - top_i)
//
// One pass over the keys with a running maximum and sum per row (the sums so far are multiplied down when the maximum rises).  The rows of
// all query heads that share a head of the cache go through the matrix instructions together (m16n8k16), so that the cache is read once for them. For up to
// 32 rows per cache head; above, zq_attn_wide.cu takes over where its layout allows (heads of 64 to 128, pages from 8). What it leaves goes through tiles of 64 rows here, each of which
// reads the cache again: 64 rows of 8 query heads a cache head of 256 over 32000 positions take 689 us, of 128 on the other kernel 76. One row each of 64 sequences at 16384 positions streams the cache at 6.6 TB/s.
//
// Work: an item is a (sequence, cache head, tile of rows); its keys are cut into units.  The units of all items, in one line, with a few
// places behind each item for what its end costs, are dealt to the CTAs (one per SM) in equal shares, so that one long sequence or many unequal ones keep all SMs at work; an item cut by a border is
// left in parts (largest score, sum of weights and weighted sums per row, f32) which a second, small kernel joins in ascending order:
// results do not depend on timing.  The lengths are on the device, so each CTA finds its share from them itself.
//
// Where all of it takes a few microseconds, the second kernel would be half of the time: there a cluster of CTAs takes an item, in equal
// runs of its units, and joins its parts through distributed shared memory.
//
// A CTA has key groups (its warps of one group share keys, each with 16 rows of its own; the groups take the keys in turn), every one with a ring
// of its own that cp.async fills: no barrier between groups until the item ends.  Shared memory rows are swizzled by 16-byte chunks so that
// ldmatrix reads without conflicts.
#include <cooperative_groups.h>

#include "zq_attn.cuh"

namespace zq {

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
constexpr int kMaxSplit = 8;  // CTAs of an item in a cluster
// What the end of an item costs, in units.  A decode step of 8 rows per cache head of 128, 4 cache heads, takes 24.8 / 40.2 / 73.1 / 66.6 us for 64 unequal sequences of up to
// 200 and 1000, 150 of 900 and 40 of 5000 positions without it, 21.6 / 35.1 / 60.7 / 61.1 with 3, 21.8 / 36.6 / 63.7 / 63.4 with 6.
constexpr int kItemEnd = 3;

// Shape of the kernel for a head of up to D values and WM warps of 16 rows.
template <int D, int WM> struct AttnShape {
    static constexpr int kGroups = WM == 4 ? 2 : 4;              // key groups of a CTA
    static constexpr int kWarps = WM * kGroups, kThreads = 32 * kWarps;
    static constexpr int kKeys = D <= 128 ? 32 : 16;             // keys per group and step
    static constexpr int kUnit = kKeys * kGroups;                // keys per unit of work
    static constexpr int kPitch = D <= 64 ? 128 : D <= 128 ? 256 : 512;  // bytes of a key in shared memory: chunks are swizzled in eights
    static constexpr int kStage = 2 * kKeys * kPitch;
    static constexpr int kStages = (200 << 10) / (kGroups * kStage) > 6 ? 6 : (200 << 10) / (kGroups * kStage);
    static constexpr int kRows = 16 * WM;
    static constexpr int kRing = kGroups * kStages * kStage;
    static constexpr int kMerge = kGroups * kRows * (D + 2) * 4;  // the groups' sums at the end of an item, in place of the ring
    static constexpr int kPartFloats = kRows * (D + 2);           // of a part: sums, largest scores, sums of weights
    static constexpr int kPartAt = kMerge, kNeed = kMerge + kPartFloats * 4;
    static constexpr int kSmem = (kRing > kNeed ? kRing : kNeed) + 1024;
    static_assert(kStages >= 2 && kSmem <= 227 << 10, "ring");
};

template <int D, int WM, bool BF16> __global__ void __launch_bounds__(AttnShape<D, WM>::kThreads, 1) tree_attention_kernel(const AttnArgs a) {
    using S = AttnShape<D, WM>;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = warp / WM, wm = warp % WM, gtid = tid - group * WM * 32;
    namespace cg = cooperative_groups;
    Share share;
    if (a.split) {
        const int per_seq = a.c.heads * a.tiles, id = blockIdx.x / a.split, rank = blockIdx.x % a.split, item = id % per_seq;
        share.seq = id / per_seq;
        share.seq_first = 0;
        const int64_t n = units_of(seq_len(a, share.seq), S::kUnit);
        share.first = item * n + rank * n / a.split;
        share.last = item * n + (rank + 1) * n / a.split;
        share.total = 0;
        share.extra = 0;
        share.ctas = 0;
    } else {
        share = find_share<S::kThreads>(a, S::kUnit, kItemEnd, smem + S::kSmem - 1024);
        if (tid == 0) a.info[blockIdx.x] = make_int4(0, 0, 0, 0);
        if (share.first >= share.last) return;
    }
    const int d = a.c.head_dim, chunks = d / 8;
    uint8_t *ring = smem + group * S::kStages * S::kStage;
    const uint32_t ring_u32 = smem_u32(ring);
    int seq = share.seq;
    int64_t seq_first = share.seq_first;
    SeqLen len = seq_len(a, seq);
    int units = units_of(len, S::kUnit);

    for (int64_t u = share.first; u < share.last || a.split;) {  // in a cluster once, with no units too
        while (!a.split && u >= seq_first + (int64_t)(units + share.extra) * a.c.heads * a.tiles) {
            seq_first += (int64_t)(units + share.extra) * a.c.heads * a.tiles;
            len = seq_len(a, ++seq);
            units = units_of(len, S::kUnit);
        }
        const int item = a.split ? (int)(blockIdx.x / a.split) % (a.c.heads * a.tiles) : (int)((u - seq_first) / (units + share.extra));
        const int64_t item_first = seq_first + (int64_t)item * (units + share.extra);
        const int head = item / a.tiles, tile = item % a.tiles;
        const int ua = (int)(u - item_first), ub = (int)min((int64_t)units, share.last - item_first);
        if (!a.split && ua >= units) {  // behind its units
            u = item_first + units + share.extra;
            continue;
        }
        const int steps = ub - ua, keys = len.rows ? len.context + len.rows : 0;
        const int row0 = tile * S::kRows + wm * 16, n_rows = len.rows * a.group;

        // ---- the ring: step s of this share holds keys [(ua + s) * kUnit + group * kKeys, + kKeys)
        const int64_t head_off = (int64_t)head * d;
        auto page_of = [&](int s) -> int64_t {  // first value of this lane's key of step s, -1 where there is none
            const int key = (ua + s) * S::kUnit + group * S::kKeys + lane % S::kKeys;
            if (s >= steps || key >= keys) return -1;
            const int64_t r = cache_row(a.c, seq, key);
            if (r < 0) atomicMax(a.status, (uint32_t)kStatusBadIndex);
            return r < 0 ? -1 : r + head_off;
        };
        auto fill = [&](int s, int64_t mine) {
            if (s < steps) {
                const uint32_t base = ring_u32 + (s % S::kStages) * S::kStage;
                constexpr int kChunks = D / 8, kCopies = S::kKeys * kChunks;
#pragma unroll 4
                for (int i = 0; i < (kCopies + WM * 32 - 1) / (WM * 32); ++i) {
                    const int idx = i * WM * 32 + gtid, key = idx / kChunks, chunk = idx % kChunks;
                    const int64_t at = __shfl_sync(0xffffffffu, mine, key % S::kKeys);
                    if (kCopies % (WM * 32) && idx >= kCopies) continue;
                    const bool there = at >= 0 && chunk < chunks;
                    const int64_t off = there ? 2 * at + 16 * chunk : 0;
                    const uint32_t dst = base + key * S::kPitch + ((chunk ^ (key & 7)) << 4);
                    cp_async16(dst, a.c.k + off, there);
                    cp_async16(dst + S::kKeys * S::kPitch, a.c.v + off, there);
                }
            }
            cp_commit();
        };
        // ---- the rows of this warp
        constexpr int kK = D / 16;
        uint32_t qf[kK][4];
        const int r_lo = row0 + lane / 4, r_hi = r_lo + 8, i_lo = r_lo / a.group, i_hi = r_hi / a.group;
        {
            const int g_lo = r_lo % a.group, g_hi = r_hi % a.group;
            const uint8_t *p_lo = a.q + 2 * (((int64_t)seq * a.rows + i_lo) * a.q_stride + (int64_t)(head * a.group + g_lo) * d), *p_hi = a.q + 2 * (((int64_t)seq * a.rows + i_hi) * a.q_stride + (int64_t)(head * a.group + g_hi) * d);
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                const int col = 16 * k + 2 * (lane & 3);
                qf[k][0] = r_lo < n_rows && col < d ? *reinterpret_cast<const uint32_t *>(p_lo + 2 * col) : 0u;
                qf[k][1] = r_hi < n_rows && col < d ? *reinterpret_cast<const uint32_t *>(p_hi + 2 * col) : 0u;
                qf[k][2] = r_lo < n_rows && col + 8 < d ? *reinterpret_cast<const uint32_t *>(p_lo + 2 * col + 16) : 0u;
                qf[k][3] = r_hi < n_rows && col + 8 < d ? *reinterpret_cast<const uint32_t *>(p_hi + 2 * col + 16) : 0u;
            }
        }
        int64_t ahead = page_of(0);
#pragma unroll 1
        for (int s = 0; s < S::kStages - 1; ++s) {  // small code: it runs once per item, at the pace of instruction fetches
            const int64_t now = ahead;
            ahead = page_of(s + 1);
            fill(s, now);
        }

        float o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

        for (int s = 0; s < steps; ++s) {
            cp_wait<S::kStages - 2>();
            if (WM == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WM * 32) : "memory");
            fill(s + S::kStages - 1, ahead);
            ahead = page_of(s + S::kStages);
            const uint32_t kb = ring_u32 + (s % S::kStages) * S::kStage, vb = kb + S::kKeys * S::kPitch;
            const int key0 = (ua + s) * S::kUnit + group * S::kKeys;

            constexpr int kN = S::kKeys / 8;
            float sc[kN][4];
#pragma unroll
            for (int n = 0; n < kN; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
            const int mi = lane >> 3, mr = lane & 7;
#pragma unroll
            for (int k = 0; k < kK; ++k) {
#pragma unroll
                for (int n = 0; n < kN; n += 2) {
                    const int key = n * 8 + (mi >> 1) * 8 + mr, chunk = 2 * k + (mi & 1);
                    uint32_t b[4];
                    ldmatrix_x4(b, kb + key * S::kPitch + ((chunk ^ (key & 7)) << 4));
                    mma16<BF16>(sc[n], qf[k], b[0], b[1]);
                    mma16<BF16>(sc[n + 1], qf[k], b[2], b[3]);
                }
            }
            const bool masked = key0 + S::kKeys > len.context;  // drafted rows among the keys, or the end
#pragma unroll
            for (int n = 0; n < kN; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] *= a.scale;
            }
            uint32_t view[2] = {0xffffffffu, 0xffffffffu};  // of the keys that the thread's two rows see
            if (masked) {
                view[0] = view32(a, seq, i_lo, key0 - len.context, len.rows);
                view[1] = view32(a, seq, i_hi, key0 - len.context, len.rows);
#pragma unroll
                for (int n = 0; n < kN; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(view[e >> 1] >> (n * 8 + 2 * (lane & 3) + (e & 1)) & 1)) sc[n][e] = -INFINITY;
                }
            }
            float base[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float m = top[h];
#pragma unroll
                for (int n = 0; n < kN; ++n) m = fmaxf(m, fmaxf(sc[n][2 * h], sc[n][2 * h + 1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                base[h] = m == -INFINITY ? 0.f : m;
                const float down = exp2f(top[h] - base[h]);
                if (__any_sync(0xffffffffu, top[h] != m)) {
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[n][2 * h] *= down;
                        o[n][2 * h + 1] *= down;
                    }
                    sum[h] *= down;
                }
                top[h] = m;
            }
            const float from[2] = {base[0] - kUp<BF16, 0>, base[1] - kUp<BF16, 0>};
            uint32_t pf[S::kKeys / 16][4];
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = exp2f(sc[n][e] - from[e >> 1]);
                    sum[e >> 1] += p[e];
                }
                pf[n / 2][(n & 1) * 2] = pack2<BF16>(p[0], p[1]);
                pf[n / 2][(n & 1) * 2 + 1] = pack2<BF16>(p[2], p[3]);
            }
            if (masked) {
                // A weight of zero times an infinity of a row that is not seen would be a NaN: such values leave the tile, and are added to the rows that see
                // them.  Lane j looks through key j (all warps of the group write the same).
                uint8_t *v = ring + (s % S::kStages) * S::kStage + S::kKeys * S::kPitch;
                bool dropped = false;
                if (lane < S::kKeys && key0 + lane >= len.context && key0 + lane < keys) {
#pragma unroll 1
                    for (int c = 0; c < D / 8; ++c) {
                        uint4 *at = reinterpret_cast<uint4 *>(v + lane * S::kPitch + ((c ^ (lane & 7)) << 4));
                        uint4 w = *at;
                        bool some = drop_nonfinite<BF16>(w.x);
                        some |= drop_nonfinite<BF16>(w.y);
                        some |= drop_nonfinite<BF16>(w.z);
                        some |= drop_nonfinite<BF16>(w.w);
                        if (some) dropped = true;
                    }
                }
                uint32_t bad = __ballot_sync(0xffffffffu, dropped);
                if (bad) {
                    if (WM > 1) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WM * 32) : "memory");  // every warp has looked
                    for (uint32_t left = bad; left; left &= left - 1) {
                        const int j = __ffs(left) - 1;
                        const int64_t row = cache_row(a.c, seq, key0 + j);
                        const uint16_t *from = reinterpret_cast<const uint16_t *>(a.c.v) + row + head_off;
                        const bool lo = view[0] >> j & 1, hi = view[1] >> j & 1;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) {
                            const int col = n * 8 + 2 * (lane & 3);
                            if (row >= 0 && col < d) {
                                const float x = unpack16<BF16>(from[col]), y = unpack16<BF16>(from[col + 1]);
                                if (!isfinite(x)) o[n][0] += lo ? x : 0.f, o[n][2] += hi ? x : 0.f;
                                if (!isfinite(y)) o[n][1] += lo ? y : 0.f, o[n][3] += hi ? y : 0.f;
                            }
                        }
                        for (int c = lane; c < D / 8; c += 32) {
                            uint4 *at = reinterpret_cast<uint4 *>(v + j * S::kPitch + ((c ^ (j & 7)) << 4));
                            uint4 w = *at;
                            drop_nonfinite<BF16>(w.x);
                            drop_nonfinite<BF16>(w.y);
                            drop_nonfinite<BF16>(w.z);
                            drop_nonfinite<BF16>(w.w);
                            *at = w;
                        }
                    }
                    if (WM > 1) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WM * 32) : "memory");
                    __syncwarp();
                }
            }
#pragma unroll
            for (int k = 0; k < S::kKeys / 16; ++k) {
#pragma unroll
                for (int n = 0; n < D / 8; n += 2) {
                    const int key = k * 16 + (mi & 1) * 8 + mr, chunk = n + (mi >> 1);
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, vb + key * S::kPitch + ((chunk ^ (key & 7)) << 4));
                    mma16<BF16>(o[n], pf[k], b[0], b[1]);
                    mma16<BF16>(o[n + 1], pf[k], b[2], b[3]);
                }
            }
        }
        cp_wait<0>();
        __syncthreads();

        // ---- the groups' sums meet in shared memory
        float *m_o = reinterpret_cast<float *>(smem), *m_top = m_o + S::kGroups * S::kRows * D, *m_sum = m_top + S::kGroups * S::kRows;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
            const int r = group * S::kRows + wm * 16 + lane / 4 + 8 * h;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2 *>(m_o + r * D + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
            if ((lane & 3) == 0) {
                m_top[r] = top[h];
                m_sum[r] = sum[h];
            }
        }
        __syncthreads();
        const bool whole = !a.split && ua == 0 && ub == units;
        float *part = a.split ? reinterpret_cast<float *>(smem + S::kPartAt) : a.parts + ((size_t)blockIdx.x * 2 + (ua == 0 ? 1 : 0)) * S::kPartFloats;  // in a cluster its own memory
        const int n_out = min(S::kRows, a.rows * a.group - tile * S::kRows) * (D / 2);  // pairs of columns of the tile's rows
        // a row's factors of the groups' sums, once, in place of their largest scores
        for (int r = tid; r < S::kRows; r += S::kThreads) {
            float m = -INFINITY, l = 0.f, f[S::kGroups];
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) m = fmaxf(m, m_top[g * S::kRows + r]);
            const float b = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) {
                f[g] = exp2f(m_top[g * S::kRows + r] - b);
                l += f[g] * m_sum[g * S::kRows + r];
            }
            const bool none = whole && (l == 0.f || (tile * S::kRows + r) / a.group >= len.rows);
            const float by = !whole ? 1.f : none ? 0.f : 1.f / l;
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) m_top[g * S::kRows + r] = none ? -1.f : f[g] * by;
            if (!whole && (tile * S::kRows + r) < a.rows * a.group) {
                part[S::kRows * D + r] = m;
                part[S::kRows * D + S::kRows + r] = l;
            }
        }
        __syncthreads();
#pragma unroll 2
        for (int idx = tid; idx < n_out; idx += S::kThreads) {
            const int r = idx / (D / 2), col = 2 * (idx % (D / 2));
            float x = 0.f, y = 0.f;
            bool none = false;
#pragma unroll
            for (int g = 0; g < S::kGroups; ++g) {
                const float w = m_top[g * S::kRows + r];
                const float2 v = *reinterpret_cast<const float2 *>(m_o + (g * S::kRows + r) * D + col);
                none = w < 0.f;
                x += w * v.x;
                y += w * v.y;
            }
            if (!whole) {
                *reinterpret_cast<float2 *>(part + r * D + col) = make_float2(x, y);
            } else if (col < d) {
                const int row = tile * S::kRows + r, i = row / a.group;
                *reinterpret_cast<uint32_t *>(a.out + 2 * ((((int64_t)seq * a.rows + i) * a.c.heads * a.group + head * a.group + row - i * a.group) * d + col)) = none ? 0u : pack2<BF16>(x, y);
            }
        }
        if (a.split) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            for (int idx = tid * a.split + (int)cluster.block_rank(); idx < n_out; idx += a.split * S::kThreads) {
                const int r = idx / (D / 2), col = 2 * (idx % (D / 2)), row = tile * S::kRows + r, i = row / a.group;
                float top_of[kMaxSplit], sum_of[kMaxSplit], m = -INFINITY, x = 0.f, y = 0.f, l = 0.f;
                float2 v[kMaxSplit];
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p) {
                    const float *f = cluster.map_shared_rank(part, p < a.split ? p : 0);
                    top_of[p] = p < a.split ? f[S::kRows * D + r] : -INFINITY;
                    sum_of[p] = f[S::kRows * D + S::kRows + r];
                    v[p] = *reinterpret_cast<const float2 *>(f + r * D + col);
                }
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p) m = fmaxf(m, top_of[p]);
                const float b = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int p = 0; p < kMaxSplit; ++p) {
                    if (p < a.split) {
                        const float w = exp2f(top_of[p] - b);
                        x += w * v[p].x;
                        y += w * v[p].y;
                        l += w * sum_of[p];
                    }
                }
                const bool none = l == 0.f || i >= len.rows;
                const float inv = none ? 0.f : 1.f / l;
                if (col < d) *reinterpret_cast<uint32_t *>(a.out + 2 * ((((int64_t)seq * a.rows + i) * a.c.heads * a.group + head * a.group + row % a.group) * d + col)) = none ? 0u : pack2<BF16>(x * inv, y * inv);
            }
            cluster.sync();  // no CTA leaves while another reads its part
            return;
        }
        if (tid == 0 && ua == 0 && ub < units) {
            const int64_t end = item_first + units;  // the CTA of the item's last unit
            const int last = (int)((end * share.ctas - 1) / share.total);
            a.info[blockIdx.x] = make_int4(seq, item, last - (int)blockIdx.x + 1, len.rows);
        }
        __syncthreads();
        u = item_first + units + share.extra;
    }
}

// Joins the parts of the item that starts in CTA blockIdx.x's share, in the order of its keys: a warp per row, a lane has four columns.  It waits for memory and little
// else, so a row's first parts, and the maxima and sums of the first 32, are on their way before any is used; weights come from the lanes that have them.
// (40 sequences of up to 5000 positions with 240 rows per cache head of 128, 30 MB of parts: 15 us; 33 with two warps a row that took four rows in turn and
// the weights from memory; 20 with four parts ahead, 34 with eight, as the code is met cold.)
constexpr int kJoinRows = 8, kJoinAhead = 2;
template <bool BF16> __global__ void __launch_bounds__(32 * kJoinRows) attention_join_kernel(const AttnArgs a, int rows, int d_pad) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int4 info = a.info[blockIdx.x];
    const int seq = info.x, head = info.y / a.tiles, tile = info.y % a.tiles, pieces = info.z, d = a.c.head_dim;
    const int lane = threadIdx.x & 31, r = kJoinRows * blockIdx.y + (threadIdx.x >> 5), row = tile * rows + r, i = row / a.group;
    if (pieces == 0 || r >= rows || i >= a.rows) return;
    const size_t floats = (size_t)rows * (d_pad + 2);
    auto part = [&](int p) { return a.parts + ((size_t)(blockIdx.x + p) * 2 + (p == 0 ? 1 : 0)) * floats; };
    auto values = [&](int p, int col) { return p < pieces && col < d ? *reinterpret_cast<const float4 *>(part(p) + (size_t)r * d_pad + col) : make_float4(0.f, 0.f, 0.f, 0.f); };
    float4 v[kJoinAhead];
#pragma unroll
    for (int p = 0; p < kJoinAhead; ++p) v[p] = values(p, 4 * lane);
    const float first_top = lane < pieces ? part(lane)[rows * d_pad + r] : -INFINITY, first_sum = lane < pieces ? part(lane)[rows * d_pad + rows + r] : 0.f;
    float m = first_top;
    for (int p = lane + 32; p < pieces; p += 32) m = fmaxf(m, part(p)[rows * d_pad + r]);
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m, first_w = exp2f(first_top - base);
    float l = first_w * first_sum;
    for (int p = lane + 32; p < pieces; p += 32) l += exp2f(part(p)[rows * d_pad + r] - base) * part(p)[rows * d_pad + rows + r];
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const bool none = l == 0.f || i >= info.w;
    const float inv = none ? 0.f : 1.f / l;
    for (int c0 = 0; c0 < d; c0 += 128) {
        const int col = c0 + 4 * lane;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float w_lane = first_w;
        auto add = [&](float w, const float4 &x) {
            sum.x += w * x.x;
            sum.y += w * x.y;
            sum.z += w * x.z;
            sum.w += w * x.w;
        };
        for (int p0 = 0; p0 < pieces; p0 += kJoinAhead) {
            float4 next[kJoinAhead];  // those behind, or the next columns' first
            const bool over = p0 + kJoinAhead >= pieces;
#pragma unroll
            for (int k = 0; k < kJoinAhead; ++k) next[k] = values(over ? k : p0 + kJoinAhead + k, over ? col + 128 : col);
            if (p0 && p0 % 32 == 0) w_lane = p0 + lane < pieces ? exp2f(part(p0 + lane)[rows * d_pad + r] - base) : 0.f;
#pragma unroll
            for (int k = 0; k < kJoinAhead; ++k) {
                const float w = __shfl_sync(0xffffffffu, w_lane, (p0 + k) & 31);
                if (p0 + k < pieces) add(w, v[k]);
                v[k] = next[k];
            }
        }
        if (col < d) {
            uint32_t *to = reinterpret_cast<uint32_t *>(a.out + 2 * ((((int64_t)seq * a.rows + i) * a.c.heads * a.group + head * a.group + row % a.group) * d + col));
            to[0] = none ? 0u : pack2<BF16>(sum.x * inv, sum.y * inv);
            to[1] = none ? 0u : pack2<BF16>(sum.z * inv, sum.w * inv);
        }
    }
}

int launch_attention_join(zq_ctx *ctx, const AttnArgs &a, bool bf16, int ctas, int rows, int d_pad, zq_error *err) {
    const int used = a.rows * a.group < rows ? a.rows * a.group : rows;
    return launch_pdl(ctx, bf16 ? attention_join_kernel<true> : attention_join_kernel<false>, dim3((unsigned)ctas, (unsigned)((used + kJoinRows - 1) / kJoinRows)), dim3(32 * kJoinRows), 0, err, a, rows, d_pad);
}

constexpr size_t kClusterBytes = size_t(512) << 10;

template <int D, int WM, bool BF16> static int launch_shape(zq_ctx *ctx, AttnArgs &a, zq_error *err) {
    using S = AttnShape<D, WM>;
    a.tiles = (a.rows * a.group + S::kRows - 1) / S::kRows;
    ZQ_CUDA_CHECK(cudaFuncSetAttribute(tree_attention_kernel<D, WM, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem), err);
    // A cluster per item where that gives each of its CTAs no more of the cache than kClusterBytes, by the room in the block table (the lengths are on the
    // device): one sequence, 8 cache heads of 128 f16 at 4000 / 8000 / 16000 positions (0.25 / 0.5 / 1 MB a CTA) takes 14.1 / 19.7 / 32.0 us in clusters and
    // 16.8 / 22.0 / 29.5 with the second kernel, heads of 64 at 1000 / 16000 (0.03 / 0.5 MB) 8.2 / 22.4 and 11.5 / 21.7.  Clusters of at most eight CTAs:
    // those of sixteen find room one after the other (17.5 us instead of 8.9 at 517 positions).
    const size_t items = (size_t)a.batch * a.c.heads * a.tiles, positions = (size_t)a.c.max_blocks << a.c.page_shift, units_most = (positions + S::kUnit - 1) / S::kUnit;
    a.split = kMaxSplit;
    while (a.split > 1 && (items * a.split > (size_t)ctx->sm_count || (size_t)a.split >= 2 * units_most)) a.split /= 2;
    if (items * a.split <= (size_t)ctx->sm_count && positions * a.c.head_dim * 4 <= kClusterBytes * a.split) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(items * a.split));
        cfg.blockDim = dim3(S::kThreads);
        cfg.dynamicSmemBytes = S::kSmem;
        cfg.stream = ctx->stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)a.split;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = ctx->disable_pdl ? 1 : 2;
        ZQ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, tree_attention_kernel<D, WM, BF16>, a), err);
        ctx->launches++;
        return ZQ_OK;
    }
    a.split = 0;
    const size_t ctas = (size_t)ctx->sm_count, bytes = ctas * 2 * S::kPartFloats * sizeof(float);
    LaunchScratch scratch;
    int rc = scratch.take(ctx, bytes + ctas * sizeof(int4), err);
    if (rc) return rc;
    a.parts = static_cast<float *>(scratch.p);
    a.info = reinterpret_cast<int4 *>(static_cast<uint8_t *>(scratch.p) + bytes);
    rc = launch_pdl(ctx, tree_attention_kernel<D, WM, BF16>, dim3((unsigned)ctas), dim3(S::kThreads), S::kSmem, err, a);
    if (rc) return rc;
    return launch_attention_join(ctx, a, BF16, (int)ctas, S::kRows, D, err);
}
template <int D, bool BF16> static int launch_rows(zq_ctx *ctx, AttnArgs &a, zq_error *err) {
    const int rows = a.rows * a.group;
    return rows <= 16 ? launch_shape<D, 1, BF16>(ctx, a, err) : rows <= 32 ? launch_shape<D, 2, BF16>(ctx, a, err) : launch_shape<D, 4, BF16>(ctx, a, err);
}
template <bool BF16> static int launch_dim(zq_ctx *ctx, AttnArgs &a, zq_error *err) {
    const int d = a.c.head_dim;
    return d <= 64 ? launch_rows<64, BF16>(ctx, a, err) : d <= 96 ? launch_rows<96, BF16>(ctx, a, err) : d <= 128 ? launch_rows<128, BF16>(ctx, a, err) : d <= 192 ? launch_rows<192, BF16>(ctx, a, err) : launch_rows<256, BF16>(ctx, a, err);
}

}  // namespace zq

using namespace zq;

extern "C" int zq_tree_attention(zq_ctx *ctx, const void *dev_q, size_t q_heads, size_t q_stride, size_t rows, const zq_kv_cache *cache, const uint64_t *dev_mask, const int32_t *dev_draft_lens, float scale, void *dev_out, zq_error *err) {
    if (!ctx || !dev_q || !dev_out) return set_error(err, ZQ_ERR_ARG, "zq_tree_attention: null argument");
    AttnArgs a = {};
    int rc = cache_args("zq_tree_attention", cache, a.c, err);
    if (rc) return rc;
    if (rows == 0 || rows > kMaxDraftRows) return set_error(err, ZQ_ERR_SHAPE, "zq_tree_attention: %zu rows of a sequence (1..%d)", rows, kMaxDraftRows);
    if (q_heads == 0 || q_heads % cache->heads || q_heads > 65536) return set_error(err, ZQ_ERR_SHAPE, "zq_tree_attention: %zu query heads for %zu heads of the cache", q_heads, cache->heads);
    if (q_stride < q_heads * cache->head_dim || q_stride % 2 || q_stride > (size_t)INT32_MAX) return set_error(err, ZQ_ERR_SHAPE, "zq_tree_attention: rows of q %zu values apart for %zu values", q_stride, q_heads * cache->head_dim);
    if (!(scale > 0) || scale > 1e30f) return set_error(err, ZQ_ERR_ARG, "zq_tree_attention: scale %g (positive)", (double)scale);
    if ((reinterpret_cast<uintptr_t>(dev_q) | reinterpret_cast<uintptr_t>(dev_out)) & 3) return set_error(err, ZQ_ERR_ARG, "zq_tree_attention: q or the output is not 4-byte aligned");
    if (reinterpret_cast<uintptr_t>(dev_mask) & 7) return set_error(err, ZQ_ERR_ARG, "zq_tree_attention: the mask is not 8-byte aligned");
    if ((uint64_t)cache->max_blocks * cache->page_size > (uint64_t)INT32_MAX - 4096) return set_error(err, ZQ_ERR_SHAPE, "zq_tree_attention: %zu blocks of %zu positions", cache->max_blocks, cache->page_size);
    if ((rc = use_device(ctx, err))) return rc;
    a.q = static_cast<const uint8_t *>(dev_q);
    a.mask = reinterpret_cast<const unsigned long long *>(dev_mask);
    a.lens = dev_draft_lens;
    a.out = static_cast<uint8_t *>(dev_out);
    a.q_stride = (int64_t)q_stride;
    a.batch = (int)cache->batch;
    a.rows = (int)rows;
    a.group = (int)(q_heads / cache->heads);
    a.words = (int)((rows + 63) / 64);
    a.scale = scale * kLog2e;
    a.status = ctx->status_dev;
    bool taken = false;
    rc = launch_attention_wide(ctx, a, cache, taken, err);
    if (rc || taken) return rc;
    return cache->dtype == ZQ_BF16 ? launch_dim<true>(ctx, a, err) : launch_dim<false>(ctx, a, err);
}
