// Attention of drafted rows over a paged cache: what the kernels share.
#pragma once
#include "zq_draft.cuh"

namespace zq {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    CacheArgs c;
    const uint8_t *q;
    const unsigned long long *mask;
    const int32_t *lens;
    uint8_t *out;
    float *parts;     // [gridDim.x][2]: rows x (D) sums, then largest scores and sums of weights
    int4 *info;       // [gridDim.x]: {sequence, head * tiles + tile, pieces, rows of the sequence} of the item that starts in this CTA's share and ends in another's
    int64_t q_stride;
    int batch, rows, group, tiles, words;  // tiles: row tiles of a (sequence, head)
    int split;        // CTAs of a cluster that share an item, 0: shares of all items in one line
    float scale;      // of the scores, log2(e) included
    uint32_t *status;
};

// A sequence's cache positions in front of its rows, and its rows.
struct SeqLen {
    int context, rows;
};
__device__ __forceinline__ SeqLen seq_len(const AttnArgs &a, int seq) {
    SeqLen s{a.c.lens[seq], draft_len(a.lens, seq, a.rows, a.status)};
    if (s.context < 0 || ((int64_t)s.context + s.rows) > ((int64_t)a.c.max_blocks << a.c.page_shift)) {
        atomicMax(a.status, (uint32_t)kStatusBadIndex);
        s = {0, 0};
    }
    return s;
}
// 32 bits of a row's view of the drafted rows, from row d on (d may be negative: the context, which it sees).
__device__ __forceinline__ uint32_t view32(const AttnArgs &a, int seq, int i, int d, int rows) {
    if (i >= rows) return 0u;
    uint32_t v;
    if (d <= -32) {
        v = 0xffffffffu;
    } else {
        const int from = d < 0 ? 0 : d, skip = d < 0 ? -d : 0;
        uint32_t bits;  // drafted rows [from, from + 32)
        if (!a.mask) {
            const int n = i - from + 1;
            bits = n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
        } else {
            const unsigned long long *m = a.mask + ((size_t)seq * a.rows + i) * a.words;
            const int w = from >> 6, o = from & 63;
            unsigned long long x = w < a.words ? m[w] >> o : 0;
            if (o > 32 && w + 1 < a.words) x |= m[w + 1] << (64 - o);
            bits = (uint32_t)x;
        }
        v = skip ? bits << skip | ((1u << skip) - 1) : bits;
    }
    const int n = rows - d;  // keys there are
    return n <= 0 ? 0u : n >= 32 ? v : v & ((1u << n) - 1);
}

// The weights are rounded to the cache's type for the second product, whose operands are of one type: by half a step of each, 2^-8 of it in bf16 and 2^-11 in f16; the
// sum of weights is one of unrounded weights, in f32. Below 2^-14 f16's steps stay as wide as they are there, and below 2^-25 nothing is left, which at 131072 keys can be 0.4 % of
// a row. Weights in f16 are therefore taken 2^kUp times as large, in the products and in the sum, so that it falls out by itself; before that they are at most 2^MOST.
template <bool BF16, int MOST> constexpr float kUp = BF16 ? 0.f : 15.f - MOST;
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
    __half2 v = __floats2half2_rn(lo, hi);
    return h2_as_u32(v);
}
template <bool BF16> __device__ __forceinline__ float unpack16(uint32_t bits) { return BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits)); }
// Values of a word whose exponent is all ones (infinities, NaN) become zero; true if there was one.
template <bool BF16> __device__ __forceinline__ bool drop_nonfinite(uint32_t &w) {
    const uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
    const bool lo = (w & e) == e, hi = (w >> 16 & e) == e;
    if (lo) w &= 0xffff0000u;
    if (hi) w &= 0x0000ffffu;
    return lo || hi;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool there) {
    const int n = there ? 16 : 0;  // 0: sixteen zero bytes, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
struct Share {
    int64_t first, last, total;  // places of this CTA; of all
    int extra;                   // places of an item behind its units'
    int ctas;                    // with a share
    int seq;                     // of the first place
    int64_t seq_first;           // first place of that sequence
};

__device__ __forceinline__ int units_of(const SeqLen &s, int unit) {
    return s.rows ? (s.context + s.rows + unit - 1) / unit : 1;  // a sequence without rows has its output set to zero by its one unit
}

// The CTA's share of the places in line: those of an item's units, and `extra` behind them for what the end of an item costs (a CTA that walks
// from one item into the next has that much less to read).  Every thread adds up some sequences, the thread whose sequences hold the first place looks for it.
template <int kThreads> __device__ Share find_share(const AttnArgs &a, int unit, int extra, uint8_t *scratch) {
    int64_t *s_sum = reinterpret_cast<int64_t *>(scratch);  // [kThreads / 32 + 3]
    const int tid = threadIdx.x, lane = tid & 31, per = (a.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    const int64_t items = (int64_t)a.c.heads * a.tiles;
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += units_of(seq_len(a, b), unit) * items;
    int64_t incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) s_sum[tid / 32] = incl;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < tid / 32) before += s_sum[w];
        total += s_sum[w];
    }
    if (total <= (int64_t)gridDim.x) extra = 0;  // a unit each: nobody walks on
    total += a.batch * items * extra;
    mine += (b1 - b0) * items * extra;
    int64_t at = before + incl + b1 * items * extra - mine;
    Share s;
    s.total = total;
    s.extra = extra;
    s.ctas = (int)min((int64_t)gridDim.x, total);
    const int64_t c = blockIdx.x;
    s.first = c < s.ctas ? c * total / s.ctas : total;
    s.last = c < s.ctas ? (c + 1) * total / s.ctas : total;
    int64_t *s_found = s_sum + kThreads / 32;
    if (s.first >= at && s.first < at + mine) {
        for (int b = b0; b < b1; ++b) {
            const int64_t n = (units_of(seq_len(a, b), unit) + extra) * items;
            if (s.first < at + n) {
                s_found[0] = b;
                s_found[1] = at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    s.seq = s.first < total ? (int)s_found[0] : 0;
    s.seq_first = s.first < total ? s_found[1] : 0;
    __syncthreads();
    return s;
}

// Joins the parts of cut items: in place behind a kernel that left them (a.parts, a.info) with `rows` rows of d_pad values per part.
int launch_attention_join(zq_ctx *ctx, const AttnArgs &a, bool bf16, int ctas, int rows, int d_pad, zq_error *err);
// Many rows per key: the kernel on tcgen05 (zq_attn_wide.cu).  `taken` false: not a shape of this kernel.
int launch_attention_wide(zq_ctx *ctx, AttnArgs &a, const zq_kv_cache *cache, bool &taken, zq_error *err);

}  // namespace zq
