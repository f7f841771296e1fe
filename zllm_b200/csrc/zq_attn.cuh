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
// Does row i of the sequence see its drafted row j?
__device__ __forceinline__ bool sees(const AttnArgs &a, int seq, int i, int j) {
    if (!a.mask) return j <= i;
    return a.mask[((size_t)seq * a.rows + i) * a.words + (j >> 6)] >> (j & 63) & 1;
}

}  // namespace zq
