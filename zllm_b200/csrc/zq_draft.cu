// Drafted trees of tokens: their positions and mask, and the cache rows that are kept of them.
//
// Both kernels are bound by latency: a launch, one dependent read of the tables, then a few bytes per row.
#include "zq_draft.cuh"

namespace zq {

int cache_args(const char *who, const zq_kv_cache *c, CacheArgs &out, zq_error *err) {
    if (!c || !c->dev_k || !c->dev_v || !c->dev_blocks || !c->dev_context_lens) return set_error(err, ZQ_ERR_ARG, "%s: null cache argument", who);
    if (c->dtype != ZQ_F16 && c->dtype != ZQ_BF16) return set_error(err, ZQ_ERR_UNSUPPORTED, "%s: a cache holds f16 or bf16, not dtype %d", who, c->dtype);
    if (c->page_size == 0 || (c->page_size & (c->page_size - 1)) || c->page_size > (size_t(1) << 20)) return set_error(err, ZQ_ERR_SHAPE, "%s: page size %zu is not a power of two up to 2^20", who, c->page_size);
    if (c->head_dim == 0 || c->head_dim % 8 || c->head_dim > 256) return set_error(err, ZQ_ERR_SHAPE, "%s: head_dim=%zu (a multiple of 8 up to 256)", who, c->head_dim);
    if (c->heads == 0 || c->heads > 4096 || c->batch == 0 || c->batch > 65535 || c->pages == 0 || c->pages > (size_t)INT32_MAX || c->max_blocks == 0 || c->max_blocks > (size_t)INT32_MAX)
        return set_error(err, ZQ_ERR_SHAPE, "%s: cache of %zu pages for %zu heads, %zu sequences of %zu blocks", who, c->pages, c->heads, c->batch, c->max_blocks);
    if (c->page_stride % 8 || c->page_stride < c->page_size * c->heads * c->head_dim) return set_error(err, ZQ_ERR_SHAPE, "%s: page stride %zu for pages of %zu values", who, c->page_stride, c->page_size * c->heads * c->head_dim);
    if ((reinterpret_cast<uintptr_t>(c->dev_k) | reinterpret_cast<uintptr_t>(c->dev_v)) & 15) return set_error(err, ZQ_ERR_ARG, "%s: the cache is not 16-byte aligned", who);
    out.k = static_cast<uint8_t *>(c->dev_k);
    out.v = static_cast<uint8_t *>(c->dev_v);
    out.blocks = c->dev_blocks;
    out.lens = c->dev_context_lens;
    out.page_stride = (int64_t)c->page_stride;
    out.row_stride = (int64_t)(c->heads * c->head_dim);
    out.pages = (int)c->pages;
    out.page_shift = 0;
    while ((size_t(1) << out.page_shift) < c->page_size) ++out.page_shift;
    out.max_blocks = (int)c->max_blocks;
    out.heads = (int)c->heads;
    out.head_dim = (int)c->head_dim;
    return ZQ_OK;
}

// One CTA per sequence, one thread per row.  A row's ancestors come in descending order, so that the thread gathers the bits of
// one word after the other while it climbs, and a parent that is not below its child ends the climb: no path is longer than the row's number.
__global__ void __launch_bounds__(1024) draft_tree_kernel(const int32_t *__restrict__ parents, int shared_parents, int rows, const int32_t *__restrict__ context, const int32_t *__restrict__ lens, int32_t *__restrict__ positions,
                                                          unsigned long long *__restrict__ mask, uint32_t *status) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    __shared__ int32_t s_parent[kMaxDraftRows];
    const int seq = blockIdx.x, i = threadIdx.x, words = (rows + 63) / 64;
    if (i < rows) s_parent[i] = parents[(shared_parents ? 0 : (size_t)seq * rows) + i];
    __syncthreads();
    if (i >= rows) return;
    const int ctx_len = context[seq];
    int n = draft_len(lens, seq, rows, status);
    if (ctx_len < 0 || ctx_len > INT32_MAX - rows) {
        if (i == 0) atomicMax(status, (uint32_t)kStatusBadIndex);
        n = 0;
    }
    int depth = 0, last = i;
    bool real = i < n;
    for (int j = i; real;) {  // is the whole path there?
        const int up = s_parent[j];
        if (up < -1 || up >= j) {
            atomicMax(status, (uint32_t)kStatusBadIndex);
            real = false;
        }
        if (up < 0) break;
        ++depth;
        j = up;
    }
    const size_t row = (size_t)seq * rows + i;
    positions[row] = real ? ctx_len + depth : -1;
    unsigned long long *out = mask + row * words;
    int word = words - 1;
    unsigned long long bits = 0;
    while (real && last >= 0) {
        for (; word > last >> 6; --word) {
            out[word] = bits;
            bits = 0;
        }
        bits |= 1ull << (last & 63);
        last = s_parent[last];
    }
    for (; word >= 0; --word) {
        out[word] = bits;
        bits = 0;
    }
}

struct KeepArgs {
    CacheArgs c;
    int64_t layer_stride;
    const int32_t *path, *accepted;
    int rows, chunks;  // 16-byte chunks of a cache row
    uint32_t *status;
};

// One CTA per (sequence, layer), one thread per 16 bytes of a row of K or of V, which it moves for all rows of the path: the
// same thread reads and writes a column, and path[k] >= k, so that no row is overwritten before it is read; eight rows are read before
// the first of them is written.
constexpr int kKeepHeld = 8;
__global__ void __launch_bounds__(256) cache_keep_path_kernel(const KeepArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    __shared__ int64_t s_from[kMaxDraftRows], s_to[kMaxDraftRows];
    const int seq = blockIdx.x, n = draft_len(a.accepted, seq, a.rows, a.status), start = a.c.lens[seq];
    for (int k = threadIdx.x; k < n; k += blockDim.x) {
        const int from = a.path[(size_t)seq * a.rows + k];
        int64_t src = -1, dst = -1;
        bool bad = from < k || from >= a.rows || start < 0;
        if (!bad && from != k) {
            src = cache_row(a.c, seq, (int64_t)start + from);
            dst = cache_row(a.c, seq, (int64_t)start + k);
            bad = src < 0 || dst < 0;
        }
        if (bad) {
            atomicMax(a.status, (uint32_t)kStatusBadIndex);
            src = -1;
        }
        s_from[k] = src;
        s_to[k] = dst;
    }
    __syncthreads();
    const int64_t layer = (int64_t)blockIdx.y * a.layer_stride;
    for (int c = threadIdx.x; c < 2 * a.chunks; c += blockDim.x) {
        uint4 *base = reinterpret_cast<uint4 *>((c < a.chunks ? a.c.k : a.c.v) + 2 * layer) + (c < a.chunks ? c : c - a.chunks);
        for (int k0 = 0; k0 < n; k0 += kKeepHeld) {
            uint4 held[kKeepHeld];
#pragma unroll
            for (int j = 0; j < kKeepHeld; ++j)
                if (k0 + j < n && s_from[k0 + j] >= 0) held[j] = base[s_from[k0 + j] / 8];
#pragma unroll
            for (int j = 0; j < kKeepHeld; ++j)
                if (k0 + j < n && s_from[k0 + j] >= 0) base[s_to[k0 + j] / 8] = held[j];
        }
    }
}

}  // namespace zq

using namespace zq;

extern "C" int zq_draft_tree(zq_ctx *ctx, const int32_t *dev_parents, int parents_shared, size_t batch, size_t rows, const int32_t *dev_context_lens, const int32_t *dev_draft_lens, int32_t *dev_positions, uint64_t *dev_mask, zq_error *err) {
    if (!ctx || !dev_parents || !dev_context_lens || !dev_positions || !dev_mask) return set_error(err, ZQ_ERR_ARG, "zq_draft_tree: null argument");
    if (batch == 0 || batch > 65535 || rows == 0 || rows > kMaxDraftRows) return set_error(err, ZQ_ERR_SHAPE, "zq_draft_tree: %zu sequences of %zu rows (1..65535, 1..%d)", batch, rows, kMaxDraftRows);
    int rc = use_device(ctx, err);
    if (rc) return rc;
    return launch_pdl(ctx, draft_tree_kernel, dim3((unsigned)batch), dim3((unsigned)((rows + 31) / 32 * 32)), 0, err, dev_parents, parents_shared, (int)rows, dev_context_lens, dev_draft_lens, dev_positions,
                      reinterpret_cast<unsigned long long *>(dev_mask), ctx->status_dev);
}

extern "C" int zq_cache_keep_path(zq_ctx *ctx, const zq_kv_cache *cache, const int32_t *dev_path, size_t rows, const int32_t *dev_accepted, zq_error *err) {
    if (!ctx || !dev_path || !dev_accepted) return set_error(err, ZQ_ERR_ARG, "zq_cache_keep_path: null argument");
    KeepArgs a;
    int rc = cache_args("zq_cache_keep_path", cache, a.c, err);
    if (rc) return rc;
    if (rows == 0 || rows > kMaxDraftRows) return set_error(err, ZQ_ERR_SHAPE, "zq_cache_keep_path: %zu rows (1..%d)", rows, kMaxDraftRows);
    if (cache->layers == 0 || cache->layers > 65535 || (cache->layers > 1 && cache->layer_stride % 8)) return set_error(err, ZQ_ERR_SHAPE, "zq_cache_keep_path: %zu layers %zu values apart", cache->layers, cache->layer_stride);
    if ((rc = use_device(ctx, err))) return rc;
    a.layer_stride = (int64_t)cache->layer_stride;
    a.path = dev_path;
    a.accepted = dev_accepted;
    a.rows = (int)rows;
    a.chunks = (int)(cache->heads * cache->head_dim / 8);
    a.status = ctx->status_dev;
    return launch_pdl(ctx, cache_keep_path_kernel, dim3((unsigned)cache->batch, (unsigned)cache->layers), dim3(256), 0, err, a);
}
