// What the operators on drafted tokens share: the cache as their kernels see it, and the launch of a kernel under the one before it.
#pragma once
#include "zq_common.cuh"

namespace zq {

constexpr int kMaxDraftRows = 1024;

struct CacheArgs {
    uint8_t *k, *v;
    const int32_t *blocks, *lens;
    int64_t page_stride, row_stride;  // in values
    int pages, page_shift, max_blocks, heads, head_dim;
};

// First value of the cache row of a position, -1 where the block table has no such page.
__device__ __forceinline__ int64_t cache_row(const CacheArgs &c, int seq, int64_t position) {
    const int64_t block = position >> c.page_shift;
    if (position < 0 || block >= c.max_blocks) return -1;
    const int page = c.blocks[(size_t)seq * c.max_blocks + block];
    if (page < 0 || page >= c.pages) return -1;
    return page * c.page_stride + (position & ((1 << c.page_shift) - 1)) * c.row_stride;
}

// Rows that sequence `seq` brings; a length out of range is reported and counts as none.
__device__ __forceinline__ int draft_len(const int32_t *lens, int seq, int rows, uint32_t *status) {
    if (!lens) return rows;
    const int n = lens[seq];
    if (n < 0 || n > rows) {
        atomicMax(status, (uint32_t)kStatusBadIndex);
        return 0;
    }
    return n;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two f32 operations at once.
__device__ __forceinline__ uint64_t pair64(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ void unpair64(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t twice(float v) { return pair64(__float_as_uint(v), __float_as_uint(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

int cache_args(const char *who, const zq_kv_cache *cache, CacheArgs &out, zq_error *err);

template <class... P, class... A> int launch_pdl(zq_ctx *ctx, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, zq_error *err, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->disable_pdl ? 0 : 1;
    ZQ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...), err);
    ctx->launches++;
    return ZQ_OK;
}

}  // namespace zq
