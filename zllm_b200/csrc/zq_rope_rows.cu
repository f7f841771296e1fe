// Rotary positions of single rows, from frequencies: the rows of a drafted tree, batches of sequences of unequal length, contexts
// longer than a table; optionally with the keys and values written to a paged cache.
//
//     (re, im) <- factor * (re cos t - im sin t, im cos t + re sin t),   t = position * inv_freq[pair]
//
// t reaches 1e6 and more, where an f32 product is off by tenths of a radian; here the product is exact (24 + 24 bits in f64), its whole
// turns come off in f64, and the rest of it, at most half a turn, goes through sincospif: 1e-7 at any position.
//
// Bound by memory, each value read and written once.  A CTA takes as many rows as fill its 128 or 256 threads.  A thread has one place in a head (a vector of
// pairs) and takes it in several heads, so that offsets and sines are computed or read once for all of them; it asks for the first three heads'
// values before anything else: the look-ups of position and page and the angles hide under the loads.
#include <cmath>
#include <type_traits>

#include "zq_draft.cuh"

namespace zq {

constexpr int kAhead = 3, kMaxRopeHead = 512;  // heads a thread asks for at once; values of a head

struct RopeRowsArgs {
    const uint8_t *q, *k, *v;
    uint8_t *q_out, *k_out;
    const int32_t *positions, *lens;
    const float *inv_freq;
    CacheArgs cache;  // cache.k null: keys go to k_out
    int64_t q_stride, k_stride, v_stride;  // values between rows
    int64_t rows;
    int rows_per_seq, q_heads, k_heads, v_heads, head_dim, rotary, start, interleaved, inverse;
    float factor;
    int log_threads, places, heads;  // threads of a row, places of a head, heads of q, k and v that the threads take at a time
    uint32_t *status;
};

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values of a word.
template <class T> __device__ __forceinline__ float2 two_f32(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T> __device__ __forceinline__ uint32_t from_two(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}

template <class T, int N> struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

// VEC values per access: 16 bytes where head, turned part, strides and addresses allow, else one value.  A place is VEC pairs (two vectors, of which an
// interleaved one is the other's neighbour) or 2 VEC values that are copied; the sines lie so that neighbouring threads read neighbouring ones.
template <class T, int VEC> __global__ void __launch_bounds__(256, 4) rope_rows_kernel(const RopeRowsArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    extern __shared__ float2 s_turn[];
    using V = Vec<T, VEC>;
    const int lane = threadIdx.x & ((1 << a.log_threads) - 1), slot = threadIdx.x >> a.log_threads, half = a.rotary / 2;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> a.log_threads) + slot;
    const int h0 = (int)((unsigned)lane / (unsigned)a.places), c = lane - h0 * a.places, all = a.q_heads + a.k_heads + a.v_heads;
    const bool here = row < a.rows && h0 < a.heads;
    // the place in a head of q or k (its first pair, or -1 outside the turned part), and in one of v; a second vector at head_dim is none
    const int pairs = half / VEC, at = 2 * VEC * (c - pairs);
    const int pair = c < pairs ? c * VEC : -1;
    const int first = pair >= 0 ? a.start + (a.interleaved ? 2 * pair : pair) : a.start ? at : a.rotary + at;
    const int second = pair >= 0 ? first + (a.interleaved ? VEC : half) : first + VEC < (a.start ? a.start : a.head_dim) ? first + VEC : a.head_dim;
    const T *q = reinterpret_cast<const T *>(a.q) + row * a.q_stride, *k = reinterpret_cast<const T *>(a.k) + row * a.k_stride, *v = reinterpret_cast<const T *>(a.v) + row * a.v_stride;

    auto load = [&](int h, V &x, V &y) {
        const bool is_v = h >= a.q_heads + a.k_heads;
        const T *src = h < a.q_heads ? q + h * a.head_dim : is_v ? v + (h - a.q_heads - a.k_heads) * a.head_dim : k + (h - a.q_heads) * a.head_dim;
        const int i = is_v ? 2 * VEC * c : first, j = is_v ? i + VEC : second;
        x = *reinterpret_cast<const V *>(src + i);
        if (j < a.head_dim) y = *reinterpret_cast<const V *>(src + j);
    };
    V xs[kAhead], ys[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        if (here && h0 + j * a.heads < all) load(h0 + j * a.heads, xs[j], ys[j]);
    const int position = row < a.rows ? a.positions[row] : -1;
    int64_t keep = -1;  // the cache row, or -1
    if (a.cache.k && row < a.rows) {
        const int seq = (int)((unsigned)row / (unsigned)a.rows_per_seq), i = (int)row - seq * a.rows_per_seq, start = a.cache.lens[seq];
        if (i < draft_len(a.lens, seq, a.rows_per_seq, a.status) && position >= 0) {
            keep = start < 0 ? -1 : cache_row(a.cache, seq, (int64_t)start + i);
            if (keep < 0) atomicMax(a.status, (uint32_t)kStatusBadIndex);
        }
    }
    float2 *turn = s_turn + slot * half;
    if (position >= 0) {
        for (int p = lane; p < half; p += 1 << a.log_threads) {
            double t = (double)position * (double)a.inv_freq[p] * 0.15915494309189533577;  // in turns
            t -= rint(t);
            float s, c;
            sincospif(2.f * (float)t, &s, &c);
            turn[p % VEC * (half / VEC) + p / VEC] = make_float2(c * a.factor, a.inverse ? -s * a.factor : s * a.factor);
        }
    }
    __syncthreads();
    if (!here) return;
    const bool turns = pair >= 0 && position >= 0;
    T *q_out = reinterpret_cast<T *>(a.q_out) + row * a.q_heads * a.head_dim, *k_out = a.cache.k ? reinterpret_cast<T *>(a.cache.k) + keep : reinterpret_cast<T *>(a.k_out) + row * a.k_heads * a.head_dim,
      *v_out = reinterpret_cast<T *>(a.cache.v) + keep;
    auto finish = [&](int h, V x, V y) {
        const bool is_v = h >= a.q_heads + a.k_heads;
        if (h >= a.q_heads && a.cache.k && keep < 0) return;
        if (turns && !is_v) {
            if constexpr (sizeof(T) == 2 && VEC > 1) {
                uint32_t xw[VEC / 2], yw[VEC / 2];
                memcpy(xw, &x, sizeof(x));
                memcpy(yw, &y, sizeof(y));
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    const float2 a0 = turn[j * pairs + c], a1 = turn[(j + 1) * pairs + c];
                    if (a.interleaved) {  // words 0..VEC/2 are x's pairs, the others y's
                        uint32_t &w0 = j < VEC / 2 ? xw[j] : yw[j - VEC / 2], &w1 = j < VEC / 2 ? xw[j + 1] : yw[j + 1 - VEC / 2];
                        const float2 s = two_f32<T>(w0), t = two_f32<T>(w1);
                        w0 = from_two<T>(s.x * a0.x - s.y * a0.y, s.y * a0.x + s.x * a0.y);
                        w1 = from_two<T>(t.x * a1.x - t.y * a1.y, t.y * a1.x + t.x * a1.y);
                    } else {
                        const float2 re = two_f32<T>(xw[j / 2]), im = two_f32<T>(yw[j / 2]);
                        xw[j / 2] = from_two<T>(re.x * a0.x - im.x * a0.y, re.y * a1.x - im.y * a1.y);
                        yw[j / 2] = from_two<T>(im.x * a0.x + re.x * a0.y, im.y * a1.x + re.y * a1.y);
                    }
                }
                memcpy(&x, xw, sizeof(x));
                memcpy(&y, yw, sizeof(y));
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const bool beside = a.interleaved && VEC > 1;
                    T &r = beside ? (2 * j < VEC ? x : y).v[2 * j % VEC] : x.v[j], &i = beside ? (2 * j < VEC ? x : y).v[(2 * j + 1) % VEC] : y.v[j];
                    const float re = to_f32(r), im = to_f32(i);
                    r = from_f32<T>(re * turn[j * pairs + c].x - im * turn[j * pairs + c].y);
                    i = from_f32<T>(im * turn[j * pairs + c].x + re * turn[j * pairs + c].y);
                }
            }
        }
        T *dst = h < a.q_heads ? q_out + h * a.head_dim : is_v ? v_out + (h - a.q_heads - a.k_heads) * a.head_dim : k_out + (h - a.q_heads) * a.head_dim;
        const int i = is_v ? 2 * VEC * c : first, j = is_v ? i + VEC : second;
        *reinterpret_cast<V *>(dst + i) = x;
        if (j < a.head_dim) *reinterpret_cast<V *>(dst + j) = y;
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        if (h0 + j * a.heads < all) finish(h0 + j * a.heads, xs[j], ys[j]);
    for (int h = h0 + kAhead * a.heads; h < all; h += a.heads) {
        V x, y;
        load(h, x, y);
        finish(h, x, y);
    }
}

static int rope_checks(const char *who, zq_ctx *ctx, const RopeRowsArgs &a, int dtype, size_t q_heads, size_t q_stride, size_t k_heads, size_t k_stride, size_t v_stride, size_t rows, size_t head_dim, size_t rotary, int layout, int placement,
                       float factor, zq_error *err) {
    if (!ctx || !a.q || !a.q_out || !a.positions || !a.inv_freq) return set_error(err, ZQ_ERR_ARG, "%s: null argument", who);
    if (dtype != ZQ_F32 && dtype != ZQ_F16 && dtype != ZQ_BF16) return set_error(err, ZQ_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if ((layout != ZQ_ROPE_SPLIT_HALF && layout != ZQ_ROPE_INTERLEAVED) || (placement != ZQ_ROPE_PREFIX && placement != ZQ_ROPE_SUFFIX)) return set_error(err, ZQ_ERR_ARG, "%s: unknown layout %d or placement %d", who, layout, placement);
    if (q_heads == 0 || rotary == 0 || rotary % 2 || head_dim == 0 || head_dim > kMaxRopeHead) return set_error(err, ZQ_ERR_SHAPE, "%s: heads=%zu head_dim=%zu rotary=%zu (a head of up to 512 values, rotary even and positive)", who, q_heads, head_dim, rotary);
    if (rotary > head_dim) return set_error(err, ZQ_ERR_SHAPE, "%s: rotary=%zu exceeds head_dim=%zu", who, rotary, head_dim);
    if (rows == 0 || rows > (size_t)INT32_MAX) return set_error(err, ZQ_ERR_SHAPE, "%s: %zu rows", who, rows);
    if ((q_heads + 2 * k_heads) * head_dim > (size_t(1) << 20) || q_heads > (size_t(1) << 20) || k_heads > (size_t(1) << 20)) return set_error(err, ZQ_ERR_SHAPE, "%s: rows of %zu and %zu heads of %zu values are too large", who, q_heads, k_heads, head_dim);
    if (q_stride < q_heads * head_dim || (a.k && k_stride < k_heads * head_dim) || (a.v && v_stride < k_heads * head_dim)) return set_error(err, ZQ_ERR_SHAPE, "%s: rows overlap (strides %zu, %zu, %zu)", who, q_stride, k_stride, v_stride);
    if (q_stride > (size_t)INT32_MAX || k_stride > (size_t)INT32_MAX || v_stride > (size_t)INT32_MAX) return set_error(err, ZQ_ERR_SHAPE, "%s: shape too large", who);
    if ((a.q_out == a.q && q_stride != q_heads * head_dim) || (a.k && a.k_out == a.k && k_stride != k_heads * head_dim)) return set_error(err, ZQ_ERR_ARG, "%s: in place only where the rows are dense", who);
    if (!std::isfinite(factor)) return set_error(err, ZQ_ERR_ARG, "%s: the factor is not finite", who);
    return ZQ_OK;
}

template <class T> static int launch_rope_rows(zq_ctx *ctx, RopeRowsArgs &a, zq_error *err) {
    constexpr int kWide = 16 / sizeof(T);
    // pairs of an item lie in two vectors: half a turned part (split halves) or two neighbours (interleaved)
    const int half = a.rotary / 2, rest = a.head_dim - a.rotary;
    bool wide = a.head_dim % kWide == 0 && a.rotary % (2 * kWide) == 0 && a.start % kWide == 0 && a.q_stride % kWide == 0 && (!a.k || a.k_stride % kWide == 0) && (!a.v || a.v_stride % kWide == 0);
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k_out);
    wide = wide && (at & 15) == 0;
    const int vec = wide ? kWide : 1;
    a.places = half / vec + (rest + 2 * vec - 1) / (2 * vec);  // of v as many: the turned part is whole places
    const int all = a.q_heads + a.k_heads + a.v_heads;
    // a row's threads: enough for its heads in three turns where rows are many (their look-ups are then fewer), in one where an SM has few
    const int64_t turns = a.rows > 4 * ctx->sm_count ? kAhead : 1;
    a.log_threads = 5;
    while (a.log_threads < 8 && ((1 << a.log_threads) < a.places || (1 << a.log_threads) / a.places * turns < all)) ++a.log_threads;
    a.heads = (1 << a.log_threads) / a.places;
    const int threads = a.log_threads < 7 ? 128 : 1 << a.log_threads, per_cta = threads >> a.log_threads;
    const dim3 grid((unsigned)((a.rows + per_cta - 1) / per_cta));
    const size_t smem = (size_t)per_cta * half * sizeof(float2);
    return wide ? launch_pdl(ctx, rope_rows_kernel<T, kWide>, grid, dim3((unsigned)threads), smem, err, a) : launch_pdl(ctx, rope_rows_kernel<T, 1>, grid, dim3((unsigned)threads), smem, err, a);
}

static int launch_rope_rows(zq_ctx *ctx, RopeRowsArgs &a, int dtype, zq_error *err) {
    int rc = use_device(ctx, err);
    if (rc) return rc;
    a.status = ctx->status_dev;
    return dtype == ZQ_F32 ? launch_rope_rows<float>(ctx, a, err) : dtype == ZQ_F16 ? launch_rope_rows<__half>(ctx, a, err) : launch_rope_rows<__nv_bfloat16>(ctx, a, err);
}

}  // namespace zq

using namespace zq;

extern "C" int zq_rope_frequencies(size_t rotary_dim, double base, int scaling, double factor, double original_context, double beta_slow, double beta_fast, const float *pair_factors, float *out_inv_freq, float *out_factor, zq_error *err) {
    if (!out_inv_freq || !out_factor) return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: null argument");
    if (rotary_dim == 0 || rotary_dim % 2 || rotary_dim > 4096) return set_error(err, ZQ_ERR_SHAPE, "zq_rope_frequencies: rotary=%zu (rotary must be even and positive)", rotary_dim);
    const bool yarn = scaling == ZQ_ROPE_SCALE_YARN || scaling == ZQ_ROPE_SCALE_YARN_PAIRS;
    if (scaling != ZQ_ROPE_SCALE_NONE && scaling != ZQ_ROPE_SCALE_LINEAR && !yarn) return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: unknown scaling %d", scaling);
    if (!(base > 0) || !std::isfinite(base)) return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: base %g", base);
    if (scaling != ZQ_ROPE_SCALE_NONE && (!(factor > 0) || !std::isfinite(factor))) return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: factor %g", factor);
    if (yarn && (!(original_context > 0) || !std::isfinite(original_context) || !(beta_fast > beta_slow) || !std::isfinite(beta_fast) || !std::isfinite(beta_slow)))
        return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: original context %g, turns %g to %g", original_context, beta_slow, beta_fast);
    if (scaling == ZQ_ROPE_SCALE_YARN_PAIRS && (!(base > 1) || !(beta_slow > 0))) return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: base %g, turns from %g: the pairs that turn so often have no number", base, beta_slow);
    const size_t half = rotary_dim / 2;
    constexpr double kTurn = 6.28318530717958647692;
    // base^(-i / half) original_context / (2 pi) turns: i from the turns
    auto number = [&](double turns) { return (double)half * std::log(original_context / (turns * kTurn)) / std::log(base); };
    auto limited = [&](double i) { return i < 0 ? 0 : i > (double)(rotary_dim - 1) ? (double)(rotary_dim - 1) : i; };
    const double low = scaling == ZQ_ROPE_SCALE_YARN_PAIRS ? limited(std::floor(number(beta_fast))) : 0, high = scaling == ZQ_ROPE_SCALE_YARN_PAIRS ? limited(std::ceil(number(beta_slow))) : 0;
    for (size_t i = 0; i < half; ++i) {
        double f = std::pow(base, -(double)i / (double)half);
        if (pair_factors) {
            if (!(pair_factors[i] > 0)) return set_error(err, ZQ_ERR_ARG, "zq_rope_frequencies: pair factor %g", (double)pair_factors[i]);
            f /= (double)pair_factors[i];
        }
        if (scaling == ZQ_ROPE_SCALE_LINEAR) f /= factor;
        if (yarn) {
            double keep;
            if (scaling == ZQ_ROPE_SCALE_YARN) keep = (original_context * f / kTurn - beta_slow) / (beta_fast - beta_slow);
            else keep = high > low ? (high - (double)i) / (high - low) : (double)i <= low ? 1 : 0;
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / factor * (1 - keep);
        }
        out_inv_freq[i] = (float)f;
    }
    *out_factor = yarn && factor > 1 ? (float)(0.1 * std::log(factor) + 1.0) : 1.f;
    return ZQ_OK;
}

extern "C" int zq_rope_rows(zq_ctx *ctx, const void *dev_q, size_t q_heads, size_t q_stride, const void *dev_k, size_t k_heads, size_t k_stride, int dtype, size_t rows, size_t head_dim, size_t rotary_dim, int layout, int placement,
                            const int32_t *dev_positions, const float *dev_inv_freq, float factor, int inverse, void *dev_q_out, void *dev_k_out, zq_error *err) {
    RopeRowsArgs a = {};
    a.q = static_cast<const uint8_t *>(dev_q);
    a.k = static_cast<const uint8_t *>(dev_k);
    a.q_out = static_cast<uint8_t *>(dev_q_out);
    a.k_out = static_cast<uint8_t *>(dev_k_out);
    a.positions = dev_positions;
    a.inv_freq = dev_inv_freq;
    int rc = rope_checks("zq_rope_rows", ctx, a, dtype, q_heads, q_stride, k_heads, k_stride, 0, rows, head_dim, rotary_dim, layout, placement, factor, err);
    if (rc) return rc;
    if (dev_k && (!dev_k_out || k_heads == 0)) return set_error(err, ZQ_ERR_ARG, "zq_rope_rows: key given without heads or without an output");
    a.q_stride = (int64_t)q_stride;
    a.k_stride = (int64_t)k_stride;
    a.rows = (int64_t)rows;
    a.rows_per_seq = 1;
    a.q_heads = (int)q_heads;
    a.k_heads = dev_k ? (int)k_heads : 0;
    a.head_dim = (int)head_dim;
    a.rotary = (int)rotary_dim;
    a.start = placement == ZQ_ROPE_SUFFIX ? (int)(head_dim - rotary_dim) : 0;
    a.interleaved = layout == ZQ_ROPE_INTERLEAVED;
    a.inverse = inverse;
    a.factor = factor;
    return launch_rope_rows(ctx, a, dtype, err);
}

extern "C" int zq_rope_append(zq_ctx *ctx, const void *dev_q, size_t q_heads, size_t q_stride, const void *dev_k, size_t k_stride, const void *dev_v, size_t v_stride, size_t rows_per_seq, const zq_kv_cache *cache, const int32_t *dev_draft_lens,
                              size_t rotary_dim, int layout, int placement, const int32_t *dev_positions, const float *dev_inv_freq, float factor, void *dev_q_out, zq_error *err) {
    if (!dev_k || !dev_v) return set_error(err, ZQ_ERR_ARG, "zq_rope_append: null argument");
    RopeRowsArgs a = {};
    int rc = cache_args("zq_rope_append", cache, a.cache, err);
    if (rc) return rc;
    a.q = static_cast<const uint8_t *>(dev_q);
    a.k = static_cast<const uint8_t *>(dev_k);
    a.v = static_cast<const uint8_t *>(dev_v);
    a.q_out = static_cast<uint8_t *>(dev_q_out);
    a.positions = dev_positions;
    a.lens = dev_draft_lens;
    a.inv_freq = dev_inv_freq;
    if (rows_per_seq == 0 || rows_per_seq > (size_t(1) << 20)) return set_error(err, ZQ_ERR_SHAPE, "zq_rope_append: %zu rows of a sequence", rows_per_seq);
    rc = rope_checks("zq_rope_append", ctx, a, cache->dtype, q_heads, q_stride, cache->heads, k_stride, v_stride, rows_per_seq * cache->batch, cache->head_dim, rotary_dim, layout, placement, factor, err);
    if (rc) return rc;
    a.q_stride = (int64_t)q_stride;
    a.k_stride = (int64_t)k_stride;
    a.v_stride = (int64_t)v_stride;
    a.rows = (int64_t)(rows_per_seq * cache->batch);
    a.rows_per_seq = (int)rows_per_seq;
    a.q_heads = (int)q_heads;
    a.k_heads = a.v_heads = (int)cache->heads;
    a.head_dim = (int)cache->head_dim;
    a.rotary = (int)rotary_dim;
    a.start = placement == ZQ_ROPE_SUFFIX ? (int)(cache->head_dim - rotary_dim) : 0;
    a.interleaved = layout == ZQ_ROPE_INTERLEAVED;
    a.factor = factor;
    return launch_rope_rows(ctx, a, cache->dtype, err);
}
