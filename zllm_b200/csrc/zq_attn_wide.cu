// Attention of many rows per key (drafted rows times query heads of a cache head) on the 5th-generation tensor cores.
//
// The same sums and the same shares as in zq_attn.cu, in tiles of 128 rows by 128 keys: S = Q K^T into tensor memory, the weights from
// there through registers back into tensor memory (the same columns), O += P V.  A CTA per SM has
//   warp 8      the copies: TMA boxes of a page by 64 values, K and V tiles in turn through one ring of 128-byte swizzled tiles;
//   warp 9      the MMAs (tcgen05, one lane);
//   warps 0..3  slot 0 and warps 4..7 slot 1: a thread has a row of S and O, so largest score and sum need no exchange.
// The slots take turns at the tensor cores: while one turns scores into weights, the other's products run.  With more than 128 rows (PAIR) they hold two row tiles
// against the same keys, else the same rows against every other tile of keys, and add up at the end of the item.
//
// O stays in tensor memory while the largest score rises by less than 2^8: the weights are taken relative to an older maximum (exact in f32,
// and the sum with them), so that the sums so far are hardly ever multiplied down.
//
// Bytes against tensor cycles: a tile of 128 keys of 128 values is 64 KB, 1.49 us at an SM's share of the memory rate (2850 cycles at 1.9 GHz, 2400 to 2550 at the 1.6 to
// 1.7 GHz of long runs); its products take 1024 cycles per slot of rows and its exponentials as many, so up to 256 rows the copies bound it. (ptxas spills 40 to 104 bytes a thread.)
//
// Padding and the end of a sequence: boxes are whole pages, and what lies behind the sequence's end must not reach a row (0 * NaN): in tiles that hold
// drafted rows or the end, a slot's threads clear those rows of V in shared memory, and infinities and NaN of drafted rows, which they
// add to O of the rows that see them.
#include <cstddef>
#include <type_traits>

#include "zq_attn.cuh"

namespace zq {

constexpr int kWideThreads = 320, kWideTile = 128, kBarBytes = 3 << 10;
constexpr int kRise = 8;  // the largest score may rise by so much, as a power of two of its weight, before the sums follow
// What the end of an item and the start of the next cost, in tiles of keys: some 10 000 cycles in which the ring stands still (the sums out of tensor memory, the first
// weights with no product beside them).  40 rows per cache head of 128, 4 cache heads: 64 unequal sequences of up to 200 and 1000, 150 of 900 and 16 of 8000
// positions take 34.7 / 50.5 / 93 / 48.4 us without it, 28.0 / 41.6 / 74 / 45.4 with 7, 27.9 / 42.5 / 74 / 45.6 with 11.
constexpr int kWideEnd = 7;

__device__ __forceinline__ bool wide_elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
}
// Waits for this thread's loads; the values pass through, so that nothing uses them before.
__device__ __forceinline__ void tm_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
        "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int head, int row, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(head), "r"(row), "r"(page)
                 : "memory");
}
// A tile of 128-byte swizzled rows, eight rows (1024 bytes) from one group to the next.  K-major (Q, K: a row is 64 values of the reduced
// dimension): the leading offset is not used.  The other way round (V: a row is a key, the reduced dimension): the leading offset leads to the next 64 values.
// sw128_low is the half that holds the address; one lane's value for the warp, so that the MMAs' operands are uniform registers.
__device__ __forceinline__ uint32_t sw128_low(uint32_t addr, uint32_t leading) { return __shfl_sync(0xffffffffu, (addr & 0x3FFFFu) >> 4 | leading >> 4 << 16, 0); }
__device__ __forceinline__ uint64_t sw128_desc(uint32_t low) { return (uint64_t)low | (uint64_t)(1024 >> 4 | 1 << 14 | 2u << 29) << 32; }

template <int D> struct WideShape {
    static constexpr int kBlocks = D / 64;
    static constexpr int kBlock = kWideTile * 128;      // bytes of 64 values of 128 rows
    static constexpr int kTileBytes = kBlocks * kBlock;
    static constexpr int kRing = D == 128 ? 5 : 10;     // K and V tiles
    static constexpr int kQ = 0, kPlace = 2 * kWideTile * 128, kRingAt = 2 * kPlace, kBars = kRingAt + kRing * kTileBytes;
    static_assert(kTileBytes <= kPlace, "a place of Q: a tile, later 32 columns of both slots' sums");
    static constexpr int kSmem = kBars + kBarBytes;     // barriers, maxima and sums of the slots' rows
    static_assert(kSmem <= 227 << 10, "shared memory");
};

struct WideBars {
    uint64_t full[10], empty[10], scores[2], weights[2], sums[2], q[2], left[2], start, end;  // 8 bytes each, at kFull and so on
    uint32_t tmem, dead, poison[2][4];     // rows of a tile of V that were cleared of infinities and NaN, per slot
    float top[2][kWideTile], sum[2][kWideTile];  // of the slots' rows, when the slots share rows
};
constexpr uint32_t kFull = 0, kEmpty = 80, kScores = 160, kWeights = 176, kSums = 192, kQ = 208, kLeft = 224, kStart = 240, kEnd = 248;
static_assert(sizeof(WideBars) <= kBarBytes && offsetof(WideBars, q) == kQ && offsetof(WideBars, left) == kLeft && offsetof(WideBars, start) == kStart && offsetof(WideBars, end) == kEnd, "barriers");

__device__ __forceinline__ bool poll(uint32_t at, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(at), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __noinline__ void wait_on(uint32_t at, uint32_t parity, volatile uint32_t *dead, uint32_t *status, uint32_t code) {
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        if (poll(at, parity) || *dead) return;
    }
    *dead = 1;
    atomicMax(status, code);
}

template <int D, bool BF16, bool PAIR> __global__ void __launch_bounds__(kWideThreads, 1) wide_attention_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using S = WideShape<D>;
    constexpr int kRows = PAIR ? 2 * kWideTile : kWideTile;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    WideBars &bar = *reinterpret_cast<WideBars *>(smem + S::kBars);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    if (tid == 0) {
        for (int i = 0; i < S::kRing; ++i) {
            mbar_init(&bar.full[i], 1);
            mbar_init(&bar.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.scores[i], 1);
            mbar_init(&bar.weights[i], kWideTile);
            mbar_init(&bar.sums[i], 1);
            mbar_init(&bar.q[i], PAIR ? kWideTile : 32);
            mbar_init(&bar.left[i], 2 * kWideTile);
        }
        mbar_init(&bar.start, kWideThreads);
        mbar_init(&bar.end, 1);
        bar.dead = 0;
        fence_mbar_init();
        a.info[blockIdx.x] = make_int4(0, 0, 0, 0);
        if (base & 1023) atomicMax(a.status, (uint32_t)kStatusTmaTimeout);  // swizzled tiles begin at multiples of 1024 bytes
    }
    if (base & 1023) return;
    const Share share = find_share<kWideThreads>(a, kWideTile, kWideEnd, smem);
    if (share.first >= share.last) return;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 8 && wide_elect()) {
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bar.tmem, 0);
    const int d = a.c.head_dim;

    // Bounded wait of a whole warp.  One that runs out is reported, and from then on the CTA waits for nothing and walks to its end.
    // (The first poll is in line and nearly always enough.  The MMA warp shares its scheduler's instruction cache with the long loops of the slots: its
    // waits took 350 cycles each while they polled, voted and computed the barrier's place in 60 instructions.)
    const uint32_t bars = base + S::kBars;
    auto wait = [&](uint32_t offset, uint32_t parity, uint32_t code) {
        if (!poll(bars + offset, parity)) wait_on(bars + offset, parity, &bar.dead, a.status, code);
        __syncwarp();
    };

    // The items of this CTA's share, one after the other; every role walks them for itself.
    int seq = share.seq;
    int64_t seq_first = share.seq_first, u = share.first;
    SeqLen len = seq_len(a, seq);
    int units = units_of(len, kWideTile), head = 0, tile = 0, ua = 0, ub = 0, item = 0, keys = 0;
    int64_t item_first = 0;
    auto next_item = [&]() {
        do {
            if (u >= share.last) return false;
            while (u >= seq_first + (int64_t)(units + share.extra) * a.c.heads * a.tiles) {
                seq_first += (int64_t)(units + share.extra) * a.c.heads * a.tiles;
                len = seq_len(a, ++seq);
                units = units_of(len, kWideTile);
            }
            item = (int)((u - seq_first) / (units + share.extra));
            item_first = seq_first + (int64_t)item * (units + share.extra);
            ua = (int)(u - item_first);
            u = item_first + units + share.extra;
        } while (ua >= units);  // a share that begins behind an item's units
        head = item / a.tiles;
        tile = item % a.tiles;
        ub = (int)min((int64_t)units, share.last - item_first);
        keys = len.rows ? len.context + len.rows : 0;
        return true;
    };

    // The rows of Q of an item into one of two tiles, in turn (slots that have rows of their own load them themselves: their tiles have no second place).  The first
    // item's by all threads, those of the next ones by the copying warp while the item before is worked on.
    int nth = 0;  // item of this CTA
    auto load_q = [&](int who, int of) {
        const uint8_t *from = a.q + 2 * ((int64_t)seq * a.rows * a.q_stride + (int64_t)head * a.group * d);
        const uint32_t to = base + S::kQ + (nth & 1) * S::kPlace;
#pragma unroll 2
        for (int idx = who; idx < kWideTile * (D / 8); idx += of) {
            const int r = idx / (D / 8), c = idx % (D / 8), q_row = tile * kRows + r, qi = (int)((unsigned)q_row / (unsigned)a.group);
            const bool there = qi < len.rows && 8 * c < d;
            cp_async16(to + (c >> 3) * S::kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4), there ? from + 2 * (qi * a.q_stride + (int64_t)(q_row - qi * a.group) * d + 8 * c) : a.q, there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto have_q = [&](uint64_t *barrier) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async();
        mbar_arrive(barrier);
    };
    bool more = next_item();
    if (!PAIR && more) load_q(tid, kWideThreads);

    if (warp == 8) {
        // ---- copies
        const int box_shift = min(a.c.page_shift, 7), boxes = kWideTile >> box_shift, box_rows = 1 << box_shift;
        uint32_t at = 0, phase = 0;  // ring place; how often round
        for (; more; more = next_item(), ++nth) {
            auto page_of = [&](int t) {
                const int key = t * kWideTile + lane * box_rows;
                if (lane >= boxes || t >= ub || key >= keys) return a.c.pages;  // no page: zeros
                const int page = a.c.blocks[(size_t)seq * a.c.max_blocks + (key >> a.c.page_shift)];
                if (page >= 0 && page < a.c.pages) return page;
                atomicMax(a.status, (uint32_t)kStatusBadIndex);
                return a.c.pages;
            };
            int ahead = page_of(ua);
            for (int t = ua; t < ub; ++t) {
                const int page = ahead, row = (t * kWideTile + lane * box_rows) & ((1 << a.c.page_shift) - 1);
                ahead = page_of(t + 1);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (phase) wait(kEmpty + 8 * at, (phase - 1) & 1, kStatusMmaTimeout);
                    if (wide_elect()) mbar_expect_tx(&bar.full[at], S::kTileBytes);
                    __syncwarp();
                    if (lane < boxes) {
                        const uint32_t dst = base + S::kRingAt + at * S::kTileBytes + lane * box_rows * 128;
#pragma unroll
                        for (int b = 0; b < S::kBlocks; ++b) tma_load_page(dst + b * S::kBlock, kv ? &map_v : &map_k, &bar.full[at], 64 * b, head, row, page);
                    }
                    if (++at == S::kRing) {
                        at = 0;
                        ++phase;
                    }
                }
                if (!PAIR && t == ua) {
                    if (nth) {
                        if (nth > 1) wait(kLeft + 8 * (nth & 1), ((nth >> 1) - 1) & 1, kStatusMmaTimeout);
                        load_q(lane, 32);
                    }
                    have_q(nth ? &bar.q[nth & 1] : &bar.start);
                }
            }
        }
        // where waits ran out, nobody has waited for the last copies
        if (*reinterpret_cast<volatile uint32_t *>(&bar.dead)) {
            for (int i = 0; i < S::kRing; ++i) {
                const uint32_t rounds = phase + (i < (int)at ? 1 : 0);
                if (rounds) mbar_wait_bounded(&bar.full[i], (rounds - 1) & 1);
            }
        }
    } else if (warp == 9) {
        // ---- MMAs
        const uint32_t type = BF16 ? 1u << 7 | 1u << 10 : 0u;
        const uint32_t idesc_s = 1u << 4 | type | (uint32_t)(kWideTile >> 3) << 17 | (uint32_t)(kWideTile >> 4) << 24;
        const uint32_t idesc_o = 1u << 4 | type | 1u << 16 | (uint32_t)(D >> 3) << 17 | (uint32_t)(kWideTile >> 4) << 24;
        uint32_t q_phase = 0, w_phase[2] = {0, 0};
        struct Place {  // in the ring: K tiles take every other one, V tiles those between
            uint32_t slot, parity;
            __device__ __forceinline__ void step() {
                slot += 2;
                if (slot >= S::kRing) {
                    slot -= S::kRing;
                    parity ^= 1;
                }
            }
        } k_at{0, 0}, v_at{1, 0};
        const uint32_t ring_k = sw128_low(base + S::kRingAt, 16), ring_v = sw128_low(base + S::kRingAt, S::kBlock);
        const uint32_t q_at[2] = {sw128_low(base + S::kQ, 16), sw128_low(base + S::kQ + S::kPlace, 16)};  // of the slots, or of this item and the next
        if (!PAIR && more) have_q(&bar.start);
        // products of slot s: scores with the K tile at k_at, sums with the V tile at v_at
        auto scores = [&](int s) {
            if (!PAIR || s == 0) wait(kFull + 8 * k_at.slot, k_at.parity, kStatusTmaTimeout);
            tc_after();
            const uint32_t q_low = q_at[PAIR ? s : nth & 1];
            const uint32_t kd = __shfl_sync(0xffffffffu, ring_k + k_at.slot * (S::kTileBytes / 16), 0), release = bars + kEmpty + 8 * k_at.slot;
            if (wide_elect()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k >> 2) * (S::kBlock / 16) + (k & 3) * 2;
                    mma_ss(tmem + s * 256, sw128_desc(q_low + off), sw128_desc(kd + off), idesc_s, k > 0);
                }
                tc_commit(bars + kScores + 8 * s);
                if (!PAIR || s == 1) tc_commit(release);
            }
            __syncwarp();
            if (!PAIR || s == 1) k_at.step();
        };
        auto sums = [&](int s) {
            if (!PAIR || s == 0) wait(kFull + 8 * v_at.slot, v_at.parity, kStatusTmaTimeout);
            wait(kWeights + 8 * s, w_phase[s], kStatusMmaTimeout);
            w_phase[s] ^= 1;
            tc_after();
            const uint32_t vd = __shfl_sync(0xffffffffu, ring_v + v_at.slot * (S::kTileBytes / 16), 0), release = bars + kEmpty + 8 * v_at.slot;
            if (wide_elect()) {
#pragma unroll
                for (int k = 0; k < kWideTile / 16; ++k) mma_ts(tmem + s * 256 + 128, tmem + s * 256 + 8 * k, sw128_desc(vd + k * (2048 / 16)), idesc_o);
                tc_commit(bars + kSums + 8 * s);
                if (!PAIR || s == 1) tc_commit(release);
            }
            __syncwarp();
            if (!PAIR || s == 1) v_at.step();
        };
        for (; more; more = next_item(), ++nth) {
            const int n = ub - ua, jobs = PAIR ? 2 * n : n;
            if (PAIR) {
                wait(kQ, q_phase, kStatusMmaTimeout);
                wait(kQ + 8, q_phase, kStatusMmaTimeout);
                q_phase ^= 1;
            } else if (nth) {
                wait(kQ + 8 * (nth & 1), (nth - 1) >> 1 & 1, kStatusMmaTimeout);
            } else {
                wait(kStart, 0, kStatusMmaTimeout);
            }
            scores(0);
            if (jobs > 1) scores(1);
#pragma unroll 1
            for (int j = 0; j < jobs; j += 2) {
                sums(0);
                if (j + 2 < jobs) scores(0);
                if (j + 1 < jobs) {
                    sums(1);
                    if (j + 3 < jobs) scores(1);
                }
            }
        }
        if (wide_elect()) tc_commit(bars + kEnd);
        __syncwarp();
        // with a limit of its own, not `wait`: where another wait ran out, MMAs may still be on their way to the tensor memory that is given back below
        if (!mbar_wait_bounded(&bar.end, 0)) atomicMax(a.status, (uint32_t)kStatusMmaTimeout);
        __syncwarp();
    } else {
        // ---- scores to weights
        const int s = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16, t_s = tmem + s * 256 + lanes, t_o = t_s + 128;
        uint32_t s_phase = 0;
        uint32_t n_sums = 0;   // products that this slot has been through
        uint32_t first = 0;
        const int chunks = d / 8;
        if (!PAIR && more) have_q(&bar.start);
        for (; more; more = next_item(), ++nth) {
            const int n = ub - ua, mine = PAIR ? n : (n + 1 - s) / 2;
            // ---- this slot's rows of Q
            if (PAIR) {
                uint8_t *q_tile = smem + S::kQ + s * S::kPlace;
                const int r0 = tile * kRows + s * kWideTile, n_rows = len.rows * a.group;
                uint4 v[D / 8];
#pragma unroll
                for (int k = 0; k < D / 8; ++k) {
                    const int r = (k * kWideTile + row) / (D / 8), c = row % (D / 8), q_row = r0 + r;
                    v[k] = make_uint4(0, 0, 0, 0);
                    if (q_row < n_rows && c < chunks)
                        v[k] = *reinterpret_cast<const uint4 *>(a.q + 2 * (((int64_t)seq * a.rows + q_row / a.group) * a.q_stride + (int64_t)(head * a.group + q_row % a.group) * d + 8 * c));
                }
#pragma unroll
                for (int k = 0; k < D / 8; ++k) {
                    const int r = (k * kWideTile + row) / (D / 8), c = row % (D / 8);
                    *reinterpret_cast<uint4 *>(q_tile + (c >> 3) * S::kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[k];
                }
                fence_proxy_async();
            }
            uint32_t zero[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) zero[e] = 0;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) tm_st32(t_o + 32 * c, zero);
            tm_st_wait();
            if (PAIR) mbar_arrive(&bar.q[s]);
            const int q_row = tile * kRows + (PAIR ? s * kWideTile : 0) + row, i = q_row / a.group;
            float top = -INFINITY, sum = 0.f;  // top: what the weights are relative to, in scores as they come

            for (int job = 0; job < mine; ++job) {
                const int step = PAIR ? job : 2 * job + s, key0 = (ua + step) * kWideTile;
                const bool masked = key0 + kWideTile > (len.rows ? len.context : 0);
                uint32_t seen[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) seen[c] = view32(a, seq, i, key0 + 32 * c - len.context, len.rows);
                }
                wait(kScores + 8 * s, s_phase, kStatusMmaTimeout);
                s_phase ^= 1;
                tc_after();
                const uint64_t scale2 = twice(a.scale);
                uint64_t sums[2] = {0, 0};
                auto most = [&](float m, const uint32_t (&z)[32]) {
                    float n = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        m = fmaxf(fmaxf(m, __uint_as_float(z[e])), __uint_as_float(z[e + 1]));
                        n = fmaxf(fmaxf(n, __uint_as_float(z[e + 2])), __uint_as_float(z[e + 3]));
                    }
                    return fmaxf(m, n);
                };
                uint32_t za[32], zb[32];
                bool done = false;
                if (!masked && !__any_sync(0xffffffffu, top == -INFINITY)) {
                    // Four chunks of 32 scores, the next one on its way while one is worked on.  The weights are taken relative to the maximum of earlier tiles
                    // and stay in registers until it is clear that this tile's is no more than 2^8 above it.
                    uint32_t p[64];
                    const uint64_t off2 = twice(kUp<BF16, kRise> - top * a.scale);
                    float m = -INFINITY;
                    tm_ld32(t_s, za);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t(&z)[32] = c & 1 ? zb : za;
                        tm_ld_wait(z);
                        if (c < 3) tm_ld32(t_s + 32 * (c + 1), c & 1 ? za : zb);
                        m = most(m, z);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const uint64_t y = fma2(pair64(z[e], z[e + 1]), scale2, off2);
                            float lo, hi;
                            unpair64(y, lo, hi);
                            lo = ex2(lo);
                            hi = ex2(hi);
                            sums[e >> 1 & 1] = add2(sums[e >> 1 & 1], pair64(__float_as_uint(lo), __float_as_uint(hi)));
                            p[16 * c + (e >> 1)] = pack2<BF16>(lo, hi);
                        }
                    }
                    if (!__any_sync(0xffffffffu, (m - top) * a.scale > kRise)) {
                        tm_st32(t_s, *reinterpret_cast<uint32_t(*)[32]>(p));
                        tm_st32(t_s + 32, *reinterpret_cast<uint32_t(*)[32]>(p + 32));
                        done = true;
                    }
                }
                if (!done) {
                    // The first tile of an item, one with a new maximum, or with keys that not every row sees: maximum first.  Small code, as the instruction
                    // cache has not seen it for a while.
                    auto hide = [&](int c) {
                        const uint32_t view = c == 0 ? seen[0] : c == 1 ? seen[1] : c == 2 ? seen[2] : seen[3];
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(view >> e & 1)) za[e] = 0xff800000u;
                    };
                    float m = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        tm_ld32(t_s + 32 * c, za);
                        tm_ld_wait(za);
                        hide(c);
                        m = most(m, za);
                    }
                    const bool rise = top == -INFINITY ? m > top : (m - top) * a.scale > kRise;
                    const float down = rise && top != -INFINITY ? ex2((top - m) * a.scale) : 1.f;
                    if (__any_sync(0xffffffffu, down != 1.f)) {
                        if (job) wait(kSums + 8 * s, (n_sums - 1) & 1, kStatusMmaTimeout);
                        tc_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            tm_ld32(t_o + 32 * c, za);
                            tm_ld_wait(za);
#pragma unroll
                            for (int e = 0; e < 32; ++e) za[e] = __float_as_uint(__uint_as_float(za[e]) * down);
                            tm_st32(t_o + 32 * c, za);
                        }
                        sum *= down;
                    }
                    if (rise) top = m;
                    const uint64_t off2 = twice(top == -INFINITY ? 0.f : kUp<BF16, kRise> - top * a.scale);
                    sums[0] = sums[1] = 0;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        tm_ld32(t_s + 32 * c, za);
                        tm_ld_wait(za);
                        hide(c);
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float lo, hi;
                            unpair64(fma2(pair64(za[e], za[e + 1]), scale2, off2), lo, hi);
                            lo = ex2(lo);
                            hi = ex2(hi);
                            sums[e >> 1 & 1] = add2(sums[e >> 1 & 1], pair64(__float_as_uint(lo), __float_as_uint(hi)));
                            p[e >> 1] = pack2<BF16>(lo, hi);
                        }
                        tm_st16(t_s + 16 * c, p);  // over scores that are read already
                    }
                }
                tm_st_wait();
                {
                    float lo, hi;
                    unpair64(add2(sums[0], sums[1]), lo, hi);
                    sum += lo + hi;
                }

                if (masked) {
                    // clear what nobody may meet in V; slot 0 does it for both where they share the keys
                    const uint32_t v_tile = first + 2 * step + 1;
                    uint8_t *v = smem + S::kRingAt + v_tile % S::kRing * S::kTileBytes;
                    if (!PAIR || s == 0) {
                        wait(kFull + 8 * (v_tile % S::kRing), v_tile / S::kRing & 1, kStatusTmaTimeout);
                        bool dropped = false;
                        const int key = key0 + row;
                        if (key >= (len.rows ? len.context : 0)) {
#pragma unroll 1
                            for (int c = 0; c < D / 8; ++c) {
                                uint4 *w = reinterpret_cast<uint4 *>(v + (c >> 3) * S::kBlock + row * 128 + (((c & 7) ^ (row & 7)) << 4));
                                uint4 y = *w;
                                if (key >= keys) {
                                    *w = make_uint4(0, 0, 0, 0);
                                } else {
                                    bool some = drop_nonfinite<BF16>(y.x);
                                    some |= drop_nonfinite<BF16>(y.y);
                                    some |= drop_nonfinite<BF16>(y.z);
                                    some |= drop_nonfinite<BF16>(y.w);
                                    if (some) *w = y;
                                    dropped |= some;
                                }
                            }
                            fence_proxy_async();
                        }
                        const uint32_t rows = __ballot_sync(0xffffffffu, dropped);
                        if (lane == 0) bar.poison[s][warp & 3] = rows;
                    }
                    asm volatile("bar.sync %0, %1;" ::"r"(PAIR ? 1 : 2 + s), "n"(PAIR ? 2 * kWideTile : kWideTile) : "memory");
                    // the rows that see such a value have it in their sums
                    uint32_t poison[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) poison[c] = bar.poison[PAIR ? 0 : s][c];
                    if (poison[0] | poison[1] | poison[2] | poison[3]) {
                        if (job) wait(kSums + 8 * s, (n_sums - 1) & 1, kStatusMmaTimeout);
                        tc_after();
                        for (int r = 0; r < kWideTile; ++r) {
                            const uint32_t bad = r < 32 ? poison[0] : r < 64 ? poison[1] : r < 96 ? poison[2] : poison[3], view = r < 32 ? seen[0] : r < 64 ? seen[1] : r < 96 ? seen[2] : seen[3];
                            if (!(bad >> (r & 31) & 1)) continue;
                            const bool mine_too = view >> (r & 31) & 1;
                            const int64_t at = cache_row(a.c, seq, key0 + r);
                            if (at < 0) continue;
                            const uint16_t *from = reinterpret_cast<const uint16_t *>(a.c.v) + at + (int64_t)head * d;
#pragma unroll 1
                            for (int c = 0; c < (d + 31) / 32; ++c) {
                                uint32_t x[32];
                                tm_ld32(t_o + 32 * c, x);
                                tm_ld_wait(x);
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    if (32 * c + e < d && mine_too) {
                                        const float y = unpack16<BF16>(from[32 * c + e]);
                                        if (!isfinite(y)) x[e] = __float_as_uint(__uint_as_float(x[e]) + y);
                                    }
                                }
                                tm_st32(t_o + 32 * c, x);
                            }
                            tm_st_wait();  // the next such row of V loads what this one has stored
                        }
                    }
                    asm volatile("bar.sync %0, %1;" ::"r"(PAIR ? 1 : 2 + s), "n"(PAIR ? 2 * kWideTile : kWideTile) : "memory");
                }
                tc_before();
                mbar_arrive(&bar.weights[s]);
                ++n_sums;
            }
            if (mine) wait(kSums + 8 * s, (n_sums - 1) & 1, kStatusMmaTimeout);
            tc_after();
            first += 2 * n;

            // ---- the item's sums
            const bool whole = ua == 0 && ub == units;
            float *part = a.parts + ((size_t)blockIdx.x * 2 + (ua == 0 ? 1 : 0)) * (size_t)(kRows * (D + 2));
            const int part_row = PAIR ? s * kWideTile + row : row;
            // first value of this thread's row in the output or in the part
            const int64_t to = i >= a.rows ? -1 : whole ? (((int64_t)seq * a.rows + i) * a.c.heads * a.group + head * a.group + q_row % a.group) * d : (int64_t)part_row * D;
            // The sums leave by way of the place of Q, which is through ([128][D / 2] f32, chunks of 16 bytes swizzled), whole lines at a time: 32 columns of the
            // warp's 32 rows.  Loops, not straight code: it runs once per item, at the pace of instruction fetches.
            auto chunk_at = [&](uint8_t *region, int r, int c) { return region + r * (PAIR ? 2 * D : 128) + ((c ^ (r & 7)) << 4); };
            auto put = [&](uint8_t *region, int c0, int col) {
                __syncwarp();
#pragma unroll 2
                for (int k = 0; k < 8; ++k) {
                    const int r = 4 * k + (lane >> 3), c = lane & 7;
                    const int64_t at = __shfl_sync(0xffffffffu, to, r);
                    const float4 v = *reinterpret_cast<const float4 *>(chunk_at(region, (row & ~31) + r, c0 + c));
                    if (at < 0) continue;
                    if (!whole) *reinterpret_cast<float4 *>(part + at + col + 4 * c) = v;
                    else if (col + 4 * c < d) *reinterpret_cast<uint2 *>(a.out + 2 * (at + col + 4 * c)) = make_uint2(pack2<BF16>(v.x, v.y), pack2<BF16>(v.z, v.w));
                }
                __syncwarp();
            };
            // A slot that saw no score but NaN has no largest one and a sum of NaN: it must not be taken for a slot that saw nothing.
            float log_top = top == -INFINITY ? (PAIR || sum == 0.f ? -INFINITY : NAN) : top * a.scale;
            uint8_t *stage = smem + S::kQ + (PAIR ? s * S::kPlace : (nth & 1) * S::kPlace + s * (S::kPlace / 2));
            uint32_t x[32];
            if (PAIR) {
                const bool none = whole && (sum == 0.f || i >= len.rows);
                const float inv = !whole ? 1.f : none ? 0.f : 1.f / sum;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    tm_ld32(t_o + 32 * c, x);
                    tm_ld_wait(x);
                    const int c0 = (8 * c) % (D / 8);
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4 *>(chunk_at(stage, row, c0 + e / 4)) = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(__uint_as_float(x[e]) * inv, __uint_as_float(x[e + 1]) * inv, __uint_as_float(x[e + 2]) * inv, __uint_as_float(x[e + 3]) * inv);
                    put(stage, c0, 32 * c);
                }
            } else {
                // each slot finishes half of the columns: it hands the other half of its sums over, relative to both slots' maximum
                bar.top[s][row] = log_top;
                bar.sum[s][row] = sum;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float other = bar.top[1 - s][row], both = fmaxf(log_top, other), scale = log_top == -INFINITY ? 0.f : ex2(log_top - both);
                sum = (scale == 0.f ? 0.f : sum * scale) + (other == -INFINITY ? 0.f : bar.sum[1 - s][row] * ex2(other - both));
                log_top = both;
                const bool none = whole && (sum == 0.f || i >= len.rows);
                const float inv = !whole ? 1.f : none ? 0.f : 1.f / sum;
                uint8_t *from = smem + S::kQ + (nth & 1) * S::kPlace + (1 - s) * (S::kPlace / 2);
#pragma unroll 1
                for (int c = 0; c < D / 64; ++c) {
                    tm_ld32(t_o + (1 - s) * (D / 2) + 32 * c, x);
                    tm_ld_wait(x);
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4 *>(chunk_at(stage, row, e / 4)) = scale == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(__uint_as_float(x[e]) * scale, __uint_as_float(x[e + 1]) * scale, __uint_as_float(x[e + 2]) * scale, __uint_as_float(x[e + 3]) * scale);
                    tm_ld32(t_o + s * (D / 2) + 32 * c, x);
                    tm_ld_wait(x);
                    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4 *at = reinterpret_cast<float4 *>(chunk_at(from, row, e / 4));
                        float4 v = *at;
                        if (scale != 0.f) {
                            v.x += __uint_as_float(x[e]) * scale;
                            v.y += __uint_as_float(x[e + 1]) * scale;
                            v.z += __uint_as_float(x[e + 2]) * scale;
                            v.w += __uint_as_float(x[e + 3]) * scale;
                        }
                        *at = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                    }
                    put(from, 0, s * (D / 2) + 32 * c);
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                }
                mbar_arrive(&bar.left[nth & 1]);
            }
            if (!whole && (PAIR || s == 0)) {
                part[kRows * D + part_row] = log_top;
                part[kRows * D + kRows + part_row] = sum;
            }
            if (PAIR) asm volatile("bar.sync %0, %1;" ::"r"(2 + s), "n"(kWideTile) : "memory");  // the next item's rows of Q go where these sums were
            if (tid == 0 && ua == 0 && ub < units) {
                const int64_t end = item_first + units;
                a.info[blockIdx.x] = make_int4(seq, item, (int)((end * share.ctas - 1) / share.total) - (int)blockIdx.x + 1, len.rows);
            }
        }
        tc_before();
    }
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

static int page_map(const zq_kv_cache *c, void *data, int box_rows, CUtensorMap *out, zq_error *err) {
    EncodeTiledFn encode = get_encode_tiled(err);
    if (!encode) return ZQ_ERR_CUDA;
    const cuuint64_t dims[4] = {c->head_dim, c->heads, c->page_size, c->pages};
    const cuuint64_t strides[3] = {c->head_dim * 2, c->heads * c->head_dim * 2, c->page_stride * 2};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)box_rows, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(out, c->dtype == ZQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(err, ZQ_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d (cache of %zu pages of %zu x %zu x %zu)", (int)r, c->pages, c->page_size, c->heads, c->head_dim);
    return ZQ_OK;
}

template <int D, bool BF16, bool PAIR> static int launch_wide(zq_ctx *ctx, AttnArgs &a, const zq_kv_cache *cache, zq_error *err) {
    constexpr int kRows = PAIR ? 2 * kWideTile : kWideTile;
    CUtensorMap map_k, map_v;
    const int box_rows = cache->page_size < kWideTile ? (int)cache->page_size : kWideTile;
    int rc = page_map(cache, cache->dev_k, box_rows, &map_k, err);
    if (rc || (rc = page_map(cache, cache->dev_v, box_rows, &map_v, err))) return rc;
    a.tiles = (a.rows * a.group + kRows - 1) / kRows;
    const size_t ctas = (size_t)ctx->sm_count, bytes = ctas * 2 * kRows * (D + 2) * sizeof(float);
    LaunchScratch scratch;
    if ((rc = scratch.take(ctx, bytes + ctas * sizeof(int4), err))) return rc;
    a.parts = static_cast<float *>(scratch.p);
    a.info = reinterpret_cast<int4 *>(static_cast<uint8_t *>(scratch.p) + bytes);
    ZQ_CUDA_CHECK(cudaFuncSetAttribute(wide_attention_kernel<D, BF16, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, WideShape<D>::kSmem), err);
    rc = launch_pdl(ctx, wide_attention_kernel<D, BF16, PAIR>, dim3((unsigned)ctas), dim3(kWideThreads), WideShape<D>::kSmem, err, a, map_k, map_v);
    if (rc) return rc;
    return launch_attention_join(ctx, a, BF16, (int)ctas, kRows, D, err);
}

// From 33 rows on.  With 24 rows of heads of 128 the kernel of zq_attn.cu takes 14.2 / 26.4 / 45.5 us for one sequence at 200, eight at 4000 and sixteen at 8000
// positions of four cache heads, this one 15.5 / 22.0 / 44.4; with 40 rows 19.5 / 38.6 / 65.2 and 15.7 / 23.1 / 45.2 (pages of 64; of 8, where a copy is a
// short box: 14.1 / 28.4 / 50.4 and 17.1 / 32.2 / 74.3 for 24 rows, 19.5 / 40.3 / 80.3 and 17.3 / 31.0 / 74.8 for 40).
int launch_attention_wide(zq_ctx *ctx, AttnArgs &a, const zq_kv_cache *cache, bool &taken, zq_error *err) {
    const int rows = a.rows * a.group, d = a.c.head_dim;
    taken = rows > 32 && d >= 64 && d <= 128 && cache->page_size >= 8 && ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 && a.q_stride % 8 == 0;
    if (!taken) return ZQ_OK;
    const bool bf16 = cache->dtype == ZQ_BF16, pair = rows > kWideTile;
    if (d == 64) return bf16 ? (pair ? launch_wide<64, true, true>(ctx, a, cache, err) : launch_wide<64, true, false>(ctx, a, cache, err)) : pair ? launch_wide<64, false, true>(ctx, a, cache, err) : launch_wide<64, false, false>(ctx, a, cache, err);
    return bf16 ? (pair ? launch_wide<128, true, true>(ctx, a, cache, err) : launch_wide<128, true, false>(ctx, a, cache, err)) : pair ? launch_wide<128, false, true>(ctx, a, cache, err) : launch_wide<128, false, false>(ctx, a, cache, err);
}

}  // namespace zq
