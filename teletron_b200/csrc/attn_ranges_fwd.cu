// Softmax attention in which every query sees one run of the keys, forward, on tcgen05 / TMEM: heads of 64 and 128, bf16 and fp16, key
// heads shared by groups of query heads, scores capped by a tanh, a bias that depends on the distance.
//
//   s = scale q . k;   s = cap tanh(s / cap);   s += bias[h, clamp(key position - query position, -R, R) + R]
//   out = softmax over the query's run of keys (s) v;   0 where the run is empty
//
// One CTA owns two tiles of 128 queries that ping-pong through the tensor core and share the loaded keys and values: the same queries of two heads of
// a group where groups are even (both tiles then have the same runs, and keys and values are read once for both), else two neighbouring tiles of one
// head.  TMEM columns [0, 256): scores of both tiles, overwritten in place by P; from 256 on: both outputs.  Warp 0 loads (and clears values that no
// query sees), warp 1 issues every product, warps 2-5 and 6-9 are the softmax of the tiles, one query per thread.  A CTA goes on with items of the
// grid that have not been launched, each role at its own pace, so that the loads and first products of one item run behind the softmax and output of
// the one before.  Tiles of keys that no query of a tile sees are not touched; whole tiles are not masked; between them a warp masks by the bits of
// its rows' runs.
//
// What bounds it is the chain of a tile (scores, softmax, P V), of which two ping-pong.  Measured (bf16, heads of 128): five clips packed into 32656
// tokens x 24 heads 2.2 - 2.3 ms (1.12 - 1.18 PFLOP/s of the visible pairs); 2 x 4095 tokens x 32 heads, causal behind a prefix, capped 355 - 385 us
// (0.73 - 0.79).  With few tiles a CTA latencies count: 8 prompts of 256 tokens 21.5 us; 4 x 512 tokens x 64 heads of 64 with a bias that is trained
// 74 us, of which the output in both types is a sixth.
#include <limits.h>

#include "attn_ranges.cuh"

namespace {

using namespace sm100;
using namespace ranges;

constexpr int kThreads = 320;
constexpr int kSlab = kTile * 128;          // [128 rows x 64 elements], 128-byte swizzle
constexpr float kRescaleThreshold = 8.0f;   // log2 units by which the running maximum may lag behind

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

struct FwdParams {
    PlanPtr plan;
    Order order;
    void* out;
    float *out32, *lse;
    const float* bias;
    int q_len, q_heads, group, pair_heads, R;
    float scale_log2;
    Cap cap;
    int* status;
};

template <int D> struct Layout {
    static constexpr int kSlabs = D / 64;
    static constexpr int kTileBytes = kSlabs * kSlab;
    static constexpr int kStages = D == 64 ? 4 : 2;         // of keys and of values each
    static constexpr int kBars = 2 + 5 * kStages + 2 + 4 + 2 + 2;
    static constexpr int kFixed = (2 + 2 * kStages) * kTileBytes + 8 * 2048 + (kBars + 1) / 2 * 16 + Queue::kBytes + 16;      // 16: abort flag, tensor memory's address
    // dynamic shared memory is declared to start at a 1024-byte boundary, and there is no static one ahead of it
    static constexpr int smem(int R) { return kFixed + (R >= 0 ? 2 * (2 * R + 1 + 2 * kPad) * 4 : 0); }
};
static_assert(Layout<128>::smem(TT_RANGES_MAX_DISTANCE) <= 232448, "shared memory of an SM");

enum { kPlain = 0, kGeneral = 1, kGeneralWide = 2 };

// kGeneral: scores are scaled (by any factor), capped and biased ahead of the softmax; kPlain: the positive scale is part of its exponent.
// kGeneralWide, for a bias that is trained and for trained calls of few keys, also writes the output before rounding, to 2^-16 instead of P's 2^-8: P is split into two 16-bit
// parts (the second one takes the 64 columns that the scores leave free) and multiplied twice.  The bias's gradient sums P (dP - delta)
// over whole diagonals in 32 bits; with delta from a product with rounded P it was good to 1e-3 only.
template <int D, bool BF16, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
ranges_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const FwdParams p) {
    using L = Layout<D>;
    constexpr bool GEN = MODE != kPlain, WIDE = MODE == kGeneralWide;
    constexpr int kStages = L::kStages, kTileBytes = L::kTileBytes;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem_raw + L::kFixed - 16);
    uint32_t& tmem_base_slot = *reinterpret_cast<uint32_t*>(smem_raw + L::kFixed - 8);

    const uint32_t base = smem_u32(smem_raw);
    if (base & 1023u) {                 // the swizzled tiles would be read wrongly
        if (threadIdx.x == 0) atomicExch(p.status, TT_ERR_ARG);
        return;
    }
    const uint32_t sQ = base, sK = base + 2 * kTileBytes, sV = sK + kStages * kTileBytes, stages = sV + kStages * kTileBytes, bars = stages + 8 * 2048;
    const uint32_t queue_base = bars + (L::kBars + 1) / 2 * 16;
    float* table = reinterpret_cast<float*>(smem_raw + L::kFixed);
    const uint32_t q_full = bars, q_empty = bars + 8u;
    auto k_full = [&](int s) { return bars + 8u * (2 + s); };
    auto k_empty = [&](int s) { return bars + 8u * (2 + kStages + s); };
    auto v_full = [&](int s) { return bars + 8u * (2 + 2 * kStages + s); };
    auto v_empty = [&](int s) { return bars + 8u * (2 + 3 * kStages + s); };
    auto v_clean = [&](int s) { return bars + 8u * (2 + 4 * kStages + s); };
    auto s_full = [&](int t) { return bars + 8u * (2 + 5 * kStages + t); };
    auto p_half = [&](int t, int h) { return bars + 8u * (4 + 5 * kStages + 2 * t + h); };       // keys [64 h, 64 h + 64) of P are in place
    auto o_final = [&](int t) { return bars + 8u * (8 + 5 * kStages + t); };
    auto table_ready = [&](int t) { return bars + 8u * (10 + 5 * kStages + t); };
    Queue queue{queue_base};

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // An item: tile t is queries [128 qt[t], 128 qt[t] + 128) of head h[t] and sees some of the tiles of keys [a[t].x, a[t].y).  The long runs of
    // causal masks are at the end of the sequence: first.
    struct Item {
        int b, qt[2], h[2], kv_head, lo, hi;
        int2 a[2];
    };
    auto item_at = [&](int bx, int by, int bz) {
        Item w;
        w.b = p.order.sample(bx, by, bz);
        const int x = p.order.tiles() - 1 - p.order.tile(bx, by, bz), head = p.order.head(bx, by, bz);
        w.qt[0] = p.pair_heads ? x : 2 * x;
        w.qt[1] = p.pair_heads ? x : 2 * x + 1;
        w.h[0] = p.pair_heads ? 2 * head : head;
        w.h[1] = p.pair_heads ? w.h[0] + 1 : w.h[0];
        w.kv_head = w.h[0] / p.group;
        const PlanView plan = p.plan.sample(w.b);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            w.a[t] = make_int2(0, 0);
            if (w.qt[t] < p.plan.q_tiles) {
                const int4 r = plan.q_tiles[w.qt[t]];
                if (r.x < r.y) w.a[t] = make_int2(r.x / kTile, (r.y + kTile - 1) / kTile);
            }
        }
        const bool some0 = w.a[0].x < w.a[0].y, some1 = w.a[1].x < w.a[1].y;
        w.lo = some0 ? (some1 ? min(w.a[0].x, w.a[1].x) : w.a[0].x) : w.a[1].x;
        w.hi = max(w.a[0].y, w.a[1].y);
        return w;
    };
    auto active = [](const Item& w, int t, int j) { return j >= w.a[t].x && j < w.a[t].y; };
    int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(k_full(s), 1);
            mbar_init(k_empty(s), 1);
            mbar_init(v_full(s), 1);
            mbar_init(v_empty(s), 1);
            mbar_init(v_clean(s), 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(s_full(t), 1);
            mbar_init(p_half(t, 0), 4);
            mbar_init(p_half(t, 1), 4);
            mbar_init(o_final(t), 1);
            mbar_init(table_ready(t), 4);
        }
        queue.init(2 + 8);
        fence_barrier_init();
        fence_proxy_async();
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_slot;

    if (warp == 0) {
        // ------------------------------------------------------------ loads
        const bool lead = elect_one();
        int i = 0, n_some = 0;              // tiles of keys, and items that have any, so far
        do {
            const Item w = item_at(bx, by, bz);
            const PlanView plan = p.plan.sample(w.b);
            if (w.lo < w.hi) {
                if (!warp_wait(q_empty, (uint32_t)n_some & 1u ^ 1u, &abort_flag)) goto done;
                if (lead) {
                    mbar_arrive_expect_tx(q_full, 2 * kTileBytes);
#pragma unroll
                    for (int s = 0; s < L::kSlabs; ++s) {
                        tma_load_4d(sQ + s * kSlab, &tmQ, q_full, s * 64, w.qt[0] * kTile, w.h[0], w.b);
                        tma_load_4d(sQ + kTileBytes + s * kSlab, &tmQ, q_full, s * 64, w.qt[1] * kTile, w.h[1], w.b);
                    }
                }
                ++n_some;
            }
            int dirty = w.lo < w.hi ? plan.dirty[w.lo] : 0;
            for (int j = w.lo; j < w.hi; ++j, ++i) {
                const int s = i % kStages;
                const uint32_t ph = (uint32_t)(i / kStages) & 1u;
                const int dirty_next = j + 1 < w.hi ? plan.dirty[j + 1] : 0;
                if (!warp_wait(k_empty(s), ph ^ 1u, &abort_flag)) goto done;
                if (lead) {
                    mbar_arrive_expect_tx(k_full(s), kTileBytes);
#pragma unroll
                    for (int h = 0; h < L::kSlabs; ++h) tma_load_4d(sK + s * kTileBytes + h * kSlab, &tmK, k_full(s), h * 64, j * kTile, w.kv_head, w.b);
                }
                if (!warp_wait(v_empty(s), ph ^ 1u, &abort_flag)) goto done;
                if (lead) {
                    mbar_arrive_expect_tx(v_full(s), kTileBytes);
#pragma unroll
                    for (int h = 0; h < L::kSlabs; ++h) tma_load_4d(sV + s * kTileBytes + h * kSlab, &tmV, v_full(s), h * 64, j * kTile, w.kv_head, w.b);
                }
                __syncwarp();
                if (dirty) {        // 0 times a NaN is a NaN: values that no query sees become 0
                    if (!warp_wait(v_full(s), ph, &abort_flag)) goto done;
                    clear_rows(sV + s * kTileBytes, L::kSlabs, plan.dead[j], lane);
                    fence_proxy_async();
                    __syncwarp();
                    if (lead) mbar_arrive(v_clean(s));
                }
                dirty = dirty_next;
            }
            if (!queue.ask(lead, &abort_flag)) goto done;
            if (!warp_wait(queue.full(), queue.parity(), &abort_flag)) goto done;
            __syncwarp();
        } while (queue.next<true>(lead, &bx, &by, &bz));
    } else if (warp == 1) {
        // ------------------------------------------------------------ products
        if (elect_one()) {
            constexpr uint32_t idesc_s = idesc<BF16>(kTile, kTile, false, false);     // S = Q K^T: both K-major
            constexpr uint32_t idesc_o = idesc<BF16>(kTile, D, false, true);          // O += P V: V is MN-major
            auto issue_s = [&](int t, int stage) {
                const uint64_t a = fresh_desc(smem_desc_sw128(sQ + t * kTileBytes, 16, 1024));
                const uint64_t k = fresh_desc(smem_desc_sw128(sK + stage * kTileBytes, 16, 1024));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint64_t off = (uint64_t)(((kk >> 2) * kSlab + (kk & 3) * 32) >> 4);
                    umma_bf16_ss(tmem + t * 128, a + off, k + off, idesc_s, kk ? 1u : 0u);
                }
                umma_commit(s_full(t));
            };
            auto issue_o = [&](int t, int stage, int half, bool accumulate) {
                const uint64_t v = fresh_desc(smem_desc_sw128(sV + stage * kTileBytes, kSlab, 1024));
#pragma unroll
                for (int k4 = 0; k4 < kTile / 32; ++k4) {
                    const int kk = half * (kTile / 32) + k4;
                    umma_bf16_ts(tmem + 256 + t * D, tmem + t * 128 + kk * 8, v + (uint64_t)(kk * (2048 >> 4)), idesc_o, (accumulate || kk) ? 1u : 0u);
                    if (WIDE) umma_bf16_ts(tmem + 256 + t * D, tmem + t * 128 + 64 + kk * 8, v + (uint64_t)(kk * (2048 >> 4)), idesc_o, 1u);
                }
            };
            int i = 0, n_some = 0;              // tiles of keys, and items that have any, so far
            uint32_t n0 = 0, n1 = 0;            // tiles of keys that each tile of queries has been through
            uint32_t cleaned = 0;               // bit s: parity of the cleaned uses of stage s
            do {
                const Item w = item_at(bx, by, bz);
                const PlanView plan = p.plan.sample(w.b);
                int dirty = 0;
                bool first0 = true, first1 = true;
                if (w.lo < w.hi) {
                    dirty = plan.dirty[w.lo];
                    if (!mbar_wait(q_full, (uint32_t)n_some++ & 1u, &abort_flag)) goto done;
                    if (!mbar_wait(k_full(i % kStages), (uint32_t)(i / kStages) & 1u, &abort_flag)) goto done;
                    tc_fence_after();
                    if (active(w, 0, w.lo)) issue_s(0, i % kStages);
                    if (active(w, 1, w.lo)) issue_s(1, i % kStages);
                    umma_commit(k_empty(i % kStages));
                    if (w.lo + 1 == w.hi) umma_commit(q_empty);
                }
                for (int j = w.lo; j < w.hi; ++j, ++i) {
                    const int s = i % kStages, s1 = (i + 1) % kStages;
                    const uint32_t ph = (uint32_t)(i / kStages) & 1u, ph1 = (uint32_t)((i + 1) / kStages) & 1u;
                    const bool more = j + 1 < w.hi;
                    const int dirty_next = more ? plan.dirty[j + 1] : 0;
                    if (dirty) {
                        if (!mbar_wait(v_clean(s), cleaned >> s & 1u, &abort_flag)) goto done;
                        cleaned ^= 1u << s;
                    } else if (!mbar_wait(v_full(s), ph, &abort_flag)) {
                        goto done;
                    }
                    if (active(w, 0, j)) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (!mbar_wait(p_half(0, h), n0 & 1u, &abort_flag)) goto done;
                            tc_fence_after();
                            issue_o(0, s, h, !first0);
                        }
                        ++n0;
                        first0 = false;
                    }
                    if (more) {
                        if (!mbar_wait(k_full(s1), ph1, &abort_flag)) goto done;
                        tc_fence_after();
                        if (active(w, 0, j + 1)) issue_s(0, s1);
                    }
                    if (active(w, 1, j)) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (!mbar_wait(p_half(1, h), n1 & 1u, &abort_flag)) goto done;
                            tc_fence_after();
                            issue_o(1, s, h, !first1);
                        }
                        ++n1;
                        first1 = false;
                    }
                    umma_commit(v_empty(s));
                    if (more) {
                        if (active(w, 1, j + 1)) issue_s(1, s1);
                        umma_commit(k_empty(s1));
                        if (j + 2 == w.hi) umma_commit(q_empty);        // the item's last scores: the next one's queries may come
                    }
                    dirty = dirty_next;
                }
                // a tile's own barrier, and only where it has had a product: its warps then are never more than a phase behind
                if (!first0) umma_commit(o_final(0));
                if (!first1) umma_commit(o_final(1));
                if (!mbar_wait(queue.full(), queue.parity(), &abort_flag)) goto done;
            } while (queue.next<false>(true, &bx, &by, &bz));
        }
    } else {
        // ------------------------------------------------------------ softmax and output (one query per thread)
        const int t = (warp - 2) >> 2, quad = warp & 3;
        const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
        const uint32_t tS = tmem + lane_sel + t * 128, tO = tmem + lane_sel + 256 + t * D;
        const int table_size = 2 * p.R + 1 + 2 * kPad;
        float* const my_table = table + t * table_size;
        // what a thread needs of an item; the next one's is read ahead of this one's output
        struct Mine {
            int b, qt, head, start, first, behind;
            int2 a;
        };
        auto mine_of = [&](int x, int y, int z) {
            const Item w = item_at(x, y, z);
            const PlanView plan = p.plan.sample(w.b);
            Mine v;
            v.b = w.b;
            v.qt = t ? w.qt[1] : w.qt[0];
            v.head = t ? w.h[1] : w.h[0];
            v.a = t ? w.a[1] : w.a[0];
            v.start = plan.start;
            const int row = v.qt * kTile + quad * 32 + lane;
            // rows behind the last query see all and count for nothing
            v.first = row < p.q_len ? plan.first[row] : 0;
            v.behind = row < p.q_len ? plan.behind[row] : INT_MAX;
            return v;
        };
        Mine v = mine_of(bx, by, bz);
        int table_head = -1;
        uint32_t n = 0, n_final = 0, n_table = 0;           // tiles of keys, outputs and tables so far
        bool go = true;
        while (go) {
            const int row = v.qt * kTile + quad * 32 + lane;
            const bool real = row < p.q_len;
            const int first = v.first, behind = v.behind;
            const bool some = real && first < behind;
            const int w_first_all = __reduce_max_sync(0xffffffffu, some || !real ? first : INT_MAX);
            const int w_behind_all = __reduce_min_sync(0xffffffffu, behind);
            const int w_first_any = __reduce_min_sync(0xffffffffu, some ? first : INT_MAX);
            const int w_behind_any = __reduce_max_sync(0xffffffffu, some ? behind : 0);
            const int pos = row + v.start;
            if (GEN && p.R >= 0 && v.head != table_head) {
                // this head's table in the log2 domain, its ends repeated, once all four warps are through with the last one
                if (lane == 0) mbar_arrive(table_ready(t));
                if (!warp_wait(table_ready(t), n_table++ & 1u, &abort_flag)) goto done;
                for (int i = quad * 32 + lane; i < table_size; i += 128)
                    my_table[i] = p.bias[(long)v.head * (2 * p.R + 1) + min(max(i - kPad, 0), 2 * p.R)] * kLog2e;
                __syncwarp();
                if (lane == 0) mbar_arrive(table_ready(t));
                if (!warp_wait(table_ready(t), n_table++ & 1u, &abort_flag)) goto done;
                table_head = v.head;
            }
            float m = -INFINITY, l = 0.f;
            for (int j = v.a.x; j < v.a.y; ++j, ++n) {
                const int k0 = j * kTile;
                if (!warp_wait(s_full(t), n & 1u, &abort_flag)) goto done;
                tc_fence_after();
                if (w_behind_any <= k0 || w_first_any >= k0 + kTile) {          // no row of this warp sees any of these keys
                    uint32_t z[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] = 0u;
#pragma unroll
                    for (int c = 0; c < (WIDE ? 8 : 4); ++c) tmem_st_32x16(tS + c * 16, z);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(p_half(t, 0));
                        mbar_arrive(p_half(t, 1));
                    }
                    continue;
                }
                uint32_t r[kTile];
#pragma unroll
                for (int c = 0; c < kTile / 32; ++c) tmem_ld_32x32(tS + c * 32, r + c * 32);
                tmem_ld_wait();
                if (GEN) {
                    float factor = p.scale_log2;            // what is left of the scale
                    if (p.cap.out != 0.f) {
                        factor = 1.f;
                        if (all_small<kTile>(p.cap, r)) {
#pragma unroll
                            for (int i = 0; i < kTile; i += 2) {
                                const float2 y = cap_small(p.cap, make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
                                r[i] = __float_as_uint(y.x);
                                r[i + 1] = __float_as_uint(y.y);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < kTile; ++i) r[i] = __float_as_uint(cap_any(p.cap, __uint_as_float(r[i])));
                        }
                    }
                    const float2 f2 = make_float2(factor, factor);
                    const int pos0 = pos - lane;                        // of the warp's first row
                    if (p.R < 0 || k0 + kTile - 1 - pos0 <= -p.R || k0 - pos0 - 31 >= p.R) {       // no bias, or all at the table's end
                        const float far = p.R < 0 ? 0.f : my_table[kPad + p.R + (k0 - pos0 > 0 ? p.R : -p.R)];
                        if (p.R >= 0 || p.cap.out == 0.f) {
#pragma unroll
                            for (int i = 0; i < kTile; i += 2) {
                                const float2 y = __ffma2_rn(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2, make_float2(far, far));
                                r[i] = __float_as_uint(y.x);
                                r[i + 1] = __float_as_uint(y.y);
                            }
                        }
                    } else {
                        const uint32_t entry = smem_u32(my_table) + 4 * (kPad + p.R + k0 - pos);
#pragma unroll
                        for (int i = 0; i < kTile; i += 2) {
                            float2 add;
                            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(add.x) : "r"(entry + 4 * i));
                            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(add.y) : "r"(entry + 4 * i + 4));
                            const float2 y = __ffma2_rn(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2, add);
                            r[i] = __float_as_uint(y.x);
                            r[i + 1] = __float_as_uint(y.y);
                        }
                    }
                }
                if (w_first_all > k0 || w_behind_all < k0 + kTile) {
#pragma unroll
                    for (int c = 0; c < kTile / 32; ++c) {
                        const uint32_t see = bits_between(first - k0 - 32 * c, behind - k0 - 32 * c);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(see >> i & 1u)) r[c * 32 + i] = 0xff800000u;      // -inf
                    }
                }
                const float2 sc2 = GEN ? make_float2(1.f, 1.f) : make_float2(p.scale_log2, p.scale_log2);
                float2 sum2a = make_float2(0.f, 0.f), sum2b = make_float2(0.f, 0.f);
                auto exp_cols = [&](int c) {
                    const float nm = m == -INFINITY ? 0.f : -m;         // no key seen so far: the scores are -inf and P is 0
                    const float2 nm2 = make_float2(nm, nm);
                    uint32_t pk[16], rest[WIDE ? 16 : 1];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 s2 = make_float2(__uint_as_float(r[c * 32 + 2 * i]), __uint_as_float(r[c * 32 + 2 * i + 1]));
                        const float2 y = GEN ? __fadd2_rn(s2, nm2) : __ffma2_rn(s2, sc2, nm2);
                        const float2 e = make_float2(exp2f(y.x), exp2f(y.y));
                        if (i & 1) sum2b = __fadd2_rn(sum2b, e);
                        else sum2a = __fadd2_rn(sum2a, e);
                        // P is rounded to the operands' type: half a step of 2^-8 (2^-11 in fp16) of each weight, as any product with 16-bit operands needs
                        pk[i] = pack2<BF16>(e.x, e.y);
                        if (WIDE) {
                            const float2 hi = unpack2<BF16>(pk[i]);
                            rest[i] = pack2<BF16>(e.x - hi.x, e.y - hi.y);
                        }
                    }
                    tmem_st_32x16(tS + c * 16, pk);
                    if (WIDE) tmem_st_32x16(tS + 64 + c * 16, rest);
                };
                // The first 32 exponentials use the running maximum as it stands; where it grows past the threshold they are redone.
                exp_cols(0);
                float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
                for (int i = 0; i < kTile; i += 8) {
                    mx0 = max3(mx0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                    mx1 = max3(mx1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
                    mx2 = max3(mx2, __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
                    mx3 = max3(mx3, __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
                }
                const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * (GEN ? 1.f : p.scale_log2);
                const bool grow = mx > m + kRescaleThreshold;           // always for the first visible key (m = -inf)
                if (__any_sync(0xffffffffu, grow)) {
                    tmem_st_wait();         // the stores that are about to be repeated have landed: the second ones win
                    if (j > v.a.x) {
                        const float alpha = grow ? exp2f(m - mx) : 1.f;
                        l *= alpha;
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld_32x16(tO + c * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st_32x16(tO + c * 16, o);
                        }
                        tmem_st_wait();
                    }
                    if (grow) m = mx;
                    sum2a = sum2b = make_float2(0.f, 0.f);
                    exp_cols(0);
                }
                exp_cols(1);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half(t, 0));               // P V over the first 64 keys can start
                exp_cols(2);
                exp_cols(3);
                l += (sum2a.x + sum2a.y) + (sum2b.x + sum2b.y);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half(t, 1));
            }
            const Mine w = v;
            if (!warp_wait(queue.full(), queue.parity(), &abort_flag)) goto done;
            go = queue.next<true>(lane == 0, &bx, &by, &bz);
            if (go) v = mine_of(bx, by, bz);
            if (w.a.x < w.a.y && !warp_wait(o_final(t), n_final++ & 1u, &abort_flag)) goto done;
            tc_fence_after();
            const bool none = !some || l == 0.f;           // sees nothing, or nothing but scores of -inf
            const float inv = none ? 0.f : 1.f / l;
            const int row0 = row - lane;
            const long at = (((long)w.b * p.q_len + row0) * p.q_heads + w.head) * D, pitch = (long)p.q_heads * D;
            uint16_t* const out = reinterpret_cast<uint16_t*>(p.out) + at;
            const uint32_t stage = stages + (warp - 2) * 2048;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld_32x32(tO + c * 32, r);
                tmem_ld_wait();
                uint4 piece[4];
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = none ? 0u : __float_as_uint(__uint_as_float(r[i]) * inv);
                const float* o = reinterpret_cast<const float*>(r);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    piece[g] = make_uint4(pack2<BF16>(o[g * 8], o[g * 8 + 1]), pack2<BF16>(o[g * 8 + 2], o[g * 8 + 3]),
                                          pack2<BF16>(o[g * 8 + 4], o[g * 8 + 5]), pack2<BF16>(o[g * 8 + 6], o[g * 8 + 7]));
                store_rows64(stage, lane, piece, [&](int i) { return row0 + i < p.q_len ? out + i * pitch + c * 32 : nullptr; });
                if (WIDE) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int i = half * 16 + g * 4;
                            piece[g] = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
                        }
                        store_rows64(stage, lane, piece, [&](int i) { return row0 + i < p.q_len ? p.out32 + at + i * pitch + c * 32 + half * 16 : nullptr; });
                    }
                }
            }
            if (w.qt < p.plan.q_tiles)
                p.lse[((long)w.b * p.q_heads + w.head) * p.plan.q_tiles * kTile + row] = none ? INFINITY : m + log2f(l);
            tc_fence_before();          // ahead of the arrivals that let the next item's first P V overwrite the output
        }
    }

done:
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        if (threadIdx.x == 0) atomicExch(p.status, TT_ERR_TIMEOUT);
        for (int i = 0; i < 200; ++i) __nanosleep(1000);         // copies in flight land
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D, bool BF16, int MODE>
int launch(const tt_ranges_args& a, FwdParams p, int dev, cudaStream_t st) {
    CUtensorMap tq, tk, tv;
    int rc;
    if ((rc = tt_make_tmap_bhsd(&tq, a.q, a.batch, a.q_heads, a.q_len, D, a.q_stride, kTile)) != TT_OK) return rc;
    if ((rc = tt_make_tmap_bhsd(&tk, a.k, a.batch, a.k_heads, a.kv_len, D, a.k_stride, kTile)) != TT_OK) return rc;
    if ((rc = tt_make_tmap_bhsd(&tv, a.v, a.batch, a.k_heads, a.kv_len, D, a.v_stride, kTile)) != TT_OK) return rc;
    auto kern = ranges_fwd_kernel<D, BF16, MODE>;
    static bool configured[64] = {false};         // per device: the attribute belongs to the device's context
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::smem(MODE != kPlain ? TT_RANGES_MAX_DISTANCE : -1));
        if (e != cudaSuccess) return tt_record_cuda(e);
        configured[dev] = true;
    }
    const int tiles = p.plan.q_tiles;
    const int items = p.pair_heads ? tiles : (tiles + 1) / 2;
    p.order = make_order(a, items);
    kern<<<p.order.grid(items, p.pair_heads ? a.q_heads / 2 : a.q_heads, a.batch), kThreads, Layout<D>::smem(MODE != kPlain ? a.max_distance : -1), st>>>(tq, tk, tv, p);
    TT_CHECK_LAUNCH();
    return TT_OK;
}

template <int D, bool BF16>
int pick(const tt_ranges_args& a, const FwdParams& p, int mode, int dev, cudaStream_t st) {
    return mode == kPlain ? launch<D, BF16, kPlain>(a, p, dev, st)
           : mode == kGeneral ? launch<D, BF16, kGeneral>(a, p, dev, st) : launch<D, BF16, kGeneralWide>(a, p, dev, st);
}

}  // namespace

extern "C" int tt_attn_ranges_fwd(const tt_ranges_args* a, void* stream) {
    int rc = tt_ranges_check(a);
    if (rc != TT_OK) return rc;
    if (tt_ranges_few_rows(*a)) return tt_attn_ranges_few(*a, (cudaStream_t)stream);
    const int dev = tt_device().dev;
    FwdParams p;
    p.plan = plan_ptr(*a);
    p.out = a->out;
    p.out32 = a->out32;
    p.lse = a->lse;
    p.bias = a->bias;
    p.q_len = a->q_len;
    p.q_heads = a->q_heads;
    p.group = a->q_heads / a->k_heads;
    p.pair_heads = p.group % 2 == 0;
    p.R = a->max_distance;
    p.scale_log2 = a->scale * kLog2e;
    p.cap = make_cap(a->scale, a->softcap);
    p.status = a->status;
    cudaStream_t st = (cudaStream_t)stream;
    const bool gen = a->softcap > 0.f || a->max_distance >= 0 || !(a->scale > 0.f) || a->out32 != nullptr;
    const int mode = a->out32 != nullptr ? kGeneralWide : gen ? kGeneral : kPlain;
    if (a->head_dim == 128)
        return a->dtype == TT_BF16 ? pick<128, true>(*a, p, mode, dev, st) : pick<128, false>(*a, p, mode, dev, st);
    return a->dtype == TT_BF16 ? pick<64, true>(*a, p, mode, dev, st) : pick<64, false>(*a, p, mode, dev, st);
}
