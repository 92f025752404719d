// Backward of the attention in which every query sees one run of the keys (attn_ranges_fwd.cu has the formulas).
//
//   P = exp(s - lse),  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO O)
//   dbias[h, d] = sum of dS over the diagonals of distance d;   dS' = dS (1 - tanh^2) behind a cap
//   dQ = scale dS' K,  dK = scale dS'^T Q,  dV = P^T dO
//
// Two kernels without atomics, so that results do not depend on the order of anything: one keeps a tile of 128 keys and goes through the
// queries that see any of them, of all heads of the group (dK and dV accumulate in TMEM; shared key heads need no second sum), the other keeps a
// tile of 128 queries and goes through its keys (dQ in TMEM).  Seven products per pair of tiles instead of five.
//
// Both are one template: stationary operands A1, A2 (K, V or Q, dO) stay in shared memory, streamed operands B1, B2 (Q, dO or K, V) come through
// rings.  TMEM: T1 = A1 B1^T (scores), T2 = A2 B2^T (dP), accumulators from column 256.  The order of the products keeps both sides busy: with
// stationary keys P overwrites the scores and dV takes it while dS is formed over dP; with stationary queries the next chunk's scores and
// dP (in a second buffer) are formed behind this chunk's dS.  Warp
// 0 loads, warp 1 issues, sixteen warps turn T1, T2 into P and dS (a thread: one stationary row, 32 streamed ones).
//
// Measured (bf16, heads of 128), dK dV and dQ: five clips packed into 32656 tokens x 24 heads 4.4 - 4.7 and 2.9 - 3.0 ms (1.1 - 1.3 PFLOP/s of the
// products executed; the power cap holds long runs to 1.38); 2 x 4095 tokens x 32 heads, causal behind a prefix, capped 590 - 640 and 470 - 510 us; 4
// x 512 tokens x 64 heads of 64 with a bias 90 us, with its gradient 111, where every item has four chunks and its first loads, sums and output are
// half of it.  dK dV has a CTA for each tile of keys and key head, whatever the heads of a group: 1000 causal tokens of 8 heads on one key head are 8
// CTAs (116 us, on two key heads 62; dQ 15), 2000 222 and 115 (dQ 24).
//
// The bias's gradient: diagonals within the largest distance hold delta's rounding (P and dS in 32 bits, delta from an output good to 2^-16), relative 2.8e-7 -
// 5.3e-7 where 32-bit arithmetic throughout has 1.9e-7 - 3.7e-7; the two ends, corrected by their rows' sums, 5.2e-7 - 9.6e-7 against 8e-7 - 2.8e-6 (512 and
// 2000 tokens, heads of 64, distances up to 128 and 1024).
#include <limits.h>

#include <type_traits>

#include "attn_ranges.cuh"

namespace {

using namespace sm100;
using namespace ranges;

constexpr int kGroups = 4;                                  // warpgroups that share a chunk's columns
constexpr int kCols = kTile / kGroups;                      // streamed rows of one thread
constexpr int kThreads = 64 + kGroups * 128;
constexpr int kSlab = kTile * 128;
constexpr int kDiagPad = 256;                               // a tile that is not wholly beyond the largest distance reaches at most 254 past it

// scores: scaled; capped; with a bias and maybe a cap; the same for a bias that gets a gradient
enum { kPlain = 0, kCapped = 1, kGeneral = 2, kGeneralDbias = 3 };

struct BwdParams {
    PlanPtr plan;
    Order order;
    const float *lse, *delta, *bias;
    void *out1, *out2;                  // dQ / dV and dK
    long s1[3], s2[3];                  // their strides
    float* partials;
    int q_len, kv_len, q_heads, group, R;
    float scale, scale_log2;
    Cap cap;
    int* status;
};

template <int D, bool KVS, int MODE> struct Layout {
    static constexpr int kSlabs = D / 64;
    static constexpr int kTileBytes = kSlabs * kSlab;
    static constexpr int kRing1 = MODE == kGeneralDbias && D == 128 ? 2 : 3, kRing2 = D == 64 ? 3 : 2;
    static constexpr int kStats = KVS ? (kRing1 + kRing2) * kTile * 4 : 0;      // lse with every slot of Q, delta with every slot of dO
    static constexpr int kBars = 2 + 3 * kRing1 + 3 * kRing2 + 7;
    static constexpr int kStage = D == 64 ? 16 * 2048 : 0;      // rows on their way out (heads of 128 leave no room)
    // barriers, the queue, the abort flag and the tensor memory's address
    static constexpr int kFixed = (2 + kRing1 + kRing2) * kTileBytes + kStats + kStage + (kBars + 1) / 2 * 16 + Queue::kBytes + 16;
    // dynamic shared memory is declared to start at a 1024-byte boundary, and there is no static one ahead of it
    static constexpr int smem(int R) { return kFixed + (MODE == kGeneralDbias ? (2 * 16 * 64 + 2 * R + 1 + 2 * kDiagPad) * 4 : 0); }
};
static_assert(Layout<128, true, kPlain>::smem(0) <= 232448, "shared memory of an SM");

template <int D, bool BF16, bool KVS, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
ranges_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmDO, const BwdParams p) {
    using L = Layout<D, KVS, MODE>;
    constexpr int kTileBytes = L::kTileBytes, kRing1 = L::kRing1, kRing2 = L::kRing2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    volatile int& abort_flag = *reinterpret_cast<volatile int*>(smem_raw + L::kFixed - 16);
    uint32_t& tmem_base_slot = *reinterpret_cast<uint32_t*>(smem_raw + L::kFixed - 8);

    const uint32_t base = smem_u32(smem_raw);
    if (base & 1023u) {                 // the swizzled tiles would be read wrongly
        if (threadIdx.x == 0) atomicExch(p.status, TT_ERR_ARG);
        return;
    }
    const uint32_t sA1 = base, sA2 = base + kTileBytes;
    const uint32_t sRing1 = base + 2 * kTileBytes, sRing2 = sRing1 + kRing1 * kTileBytes;
    const uint32_t sLse = sRing2 + kRing2 * kTileBytes, sDelta = sLse + kRing1 * kTile * 4;     // KVS
    const uint32_t stages = sRing2 + kRing2 * kTileBytes + L::kStats, bars = stages + L::kStage;
    float* scratch = reinterpret_cast<float*>(smem_raw + L::kFixed);      // [2][16 warps][64]: diagonals of a warp's block
    float* diag = scratch + 2 * 16 * 64;                                                                // [2 R + 1 + 2 kDiagPad]
    const uint32_t a_full = bars, a_empty = bars + 8u;
    auto b1_full = [&](int s) { return bars + 8u * (2 + s); };
    auto b1_empty = [&](int s) { return bars + 8u * (2 + kRing1 + s); };
    auto b1_clean = [&](int s) { return bars + 8u * (2 + 2 * kRing1 + s); };
    auto b2_full = [&](int s) { return bars + 8u * (2 + 3 * kRing1 + s); };
    auto b2_empty = [&](int s) { return bars + 8u * (2 + 3 * kRing1 + kRing2 + s); };
    auto b2_clean = [&](int s) { return bars + 8u * (2 + 3 * kRing1 + 2 * kRing2 + s); };
    const uint32_t s_full = bars + 8u * (2 + 3 * kRing1 + 3 * kRing2);      // T1 holds this chunk's scores
    auto dp_full = [&](int c) { return s_full + 8u + (KVS ? 0u : 40u * (uint32_t)(c & 1)); };      // the chunk's dP is there (dQ: two buffers)
    const uint32_t p_ready = s_full + 16u;                     // every softmax warp has read the scores
    const uint32_t ds_ready = s_full + 24u;                    // P and dS have been written over dP
    const uint32_t acc_final = s_full + 32u;
    const uint32_t diag_ready = s_full + 40u;                  // every softmax warp has left its diagonals in the scratch

    Queue queue{bars + (L::kBars + 1) / 2 * 16};

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // An item: a stationary tile of 128 rows from r0 on and the streamed tiles [lo, hi), KVS for all heads of the group one after the other
    struct Item {
        int b, tile, head, kv_head, lo, per_head, chunks;       // head: the first one
    };
    auto item_at = [&](int bx, int by, int bz) {
        Item w;
        const int head = p.order.head(bx, by, bz);
        w.b = p.order.sample(bx, by, bz);
        w.tile = p.order.tile(bx, by, bz);
        if (!KVS) w.tile = p.order.tiles() - 1 - w.tile;
        w.head = KVS ? head * p.group : head;
        w.kv_head = KVS ? head : head / p.group;
        const PlanView plan = p.plan.sample(w.b);
        int hi = 0;
        w.lo = 0;
        if (KVS) {
            const int2 k = plan.k_tiles[w.tile];
            w.lo = k.x;
            hi = k.y;
        } else {
            const int4 r = plan.q_tiles[w.tile];
            if (r.x < r.y) {
                w.lo = r.x / kTile;
                hi = (r.y + kTile - 1) / kTile;
            }
        }
        w.per_head = max(hi - w.lo, 0);
        w.chunks = w.per_head * (KVS ? p.group : 1);
        return w;
    };
    struct Chunk {
        int head, t;
    };
    auto chunk_at = [&](const Item& w, int c) {
        if (!KVS) return Chunk{w.head, w.lo + c};
        const int g = c / w.per_head;
        return Chunk{w.head + g, w.lo + c - g * w.per_head};
    };
    auto lds4 = [](uint32_t at, float4& v) { asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at)); };
    auto slope_of = [&](float2 y) {         // of the cap, from capped scores in the log2 domain
        const float2 t = __fmul2_rn(y, make_float2(p.cap.inv_out, p.cap.inv_out));
        return __ffma2_rn(t, make_float2(-t.x, -t.y), make_float2(1.f, 1.f));
    };
    // a streamed tile with rows that no run reaches: queries that see nothing, keys that nothing sees
    auto is_dirty = [&](const Item& w, const PlanView& plan, int c) {
        return c < w.chunks ? (KVS ? plan.q_tiles[chunk_at(w, c).t].w == 0 : plan.dirty[w.lo + c] != 0) : false;
    };
    int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        mbar_init(a_full, 1);
        mbar_init(a_empty, 1);
        queue.init(2 + 4 * kGroups);
        for (int s = 0; s < kRing1; ++s) {
            mbar_init(b1_full(s), 1);
            mbar_init(b1_empty(s), 1);
            mbar_init(b1_clean(s), 1);
        }
        for (int s = 0; s < kRing2; ++s) {
            mbar_init(b2_full(s), 1);
            mbar_init(b2_empty(s), 1);
            mbar_init(b2_clean(s), 1);
        }
        mbar_init(s_full, 1);
        mbar_init(dp_full(0), 1);
        if (!KVS) mbar_init(dp_full(1), 1);
        mbar_init(p_ready, 4 * kGroups);
        mbar_init(ds_ready, 4 * kGroups);
        mbar_init(acc_final, 1);
        mbar_init(diag_ready, 4 * kGroups);
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), 512);
        tmem_relinquish();
    }
    if (MODE == kGeneralDbias)
        for (int i = threadIdx.x; i < 2 * p.R + 1 + 2 * kDiagPad; i += kThreads) diag[i] = 0.f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_slot;
    constexpr uint32_t kT1 = 0, kT2 = 128, kAcc1 = 256, kAcc2 = 256 + D, kT3 = 384;       // kT3: the second dP of the dQ kernel, which has no kAcc2

    if (warp == 0) {
        // ------------------------------------------------------------ loads
        const bool lead = elect_one();
        int i = 0, n_some = 0;              // chunks, and items that have any, so far
        do {
            const Item w = item_at(bx, by, bz);
            const PlanView plan = p.plan.sample(w.b);
            if (w.chunks > 0) {
                if (!warp_wait(a_empty, (uint32_t)n_some & 1u ^ 1u, &abort_flag)) goto done;
                if (lead) {
                    mbar_arrive_expect_tx(a_full, 2 * kTileBytes);
#pragma unroll
                    for (int h = 0; h < L::kSlabs; ++h) {
                        tma_load_4d(sA1 + h * kSlab, KVS ? &tmK : &tmQ, a_full, h * 64, w.tile * kTile, KVS ? w.kv_head : w.head, w.b);
                        tma_load_4d(sA2 + h * kSlab, KVS ? &tmV : &tmDO, a_full, h * 64, w.tile * kTile, KVS ? w.kv_head : w.head, w.b);
                    }
                }
                ++n_some;
            }
            bool dirty = is_dirty(w, plan, 0);
            for (int c = 0; c < w.chunks; ++c, ++i) {
                const int s1 = i % kRing1, s2 = i % kRing2;
                const uint32_t ph1 = (uint32_t)(i / kRing1) & 1u, ph2 = (uint32_t)(i / kRing2) & 1u;
                const Chunk ch = chunk_at(w, c);
                const int row = ch.t * kTile, head = KVS ? ch.head : w.kv_head;
                const bool dirty_next = is_dirty(w, plan, c + 1);
                const uint32_t d1 = sRing1 + s1 * kTileBytes, d2 = sRing2 + s2 * kTileBytes;
                const long stat = (((long)w.b * p.q_heads + head) * p.plan.q_tiles + ch.t) * kTile;
                if (!warp_wait(b1_empty(s1), ph1 ^ 1u, &abort_flag)) goto done;
                if (lead) {
                    mbar_arrive_expect_tx(b1_full(s1), kTileBytes + (KVS ? kTile * 4 : 0));
                    if (KVS) bulk_load_1d(sLse + s1 * kTile * 4, p.lse + stat, kTile * 4, b1_full(s1));
#pragma unroll
                    for (int h = 0; h < L::kSlabs; ++h) tma_load_4d(d1 + h * kSlab, KVS ? &tmQ : &tmK, b1_full(s1), h * 64, row, head, w.b);
                }
                if (!warp_wait(b2_empty(s2), ph2 ^ 1u, &abort_flag)) goto done;
                if (lead) {
                    mbar_arrive_expect_tx(b2_full(s2), kTileBytes + (KVS ? kTile * 4 : 0));
                    if (KVS) bulk_load_1d(sDelta + s2 * kTile * 4, p.delta + stat, kTile * 4, b2_full(s2));
#pragma unroll
                    for (int h = 0; h < L::kSlabs; ++h) tma_load_4d(d2 + h * kSlab, KVS ? &tmDO : &tmV, b2_full(s2), h * 64, row, head, w.b);
                }
                __syncwarp();
                if (dirty) {        // their P and dS are 0, and 0 times a NaN is a NaN
                    uint4 bits;
                    if (KVS) {
                        uint32_t m[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int r = row + q * 32 + lane;
                            m[q] = __ballot_sync(0xffffffffu, r < p.q_len && plan.first[r] >= plan.behind[r]);
                        }
                        bits = make_uint4(m[0], m[1], m[2], m[3]);
                    } else {
                        bits = plan.dead[ch.t];
                    }
                    if (!warp_wait(b1_full(s1), ph1, &abort_flag)) goto done;
                    clear_rows(d1, L::kSlabs, bits, lane);
                    if (KVS) {      // V only meets dS through a selection by the mask
                        if (!warp_wait(b2_full(s2), ph2, &abort_flag)) goto done;
                        clear_rows(d2, L::kSlabs, bits, lane);
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lead) {
                        mbar_arrive(b1_clean(s1));
                        if (KVS) mbar_arrive(b2_clean(s2));
                    }
                }
                dirty = dirty_next;
            }
            if (!queue.ask(lead, &abort_flag)) goto done;
            if (!warp_wait(queue.full(), queue.parity(), &abort_flag)) goto done;
        } while (queue.next<true>(lead, &bx, &by, &bz));
    } else if (warp == 1) {
        // ------------------------------------------------------------ products
        if (elect_one()) {
            constexpr uint32_t idesc_t = idesc<BF16>(kTile, kTile, false, false);   // T = A B^T, both K-major
            constexpr uint32_t idesc_a = idesc<BF16>(kTile, D, false, true);        // acc += P B, B MN-major
            auto issue_t = [&](uint32_t t_col, uint32_t sa, uint32_t sb) {
                const uint64_t a = fresh_desc(smem_desc_sw128(sa, 16, 1024)), k = fresh_desc(smem_desc_sw128(sb, 16, 1024));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint64_t off = (uint64_t)(((kk >> 2) * kSlab + (kk & 3) * 32) >> 4);
                    umma_bf16_ss(tmem + t_col, a + off, k + off, idesc_t, kk ? 1u : 0u);
                }
            };
            // acc[128 x D] += A (pairs in tensor memory, 128 stationary x 128 streamed rows) x chunk (MN-major B)
            auto issue_acc = [&](uint32_t acc_col, uint32_t a_col, uint32_t sb, bool first) {
                const uint64_t k = fresh_desc(smem_desc_sw128(sb, kSlab, 1024));
#pragma unroll
                for (int kk = 0; kk < kTile / 16; ++kk)
                    umma_bf16_ts(tmem + acc_col, tmem + a_col + (kk >> 1) * kCols + (kk & 1) * 8, k + (uint64_t)(kk * (2048 >> 4)), idesc_a,
                                 (first && kk == 0) ? 0u : 1u);
            };
            uint32_t cleaned1 = 0, cleaned2 = 0;        // bit s: parity of the cleaned uses of slot s
            auto wait_b1 = [&](int i, bool dirty) {
                const int s = i % kRing1;
                if (!dirty) return mbar_wait(b1_full(s), (uint32_t)(i / kRing1) & 1u, &abort_flag);
                const uint32_t par = cleaned1 >> s & 1u;
                cleaned1 ^= 1u << s;
                return mbar_wait(b1_clean(s), par, &abort_flag);
            };
            auto wait_b2 = [&](int i, bool dirty) {
                const int s = i % kRing2;
                if (!KVS || !dirty) return mbar_wait(b2_full(s), (uint32_t)(i / kRing2) & 1u, &abort_flag);
                const uint32_t par = cleaned2 >> s & 1u;
                cleaned2 ^= 1u << s;
                return mbar_wait(b2_clean(s), par, &abort_flag);
            };
            auto slot1 = [&](int i) { return sRing1 + i % kRing1 * kTileBytes; };
            auto slot2 = [&](int i) { return sRing2 + i % kRing2 * kTileBytes; };
            auto t2_of = [&](int i) { return KVS || !(i & 1) ? kT2 : kT3; };
            int i = 0, n_some = 0;              // chunks, and items that have any, so far
            do {
                const Item w = item_at(bx, by, bz);
                const PlanView plan = p.plan.sample(w.b);
                if (w.chunks > 0) {
                    const bool dirty = is_dirty(w, plan, 0);
                    if (!mbar_wait(a_full, (uint32_t)n_some++ & 1u, &abort_flag)) goto done;
                    if (!wait_b1(i, dirty)) goto done;
                    tc_fence_after();
                    issue_t(kT1, sA1, slot1(i));
                    umma_commit(s_full);
                    if (!wait_b2(i, dirty)) goto done;
                    tc_fence_after();
                    issue_t(t2_of(i), sA2, slot2(i));
                    umma_commit(dp_full(i));
                    if (!KVS) umma_commit(b2_empty(i % kRing2));
                    if (w.chunks == 1) umma_commit(a_empty);
                }
                for (int c = 0; c < w.chunks; ++c, ++i) {
                    const uint32_t par = (uint32_t)i & 1u;
                    const bool more = c + 1 < w.chunks;
                    const bool dirty_next = is_dirty(w, plan, c + 1);
                    if (!mbar_wait(p_ready, par, &abort_flag)) goto done;
                    tc_fence_after();
                    if (KVS) {
                        // T1 holds P: dV takes it while dS is formed, then the next chunk's scores take T1
                        issue_acc(kAcc1, kT1, slot2(i), c == 0);                    // dV += P^T dO
                        if (more) {
                            if (!wait_b1(i + 1, dirty_next)) goto done;
                            tc_fence_after();
                            issue_t(kT1, sA1, slot1(i + 1));
                            umma_commit(s_full);
                        }
                        if (!mbar_wait(ds_ready, par, &abort_flag)) goto done;
                        tc_fence_after();
                        issue_acc(kAcc2, kT2, slot1(i), c == 0);                    // dK += dS^T Q
                        umma_commit(b1_empty(i % kRing1));
                        umma_commit(b2_empty(i % kRing2));         // not behind dV: delta lies in the slot until dS is formed
                        if (more) {
                            if (!wait_b2(i + 1, dirty_next)) goto done;
                            tc_fence_after();
                            issue_t(kT2, sA2, slot2(i + 1));
                            umma_commit(dp_full(i + 1));
                        }
                    } else {
                        // the scores have been read: the next chunk's, and its dP in the other buffer, overlap this chunk's dS
                        if (more) {
                            if (!wait_b1(i + 1, dirty_next)) goto done;
                            tc_fence_after();
                            issue_t(kT1, sA1, slot1(i + 1));
                            umma_commit(s_full);
                            if (!wait_b2(i + 1, dirty_next)) goto done;
                            tc_fence_after();
                            issue_t(t2_of(i + 1), sA2, slot2(i + 1));
                            umma_commit(dp_full(i + 1));
                            umma_commit(b2_empty((i + 1) % kRing2));
                        }
                        if (!mbar_wait(ds_ready, par, &abort_flag)) goto done;
                        tc_fence_after();
                        issue_acc(kAcc1, t2_of(i), slot1(i), c == 0);               // dQ += dS K
                        umma_commit(b1_empty(i % kRing1));
                    }
                    if (c + 2 == w.chunks) umma_commit(a_empty);        // the item's last scores and dP: the next one's operands may come
                }
                if (w.chunks > 0) umma_commit(acc_final);
                if (!mbar_wait(queue.full(), queue.parity(), &abort_flag)) goto done;
            } while (queue.next<false>(true, &bx, &by, &bz));
        }
    } else {
        // ------------------------------------------------------------ P and dS
        const int part = (warp - 2) >> 2, quad = warp & 3;
        const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
        const uint32_t t1 = tmem + lane_sel + kT1 + part * kCols, t2 = tmem + lane_sel + kT2 + part * kCols;
        // what a thread needs of an item; the next one's is read ahead of this one's results
        struct Mine {
            Item w;
            float lse, delta;
            int first, behind, start;
        };
        auto mine_of = [&](int x, int y, int z) {
            Mine v;
            v.w = item_at(x, y, z);
            const PlanView plan = p.plan.sample(v.w.b);
            v.start = plan.start;
            v.lse = v.delta = 0.f;
            v.first = v.behind = 0;
            if (!KVS) {
                const int row = v.w.tile * kTile + quad * 32 + lane;
                const long at = ((long)v.w.b * p.q_heads + v.w.head) * p.plan.q_tiles * kTile + row;
                v.lse = p.lse[at];             // +inf behind the last query: its P is 0
                v.delta = p.delta[at];
                if (row < p.q_len) {
                    v.first = plan.first[row];
                    v.behind = plan.behind[row];
                }
            }
            return v;
        };
        Mine v = mine_of(bx, by, bz);
        int i = 0, n_diag = 0, n_final = 0;
        bool go = true;
        while (go) {
            const Item w = v.w;
            const PlanView plan = p.plan.sample(w.b);
            const int r0 = w.tile * kTile, row = r0 + quad * 32 + lane;         // key (KVS) or query
            const int start = v.start;
            float far_sum = 0.f, near_sum = 0.f;    // of dS beyond the largest distance: ahead of the query, behind it
            float far_p = 0.f, near_p = 0.f, all_sum = 0.f;     // of P there, and of all dS
            for (int c = 0; c < w.chunks; ++c, ++i) {
                const uint32_t par = (uint32_t)i & 1u;
                const Chunk ch = chunk_at(w, c);
                const int col0 = ch.t * kTile + part * kCols;         // first streamed row of this thread's 32
                uint32_t see = 0xffffffffu;
                bool one = false;           // the query (KVS: of column `lane`) sees one key
                if (KVS) {
                    const int4 r = plan.q_tiles[ch.t];
                    if (r.z > r0 || r.w < min(r0 + kTile, p.kv_len) || p.kv_len - r0 == 1) {        // some query does not see all of these keys, or it is one
                        const int q = col0 + lane, k0 = r0 + quad * 32;
                        uint32_t mine = 0u;                                    // keys of this warp that query `lane` sees
                        if (q < p.q_len) {
                            const int first = plan.first[q], behind = plan.behind[q];
                            mine = bits_between(first - k0, behind - k0);
                            one = behind - first == 1;
                        }
                        see = 0u;
#pragma unroll
                        for (int e = 0; e < 32; ++e) see |= (__shfl_sync(0xffffffffu, mine, e) >> lane & 1u) << e;
                    }
                } else {
                    see = bits_between(v.first - col0, v.behind - col0);
                }
                const bool clean = __all_sync(0xffffffffu, see == 0xffffffffu);
                // distance of column e: pos0 + e, KVS pos0 - e
                const int pos0 = KVS ? row - (start + col0) : col0 - (start + row);
                bool at_end = false, inside = false;
                float end_bias = 0.f;
                const float* bias_row = nullptr;
                if (MODE >= kGeneral) {
                    bias_row = p.bias + (long)ch.head * (2 * p.R + 1) + p.R;
                    const int w0 = __shfl_sync(0xffffffffu, pos0, 0), w31 = __shfl_sync(0xffffffffu, pos0, 31);
                    const int least = KVS ? w0 - 31 : w31, most = KVS ? w31 : w0 + 31;
                    at_end = most <= -p.R || least >= p.R;
                    inside = least >= -p.R && most <= p.R;
                    if (at_end) end_bias = bias_row[least >= p.R ? p.R : -p.R] * kLog2e;
                }
                uint32_t tk[MODE >= kGeneral ? 16 : 1], a[32];
                if (!warp_wait(s_full, par, &abort_flag)) goto done;
                tc_fence_after();
                tmem_ld_32x32(t1, a);
                tmem_ld_wait();
                // raw scores to the log2 domain (kPlain: with the exponential)
                if (MODE == kCapped || (MODE >= kGeneral && p.cap.out != 0.f)) {
                    if (all_small<32>(p.cap, a)) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 y = cap_small(p.cap, make_float2(__uint_as_float(a[e]), __uint_as_float(a[e + 1])));
                            a[e] = __float_as_uint(y.x);
                            a[e + 1] = __float_as_uint(y.y);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(cap_any(p.cap, __uint_as_float(a[e])));
                    }
                    if (MODE >= kGeneral) {         // the slope ahead of the bias, in fp16: 2^-11 of a factor that is rounded to 16 bits with its dS below
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float2 f = slope_of(make_float2(__uint_as_float(a[2 * e]), __uint_as_float(a[2 * e + 1])));
                            tk[e] = pack2<false>(f.x, f.y);
                        }
                    }
                } else if (MODE >= kGeneral) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(__uint_as_float(a[e]) * p.scale_log2);
                }
                if (MODE >= kGeneral) {
                    if (at_end) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(__uint_as_float(a[e]) + end_bias);
                    } else if (inside) {
                        const float* entry = bias_row + pos0;
#pragma unroll
                        for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(fmaf(__ldg(KVS ? entry - e : entry + e), kLog2e, __uint_as_float(a[e])));
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            a[e] = __float_as_uint(fmaf(__ldg(bias_row + max(-p.R, min(p.R, KVS ? pos0 - e : pos0 + e))), kLog2e, __uint_as_float(a[e])));
                    }
                }
                if (KVS && !warp_wait(b1_full(i % kRing1), (uint32_t)(i / kRing1) & 1u, &abort_flag)) goto done;       // has the copied lse: long complete
                // P in 32 bits over the scores.  For the product with dO it is rounded, half a step of the operands' type; for dS it stays, behind a
                // cap alone times the cap's slope.
                uint32_t pk[KVS ? 16 : 1];
                auto exponentials = [&](auto whole) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        float4 l4 = make_float4(v.lse, v.lse, v.lse, v.lse);
                        if (KVS) lds4(sLse + ((i % kRing1) * kTile + part * kCols + 4 * q) * 4, l4);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int e = 4 * q + 2 * h;
                            const float2 s2 = make_float2(__uint_as_float(a[e]), __uint_as_float(a[e + 1]));
                            const float2 n2 = h ? make_float2(-l4.z, -l4.w) : make_float2(-l4.x, -l4.y);
                            const float2 y = MODE == kPlain ? __ffma2_rn(s2, make_float2(p.scale_log2, p.scale_log2), n2) : __fadd2_rn(s2, n2);
                            float2 pr = make_float2(exp2f(y.x), exp2f(y.y)), f = MODE == kCapped ? slope_of(s2) : make_float2(1.f, 1.f);
                            if (!whole) {       // P and slope of a key or a query that no run reaches may be anything
                                if (!(see >> e & 1u)) pr.x = f.x = 0.f;
                                if (!(see >> (e + 1) & 1u)) pr.y = f.y = 0.f;
                            }
                            if (KVS) pk[e >> 1] = pack2<BF16>(pr.x, pr.y);
                            if (MODE == kCapped) pr = __fmul2_rn(pr, f);
                            a[e] = __float_as_uint(pr.x);
                            a[e + 1] = __float_as_uint(pr.y);
                        }
                    }
                };
                // With stationary queries one form for both is the faster one (3430 -> 2960 us at 32656 packed tokens), with stationary keys two are
                // (4556 against 4658).
                if (!KVS) exponentials(clean);
                else if (clean) exponentials(std::true_type());
                else exponentials(std::false_type());
                if (KVS) {
                    tmem_st_32x16(t1, pk);
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready);
                // a query that sees one key weighs it 1 whatever its score: dP - delta is nothing but rounding
                if (KVS) see &= ~__ballot_sync(0xffffffffu, one);
                else if (v.behind - v.first == 1) see = 0u;

                // beyond the largest distance the bias's gradient takes sums only
                const int corner = ch.t * kTile - (start + r0);         // distance of the tile's first key from its first query
                const bool beyond = MODE == kGeneralDbias && (corner + kTile - 1 <= -p.R || corner - kTile + 1 >= p.R);
                if (MODE == kGeneralDbias && beyond) {
                    float s = 0.f;
#pragma unroll
                    for (int e = 0; e < 32; ++e) s += __uint_as_float(a[e]);
                    if (corner < 0) near_p += s;
                    else far_p += s;
                }

                const uint32_t t2c = KVS || !(i & 1) ? t2 : t2 + (kT3 - kT2);
                if (!warp_wait(dp_full(i), KVS ? par : (uint32_t)(i >> 1) & 1u, &abort_flag)) goto done;
                tc_fence_after();
                if (KVS && !warp_wait(b2_full(i % kRing2), (uint32_t)(i / kRing2) & 1u, &abort_flag)) goto done;       // and delta
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t g[16], dk[8];
                    tmem_ld_32x16(t2c + 16 * half, g);
                    tmem_ld_wait();
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float4 d4 = make_float4(v.delta, v.delta, v.delta, v.delta);
                        if (KVS) lds4(sDelta + ((i % kRing2) * kTile + part * kCols + 16 * half + 4 * q) * 4, d4);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int e = 4 * q + 2 * h, k = 16 * half + e;
                            const float2 n2 = h ? make_float2(-d4.z, -d4.w) : make_float2(-d4.x, -d4.y);
                            float2 ds = __fmul2_rn(make_float2(__uint_as_float(a[k]), __uint_as_float(a[k + 1])),
                                                   __fadd2_rn(make_float2(__uint_as_float(g[e]), __uint_as_float(g[e + 1])), n2));
                            float2 f = make_float2(1.f, 1.f);
                            if (MODE >= kGeneral && p.cap.out != 0.f) f = unpack2<false>(tk[k >> 1]);
                            if (!clean) {           // dP and slope of a key or a query that no run reaches may be anything
                                if (!(see >> k & 1u)) ds.x = f.x = 0.f;
                                if (!(see >> (k + 1) & 1u)) ds.y = f.y = 0.f;
                            }
                            if (MODE == kGeneralDbias) {
                                a[k] = __float_as_uint(ds.x);
                                a[k + 1] = __float_as_uint(ds.y);
                            }
                            if (MODE >= kGeneral) ds = __fmul2_rn(ds, f);
                            // rounded to the operands' type, as the products take it: half a step of each dS
                            dk[e >> 1] = pack2<BF16>(ds.x, ds.y);
                        }
                    }
                    tmem_st_32x8(t2c + 8 * half, dk);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_ready);

                if (MODE == kGeneralDbias) {
                    float s = 0.f;
#pragma unroll
                    for (int e = 0; e < 32; ++e) s += __uint_as_float(a[e]);
                    all_sum += s;
                    if (beyond) {
                        if (corner < 0) near_sum += s;
                        else far_sum += s;
                    } else {
                        // Sums along the diagonals of the warp's 32 x 32 block: a partial sum moves down one row per column.  Slot
                        // c - row + 31; what leaves the last row at column c is slot c, what is left at the end belongs to slots 62 - row.
                        float* slots = scratch + ((n_diag & 1) * 16 + part * 4 + quad) * 64;
                        float acc = 0.f;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float above = __shfl_up_sync(0xffffffffu, acc, 1);
                            acc = (lane == 0 ? 0.f : above) + __uint_as_float(a[e]);
                            if (lane == 31) slots[e] = acc;
                        }
                        if (lane < 31) slots[62 - lane] = acc;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(diag_ready);
                        if (!warp_wait(diag_ready, (uint32_t)n_diag & 1u, &abort_flag)) goto done;
                        // one diagonal of the tile a thread, its warps' shares in a fixed order
                        const int x = (int)threadIdx.x - 64;
                        if (x < 2 * kTile - 1) {
                            const int d = x - (kTile - 1);
                            float sum = 0.f;
                            for (int q = 0; q < 4; ++q)
                                for (int k = 0; k < 4; ++k) {
                                    const int slot = d - 32 * (k - q) + 31;
                                    if (slot >= 0 && slot < 63) sum += scratch[((n_diag & 1) * 16 + k * 4 + q) * 64 + slot];
                                }
                            diag[kDiagPad + p.R + corner + d] += sum;
                        }
                        ++n_diag;
                    }
                }
            }
            if (MODE == kGeneralDbias) {
                // The sums beyond the largest distance are sums of whole rows, and a row of dS sums to nothing: what it sums to is delta's
                // error, which leaves them again by its share of P.  Row by row over the four parts of the row, then row after row.
                float* slots = scratch + (n_diag & 1) * 16 * 64;
                slots[(part * 4 + quad) * 64 + lane] = all_sum;
                __syncwarp();
                if (lane == 0) mbar_arrive(diag_ready);
                if (!warp_wait(diag_ready, (uint32_t)n_diag & 1u, &abort_flag)) goto done;
                float over = 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q) over += slots[(q * 4 + quad) * 64 + lane];
                near_sum -= near_p * over;
                far_sum -= far_p * over;
                for (int o = 16; o > 0; o >>= 1) {
                    near_sum += __shfl_xor_sync(0xffffffffu, near_sum, o);
                    far_sum += __shfl_xor_sync(0xffffffffu, far_sum, o);
                }
                ++n_diag;
                slots = scratch + (n_diag & 1) * 16 * 64;
                if (lane == 0) {
                    slots[2 * (part * 4 + quad)] = near_sum;
                    slots[2 * (part * 4 + quad) + 1] = far_sum;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(diag_ready);
                if (!warp_wait(diag_ready, (uint32_t)n_diag & 1u, &abort_flag)) goto done;
                ++n_diag;
                float* out = p.partials + (((long)w.b * p.q_heads + w.head) * p.plan.q_tiles + w.tile) * (2 * p.R + 1);
                for (int e = (int)threadIdx.x - 64; e < 2 * p.R + 1; e += kThreads - 64) {
                    float s = diag[kDiagPad + e];
                    if (e == 0) {
                        for (int q = 0; q < kDiagPad; ++q) s += diag[q];
                        for (int q = 0; q < 16; ++q) s += slots[2 * q];
                    }
                    if (e == 2 * p.R) {
                        for (int q = 0; q < kDiagPad; ++q) s += diag[kDiagPad + 2 * p.R + 1 + q];
                        for (int q = 0; q < 16; ++q) s += slots[2 * q + 1];
                    }
                    out[e] = s;
                }
                // cleared for the next item once all have read it; its first addition is behind another wait of all
                __syncwarp();
                if (lane == 0) mbar_arrive(diag_ready);
                if (!warp_wait(diag_ready, (uint32_t)n_diag & 1u, &abort_flag)) goto done;
                ++n_diag;
                for (int e = (int)threadIdx.x - 64; e < 2 * p.R + 1 + 2 * kDiagPad; e += kThreads - 64) diag[e] = 0.f;
            }
            // ------------------------------------------------------------ gradients
            if (!warp_wait(queue.full(), queue.parity(), &abort_flag)) goto done;
            go = queue.next<true>(lane == 0, &bx, &by, &bz);
            if (go) v = mine_of(bx, by, bz);
            if (w.chunks > 0 && !warp_wait(acc_final, (uint32_t)n_final++ & 1u, &abort_flag)) goto done;
            tc_fence_after();
            const int rows = KVS ? p.kv_len : p.q_len, row0 = row - lane;
#pragma unroll 1
            for (int which = 0; which < (KVS ? 2 : 1); ++which) {
                const long* st = which == 0 ? p.s1 : p.s2;
                uint16_t* const dst = reinterpret_cast<uint16_t*>(which == 0 ? p.out1 : p.out2) + w.b * st[0] + (KVS ? w.kv_head : w.head) * st[1] + row0 * st[2];
                const float mul = (KVS && which == 0) ? 1.f : p.scale;         // dV is unscaled
                const uint32_t tacc = tmem + lane_sel + (which == 0 ? kAcc1 : kAcc2);
#pragma unroll 1
                for (int cch = part; cch < D / 32; cch += kGroups) {        // the warpgroups share the accumulator's columns
                    uint32_t r[32];
                    tmem_ld_32x32(tacc + cch * 32, r);
                    tmem_ld_wait();
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = w.chunks == 0 ? 0.f : __uint_as_float(r[e]) * mul;
                    uint4 piece[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        piece[g] = make_uint4(pack2<BF16>(o[g * 8], o[g * 8 + 1]), pack2<BF16>(o[g * 8 + 2], o[g * 8 + 3]),
                                              pack2<BF16>(o[g * 8 + 4], o[g * 8 + 5]), pack2<BF16>(o[g * 8 + 6], o[g * 8 + 7]));
                    if (L::kStage > 0) {
                        store_rows64(stages + (warp - 2) * 2048, lane, piece, [&](int e) { return row0 + e < rows ? dst + e * st[2] + cch * 32 : nullptr; });
                    } else if (row < rows) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(dst + lane * st[2] + cch * 32 + g * 8) = piece[g];
                    }
                }
            }
            tc_fence_before();          // ahead of the arrivals that let the next item's first products overwrite the accumulators
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

// delta = rowsum(dO O) in fp32; 0 for queries that see nothing (their dO may be anything) and behind the last.  D / 8 lanes a row.
template <int D, bool BF16, bool WIDE>
__global__ void __launch_bounds__(256) ranges_delta_kernel(const PlanPtr plan, const uint16_t* __restrict__ dout, const void* __restrict__ out,
                                                           float* __restrict__ delta, long rows, int q_len, int q_heads) {
    constexpr int kLanes = D / 8;
    const int pitch = plan.q_tiles * kTile, l = threadIdx.x % kLanes;
    for (long w = ((long)blockIdx.x * 256 + threadIdx.x) / kLanes; w < rows; w += (long)gridDim.x * (256 / kLanes)) {
        // heads of a query are neighbours in memory: w counts [batch, padded queries, heads]
        const int h = (int)(w % q_heads);
        const long bi = w / q_heads;
        const int i = (int)(bi % pitch);
        const long b = bi / pitch;
        float s = 0.f;
        if (i < q_len && plan.base[plan.at.first + b * q_len + i] < plan.base[plan.at.behind + b * q_len + i]) {
            const long at = ((b * q_len + i) * q_heads + h) * D + l * 8;
            const uint4 g = *reinterpret_cast<const uint4*>(dout + at);
            float2 o[4];
            if (WIDE) {
                const float4 u = reinterpret_cast<const float4*>((const float*)out + at)[0], v = reinterpret_cast<const float4*>((const float*)out + at)[1];
                o[0] = make_float2(u.x, u.y);
                o[1] = make_float2(u.z, u.w);
                o[2] = make_float2(v.x, v.y);
                o[3] = make_float2(v.z, v.w);
            } else {
                const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*)out + at);
                o[0] = unpack2<BF16>(u.x);
                o[1] = unpack2<BF16>(u.y);
                o[2] = unpack2<BF16>(u.z);
                o[3] = unpack2<BF16>(u.w);
            }
            const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 d = unpack2<BF16>(gw[e]);
                s += d.x * o[e].x + d.y * o[e].y;
            }
        }
#pragma unroll
        for (int m = kLanes / 2; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m, kLanes);
        if (l == 0) delta[(b * q_heads + h) * pitch + i] = s;
    }
}

// dbias[h, e]: the tiles' rows of the table, summed in a fixed order.  32 entries a CTA, 32 threads an entry.
__global__ void __launch_bounds__(1024) ranges_dbias_kernel(const float* __restrict__ partials, float* __restrict__ dbias, int batch, int q_heads,
                                                            int q_tiles, int entries) {
    __shared__ float fold[32][33];
    const int e = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5, h = blockIdx.y;
    float s = 0.f;
    if (e < entries)
        for (int i = g; i < batch * q_tiles; i += 32) {
            const int b = i / q_tiles, t = i - b * q_tiles;
            s += partials[(((long)b * q_heads + h) * q_tiles + t) * entries + e];
        }
    fold[g][threadIdx.x & 31] = s;
    __syncthreads();
    if (g == 0 && e < entries) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += fold[i][threadIdx.x];
        dbias[(long)h * entries + e] = s;
    }
}

struct Maps {
    CUtensorMap q, k, v, dout;
};

template <int D, bool BF16, bool KVS, int MODE>
int launch(const tt_ranges_args& a, const Maps& m, BwdParams p, int dev, cudaStream_t st) {
    auto kern = ranges_bwd_kernel<D, BF16, KVS, MODE>;
    using L = Layout<D, KVS, MODE>;
    static bool configured[64] = {false};         // per device: the attribute belongs to the device's context
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(TT_RANGES_MAX_DISTANCE));
        if (e != cudaSuccess) return tt_record_cuda(e);
        configured[dev] = true;
    }
    p.out1 = KVS ? a.dv : a.dq;
    p.out2 = KVS ? a.dk : nullptr;
    for (int i = 0; i < 3; ++i) {
        p.s1[i] = KVS ? a.dv_stride[i] : a.dq_stride[i];
        p.s2[i] = KVS ? a.dk_stride[i] : 0;
    }
    const int tiles = KVS ? p.plan.k_tiles : p.plan.q_tiles;
    p.order = make_order(a, tiles);
    kern<<<p.order.grid(tiles, KVS ? a.k_heads : a.q_heads, a.batch), kThreads, L::smem(a.max_distance), st>>>(m.q, m.k, m.v, m.dout, p);
    TT_CHECK_LAUNCH();
    return TT_OK;
}

template <int D, bool BF16>
int run(const tt_ranges_args& a, const BwdParams& p, int dev, int sms, cudaStream_t st) {
    Maps m;
    int rc;
    const long dout_stride[3] = {(long)a.q_len * a.q_heads * D, D, (long)a.q_heads * D};
    if ((rc = tt_make_tmap_bhsd(&m.q, a.q, a.batch, a.q_heads, a.q_len, D, a.q_stride, kTile)) != TT_OK) return rc;
    if ((rc = tt_make_tmap_bhsd(&m.k, a.k, a.batch, a.k_heads, a.kv_len, D, a.k_stride, kTile)) != TT_OK) return rc;
    if ((rc = tt_make_tmap_bhsd(&m.v, a.v, a.batch, a.k_heads, a.kv_len, D, a.v_stride, kTile)) != TT_OK) return rc;
    if ((rc = tt_make_tmap_bhsd(&m.dout, a.dout, a.batch, a.q_heads, a.q_len, D, dout_stride, kTile)) != TT_OK) return rc;
    const long rows = (long)a.batch * a.q_heads * p.plan.q_tiles * kTile, want = (rows * (D / 8) + 255) / 256;
    const int grid = (int)(want < sms * 16L ? want : sms * 16L);
    if (a.out32 != nullptr)
        ranges_delta_kernel<D, BF16, true><<<grid, 256, 0, st>>>(p.plan, (const uint16_t*)a.dout, a.out32, a.delta, rows, a.q_len, a.q_heads);
    else
        ranges_delta_kernel<D, BF16, false><<<grid, 256, 0, st>>>(p.plan, (const uint16_t*)a.dout, a.out, a.delta, rows, a.q_len, a.q_heads);
    TT_CHECK_LAUNCH();
    const bool bias = a.max_distance >= 0, cap = a.softcap > 0.f;
    rc = bias ? launch<D, BF16, true, kGeneral>(a, m, p, dev, st)
         : cap ? launch<D, BF16, true, kCapped>(a, m, p, dev, st) : launch<D, BF16, true, kPlain>(a, m, p, dev, st);
    if (rc != TT_OK) return rc;
    if (a.dbias == nullptr)
        return bias ? launch<D, BF16, false, kGeneral>(a, m, p, dev, st)
               : cap ? launch<D, BF16, false, kCapped>(a, m, p, dev, st) : launch<D, BF16, false, kPlain>(a, m, p, dev, st);
    if ((rc = launch<D, BF16, false, kGeneralDbias>(a, m, p, dev, st)) != TT_OK) return rc;
    const int entries = 2 * a.max_distance + 1;
    ranges_dbias_kernel<<<dim3((entries + 31) / 32, a.q_heads), 1024, 0, st>>>(a.partials, a.dbias, a.batch, a.q_heads, p.plan.q_tiles, entries);
    TT_CHECK_LAUNCH();
    return TT_OK;
}

}  // namespace

extern "C" int tt_attn_ranges_bwd(const tt_ranges_args* a, void* stream) {
    int rc = tt_ranges_check(a);
    if (rc != TT_OK) return rc;
    if (a->dout == nullptr || a->delta == nullptr || a->dq == nullptr || a->dk == nullptr || a->dv == nullptr) return TT_ERR_ARG;
    for (const void* x : {a->dout, (const void*)a->lse, (const void*)a->delta, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
        if ((uintptr_t)x & 15) return TT_ERR_ARG;
    for (const long* s : {a->dq_stride, a->dk_stride, a->dv_stride})
        if (s[0] % 8 || s[1] % 8 || s[2] % 8) return TT_ERR_ARG;
    if (a->dbias != nullptr && (a->partials == nullptr || a->max_distance < 0)) return TT_ERR_ARG;
    const tt_device_info dev = tt_device();
    BwdParams p;
    p.plan = plan_ptr(*a);
    p.lse = a->lse;
    p.delta = a->delta;
    p.bias = a->bias;
    p.partials = a->partials;
    p.q_len = a->q_len;
    p.kv_len = a->kv_len;
    p.q_heads = a->q_heads;
    p.group = a->q_heads / a->k_heads;
    p.R = a->max_distance;
    p.scale = a->scale;
    p.scale_log2 = a->scale * kLog2e;
    p.cap = make_cap(a->scale, a->softcap);
    p.status = a->status;
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = a->dtype == TT_BF16;
    if (a->head_dim == 128) return bf ? run<128, true>(*a, p, dev.dev, dev.sms, st) : run<128, false>(*a, p, dev.dev, dev.sms, st);
    return bf ? run<64, true>(*a, p, dev.dev, dev.sms, st) : run<64, false>(*a, p, dev.dev, dev.sms, st);
}
