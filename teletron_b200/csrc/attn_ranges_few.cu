// The attention of attn_ranges_fwd.cu for few queries over long keys (new tokens over a cache): at most 32 rows of a key head's group.
//
// What bounds it is reading keys and values once, so the keys of a sample and key head are split over CTAs and, in steps of 16, over
// their four warps.  Every warp streams its keys and values through a ring of its own in shared memory (16-byte asynchronous copies, three steps
// deep: 96 KB in flight per CTA at heads of 128) and keeps running maxima, sums and outputs of its 16 or 32 rows (the queries of all heads of the
// group, so that shared keys are read once) in registers; the products are mma.sync of 16 x 8 x 16, which a tile of 128 queries on
// tcgen05 would leave seven eighths empty.  Warps are joined through shared memory, CTAs by a second kernel in a fixed order.
#include <limits.h>

#include "attn_ranges.cuh"

namespace {

using namespace ranges;

constexpr int kWarps = 4, kThreads = kWarps * 32, kStep = 16, kStages = 3;
constexpr int kMaxRows = 32;

struct FewParams {
    PlanPtr plan;
    const uint16_t *q, *k, *v;
    long qs[3], ks[3], vs[3];
    uint16_t* out;
    float *lse, *partials;
    const float* bias;
    int q_len, q_heads, k_heads, group, R, splits;
    float scale_log2;
    Cap cap;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");     // zeros where not in
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <bool TRANS> __device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t* r) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool BF16> __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Rows of D 16-bit elements in shared memory, their 16-byte pieces exchanged by row so that eight rows' same piece lies in eight banks
template <int D> __device__ __forceinline__ uint32_t place(uint32_t base, int row, int piece) {
    return base + row * (D * 2) + ((piece ^ (row & 7)) << 4);
}

template <int D, int MT> struct Few {
    static constexpr int kTileBytes = kStep * D * 2;                        // 16 keys
    static constexpr int kRing = kStages * 2 * kTileBytes;                  // of one warp
    static constexpr int kQ = MT * 16 * D * 2;
    static constexpr int kSmem = kWarps * kRing + kQ;
    static_assert(kRing >= MT * 16 * D * 4, "a warp's outputs are joined in its ring");
};

template <int D, bool BF16, bool GEN, int MT>
__global__ void __launch_bounds__(kThreads) few_kernel(const FewParams p) {
    using F = Few<D, MT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float stats[kWarps][kMaxRows][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, kv_head = blockIdx.y, b = blockIdx.z;
    const PlanView plan = p.plan.sample(b);
    const int rows = p.group * p.q_len;             // row r: query r / group of head r % group
    const uint32_t sQ = sm100::smem_u32(smem) + kWarps * F::kRing, ring = sm100::smem_u32(smem) + warp * F::kRing;

    const int4 bounds = plan.q_tiles[0];
    const int k_lo = bounds.x < bounds.y ? bounds.x / kStep * kStep : 0, k_hi = bounds.x < bounds.y ? bounds.y : 0;
    const int steps = (k_hi - k_lo + kStep - 1) / kStep;
    const int s0 = (int)((long)steps * split / p.splits), s1 = (int)((long)steps * (split + 1) / p.splits);

    const uint16_t* kp = p.k + b * p.ks[0] + kv_head * p.ks[1];
    const uint16_t* vp = p.v + b * p.vs[0] + kv_head * p.vs[1];
    // bit i: key i of a step is one that no query sees; read a fetch ahead, so that no copy waits for it
    auto dead_of = [&](int step) {
        const int key = k_lo + step * kStep;
        if (step >= s1) return 0u;
        return reinterpret_cast<const uint32_t*>(plan.dead + key / kTile)[key % kTile / 32] >> (key % 32) & 0xffffu;
    };
    auto fetch = [&](int step, int slot, uint32_t dead) {          // keys and values of a step; behind the last, and where no query looks, zeros
        const uint32_t dk = ring + slot * (2 * F::kTileBytes), dv = dk + F::kTileBytes;
        const int key0 = k_lo + step * kStep, behind = step < s1 ? k_hi - key0 : 0;
#pragma unroll
        for (int i = 0; i < kStep * D / 8 / 32; ++i) {
            const int c = i * 32 + lane, r = c / (D / 8), piece = c % (D / 8);
            const bool in = r < behind && !(dead >> r & 1u);
            const long at = in ? (long)(key0 + r) : 0L;
            copy16(place<D>(dk, r, piece), kp + at * p.ks[2] + piece * 8, in);
            copy16(place<D>(dv, r, piece), vp + at * p.vs[2] + piece * 8, in);
        }
        copy_commit();
    };
    uint32_t dead = dead_of(s0 + warp);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        const uint32_t next = dead_of(s0 + warp + (i + 1) * kWarps);
        fetch(s0 + warp + i * kWarps, i, dead);
        dead = next;
    }

    for (int c = threadIdx.x; c < MT * 16 * (D / 8); c += kThreads) {
        const int r = c / (D / 8), piece = c % (D / 8);
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows)
            u = *reinterpret_cast<const uint4*>(p.q + b * p.qs[0] + (long)(kv_head * p.group + r % p.group) * p.qs[1] + (long)(r / p.group) * p.qs[2] + piece * 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place<D>(sQ, r, piece)), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
    }
    __syncthreads();

    // this thread's rows: two per tile of 16
    int first[MT][2], behind[MT][2], pos[MT][2];
    const float* bias[MT][2];
    float m[MT][2], l[MT][2], o[MT][D / 8][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = t * 16 + h * 8 + lane / 4, i = r / p.group;
            first[t][h] = r < rows ? plan.first[i] : 0;
            behind[t][h] = r < rows ? plan.behind[i] : 0;
            pos[t][h] = plan.start + i;
            bias[t][h] = GEN && p.R >= 0 && r < rows ? p.bias + (long)(kv_head * p.group + r % p.group) * (2 * p.R + 1) + p.R : nullptr;
            m[t][h] = -INFINITY;
            l[t][h] = 0.f;
        }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][d][e] = 0.f;

    const int mat = lane >> 3, row8 = lane & 7;
    uint32_t qf[MT == 1 ? D / 16 : 1][4];
    if (MT == 1)
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) ldmatrix4<false>(place<D>(sQ, (mat & 1) * 8 + row8, kk * 2 + (mat >> 1)), qf[kk]);

    int slot = 0;
    for (int step = s0 + warp; step < s1; step += kWarps) {
        copy_wait<kStages - 2>();
        __syncwarp();               // and all lanes are through with the slot of the step before, which the next fetch overwrites
        const uint32_t next = dead_of(step + kStages * kWarps);
        fetch(step + (kStages - 1) * kWarps, (slot + kStages - 1) % kStages, dead);
        dead = next;
        const uint32_t tk = ring + slot * (2 * F::kTileBytes), tv = tk + F::kTileBytes;
        float s[MT][2][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][0][e] = s[t][1][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t kf[4];
            ldmatrix4<false>(place<D>(tk, (mat >> 1) * 8 + row8, kk * 2 + (mat & 1)), kf);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t a[4];
                if (MT > 1) ldmatrix4<false>(place<D>(sQ, t * 16 + (mat & 1) * 8 + row8, kk * 2 + (mat >> 1)), a);
                mma<BF16>(s[t][0], MT == 1 ? qf[kk] : a, kf[0], kf[1]);
                mma<BF16>(s[t][1], MT == 1 ? qf[kk] : a, kf[2], kf[3]);
            }
        }
        const int key0 = k_lo + step * kStep + (lane & 3) * 2;         // element e of tile n: key key0 + 8 n + (e & 1), row half e >> 1
        uint32_t pf[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            bool small = true;
            if (GEN && p.cap.out != 0.f) {
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(s[t][0][e]), fabsf(s[t][1][e])));
                small = __all_sync(0xffffffffu, top <= p.cap.small);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int h = e >> 1, key = key0 + 8 * n + (e & 1);
                    float y = s[t][n][e];
                    if (GEN && p.cap.out != 0.f) y = small ? cap_small(p.cap, make_float2(y, 0.f)).x : cap_any(p.cap, y);
                    else y *= p.scale_log2;
                    const bool sees = key >= first[t][h] && key < behind[t][h];
                    if (GEN && p.R >= 0 && sees) y += bias[t][h][max(-p.R, min(p.R, key - pos[t][h]))] * kLog2e;
                    s[t][n][e] = sees ? y : -INFINITY;
                }
            float grown[2];
            bool any = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = fmaxf(fmaxf(s[t][0][2 * h], s[t][0][2 * h + 1]), fmaxf(s[t][1][2 * h], s[t][1][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                grown[h] = fmaxf(m[t][h], x);
                any |= grown[h] > m[t][h];
            }
            if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float alpha = grown[h] > m[t][h] ? exp2f(m[t][h] - grown[h]) : 1.f;
                    m[t][h] = grown[h];
                    l[t][h] *= alpha;
#pragma unroll
                    for (int d = 0; d < D / 8; ++d) {
                        o[t][d][2 * h] *= alpha;
                        o[t][d][2 * h + 1] *= alpha;
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float base = m[t][h] == -INFINITY ? 0.f : m[t][h];
                    const float e0 = exp2f(s[t][n][2 * h] - base), e1 = exp2f(s[t][n][2 * h + 1] - base);
                    l[t][h] += e0 + e1;
                    pf[t][2 * n + h] = pack2<BF16>(e0, e1);         // rounded for the product: half a step of the operands' type
                }
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t vf[4];
            ldmatrix4<true>(place<D>(tv, (mat & 1) * 8 + row8, 2 * d + (mat >> 1)), vf);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                mma<BF16>(o[t][2 * d], pf[t], vf[0], vf[1]);
                mma<BF16>(o[t][2 * d + 1], pf[t], vf[2], vf[3]);
            }
        }
        slot = (slot + 1) % kStages;
    }
    copy_wait<0>();
    __syncthreads();

    // the warps' results, joined by the threads in the warps' order
    float* mine = reinterpret_cast<float*>(smem + warp * F::kRing);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = t * 16 + h * 8 + lane / 4;
            float sum = l[t][h];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if ((lane & 3) == 0) {
                stats[warp][r][0] = m[t][h];
                stats[warp][r][1] = sum;
            }
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
                *reinterpret_cast<float2*>(mine + r * D + d * 8 + (lane & 3) * 2) = make_float2(o[t][d][2 * h], o[t][d][2 * h + 1]);
        }
    __syncthreads();
    for (int c = threadIdx.x; c < rows * (D / 2); c += kThreads) {
        const int r = c / (D / 2), d = c % (D / 2) * 2;
        float top = -INFINITY, sum = 0.f;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[w][r][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float a = stats[w][r][0] == -INFINITY ? 0.f : exp2f(stats[w][r][0] - top);
            const float2 x = *reinterpret_cast<const float2*>(reinterpret_cast<float*>(smem + w * F::kRing) + r * D + d);
            sum += a * stats[w][r][1];
            acc.x += a * x.x;
            acc.y += a * x.y;
        }
        const int head = kv_head * p.group + r % p.group, i = r / p.group;
        if (p.splits == 1) {
            const bool none = sum == 0.f;
            const float inv = none ? 0.f : 1.f / sum;
            *reinterpret_cast<uint32_t*>(p.out + (((long)b * p.q_len + i) * p.q_heads + head) * D + d) = none ? 0u : pack2<BF16>(acc.x * inv, acc.y * inv);
            if (d == 0) p.lse[((long)b * p.q_heads + head) * kTile + i] = none ? INFINITY : top + log2f(sum);
        } else {        // [batch, key heads, rows, splits]: D outputs, maximum, sum
            float* part = p.partials + ((((long)b * p.k_heads + kv_head) * rows + r) * p.splits + split) * (D + 2);
            *reinterpret_cast<float2*>(part + d) = acc;
            if (d == 0) {
                part[D] = top;
                part[D + 1] = sum;
            }
        }
    }
    if (split == 0)         // the rest of the statistics' tile says "no such query" to the backward
        for (int c = threadIdx.x; c < p.group * (kTile - p.q_len); c += kThreads) {
            const int g = c / (kTile - p.q_len), i = p.q_len + c % (kTile - p.q_len);
            p.lse[((long)b * p.q_heads + kv_head * p.group + g) * kTile + i] = INFINITY;
        }
}

// One CTA a row: eight warps add the splits' results, each its own in their order, then the warps' sums in theirs.
constexpr int kMaxSplits = 256, kJoinThreads = 256;
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) few_join_kernel(const float* __restrict__ partials, uint16_t* __restrict__ out, float* __restrict__ lse, int rows,
                                                       int splits, int group, int q_len, int q_heads) {
    __shared__ float weight[kMaxSplits], red[kJoinThreads / 32], sums[kJoinThreads / 32][D + 1];
    const long w = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, s0 = threadIdx.x;
    const int r = (int)(w % rows), k_heads = q_heads / group;
    const long bk = w / rows;
    const int head = (int)(bk % k_heads) * group + r % group, i = r / group;
    const long b = bk / k_heads;
    const float* part = partials + w * splits * (D + 2);
    const float mine = s0 < splits ? part[(long)s0 * (D + 2) + D] : -INFINITY;
    float top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int i8 = 1; i8 < kJoinThreads / 32; ++i8) top = fmaxf(top, red[i8]);
    if (s0 < splits) weight[s0] = mine == -INFINITY ? 0.f : exp2f(mine - top);
    __syncthreads();
    float sum = 0.f;
    float2 acc[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int s = warp; s < splits; s += kJoinThreads / 32) {
        const float* q = part + (long)s * (D + 2);
        const float a = weight[s];
        sum += a * q[D + 1];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            const float2 x = *reinterpret_cast<const float2*>(q + c * 64 + lane * 2);
            acc[c].x += a * x.x;
            acc[c].y += a * x.y;
        }
    }
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        sums[warp][c * 64 + lane * 2] = acc[c].x;
        sums[warp][c * 64 + lane * 2 + 1] = acc[c].y;
    }
    if (lane == 0) sums[warp][D] = sum;
    __syncthreads();
    const int d = threadIdx.x * 2;
    if (d < D) {
        float2 o2 = make_float2(0.f, 0.f);
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < kJoinThreads / 32; ++k) {
            o2.x += sums[k][d];
            o2.y += sums[k][d + 1];
            sum += sums[k][D];
        }
        const bool none = sum == 0.f;
        const float inv = none ? 0.f : 1.f / sum;
        *reinterpret_cast<uint32_t*>(out + ((b * q_len + i) * q_heads + head) * D + d) = none ? 0u : pack2<BF16>(o2.x * inv, o2.y * inv);
        if (d == 0) lse[(b * q_heads + head) * kTile + i] = none ? INFINITY : top + log2f(sum);
    }
}

// CTAs that share the keys of a sample and key head.  Two fit an SM; a wave of them takes what its longest share does, about 1.5 us for 64
// keys (of two CTAs at the memory's rate) and 3 us besides: the number of shares with the cheapest waves.
int few_splits(const tt_ranges_args& a, int sms) {
    const long units = (long)a.batch * a.k_heads, slots = 2L * sms, blocks = (a.kv_len + 63) / 64;
    int best = 1;
    double least = 1e300;
    for (int n = 1; n <= kMaxSplits && n <= blocks; ++n) {
        const double cost = (double)((units * n + slots - 1) / slots) * (1.5 * (double)((blocks + n - 1) / n) + 3.0) + (n > 1 ? 4.0 : 0.0);
        if (cost < least) {
            least = cost;
            best = n;
        }
    }
    return best;
}

template <int D, bool BF16, bool GEN, int MT>
int launch(const tt_ranges_args& a, const FewParams& p, int dev, cudaStream_t st) {
    auto kern = few_kernel<D, BF16, GEN, MT>;
    static bool configured[64] = {false};         // per device: the attribute belongs to the device's context
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<D, MT>::kSmem);
        if (e != cudaSuccess) return tt_record_cuda(e);
        configured[dev] = true;
    }
    kern<<<dim3(p.splits, a.k_heads, a.batch), kThreads, Few<D, MT>::kSmem, st>>>(p);
    TT_CHECK_LAUNCH();
    if (p.splits > 1) {
        const int rows = p.group * p.q_len;
        const long total = (long)a.batch * a.k_heads * rows;
        if (total > INT_MAX) return TT_ERR_LIMIT;
        few_join_kernel<D, BF16><<<(unsigned)total, kJoinThreads, 0, st>>>(p.partials, p.out, p.lse, rows, p.splits, p.group, p.q_len, p.q_heads);
        TT_CHECK_LAUNCH();
    }
    return TT_OK;
}

template <int D, bool BF16>
int pick(const tt_ranges_args& a, const FewParams& p, bool gen, int dev, cudaStream_t st) {
    if (p.group * p.q_len <= 16) return gen ? launch<D, BF16, true, 1>(a, p, dev, st) : launch<D, BF16, false, 1>(a, p, dev, st);
    return gen ? launch<D, BF16, true, 2>(a, p, dev, st) : launch<D, BF16, false, 2>(a, p, dev, st);
}

}  // namespace

bool tt_ranges_few_rows(const tt_ranges_args& a) { return a.out32 == nullptr && (long)(a.q_heads / a.k_heads) * a.q_len <= kMaxRows; }

extern "C" long tt_attn_ranges_fwd_floats(const tt_ranges_args* a) {
    if (tt_ranges_check(a) != TT_OK || !tt_ranges_few_rows(*a)) return 0;
    const int splits = few_splits(*a, tt_device().sms);
    return splits == 1 ? 0 : (long)a->batch * a->q_heads * a->q_len * splits * (a->head_dim + 2);
}

int tt_attn_ranges_few(const tt_ranges_args& a, cudaStream_t st) {
    const tt_device_info dev = tt_device();
    for (const void* x : {a.q, a.k, a.v, (const void*)a.partials})
        if ((uintptr_t)x & 15) return TT_ERR_ARG;
    FewParams p;
    // rows start at 16-byte boundaries; the stride of a dimension of one is never stepped over
    const auto aligned = [](const long* s, int batch, int heads, int tokens) {
        return !((batch > 1 && s[0] & 7) || (heads > 1 && s[1] & 7) || (tokens > 1 && s[2] & 7));
    };
    if (!aligned(a.q_stride, a.batch, a.q_heads, a.q_len) || !aligned(a.k_stride, a.batch, a.k_heads, a.kv_len) ||
        !aligned(a.v_stride, a.batch, a.k_heads, a.kv_len))
        return TT_ERR_ARG;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a.q_stride[i];
        p.ks[i] = a.k_stride[i];
        p.vs[i] = a.v_stride[i];
    }
    p.plan = plan_ptr(a);
    p.q = (const uint16_t*)a.q;
    p.k = (const uint16_t*)a.k;
    p.v = (const uint16_t*)a.v;
    p.out = (uint16_t*)a.out;
    p.lse = a.lse;
    p.partials = a.partials;
    p.bias = a.bias;
    p.q_len = a.q_len;
    p.q_heads = a.q_heads;
    p.k_heads = a.k_heads;
    p.group = a.q_heads / a.k_heads;
    p.R = a.max_distance;
    p.splits = few_splits(a, dev.sms);
    if (p.splits > 1 && a.partials == nullptr) return TT_ERR_ARG;
    p.scale_log2 = a.scale * kLog2e;
    p.cap = make_cap(a.scale, a.softcap);
    const bool gen = a.softcap > 0.f || a.max_distance >= 0, bf = a.dtype == TT_BF16;
    if (a.head_dim == 128) return bf ? pick<128, true>(a, p, gen, dev.dev, st) : pick<128, false>(a, p, gen, dev.dev, st);
    return bf ? pick<64, true>(a, p, gen, dev.dev, st) : pick<64, false>(a, p, gen, dev.dev, st);
}
