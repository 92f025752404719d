// The attention of attn_ranges_fwd.cu for few queries over long keys (new tokens over a cache): at most 32 rows of a key head's group.
//
// What bounds it is reading keys and values once, so the steps of 16 keys of all samples and key heads, counted as the samples' runs have them, are
// dealt to the CTAs in equal shares, and a share's steps to its four warps.  Every warp streams its keys and values through a ring of its own in
// shared memory (16-byte asynchronous copies; three steps of 8 KB a warp at heads of 128, 96 KB a CTA, of which two steps are under way while the third is
// worked on: 64 KB) and keeps running maxima, sums and outputs
// of its 16 or 32 rows (the queries of all heads of the group, so that shared keys are read once) in registers; the products are mma.sync of 16 x 8 x
// 16, which a tile of 128 queries on tcgen05 would leave seven eighths empty.  Warps are joined through shared memory, CTAs by a second kernel in a
// fixed order.
//
// Measured: one token each of eight samples over up to 8192 keys (32 heads of 128 on 8) 43.7 us, 4.7 TB/s; of 76 samples over up to 8192 keys 305 us
// (6.7 TB/s).  The rest is the first loads of every share, the border of heads inside some of them, and the join.
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
    int q_len, q_heads, k_heads, group, R, batch, ctas;        // ctas 0: one CTA for each sample and key head, results written by it
    float scale_log2;
    Cap cap;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");     // zeros where not in
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// (ordered among the copies' waits and the warp's barriers, as they are volatile too; the products between them are free to move)
template <bool TRANS> __device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t* r) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
template <bool BF16> __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Rows of D 16-bit elements in shared memory, their 16-byte pieces exchanged by row so that eight rows' same piece lies in eight banks
template <int D> __device__ __forceinline__ uint32_t place(uint32_t base, int row, int piece) {
    return base + row * (D * 2) + ((piece ^ (row & 7)) << 4);
}

// of shared steps; more samples are many CTAs by themselves (one key head, 4 rows, us: 128 samples in shares against 129 without, 1024 keys 24.6 / 24.6, 4096
// 65.5 / 65.5, 8192 114.7 / 110.6)
constexpr int kMaxBatch = 128;
static_assert(kMaxBatch <= kThreads, "a thread a sample");

template <int D, int MT> struct Few {
    static constexpr int kTileBytes = kStep * D * 2;                        // 16 keys
    static constexpr int kRing = kStages * 2 * kTileBytes;                  // of one warp
    static constexpr int kQ = MT * 16 * D * 2;
    static constexpr int kSmem = kWarps * kRing + kQ;
    static_assert(kRing >= MT * 16 * D * 4, "a warp's outputs are joined in its ring");
};

constexpr int kMinSteps = 2 * kWarps;   // of a share

// The keys that any of a sample's queries sees, from a multiple of a step on
__device__ __forceinline__ void run_of(const PlanPtr& plan, int b, int* lo, int* hi) {
    const int4 r = plan.sample(b).q_tiles[0];
    *lo = r.x < r.y ? r.x / kStep * kStep : 0;
    *hi = r.x < r.y ? r.y : 0;
}

// How the steps of all samples and key heads are dealt to the CTAs: in equal shares, sample after sample and head after head.  A share that
// ends inside a head's steps goes on with the next head's, so share c has at most one piece of unit u (sample and head), and pieces are
// numbered u + c.
struct Shares {
    long before[kMaxBatch + 1];         // steps of the samples ahead
    long warps[kMaxBatch / 32];         // of 32 samples
    int ctas;
    __device__ void count(const PlanPtr& plan, int batch, int k_heads, int most) {       // whole CTA, of kMaxBatch threads or more
        const int b = threadIdx.x, lane = b & 31, warp = b >> 5;
        long sum = 0;
        if (b < batch) {
            int lo, hi;
            run_of(plan, b, &lo, &hi);
            sum = (long)((hi - lo + kStep - 1) / kStep) * k_heads;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 31 && warp < kMaxBatch / 32) warps[warp] = sum;
        __syncthreads();
        long total = 0;
#pragma unroll
        for (int w = 0; w < kMaxBatch / 32; ++w) {
            if (w < warp) sum += warps[w];
            total += warps[w];
        }
        if (b < batch) before[b + 1] = sum;
        if (b == 0) {
            before[0] = 0;
            const long wanted = (total + kMinSteps - 1) / kMinSteps;
            ctas = (int)(wanted < most ? wanted : most);
            samples = batch;
        }
        __syncthreads();
    }
    __device__ __forceinline__ long first_of(int c) const { return before[samples] * c / ctas; }
    __device__ __forceinline__ int sample_of(long step) const {        // the last with no more than `step` steps ahead
        int l = 0, h = samples;
        while (l + 1 < h) {
            const int m = (l + h) >> 1;
            if (before[m] <= step) l = m;
            else h = m;
        }
        return l;
    }
    __device__ __forceinline__ int share_of(long step) const {
        int c = (int)(step * ctas / before[samples]);
        while (c + 1 < ctas && first_of(c + 1) <= step) ++c;
        return c;
    }
    int samples;
};

// The rest of the statistics' tile says "no such query" to the backward.
__device__ __forceinline__ void write_padding(float* lse, long b, int q_heads, int head0, int heads, int q_len) {
    for (int c = threadIdx.x; c < heads * (kTile - q_len); c += blockDim.x)
        lse[(b * q_heads + head0 + c / (kTile - q_len)) * kTile + q_len + c % (kTile - q_len)] = INFINITY;
}

template <int D, bool BF16, bool GEN, int MT>
__global__ void __launch_bounds__(kThreads) few_kernel(const FewParams p) {
    using F = Few<D, MT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float stats[kWarps][kMaxRows][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ Shares shares;
    const int rows = p.group * p.q_len;             // row r: query r / group of head r % group
    const uint32_t sQ = sm100::smem_u32(smem) + kWarps * F::kRing, ring = sm100::smem_u32(smem) + warp * F::kRing;
    const bool whole = p.ctas == 0;
    long at_step = 0, end_step = 1;
    if (!whole) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");        // the join: it waits for this grid's end before it reads a result
        shares.count(p.plan, p.batch, p.k_heads, p.ctas);
        if ((int)blockIdx.x >= shares.ctas) return;
        at_step = shares.first_of(blockIdx.x);
        end_step = shares.first_of(blockIdx.x + 1);
    }
    while (at_step < end_step) {
        int b, kv_head, s0, s1, k_lo, k_hi;
        if (whole) {
            b = blockIdx.x / p.k_heads;
            kv_head = blockIdx.x - b * p.k_heads;
            run_of(p.plan, b, &k_lo, &k_hi);
            s0 = 0;
            s1 = (k_hi - k_lo + kStep - 1) / kStep;
            at_step = end_step;
        } else {
            b = shares.sample_of(at_step);
            run_of(p.plan, b, &k_lo, &k_hi);
            const int steps = (k_hi - k_lo + kStep - 1) / kStep;
            const long in_sample = at_step - shares.before[b];
            kv_head = (int)(in_sample / steps);
            s0 = (int)(in_sample - (long)kv_head * steps);
            s1 = (int)min((long)steps, s0 + (end_step - at_step));
            at_step += s1 - s0;
        }
        const PlanView plan = p.plan.sample(b);
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
            if (whole) {
                const bool none = sum == 0.f;
                const float inv = none ? 0.f : 1.f / sum;
                *reinterpret_cast<uint32_t*>(p.out + (((long)b * p.q_len + i) * p.q_heads + head) * D + d) = none ? 0u : pack2<BF16>(acc.x * inv, acc.y * inv);
                if (d == 0) p.lse[((long)b * p.q_heads + head) * kTile + i] = none ? INFINITY : top + log2f(sum);
            } else {        // [share + sample and key head, rows]: D outputs, maximum, sum
                float* part = p.partials + (((long)b * p.k_heads + kv_head + blockIdx.x) * rows + r) * (D + 2);
                *reinterpret_cast<float2*>(part + d) = acc;
                if (d == 0) {
                    part[D] = top;
                    part[D + 1] = sum;
                }
            }
        }
        if (whole) write_padding(p.lse, b, p.q_heads, kv_head * p.group, p.group, p.q_len);
        __syncthreads();            // the rings and the queries' tile are free for the next sample or head
    }
}

// W warps a row, 8 / W rows a CTA: every warp adds its share of the row's pieces in their order, then the warps' sums are added in theirs.
constexpr int kJoinThreads = 256;
template <int D, bool BF16, int W>
__global__ void __launch_bounds__(kJoinThreads) few_join_kernel(const FewParams p) {
    __shared__ Shares shares;
    __shared__ float sums[W > 1 ? W : 1][D + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first_piece = W > 1 ? warp : 0;
    const int rows = p.group * p.q_len;
    const long row = (long)blockIdx.x * (8 / W) + (W > 1 ? 0 : warp);
    shares.count(p.plan, p.batch, p.k_heads, p.ctas);
    if (row >= (long)p.batch * p.k_heads * rows) return;        // (W == 1: whole warps, with no barrier to come)
    const int unit = (int)(row / rows), r = (int)(row - (long)unit * rows);
    const int b = unit / p.k_heads, kv_head = unit - b * p.k_heads, head = kv_head * p.group + r % p.group, i = r / p.group;
    const long steps = (shares.before[b + 1] - shares.before[b]) / p.k_heads, first = shares.before[b] + kv_head * steps;
    const int c0 = steps > 0 ? shares.share_of(first) : 0, n = steps > 0 ? shares.share_of(first + steps - 1) - c0 + 1 : 0;
    const float* part = p.partials + ((long)(unit + c0) * rows + r) * (D + 2);
    const long next = (long)rows * (D + 2);         // of the next piece
    asm volatile("griddepcontrol.wait;" ::: "memory");          // the kernel ahead has ended and its results are in memory
    // the first piece, often a warp's only one, is read with the maxima
    float m1 = -INFINITY, l1 = 0.f;
    float2 acc[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
    if (first_piece < n) {
        const float* q = part + first_piece * next;
        m1 = q[D];
        l1 = q[D + 1];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] = *reinterpret_cast<const float2*>(q + c * 64 + lane * 2);
    }
    float top = -INFINITY;
    for (int s = lane; s < n; s += 32) top = fmaxf(top, part[s * next + D]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float a1 = m1 == -INFINITY ? 0.f : exp2f(m1 - top);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(a1 * acc[c].x, a1 * acc[c].y);
    float sum = lane == 0 ? a1 * l1 : 0.f;
    for (int s0 = first_piece + W; s0 < n; s0 += 32 * W) {
        const int mine = s0 + lane * W, count = min(32, (n - s0 + W - 1) / W);
        float weight = 0.f;
        if (mine < n) {
            const float m = part[mine * next + D];
            weight = m == -INFINITY ? 0.f : exp2f(m - top);
            sum += weight * part[mine * next + D + 1];
        }
#pragma unroll 8
        for (int k = 0; k < count; ++k) {
            const float* q = part + (s0 + k * W) * next;
            const float a = __shfl_sync(0xffffffffu, weight, k);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const float2 x = *reinterpret_cast<const float2*>(q + c * 64 + lane * 2);
                acc[c].x += a * x.x;
                acc[c].y += a * x.y;
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (W > 1) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            sums[warp][c * 64 + lane * 2] = acc[c].x;
            sums[warp][c * 64 + lane * 2 + 1] = acc[c].y;
        }
        if (lane == 0) sums[warp][D] = sum;
        __syncthreads();
        if (warp > 0) return;
        sum = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            sum += sums[k][D];
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                acc[c].x += sums[k][c * 64 + lane * 2];
                acc[c].y += sums[k][c * 64 + lane * 2 + 1];
            }
        }
    }
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : 1.f / sum;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
        *reinterpret_cast<uint32_t*>(p.out + (((long)b * p.q_len + i) * p.q_heads + head) * D + c * 64 + lane * 2) =
            none ? 0u : pack2<BF16>(acc[c].x * inv, acc[c].y * inv);
    float* const lse = p.lse + ((long)b * p.q_heads + head) * kTile;
    if (lane == 0) lse[i] = none ? INFINITY : top + log2f(sum);
    if (i == 0)         // the rest of the statistics' tile says "no such query" to the backward
        for (int c = p.q_len + lane; c < kTile; c += 32) lse[c] = INFINITY;
}

// CTAs of equal shares, two of which fit an SM; 0: a CTA for each sample and key head, which needs no join.  Those leave a share of the device idle
// in their last round, for as long as a sample's keys take; shares cost a second kernel and a few more loads, ~6 us and more with
// many rows.  Measured, one CTA each against shares, in us (heads of 128, 4 rows): 8 units of 512 keys 8.4 / 10.0, of 1024 12.4 / 11.2, of
// 2048 19.3 / 12.0; 64 units of 512 11.4 / 14.5, of 1024 17.1 / 17.4, of 4096 50.7 / 29.5; 256 units of 1024 25.4 / 30.4, of 8192 139 / 135;
// 304 units of 4096 110 / 87; 512 units of 2048 75 / 77.  With 32 rows: 64 units of 1024 28.4 / 31.4, of 4096 77 / 46; 512 of 2048 108 / 118.
int few_ctas(const tt_ranges_args& a, int sms) {
    const long units = (long)a.batch * a.k_heads, slots = 2L * sms, rounds = (units + slots - 1) / slots;
    const long idle_keys = a.kv_len * (rounds * slots - units) / (rounds * slots);
    if (idle_keys < 768 + units * (a.q_heads / a.k_heads) * a.q_len / 24 || a.batch > kMaxBatch) return 0;
    return (int)slots;
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
    const long units = (long)a.batch * a.k_heads, rows = (long)p.group * p.q_len;
    if (units * rows > INT_MAX) return TT_ERR_LIMIT;
    kern<<<p.ctas ? p.ctas : (int)units, kThreads, Few<D, MT>::kSmem, st>>>(p);
    TT_CHECK_LAUNCH();
    if (p.ctas) {
        // started while the pieces are still computed, so that neither its launch nor the counting of the shares is waited for
        const bool wide = units * rows <= 4L * tt_device().sms;
        cudaLaunchAttribute early = {};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(wide ? units * rows : (units * rows + 7) / 8));
        cfg.blockDim = dim3(kJoinThreads);
        cfg.stream = st;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        const cudaError_t e = wide ? cudaLaunchKernelEx(&cfg, few_join_kernel<D, BF16, 8>, p) : cudaLaunchKernelEx(&cfg, few_join_kernel<D, BF16, 1>, p);
        if (e != cudaSuccess) return tt_record_cuda(e);
    }
    return TT_OK;
}

template <int D, bool BF16>
int pick(const tt_ranges_args& a, const FewParams& p, bool gen, int dev, cudaStream_t st) {
    if (p.group * p.q_len <= 16) return gen ? launch<D, BF16, true, 1>(a, p, dev, st) : launch<D, BF16, false, 1>(a, p, dev, st);
    return gen ? launch<D, BF16, true, 2>(a, p, dev, st) : launch<D, BF16, false, 2>(a, p, dev, st);
}

}  // namespace

// At most 32 rows of a group (beyond them, and from 17 on over few short caches, the kernel for tiles is the faster one).  In us, tiles against this:
// 64 units of 8192 keys, heads of 128, 32 rows 106 / 76, 4 rows 106 / 46; 8 units of 1024 keys, 16 rows 14.5 / 13.5, 32 rows 14.5 / 20.2; 64 units of
// 1024, 32 rows 20.7 / 28.4, of 4096 57 / 46; 256 units of 256, 32 rows 29 / 21.  Heads of 64, 32 rows: 64 units of 1024 19.0 / 18.2.
// Beyond them long caches are far from their floor, as the kernel for tiles gives one CTA two heads' tiles and all keys: eight heads on one key head over 65536
// keys, 4 new tokens 43 us, 5 776; 32 heads on 8 key heads over as many, 8 new tokens 72, 9 778, 128 789.
bool tt_ranges_few_rows(const tt_ranges_args& a) {
    const long rows = (long)(a.q_heads / a.k_heads) * a.q_len, units = (long)a.batch * a.k_heads;
    const bool short_caches = rows > 16 && a.head_dim == 128 && a.kv_len <= 1536 && 2 * units <= tt_device().sms;
    return a.out32 == nullptr && rows <= kMaxRows && !short_caches;
}

extern "C" long tt_attn_ranges_fwd_floats(const tt_ranges_args* a) {
    if (tt_ranges_check(a) != TT_OK || !tt_ranges_few_rows(*a)) return 0;
    const int ctas = few_ctas(*a, tt_device().sms);
    return ctas == 0 ? 0 : ((long)a->batch * a->k_heads + ctas) * (a->q_heads / a->k_heads) * a->q_len * (a->head_dim + 2);
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
    p.batch = a.batch;
    p.ctas = few_ctas(a, dev.sms);
    if (p.ctas && a.partials == nullptr) return TT_ERR_ARG;
    p.scale_log2 = a.scale * kLog2e;
    p.cap = make_cap(a.scale, a.softcap);
    const bool gen = a.softcap > 0.f || a.max_distance >= 0, bf = a.dtype == TT_BF16;
    if (a.head_dim == 128) return bf ? pick<128, true>(a, p, gen, dev.dev, st) : pick<128, false>(a, p, gen, dev.dev, st);
    return bf ? pick<64, true>(a, p, gen, dev.dev, st) : pick<64, false>(a, p, gen, dev.dev, st);
}
