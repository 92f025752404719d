// Shared by the attention kernels in which every query sees one run of the keys (attn_ranges_*.cu).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "sm100.cuh"
#include "teletron_b200.h"

namespace ranges {

constexpr int kTile = TT_RANGES_TILE;
constexpr float kLog2e = 1.4426950408889634f;
// The bias table lies in shared memory with its end values repeated for kPad entries, so that a tile that is not wholly beyond the
// largest distance needs no clamp: its distances reach at most 127 + 31 past it.
constexpr int kPad = 160;

// A plan's parts for one sample.
struct PlanView {
    const int4* q_tiles;
    const uint4* dead;
    const int2* k_tiles;
    const int* dirty;
    const int *first, *behind;
    int start;
};

struct PlanPtr {
    const int* base;
    tt_ranges_layout at;
    int q_len, q_tiles, k_tiles;
    __device__ __forceinline__ PlanView sample(int b) const {
        PlanView v;
        v.q_tiles = reinterpret_cast<const int4*>(base + at.q_tiles) + (long)b * q_tiles;
        v.dead = reinterpret_cast<const uint4*>(base + at.dead) + (long)b * k_tiles;
        v.k_tiles = reinterpret_cast<const int2*>(base + at.k_tiles) + (long)b * k_tiles;
        v.dirty = base + at.dirty + (long)b * k_tiles;
        v.first = base + at.first + (long)b * q_len;
        v.behind = base + at.behind + (long)b * q_len;
        v.start = base[at.start + b];
        return v;
    }
};

inline PlanPtr plan_ptr(const tt_ranges_args& a) {
    PlanPtr p;
    p.base = a.plan;
    tt_key_ranges_layout(a.batch, a.q_len, a.kv_len, &p.at);
    p.q_len = a.q_len;
    p.q_tiles = (a.q_len + kTile - 1) / kTile;
    p.k_tiles = (a.kv_len + kTile - 1) / kTile;
    return p;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
template <bool BF16> __device__ __forceinline__ float2 unpack2(uint32_t u) {
    if (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// Instruction descriptor of kind::f16 with fp32 accumulation; both operands bf16 or both fp16.
template <bool BF16> __host__ __device__ constexpr uint32_t idesc(int m, int n, bool a_mn, bool b_mn) {
    const uint32_t d = sm100::idesc_bf16(m, n, a_mn, b_mn);
    return BF16 ? d : d & ~((1u << 7) | (1u << 10));
}

// The wait of a whole warp: all lanes get the same answer, so that none is left behind at a later warp-wide instruction.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, sm100::mbar_wait(bar, parity, abort_flag));
}

// Grids are (tiles, heads, samples), the long runs of causal masks first.  Where all heads' long runs should come ahead of all short ones (a causal
// mask: the last heads' long ones would be started when other CTAs run dry) the tiles are the slowest index instead of the fastest, in which
// CTAs that run together share a head's operands.
struct Order {
    int tiles_last;
    dim3 grid(int tiles, int heads, int batch) const { return tiles_last ? dim3(heads, batch, tiles) : dim3(tiles, heads, batch); }
    __device__ __forceinline__ int tile(int x, int, int z) const { return tiles_last ? z : x; }
    __device__ __forceinline__ int head(int x, int y, int) const { return tiles_last ? x : y; }
    __device__ __forceinline__ int sample(int, int y, int z) const { return tiles_last ? y : z; }
    __device__ __forceinline__ int tiles() const { return tiles_last ? (int)gridDim.z : (int)gridDim.x; }
};
inline Order make_order(const tt_ranges_args& a, int tiles) { return Order{a.causal && tiles <= 65535 ? 1 : 0}; }

// The items of a CTA: its own block index, then ones of the launch that have not been started, so that an item's first loads and products
// run behind the last one's.  The loading warp asks for the next item when all of one's loads are under way (at its beginning, long items were
// claimed by CTAs that were busy while others ran dry: 21 % on a causal mask's dK dV); every role reads the answer when it is through.
struct Queue {
    static constexpr int kBytes = 64;               // two answers of 16 bytes, two pairs of barriers
    uint32_t base;
    int n = 0;                                      // items begun
    __device__ __forceinline__ uint32_t answer() const { return base + 16u * (n & 1); }
    __device__ __forceinline__ uint32_t full() const { return base + 32u + 8u * (n & 1); }
    __device__ __forceinline__ uint32_t empty() const { return base + 48u + 8u * (n & 1); }
    __device__ __forceinline__ void init(int readers) const {         // one thread
        for (int i = 0; i < 2; ++i) {
            sm100::mbar_init(base + 32u + 8u * i, 1);
            sm100::mbar_init(base + 48u + 8u * i, readers);
        }
    }
    // the loading warp, once per item; its `lead` lane asks
    __device__ __forceinline__ bool ask(bool lead, volatile int* abort_flag) const {
        if (!warp_wait(empty(), (uint32_t)(n >> 1) & 1u ^ 1u, abort_flag)) return false;
        if (lead) {
            sm100::fence_proxy_async();             // the readers of the answer before last were ordinary loads
            sm100::mbar_arrive_expect_tx(full(), 16);
            sm100::launch_take(answer(), full());
        }
        return true;
    }
    __device__ __forceinline__ uint32_t parity() const { return (uint32_t)(n >> 1) & 1u; }
    // the next item's block index, once full() has completed; a reader is a whole warp, of which one lane arrives, or a single thread
    template <bool WARP> __device__ __forceinline__ bool next(bool arrive, int* x, int* y, int* z) {
        const bool ok = sm100::launch_taken(answer(), x, y, z);
        if (WARP) __syncwarp();
        if (arrive) sm100::mbar_arrive(empty());
        ++n;
        return ok;
    }
};

// Bits [lo, hi) of a 32-bit word, for any lo and hi.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
    const uint32_t below_hi = hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u;
    const uint32_t below_lo = lo >= 32 ? 0xffffffffu : lo <= 0 ? 0u : (1u << lo) - 1u;
    return below_hi & ~below_lo;
}

// Clears the rows of a tile (slabs of [128 rows x 128 bytes], as TMA wrote them) whose bit is set; one warp.
__device__ __forceinline__ void clear_rows(uint32_t tile, int slabs, uint4 bits, int lane) {
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (!(w[q] >> lane & 1u)) continue;
        for (int s = 0; s < slabs; ++s)
#pragma unroll
            for (int c = 0; c < 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + s * (kTile * 128) + (q * 32 + lane) * 128 + c * 16), "r"(0) : "memory");
    }
}

// 64 bytes of each of a warp's 32 rows to memory through 2 KB of shared memory: a lane has its row's four 16-byte pieces, and stores the pieces of
// eight rows with three others (stored by the lanes that have them, 32 rows' pieces are as many lines an instruction, and the output of two
// tiles of 128 x 128 took 5000 clocks).  `dst(row)`: where a row's 64 bytes go, or null.
template <typename F> __device__ __forceinline__ void store_rows64(uint32_t stage, int lane, const uint4* piece, F&& dst) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)), "r"(piece[q].x), "r"(piece[q].y),
                     "r"(piece[q].z), "r"(piece[q].w)
                     : "memory");
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2), q = lane & 3;
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(stage + row * 64 + ((q ^ (row >> 1 & 3)) << 4)) : "memory");
        uint4* to = reinterpret_cast<uint4*>(dst(row));
        if (to != nullptr) to[q] = v;
    }
    __syncwarp();
}

// cap tanh(scale z / cap) log2(e) of raw scores z, in the log2 domain.  Where all of a warp's scores are small against the cap the odd Taylor
// series up to the ninth power (|u| <= 0.3: the next term is below 2^-24 of the value) takes six packed multiply-adds a pair; else
// tanh u = 1 - 2 / (1 + e^2u), two special functions a score, exact to a few roundings of the cap.
struct Cap {
    float two_u, out, inv_out;      // 2 / cap * scale * log2(e); cap * log2(e), and its inverse; two_u and out 0: no cap
    float small;                    // largest |z| of the series
    float c[5];                     // its coefficients times scale * log2(e)
};
inline Cap make_cap(float scale, float softcap) {
    Cap k = {};
    if (!(softcap > 0.f)) return k;
    const double u = (double)scale / softcap, t[5] = {1.0, -1.0 / 3, 2.0 / 15, -17.0 / 315, 62.0 / 2835};
    double power = (double)scale * kLog2e;
    for (int i = 0; i < 5; ++i, power *= u * u) k.c[i] = (float)(t[i] * power);
    k.two_u = (float)(2.0 * u * kLog2e);
    k.out = softcap * kLog2e;
    k.inv_out = 1.f / k.out;
    k.small = scale != 0.f ? (float)fmin(0.3 / fabs(u), 3e38) : 3e38f;
    for (float c : k.c)
        if (!isfinite(c)) k.small = -1.f;           // a cap so far below the scale that the series has no coefficients in 32 bits
    return k;
}
__device__ __forceinline__ float2 cap_small(const Cap& k, float2 z) {
    const float2 zz = __fmul2_rn(z, z);
    float2 q = __ffma2_rn(zz, make_float2(k.c[4], k.c[4]), make_float2(k.c[3], k.c[3]));
    q = __ffma2_rn(q, zz, make_float2(k.c[2], k.c[2]));
    q = __ffma2_rn(q, zz, make_float2(k.c[1], k.c[1]));
    q = __ffma2_rn(q, zz, make_float2(k.c[0], k.c[0]));
    return __fmul2_rn(z, q);
}
__device__ __forceinline__ float cap_any(const Cap& k, float z) { return k.out * (1.f - __fdividef(2.f, 1.f + exp2f(z * k.two_u))); }
// whether the largest magnitude of N scores of every lane is one of the series
template <int N> __device__ __forceinline__ bool all_small(const Cap& k, const uint32_t* z) {
    float m = 0.f, m2 = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 4) {        // three-input maxima
        asm("max.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(__uint_as_float(z[i]))), "f"(fabsf(__uint_as_float(z[i + 1]))));
        asm("max.f32 %0, %0, %1, %2;" : "+f"(m2) : "f"(fabsf(__uint_as_float(z[i + 2]))), "f"(fabsf(__uint_as_float(z[i + 3]))));
    }
    m = fmaxf(m, m2);
    return __all_sync(0xffffffffu, m <= k.small);
}

}  // namespace ranges

// [batch, heads, tokens, head_dim] of 16-bit elements with any strides, box [box_rows, 64], 128-byte swizzle: coordinates (element, token, head, batch)
int tt_make_tmap_bhsd(CUtensorMap* out, const void* base, int batch, int heads, int tokens, int head_dim, const long* stride, int box_rows);
// validates what every entry point needs; fills in nothing
int tt_ranges_check(const tt_ranges_args* a);
// few queries (attn_ranges_few.cu)
bool tt_ranges_few_rows(const tt_ranges_args& a);
int tt_attn_ranges_few(const tt_ranges_args& a, cudaStream_t st);
