// Rotary positions of queries and keys, alone or behind an RMS norm of every head, forward and backward.
//
//   y[p0] = A (x[p0] cos t - x[p1] sin t),   y[p1] = A (x[p1] cos t + x[p0] sin t),   t = position[axis(p)] * w_p
//
// for pairs p < P of a head of D >= 2 P elements: (p, P + p) in the half layout, (2 p, 2 p + 1) in the interleaved one; elements
// from 2 P on pass.  The transpose of a rotation is the rotation by -t, so the backward of the plain form is the same kernel.
// With the norm x is replaced by x^ w, x^ = r x, r = rsqrt(mean x^2 + eps); backward, with g' the rotated-back gradient:
// dw = sum over rows of g' x^, dx = r (g' w - x^ mean(g' w x^)).
//
// No table is read: the angle of a (token, pair) is shared by all heads, so a warp forms it once per token, in 64 bits (in 32 a position of 10^5 times a
// frequency near 1 is off by up to 2^-8 of a radian), reduced to a part of a turn and spread over the lanes while the first heads'
// elements are being loaded.  The kernels are bound by memory: 2 passes over q and k forward, 3 for the norm's backward.  Measured (bf16, heads of
// 128): 24 + 24 heads of 32400 tokens, rotation there and back 252 us (6.3 TB/s), norm and rotation forward 138 (5.8), backward 199 (6.0) and 4 for
// the weights' gradients; 4 x 8192 tokens of 32 + 8 heads (fp16) 107 (6.3); eight tokens 3.4, most of it the launch.  fp32 heads of 80 with 20
// rotated elements go two elements a lane, as do all pairs in the half layout that 16 bytes do not divide (142 MB there and back in 56 us, 2.5 TB/s).
#include <cuda_fp16.h>
#include <limits.h>

#include "common.cuh"
#include "sm100.cuh"
#include "teletron_b200.h"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxD = 256;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// V elements as they are in memory
template <typename T, int V> struct Pack {
    using R = typename Raw<sizeof(T) * V>::type;
    union {
        R raw;
        T v[V];
    };
    __device__ __forceinline__ Pack() : raw() {}
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const R*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<R*>(p) = raw; }
};

// Packed arithmetic on neighbours of an array: half the instructions, which are what the kernels spend next to their loads.
template <int V, typename F2, typename F1> __device__ __forceinline__ void pairwise(F2&& two, F1&& one) {
    if (V % 2 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 2) two(e);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) one(e);
    }
}
__device__ __forceinline__ float2 at2(const float* f, int e) { return make_float2(f[e], f[e + 1]); }
__device__ __forceinline__ void put2(float* f, int e, float2 v) {
    f[e] = v.x;
    f[e + 1] = v.y;
}
// x *= y;  x += y z
template <int V> __device__ __forceinline__ void mul(float* x, const float* y) {
    pairwise<V>([&](int e) { put2(x, e, __fmul2_rn(at2(x, e), at2(y, e))); }, [&](int e) { x[e] *= y[e]; });
}
template <int V> __device__ __forceinline__ void scale(float* x, float y) {
    pairwise<V>([&](int e) { put2(x, e, __fmul2_rn(at2(x, e), make_float2(y, y))); }, [&](int e) { x[e] *= y; });
}
template <int V> __device__ __forceinline__ void add_product(float* x, const float* y, const float* z) {
    pairwise<V>([&](int e) { put2(x, e, __ffma2_rn(at2(y, e), at2(z, e), at2(x, e))); }, [&](int e) { x[e] += y[e] * z[e]; });
}

template <int V> __device__ __forceinline__ float total(float* x) {
#pragma unroll
    for (int n = V / 2; n >= 2; n /= 2)
#pragma unroll
        for (int e = 0; e < n; e += 2) put2(x, e, __fadd2_rn(at2(x, e), at2(x, e + n)));
    return V > 1 ? x[0] + x[1] : x[0];
}

// A lane's share of a head: NV chunks of V pairs, each as two vectors of V elements at off0 and off1.  In the half layout the vectors hold the
// pairs' first and second elements; in the interleaved one V / 2 whole pairs each, and full-width vectors lie one lane apart, so that a
// group of lanes reads neighbouring addresses.  Chunks behind the rotated elements pass.
template <int V, int NV, bool INTER> struct Geometry {
    static constexpr bool kWhole = INTER && V > 1;         // vectors of whole pairs
    int off0[NV], off1[NV];
    __device__ __forceinline__ Geometry(int l, int log_l, int P) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = l + (i << log_l);
            if (kWhole) {
                off0[i] = NV == 1 ? c * V : c * 2 * V;
                off1[i] = NV == 1 ? off0[i] + (V << log_l) : off0[i] + V;
            } else if (c * V < P) {
                off0[i] = INTER ? 2 * c : c * V;
                off1[i] = INTER ? 2 * c + 1 : P + c * V;
            } else {
                off0[i] = 2 * P + (c - P / V) * 2 * V;
                off1[i] = off0[i] + V;
            }
        }
    }
    // Where pair p's cos and sin lie.  A lane of the half layout takes eight neighbours: their two 16-byte halves are kept apart, so that
    // neighbouring lanes read neighbouring banks.
    __device__ __forceinline__ static int place(int p, int P) {
        return V == 8 && !INTER ? (p % 8 / 4) * ((P + 7) / 8 * 4) + p / 8 * 4 + p % 4 : p;
    }
    // cos or sin of chunk i's pairs, read from shared memory where they are used: kept in registers they cost 16 a thread, and with them a
    // third of the warps that hide the loads
    __device__ __forceinline__ void angles(uint32_t table, int i, int l, int log_l, int P, float* f) const {
        const int c = l + (i << log_l);
        if (V == 8) {
            const int second = INTER ? 1 << log_l : (P + 7) / 8;
            quad(table + 16 * c, f);
            quad(table + 16 * (c + second), f + 4);
        } else if (V == 4 && INTER) {
            two(table + 8 * c, f);
            two(table + 8 * (c + (1 << log_l)), f + 2);
        } else if (V == 4) {
            quad(table + 16 * c, f);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[e]) : "r"(table + 4 * min(c * V + e, kMaxD / 2 - 1)));
        }
    }
    __device__ __forceinline__ static void quad(uint32_t at, float* f) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]) : "r"(at));
    }
    __device__ __forceinline__ static void two(uint32_t at, float* f) { asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f[0]), "=f"(f[1]) : "r"(at)); }
};

// The pairs' first and second elements of two vectors, and back
template <typename T, int V, bool WHOLE> __device__ __forceinline__ void unpack(const Pack<T, V>& p0, const Pack<T, V>& p1, float* a, float* b) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (!WHOLE) {
            a[e] = to_f(p0.v[e]);
            b[e] = to_f(p1.v[e]);
        } else {
            const Pack<T, V>& p = e < V / 2 ? p0 : p1;
            a[e] = to_f(p.v[2 * e % V]);
            b[e] = to_f(p.v[(2 * e + 1) % V]);
        }
    }
}
template <typename T, int V, bool WHOLE> __device__ __forceinline__ void pack(const float* a, const float* b, Pack<T, V>& p0, Pack<T, V>& p1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (!WHOLE) {
            p0.v[e] = from_f<T>(a[e]);
            p1.v[e] = from_f<T>(b[e]);
        } else {
            Pack<T, V>& p = e < V / 2 ? p0 : p1;
            p.v[2 * e % V] = from_f<T>(a[e]);
            p.v[(2 * e + 1) % V] = from_f<T>(b[e]);
        }
    }
}

// (a, b) -> (a c - b s, b c + a s) for the pairs that are rotated (`partial`: not all are); the second half of a chunk of whole pairs has a flag
// of its own
template <int V, bool WHOLE> __device__ __forceinline__ void rotate(float* a, float* b, const float* c, const float* s, bool partial, bool rot0, bool rot1) {
    float y[V], z[V];
    pairwise<V>(
        [&](int e) {
            const float2 a2 = at2(a, e), b2 = at2(b, e), c2 = at2(c, e), s2 = at2(s, e);
            const float2 t = __fmul2_rn(b2, s2);
            put2(y, e, __ffma2_rn(a2, c2, make_float2(-t.x, -t.y)));
            put2(z, e, __ffma2_rn(b2, c2, __fmul2_rn(a2, s2)));
        },
        [&](int e) {
            y[e] = a[e] * c[e] - b[e] * s[e];
            z[e] = b[e] * c[e] + a[e] * s[e];
        });
    if (partial) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const bool rot = WHOLE && e >= V / 2 ? rot1 : rot0;
            y[e] = rot ? y[e] : a[e];
            z[e] = rot ? z[e] : b[e];
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        a[e] = y[e];
        b[e] = z[e];
    }
}

enum { kRotate = 0, kNorm = 1, kNormBwd = 2 };
constexpr int kAhead = 2;           // rows that the asynchronous copies run ahead
constexpr int ring_bytes(int vector_bytes, int nv, int mode) {
    return vector_bytes >= 4 ? kWarps * (kAhead + 1) * (mode == kNormBwd ? 4 : 2) * nv * 32 * vector_bytes : 0;
}

template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool in) {         // zeros where not in
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(in ? BYTES : 0) : "memory");
}
template <typename R> __device__ __forceinline__ R load_shared(uint32_t from) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (sizeof(R) == 16)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    else if (sizeof(R) == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(from) : "memory");
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v.x) : "r"(from) : "memory");
    return *reinterpret_cast<const R*>(&v);
}

// Queries or keys.  Read from the constant bank where it is used (the index is the same for a whole CTA).
struct Side {
    const void *x, *g, *w;
    void* y;
    long xs[3], gs[3], ys[3];
    int heads, hpu, parts;         // heads, heads per unit, units per token
};
struct Params {
    Side side[2];
    const void* positions;
    const double* half_turns;
    const int* axis;
    float* partials;
    long pos_stride[3], batch_tokens;
    int tokens, D, P, pos_is_64, whole, ctas_q;
    float amplitude, sin_amplitude, eps, inv_D;
};

// Three CTAs an SM leave 80 registers a thread, of which the norm's forward on eight 16-bit elements a lane spills 72 - 84 bytes.  Two CTAs without spills: 24 + 24
// heads of 32400 tokens 148.5 us against 146.5, 8 x 256 tokens of 32 + 8 heads 15.5 - 16.4 against 17.4, 3 x 1001 of 12 + 4 heads of 64 level.
//
// A group of 2^log_l lanes holds one head of one token; a warp's groups take consecutive heads.  A unit is a token with all heads of q and k
// (`whole`), or with `hpu` heads of one of them; consecutive warps take consecutive tokens, whose rows are neighbours in the head-major
// output.  The norm's backward keeps q and k apart, since a CTA sums one weight's gradient: CTAs below ctas_q work on q, the others on k.
template <typename T, int V, int NV, bool INTER, int MODE, int LOGL>
__global__ void __launch_bounds__(kThreads, MODE == kRotate ? 3 : MODE == kNorm ? 3 : 2) rotary_kernel(const __grid_constant__ Params a, const int any_log_l) {
    constexpr bool WHOLE = Geometry<V, NV, INTER>::kWhole, ASYNC = V * sizeof(T) >= 4;
    constexpr int VB = V * sizeof(T), kVectors = (MODE == kNormBwd ? 4 : 2) * NV;         // of a lane and row
    extern __shared__ __align__(16) uint8_t ring_raw[];
    const uint32_t ring = sm100::smem_u32(ring_raw);
    __shared__ alignas(16) float angle[kWarps][2][kMaxD / 2];         // cos, sin
    __shared__ float fold[MODE == kNormBwd ? kWarps : 1][MODE == kNormBwd ? kMaxD : 1];
    const int log_l = LOGL >= 0 ? LOGL : any_log_l;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int l = lane & ((1 << log_l) - 1), sub = lane >> log_l, rows = 32 >> log_l;
    const int D = a.D, P = a.P;
    const Geometry<V, NV, INTER> geo(l, log_l, P);
    bool in0[NV], in1[NV], rot0[NV], rot1[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        in0[i] = geo.off0[i] < D;
        in1[i] = geo.off1[i] < D;
        rot0[i] = WHOLE ? geo.off0[i] < 2 * P : (l + (i << log_l)) * V < P;
        rot1[i] = geo.off1[i] < 2 * P;
    }
    const bool partial = 2 * P < (2 * V * NV << log_l);         // some lane has elements that are not rotated, or none at all
    const uint32_t cos_table = sm100::smem_u32(&angle[warp][0][0]);
    const int only = MODE != kNormBwd ? -1 : (int)blockIdx.x >= a.ctas_q ? 1 : 0;
    const int cta = (int)blockIdx.x - (only == 1 ? a.ctas_q : 0), n_ctas = only < 0 ? (int)gridDim.x : only ? (int)gridDim.x - a.ctas_q : a.ctas_q;
    const int parts = only >= 0 ? a.side[only].parts : a.whole ? 1 : a.side[0].parts + a.side[1].parts;
    const long units = a.batch_tokens * parts;

    float acc0[NV][V], acc1[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) acc0[i][e] = acc1[i][e] = 0.f;
    auto group_sum = [&](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o < 1 << log_l) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };

    // A unit's token and heads: of q and k, or (last == which + 1) of one of them.
    struct Unit {
        long b;
        int t, part, which, last;
    };
    auto unit_at = [&](long unit) {
        Unit w;
        long token = unit;
        w.part = 0;
        if (parts > 1) {
            w.part = (int)(unit / a.batch_tokens);
            token = unit - (long)w.part * a.batch_tokens;
        }
        w.b = 0;
        w.t = (int)token;
        if (a.batch_tokens > a.tokens) {
            w.b = a.batch_tokens <= INT_MAX ? (int)token / a.tokens : token / a.tokens;
            w.t = (int)(token - w.b * a.tokens);
        }
        w.which = only >= 0 ? only : !a.whole && w.part >= a.side[0].parts ? 1 : 0;
        if (only < 0 && w.which) w.part -= a.side[0].parts;
        w.last = only < 0 && a.whole ? 2 : w.which + 1;
        return w;
    };
    const long unit_step = (long)n_ctas * kWarps, first_unit = (long)cta * kWarps + warp;

    // Loads run kAhead rows ahead of the arithmetic, over the borders of heads, q and k, and tokens: vectors are copied asynchronously into
    // slots of shared memory that a lane has to itself, which costs no registers.  (24 + 24 heads of 32400 tokens with one row ahead in registers:
    // rotation there and back 289 us, the norm's forward 176 and backward 281; so 252, 139 and 198.)  Single elements of 16 bits, which
    // the copies do not take, go through registers, one row ahead.
    struct Rows {
        long unit;
        int which, last, part, t, h0, h_end;
        long b;
        const T *x, *g;
        bool any;
    } ahead;
    auto enter = [&] {              // the first rows of side ahead.which, or of the next one that has any
        while (true) {
            if (ahead.which < ahead.last) {
                const Side& side = a.side[ahead.which];
                ahead.h0 = ahead.part * side.hpu + sub;
                ahead.h_end = min(side.heads, (ahead.part + 1) * side.hpu);
                if (ahead.h0 - sub < ahead.h_end) {
                    ahead.x = (const T*)side.x + ahead.b * side.xs[0] + ahead.t * side.xs[2] + ahead.h0 * side.xs[1];
                    if (MODE == kNormBwd) ahead.g = (const T*)side.g + ahead.b * side.gs[0] + ahead.t * side.gs[2] + ahead.h0 * side.gs[1];
                    return;
                }
                ++ahead.which;
                continue;
            }
            ahead.unit += unit_step;
            ahead.any = ahead.unit < units;
            if (!ahead.any) return;
            const Unit w = unit_at(ahead.unit);
            ahead.which = w.which;
            ahead.last = w.last;
            ahead.part = w.part;
            ahead.b = w.b;
            ahead.t = w.t;
        }
    };
    auto advance = [&] {
        ahead.h0 += rows;
        if (ahead.h0 - sub < ahead.h_end) {
            ahead.x += rows * a.side[ahead.which].xs[1];
            if (MODE == kNormBwd) ahead.g += rows * a.side[ahead.which].gs[1];
        } else {
            ++ahead.which;
            enter();
        }
    };
    Pack<T, V> nx0[NV], nx1[NV], ng0[NV], ng1[NV];
    const uint32_t slots = ring + ((uint32_t)warp * (kAhead + 1) * kVectors * 32 + lane) * VB;
    int fetched = 0, taken = 0;     // of kAhead + 1 slots
    auto fetch = [&] {              // rows behind the last head are 0: they count for nothing in the weights' gradient
        const bool ok = ahead.any && ahead.h0 < ahead.h_end;
        if (ASYNC) {
            uint32_t to = slots + fetched * (kVectors * 32 * VB);
#pragma unroll
            for (int i = 0; i < NV; ++i, to += kVectors / NV * 32 * VB) {
                const bool c0 = ok && in0[i], c1 = ok && in1[i];
                copy_async<VB < 4 ? 4 : VB>(to, c0 ? (const void*)(ahead.x + geo.off0[i]) : a.half_turns, c0);
                copy_async<VB < 4 ? 4 : VB>(to + 32 * VB, c1 ? (const void*)(ahead.x + geo.off1[i]) : a.half_turns, c1);
                if (MODE == kNormBwd) {
                    copy_async<VB < 4 ? 4 : VB>(to + 64 * VB, c0 ? (const void*)(ahead.g + geo.off0[i]) : a.half_turns, c0);
                    copy_async<VB < 4 ? 4 : VB>(to + 96 * VB, c1 ? (const void*)(ahead.g + geo.off1[i]) : a.half_turns, c1);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            fetched = fetched == kAhead ? 0 : fetched + 1;
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                nx0[i] = nx1[i] = Pack<T, V>();
                if (ok && in0[i]) nx0[i].load(ahead.x + geo.off0[i]);
                if (ok && in1[i]) nx1[i].load(ahead.x + geo.off1[i]);
                if (MODE == kNormBwd) {
                    ng0[i] = ng1[i] = Pack<T, V>();
                    if (ok && in0[i]) ng0[i].load(ahead.g + geo.off0[i]);
                    if (ok && in1[i]) ng1[i].load(ahead.g + geo.off1[i]);
                }
            }
        }
        if (ahead.any) advance();
    };
    if (first_unit < units) {
        const Unit w = unit_at(first_unit);
        ahead = {first_unit, w.which, w.last, w.part, w.t, 0, 0, w.b, nullptr, nullptr, true};
        enter();
#pragma unroll
        for (int i = 0; i < (ASYNC ? kAhead : 1); ++i) fetch();
    }

    for (long unit = first_unit; unit < units; unit += unit_step) {
        Unit w = unit_at(unit);
        {       // every pair's angle once per token and warp, spread over the lanes
            const long at = w.b * a.pos_stride[0] + w.t * a.pos_stride[2];
            __syncwarp();
            for (int p = lane; p < P; p += 32) {
                const long q = at + (a.axis != nullptr ? a.axis[p] * a.pos_stride[1] : 0L);
                const double pos = a.pos_is_64 ? (double)((const long long*)a.positions)[q] : (double)((const int*)a.positions)[q];
                const double h = pos * a.half_turns[p];                // angle / pi
                float c, s;
                sincospif((float)(h - 2.0 * rint(0.5 * h)), &s, &c);
                const int place = Geometry<V, NV, INTER>::place(p, P);
                angle[warp][0][place] = c * a.amplitude;
                angle[warp][1][place] = s * a.sin_amplitude;
            }
            __syncwarp();
        }
        for (; w.which < w.last; ++w.which) {
            const Side& side = a.side[w.which];
            const int h_end = min(side.heads, (w.part + 1) * side.hpu);
            int h0 = w.part * side.hpu + sub;
            if (h0 - sub >= h_end) continue;        // no heads
            T* yr = (T*)side.y + w.b * side.ys[0] + w.t * side.ys[2] + h0 * side.ys[1];
            Pack<T, V> pw0[NV], pw1[NV];
            if (MODE != kRotate) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (in0[i]) pw0[i].load((const T*)side.w + geo.off0[i]);
                    if (in1[i]) pw1[i].load((const T*)side.w + geo.off1[i]);
                }
            }
            for (; h0 - sub < h_end; h0 += rows, yr += rows * side.ys[1]) {
                Pack<T, V> px0[NV], px1[NV], pg0[NV], pg1[NV];
                if (ASYNC) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
                    uint32_t from = slots + taken * (kVectors * 32 * VB);
                    using R = typename Pack<T, V>::R;
#pragma unroll
                    for (int i = 0; i < NV; ++i, from += kVectors / NV * 32 * VB) {
                        px0[i].raw = load_shared<R>(from);
                        px1[i].raw = load_shared<R>(from + 32 * VB);
                        if (MODE == kNormBwd) {
                            pg0[i].raw = load_shared<R>(from + 64 * VB);
                            pg1[i].raw = load_shared<R>(from + 96 * VB);
                        }
                    }
                    taken = taken == kAhead ? 0 : taken + 1;
                } else {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        px0[i] = nx0[i];
                        px1[i] = nx1[i];
                        if (MODE == kNormBwd) {
                            pg0[i] = ng0[i];
                            pg1[i] = ng1[i];
                        }
                    }
                }
                fetch();
                float f0[NV][V], f1[NV][V];
#pragma unroll
                for (int i = 0; i < NV; ++i) unpack<T, V, WHOLE>(px0[i], px1[i], f0[i], f1[i]);
                if (MODE != kRotate) {
                    float sq[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) sq[e] = 0.f;
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        add_product<V>(sq, f0[i], f0[i]);
                        add_product<V>(sq, f1[i], f1[i]);
                    }
                    const float ss = total<V>(sq);
                    float r = rsqrtf(group_sum(ss) * a.inv_D + a.eps);
                    if (MODE == kNormBwd && h0 >= h_end) r = 0.f;         // a row behind the last head; without eps it would be NaN
                    float g0[NV][V], g1[NV][V], dots[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) dots[e] = 0.f;
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        float w0[V], w1[V];
                        unpack<T, V, WHOLE>(pw0[i], pw1[i], w0, w1);
                        scale<V>(f0[i], r);
                        scale<V>(f1[i], r);
                        if (MODE == kNorm) {
                            mul<V>(f0[i], w0);
                            mul<V>(f1[i], w1);
                        } else {
                            float cs[V], sn[V];
                            geo.angles(cos_table, i, l, log_l, P, cs);
                            geo.angles(cos_table + 4 * (kMaxD / 2), i, l, log_l, P, sn);
                            unpack<T, V, WHOLE>(pg0[i], pg1[i], g0[i], g1[i]);
                            rotate<V, WHOLE>(g0[i], g1[i], cs, sn, partial, rot0[i], rot1[i]);
                            add_product<V>(acc0[i], g0[i], f0[i]);
                            add_product<V>(acc1[i], g1[i], f1[i]);
                            mul<V>(g0[i], w0);
                            mul<V>(g1[i], w1);
                            add_product<V>(dots, g0[i], f0[i]);
                            add_product<V>(dots, g1[i], f1[i]);
                        }
                    }
                    if (MODE == kNormBwd) {
                        const float dot = -group_sum(total<V>(dots)) * a.inv_D;
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            // r (g' w - x^ mean(g' w x^))
                            pairwise<V>(
                                [&](int e) {
                                    const float2 d2 = make_float2(dot, dot), r2 = make_float2(r, r);
                                    put2(f0[i], e, __fmul2_rn(r2, __ffma2_rn(at2(f0[i], e), d2, at2(g0[i], e))));
                                    put2(f1[i], e, __fmul2_rn(r2, __ffma2_rn(at2(f1[i], e), d2, at2(g1[i], e))));
                                },
                                [&](int e) {
                                    f0[i][e] = r * (g0[i][e] + f0[i][e] * dot);
                                    f1[i][e] = r * (g1[i][e] + f1[i][e] * dot);
                                });
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (MODE != kNormBwd) {
                        float cs[V], sn[V];
                        geo.angles(cos_table, i, l, log_l, P, cs);
                        geo.angles(cos_table + 4 * (kMaxD / 2), i, l, log_l, P, sn);
                        rotate<V, WHOLE>(f0[i], f1[i], cs, sn, partial, rot0[i], rot1[i]);
                    }
                    Pack<T, V> o0, o1;
                    pack<T, V, WHOLE>(f0[i], f1[i], o0, o1);
                    if (h0 < h_end && in0[i]) o0.store(yr + geo.off0[i]);
                    if (h0 < h_end && in1[i]) o1.store(yr + geo.off1[i]);
                }
            }
        }
    }
    if (ASYNC) asm volatile("cp.async.wait_all;" ::: "memory");
    if (MODE == kNormBwd) {     // this CTA's share of the weight gradient, in a fixed order
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e)
                for (int o = 1 << log_l; o < 32; o <<= 1) {
                    acc0[i][e] += __shfl_xor_sync(0xffffffffu, acc0[i][e], o);
                    acc1[i][e] += __shfl_xor_sync(0xffffffffu, acc1[i][e], o);
                }
        if (sub == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) {       // where unpack took entry e from
                    const bool second = WHOLE && e >= V / 2;
                    const int at0 = !WHOLE ? geo.off0[i] + e : (second ? geo.off1[i] : geo.off0[i]) + 2 * e % V;
                    const int at1 = !WHOLE ? geo.off1[i] + e : at0 + 1;
                    if (at0 < D) fold[warp][at0] = acc0[i][e];
                    if (at1 < D) fold[warp][at1] = acc1[i][e];
                }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kThreads) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) s += fold[i][d];
            a.partials[(long)blockIdx.x * D + d] = s;
        }
    }
}

// Column sums of the CTAs' partial rows: 16 columns a CTA, 64 threads a column, folded in a fixed order.
constexpr int kFinCols = 16, kFinRows = 64;
template <typename T>
__global__ void __launch_bounds__(kFinCols * kFinRows) rotary_weight_kernel(const float* __restrict__ partials, T* __restrict__ dq, T* __restrict__ dk,
                                                                           int D, int ctas_q, int ctas) {
    __shared__ float fold[kFinRows][kFinCols + 1];
    const int cl = threadIdx.x % kFinCols, r = threadIdx.x / kFinCols;
    const int c = blockIdx.x * kFinCols + cl, which = ctas_q == 0 ? 1 : blockIdx.y;       // only operands that there are
    const int first = which ? ctas_q : 0, last = which ? ctas : ctas_q;
    float s = 0.f;
    if (c < D)
        for (int i = first + r; i < last; i += kFinRows) s += partials[(long)i * D + c];
    fold[r][cl] = s;
    __syncthreads();
    if (r == 0 && c < D) {
        s = 0.f;
#pragma unroll 8
        for (int i = 0; i < kFinRows; ++i) s += fold[i][cl];
        (which ? dk : dq)[c] = from_f<T>(s);
    }
}

struct Plan {
    int width, log_l, whole, ctas_q, ctas_k, hpu_q, hpu_k;      // forward: ctas_q for both
};

int elem_size(int dtype) { return dtype == TT_FP32 ? 4 : 2; }

// Elements a lane moves at once: 16 bytes where the pairs' halves, the rows and the pointers allow it, else 2 or 1.
int vector_width(const tt_rotary_args& a) {
    const int size = elem_size(a.dtype);
    for (int v : {16 / size, 2, 1}) {
        bool ok = a.head_dim % v == 0 && (a.interleaved ? (2 * a.pairs) % v == 0 : a.pairs % v == 0);
        auto test = [&](const void* p, const long* s, int heads) {
            if (p == nullptr || heads == 0) return;
            ok = ok && (uintptr_t)p % (v * size) == 0 && (s == nullptr || (s[0] % v == 0 && s[1] % v == 0 && s[2] % v == 0));
        };
        test(a.q, a.q_stride, a.q_heads);
        test(a.k, a.k_stride, a.k_heads);
        test(a.gq, a.gq_stride, a.q_heads);
        test(a.gk, a.gk_stride, a.k_heads);
        test(a.out_q, a.out_q_stride, a.q_heads);
        test(a.out_k, a.out_k_stride, a.k_heads);
        test(a.q_weight, nullptr, a.q_heads);
        test(a.k_weight, nullptr, a.k_heads);
        if (ok) return v;
    }
    return 1;
}

Plan plan(const tt_rotary_args& a, int sms, int mode) {
    Plan p;
    p.width = vector_width(a);
    const int chunks = (a.head_dim + 2 * p.width - 1) / (2 * p.width);
    p.log_l = 0;
    while ((1 << p.log_l) < chunks && p.log_l < 5) ++p.log_l;
    const int rows = 32 >> p.log_l;
    const long tokens = a.batch * a.tokens;
    // All heads of a token in one unit share its angles.  With fewer tokens than three quarters of the device's warps at a CTA an SM a unit takes
    // fewer heads, so that the units cover the device (32 + 8 heads of 128, parts against whole tokens: 256 tokens 4.0 / 6.0 us, 600
    // 5.4 / 6.1, 1100 7.9 / 6.8, 2000 9.8 / 8.8).
    p.whole = tokens >= (long)sms * (kWarps * 3 / 4);
    auto heads_per_unit = [&](int heads) {
        int per = (heads + rows - 1) / rows;
        while (!p.whole && per > 1 && tokens * ((heads + rows * per - 1) / (rows * per)) < (long)sms * kWarps) per = (per + 1) / 2;
        return rows * (per > 0 ? per : 1);
    };
    p.hpu_q = heads_per_unit(a.q_heads);
    p.hpu_k = heads_per_unit(a.k_heads);
    const long cap = (long)sms * 8;
    auto ctas = [&](long parts, long most) {
        const long want = (tokens * parts + kWarps - 1) / kWarps;
        return (int)(want < most ? want : most);
    };
    const long parts_q = (a.q_heads + p.hpu_q - 1) / p.hpu_q, parts_k = (a.k_heads + p.hpu_k - 1) / p.hpu_k;
    if (mode != kNormBwd) {
        p.ctas_q = ctas(p.whole ? 1 : parts_q + parts_k, INT_MAX);
        p.ctas_k = 0;
    } else {
        p.ctas_q = ctas(parts_q, (cap * a.q_heads + a.q_heads + a.k_heads - 1) / (a.q_heads + a.k_heads));
        p.ctas_k = ctas(parts_k, (cap * a.k_heads + a.q_heads + a.k_heads - 1) / (a.q_heads + a.k_heads));
    }
    return p;
}

Params params(const tt_rotary_args& a, const Plan& p, int mode) {
    Params k;
    k.side[0] = {a.q, a.gq, a.q_weight, a.out_q, {}, {}, {}, a.q_heads, p.hpu_q, (a.q_heads + p.hpu_q - 1) / p.hpu_q};
    k.side[1] = {a.k, a.gk, a.k_weight, a.out_k, {}, {}, {}, a.k_heads, p.hpu_k, (a.k_heads + p.hpu_k - 1) / p.hpu_k};
    for (int i = 0; i < 3; ++i) {
        k.side[0].xs[i] = a.q_stride[i];
        k.side[0].gs[i] = a.gq_stride[i];
        k.side[0].ys[i] = a.out_q_stride[i];
        k.side[1].xs[i] = a.k_stride[i];
        k.side[1].gs[i] = a.gk_stride[i];
        k.side[1].ys[i] = a.out_k_stride[i];
        k.pos_stride[i] = a.pos_stride[i];
    }
    k.positions = a.positions;
    k.half_turns = a.half_turns;
    k.axis = a.axis;
    k.partials = a.partials;
    k.batch_tokens = a.batch * a.tokens;
    k.tokens = (int)a.tokens;
    k.D = a.head_dim;
    k.P = a.pairs;
    k.pos_is_64 = a.pos_is_64;
    k.whole = p.whole;
    k.ctas_q = p.ctas_q;
    k.amplitude = a.amplitude;
    k.sin_amplitude = mode == kNormBwd || a.transpose ? -a.amplitude : a.amplitude;
    k.eps = a.eps;
    k.inv_D = 1.f / (float)a.head_dim;
    return k;
}

template <typename T, int V, int NV, bool INTER, int LOGL = -1>
int launch(const tt_rotary_args& a, const Plan& p, int mode, cudaStream_t st) {
    const int grid = p.ctas_q + p.ctas_k;
    const Params k = params(a, p, mode);
    const int ring = ring_bytes(V * sizeof(T), NV, mode);
    if (mode == kRotate) rotary_kernel<T, V, NV, INTER, kRotate, LOGL><<<grid, kThreads, ring, st>>>(k, p.log_l);
    else if (mode == kNorm) rotary_kernel<T, V, NV, INTER, kNorm, LOGL><<<grid, kThreads, ring, st>>>(k, p.log_l);
    else {
        static bool configured[64] = {false};         // per device: the attribute belongs to the device's context
        const int dev = tt_device().dev;
        if (!configured[dev]) {         // 64 KB with the static part
            cudaError_t e = cudaFuncSetAttribute(rotary_kernel<T, V, NV, INTER, kNormBwd, LOGL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 ring_bytes(V * sizeof(T), NV, kNormBwd));
            if (e != cudaSuccess) return tt_record_cuda(e);
            configured[dev] = true;
        }
        rotary_kernel<T, V, NV, INTER, kNormBwd, LOGL><<<grid, kThreads, ring, st>>>(k, p.log_l);
    }
    return TT_OK;
}

// Full-width vectors of 16-bit heads of 64 and 128 (four and eight lanes) have the lanes of a head compiled in.
template <typename T>
int dispatch(const tt_rotary_args& a, const Plan& p, int mode, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T), A = W == 8 ? 3 : -1, B = W == 8 ? 2 : -1;
    if (p.width == W && W == 8 && p.log_l == 3) return a.interleaved ? launch<T, W, 1, true, A>(a, p, mode, st) : launch<T, W, 1, false, A>(a, p, mode, st);
    if (p.width == W && W == 8 && p.log_l == 2) return a.interleaved ? launch<T, W, 1, true, B>(a, p, mode, st) : launch<T, W, 1, false, B>(a, p, mode, st);
    if (p.width == W) return a.interleaved ? launch<T, W, 1, true>(a, p, mode, st) : launch<T, W, 1, false>(a, p, mode, st);
    if (p.width == 2) return a.interleaved ? launch<T, 2, 2, true>(a, p, mode, st) : launch<T, 2, 2, false>(a, p, mode, st);
    return a.interleaved ? launch<T, 1, 4, true>(a, p, mode, st) : launch<T, 1, 4, false>(a, p, mode, st);
}

int check(const tt_rotary_args* a) {
    if (a == nullptr || a->struct_size != (long)sizeof(tt_rotary_args)) return TT_ERR_ARG;
    if (a->batch <= 0 || a->tokens <= 0 || a->tokens > INT_MAX || a->batch > INT_MAX || a->q_heads < 0 || a->k_heads < 0 || a->q_heads + a->k_heads == 0) return TT_ERR_ARG;
    if (a->head_dim <= 0 || a->head_dim % 2 || a->pairs <= 0 || 2 * a->pairs > a->head_dim) return TT_ERR_ARG;
    if (a->head_dim > kMaxD) return TT_ERR_LIMIT;
    if (a->dtype != TT_BF16 && a->dtype != TT_FP16 && a->dtype != TT_FP32) return TT_ERR_ARG;
    if (a->positions == nullptr || a->half_turns == nullptr) return TT_ERR_ARG;
    if (a->q_heads > 0 && (a->q == nullptr || a->out_q == nullptr)) return TT_ERR_ARG;
    if (a->k_heads > 0 && (a->k == nullptr || a->out_k == nullptr)) return TT_ERR_ARG;
    return TT_OK;
}

int run(const tt_rotary_args* a, int mode, void* stream) {
    const int rc = check(a);
    if (rc != TT_OK) return rc;
    if (mode != kRotate && ((a->q_heads > 0 && a->q_weight == nullptr) || (a->k_heads > 0 && a->k_weight == nullptr))) return TT_ERR_ARG;
    if (mode == kNormBwd && (a->partials == nullptr || (a->q_heads > 0 && (a->gq == nullptr || a->dq_weight == nullptr)) ||
                             (a->k_heads > 0 && (a->gk == nullptr || a->dk_weight == nullptr))))
        return TT_ERR_ARG;
    const Plan p = plan(*a, tt_device().sms, mode);
    if (mode == kNormBwd && a->partial_floats < (long)(p.ctas_q + p.ctas_k) * a->head_dim) return TT_ERR_ARG;
    cudaStream_t st = (cudaStream_t)stream;
    const int rc2 = a->dtype == TT_BF16 ? dispatch<__nv_bfloat16>(*a, p, mode, st)
                    : a->dtype == TT_FP16 ? dispatch<__half>(*a, p, mode, st) : dispatch<float>(*a, p, mode, st);
    if (rc2 != TT_OK) return rc2;
    TT_CHECK_LAUNCH();
    if (mode == kNormBwd) {
        const dim3 grid((a->head_dim + kFinCols - 1) / kFinCols, (a->q_heads > 0) + (a->k_heads > 0));
        if (a->dtype == TT_BF16)
            rotary_weight_kernel<<<grid, kFinCols * kFinRows, 0, st>>>(a->partials, (__nv_bfloat16*)a->dq_weight, (__nv_bfloat16*)a->dk_weight,
                                                                       a->head_dim, p.ctas_q, p.ctas_q + p.ctas_k);
        else if (a->dtype == TT_FP16)
            rotary_weight_kernel<<<grid, kFinCols * kFinRows, 0, st>>>(a->partials, (__half*)a->dq_weight, (__half*)a->dk_weight, a->head_dim,
                                                                       p.ctas_q, p.ctas_q + p.ctas_k);
        else
            rotary_weight_kernel<<<grid, kFinCols * kFinRows, 0, st>>>(a->partials, (float*)a->dq_weight, (float*)a->dk_weight, a->head_dim,
                                                                       p.ctas_q, p.ctas_q + p.ctas_k);
        TT_CHECK_LAUNCH();
    }
    return TT_OK;
}

}  // namespace

extern "C" long tt_rotary_partial_floats(const tt_rotary_args* a) {
    if (check(a) != TT_OK) return -1;
    const Plan p = plan(*a, tt_device().sms, kNormBwd);
    return (long)(p.ctas_q + p.ctas_k) * a->head_dim;
}
extern "C" int tt_rotary(const tt_rotary_args* a, void* stream) { return run(a, kRotate, stream); }
extern "C" int tt_norm_rotary_fwd(const tt_rotary_args* a, void* stream) { return run(a, kNorm, stream); }
extern "C" int tt_norm_rotary_bwd(const tt_rotary_args* a, void* stream) { return run(a, kNormBwd, stream); }
