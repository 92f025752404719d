// Rotary positions of queries and keys, alone or behind an RMS norm of every head, forward and backward.
//
//   y[p0] = A (x[p0] cos t - x[p1] sin t),   y[p1] = A (x[p1] cos t + x[p0] sin t),   t = position[axis(p)] * w_p
//
// for pairs p < P of a head of D >= 2 P elements: (p, P + p) in the half layout, (2 p, 2 p + 1) in the interleaved one; elements
// from 2 P on pass.  The transpose of a rotation is the rotation by -t, so the backward of the plain form is the same kernel.
// With the norm x is replaced by x^ w, x^ = r x, r = rsqrt(mean x^2 + eps); backward, with g' the rotated-back gradient:
// dw = sum over rows of g' x^, dx = r (g' w - x^ mean(g' w x^)).
//
// No table is read: the angle of a (token, pair) is shared by all heads, so a warp forms it once per token, in 64 bits (a
// position of 10^5 times a frequency near 1 leaves 2^-7 of a turn's fraction in 32 bits), reduced to a part of a turn, and keeps cos and sin
// in registers over the token's heads.  The kernels are bound by memory: 2 passes over q and k forward, 3 for the norm's backward.
#include <cuda_fp16.h>

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
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f(v[i]);
    }
    __device__ __forceinline__ void set(const float* f) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = from_f<T>(f[i]);
    }
};

// A lane's share of a head: NV chunks of V pairs, each as two vectors of V elements at off0 and off1.
template <int V, int NV, bool INTER> struct Geometry {
    int off0[NV], off1[NV];
    bool in0[NV], in1[NV], rot0[NV], rot1[NV];
    __device__ __forceinline__ Geometry(int l, int log_l, int D, int P) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = l + (i << log_l);
            if (INTER && V > 1) {
                off0[i] = c * 2 * V;
                off1[i] = off0[i] + V;
                rot0[i] = off0[i] < 2 * P;
                rot1[i] = off1[i] < 2 * P;
            } else if (c * V < P) {
                off0[i] = INTER ? 2 * c : c * V;
                off1[i] = INTER ? 2 * c + 1 : P + c * V;
                rot0[i] = rot1[i] = true;
            } else {
                off0[i] = 2 * P + (c - P / V) * 2 * V;
                off1[i] = off0[i] + V;
                rot0[i] = rot1[i] = false;
            }
            in0[i] = off0[i] < D;
            in1[i] = off1[i] < D;
        }
    }
    // the pair whose angle entry e of chunk i belongs to
    __device__ __forceinline__ int pair(int i, int e, int l, int log_l) const {
        if (INTER && V > 1) return e < V / 2 ? off0[i] / 2 + e : off1[i] / 2 + e - V / 2;
        return (l + (i << log_l)) * V + e;
    }
};

template <int V, bool INTER>
__device__ __forceinline__ void rotate(float* u, float* v, const float* c, const float* s, bool rot0, bool rot1) {
    if (INTER && V > 1) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const float a0 = u[2 * e], a1 = u[2 * e + 1], b0 = v[2 * e], b1 = v[2 * e + 1];
            if (rot0) {
                u[2 * e] = a0 * c[e] - a1 * s[e];
                u[2 * e + 1] = a1 * c[e] + a0 * s[e];
            }
            if (rot1) {
                v[2 * e] = b0 * c[V / 2 + e] - b1 * s[V / 2 + e];
                v[2 * e + 1] = b1 * c[V / 2 + e] + b0 * s[V / 2 + e];
            }
        }
    } else if (rot0) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float a = u[e], b = v[e];
            u[e] = a * c[e] - b * s[e];
            v[e] = b * c[e] + a * s[e];
        }
    }
}

enum { kRotate = 0, kNorm = 1, kNormBwd = 2 };

// A group of 2^log_l lanes holds one head of one token; a warp's groups take consecutive heads of the same token, U rows per group at a
// time so that 2 U (backward 4 U) loads are in flight.  A unit is one token with heads_per_unit heads; consecutive warps take
// consecutive tokens, whose rows are neighbours in the head-major output.  CTAs below ctas_q work on q, the others on k.
template <typename T, int V, int NV, bool INTER, int MODE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const tt_rotary_args a, const int log_l, const int ctas_q, const int hpu_q, const int hpu_k) {
    constexpr int U = MODE == kNormBwd ? (NV * V >= 8 ? 1 : 2) : (NV * V >= 4 ? 4 : 4);
    __shared__ float fold[MODE == kNormBwd ? kWarps : 1][MODE == kNormBwd ? kMaxD : 1];
    const int which = (int)blockIdx.x >= ctas_q;
    const long cta = which ? (long)blockIdx.x - ctas_q : blockIdx.x, n_ctas = which ? (long)gridDim.x - ctas_q : ctas_q;
    const int heads = which ? a.k_heads : a.q_heads, hpu = which ? hpu_k : hpu_q;
    const T* __restrict__ x = (const T*)(which ? a.k : a.q);
    const T* __restrict__ g = (const T*)(which ? a.gk : a.gq);
    const T* __restrict__ w = (const T*)(which ? a.k_weight : a.q_weight);
    T* __restrict__ y = (T*)(which ? a.out_k : a.out_q);
    const long *xs = which ? a.k_stride : a.q_stride, *gs = which ? a.gk_stride : a.gq_stride, *ys = which ? a.out_k_stride : a.out_q_stride;
    const long xb = xs[0], xh = xs[1], xt = xs[2], gb = gs[0], gh = gs[1], gt = gs[2], yb = ys[0], yh = ys[1], yt = ys[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int l = lane & ((1 << log_l) - 1), sub = lane >> log_l, rows = 32 >> log_l;
    const int D = a.head_dim, P = a.pairs;
    const Geometry<V, NV, INTER> geo(l, log_l, D, P);
    const long tokens = (long)a.batch * a.tokens;
    const int parts = (heads + hpu - 1) / hpu;
    const long units = tokens * parts;

    float w0[NV][V], w1[NV][V], acc0[NV][V], acc1[NV][V];
    if (MODE != kRotate) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Pack<T, V> p0, p1;
            if (geo.in0[i]) p0.load(w + geo.off0[i]);
            if (geo.in1[i]) p1.load(w + geo.off1[i]);
            p0.get(w0[i]);
            p1.get(w1[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) acc0[i][e] = acc1[i][e] = 0.f;
        }
    }
    auto group_sum = [&](float v) {
        for (int o = 1 << log_l >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };

    for (long unit = cta * kWarps + warp; unit < units; unit += n_ctas * kWarps) {
        const int part = parts == 1 ? 0 : (int)(unit / tokens);
        const long token = parts == 1 ? unit : unit - (long)part * tokens;
        const long b = token / a.tokens, t = token - b * a.tokens;
        const int h_end = min(heads, (part + 1) * hpu);
        float cs[NV][V], sn[NV][V];
        {
            const long at = b * a.pos_stride[0] + t * a.pos_stride[2];
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int p = geo.pair(i, e, l, log_l);
                    cs[i][e] = 1.f;
                    sn[i][e] = 0.f;
                    if (p < P) {
                        const long q = at + (a.axis != nullptr ? a.axis[p] * a.pos_stride[1] : 0L);
                        const double pos = a.pos_is_64 ? (double)((const long long*)a.positions)[q] : (double)((const int*)a.positions)[q];
                        const double h = pos * a.half_turns[p];                // angle / pi
                        sincospif((float)(h - 2.0 * rint(0.5 * h)), &sn[i][e], &cs[i][e]);
                        cs[i][e] *= a.amplitude;
                        sn[i][e] *= MODE == kNormBwd || a.transpose ? -a.amplitude : a.amplitude;
                    }
                }
        }
        const T* xp = x + b * xb + t * xt;
        const T* gp = g + b * gb + t * gt;
        T* yp = y + b * yb + t * yt;
        for (int h0 = part * hpu + sub; h0 - sub < h_end; h0 += rows * U) {
            Pack<T, V> px0[U][NV], px1[U][NV], pg0[U][NV], pg1[U][NV];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * rows;
                if (h < h_end) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        if (geo.in0[i]) px0[u][i].load(xp + h * xh + geo.off0[i]);
                        if (geo.in1[i]) px1[u][i].load(xp + h * xh + geo.off1[i]);
                        if (MODE == kNormBwd) {
                            if (geo.in0[i]) pg0[u][i].load(gp + h * gh + geo.off0[i]);
                            if (geo.in1[i]) pg1[u][i].load(gp + h * gh + geo.off1[i]);
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * rows;
                float f0[NV][V], f1[NV][V];
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    px0[u][i].get(f0[i]);
                    px1[u][i].get(f1[i]);
                }
                if (MODE != kRotate) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) ss += f0[i][e] * f0[i][e] + f1[i][e] * f1[i][e];
                    const float r = rsqrtf(group_sum(ss) / (float)D + a.eps);
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            f0[i][e] *= MODE == kNorm ? r * w0[i][e] : r;
                            f1[i][e] *= MODE == kNorm ? r * w1[i][e] : r;
                        }
                    if (MODE == kNormBwd) {
                        float g0[NV][V], g1[NV][V], dot = 0.f;
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            pg0[u][i].get(g0[i]);
                            pg1[u][i].get(g1[i]);
                            rotate<V, INTER>(g0[i], g1[i], cs[i], sn[i], geo.rot0[i], geo.rot1[i]);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                acc0[i][e] += g0[i][e] * f0[i][e];
                                acc1[i][e] += g1[i][e] * f1[i][e];
                                g0[i][e] *= w0[i][e];
                                g1[i][e] *= w1[i][e];
                                dot += g0[i][e] * f0[i][e] + g1[i][e] * f1[i][e];
                            }
                        }
                        dot = group_sum(dot) / (float)D;
#pragma unroll
                        for (int i = 0; i < NV; ++i)
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                f0[i][e] = r * (g0[i][e] - f0[i][e] * dot);
                                f1[i][e] = r * (g1[i][e] - f1[i][e] * dot);
                            }
                    }
                }
                if (h < h_end) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        if (MODE != kNormBwd) rotate<V, INTER>(f0[i], f1[i], cs[i], sn[i], geo.rot0[i], geo.rot1[i]);
                        Pack<T, V> o0, o1;
                        o0.set(f0[i]);
                        o1.set(f1[i]);
                        if (geo.in0[i]) o0.store(yp + h * yh + geo.off0[i]);
                        if (geo.in1[i]) o1.store(yp + h * yh + geo.off1[i]);
                    }
                }
            }
        }
    }
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
                for (int e = 0; e < V; ++e) {
                    if (geo.in0[i]) fold[warp][geo.off0[i] + e] = acc0[i][e];
                    if (geo.in1[i]) fold[warp][geo.off1[i] + e] = acc1[i][e];
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
    int width, log_l, ctas_q, ctas_k, hpu_q, hpu_k;
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

Plan plan(const tt_rotary_args& a, int sms) {
    Plan p;
    p.width = vector_width(a);
    const int chunks = (a.head_dim + 2 * p.width - 1) / (2 * p.width);
    p.log_l = 0;
    while ((1 << p.log_l) < chunks && p.log_l < 5) ++p.log_l;
    const int rows = 32 >> p.log_l;
    const long tokens = (long)a.batch * a.tokens;
    // All heads of a token in one unit share its angles.  With few tokens a unit takes fewer heads, so that the units cover the device.
    auto heads_per_unit = [&](int heads) {
        int per = (heads + rows - 1) / rows;
        while (per > 1 && tokens * ((heads + rows * per - 1) / (rows * per)) < (long)sms * kWarps) per = (per + 1) / 2;
        return rows * (per > 0 ? per : 1);
    };
    p.hpu_q = heads_per_unit(a.q_heads);
    p.hpu_k = heads_per_unit(a.k_heads);
    const long cap = (long)sms * 8;
    auto ctas = [&](int heads, int hpu) {
        if (heads == 0) return 0L;
        const long units = tokens * ((heads + hpu - 1) / hpu), want = (units + kWarps - 1) / kWarps;
        const long most = (cap * heads + a.q_heads + a.k_heads - 1) / (a.q_heads + a.k_heads);
        return want < most ? want : most;
    };
    p.ctas_q = (int)ctas(a.q_heads, p.hpu_q);
    p.ctas_k = (int)ctas(a.k_heads, p.hpu_k);
    return p;
}

template <typename T, int V, int NV, bool INTER>
void launch(const tt_rotary_args& a, const Plan& p, int mode, cudaStream_t st) {
    const int grid = p.ctas_q + p.ctas_k;
    if (mode == kRotate) rotary_kernel<T, V, NV, INTER, kRotate><<<grid, kThreads, 0, st>>>(a, p.log_l, p.ctas_q, p.hpu_q, p.hpu_k);
    else if (mode == kNorm) rotary_kernel<T, V, NV, INTER, kNorm><<<grid, kThreads, 0, st>>>(a, p.log_l, p.ctas_q, p.hpu_q, p.hpu_k);
    else rotary_kernel<T, V, NV, INTER, kNormBwd><<<grid, kThreads, 0, st>>>(a, p.log_l, p.ctas_q, p.hpu_q, p.hpu_k);
}

template <typename T>
void dispatch(const tt_rotary_args& a, const Plan& p, int mode, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    if (p.width == W && a.interleaved) launch<T, W, 1, true>(a, p, mode, st);
    else if (p.width == W) launch<T, W, 1, false>(a, p, mode, st);
    else if (p.width == 2 && a.interleaved) launch<T, 2, 2, true>(a, p, mode, st);
    else if (p.width == 2) launch<T, 2, 2, false>(a, p, mode, st);
    else if (a.interleaved) launch<T, 1, 4, true>(a, p, mode, st);
    else launch<T, 1, 4, false>(a, p, mode, st);
}

int check(const tt_rotary_args* a) {
    if (a == nullptr || a->struct_size != (long)sizeof(tt_rotary_args)) return TT_ERR_ARG;
    if (a->batch <= 0 || a->tokens <= 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads + a->k_heads == 0) return TT_ERR_ARG;
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
    const Plan p = plan(*a, tt_device().sms);
    if (mode == kNormBwd && a->partial_floats < (long)(p.ctas_q + p.ctas_k) * a->head_dim) return TT_ERR_ARG;
    cudaStream_t st = (cudaStream_t)stream;
    if (a->dtype == TT_BF16) dispatch<__nv_bfloat16>(*a, p, mode, st);
    else if (a->dtype == TT_FP16) dispatch<__half>(*a, p, mode, st);
    else dispatch<float>(*a, p, mode, st);
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
    const Plan p = plan(*a, tt_device().sms);
    return (long)(p.ctas_q + p.ctas_k) * a->head_dim;
}
extern "C" int tt_rotary(const tt_rotary_args* a, void* stream) { return run(a, kRotate, stream); }
extern "C" int tt_norm_rotary_fwd(const tt_rotary_args* a, void* stream) { return run(a, kNorm, stream); }
extern "C" int tt_norm_rotary_bwd(const tt_rotary_args* a, void* stream) { return run(a, kNormBwd, stream); }
