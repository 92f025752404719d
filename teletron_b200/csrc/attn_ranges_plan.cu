// The plan of an attention in which every query sees one run of the keys: causal, prefix and document masks, lengths of padded
// batches and of caches are all of this form.  Query i at position p = query_start + i sees
//   [start of its document, min(end of its document, keys in use, causal ? max(p + 1, start + prefix) : all)).
// Besides the runs the plan holds, for tiles of 128, what the kernels need to skip and to mask: bounds of the runs of a tile of queries,
// the tiles of queries that see a tile of keys, and the keys that no query sees (their values are never used, not even times 0).
#include <limits.h>

#include "attn_ranges.cuh"

namespace {

using ranges::kTile;
constexpr int kMaxLen = 1 << 30;

struct Rule {
    int q_len, kv_len, causal;
    const int* documents;
    int n_documents;
    long document_stride;
    const int* prefix;
    long prefix_stride;
    int prefix_per_document, prefix_len;
    const int *kv_valid_len, *query_start;
};

__device__ __forceinline__ int2 run_of(const Rule& r, int b, int i) {
    int lo = 0, hi = r.kv_len, start = 0, doc = 0;
    if (r.kv_valid_len != nullptr) hi = min(hi, r.kv_valid_len[b]);
    const long at = (long)i + (r.query_start != nullptr ? r.query_start[b] : 0);
    if (r.documents != nullptr) {
        const int* off = r.documents + b * r.document_stride;
        int l = 0, h = r.n_documents + 1;          // how many offsets are at or below i
        while (l < h) {
            const int m = (l + h) >> 1;
            if (off[m] <= i) l = m + 1;
            else h = m;
        }
        if (l == 0 || l > r.n_documents) return make_int2(0, 0);       // ahead of the first document, or behind the last
        doc = l - 1;
        start = max(off[doc], 0);
        lo = start;
        hi = min(hi, off[l]);
    }
    if (r.causal) {
        int prefix = r.prefix_len;
        if (r.prefix != nullptr) prefix = r.prefix[b * r.prefix_stride + (r.prefix_per_document ? doc : 0)];
        const long reach = max(at + 1, (long)start + max(prefix, 0));
        if (reach < hi) hi = (int)max(reach, 0L);
    }
    return lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
}

__global__ void __launch_bounds__(kTile) runs_kernel(int* __restrict__ plan, const tt_ranges_layout at, const Rule r, int q_tiles) {
    const int b = blockIdx.y, i = blockIdx.x * kTile + threadIdx.x;
    // positions stay within what the distances of 32 bits can hold; beyond that a bias has its end value anyway
    if (i == 0) plan[at.start + b] = r.query_start != nullptr ? max(-kMaxLen, min(kMaxLen, r.query_start[b])) : 0;
    int first_any = INT_MAX, behind_any = 0, first_all = 0, behind_all = INT_MAX;
    if (i < r.q_len) {
        const int2 run = run_of(r, b, i);
        plan[at.first + (long)b * r.q_len + i] = run.x;
        plan[at.behind + (long)b * r.q_len + i] = run.y;
        if (run.x < run.y) {
            first_any = first_all = run.x;
            behind_any = behind_all = run.y;
        } else {            // no tile is whole for a query that sees nothing
            first_all = INT_MAX;
            behind_all = 0;
        }
    }
    __shared__ int4 part[kTile / 32];
    const int4 mine = make_int4(__reduce_min_sync(0xffffffffu, first_any), __reduce_max_sync(0xffffffffu, behind_any),
                                __reduce_max_sync(0xffffffffu, first_all), __reduce_min_sync(0xffffffffu, behind_all));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        int4 t = part[0];
        for (int w = 1; w < kTile / 32; ++w)
            t = make_int4(min(t.x, part[w].x), max(t.y, part[w].y), max(t.z, part[w].z), min(t.w, part[w].w));
        reinterpret_cast<int4*>(plan + at.q_tiles)[(long)b * q_tiles + blockIdx.x] = t;
    }
}

__global__ void __launch_bounds__(kTile) tiles_kernel(int* __restrict__ plan, const tt_ranges_layout at, int q_len, int kv_len, int q_tiles, int k_tiles) {
    const int b = blockIdx.y, j0 = blockIdx.x * kTile, j1 = min(j0 + kTile, kv_len);
    const int4* qt = reinterpret_cast<const int4*>(plan + at.q_tiles) + (long)b * q_tiles;
    __shared__ int lo_s, hi_s, whole_s;
    __shared__ uint32_t seen[4];
    if (threadIdx.x == 0) {
        lo_s = q_tiles;
        hi_s = whole_s = 0;
    }
    if (threadIdx.x < 4) seen[threadIdx.x] = 0u;
    __syncthreads();
    int lo = q_tiles, hi = 0, whole = 0;
    for (int t = threadIdx.x; t < q_tiles; t += kTile) {
        const int4 v = qt[t];
        if (v.x < j1 && v.y > j0) {
            lo = min(lo, t);
            hi = max(hi, t + 1);
            whole |= v.z <= j0 && v.w >= j1;
        }
    }
    if (lo < q_tiles) atomicMin(&lo_s, lo);
    if (hi > 0) atomicMax(&hi_s, hi);
    if (whole) whole_s = 1;
    __syncthreads();
    lo = lo_s;
    hi = hi_s;
    if (!whole_s) {         // no tile of queries sees all: mark what single queries see
        for (long i = (long)lo * kTile + threadIdx.x; i < (long)hi * kTile && i < q_len; i += kTile) {
            const int a = plan[at.first + (long)b * q_len + i] - j0, e = plan[at.behind + (long)b * q_len + i] - j0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t m = ranges::bits_between(a - 32 * w, e - 32 * w);
                if (m & ~seen[w]) atomicOr(&seen[w], m);
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        reinterpret_cast<int2*>(plan + at.k_tiles)[(long)b * k_tiles + blockIdx.x] = make_int2(lo, max(hi, lo));
        uint32_t dead[4];
        for (int w = 0; w < 4; ++w) dead[w] = whole_s ? 0u : ranges::bits_between(-32 * w, j1 - j0 - 32 * w) & ~seen[w];
        reinterpret_cast<uint4*>(plan + at.dead)[(long)b * k_tiles + blockIdx.x] = make_uint4(dead[0], dead[1], dead[2], dead[3]);
        plan[at.dirty + (long)b * k_tiles + blockIdx.x] = (dead[0] | dead[1] | dead[2] | dead[3]) != 0u;
    }
}

}  // namespace

extern "C" void tt_key_ranges_layout(int batch, int q_len, int kv_len, tt_ranges_layout* out) {
    const long qt = (q_len + kTile - 1) / kTile, kt = (kv_len + kTile - 1) / kTile;
    out->q_tiles = 0;
    out->dead = out->q_tiles + batch * qt * 4;
    out->k_tiles = out->dead + batch * kt * 4;
    out->dirty = out->k_tiles + batch * kt * 2;
    out->first = out->dirty + batch * kt;
    out->behind = out->first + (long)batch * q_len;
    out->start = out->behind + (long)batch * q_len;
    out->ints = out->start + batch;
}

extern "C" int tt_key_ranges(int* plan, int batch, int q_len, int kv_len, int causal, const int* documents, int n_documents, long document_stride,
                             const int* prefix, long prefix_stride, int prefix_per_document, int prefix_len, const int* kv_valid_len,
                             const int* query_start, void* stream) {
    if (plan == nullptr || ((uintptr_t)plan & 15) || batch <= 0 || batch > 65535 || q_len <= 0 || kv_len <= 0 || kv_len > kMaxLen || q_len > kMaxLen)
        return TT_ERR_ARG;
    if (documents != nullptr && (n_documents <= 0 || q_len != kv_len || query_start != nullptr)) return TT_ERR_ARG;
    tt_ranges_layout at;
    tt_key_ranges_layout(batch, q_len, kv_len, &at);
    const Rule r = {q_len, kv_len, causal, documents, n_documents, document_stride, prefix, prefix_stride, prefix_per_document && documents != nullptr,
                    prefix_len, kv_valid_len, query_start};
    const int q_tiles = (q_len + kTile - 1) / kTile, k_tiles = (kv_len + kTile - 1) / kTile;
    runs_kernel<<<dim3(q_tiles, batch), kTile, 0, (cudaStream_t)stream>>>(plan, at, r, q_tiles);
    TT_CHECK_LAUNCH();
    tiles_kernel<<<dim3(k_tiles, batch), kTile, 0, (cudaStream_t)stream>>>(plan, at, q_len, kv_len, q_tiles, k_tiles);
    TT_CHECK_LAUNCH();
    return TT_OK;
}

int tt_make_tmap_bhsd(CUtensorMap* out, const void* base, int batch, int heads, int tokens, int head_dim, const long* stride, int box_rows) {
    tt_encode_tiled_fn enc = tt_get_encode_tiled();
    if (enc == nullptr) return TT_ERR_CUDA;
    if ((uintptr_t)base & 15) return TT_ERR_ARG;
    cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)batch};
    cuuint64_t strides[3];
    const long s[3] = {stride[2], stride[1], stride[0]};
    for (int i = 0; i < 3; ++i) {
        if (dims[i + 1] > 1 && (s[i] <= 0 || s[i] % 8)) return TT_ERR_ARG;
        strides[i] = dims[i + 1] > 1 ? (cuuint64_t)s[i] * 2 : (cuuint64_t)head_dim * 2;       // never stepped
    }
    cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TT_OK : TT_ERR_ARG;
}

int tt_ranges_check(const tt_ranges_args* a) {
    if (a == nullptr || a->struct_size != (long)sizeof(tt_ranges_args)) return TT_ERR_ARG;
    if (a->batch <= 0 || a->batch > 65535 || a->q_len <= 0 || a->kv_len <= 0 || a->q_heads <= 0 || a->k_heads <= 0 || a->q_heads % a->k_heads ||
        a->q_heads > 65535 || a->kv_len > kMaxLen || a->q_len > kMaxLen)
        return TT_ERR_ARG;
    if (a->head_dim != 64 && a->head_dim != 128) return TT_ERR_LIMIT;
    if (a->dtype != TT_BF16 && a->dtype != TT_FP16) return TT_ERR_ARG;
    if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->out == nullptr || a->lse == nullptr || a->plan == nullptr || a->status == nullptr)
        return TT_ERR_ARG;
    if (((uintptr_t)a->plan & 15) || ((uintptr_t)a->out & 15) || ((uintptr_t)a->out32 & 15)) return TT_ERR_ARG;
    if (a->max_distance < -1) return TT_ERR_ARG;
    if (a->max_distance > TT_RANGES_MAX_DISTANCE) return TT_ERR_LIMIT;
    if ((a->max_distance >= 0) != (a->bias != nullptr)) return TT_ERR_ARG;
    if (!(a->softcap >= 0.f) || isinf(a->softcap) || isnan(a->scale) || isinf(a->scale)) return TT_ERR_ARG;
    return TT_OK;
}
