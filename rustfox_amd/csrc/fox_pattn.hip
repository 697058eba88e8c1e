// fox_pattn.hip -- attention of one token a row over a paged cache.
#include "fox_paged_dev.h"

#include <cfloat>
#include <cmath>

#define PA_THREADS 256

struct PagedAttnArgs {
    PagedDev C;
    const float *q;
    float *out;
    size_t q_stride, out_stride;
    const uint32_t *length, *seq;
    uint32_t G, M;
    float score;                  // log2(e) / sqrt(hd)
    float *stats;                 // every head's maximum and sum
};

// sum or maximum over the workgroup
template <bool MAX>
__device__ __forceinline__ float block_all(float v, float *lds)
{
    for (int m = 32; m; m >>= 1) {
        const float o = __shfl_xor(v, m);
        v = MAX ? fmaxf(v, o) : v + o;
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int i = 0; i < PA_THREADS / 64; i++) v = i == 0 ? lds[0] : MAX ? fmaxf(v, lds[i]) : v + lds[i];
    __syncthreads();
    return v;
}

// log2 of the softmax's exponent for row r of the head in x
template <bool BF>
__device__ __forceinline__ float score_of(const PagedAttnArgs &A, const float *x, size_t at)
{
    const uint16_t *k = (const uint16_t *)A.C.k + at;
    float s = 0.0f;
    for (uint32_t d = 0; d < A.C.hd; d++) s = __builtin_fmaf(x[d], paged_float<BF>(k[d]), s);
    return s * A.score;
}

// One workgroup per (row, kv head), its query heads in turn: a thread a
// position for the scores, a thread a dimension for the values.
template <bool BF>
__global__ __launch_bounds__(PA_THREADS) void paged_attn_k(PagedAttnArgs A)
{
    __shared__ float x[256], p[PA_THREADS], lds[PA_THREADS / 64];
    __shared__ size_t rows[PA_THREADS];
    const uint32_t kvh = blockIdx.x, t = blockIdx.y, tid = threadIdx.x, hd = A.C.hd;
    const uint32_t s = A.seq ? A.seq[t] : t;
    const uint32_t n = s < A.C.n_seqs ? min(A.length[t], A.C.cap) : 0;
    for (uint32_t g = 0; g < A.G; g++) {
        const size_t head = (size_t)(kvh * A.G + g) * hd;
        if (tid < hd) x[tid] = A.q[t * A.q_stride + head + tid];
        __syncthreads();
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (uint32_t base = 0; base < n; base += PA_THREADS) {
            const uint32_t i = base + tid;
            const size_t at = i < n ? paged_row(A.C, s, kvh, i) : ~(size_t)0;
            const bool seen = at != ~(size_t)0;
            const float sc = seen ? score_of<BF>(A, x, at) : -INFINITY;
            const float mx = fmaxf(m, block_all<true>(seen ? sc : -INFINITY, lds));
            const float f = m == mx ? 1.0f : exp2f(m - mx);
            p[tid] = seen ? exp2f(sc - mx) : 0.0f;
            rows[tid] = at;
            l = l * f + block_all<false>(p[tid], lds);
            if (tid < hd) {
                o *= f;
                for (uint32_t r = 0; r < PA_THREADS && base + r < n; r++)
                    if (rows[r] != ~(size_t)0)
                        o = __builtin_fmaf(p[r], paged_float<BF>(((const uint16_t *)A.C.v)[rows[r] + tid]), o);
            }
            m = mx;
            __syncthreads();
        }
        if (tid < hd) A.out[t * A.out_stride + head + tid] = l == 0.0f ? 0.0f : o / l;
        if (tid == 0) {
            A.stats[2 * (t * A.C.n_kv * A.G + kvh * A.G + g)] = m;
            A.stats[2 * (t * A.C.n_kv * A.G + kvh * A.G + g) + 1] = l;
        }
        __syncthreads();
    }
}

// the group's weights of a row, summed before they are added to what it has
template <bool BF>
__global__ __launch_bounds__(PA_THREADS) void paged_weigh_k(PagedAttnArgs A)
{
    const uint32_t kvh = blockIdx.x, t = blockIdx.y;
    const uint32_t n = min(A.length[t], A.C.cap);
    float *weight = A.C.weight + ((size_t)t * A.C.n_kv + kvh) * A.C.cap;
    for (uint32_t i = threadIdx.x; i < n; i += PA_THREADS) {
        const size_t at = paged_row(A.C, t, kvh, i);
        if (at == ~(size_t)0) continue;
        float sum = 0.0f;
        for (uint32_t g = 0; g < A.G; g++) {
            const float *ml = A.stats + 2 * (t * A.C.n_kv * A.G + kvh * A.G + g);
            const float *x = A.q + t * A.q_stride + (size_t)(kvh * A.G + g) * A.C.hd;
            sum += exp2f(score_of<BF>(A, x, at) - ml[0]) / ml[1];
        }
        weight[i] += sum;
    }
}

extern "C" fox_gpu_status fox_gpu_paged_attention(fox_gpu_ctx *ctx, const fox_gpu_paged *cache, float *out,
                                                  size_t out_stride, const float *q, size_t q_stride, size_t n_head,
                                                  size_t M, const uint32_t *length, const uint32_t *seq, int weigh)
{
    if (!ctx || !out || !q || !length || n_head == 0 || M == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: bad argument");
    PagedAttnArgs A = {};
    fox_gpu_status st = fox_paged_check("paged_attention", cache, weigh != 0, &A.C);
    if (st) return st;
    if (n_head % cache->n_head_kv || n_head > 65535)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: %zu heads over %zu kv heads", n_head, cache->n_head_kv);
    if (M > FOX_GPU_BATCH_TOKENS) return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: too many tokens");
    const size_t width = n_head * cache->head_dim;
    if (M > 1 && (q_stride < width || out_stride < width))
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: a stride below the row's width");
    if (!seq && M > cache->n_seqs)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: %zu tokens for %zu sequences", M, cache->n_seqs);
    if (weigh && seq)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: weights are added to for a token of each sequence, "
                        "without seq");
    A.q = q;
    A.out = out;
    A.q_stride = q_stride;
    A.out_stride = out_stride;
    A.length = length;
    A.seq = seq;
    A.G = (uint32_t)(n_head / cache->n_head_kv);
    A.M = (uint32_t)M;
    A.score = (float)(1.4426950408889634 / std::sqrt((double)cache->head_dim));
    if ((st = fox_ws_reserve(ctx, M * n_head * 2 * sizeof(float)))) return st;
    A.stats = (float *)ctx->ws;
    FOX_HIP(hipSetDevice(ctx->device));
    const dim3 grid((unsigned)cache->n_head_kv, (unsigned)M);
    if (cache->type == FOX_GPU_BF16)
        paged_attn_k<true><<<grid, dim3(PA_THREADS), 0, ctx->stream>>>(A);
    else
        paged_attn_k<false><<<grid, dim3(PA_THREADS), 0, ctx->stream>>>(A);
    if (weigh) {
        if (cache->type == FOX_GPU_BF16)
            paged_weigh_k<true><<<grid, dim3(PA_THREADS), 0, ctx->stream>>>(A);
        else
            paged_weigh_k<false><<<grid, dim3(PA_THREADS), 0, ctx->stream>>>(A);
    }
    FOX_LAUNCHED("paged_attention");
    return FOX_GPU_OK;
}
