// fox_kvattn.hip -- causal attention over a quantised cache.
#include "fox_kvq_dev.h"
#include "fox_internal.h"

#include <cfloat>
#include <cmath>

// One workgroup per (query head, token): a position a thread for the scores,
// a running maximum and sum, a column a thread for the values.
template <int BITS>
__global__ __launch_bounds__(256) void kv_attn_plain(float *out, size_t out_stride, const float *q,
                                                     size_t q_stride, const uint8_t *cache,
                                                     int n_head, int n_head_kv, int hd,
                                                     const uint32_t *pos, size_t n_ctx)
{
    constexpr int H = 1 << (BITS - 1);
    __shared__ float qs[KVQ_MAXHD], ps[256], red[4];
    const int tid = threadIdx.x, h = blockIdx.x, t = blockIdx.y, kvh = h / (n_head / n_head_kv);
    const size_t upto = min((size_t)pos[0] + (size_t)t + 1, n_ctx);
    const KvqLayout L = kvq_layout(BITS, hd);
    const uint8_t *base = cache + (size_t)kvh * ((n_ctx + KVQ_TILE - 1) / KVQ_TILE) * L.record;
    if (tid < hd) qs[tid] = q[(size_t)t * q_stride + (size_t)h * hd + tid];
    __syncthreads();
    float m = -FLT_MAX, l = 0.0f, o = 0.0f;
    for (size_t p0 = 0; p0 < upto; p0 += 256) {
        const size_t p = p0 + tid;
        float s = -INFINITY;
        if (p < upto) {
            const uint8_t *rec = base + p / KVQ_TILE * L.record;
            const int r = (int)(p % KVQ_TILE);
            s = 0.0f;
            for (int d = 0; d < hd; d++) {
                const int e = d & 7;
                const uint8_t *w = rec + (size_t)r * (L.width * BITS / 8) + (d >> 3) * BITS;
                const int c = BITS == 4 ? (int)(*(const uint32_t *)w >> (4 * (e / 2 + 4 * (e & 1))) & 15u)
                                        : (int)w[e];
                s = __builtin_fmaf(qs[d], (float)(c - H) * kvq_scale(rec[L.ks + kvq_k_scale(d >> 5, r)]), s);
            }
            s /= sqrtf((float)hd);
        }
        float mx = s;
        for (int k = 32; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float e = p < upto ? expf(s - mn) : 0.0f, f = expf(m - mn);
        ps[tid] = e;
        float sum = e;
        for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = sum;
        __syncthreads();
        l = l * f + (red[0] + red[1] + red[2] + red[3]);
        m = mn;
        if (tid < hd) {
            o *= f;
            const int n = (int)min((size_t)256, upto - p0);
            for (int i = 0; i < n; i++) {
                const uint8_t *rec = base + (p0 + i) / KVQ_TILE * L.record;
                const int r = (int)((p0 + i) % KVQ_TILE), pl = kvq_v_place(r);
                const uint8_t *w = rec + L.v + ((size_t)tid * 4 + kvq_v_chunk(r)) * BITS;
                const int c = BITS == 4 ? (int)(*(const uint32_t *)w >> (4 * (pl / 2 + 4 * (pl & 1))) & 15u)
                                        : (int)w[pl];
                o = __builtin_fmaf(ps[i], (float)(c - H) * kvq_scale(rec[L.vs + kvq_v_scale(tid >> 5, r)]), o);
            }
        }
        __syncthreads();
    }
    if (tid < hd) out[(size_t)t * out_stride + (size_t)h * hd + tid] = o / l;
}

extern "C" fox_gpu_status fox_gpu_kvq_attention(fox_gpu_ctx *ctx, float *out, size_t out_stride,
                                                const float *q, size_t q_stride, int kv_type,
                                                const void *cache, size_t n_head, size_t n_head_kv,
                                                size_t head_dim, size_t M, const uint32_t *pos,
                                                size_t n_ctx)
{
    if (!ctx || !out || !q || !cache || !pos || n_head == 0 || M == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: bad argument");
    fox_gpu_status st = fox_kvq_shape("kvq_attention", kv_type, n_ctx, n_head_kv, head_dim);
    if (st) return st;
    if (n_head % n_head_kv || n_head > 65535)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: %zu heads over %zu kv heads", n_head,
                        n_head_kv);
    if (M > FOX_GPU_BATCH_TOKENS) return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: too many tokens");
    if (M > 1 && (q_stride < n_head * head_dim || out_stride < n_head * head_dim))
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: a stride below the row's width");
    if ((uintptr_t)cache % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: the cache must be 16-byte aligned");
    FOX_HIP(hipSetDevice(ctx->device));
    const dim3 grid((unsigned)n_head, (unsigned)M);
    if (kv_type == FOX_GPU_KV_Q4)
        hipLaunchKernelGGL(kv_attn_plain<4>, grid, dim3(256), 0, ctx->stream, out, out_stride, q,
                           q_stride, (const uint8_t *)cache, (int)n_head, (int)n_head_kv,
                           (int)head_dim, pos, n_ctx);
    else
        hipLaunchKernelGGL(kv_attn_plain<8>, grid, dim3(256), 0, ctx->stream, out, out_stride, q,
                           q_stride, (const uint8_t *)cache, (int)n_head, (int)n_head_kv,
                           (int)head_dim, pos, n_ctx);
    FOX_LAUNCHED("kvq attention");
    return FOX_GPU_OK;
}
