// fox_kvq.hip -- quantised caches: rows quantised as they are written, read
// back as floats, and the norm + rotation + store of a pass's queries, keys
// and values in one launch (into a quantised cache or the float ones).
#include "fox_kvq_dev.h"
#include "fox_internal.h"

#define KS_THREADS 256

// ------------------------------------------------------------- quantising

template <int CTRL>
__device__ __forceinline__ float quad_f(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ uint32_t quad_u(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}

// Codes (c + h) of the eight values x of one lane, whose group of 32 is held
// by its four-lane quad (all four active); returns the scale byte.  Every
// decision is exact: (h +- 1/2) d and r d are products of few bits, and
// x - r d, within d / 2 of a border, is a multiple of d 2^-24.
template <int BITS>
__device__ __forceinline__ uint32_t quantise_8(const float x[8], uint32_t code[8])
{
    constexpr int H = 1 << (BITS - 1);
    float hi = 0.0f, lo = 0.0f;
    uint32_t top = 0;                                   // largest |x| as bits: NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; i++) {
        hi = fmaxf(hi, x[i]);
        lo = fminf(lo, x[i]);
        top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    }
    hi = fmaxf(hi, quad_f<0xB1>(hi));
    lo = fminf(lo, quad_f<0xB1>(lo));
    top = max(top, quad_u<0xB1>(top));
    hi = fmaxf(hi, quad_f<0x4E>(hi));
    lo = fminf(lo, quad_f<0x4E>(lo));
    top = max(top, quad_u<0x4E>(top));
    // the scale byte: truncated from the needed scale, which rounding may have
    // put one byte low, then raised while it does not cover the group
    const float need = fmaxf(hi * (1.0f / (H - 0.5f)), lo * (-1.0f / (H + 0.5f))) * 4.0f;
    int b = need < 0x1p-14f ? (int)(need * 0x1p17f)
                            : (int)(__float_as_uint(need) >> 20) - ((127 - 15) << 3);
    b = min(b, KVQ_CAP(BITS));
    float d = kvq_scale((uint32_t)b);
#pragma unroll
    for (int k = 0; k < 2; k++)
        if ((hi > (H - 0.5f) * d || -lo > (H + 0.5f) * d) && b < KVQ_CAP(BITS))
            d = kvq_scale((uint32_t)++b);
    const float inv = b ? 1.0f / d : 0.0f, half = 0.5f * d;
    const bool bad = top >= 0x7F800000u;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float r = rintf(fminf(fmaxf(x[i] * inv, -H - 1.0f), H + 1.0f));
        const float e = __builtin_fmaf(-r, d, x[i]);
        const bool odd = ((int)r & 1) != 0;
        if (e > half || (e == half && odd)) r += 1.0f;
        else if (e < -half || (e == -half && odd)) r -= 1.0f;
        const int c = (int)fminf(fmaxf(r, (float)-H), (float)(H - 1));
        code[i] = bad ? (uint32_t)H : (uint32_t)(c + H);
    }
    return bad ? (uint32_t)KVQ_NAN : (uint32_t)b;
}

// Eight codes as the bytes of a K row or a V chunk.
template <int BITS>
__device__ __forceinline__ void put_codes(uint8_t *dst, const uint32_t code[8])
{
    if (BITS == 4) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= code[e] << (4 * (e / 2 + 4 * (e & 1)));
        *(uint32_t *)dst = w;
    } else {
        uint2 w = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w.x |= code[e] << (8 * e);
            w.y |= code[e + 4] << (8 * e);
        }
        *(uint2 *)dst = w;
    }
}

// ----------------------------------------------------------------- storing

struct StoreArgs {
    const float *k, *v, *q;
    size_t k_stride, v_stride, q_stride, qo_stride;
    float *q_out;
    int n_head, n_head_kv, hd, halves;
    const float *q_norm, *k_norm, *cos_t, *sin_t;
    float eps;
    const uint32_t *pos;
    size_t M, n_ctx;
    uint8_t *cache;             // quantised cache, or
    float *k_cache, *v_cache;   // the float ones
    int wide;                   // rows take 16-byte loads and stores
};

// eight values of a row from column d on (zero past hd)
__device__ __forceinline__ void load_8(float x[8], const float *row, int d, int hd, int wide)
{
    if (wide) {
        *(float4 *)x = *(const float4 *)(row + d);
        *(float4 *)(x + 4) = *(const float4 *)(row + d + 4);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = d + i < hd ? row[d + i] : 0.0f;
}

// The eight pairs j0 .. j0 + 7 of one head's row, or of the norm's weights
// (both laid out by dimension): first members a, second members b; zero past
// the last pair.
__device__ __forceinline__ void load_pairs(float a[8], float b[8], const float *row, int j0, int hd,
                                           int halves, int wide)
{
    const int half = hd >> 1;
    if (wide) {
        float x[16];
#pragma unroll
        for (int u = 0; u < 4; u++)
            *(float4 *)(x + 4 * u) =
                *(const float4 *)(row + (halves ? (u < 2 ? j0 : half + j0 - 8) : 2 * j0) + 4 * u);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            a[i] = halves ? x[i] : x[2 * i];
            b[i] = halves ? x[8 + i] : x[2 * i + 1];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int j = j0 + i;
        a[i] = j < half ? row[halves ? j : 2 * j] : 0.0f;
        b[i] = j < half ? row[halves ? half + j : 2 * j + 1] : 0.0f;
    }
}

__device__ __forceinline__ void store_pairs(float *row, const float a[8], const float b[8], int j0,
                                            int hd, int halves, int wide)
{
    const int half = hd >> 1;
    if (wide) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[halves ? i : 2 * i] = a[i];
            x[halves ? 8 + i : 2 * i + 1] = b[i];
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            *(float4 *)(row + (halves ? (u < 2 ? j0 : half + j0 - 8) : 2 * j0) + 4 * u) =
                *(float4 *)(x + 4 * u);
        return;
    }
    for (int i = 0; i < 8 && j0 + i < half; i++) {
        row[halves ? j0 + i : 2 * (j0 + i)] = a[i];
        row[halves ? half + j0 + i : 2 * (j0 + i) + 1] = b[i];
    }
}

#define KS_PAIRS 16                                    // pair items of a token, at most
#define KS_ROW (KVQ_MAXHD + 4)

// One workgroup per (tile of 32 positions, head): the tile's tokens of a kv
// head (blockIdx.y < n_head_kv), quantised into the tile's record (BITS 4, 8)
// or stored as floats (32); or of a query head.  ROPE: keys and queries are
// normed and rotated on the way, eight pairs of a token an item, so a query
// may be turned in place.  That arithmetic is in double, rounded to float
// once: a key's code may hang on its last bit.  A quantiser's item is eight
// columns of one token, a group of 32 a lane quad.  The V codes of a position
// share their words with other positions', so a workgroup owns its tile's
// words: codes pass through LDS, and words that hold positions outside the
// pass keep those.
template <int BITS, bool ROPE>
__global__ __launch_bounds__(KS_THREADS) void kv_store_k(StoreArgs A)
{
    __shared__ double ss[32 * KS_PAIRS];               // sums of squares, [token][item]
    __shared__ float kf[ROPE && BITS != 32 ? 32 * KS_ROW : 1];   // turned keys, [token][dim]
    __shared__ uint8_t vc[BITS != 32 ? 32 * KS_ROW : 1];   // V codes, [position in tile][dim]
    const int tid = threadIdx.x, head = blockIdx.y, hd = A.hd;
    const size_t p_first = A.pos[0], p_end = min(p_first + A.M, A.n_ctx);
    const size_t t0 = (p_first / KVQ_TILE + blockIdx.x) * KVQ_TILE;
    const size_t lo = max(p_first, t0), hi = min(p_end, t0 + KVQ_TILE);
    if (lo >= hi) return;                              // (uniform)
    const int nt = (int)(hi - lo), r0 = (int)(lo - t0);
    const KvqLayout L = kvq_layout(BITS == 32 ? 8 : BITS, hd);
    const bool is_q = ROPE && head >= A.n_head_kv;
    const int h = is_q ? head - A.n_head_kv : head;
    const size_t tok0 = lo - p_first;                  // first token of the tile
    if constexpr (ROPE) {
        const float *src = is_q ? A.q : A.k, *w = is_q ? A.q_norm : A.k_norm;
        const size_t stride = is_q ? A.q_stride : A.k_stride;
        const int ni = (hd + 15) / 16, half = hd >> 1;
        const size_t kvd = (size_t)A.n_head_kv * hd;
        float a[2][8], b[2][8];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int it = tid + s * KS_THREADS;
            if (it >= nt * ni) continue;
            const int t = it / ni, i = it % ni;
            load_pairs(a[s], b[s], src + (tok0 + t) * stride + (size_t)h * hd, 8 * i, hd, A.halves,
                       A.wide);
            double x = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j++)
                x += (double)a[s][j] * (double)a[s][j] + (double)b[s][j] * (double)b[s][j];
            ss[t * KS_PAIRS + i] = x;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int it = tid + s * KS_THREADS;
            if (it >= nt * ni) continue;
            const int t = it / ni, i = it % ni;
            double inv = 1.0;
            float wa[8], wb[8], ya[8], yb[8];
            if (w) {
                double x = 0.0;
                for (int j = 0; j < ni; j++) x += ss[t * KS_PAIRS + j];
                inv = 1.0 / sqrt(x / (double)hd + (double)A.eps);
                load_pairs(wa, wb, w, 8 * i, hd, A.halves, 0);
            }
            const float *cr = A.cos_t + (lo + t) * half, *sr = A.sin_t + (lo + t) * half;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int at = min(8 * i + j, half - 1);
                double x = (double)a[s][j] * inv, y = (double)b[s][j] * inv;
                if (w) {
                    x *= (double)wa[j];
                    y *= (double)wb[j];
                }
                const double c = cr[at], sn = sr[at];
                ya[j] = (float)(x * c - y * sn);
                yb[j] = (float)(x * sn + y * c);
            }
            float *dst;
            if (is_q) dst = A.q_out + (tok0 + t) * A.qo_stride + (size_t)h * hd;
            else if (BITS == 32) dst = A.k_cache + (lo + t) * kvd + (size_t)h * hd;
            else dst = kf + t * KS_ROW;
            store_pairs(dst, ya, yb, 8 * i, hd, A.halves, is_q ? A.wide : 0);
        }
        if (is_q) return;
        __syncthreads();
    }
    const int no = (hd + 7) / 8, nw = BITS == 32 ? no : L.width / 8;
    if constexpr (BITS == 32) {
        const size_t kvd = (size_t)A.n_head_kv * hd;
        for (int it = tid; it < nt * no; it += KS_THREADS) {
            const int t = it / no, d = it % no * 8;
            const size_t p = lo + t;
            float x[8];
            load_8(x, A.v + (tok0 + t) * A.v_stride + (size_t)h * hd, d, hd, A.wide);
            for (int i = 0; i < 8 && d + i < hd; i++)
                A.v_cache[((p >> 2) * kvd + (size_t)h * hd + d + i) * 4 + (p & 3)] = x[i];
        }
    } else {
        uint8_t *rec = A.cache + ((size_t)h * ((A.n_ctx + KVQ_TILE - 1) / KVQ_TILE) +
                                  t0 / KVQ_TILE) * (size_t)L.record;
        for (int it = tid; it < 2 * nt * nw; it += KS_THREADS) {
            const bool is_v = it >= nt * nw;
            const int u = is_v ? it - nt * nw : it, t = u / nw, o = u % nw, d = 8 * o, r = r0 + t;
            float x[8] = {};
            if (d < hd) {
                if (is_v) {
                    load_8(x, A.v + (tok0 + t) * A.v_stride + (size_t)h * hd, d, hd, A.wide);
                } else if (ROPE) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = d + i < hd ? kf[t * KS_ROW + d + i] : 0.0f;
                } else {
                    load_8(x, A.k + (tok0 + t) * A.k_stride + (size_t)h * hd, d, hd, A.wide);
                }
            }
            uint32_t code[8];
            const uint32_t b = quantise_8<BITS>(x, code);
            const int g = o >> 2;
            if (!is_v) {
                put_codes<BITS>(rec + (size_t)r * (L.width * BITS / 8) + o * BITS, code);
                if ((o & 3) == 0) rec[L.ks + kvq_k_scale(g, r)] = (uint8_t)b;
            } else {
                if ((o & 3) == 0) rec[L.vs + kvq_v_scale(g, r)] = (uint8_t)b;
#pragma unroll
                for (int i = 0; i < 8; i++) vc[r * KS_ROW + d + i] = (uint8_t)code[i];
            }
        }
        __syncthreads();
        // V words: item (dim, chunk) has eight positions
        for (int it = tid; it < L.width * 4; it += KS_THREADS) {
            const int dim = it >> 2, c = it & 3;
            uint8_t *dst = rec + L.v + (size_t)it * BITS;
            uint32_t code[8];
            bool any = false, all = true, on[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = (e & 3) + 4 * c + 16 * (e >> 2);
                on[e] = r >= r0 && r < r0 + nt;
                any |= on[e];
                all &= on[e];
                code[e] = on[e] ? vc[r * KS_ROW + dim] : 0;
            }
            if (!any) continue;
            if (!all) {
                if (BITS == 4) {
                    const uint32_t old = *(const uint32_t *)dst;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (!on[e]) code[e] = old >> (4 * (e / 2 + 4 * (e & 1))) & 15u;
                } else {
                    const uint2 old = *(const uint2 *)dst;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (!on[e]) code[e] = (e < 4 ? old.x >> (8 * e) : old.y >> (8 * e - 32)) & 255u;
                }
            }
            put_codes<BITS>(dst, code);
        }
    }
}

// ----------------------------------------------------------------- reading

// One workgroup per (tile, kv head): rows p0 .. p0 + n - 1 as floats.
template <int BITS>
__global__ __launch_bounds__(KS_THREADS) void kv_read_k(const uint8_t *__restrict__ cache,
                                                        size_t n_ctx, int hd, size_t p0, size_t n,
                                                        float *__restrict__ k, size_t k_stride,
                                                        float *__restrict__ v, size_t v_stride)
{
    constexpr int H = 1 << (BITS - 1);
    const int tid = threadIdx.x, h = blockIdx.y;
    const size_t t0 = (p0 / KVQ_TILE + blockIdx.x) * KVQ_TILE;
    const KvqLayout L = kvq_layout(BITS, hd);
    const uint8_t *rec = cache + ((size_t)h * ((n_ctx + KVQ_TILE - 1) / KVQ_TILE) +
                                  t0 / KVQ_TILE) * (size_t)L.record;
    const int lo = t0 < p0 ? (int)(p0 - t0) : 0;
    const int hi = (int)min((size_t)KVQ_TILE, p0 + n - t0);
    for (int it = tid; it < KVQ_TILE * L.width; it += KS_THREADS) {
        const int r = it / L.width, d = it % L.width, e = d & 7;
        if (r < lo || r >= hi || d >= hd) continue;
        const size_t row = t0 + r - p0;
        if (k) {
            const uint8_t *w = rec + (size_t)r * (L.width * BITS / 8) + (d >> 3) * BITS;
            const int c = BITS == 4 ? (int)(*(const uint32_t *)w >> (4 * (e / 2 + 4 * (e & 1))) & 15u)
                                    : (int)w[e];
            k[row * k_stride + (size_t)h * hd + d] =
                (float)(c - H) * kvq_scale(rec[L.ks + kvq_k_scale(d >> 5, r)]);
        }
        if (v) {
            const int pl = kvq_v_place(r);
            const uint8_t *w = rec + L.v + ((size_t)d * 4 + kvq_v_chunk(r)) * BITS;
            const int c = BITS == 4 ? (int)(*(const uint32_t *)w >> (4 * (pl / 2 + 4 * (pl & 1))) & 15u)
                                    : (int)w[pl];
            v[row * v_stride + (size_t)h * hd + d] =
                (float)(c - H) * kvq_scale(rec[L.vs + kvq_v_scale(d >> 5, r)]);
        }
    }
}

// ------------------------------------------------------------- entry points

// the shape every entry point here takes; `what` names the caller
fox_gpu_status fox_kvq_shape(const char *what, int kv_type, size_t n_ctx, size_t n_head_kv,
                             size_t head_dim)
{
    if (n_ctx == 0 || n_head_kv == 0 || head_dim == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: a zero size", what);
    if (kv_type != FOX_GPU_KV_Q4 && kv_type != FOX_GPU_KV_Q8)
        return fox_fail(FOX_GPU_ERR_UNSUPPORTED, "%s: unknown cache type %d", what, kv_type);
    if (head_dim > KVQ_MAXHD || head_dim % 2)
        return fox_fail(FOX_GPU_ERR_UNSUPPORTED, "%s: head_dim is even and at most %d, not %zu",
                        what, KVQ_MAXHD, head_dim);
    if (n_ctx > (1u << 30) || n_head_kv > 32767)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: %zu positions of %zu kv heads are too many", what,
                        n_ctx, n_head_kv);
    return FOX_GPU_OK;
}

extern "C" size_t fox_gpu_kvq_bytes(int kv_type, size_t n_ctx, size_t n_head_kv, size_t head_dim)
{
    if (fox_kvq_shape("kvq_bytes", kv_type, n_ctx, n_head_kv, head_dim)) return 0;
    return n_head_kv * ((n_ctx + KVQ_TILE - 1) / KVQ_TILE) *
           (size_t)kvq_layout(kv_type, (int)head_dim).record;
}

static bool wide_rows(const float *p, size_t stride) { return (uintptr_t)p % 16 == 0 && stride % 4 == 0; }

template <int BITS, bool ROPE>
static fox_gpu_status launch_store(fox_gpu_ctx *ctx, const StoreArgs &A)
{
    const size_t most = A.M < A.n_ctx ? A.M : A.n_ctx;       // rows that can be stored
    const size_t tiles = (most + KVQ_TILE - 1) / KVQ_TILE + 1;
    FOX_HIP(hipSetDevice(ctx->device));
    hipLaunchKernelGGL((kv_store_k<BITS, ROPE>),
                       dim3((unsigned)tiles, (unsigned)(A.n_head_kv + (ROPE ? A.n_head : 0))),
                       dim3(KS_THREADS), 0, ctx->stream, A);
    FOX_LAUNCHED("kv store");
    return FOX_GPU_OK;
}

extern "C" fox_gpu_status fox_gpu_kvq_write(fox_gpu_ctx *ctx, int kv_type, void *cache,
                                            size_t n_ctx, size_t n_head_kv, size_t head_dim,
                                            const uint32_t *pos, size_t M, const float *k,
                                            size_t k_stride, const float *v, size_t v_stride)
{
    if (!ctx || !cache || !pos || !k || !v || M == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_write: bad argument");
    fox_gpu_status st = fox_kvq_shape("kvq_write", kv_type, n_ctx, n_head_kv, head_dim);
    if (st) return st;
    if (M > n_ctx) return fox_fail(FOX_GPU_ERR_ARG, "kvq_write: %zu rows of %zu", M, n_ctx);
    if (M > 1 && (k_stride < n_head_kv * head_dim || v_stride < n_head_kv * head_dim))
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_write: a stride below the row's width");
    if ((uintptr_t)cache % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_write: the cache must be 16-byte aligned");
    StoreArgs A = {};
    A.k = k;
    A.v = v;
    A.k_stride = k_stride;
    A.v_stride = v_stride;
    A.n_head_kv = (int)n_head_kv;
    A.hd = (int)head_dim;
    A.pos = pos;
    A.M = M;
    A.n_ctx = n_ctx;
    A.cache = (uint8_t *)cache;
    A.wide = head_dim % 8 == 0 && wide_rows(k, M > 1 ? k_stride : 0) && wide_rows(v, M > 1 ? v_stride : 0);
    return kv_type == FOX_GPU_KV_Q4 ? launch_store<4, false>(ctx, A) : launch_store<8, false>(ctx, A);
}

extern "C" fox_gpu_status fox_gpu_kvq_read(fox_gpu_ctx *ctx, int kv_type, const void *cache,
                                           size_t n_ctx, size_t n_head_kv, size_t head_dim,
                                           size_t p0, size_t n, float *k, size_t k_stride,
                                           float *v, size_t v_stride)
{
    if (!ctx || !cache || (!k && !v) || n == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: bad argument");
    fox_gpu_status st = fox_kvq_shape("kvq_read", kv_type, n_ctx, n_head_kv, head_dim);
    if (st) return st;
    if (p0 >= n_ctx || n > n_ctx - p0)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: %zu rows from %zu on are outside the %zu-row "
                        "cache", n, p0, n_ctx);
    if (n > 1 && ((k && k_stride < n_head_kv * head_dim) || (v && v_stride < n_head_kv * head_dim)))
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: a stride below the row's width");
    if ((uintptr_t)cache % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: the cache must be 16-byte aligned");
    const unsigned tiles = (unsigned)((p0 + n - 1) / KVQ_TILE - p0 / KVQ_TILE + 1);
    FOX_HIP(hipSetDevice(ctx->device));
    if (kv_type == FOX_GPU_KV_Q4)
        hipLaunchKernelGGL(kv_read_k<4>, dim3(tiles, (unsigned)n_head_kv), dim3(KS_THREADS), 0,
                           ctx->stream, (const uint8_t *)cache, n_ctx, (int)head_dim, p0, n, k,
                           k_stride, v, v_stride);
    else
        hipLaunchKernelGGL(kv_read_k<8>, dim3(tiles, (unsigned)n_head_kv), dim3(KS_THREADS), 0,
                           ctx->stream, (const uint8_t *)cache, n_ctx, (int)head_dim, p0, n, k,
                           k_stride, v, v_stride);
    FOX_LAUNCHED("kv read");
    return FOX_GPU_OK;
}

// arguments the two norm + rotation entries share
static fox_gpu_status rope_args(const char *what, fox_gpu_ctx *ctx, const float *q, size_t q_stride,
                                float *q_out, size_t qo_stride, const float *k, size_t k_stride,
                                const float *v, size_t v_stride, size_t n_head, size_t n_head_kv,
                                size_t head_dim, size_t M, const float *q_norm, const float *k_norm,
                                float eps, int pairs, const float *cos_t, const float *sin_t,
                                const uint32_t *pos, size_t n_ctx, StoreArgs *A)
{
    const size_t nq = n_head * head_dim, nkv = n_head_kv * head_dim;
    if (!ctx || !q || !q_out || !k || !v || !cos_t || !sin_t || !pos || n_head == 0 || M == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: bad argument", what);
    fox_gpu_status st = fox_kvq_shape(what, FOX_GPU_KV_Q4, n_ctx, n_head_kv, head_dim);
    if (st) return st;
    if (pairs != FOX_GPU_PAIRS_ADJACENT && pairs != FOX_GPU_PAIRS_HALVES)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: unknown pairing %d", what, pairs);
    if (M > FOX_GPU_BATCH_TOKENS) return fox_fail(FOX_GPU_ERR_ARG, "%s: too many tokens", what);
    if (n_head > 32767) return fox_fail(FOX_GPU_ERR_ARG, "%s: too many heads", what);
    if (M > 1 && (q_stride < nq || qo_stride < nq || k_stride < nkv || v_stride < nkv))
        return fox_fail(FOX_GPU_ERR_ARG, "%s: a stride below the row's width", what);
    *A = {};
    A->q = q;
    A->q_stride = q_stride;
    A->q_out = q_out;
    A->qo_stride = qo_stride;
    A->k = k;
    A->k_stride = k_stride;
    A->v = v;
    A->v_stride = v_stride;
    A->n_head = (int)n_head;
    A->n_head_kv = (int)n_head_kv;
    A->hd = (int)head_dim;
    A->halves = pairs == FOX_GPU_PAIRS_HALVES;
    A->q_norm = q_norm;
    A->k_norm = k_norm;
    A->eps = eps;
    A->cos_t = cos_t;
    A->sin_t = sin_t;
    A->pos = pos;
    A->M = M;
    A->n_ctx = n_ctx;
    A->wide = head_dim % 16 == 0 && wide_rows(q, M > 1 ? q_stride : 0) &&
              wide_rows(q_out, M > 1 ? qo_stride : 0) && wide_rows(k, M > 1 ? k_stride : 0) &&
              wide_rows(v, M > 1 ? v_stride : 0);
    return FOX_GPU_OK;
}

extern "C" fox_gpu_status fox_gpu_norm_rope_store(
    fox_gpu_ctx *ctx, const float *q, size_t q_stride, float *q_out, size_t q_out_stride,
    const float *k, size_t k_stride, const float *v, size_t v_stride, size_t n_head,
    size_t n_head_kv, size_t head_dim, size_t M, const float *q_norm, const float *k_norm, float eps,
    int pairs, const float *cos_t, const float *sin_t, const uint32_t *pos, size_t n_ctx,
    float *k_cache, float *v_cache)
{
    StoreArgs A;
    fox_gpu_status st = rope_args("norm_rope_store", ctx, q, q_stride, q_out, q_out_stride, k,
                                  k_stride, v, v_stride, n_head, n_head_kv, head_dim, M, q_norm,
                                  k_norm, eps, pairs, cos_t, sin_t, pos, n_ctx, &A);
    if (st) return st;
    if (!k_cache || !v_cache) return fox_fail(FOX_GPU_ERR_ARG, "norm_rope_store: null cache");
    A.k_cache = k_cache;
    A.v_cache = v_cache;
    return launch_store<32, true>(ctx, A);
}

extern "C" fox_gpu_status fox_gpu_kvq_norm_rope_store(
    fox_gpu_ctx *ctx, const float *q, size_t q_stride, float *q_out, size_t q_out_stride,
    const float *k, size_t k_stride, const float *v, size_t v_stride, size_t n_head,
    size_t n_head_kv, size_t head_dim, size_t M, const float *q_norm, const float *k_norm, float eps,
    int pairs, const float *cos_t, const float *sin_t, const uint32_t *pos, int kv_type,
    void *cache, size_t n_ctx)
{
    StoreArgs A;
    fox_gpu_status st = rope_args("kvq_norm_rope_store", ctx, q, q_stride, q_out, q_out_stride, k,
                                  k_stride, v, v_stride, n_head, n_head_kv, head_dim, M, q_norm,
                                  k_norm, eps, pairs, cos_t, sin_t, pos, n_ctx, &A);
    if (st) return st;
    if ((st = fox_kvq_shape("kvq_norm_rope_store", kv_type, n_ctx, n_head_kv, head_dim))) return st;
    if (!cache || (uintptr_t)cache % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_norm_rope_store: the cache must be 16-byte aligned");
    A.cache = (uint8_t *)cache;
    return kv_type == FOX_GPU_KV_Q4 ? launch_store<4, true>(ctx, A) : launch_store<8, true>(ctx, A);
}
