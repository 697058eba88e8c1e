// fox_kvq.hip -- quantised caches: rows quantised as they are written, read
// back as floats, and the norm + rotation + store of a pass's queries, keys
// and values in one launch (into a quantised cache or the float ones).
#include "fox_kvq_dev.h"
#include "fox_internal.h"

typedef float f4v __attribute__((ext_vector_type(4)));

#define KS_THREADS 256
#define KVQ_MAXROWS (1u << 28)       // rows of one call (2^32 threads are a launch's most)

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

// Codes (c + h), a byte each, of the eight values x of one lane, whose group of
// 32 is held by its four-lane quad (all four active); returns the scale byte.
//
// x / d is rounded by adding 1.5 2^23 + h, which leaves the code in the float's
// low byte.  That quotient, from an approximate 1 / d, is off by less than
// h 2^-21, so only codes that close to a half (and saturating groups, and ones
// that are not finite) take the exact way: x against the borders (r +- 1/2) d,
// where r d has few bits and x - r d is a multiple of d 2^-24.
template <int BITS>
__device__ __forceinline__ uint32_t quantise_8(const float x[8], uint32_t code[2])
{
    constexpr int H = 1 << (BITS - 1);
    constexpr float MAGIC = 12582912.0f + H, NEAR = 0.5f - H * 0x1p-21f;
    float hi = fmaxf(x[0], 0.0f), lo = fminf(x[0], 0.0f), sum = x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        hi = fmaxf(hi, x[i]);
        lo = fminf(lo, x[i]);
        sum += x[i];
    }
    hi = fmaxf(hi, quad_f<0xB1>(hi));
    lo = fminf(lo, quad_f<0xB1>(lo));
    sum += quad_f<0xB1>(sum);
    hi = fmaxf(hi, quad_f<0x4E>(hi));
    lo = fminf(lo, quad_f<0x4E>(lo));
    sum += quad_f<0x4E>(sum);
    // the scale byte: truncated from the needed scale, which rounding may have
    // put one byte low, then raised while it does not cover the group
    const float need = fmaxf(hi * (1.0f / (H - 0.5f)), lo * (-1.0f / (H + 0.5f))) * 4.0f;
    int b = need < 0x1p-14f ? (int)(need * 0x1p17f)
                            : (int)(__float_as_uint(need) >> 20) - ((127 - 15) << 3);
    b = min(b, KVQ_CAP(BITS));
    float d = kvq_scale((uint32_t)b);
    bool over = hi > (H - 0.5f) * d || -lo > (H + 0.5f) * d;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        b += over && b < KVQ_CAP(BITS);
        d = kvq_scale((uint32_t)b);
        over = hi > (H - 0.5f) * d || -lo > (H + 0.5f) * d;
    }
    const float inv = b ? __builtin_amdgcn_rcpf(d) : 0.0f;
    uint32_t c[8];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = __builtin_fmaf(x[i], inv, MAGIC);
        off = fmaxf(off, fabsf(__builtin_fmaf(x[i], inv, MAGIC - y)));
        c[i] = __float_as_uint(y);
    }
    const bool odd_sum = !(fabsf(sum) <= 3.4028235e38f);
    if (off > NEAR || over || odd_sum) {
        const float half = 0.5f * d;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float r = rintf(fminf(fmaxf(x[i] * inv, -H - 1.0f), H + 1.0f));
            const float e = __builtin_fmaf(-r, d, x[i]);
            const bool odd = ((int)r & 1) != 0;
            if (e > half || (e == half && odd)) r += 1.0f;
            else if (e < -half || (e == -half && odd)) r -= 1.0f;
            c[i] = (uint32_t)((int)fminf(fmaxf(r, (float)-H), (float)(H - 1)) + H);
        }
    }
    bool bad = false;
    if (odd_sum) {                                      // (the quad has one sum: all of it or none is here)
        uint32_t top = 0;                               // largest |x| as bits: NaN above infinity
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        top = max(top, quad_u<0xB1>(top));
        top = max(top, quad_u<0x4E>(top));
        bad = top >= 0x7F800000u;
        if (bad)
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = H;
    }
#pragma unroll
    for (int k = 0; k < 2; k++)
        code[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * k + 3], c[4 * k + 2], 0x0C0C0400u),
                                        __builtin_amdgcn_perm(c[4 * k + 1], c[4 * k], 0x0C0C0400u),
                                        0x05040100u);
    return bad ? (uint32_t)KVQ_NAN : (uint32_t)b;
}

// Eight codes in bytes as they are held in a K row.
template <int BITS>
__device__ __forceinline__ void put_codes(uint8_t *dst, const uint32_t code[2])
{
    if (BITS == 4) {
        // values 0 2 4 6 to the nibbles of the lower half, 1 3 5 7 of the upper
        const uint32_t even = __builtin_amdgcn_perm(code[1], code[0], 0x06040200u);
        const uint32_t odd = __builtin_amdgcn_perm(code[1], code[0], 0x07050301u);
        *(uint32_t *)dst = __builtin_amdgcn_perm(odd | odd >> 4, even | even >> 4, 0x06040200u);
    } else {
        *(uint2 *)dst = uint2{code[0], code[1]};
    }
}

// column k of the 4x4 bytes a, b, c, d for k = 0..3
__device__ __forceinline__ void transpose_4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t o[4])
{
    const uint32_t p = __builtin_amdgcn_perm(b, a, 0x05010400u), q = __builtin_amdgcn_perm(b, a, 0x07030602u);
    const uint32_t r = __builtin_amdgcn_perm(d, c, 0x05010400u), s = __builtin_amdgcn_perm(d, c, 0x07030602u);
    o[0] = __builtin_amdgcn_perm(r, p, 0x05040100u);
    o[1] = __builtin_amdgcn_perm(r, p, 0x07060302u);
    o[2] = __builtin_amdgcn_perm(s, q, 0x05040100u);
    o[3] = __builtin_amdgcn_perm(s, q, 0x07060302u);
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
    bool wide;                  // rows take 16-byte loads and stores
};

// eight values of a row from column d on (zero past hd)
__device__ __forceinline__ void load_8(float x[8], const float *row, int d, int hd, bool wide)
{
    if (wide) {
        const bool in = d < hd;                        // (whole eights)
        *(float4 *)x = in ? *(const float4 *)(row + d) : float4{0, 0, 0, 0};
        *(float4 *)(x + 4) = in ? *(const float4 *)(row + d + 4) : float4{0, 0, 0, 0};
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = d + i < hd ? row[d + i] : 0.0f;
}

// The eight pairs j0 .. j0 + 7 of one head's row, or of the norm's weights
// (both laid out by dimension): first members a, second members b; zero past
// the last pair.
__device__ __forceinline__ void load_pairs(float a[8], float b[8], const float *row, int j0, int hd,
                                           int halves, bool wide)
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
                                            int hd, int halves, bool wide)
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

// One workgroup per (tile of 32 positions, row of heads): the tile's tokens of
// one head's keys (blockIdx.y < n_head_kv), values (< 2 n_head_kv) or queries.
// Keys and values are quantised into the tile's record (BITS 4, 8) or stored
// as floats (32).  ROPE: keys and queries are normed and rotated on the way, eight
// pairs of a token an item, so a query may be turned in place.  That
// arithmetic is in double, rounded to float once: a key's code may hang on
// its last bit (the vector unit adds and multiplies doubles at the rate of
// floats).  A quantiser's item is eight columns of one token, a group of 32 a
// lane quad.  The V codes of a position share their words with other
// positions', so a workgroup owns its tile's words: codes pass through LDS, and
// words that hold positions outside the pass keep those.
// HD: head_dim where rows take 16-byte loads and head_dim is a stored width, else
// 0: any head_dim, by 16 bytes where that is a multiple of 16.
template <int BITS, bool ROPE, int HD>
__global__ __launch_bounds__(KS_THREADS) void kv_store_k(StoreArgs A)
{
    constexpr int LROW = (HD ? HD : KVQ_MAXHD) + 4;
    __shared__ double ss[ROPE ? 32 * KS_PAIRS : 1];    // sums of squares, [token][item]
    // turned keys [token][dim], or V codes [position in tile][dim]
    __shared__ __attribute__((aligned(16))) uint8_t lds[BITS != 32 ? 32 * LROW * (ROPE ? 4 : 1) : 16];
    const int tid = threadIdx.x, hd = HD ? HD : A.hd;
    const bool wide = HD || (A.wide && hd % 16 == 0);
    const size_t p_first = A.pos[0], p_end = min(p_first + A.M, A.n_ctx);
    const size_t t0 = (p_first / KVQ_TILE + blockIdx.x) * KVQ_TILE;
    const size_t lo = max(p_first, t0), hi = min(p_end, t0 + KVQ_TILE);
    if (lo >= hi) return;                              // (uniform)
    const int nt = (int)(hi - lo), r0 = (int)(lo - t0);
    const KvqLayout L = kvq_layout(BITS == 32 ? 8 : BITS, hd);
    const int part = blockIdx.y < A.n_head_kv ? 0 : blockIdx.y < 2 * A.n_head_kv ? 1 : 2;
    const bool is_q = part == 2;
    const int h = blockIdx.y - part * A.n_head_kv;
    const size_t tok0 = lo - p_first;                  // first token of the tile
    const size_t kvd = (size_t)A.n_head_kv * hd;
    if constexpr (ROPE) {
        if (part != 1) {
            const float *src = is_q ? A.q : A.k, *w = is_q ? A.q_norm : A.k_norm;
            const size_t stride = is_q ? A.q_stride : A.k_stride;
            const int ni = (hd + 15) / 16, half = hd >> 1;
            constexpr int SLOTS = HD ? (2 * HD + KS_THREADS - 1) / KS_THREADS : 2;
            float a[SLOTS][8], b[SLOTS][8];
#pragma unroll
            for (int s = 0; s < SLOTS; s++) {
                const int it = tid + s * KS_THREADS;
                if (it >= nt * ni) continue;
                const int t = it / ni, i = it % ni;
                load_pairs(a[s], b[s], src + (tok0 + t) * stride + (size_t)h * hd, 8 * i, hd, A.halves,
                           wide);
                double x = 0.0;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    x += (double)a[s][j] * (double)a[s][j] + (double)b[s][j] * (double)b[s][j];
                ss[t * KS_PAIRS + i] = x;
            }
            __syncthreads();
#pragma unroll
            for (int s = 0; s < SLOTS; s++) {
                const int it = tid + s * KS_THREADS;
                if (it >= nt * ni) continue;
                const int t = it / ni, i = it % ni;
                float wa[8], wb[8], cs[8], sn[8], ya[8], yb[8];
                const float *cr = A.cos_t + (lo + t) * half, *sr = A.sin_t + (lo + t) * half;
                if (w) load_pairs(wa, wb, w, 8 * i, hd, A.halves, wide);
                load_8(cs, cr, 8 * i, half, wide);
                load_8(sn, sr, 8 * i, half, wide);
                double inv = 1.0;
                if (w) {
                    double x = 0.0;
#pragma unroll
                    for (int j = 0; j < (HD ? HD / 16 : KS_PAIRS); j++)
                        if (HD || j < ni) x += ss[t * KS_PAIRS + j];
                    inv = 1.0 / sqrt(x / (double)hd + (double)A.eps);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    double x = (double)a[s][j] * inv, y = (double)b[s][j] * inv;
                    if (w) {
                        x *= (double)wa[j];
                        y *= (double)wb[j];
                    }
                    ya[j] = (float)(x * (double)cs[j] - y * (double)sn[j]);
                    yb[j] = (float)(x * (double)sn[j] + y * (double)cs[j]);
                }
                float *dst;
                if (is_q) dst = A.q_out + (tok0 + t) * A.qo_stride + (size_t)h * hd;
                else if (BITS == 32) dst = A.k_cache + (lo + t) * kvd + (size_t)h * hd;
                else dst = (float *)lds + t * LROW;
                store_pairs(dst, ya, yb, 8 * i, hd, A.halves, wide);
            }
            if (is_q || BITS == 32) return;
            __syncthreads();
        }
    }
    if constexpr (BITS == 32) {                        // values: a column of four positions
        const float *row = A.v + tok0 * A.v_stride + (size_t)h * hd;
        for (int it = tid; it < KVQ_TILE / 4 * hd; it += KS_THREADS) {
            const int r = it / hd * 4 - r0, c = it % hd;   // first token of the four
            if (r <= -4 || r >= nt) continue;
            float *dst = A.v_cache + (((lo + r) >> 2) * kvd + (size_t)h * hd + c) * 4;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (r + i >= 0 && r + i < nt) x[i] = row[(size_t)(r + i) * A.v_stride + c];
            if (wide && r >= 0 && r + 4 <= nt) {
                *(float4 *)dst = *(const float4 *)x;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r + i >= 0 && r + i < nt) dst[i] = x[i];
            }
        }
    } else {
        const int nw = HD ? HD / 8 : L.width / 8;
        uint8_t *rec = A.cache + ((size_t)h * ((A.n_ctx + KVQ_TILE - 1) / KVQ_TILE) +
                                  t0 / KVQ_TILE) * (size_t)L.record;
        const float *row = part ? A.v + tok0 * A.v_stride : A.k + tok0 * A.k_stride;
        const size_t stride = part ? A.v_stride : A.k_stride;
        // V words: item (four dims, chunk).  Those of a tile partly outside the
        // pass are read early, and keep what `on` leaves out
        constexpr int NWORD = (HD ? HD : KVQ_MAXHD) / KS_THREADS + (HD % KS_THREADS != 0);
        uint32_t old[NWORD][4][BITS / 4], on[BITS / 4] = {};
        const bool whole = nt == KVQ_TILE;
        {
            // (a thread's items have one chunk: KS_THREADS is a multiple of 4)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = kvq_v_pos(tid & 3, e);
                if (r < r0 || r >= r0 + nt) continue;
                if (BITS == 4) on[0] |= 15u << (4 * (e / 2 + 4 * (e & 1)));
                else on[(e >> 2) & (BITS / 4 - 1)] |= 255u << (8 * (e & 3));
            }
        }
        if (part && !whole) {
#pragma unroll
            for (int s = 0; s < NWORD; s++) {
                const int it = tid + s * KS_THREADS;
                if (it >= L.width || !(on[0] | on[BITS / 4 - 1])) continue;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    __builtin_memcpy(old[s][k], __builtin_assume_aligned(
                        rec + L.v + (size_t)((it & ~3) * 4 + 4 * k + (it & 3)) * BITS, BITS), BITS);
            }
        }
        // (a thread's loads together)
        constexpr int IT = HD ? (4 * HD + KS_THREADS - 1) / KS_THREADS : 1;
        for (int it0 = tid; it0 < nt * nw; it0 += IT * KS_THREADS) {
            float x[IT][8];
#pragma unroll
            for (int u = 0; u < IT; u++) {
                const int it = min(it0 + u * KS_THREADS, nt * nw - 1), t = it / nw, d = it % nw * 8;
                if (ROPE && !part) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        x[u][i] = HD || d + i < hd ? ((const float *)lds)[t * LROW + d + i] : 0.0f;
                } else {
                    load_8(x[u], row + t * stride + (size_t)h * hd, d, hd, wide);
                }
            }
#pragma unroll
            for (int u = 0; u < IT; u++) {
                const int it = it0 + u * KS_THREADS, t = it / nw, o = it % nw, r = r0 + t, g = o >> 2;
                if (it >= nt * nw) break;
                uint32_t code[2];
                const uint32_t b = quantise_8<BITS>(x[u], code);
                if (!part) {
                    put_codes<BITS>(rec + (size_t)r * (L.width * BITS / 8) + o * BITS, code);
                    if ((o & 3) == 0) rec[L.ks + kvq_k_scale(g, r)] = (uint8_t)b;
                } else {
                    if ((o & 3) == 0) rec[L.vs + kvq_v_scale(g, r)] = (uint8_t)b;
                    uint32_t *dst = (uint32_t *)(lds + r * LROW + 8 * o);
                    dst[0] = code[0];
                    dst[1] = code[1];
                }
            }
        }
        if (!part) return;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < NWORD; s++) {
            const int it = tid + s * KS_THREADS;
            if (it >= L.width || !(on[0] | on[BITS / 4 - 1])) continue;
            const int d0 = it & ~3, c = it & 3;
            uint32_t w[8], o[2][4];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                w[e] = *(const uint32_t *)(lds + kvq_v_pos(c, e) * LROW + d0);
                if (BITS == 4 && !whole) w[e] &= 0x0F0F0F0Fu;    // (rows outside the pass: anything)
            }
            if (BITS == 4)
                transpose_4(w[0] | w[2] << 4, w[4] | w[6] << 4, w[1] | w[3] << 4, w[5] | w[7] << 4, o[0]);
            else {
                transpose_4(w[0], w[1], w[2], w[3], o[0]);
                transpose_4(w[4], w[5], w[6], w[7], o[1]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t v[BITS / 4];
#pragma unroll
                for (int i = 0; i < BITS / 4; i++)
                    v[i] = whole ? o[i][k] : (o[i][k] & on[i]) | (old[s][k][i] & ~on[i]);
                __builtin_memcpy(__builtin_assume_aligned(rec + L.v + (size_t)((d0 + k) * 4 + c) * BITS, BITS),
                                 v, BITS);
            }
        }
    }
}

// ----------------------------------------------------------------- reading

// value e of eight
template <int BITS>
__device__ __forceinline__ int code_of(const uint32_t *w, int e)
{
    return BITS == 4 ? (int)(w[0] >> (4 * (e / 2 + 4 * (e & 1))) & 15u)
                     : (int)(w[e >> 2] >> (8 * (e & 3)) & 255u);
}

__device__ __forceinline__ void put_quad(float *dst, const float x[4], int d, int hd, bool wide)
{
    if (wide) {
        // (past the caches: 16077 rows of 8 heads of 128, into three outputs in turn, take 34.8 us
        // instead of 44.8; into one output alone both ways 26.5)
        __builtin_nontemporal_store(*(const f4v *)x, (f4v *)(dst + d));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (d + i < hd) dst[d + i] = x[i];
}

// One workgroup per (tile, kv head): rows p0 .. p0 + n - 1 as floats.  Half of
// the waves take the keys, an item four columns of a row; half the values, an
// item four columns of a chunk's eight rows: 8 x 16 bytes stored by a thread
// either way (head_dim 128), whole 512-byte row pieces by half a wave.
template <int BITS, int HD>
__global__ __launch_bounds__(KS_THREADS) void kv_read_k(const uint8_t *__restrict__ cache,
                                                        size_t n_ctx, int hd_, size_t p0, size_t n,
                                                        float *__restrict__ k, size_t k_stride,
                                                        float *__restrict__ v, size_t v_stride,
                                                        bool wide_)
{
    constexpr int H = 1 << (BITS - 1), HALF_WG = KS_THREADS / 2;
    const int hd = HD ? HD : hd_, h = blockIdx.y;
    const bool wide = HD || (wide_ && hd % 4 == 0);
    const size_t t0 = (p0 / KVQ_TILE + blockIdx.x) * KVQ_TILE;
    const KvqLayout L = kvq_layout(BITS, hd);
    const uint8_t *rec = cache + ((size_t)h * ((n_ctx + KVQ_TILE - 1) / KVQ_TILE) +
                                  t0 / KVQ_TILE) * (size_t)L.record;
    const int lo = t0 < p0 ? (int)(p0 - t0) : 0;
    const int hi = (int)min((size_t)KVQ_TILE, p0 + n - t0);
    const int tid = threadIdx.x & (HALF_WG - 1);
    if (threadIdx.x < HALF_WG) {
        if (!k) return;
        const int nq = HD ? HD / 4 : (hd + 3) / 4;
        k += (t0 - p0) * k_stride + (size_t)h * hd;    // (row r of the tile; may wrap, r >= lo does not)
#pragma unroll 4
        for (int it = tid; it < KVQ_TILE * nq; it += HALF_WG) {
            const int r = it / nq, q = it % nq;
            // four columns: half of a dword's nibbles, or a dword's bytes
            uint32_t w = *(const uint32_t *)(rec + (size_t)r * (L.width * BITS / 8) +
                                             (BITS == 4 ? (q >> 1) * 4 : q * 4));
            if (BITS == 4) w >>= 8 * (q & 1);
            const float d = kvq_scale(rec[L.ks + kvq_k_scale(q >> 3, r)]);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = (float)(code_of<BITS>(&w, e) - H) * d;
            if (r >= lo && r < hi) put_quad(k + (size_t)r * k_stride, x, 4 * q, hd, wide);
        }
    } else {
        if (!v) return;
        const int nq = HD ? HD / 4 : (hd + 3) / 4;
        v += (t0 - p0) * v_stride + (size_t)h * hd;
        for (int it = tid; it < 4 * nq; it += HALF_WG) {
            const int c = it / nq, d0 = it % nq * 4;
            uint32_t w[4][2];
#pragma unroll
            for (int i = 0; i < 4; i++)
                __builtin_memcpy(w[i], __builtin_assume_aligned(rec + L.v + ((size_t)(d0 + i) * 4 + c) * BITS, BITS), BITS);
            const uint2 s = *(const uint2 *)(rec + L.vs + (d0 >> 5) * 32 + c * 8);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = kvq_v_pos(c, e);
                const float d = kvq_scale((e < 4 ? s.x : s.y) >> (8 * (e & 3)) & 255u);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = (float)(code_of<BITS>(w[i], e) - H) * d;
                if (r >= lo && r < hi) put_quad(v + (size_t)r * v_stride, x, d0, hd, wide);
            }
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

// A kernel's instance for a head_dim that is a stored width, where rows take
// 16-byte accesses (wide), else the one for any.
#define FOX_BY_WIDTH(wide, hd, F)                                                            \
    (!(wide) ? F(0) : (hd) == 32 ? F(32) : (hd) == 64 ? F(64) : (hd) == 96 ? F(96)           \
                    : (hd) == 128 ? F(128) : (hd) == 192 ? F(192) : (hd) == 256 ? F(256) : F(0))

template <int BITS, bool ROPE>
static fox_gpu_status launch_store(fox_gpu_ctx *ctx, StoreArgs A)
{
    const size_t most = A.M < A.n_ctx ? A.M : A.n_ctx;       // rows that can be stored
    // (the position is not known here: the rows may begin at a tile's end)
    const size_t tiles = (most + KVQ_TILE - 2) / KVQ_TILE + 1;
#define FOX_STORE(hd) ((const void *)kv_store_k<BITS, ROPE, hd>)
    const void *k = FOX_BY_WIDTH(A.wide, A.hd, FOX_STORE);
#undef FOX_STORE
    void *args[] = {&A};
    FOX_HIP(hipSetDevice(ctx->device));
    FOX_HIP(hipLaunchKernel(k, dim3((unsigned)tiles, (unsigned)(2 * A.n_head_kv + (ROPE ? A.n_head : 0))),
                            dim3(KS_THREADS), args, 0, ctx->stream));
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
    if (M > n_ctx || M > KVQ_MAXROWS)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_write: %zu rows of %zu, at most %u a call", M, n_ctx,
                        KVQ_MAXROWS);
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
    A.wide = wide_rows(k, M > 1 ? k_stride : 0) && wide_rows(v, M > 1 ? v_stride : 0);
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
    if (n > KVQ_MAXROWS)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: %zu rows, at most %u a call", n, KVQ_MAXROWS);
    if (n > 1 && ((k && k_stride < n_head_kv * head_dim) || (v && v_stride < n_head_kv * head_dim)))
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: a stride below the row's width");
    if ((uintptr_t)cache % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_read: the cache must be 16-byte aligned");
    const unsigned tiles = (unsigned)((p0 + n - 1) / KVQ_TILE - p0 / KVQ_TILE + 1);
    bool wide = wide_rows(k, n > 1 ? k_stride : 0) && wide_rows(v, n > 1 ? v_stride : 0);
    int hd = (int)head_dim;
#define FOX_READ4(hd) ((const void *)kv_read_k<4, hd>)
#define FOX_READ8(hd) ((const void *)kv_read_k<8, hd>)
    const void *f = kv_type == FOX_GPU_KV_Q4 ? FOX_BY_WIDTH(wide, hd, FOX_READ4)
                                             : FOX_BY_WIDTH(wide, hd, FOX_READ8);
#undef FOX_READ4
#undef FOX_READ8
    void *args[] = {(void *)&cache, &n_ctx, &hd, &p0, &n, &k, &k_stride, &v, &v_stride, &wide};
    FOX_HIP(hipSetDevice(ctx->device));
    FOX_HIP(hipLaunchKernel(f, dim3(tiles, (unsigned)n_head_kv), dim3(KS_THREADS), args, 0,
                            ctx->stream));
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
    if (n_head > 65535 || n_head + 2 * n_head_kv > 65535)    // (rows of the grid; the sum may wrap)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: %zu heads beside %zu kv heads are too many", what, n_head,
                        n_head_kv);
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
    A->wide = wide_rows(q, M > 1 ? q_stride : 0) && wide_rows(q_out, M > 1 ? qo_stride : 0) &&
              wide_rows(k, M > 1 ? k_stride : 0) && wide_rows(v, M > 1 ? v_stride : 0) &&
              wide_rows(q_norm, 0) && wide_rows(k_norm, 0) && wide_rows(cos_t, 0) &&
              wide_rows(sin_t, 0);
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
    A.wide = A.wide && wide_rows(k_cache, 0) && wide_rows(v_cache, 0);
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
