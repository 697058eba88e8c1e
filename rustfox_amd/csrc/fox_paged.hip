// fox_paged.hip -- paged caches of many sequences: tables of the rotation,
// a pass's queries, keys and values normed, rotated and stored into pages, and
// eviction of the rows that got the least attention.
#include "fox_paged_dev.h"

#include <cmath>
#include <cstring>

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));

#define PG_THREADS 256

// ------------------------------------------------------------------ shapes

fox_gpu_status fox_paged_check(const char *what, const fox_gpu_paged *c, bool track, PagedDev *out)
{
    if (!c) return fox_fail(FOX_GPU_ERR_ARG, "%s: no cache", what);
    if (!c->k || !c->v || !c->table || c->n_pages == 0 || c->page_size == 0 || c->n_head_kv == 0 ||
        c->head_dim == 0 || c->n_seqs == 0 || c->max_pages == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: the cache has a null pointer or a zero size", what);
    if (c->type != FOX_GPU_F16 && c->type != FOX_GPU_BF16)
        return fox_fail(FOX_GPU_ERR_UNSUPPORTED, "%s: a paged cache is F16 or BF16, not type %d", what, c->type);
    if (c->head_dim % 8 || c->head_dim > 256)
        return fox_fail(FOX_GPU_ERR_UNSUPPORTED, "%s: head_dim is a multiple of 8 up to 256, not %zu", what,
                        c->head_dim);
    if (c->page_size & (c->page_size - 1) || c->page_size < 16 || c->page_size > 4096)
        return fox_fail(FOX_GPU_ERR_UNSUPPORTED, "%s: page_size is a power of two from 16 to 4096, not %zu", what,
                        c->page_size);
    if (c->n_pages > (1u << 31) || c->n_seqs > 65535 || c->n_head_kv > 4096 ||
        c->n_seqs * c->n_head_kv > (1u << 20) || c->max_pages > (1u << 30) / c->page_size)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: %zu pages, %zu sequences of %zu pages, %zu kv heads are too many",
                        what, c->n_pages, c->n_seqs, c->max_pages, c->n_head_kv);
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: the pools must be 16-byte aligned", what);
    if ((c->weight == nullptr) != (c->position == nullptr))
        return fox_fail(FOX_GPU_ERR_ARG, "%s: the cache has one of weight and position", what);
    if ((uintptr_t)c->weight % 16 || (uintptr_t)c->position % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: weight and position must be 16-byte aligned", what);
    if (track && !c->weight)
        return fox_fail(FOX_GPU_ERR_ARG, "%s: the cache has no weight and position", what);
    *out = {};
    out->k = c->k;
    out->v = c->v;
    out->table = c->table;
    out->weight = c->weight;
    out->position = c->position;
    out->n_pages = (uint32_t)c->n_pages;
    out->n_seqs = (uint32_t)c->n_seqs;
    out->max_pages = (uint32_t)c->max_pages;
    out->n_kv = (uint32_t)c->n_head_kv;
    out->hd = (uint32_t)c->head_dim;
    while (((size_t)1 << out->shift) < c->page_size) out->shift++;
    out->cap = (uint32_t)(c->max_pages * c->page_size);
    return FOX_GPU_OK;
}

bool fox_rows_overlap(const float *a, size_t a_stride, size_t a_width, const float *b, size_t b_stride, size_t b_width, size_t M)
{
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    const size_t as = (M > 1 ? a_stride : a_width) * sizeof(float), bs = (M > 1 ? b_stride : b_width) * sizeof(float);
    const size_t aw = a_width * sizeof(float), bw = b_width * sizeof(float);
    if (a0 >= b0 + (M - 1) * bs + bw || b0 >= a0 + (M - 1) * as + aw) return false;
    // (rows may lie between each other's: a row of a meets the last of b's that begins before it ends, or none)
    for (size_t i = 0; i < M; i++) {
        const uintptr_t lo = a0 + i * as, hi = lo + aw;
        if (hi <= b0) continue;
        const size_t j = (hi - 1 - b0) / bs < M - 1 ? (hi - 1 - b0) / bs : M - 1;
        if (b0 + j * bs + bw > lo) return true;
    }
    return false;
}

// ------------------------------------------------------------------ tables

#define RT_ROWS 4                // rows of a thread

struct FreqArgs {
    double turn[128];             // turns a position, pair by pair
    double magnitude;
    const float *factors;
    float *cos_t, *sin_t;
    uint32_t half, p0, n;
    bool wide;                    // rows take 16-byte stores
};

// (2 pi)^k / k!
struct Terms {
    double t[14];
    constexpr __host__ __device__ Terms() : t()
    {
        t[0] = 1.0;
        for (int k = 1; k < 14; k++) t[k] = t[k - 1] * 6.283185307179586476925 / k;
    }
};

// Angles are counted in turns: what is left of p turn[j] after the nearest quarter is exact,
// and within an eighth of a turn seven terms each of sine and cosine are good to 2^-41.
// (Angles in floats would be off by 2^-24 of all the turns made.)
//
// A thread has four pairs and RT_ROWS rows of them, so speeds are read once; the two tables are
// all that moves, and their writes bound it: 131072 positions of 64 pairs (67 MB) 15.1 us, 4.4 TB/s
// (with the library's sine and cosine in double, a value a thread, 43).
__global__ __launch_bounds__(PG_THREADS) void rope_tables_k(FreqArgs A)
{
    const uint32_t quads = (A.half + 3) / 4, rows = PG_THREADS / quads;      // (quads <= 32)
    const uint32_t side = threadIdx.x / quads, j0 = threadIdx.x % quads * 4;
    if (side >= rows) return;
    constexpr Terms T;
    double turn[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t j = min(j0 + i, A.half - 1);
        turn[i] = A.turn[j];
        if (A.factors) turn[i] = turn[i] / (double)A.factors[j];
    }
#pragma unroll
    for (int k = 0; k < RT_ROWS; k++) {
        const uint64_t row = ((uint64_t)blockIdx.x * RT_ROWS + k) * rows + side;
        if (row >= A.n) return;
        float cs[4], sn[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double a = (double)(A.p0 + row) * turn[i], n = rint(4.0 * a);
            const double x = __builtin_fma(-0.25, n, a), y = x * x;
            double s = T.t[13], c = T.t[12];
            // (signs alternate: by -y)
#pragma unroll
            for (int m = 11; m > 0; m -= 2) s = __builtin_fma(s, -y, T.t[m]);
#pragma unroll
            for (int m = 10; m >= 0; m -= 2) c = __builtin_fma(c, -y, T.t[m]);
            s *= x;
            const uint32_t quarter = (uint32_t)(int64_t)n;
            const float u = (float)(A.magnitude * (quarter & 1 ? s : c)), v = (float)(A.magnitude * (quarter & 1 ? c : s));
            cs[i] = (quarter + 1) & 2 ? -u : u;
            sn[i] = quarter & 2 ? -v : v;
        }
        const uint64_t at = row * A.half + j0;
        if (A.wide) {
            *(f4v *)(A.cos_t + at) = *(const f4v *)cs;
            *(f4v *)(A.sin_t + at) = *(const f4v *)sn;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (j0 + i < A.half) {
                    A.cos_t[at + i] = cs[i];
                    A.sin_t[at + i] = sn[i];
                }
        }
    }
}

extern "C" fox_gpu_status fox_gpu_rope_tables(fox_gpu_ctx *ctx, float *cos_t, float *sin_t, size_t p0, size_t n,
                                              size_t n_rot, const fox_gpu_rope_freq *f)
{
    if (!ctx || !cos_t || !sin_t || !f || n == 0 || n_rot == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "rope_tables: bad argument");
    if (n_rot % 2 || n_rot > 256)
        return fox_fail(FOX_GPU_ERR_UNSUPPORTED, "rope_tables: n_rot is even and at most 256, not %zu", n_rot);
    if (p0 > (1u << 30) || n > (1u << 30) - p0)
        return fox_fail(FOX_GPU_ERR_ARG, "rope_tables: %zu positions from %zu on are too many", n, p0);
    // (a NaN fails every comparison)
    if (!(f->base > 0.0 && std::isfinite(f->base) && std::isfinite(f->scale) && std::isfinite(f->ext) &&
          std::isfinite(f->magnitude)))
        return fox_fail(FOX_GPU_ERR_ARG, "rope_tables: base must be above 0 and every figure finite");
    double lo = 0.0, hi = 0.0;
    if (f->ext != 0.0) {
        if (!(f->base > 1.0 && f->beta_fast > 0.0 && f->beta_slow > 0.0 && f->orig_ctx > 0.0 &&
              std::isfinite(f->beta_fast) && std::isfinite(f->beta_slow) && std::isfinite(f->orig_ctx)))
            return fox_fail(FOX_GPU_ERR_ARG, "rope_tables: with ext, base must be above 1, beta_fast, beta_slow "
                            "and orig_ctx above 0");
        const double by = (double)n_rot / (2.0 * std::log(f->base));
        lo = std::fmax(0.0, std::floor(by * std::log(f->orig_ctx / (2.0 * M_PI * f->beta_fast))));
        hi = std::fmin((double)n_rot - 1.0, std::ceil(by * std::log(f->orig_ctx / (2.0 * M_PI * f->beta_slow))));
    }
    FreqArgs A = {};
    A.half = (uint32_t)(n_rot / 2);
    for (uint32_t j = 0; j < A.half; j++) {
        double mix = 0.0;
        if (f->ext != 0.0) {
            const double ramp = ((double)j - lo) / std::fmax(hi - lo, 0.001);
            mix = f->ext * (1.0 - std::fmin(std::fmax(ramp, 0.0), 1.0));
        }
        A.turn[j] = std::pow(f->base, -2.0 * j / (double)n_rot) * (f->scale * (1.0 - mix) + mix) / (2.0 * M_PI);
    }
    A.magnitude = f->magnitude;
    A.factors = f->factors;
    A.cos_t = cos_t;
    A.sin_t = sin_t;
    A.p0 = (uint32_t)p0;
    A.n = (uint32_t)n;
    A.wide = A.half % 4 == 0 && (uintptr_t)cos_t % 16 == 0 && (uintptr_t)sin_t % 16 == 0;
    const size_t rows = PG_THREADS / ((A.half + 3) / 4) * RT_ROWS;
    if ((n + rows - 1) / rows > 0xFFFFFFFFu / PG_THREADS)
        return fox_fail(FOX_GPU_ERR_ARG, "rope_tables: %zu positions of %zu pairs are too many", n, n_rot / 2);
    FOX_HIP(hipSetDevice(ctx->device));
    rope_tables_k<<<dim3((unsigned)((n + rows - 1) / rows)), dim3(PG_THREADS), 0, ctx->stream>>>(A);
    FOX_LAUNCHED("rope_tables");
    return FOX_GPU_OK;
}

// ----------------------------------------------------------------- storing

struct PagedStoreArgs {
    PagedDev C;
    const float *q, *k, *v, *q_norm, *k_norm, *cos_t, *sin_t;
    float *q_out;
    size_t q_stride, qo_stride, k_stride, v_stride;
    const uint32_t *pos, *seq, *row;
    uint32_t n_head, n_rot, n_table;
    double by_hd;                 // 1 / head_dim
    float eps;
    int halves;
};

// the sum of x over LANES neighbouring lanes, in every one of them
template <int LANES>
__device__ __forceinline__ double sum_of(double x)
{
#define FOX_DPP(ctrl)                                                                                          \
    {                                                                                                          \
        const uint64_t u = __builtin_bit_cast(uint64_t, x);                                                    \
        const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, ctrl, 0xF, 0xF, true);        \
        const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), ctrl, 0xF, 0xF, true); \
        x += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                                              \
    }
    FOX_DPP(0xB1)                // lane ^ 1, ^ 2, then the other half of 8 and of 16
    FOX_DPP(0x4E)
    FOX_DPP(0x141)
    if (LANES > 8) FOX_DPP(0x140)
    if (LANES > 16) x += __shfl_xor(x, 16);
#undef FOX_DPP
    return x;
}

__device__ __forceinline__ void load_eight(float x[8], const float *p, bool wide)
{
    if (wide) {
        *(f4v *)x = *(const f4v *)p;
        *(f4v *)(x + 4) = *(const f4v *)(p + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
    }
}

// LANES lanes, of eight dimensions each, have one head's row of one token: keys' heads first, then
// values', then queries'; a workgroup has rows of one token, so what tells where it goes is read once.
// Norm and rotation are in double (a 16-bit key may hang on the last bit; the vector unit multiplies
// doubles at the rate of floats).  A pair's other half is another lane's: it is read
// again, from the first cache, not passed on.  All of a row is read before any of it
// is written, so a query may be turned in place.
//
// FAST: rows, tables and weights take 16-byte accesses, and eight dimensions have eight (four) pairs' angles
// that stand side by side.  Without, values come one by one: the prompt below takes 49 us with rows that are
// not aligned, 36 with 120 dimensions turned.
//
// Bound by its reads and writes where there are many tokens: 1001 tokens of 32 + 16 + 16 heads of 128 (58 MB)
// 14.5 us, 4.0 TB/s; 12.5 without norms. (A wave a row, a value a lane: 33.5.)
template <bool BF, int LANES, bool FAST>
__global__ __launch_bounds__(PG_THREADS) void paged_store_k(PagedStoreArgs A)
{
    const uint32_t t = blockIdx.y, hd = A.C.hd, half = A.n_rot / 2;
    const uint32_t at = blockIdx.x * (PG_THREADS / LANES) + threadIdx.x / LANES, d0 = threadIdx.x % LANES * 8;
    const uint32_t s = A.seq ? A.seq[t] : t, p = A.pos[t], r = A.row ? A.row[t] : p;
    if (s >= A.C.n_seqs || p >= A.n_table) return;       // (uniform)
    if (at >= A.n_head + 2 * A.C.n_kv) return;           // (of a whole row)
    const uint32_t part = at < A.C.n_kv ? 0 : at < 2 * A.C.n_kv ? 1 : 2, h = at - part * A.C.n_kv;
    const bool on = d0 < hd;
    const float *row = part == 0 ? A.k + t * A.k_stride : part == 1 ? A.v + t * A.v_stride : A.q + t * A.q_stride;
    const float *w = part == 0 ? A.k_norm : part == 1 ? nullptr : A.q_norm;
    row += (size_t)h * hd;
    float x[8] = {};
    if (on) load_eight(x, row + d0, FAST);
    if (part != 1) {
        const bool turned = on && d0 < A.n_rot;
        const float *cos_t = A.cos_t + (size_t)p * half, *sin_t = A.sin_t + (size_t)p * half;
        // the other halves' values and weights, and the angles, dimension by dimension
        float other[8] = {}, ws[8], wo[8], cs[8] = {}, sn[8] = {};
        if (turned && FAST) {
            if (A.halves) {
                const uint32_t o = d0 < half ? d0 + half : d0 - half, j = d0 < half ? d0 : o;
                load_eight(other, row + o, true);
                if (w) load_eight(wo, w + o, true);
                load_eight(cs, cos_t + j, true);
                load_eight(sn, sin_t + j, true);
            } else {
                const f4v c = *(const f4v *)(cos_t + d0 / 2), z = *(const f4v *)(sin_t + d0 / 2);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    cs[i] = c[i / 2];
                    sn[i] = z[i / 2];
                }
            }
        }
        if (turned && !FAST)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t d = d0 + i;
                if (d < A.n_rot) {
                    const uint32_t o = !A.halves ? d ^ 1 : d < half ? d + half : d - half;
                    const uint32_t j = !A.halves ? d / 2 : d < half ? d : o;
                    other[i] = row[o];
                    if (w) wo[i] = w[o];
                    cs[i] = cos_t[j];
                    sn[i] = sin_t[j];
                }
            }
        double y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = (double)x[i];
        double z[8];
#pragma unroll
        for (int i = 0; i < 8; i++) z[i] = (double)other[i];
        if (w) {
            if (on) load_eight(ws, w + d0, FAST);
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; i++) ss += y[i] * y[i];
            const double inv = rsqrt(sum_of<LANES>(ss) * A.by_hd + (double)A.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                y[i] = y[i] * inv * (double)ws[i];
                z[i] = z[i] * inv * (double)wo[i];
            }
        }
        if (turned) {
            double out[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t d = d0 + i;
                const bool second = A.halves ? d >= half : i & 1;
                const double b = FAST && !A.halves ? y[i ^ 1] : z[i];
                const double turn = y[i] * (double)cs[i] + b * (double)(second ? sn[i] : -sn[i]);
                out[i] = FAST || d < A.n_rot ? turn : y[i];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = out[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)y[i];
        if (part == 2) {
            float *to = A.q_out + t * A.qo_stride + (size_t)h * hd + d0;
            if (!on) return;
            if (FAST) {
                *(f4v *)to = *(const f4v *)x;
                *(f4v *)(to + 4) = *(const f4v *)(x + 4);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) to[i] = x[i];
            }
            return;
        }
    }
    if (r >= A.C.cap) return;
    const size_t to = paged_row(A.C, s, h, r);
    if (to == ~(size_t)0) return;
    if (on) {
        u4v o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = paged_round<BF>(x[2 * i]) | (uint32_t)paged_round<BF>(x[2 * i + 1]) << 16;
        *(u4v *)((uint16_t *)(part ? A.C.v : A.C.k) + to + d0) = o;
    }
    if (part == 0 && d0 == 0 && A.C.weight) {
        const size_t i = ((size_t)s * A.C.n_kv + h) * A.C.cap + r;
        A.C.weight[i] = 0.0f;
        A.C.position[i] = p;
    }
}

extern "C" fox_gpu_status fox_gpu_paged_rope_store(
    fox_gpu_ctx *ctx, const fox_gpu_paged *cache, const float *q, size_t q_stride, float *q_out,
    size_t q_out_stride, size_t n_head, const float *k, size_t k_stride, const float *v,
    size_t v_stride, size_t M, const float *q_norm, const float *k_norm, float eps, int pairs,
    size_t n_rot, const float *cos_t, const float *sin_t, size_t n_table, const uint32_t *pos,
    const uint32_t *seq, const uint32_t *row)
{
    if (!ctx || !q || !q_out || !k || !v || !cos_t || !sin_t || !pos || n_head == 0 || M == 0 || n_table == 0)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: bad argument");
    PagedStoreArgs A = {};
    fox_gpu_status st = fox_paged_check("paged_rope_store", cache, false, &A.C);
    if (st) return st;
    const size_t nq = n_head * cache->head_dim, nkv = cache->n_head_kv * cache->head_dim;
    if (pairs != FOX_GPU_PAIRS_ADJACENT && pairs != FOX_GPU_PAIRS_HALVES)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: unknown pairing %d", pairs);
    if (n_rot == 0 || n_rot % 2 || n_rot > cache->head_dim)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: n_rot is even and at most head_dim, not %zu", n_rot);
    if (M > FOX_GPU_BATCH_TOKENS) return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: too many tokens");
    if (n_head > 65535) return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: %zu heads are too many", n_head);
    if (n_table > (1u << 30))
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: tables of %zu positions are too long", n_table);
    if (M > 1 && (q_stride < nq || q_out_stride < nq || k_stride < nkv || v_stride < nkv))
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: a stride below the row's width");
    if (!seq && M > cache->n_seqs)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: %zu tokens for %zu sequences", M, cache->n_seqs);
    if ((q_out != q || (M > 1 && q_out_stride != q_stride)) && fox_rows_overlap(q_out, q_out_stride, nq, q, q_stride, nq, M))
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: q_out overlaps q and is not q with its stride");
    if (fox_rows_overlap(q_out, q_out_stride, nq, k, k_stride, nkv, M) ||
        fox_rows_overlap(q_out, q_out_stride, nq, v, v_stride, nkv, M))
        return fox_fail(FOX_GPU_ERR_ARG, "paged_rope_store: q_out overlaps k or v");
    A.q = q;
    A.k = k;
    A.v = v;
    A.q_norm = q_norm;
    A.k_norm = k_norm;
    A.cos_t = cos_t;
    A.sin_t = sin_t;
    A.q_out = q_out;
    A.q_stride = q_stride;
    A.qo_stride = q_out_stride;
    A.k_stride = k_stride;
    A.v_stride = v_stride;
    A.pos = pos;
    A.seq = seq;
    A.row = row;
    A.n_head = (uint32_t)n_head;
    A.n_rot = (uint32_t)n_rot;
    A.n_table = (uint32_t)n_table;
    A.by_hd = 1.0 / (double)cache->head_dim;
    A.eps = eps;
    A.halves = pairs == FOX_GPU_PAIRS_HALVES;
    FOX_HIP(hipSetDevice(ctx->device));
    // (eight dimensions of a lane are all turned or none, and their pairs' angles aligned)
    auto wide = [](const float *x, size_t stride) { return (uintptr_t)x % 16 == 0 && stride % 4 == 0; };
    const bool fast = n_rot % (A.halves ? 16 : 8) == 0 && wide(q, M > 1 ? q_stride : 0) &&
                      wide(q_out, M > 1 ? q_out_stride : 0) && wide(k, M > 1 ? k_stride : 0) &&
                      wide(v, M > 1 ? v_stride : 0) && wide(q_norm, 0) && wide(k_norm, 0) && wide(cos_t, 0) && wide(sin_t, 0);
    const size_t lanes = cache->head_dim <= 64 ? 8 : cache->head_dim <= 128 ? 16 : 32, rows = PG_THREADS / lanes;
#define FOX_STORE(bf, f)                                                                                  \
    (lanes == 8 ? (const void *)paged_store_k<bf, 8, f> : lanes == 16 ? (const void *)paged_store_k<bf, 16, f> \
                                                        : (const void *)paged_store_k<bf, 32, f>)
    const void *kern = cache->type == FOX_GPU_BF16 ? fast ? FOX_STORE(true, true) : FOX_STORE(true, false)
                                                   : fast ? FOX_STORE(false, true) : FOX_STORE(false, false);
#undef FOX_STORE
    void *args[] = {&A};
    FOX_HIP(hipLaunchKernel(kern, dim3((unsigned)((n_head + 2 * cache->n_head_kv + rows - 1) / rows), (unsigned)M),
                            dim3(PG_THREADS), args, 0, ctx->stream));
    return FOX_GPU_OK;
}

// ---------------------------------------------------------------- eviction

#define EV_COPIES 2              // of a histogram: lanes that meet in one place wait for each other
// So many rows are moved by the workgroup that finds them (100 of 128 dimensions: 13 to 15 us in one
// launch, 13.0 in two; one, where 100 could: 7.8 and 9.3; 240: 19.5 and 13.3).
#define EV_FEW 128
#define EV_ONES 8                // so many rows to give up are found one by one
#define EV_DEEP 2                // rows that a thread of the mover has on the way (4: 22 us instead of 17.5, for registers)

struct EvictArgs {
    PagedDev C;
    const uint32_t *length;
    uint32_t *kept, *list;        // places, then rows to move, of every kv head: 2 room each
    uint32_t *count;              // rows to move of every kv head
    uint32_t keep, recent, room;
    uint32_t movers;              // workgroups that move a kv head's rows
};

// a row's rank: the newest before all, then by weight (0 and above)
__device__ __forceinline__ uint32_t evict_key(float w, uint32_t p, uint32_t newest, uint32_t recent)
{
    if (newest - p < recent) return 0xFFFFFFFFu;
    return w > 0.0f ? __float_as_uint(w) : 0u;
}

// how many lanes below this one are in the mask
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask)
{
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// one 16-byte piece of a moved row, keys' pieces before values'; the first takes weight and position along
__device__ __forceinline__ void move_piece(const EvictArgs &A, size_t head, uint32_t s, uint32_t h, const uint32_t *to,
                                           const uint32_t *from, uint32_t piece, uint32_t pieces, bool on)
{
    u4v x[EV_DEEP];
    size_t at[EV_DEEP];
    float w[EV_DEEP];
    uint32_t p[EV_DEEP];
    uint16_t *pool = (uint16_t *)(piece < pieces ? A.C.k : A.C.v) + piece % pieces * 8;
    const size_t base = head * A.C.cap;
#pragma unroll
    for (int i = 0; i < EV_DEEP; i++) {
        at[i] = ~(size_t)0;
        x[i] = u4v{0, 0, 0, 0};
        w[i] = 0.0f;
        p[i] = 0;
        if (on && to[i] != ~0u) {
            const size_t src = paged_row(A.C, s, h, from[i]);
            if (src != ~(size_t)0) at[i] = paged_row(A.C, s, h, to[i]);
            if (at[i] != ~(size_t)0) x[i] = *(const u4v *)(pool + src);
            if (piece == 0) {
                w[i] = A.C.weight[base + from[i]];
                p[i] = A.C.position[base + from[i]];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < EV_DEEP; i++) {
        if (at[i] != ~(size_t)0) *(u4v *)(pool + at[i]) = x[i];
        if (on && to[i] != ~0u && piece == 0) {
            A.C.weight[base + to[i]] = w[i];
            A.C.position[base + to[i]] = p[i];
        }
    }
}

// The bin of BINS that holds the want-th key from the top, its keys, and want less those
// above it.  A wave sums its share of the bins, from the highest wave 0's; then
// each finds the share, and in that the bin, for itself.  By the workgroup.
template <int BINS, int WAVES>
__device__ __forceinline__ uint32_t find_bin(const uint32_t (*hist)[BINS], uint32_t *shares, uint32_t &want, uint32_t &in)
{
    constexpr int SHARE = BINS / WAVES, EACH = SHARE / 64;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto bins = [&](uint32_t share, uint32_t x[EACH]) -> uint32_t {      // a lane's bins, the highest first
        uint32_t sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            x[i] = 0;
#pragma unroll
            for (int k = 0; k < EV_COPIES; k++) x[i] += hist[k][BINS - 1 - share * SHARE - lane * EACH - i];
            sum += x[i];
        }
        return sum;
    };
    uint32_t x[EACH];
    __syncthreads();
    uint32_t above = wave_scan(bins(wave, x));
    if (lane == 63) shares[wave] = above;
    __syncthreads();
    uint32_t sum = lane < WAVES ? shares[lane] : 0;
    above = wave_scan(sum);
    const uint32_t share = (uint32_t)__ffsll(__ballot(above >= want)) - 1;
    want -= (uint32_t)__builtin_amdgcn_readlane((int)(above - sum), (int)share);
    sum = bins(share, x);
    above = wave_scan(sum);
    const int owner = __ffsll(__ballot(above >= want)) - 1;
    // (the first of the lane's bins that reaches it)
    uint32_t before = above - sum, bin = EACH - 1;
#pragma unroll
    for (int i = 0; i < EACH - 1; i++)
        if (bin == EACH - 1) {
            if (before + x[i] >= want) bin = i;
            else before += x[i];
        }
    in = x[EACH - 1];
#pragma unroll
    for (int i = 0; i < EACH - 1; i++)
        if (bin == i) in = x[i];
    want -= (uint32_t)__builtin_amdgcn_readlane((int)before, owner);
    in = (uint32_t)__builtin_amdgcn_readlane((int)in, owner);
    return BINS - 1 - share * SHARE - owner * EACH - (uint32_t)__builtin_amdgcn_readlane((int)bin, owner);
}

// Exclusive sums pre[0 .. N) of cnt, and the total, by every wave for itself: each writes the
// same values and reads its own, so the workgroup need not wait.
template <uint32_t N>
__device__ __forceinline__ uint32_t scan_counts(const uint32_t *cnt, uint32_t *pre)
{
    constexpr uint32_t EACH = N / 64;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t v[EACH], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < EACH; i++) sum += v[i] = cnt[lane * EACH + i];
    uint32_t x = wave_scan(sum);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
    x -= sum;
#pragma unroll
    for (uint32_t i = 0; i < EACH; i++) {
        pre[lane * EACH + i] = x;
        x += v[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    return total;
}

// One workgroup per (kv head, sequence) finds the least key that is kept, by its 12
// highest bits (exponent and 3 bits more: most keys are told apart), then 10 and 10: a
// histogram of the keys that share the bits found so far says which next ones
// the keep-th key has, and a bin that is wholly kept ends the search.
// Rows above it and the first of those equal to it are kept; the places and the rows that fill
// them are listed in order: each wave's 64 rows are counted by a ballot, the counts
// summed once.  Keys stay in registers, HELD a thread; of longer sequences
// each turn reads weights and positions anew.  Few rows are moved here; FEW: there are never more.
//
// It waits, for loads, LDS and other waves, more than it works: 48 kv heads of up to 20011 rows 19 us
// (of it 3.5 us the rows' way to one compute unit, 4 the histograms, 6 the lists), one row too many of
// 2049 in 128 kv heads 6.3 us.
template <bool FEW, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void evict_select_k(EvictArgs A)
{
    constexpr int WAVES = THREADS / 64, ROWS = THREADS * HELD;
    static_assert(WAVES * HELD % 64 == 0, "scan_counts");
    __shared__ uint32_t high[EV_COPIES][4096], low[2][EV_COPIES][1024], shares[3][WAVES], cnt[2][HELD * WAVES], pre[2][HELD * WAVES], red[WAVES];
    __shared__ uint32_t few[2 * EV_FEW], ones[2][2][WAVES];
    __shared__ uint64_t words[HELD * WAVES];
    const uint32_t h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t head = (size_t)s * A.C.n_kv + h;
    const uint32_t n = min(A.length[s], A.C.cap);
    if (h == 0 && tid == 0) A.kept[s] = min(n, A.keep);
    if (n <= A.keep) {
        if (!FEW && tid == 0) A.count[head] = 0;
        return;
    }
    const float *weight = A.C.weight + head * A.C.cap;
    const uint32_t *position = A.C.position + head * A.C.cap;
    const bool held = n <= ROWS;
    uint32_t key[HELD], pos[HELD], newest = 0;

    // the greatest position; of a short sequence the keys, too
    for (uint32_t base = 0; base < n; base += ROWS) {
#pragma unroll
        for (int c = 0; c < HELD; c++) {
            const uint32_t b = base + c * THREADS, i = min(b + tid, n - 1);
            if (b < n) {                                     // (uniform)
                pos[c] = position[i];
                if (held) key[c] = __float_as_uint(weight[i]);
            }
        }
        if (base == 0) {
            for (uint32_t i = tid; i < EV_COPIES * 4096; i += THREADS) (&high[0][0])[i] = 0;
            for (uint32_t i = tid; i < EV_COPIES * 2048; i += THREADS) (&low[0][0][0])[i] = 0;
        }
#pragma unroll
        for (int c = 0; c < HELD; c++)
            if (base + c * THREADS < n) newest = max(newest, pos[c]);
    }
    newest = wave_max(newest);
    if (lane == 0) red[wave] = newest;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) newest = max(newest, red[i]);
    if (held) {
#pragma unroll
        for (int c = 0; c < HELD; c++)
            if (c * THREADS < n) key[c] = evict_key(__uint_as_float(key[c]), pos[c], newest, A.recent);
    }
    auto read = [&](uint32_t base) {                         // keys of rows base .., where they are not held
        if (held) return;
#pragma unroll
        for (int c = 0; c < HELD; c++) {
            const uint32_t b = base + c * THREADS, i = min(b + tid, n - 1);
            if (b < n) key[c] = evict_key(weight[i], position[i], newest, A.recent);
        }
    };

    const uint32_t pieces = A.C.hd / 8, side = THREADS / (2 * pieces);
    auto move_few = [&](uint32_t rows) {                     // the places and rows of few[]
        for (uint32_t m = tid / (2 * pieces); m < rows; m += side * EV_DEEP) {
            uint32_t t[EV_DEEP], f[EV_DEEP];
#pragma unroll
            for (int i = 0; i < EV_DEEP; i++) {
                const bool in = m + i * side < rows;
                t[i] = in ? few[m + i * side] : ~0u;
                f[i] = in ? few[EV_FEW + m + i * side] : 0u;
            }
            move_piece(A, head, s, h, t, f, tid % (2 * pieces), pieces, tid < side * 2 * pieces);
        }
    };

    // A step's one row too many (a few): the least key, of equal ones the highest row, is found and
    // taken out, as often as rows have to go.  evict-step-8b 12.0 us by histograms, 8 so.
    if (held && n - A.keep <= EV_ONES) {
        const uint32_t go = n - A.keep;
        uint32_t out = 0, gone[EV_ONES];                     // a bit a row
#pragma unroll
        for (int e = 0; e < EV_ONES; e++) {
            gone[e] = ~0u;
            if (e >= go) continue;                           // (uniform)
            uint32_t k = 0xFFFFFFFFu, r = 0;
            bool any = false;
#pragma unroll
            for (int c = 0; c < HELD; c++)
                if (c * THREADS < n && c * THREADS + tid < n && !(out >> c & 1) && key[c] <= k) {
                    k = key[c];                              // (rows rise with c)
                    r = c * THREADS + tid;
                    any = true;
                }
            const uint32_t least = ~wave_max(~k);
            const uint32_t most = wave_max(any && k == least ? r + 1 : 0);   // 0: no row is left
            if (lane == 0) {
                ones[e & 1][0][wave] = least;
                ones[e & 1][1][wave] = most;
            }
            __syncthreads();
            const uint32_t kw = lane < WAVES && ones[e & 1][1][lane % WAVES] ? ones[e & 1][0][lane % WAVES] : 0xFFFFFFFFu;
            const uint32_t all = ~wave_max(~kw);
            gone[e] = wave_max(lane < WAVES && kw == all ? ones[e & 1][1][lane % WAVES] : 0) - 1;
            if (gone[e] % THREADS == tid) out |= 1u << (gone[e] / THREADS);
        }
        // of the rows from keep on, those that are not gone fill the places below it, both in order
        uint32_t rows = 0;
#pragma unroll
        for (int e = 0; e < EV_ONES; e++) {
            uint32_t rank = 0, moves = 0;
            bool left = A.keep + e < n;
#pragma unroll
            for (int x = 0; x < EV_ONES; x++) {
                rank += gone[x] < gone[e];
                left = left && gone[x] != A.keep + e;
                moves += gone[x] >= A.keep && gone[x] < A.keep + e;
            }
            if (gone[e] < A.keep) {
                rows++;
                if (tid == 0) few[rank] = gone[e];
            }
            if (left && tid == 0) few[EV_FEW + e - moves] = A.keep + e;
        }
        if (!FEW && tid == 0) A.count[head] = 0;
        __syncthreads();
        move_few(rows);
        return;
    }

    uint32_t least = 0, want = A.keep, in;   // the bits found; rows still to take among those that share them
    const uint32_t copy = lane % EV_COPIES;
    uint32_t newer = 0;                      // rows of the greatest key, one place for all: added up first
    for (uint32_t base = 0; base < n; base += ROWS) {
        read(base);
#pragma unroll
        for (int c = 0; c < HELD; c++)
            if (base + c * THREADS < n && base + c * THREADS + tid < n) {
                if (key[c] == 0xFFFFFFFFu) newer++;
                else atomicAdd(&high[copy][key[c] >> 20], 1u);
            }
    }
    newer = wave_scan(newer);
    if (lane == 63) atomicAdd(&high[0][4095], newer);
    least = find_bin<4096, WAVES>(high, shares[0], want, in) << 20;
    bool every = in == want;                 // those are all taken
#pragma unroll
    for (int turn = 0; turn < 2; turn++) {
        if (every) break;
        const int at = turn ? 0 : 10;
        for (uint32_t base = 0; base < n; base += ROWS) {
            read(base);
#pragma unroll
            for (int c = 0; c < HELD; c++)
                if (base + c * THREADS < n && base + c * THREADS + tid < n && (key[c] ^ least) >> (at + 10) == 0)
                    atomicAdd(&low[turn][copy][key[c] >> at & 1023u], 1u);
        }
        least |= find_bin<1024, WAVES>(low[turn], shares[1 + turn], want, in) << at;
        every = in == want;
    }

    uint32_t *to = FEW ? nullptr : A.list + head * 2 * A.room, *from = FEW ? nullptr : to + A.room;
    uint32_t ties = 0, places = 0, moves = 0;
    for (uint32_t base = 0; base < n; base += ROWS) {
        if (base) __syncthreads();
        read(base);
        uint32_t stays = 0;                                  // a bit a row
        if (every) {
#pragma unroll
            for (int c = 0; c < HELD; c++)
                if (base + c * THREADS < n && base + c * THREADS + tid < n && key[c] >= least) stays |= 1u << c;
        } else {
#pragma unroll
            for (int c = 0; c < HELD; c++) {
                const uint64_t tie = __ballot(base + c * THREADS < n && base + c * THREADS + tid < n && key[c] == least);
                if (lane == 0) cnt[0][c * WAVES + wave] = __popcll(tie);
            }
            __syncthreads();
            const uint32_t all = scan_counts<HELD * WAVES>(cnt[0], pre[0]);
#pragma unroll
            for (int c = 0; c < HELD; c++)
                if (base + c * THREADS < n) {
                    const bool in = base + c * THREADS + tid < n, tie = in && key[c] == least;
                    const uint32_t rank = ties + pre[0][c * WAVES + wave] + lanes_below(__ballot(tie));
                    if ((in && key[c] > least) || (tie && rank < want)) stays |= 1u << c;
                }
            ties += all;
        }
        // A wave's rows as masks, kept by lane c, then counted by a thread a mask: places in the low half, rows
        // to move in the high half.
        uint64_t mine = 0;
#pragma unroll
        for (int c = 0; c < HELD; c++) {
            const uint64_t mask = __ballot(stays >> c & 1);
            mine = lane == c ? mask : mine;
        }
        if (lane < HELD) words[lane * WAVES + wave] = mine;
        __syncthreads();
        if (tid < HELD * WAVES) {
            const uint32_t r0 = base + tid * 64;
            const uint64_t low = r0 >= A.keep ? 0 : A.keep - r0 >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << (A.keep - r0)) - 1;
            cnt[1][tid] = __popcll(~words[tid] & low) | __popcll(words[tid] & ~low) << 16;
        }
        __syncthreads();
        const uint32_t all = scan_counts<HELD * WAVES>(cnt[1], pre[1]);
#pragma unroll
        for (int c = 0; c < HELD; c++) {
            const uint32_t r0 = base + c * THREADS + wave * 64;
            if (r0 < n) {
                const bool stay = stays >> c & 1;
                const uint32_t x = pre[1][c * WAVES + wave];
                if (r0 < A.keep) {
                    const bool place = !stay && r0 + lane < A.keep;
                    const uint32_t a = places + (x & 0xFFFFu) + lanes_below(__ballot(place));
                    if (place && a < EV_FEW) few[a] = r0 + lane;
                    if (!FEW && place && a < A.room) to[a] = r0 + lane;
                }
                if (r0 + 64 > A.keep) {
                    const bool mover = stay && r0 + lane >= A.keep;
                    const uint32_t b = moves + (x >> 16) + lanes_below(__ballot(mover));
                    if (mover && b < EV_FEW) few[EV_FEW + b] = r0 + lane;
                    if (!FEW && mover && b < A.room) from[b] = r0 + lane;
                }
            }
        }
        places += all & 0xFFFFu;
        moves += all >> 16;
    }
    const uint32_t rows = min(min(places, moves), A.room);   // (places and moves are equal)
    if (!FEW && tid == 0) A.count[head] = rows > EV_FEW ? rows : 0;
    if (rows > EV_FEW) return;
    __syncthreads();
    move_few(rows);
}

// Rows to their places: no place is another's row, so in any order.  A thread has EV_DEEP
// rows' pieces on the way, since each waits for the list, the table and the row in turn: 71 MB read and
// written in 17.5 us, 4.1 TB/s.
__global__ __launch_bounds__(PG_THREADS) void evict_move_k(EvictArgs A)
{
    const uint32_t head = blockIdx.x / A.movers, part = blockIdx.x % A.movers, h = head % A.C.n_kv, s = head / A.C.n_kv;
    const uint32_t n = min(A.count[head], A.room), pieces = A.C.hd / 8, side = PG_THREADS / (2 * pieces);
    const uint32_t *to = A.list + (size_t)head * 2 * A.room, *from = to + A.room;
    for (uint64_t m = (uint64_t)part * side * EV_DEEP + threadIdx.x / (2 * pieces); m < n;
         m += (uint64_t)A.movers * side * EV_DEEP) {
        uint32_t t[EV_DEEP], f[EV_DEEP];
#pragma unroll
        for (int i = 0; i < EV_DEEP; i++) {
            const bool in = m + i * side < n;
            t[i] = in ? to[m + i * side] : ~0u;
            f[i] = in ? from[m + i * side] : 0u;
        }
        move_piece(A, head, s, h, t, f, threadIdx.x % (2 * pieces), pieces, threadIdx.x < side * 2 * pieces);
    }
}

extern "C" fox_gpu_status fox_gpu_paged_evict(fox_gpu_ctx *ctx, const fox_gpu_paged *cache, const uint32_t *length,
                                              uint32_t *kept, size_t keep, size_t recent)
{
    if (!ctx || !length || !kept || keep == 0) return fox_fail(FOX_GPU_ERR_ARG, "paged_evict: bad argument");
    EvictArgs A = {};
    fox_gpu_status st = fox_paged_check("paged_evict", cache, true, &A.C);
    if (st) return st;
    if (recent > keep)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_evict: the %zu newest rows are more than the %zu kept", recent, keep);
    const uintptr_t la = (uintptr_t)length, ka = (uintptr_t)kept, size = cache->n_seqs * sizeof(uint32_t);
    if (la < ka + size && ka < la + size)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_evict: kept must be another array than length");
    A.length = length;
    A.kept = kept;
    A.keep = (uint32_t)(keep < A.C.cap ? keep : A.C.cap);
    A.recent = (uint32_t)(recent < A.C.cap ? recent : A.C.cap);
    // at most so many rows can move
    A.room = A.C.cap - A.keep < A.keep ? A.C.cap - A.keep : A.keep;
    const size_t heads = cache->n_seqs * cache->n_head_kv;
    // Short sequences by 512 threads of 8 rows, longer ones by 1024 of 8 or 24 (4631 rows, 1915 of them kept:
    // 13.6 us by 8, 18.1 by 24: less code to meet); the few rows that a step can give up are moved in the same launch.
    const bool few = A.room <= EV_FEW;
#define FOX_SELECT(f)                                                                               \
    (A.C.cap <= 4096 ? (const void *)evict_select_k<f, 512, 8> : A.C.cap <= 8192 ? (const void *)evict_select_k<f, 1024, 8> \
                                                               : (const void *)evict_select_k<f, 1024, 24>)
    const void *k = few ? FOX_SELECT(true) : FOX_SELECT(false);
#undef FOX_SELECT
    const dim3 grid((unsigned)cache->n_head_kv, (unsigned)cache->n_seqs), block(A.C.cap <= 4096 ? 512 : 1024);
    void *args[] = {&A};
    FOX_HIP(hipSetDevice(ctx->device));
    if (few) {
        FOX_HIP(hipLaunchKernel(k, grid, block, args, 0, ctx->stream));
        return FOX_GPU_OK;
    }
    if ((st = fox_ws_reserve(ctx, (heads + heads * 2 * A.room) * sizeof(uint32_t)))) return st;
    A.count = (uint32_t *)ctx->ws;
    A.list = A.count + heads;
    // one round of rows a workgroup, unless the heads alone are many
    const size_t round = PG_THREADS / (cache->head_dim / 4) * EV_DEEP, rounds = (A.room + round - 1) / round;
    const size_t most = (size_t)32 * ctx->n_cu / heads + 1;
    A.movers = (uint32_t)(rounds < most ? rounds : most);
    FOX_HIP(hipLaunchKernel(k, grid, block, args, 0, ctx->stream));
    evict_move_k<<<dim3((unsigned)(heads * A.movers)), dim3(PG_THREADS), 0, ctx->stream>>>(A);
    FOX_LAUNCHED("paged_evict");
    return FOX_GPU_OK;
}
