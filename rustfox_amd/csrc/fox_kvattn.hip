// fox_kvattn.hip -- causal attention over a quantised cache on the matrix
// cores.
//
// Arithmetic.  The cache's values are exactly halves (fox_kvq_dev.h), so an
// f16 MFMA multiplies them without rounding; the other operand, the query or the
// softmax's weight, is the sum of two halves (22 bits of it), each its own MFMA into
// the same float sums.  A query head's row is multiplied by log2(e) / sqrt(hd) and a
// power of two first, its largest value to 2^14, so that the lower half is not lost
// below the half's range.  Scores are then a power of two away from exponents: the
// largest one's product with it, the maximum, is exact, and that score's weight, 2^7
// (1 to 2^8 from 2^24 on, where the 7 is rounded to the maximum's last bit), stays a
// half however large the score is.
//
// A step is 32 positions (a tile) of one kv head by 16 or 32 query rows (row =
// token * G + head in the group of G = n_head / n_head_kv that share it):
//   S[pos][row] = sum_d K[pos][d] q[row][d]
//   O[dim][row] += sum_pos V[dim][pos] P[pos][row]
// A lane's scores in S are of the eight positions of a V word (kvq_v_pos), so the
// weights of those positions are the second product's operand as they stand.
// The running maximum only follows scores that pass it by 8 (in powers of two):
// weights are exp2(s - m + 7) <= 2^15, within a half; between updates no lane
// needs another's maximum.  A weight ends at 2^-24, 2^-31 of the largest.
#include "fox_kvq_dev.h"
#include "fox_internal.h"

#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

#define KA_WAVES 4
#define KA_ROOM 8.0f            // how far scores may pass the running maximum
#define KA_LIFT 7.0f            // weights are scaled by 2^7: 2^(8 + 7) is within a half

struct AttnArgs {
    float *out, *part;
    size_t out_stride, q_stride;
    const float *q;
    const uint8_t *cache;
    int n_ctx, n_head_kv, G, splits;
    uint32_t by_g;                // row / G: see token_of
    float score;                  // log2(e) / sqrt(hd)
    int from;                     // positions from which kv_attn_many takes the call, kv_attn_few below
    uint16_t hd, M;
    uint8_t g_shift;
    bool q_wide, out_wide;        // rows take 16-byte accesses
};

// positions that the call's last token sees
__device__ __forceinline__ int seen_of(const AttnArgs &A, size_t p0) { return (int)min(p0 + A.M, (size_t)A.n_ctx); }

// row / G without a division (some thirty instructions, each met cold in a short
// call): by_g = 2^(30 + g_shift) / G rounded up, 2^g_shift >= G, which is exact for row < 2^30
__device__ __forceinline__ int token_of(const AttnArgs &A, int row)
{
    return (int)(__umulhi((uint32_t)row << 2, A.by_g) >> A.g_shift);
}

__device__ __forceinline__ h2v as_h2(uint32_t v) { return __builtin_bit_cast(h2v, v); }
__device__ __forceinline__ uint32_t as_u(h2v v) { return __builtin_bit_cast(uint32_t, v); }

// eight values 4 d (c) as halves from their codes w and the scales' halves d
// (a pair per two values): 4 bits as (64 + n) d - 72 d, one rounding of an
// exact result; 8 bits as ((1024 + n) - 1152) d
template <int BITS>
__device__ __forceinline__ h8v unpack(const uint32_t *w, const h2v d[4], const h2v m72[4])
{
    uint32_t r[4];
    if (BITS == 4) {
        // (in registers, where one instruction takes both: of two literals it takes neither)
        uint32_t mask = 0x00F000F0u, base = 0x54005400u;
        asm("" : "+s"(mask));
        asm("" : "+v"(base));
        const uint32_t x[4] = {w[0] << 4, w[0], w[0] >> 4, w[0] >> 8};
#pragma unroll
        for (int i = 0; i < 4; i++)
            r[i] = as_u(__builtin_elementwise_fma(as_h2((x[i] & mask) | base), d[i], m72[i]));
    } else {
        const h2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
        for (int i = 0; i < 4; i++)
            r[i] = as_u((as_h2(__builtin_amdgcn_perm(0x64646464u, w[i >> 1],
                                                     i & 1 ? 0x07030702u : 0x05010500u)) + off) * d[i]);
    }
    return __builtin_bit_cast(h8v, *(u4v *)r);
}

__device__ __forceinline__ float quad_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quad_sum(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// eight scales' halves as pairs, and -72 of them
__device__ __forceinline__ void v_scales(uint2 b, h2v d[4], h2v m72[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        d[i] = as_h2(__builtin_amdgcn_perm(0, i < 2 ? b.x : b.y, i & 1 ? 0x0C030C02u : 0x0C010C00u) << 7);
        m72[i] = d[i] * (h2v){(_Float16)-72.0f, (_Float16)-72.0f};
    }
}
// (one scale for the eight: byte i of `bytes`)
template <int BITS>
__device__ __forceinline__ h8v unpack_k(const uint32_t *w, uint32_t bytes, int i)
{
    const h2v d1 = as_h2(__builtin_amdgcn_perm(0, bytes, i ? 0x0C010C01u : 0x0C000C00u) << 7);
    const h2v m1 = d1 * (h2v){(_Float16)-72.0f, (_Float16)-72.0f};
    const h2v d[4] = {d1, d1, d1, d1}, mm[4] = {m1, m1, m1, m1};
    return unpack<BITS>(w, d, mm);
}

// A tile that not every row sees whole: V's scale bytes of chunk c of a group.
// Positions from `last` on, that no row sees, count as zero whatever the cache
// holds there; NaN scales are taken out of the product.  Returns the first
// position of those (or INT_MAX), to be put into the sums of the rows that see it.
__device__ __forceinline__ int trim_scales(uint2 &b2, int tp, int c, int last)
{
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 1; i >= 0; i--) {
        const int p = tp + kvq_v_pos(c, 4 * i), n = min(max(last - p, 0), 4);
        uint32_t b = (i ? b2.y : b2.x) & (n == 4 ? ~0u : (1u << 8 * n) - 1);
        const uint32_t nan = ((b & 0x78787878u) + 0x08080808u) & b & 0x80808080u;   // from 0xF8 on
        b &= ~((nan << 1) - (nan >> 7));
        if (nan) at = p + (__builtin_ctz(nan) >> 3);
        (i ? b2.y : b2.x) = b;
    }
    return at;
}

// a - (float)h in one instruction: the -1 is kept from the compiler, which
// would convert and subtract
__device__ __forceinline__ float less(float a, _Float16 h)
{
    float minus = -1.0f;
    asm("" : "+s"(minus));
    return __builtin_fmaf((float)h, minus, a);
}

// score 2^(14 - exponent of a row's largest value times score), the exponent kept
// at -100 or above and at 127, a float's largest, for rows with an infinity or a NaN:
// both powers are normal floats.  back turns a score of the scaled row into powers of
// two (the cache's halves are 4 times its values); it is one itself, see above
__device__ __forceinline__ float query_scale(float top, float score, float &back)
{
    const int ex = min(max((int)(__float_as_uint(top * score) >> 23) - 127, -100), 127);
    back = __uint_as_float((uint32_t)(127 - 16 + ex) << 23);
    return score * __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
}

// eight scaled values as two halves each
__device__ __forceinline__ void split_8(const float x[8], float up, h8v &hi, h8v &lo)
{
    h2v h[4], d[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = x[2 * i] * up, b = x[2 * i + 1] * up;
        // (one value of the upper halves: the compiler forms them from the product and from
        // its float, whose roundings differ now and then, and would subtract the other one)
        uint32_t hw = as_u(h2v{(_Float16)a, (_Float16)b});
        asm("" : "+v"(hw));
        h[i] = as_h2(hw);
        d[i] = h2v{(_Float16)less(a, h[i][0]), (_Float16)less(b, h[i][1])};
    }
    hi = __builtin_bit_cast(h8v, *(u4v *)h);
    lo = __builtin_bit_cast(h8v, *(u4v *)d);
}

// four floats of a query row from dimension d on (zero past hd)
__device__ __forceinline__ float4 query_quad(const float *row, int d, const AttnArgs &A)
{
    if (A.q_wide) return d < A.hd ? *(const float4 *)(row + d) : float4{0, 0, 0, 0};
    return float4{d < A.hd ? row[d] : 0.0f, d + 1 < A.hd ? row[d + 1] : 0.0f,
                  d + 2 < A.hd ? row[d + 2] : 0.0f, d + 3 < A.hd ? row[d + 3] : 0.0f};
}
__device__ __forceinline__ const float *query_row(const AttnArgs &A, int kvh, int row)
{
    const int tok = token_of(A, row);
    return A.q + (size_t)tok * A.q_stride + (uint32_t)((kvh * A.G + row - tok * A.G) * A.hd);
}
__device__ __forceinline__ float *out_row(const AttnArgs &A, int kvh, int row)
{
    const int tok = token_of(A, row);
    return A.out + (size_t)tok * A.out_stride + (uint32_t)((kvh * A.G + row - tok * A.G) * A.hd);
}

// Exponents of a row's N weights from its scores s, x = s sc - m + KA_LIFT.  Where one passes
// the maximum m by more than KA_ROOM, m becomes the largest score (of the row's
// PARTS lanes, 64 / PARTS apart) and the row's sum l and sums o follow.
template <int N, int PARTS, typename V, int ND>
__device__ __forceinline__ void exponents(float x[N], const float s[N], float sc, float &m, float &l,
                                          V (&o)[ND])
{
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; e++) {
        x[e] = __builtin_fmaf(s[e], sc, KA_LIFT - m);
        top = fmaxf(top, x[e]);
    }
    if (__any(top > KA_LIFT + KA_ROOM)) {
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < N; e++) mx = fmaxf(mx, s[e]);
        if (PARTS == 4) mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)) * sc);
        const float f = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] *= f;
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = __builtin_fmaf(s[e], sc, KA_LIFT - m);
    }
}

// The weights of eight positions, as two halves each, and their sum.  Both halves are
// truncated, which leaves up to 2^-21 of a weight out of the products, not of the sum.  Rounded
// to the nearest, whole passes are off by as much (777 tokens at 8000 positions 1.01e-6 / 1.00e-6 of the
// result, 512 at none 3.6e-7 / 3.5e-7: scores' errors count more) and take 1 to 5% longer.
__device__ __forceinline__ void weigh(const float x[8], float &l, h8v &ph, h8v &pl)
{
    h2v hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = __builtin_amdgcn_exp2f(x[2 * i]), b = __builtin_amdgcn_exp2f(x[2 * i + 1]);
        l += a + b;
        hi[i] = __builtin_bit_cast(h2v, __builtin_amdgcn_cvt_pkrtz(a, b));
        lo[i] = __builtin_bit_cast(h2v, __builtin_amdgcn_cvt_pkrtz(less(a, hi[i][0]), less(b, hi[i][1])));
    }
    ph = __builtin_bit_cast(h8v, *(u4v *)hi);
    pl = __builtin_bit_cast(h8v, *(u4v *)lo);
}

// the value of lane r ^ 8 of each 16
__device__ __forceinline__ float other_half(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, true));
}

__device__ __forceinline__ f4v mfma(h8v a, h8v b, f4v c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma(h8v a, h8v b, f16v c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// four results of a row from dimension `dim` on
__device__ __forceinline__ void put_row(const AttnArgs &A, int kvh, int row, int dim, f4v v)
{
    float *dst = out_row(A, kvh, row) + dim;
    if (A.out_wide) {
        if (dim < A.hd) *(f4v *)dst = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (dim + e < A.hd) dst[e] = v[e];
    }
}

// Four sums of one row at dimension `dim` of kv head kvh: the result, or a split's record.
__device__ __forceinline__ void put_sums(const AttnArgs &A, int kvh, int row, int dim, f4v v, float m,
                                         float l, bool whole, int split, int width)
{
    if (whole) {
        put_row(A, kvh, row, dim, v * (0.25f / l));
    } else {
        float *dst = A.part + (((size_t)kvh * A.M * A.G + row) * A.splits + split) * (4 + width);
        if (dim == 0) {
            dst[0] = m;
            dst[1] = l;
        }
        *(f4v *)(dst + 4 + dim) = v;
    }
}

// One tile's bytes as a lane holds them.
template <int BITS, int NG>
struct Tile {
    static constexpr int NS = NG % 4 == 0 ? NG / 4 : NG < 3 ? 1 : NG;   // K scale pairs of a lane
    uint32_t k[2][NG * BITS / 4], v[2 * NG][BITS / 4];
    uint16_t ks[NS];
    uint2 vs[NG];

    __device__ __forceinline__ void load_k(const uint8_t *rec, int lane)
    {
        constexpr int CODES = KVQ_TILE * NG * 32 * BITS / 8;
        const uint32_t r = lane & 15, c = lane >> 4;
#pragma unroll
        for (int i = 0; i < 2; i++)
            __builtin_memcpy(k[i], __builtin_assume_aligned(rec + (16 * (r >> 3) + 8 * i + (r & 7)) * (4 * NG * BITS) + c * NG * BITS, 4 * (NG % 4 == 0 ? 4 : NG % 2 == 0 ? 2 : 1)),
                             sizeof(k[i]));
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const uint32_t g = NS == NG ? (NG * c + s) / 4 : NG % 4 == 0 ? c * (NG / 4) + s : NG * c / 4;
            ks[s] = *(const uint16_t *)(rec + 2 * CODES + g * 32 + r * 2);
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t *rec, int lane)
    {
        constexpr int CODES = KVQ_TILE * NG * 32 * BITS / 8;
        const uint32_t r = lane & 15, c = lane >> 4;
#pragma unroll
        for (int t = 0; t < 2 * NG; t++)
            __builtin_memcpy(v[t], __builtin_assume_aligned(rec + CODES + ((16 * t + r) * 4 + c) * BITS, BITS),
                             sizeof(v[t]));
#pragma unroll
        for (int g = 0; g < NG; g++)
            vs[g] = *(const uint2 *)(rec + 2 * CODES + 32 * NG + g * 32 + c * 8);
    }
    // scale pair of MFMA step j's dimensions
    __device__ __forceinline__ uint32_t kscale(int j) const
    {
        return ks[NS == NG ? j : NG % 4 == 0 ? j / 4 : 0];
    }
};

// Few rows: partial attention of ROWS query rows over the tiles that fall to one
// wave (w0, w0 + step, ...), unpacked in its registers; the four waves of a
// workgroup are merged through LDS, and with several splits per kv head a record
// (m, l, -, -, o) goes to the workspace for the merge kernels.
// ROWS 8: the columns of one product hold the rows' upper halves and their
// lower ones, so a tile takes half the products; the two columns of a row are
// added where a score is used and at the end.
// What bounds it is unpacking, then the read: one row of 32 heads over 8 of 128
// dimensions, 4 bits, at 131,071 positions (143 MB) takes 36 to 37 us a call with its
// merge, 3.9 TB/s, the vector units busy 52% and the matrix cores 9% of the time.
// Reading two tiles ahead is slower (39.4 us for 36.5), as is one copy of the loop's
// body that reads past its last tile (8.4 -> 8.8 us at 1500 positions).
// Short contexts are a launch and 2 to 4 us: 34 positions of 6 heads 3.8 to 4.8 us in all.
// ONE: a single split, whose first tiles are read before the position is known (that row
// at 300 positions 6.7 -> 6.3 us; with more splits most such reads would be for nothing
// where a long cache is not full: 8.1 -> 8.7 us at 1000 of 32768 positions).
template <int BITS, int NG, int ROWS, bool ONE>
__global__ __launch_bounds__(64 * KA_WAVES, NG > 4 ? 1 : 2) void kv_attn_few(const uint32_t *pos, AttnArgs A)
{
    constexpr bool PACK = ROWS == 8;
    constexpr int WIDTH = 32 * NG, T = ROWS == 32 ? 2 : 1, NT = T * 2 * NG, NQ = PACK ? 1 : 2;
    constexpr int ROUND = NT < 8 ? NT : 8;                       // tiles of sums merged at a time
    constexpr int JW = (NG + KA_WAVES - 1) / KA_WAVES;           // product steps a wave prepares
    __shared__ h8v sq[T * NG * NQ][64];                          // query operands
    __shared__ f4v so[KA_WAVES][ROUND][PACK ? 32 : 64];
    __shared__ float tops[KA_WAVES][T][16], sm[KA_WAVES][T][16], sl[KA_WAVES][T][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int split = blockIdx.x, kvh = blockIdx.y, row0 = (gridDim.z - 1 - blockIdx.z) * ROWS;   // (longest rows first)
    const int rows = A.M * A.G;
    // queries: lane (r, c) has row r's dimensions of chunk c, product step j the
    // eight from 8 (NG c + j) on; a wave prepares some steps for all
    float x[T][JW][8];
    const int rq = PACK ? r & 7 : r;
#pragma unroll
    for (int t = 0; t < T; t++) {
        const float *qr = query_row(A, kvh, min(row0 + 16 * t + rq, rows - 1));
#pragma unroll
        for (int u = 0; u < JW; u++) {
            const int j = min(wave + KA_WAVES * u, NG - 1);
            *(float4 *)x[t][u] = query_quad(qr, 8 * (NG * c + j), A);
            *(float4 *)(x[t][u] + 4) = query_quad(qr, 8 * (NG * c + j) + 4, A);
        }
    }
    const int recs = (A.n_ctx + KVQ_TILE - 1) / KVQ_TILE;
    constexpr int REC = 2 * (KVQ_TILE * WIDTH * BITS / 8 + KVQ_TILE * NG);
    const uint8_t *base = A.cache + (size_t)kvh * recs * REC;
    int tile = split * KA_WAVES + wave;
    Tile<BITS, NG> cur;
    if (ONE) {
        cur.load_k(base + (size_t)min(tile, recs - 1) * REC, lane);
        cur.load_v(base + (size_t)min(tile, recs - 1) * REC, lane);
    }
    const size_t p0 = pos[0];
    auto end_of = [&](int row) { return (int)min(p0 + (size_t)token_of(A, row) + 1, (size_t)A.n_ctx); };
    const int last = end_of(min(row0 + ROWS, rows) - 1);         // positions any row sees
    const int first = end_of(row0);                              // and all rows see
    const int n_tiles = (last + KVQ_TILE - 1) / KVQ_TILE, step = A.splits * KA_WAVES;
    if (split * KA_WAVES >= n_tiles || seen_of(A, p0) >= A.from) return;   // (uniform)
    const int used = min(A.splits, (n_tiles + KA_WAVES - 1) / KA_WAVES);
    if (!ONE && tile < n_tiles) {
        cur.load_k(base + (size_t)tile * REC, lane);
        cur.load_v(base + (size_t)tile * REC, lane);
    }

    h8v q[T][NQ][NG];
    float sc[T], m[T], l[T];
    int end[T];
    f4v o[T][2 * NG];
#pragma unroll
    for (int t = 0; t < T; t++) {
        float top = 0.0f;
#pragma unroll
        for (int u = 0; u < JW; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[t][u][e]));
        top = quad_max(top);
        if (c == 0) tops[wave][t][r] = top;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < T; t++) {
        const float top = fmaxf(fmaxf(tops[0][t][r], tops[1][t][r]), fmaxf(tops[2][t][r], tops[3][t][r]));
        const float up = query_scale(top, A.score, sc[t]);
#pragma unroll
        for (int u = 0; u < JW; u++) {
            const int j = wave + KA_WAVES * u;
            h8v hi, lo;
            split_8(x[t][u], up, hi, lo);
            if (j >= NG) continue;
            if (PACK) {
                sq[t * NG + j][lane] = r < 8 ? hi : lo;
            } else {
                sq[(t * NG + j) * 2][lane] = hi;
                sq[(t * NG + j) * 2 + 1][lane] = lo;
            }
        }
        end[t] = end_of(min(row0 + 16 * t + rq, rows - 1));
        m[t] = -FLT_MAX;
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < 2 * NG; d++) o[t][d] = f4v{0, 0, 0, 0};
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
            for (int i = 0; i < NQ; i++) q[t][i][j] = sq[(t * NG + j) * NQ + i][lane];

    // (the next tile's keys are read into their registers once these are unpacked,
    // its values a phase later: no copies, and room for a third wave)
    auto take = [&](auto more) __attribute__((always_inline)) {
        const int tp = tile * KVQ_TILE;
        const bool edge = tp + KVQ_TILE > first;                 // (uniform)
        if (edge) {
            int at[NG], any = 0x7FFFFFFF;
#pragma unroll
            for (int g = 0; g < NG; g++) any = min(any, at[g] = trim_scales(cur.vs[g], tp, c, last));
            if (__any(any != 0x7FFFFFFF)) {
                const float bad = __uint_as_float(0x7FC00000u);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    int p = min(at[g], __shfl_xor(at[g], 16));   // the group's first one
                    p = min(p, __shfl_xor(p, 32));
#pragma unroll
                    for (int t = 0; t < T; t++)
                        if (p < end[t]) o[t][2 * g] = o[t][2 * g + 1] = f4v{bad, bad, bad, bad};
                }
            }
        }
        f4v s[T][2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int t = 0; t < T; t++) s[t][i] = f4v{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const h8v kf = unpack_k<BITS>(cur.k[i] + j * BITS / 4, cur.kscale(j), i);
#pragma unroll
                for (int u = 0; u < NQ; u++)
#pragma unroll
                    for (int t = 0; t < T; t++) s[t][i] = mfma(kf, q[t][u][j], s[t][i]);
            }
        }
        if constexpr (decltype(more)::value) cur.load_k(base + (size_t)(tile + step) * REC, lane);
        h8v p[T][NQ];
#pragma unroll
        for (int t = 0; t < T; t++) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = s[t][e >> 2][e & 3];
                if (PACK) y[e] += other_half(y[e]);
            }
            if (edge) {
                asm volatile("");                                // (a branch, not eight selects for every tile)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (tp + kvq_v_pos(c, e) >= end[t]) y[e] = -INFINITY;
            }
            float x[8];
            h8v hi, lo;
            exponents<8, 4>(x, y, sc[t], m[t], l[t], o[t]);
            weigh(x, l[t], hi, lo);
            if (PACK) {
                p[t][0] = r < 8 ? hi : lo;
            } else {
                p[t][0] = hi;
                p[t][NQ - 1] = lo;
            }
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
            h2v d[4], mm[4];
            v_scales(cur.vs[g], d, mm);
            h8v vf[2];
#pragma unroll
            for (int k = 0; k < 2; k++) vf[k] = unpack<BITS>(cur.v[2 * g + k], d, mm);
#pragma unroll
            for (int u = 0; u < NQ; u++)
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int t = 0; t < T; t++) o[t][2 * g + k] = mfma(vf[k], p[t][u], o[t][2 * g + k]);
        }
        if constexpr (decltype(more)::value) cur.load_v(base + (size_t)(tile + step) * REC, lane);
    };
    for (; tile + step < n_tiles; tile += step) take(std::true_type{});
    if (tile < n_tiles) take(std::false_type{});

    // the four waves' sums at their common maximum (a wave without tiles has
    // m = -FLT_MAX and l = 0), ROUND 16-dimension tiles of 16 rows at a time
#pragma unroll
    for (int t = 0; t < T; t++) {
        l[t] = quad_sum(l[t]);
        if (c == 0) {
            sm[wave][t][r] = m[t];
            sl[wave][t][r] = l[t];
        }
    }
    // (PACK: a row's two columns first; its sums are in lanes r < 8)
    const int sums = PACK ? 8 * c + r : lane;
#pragma unroll
    for (int k0 = 0; k0 < NT; k0 += ROUND) {
        if (k0) __syncthreads();                                 // (the last round is read)
#pragma unroll
        for (int k = k0; k < k0 + ROUND && k < NT; k++) {
            f4v v = o[k / (2 * NG)][k % (2 * NG)];
            if (PACK) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += other_half(v[e]);
                if (r < 8) so[wave][k - k0][sums] = v;
            } else {
                so[wave][k - k0][sums] = v;
            }
        }
        __syncthreads();
        // item: four sums of a row; in a PACK round's 32 of a tile, half a wave
        constexpr int PER = PACK ? 32 : 64;
#pragma unroll
        for (int it = 0; it < (ROUND * PER + 64 * KA_WAVES - 1) / (64 * KA_WAVES); it++) {
            const int at = threadIdx.x + it * 64 * KA_WAVES, k = k0 + at / PER, i = at % PER;
            const int rr = PACK ? i & 7 : i & 15, cc = PACK ? i >> 3 : i >> 4;
            const int t = T == 1 ? 0 : k / (2 * NG), row = row0 + 16 * t + rr;
            if (k >= NT || k >= k0 + ROUND || row >= rows) continue;
            float mx = sm[0][t][rr], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < KA_WAVES; w++) mx = fmaxf(mx, sm[w][t][rr]);
            f4v v = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < KA_WAVES; w++) {
                const float f = __builtin_amdgcn_exp2f(sm[w][t][rr] - mx);
                sum += sl[w][t][rr] * f;
                v += so[w][k - k0][i] * f;
            }
            put_sums(A, kvh, row, 16 * (k % (2 * NG)) + 4 * cc, v, mx, sum, used == 1, split, WIDTH);
        }
    }
}

// Many rows: four waves of 32 rows each share a tile's unpacked halves in LDS, a
// quarter unpacked by each of them, and PW such groups of a workgroup take tiles in
// turn, added at the end.  Products are 32x32x16: at the 16x16x32 form's
// back-to-back rate the matrix cores idle half the time (32 cycles an
// instruction against 16, measured; with vector instructions between, 19 to 23
// against 17 to 19).  A tile's weights are formed beside the next one's scores; a tile is
// unpacked while the one before it is multiplied, its words read a step
// earlier still.  777 tokens on 8000 positions of 32 heads over 8 of 128 take 217 to 226 us a
// call, 945 to 985 TFLOP/s of half products (two a product, see above) where a large library
// product of halves reaches 1136 to 1167: matrix cores busy 41%, vector units 38% of the time.
template <int BITS, int NG, int PW>
__global__ __launch_bounds__(256 * PW, NG > 4 ? 1 : 2) void kv_attn_many(const uint32_t *pos, AttnArgs A)
{
    constexpr int WIDTH = 32 * NG, NF = 2 * NG;
    constexpr int FW = (NF + 3) / 4;                             // fragments a wave unpacks, of K and V each
    constexpr int CODES = KVQ_TILE * WIDTH * BITS / 8, REC = 2 * (CODES + KVQ_TILE * NG);
    static_assert(2 * PW * 2 * NF * 1024 + 4096 <= 160 * 1024 &&
                  128 * PW * (WIDTH + 4) * 4 + 4096 <= 160 * 1024, "LDS");
    // [buffer][group][K fragments, V fragments][lane]: a fragment is an MFMA
    // operand; f of K holds 8 dimensions of each half of the 32 positions' rows, from
    // 8 f and from WIDTH / 2 + 8 f on; f of V dimensions 32 (f / 2) + 0..31 of
    // positions 16 (f % 2) + 0..15
    extern __shared__ h8v frag[];
    constexpr int ROW = WIDTH + 4;                               // floats of a row in LDS, when rows pass through it
    __shared__ int nan_at[2][PW][NG];
    __shared__ float sm[PW][4][32], sl[PW][4][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, c = lane >> 5, rw = wave % 4, pw = wave / 4;
    // workgroups that share a kv head's cache get the same blockIdx % n_head_kv; the
    // longest rows first
    const int rows = A.M * A.G, blocks = (rows + 127) / 128;
    const int kvh = blockIdx.x % A.n_head_kv, item = blockIdx.x / A.n_head_kv;
    const int split = item % A.splits, row0 = (blocks - 1 - item / A.splits) * 128;
    const size_t p0 = pos[0];
    auto end_of = [&](int row) { return (int)min(p0 + (size_t)token_of(A, row) + 1, (size_t)A.n_ctx); };
    const int last = end_of(min(row0 + 128, rows) - 1), first = end_of(row0);
    const int n_tiles = (last + KVQ_TILE - 1) / KVQ_TILE, step = A.splits * PW;
    if (split * PW >= n_tiles || seen_of(A, p0) < A.from) return;   // (uniform)
    const int used = min(A.splits, (n_tiles + PW - 1) / PW);
    const int row = row0 + 32 * rw + r, end = end_of(min(row, rows - 1));
    const uint8_t *base = A.cache + (size_t)kvh * ((A.n_ctx + KVQ_TILE - 1) / KVQ_TILE) * REC;

    // the words of this wave's fragments, and where they are in a record
    uint32_t kw[FW][BITS / 4], vw[FW][BITS / 4], kat[FW], sat[FW], vat[FW], wat[FW];
    uint8_t ks[FW];
    uint2 vs[FW];
#pragma unroll
    for (int u = 0; u < FW; u++) {
        const int f = min(rw * FW + u, NF - 1), oct = c * NF + f;
        kat[u] = r * (4 * NG * BITS) + oct * BITS;
        sat[u] = 2 * CODES + kvq_k_scale(oct >> 2, r);
        vat[u] = CODES + ((32 * (f >> 1) + r) * 4 + 2 * (f & 1) + c) * BITS;
        wat[u] = 2 * CODES + 32 * NG + (f >> 1) * 32 + (2 * (f & 1) + c) * 8;
    }
    auto record = [&](int tile) __attribute__((always_inline)) {
        return base + (size_t)min(tile, n_tiles - 1) * REC;
    };
    auto fetch_k = [&](int tile) __attribute__((always_inline)) {
        const uint8_t *rec = record(tile);
#pragma unroll
        for (int u = 0; u < FW; u++) {
            __builtin_memcpy(kw[u], __builtin_assume_aligned(rec + kat[u], BITS), BITS);
            ks[u] = rec[sat[u]];
        }
    };
    auto fetch_v = [&](int tile) __attribute__((always_inline)) {
        const uint8_t *rec = record(tile);
#pragma unroll
        for (int u = 0; u < FW; u++) {
            __builtin_memcpy(vw[u], __builtin_assume_aligned(rec + vat[u], BITS), BITS);
            vs[u] = *(const uint2 *)(rec + wat[u]);
        }
    };
    auto place = [&](int buf) __attribute__((always_inline)) {   // a tile's K fragments; V's NF further on
        return frag + (size_t)(buf * PW + pw) * 2 * NF * 64 + lane;
    };
    auto stage_k = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < FW; u++) {
            const int f = rw * FW + u;
            if (4 * FW > NF && f >= NF) break;
            place(buf)[f * 64] = unpack_k<BITS>(kw[u], ks[u], 0);
        }
    };
    auto stage_v = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < FW; u++) {
            const int f = rw * FW + u;
            if (4 * FW > NF && f >= NF) break;
            h2v d[4], mm[4];
            v_scales(vs[u], d, mm);
            place(buf)[(NF + f) * 64] = unpack<BITS>(vw[u], d, mm);
        }
    };
    // the fetched V words' scales, where not every row sees the tile whole
    auto trim = [&](int tile, int buf) __attribute__((always_inline)) {
        const int tp = tile * KVQ_TILE;
        if (tp + KVQ_TILE <= first) return;                      // (uniform)
#pragma unroll
        for (int u = 0; u < FW; u++) {
            const int f = rw * FW + u;
            int p = trim_scales(vs[u], tp, 2 * (f & 1) + c, last);
            p = min(p, __shfl_xor(p, 32));
            if (lane == 0 && f < NF) atomicMin(&nan_at[buf][pw][f >> 1], p);
        }
    };

    if (threadIdx.x < 2 * PW * NG) (&nan_at[0][0][0])[threadIdx.x] = 0x7FFFFFFF;
    int tile = split * PW + pw;
    fetch_k(tile);
    fetch_v(tile);
    // queries, through LDS: a row's pieces side by side from memory (a lane a
    // row touches 64 lines with every load)
    float *rowbuf = (float *)frag;
    constexpr int QUADS = WIDTH / 4, AT_ONCE = 256 * PW / QUADS;   // rows that the threads cover at once
    const int rr0 = threadIdx.x / QUADS, d0 = threadIdx.x % QUADS * 4;
    if (rr0 < AT_ONCE) {
        if (A.q_wide) {
#pragma unroll 8
            for (int rr = rr0; rr < 128; rr += AT_ONCE)
                *(f4v *)(rowbuf + rr * ROW + d0) =
                    d0 < A.hd ? *(const f4v *)(query_row(A, kvh, min(row0 + rr, rows - 1)) + d0) : f4v{0, 0, 0, 0};
        } else {
#pragma unroll 1
            for (int rr = rr0; rr < 128; rr += AT_ONCE)
                *(float4 *)(rowbuf + rr * ROW + d0) =
                    query_quad(query_row(A, kvh, min(row0 + rr, rows - 1)), d0, A);
        }
    }
    __syncthreads();
    h8v qh[NF], ql[NF];
    float sc;
    {
        float x[NF][8];
#pragma unroll
        for (int j = 0; j < 2 * NF; j++)
            *(float4 *)&x[j >> 1][4 * (j & 1)] =
                *(const float4 *)(rowbuf + (32 * rw + r) * ROW + 8 * NF * c + 4 * j);
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < NF; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[j][e]));
        const float up = query_scale(fmaxf(top, __shfl_xor(top, 32)), A.score, sc);
#pragma unroll
        for (int j = 0; j < NF; j++) split_8(x[j], up, qh[j], ql[j]);
    }
    float m = -FLT_MAX, l = 0.0f;
    f16v o[NG], s;
#pragma unroll
    for (int d = 0; d < NG; d++) o[d] = f16v{};
    auto score = [&](int buf) __attribute__((always_inline)) {
        const h8v *src = place(buf);
        s = f16v{};
#pragma unroll
        for (int f = 0; f < NF; f++) {
            const h8v kf = src[f * 64];
            s = mfma(kf, qh[f], s);
            s = mfma(kf, ql[f], s);
        }
    };
    __syncthreads();                                             // (nan_at; the queries are read)
    trim(tile, 0);
    stage_k(0);
    stage_v(0);
    fetch_k(tile + step);
    stage_k(1);
    fetch_k(tile + 2 * step);
    fetch_v(tile + step);
    __syncthreads();
    score(0);
    __syncthreads();                                             // (the loop writes K's buffer 0 again)
    const int n_steps = (n_tiles - split * PW + step - 1) / step;
    for (int n = 0; n < n_steps; n++, tile += step) {
        const int buf = n & 1, tp = tile * KVQ_TILE;
        if (tp + KVQ_TILE > first) {                             // (uniform)
            asm volatile("");                                    // (a branch, not selects for every tile)
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (tp + 8 * (e >> 2) + 4 * c + (e & 3) >= end) s[e] = -INFINITY;
#pragma unroll
            for (int g = 0; g < NG; g++)
                if (nan_at[buf][pw][g] < end) o[g] = f16v{} + __uint_as_float(0x7FC00000u);
        }
        trim(tile + step, buf ^ 1);
        // this tile's weights beside the next one's scores
        float y[16], x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) y[e] = s[e];
        exponents<16, 2>(x, y, sc, m, l, o);
        h8v ph[2], pl[2];
        weigh(x, l, ph[0], pl[0]);
        weigh(x + 8, l, ph[1], pl[1]);
        score(buf ^ 1);
        // its values beside the unpacking of the next one's, and of the keys after those
        stage_k(buf);
        stage_v(buf ^ 1);
        fetch_k(tile + 3 * step);
        fetch_v(tile + 2 * step);
        const h8v *src = place(buf) + NF * 64;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int d = 0; d < NG; d++) {
                const h8v vf = src[(2 * d + i) * 64];
                o[d] = mfma(vf, ph[i], o[d]);
                o[d] = mfma(vf, pl[i], o[d]);
            }
        __syncthreads();
    }

    // the groups' sums through LDS, added at their common maximum; rows whole to
    // memory, every thread a column quad of some (in loops: code that a workgroup
    // runs once costs its way to the instruction cache, 0.2 us a 128 bytes)
    l += __shfl_xor(l, 32);
    if (c == 0) {
        sm[pw][rw][r] = m;
        sl[pw][rw][r] = l;
    }
    float *mine = rowbuf + ((pw * 4 + rw) * 32 + r) * ROW + 4 * c;
#pragma unroll
    for (int k = 0; k < 4 * NG; k++)
        *(f4v *)(mine + 8 * k) = f4v{o[k >> 2][4 * (k & 3)], o[k >> 2][4 * (k & 3) + 1],
                                     o[k >> 2][4 * (k & 3) + 2], o[k >> 2][4 * (k & 3) + 3]};
    __syncthreads();
    int thread = threadIdx.x;
    asm("" : "+v"(thread));                                      // (found again, not kept through the loop)
    const int d1 = thread % QUADS * 4;
    if (thread / QUADS >= AT_ONCE) return;
#pragma unroll 2
    for (int rr = thread / QUADS; rr < 128; rr += AT_ONCE) {
        const int at = row0 + rr;
        if (at >= rows) break;
        float mx = sm[0][0][rr], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < PW; w++) mx = fmaxf(mx, sm[w][0][rr]);
        f4v v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < PW; w++) {
            const float f = __builtin_amdgcn_exp2f(sm[w][0][rr] - mx);
            sum += sl[w][0][rr] * f;
            v += *(const f4v *)(rowbuf + (w * 128 + rr) * ROW + d1) * f;
        }
        if (used > 1) {
            float *dst = A.part + (((size_t)kvh * rows + at) * A.splits + split) * (4 + WIDTH);
            *(f4v *)(dst + 4 + d1) = v;
            if (d1 == 0) {
                dst[0] = mx;
                dst[1] = sum;
            }
        } else {
            put_row(A, kvh, at, d1, v * (0.25f / sum));
        }
    }
}

// One workgroup per (row, kv head): the splits' records at their common
// maximum.  32 threads to a column quad's splits, eight split groups.  (EITHER: both
// kernels were launched; otherwise the position is not waited for.)
template <bool EITHER>
__global__ __launch_bounds__(256) void kv_merge_k(const uint32_t *pos, AttnArgs A, int width, KvqParts few, KvqParts many)
{
    __shared__ float sm[8], sl[8];
    __shared__ f4v so[8][32];
    const int row = blockIdx.x, kvh = blockIdx.y, rows = A.M * A.G;
    const int tid = threadIdx.x, sg = tid >> 5, cq = tid & 31;
    const size_t rec = 4 + (size_t)width;
    // the splits that hold this row: of its block of P.rows rows, P.tiles tiles
    // of a split at a time
    const KvqParts P = EITHER && seen_of(A, pos[0]) >= A.from ? many : few;
    const float *base = A.part + ((size_t)kvh * rows + row) * P.splits * rec;
    const int row_last = min(row / P.rows * P.rows + P.rows, rows) - 1;
    const int last = (int)min((size_t)pos[0] + (size_t)token_of(A, row_last) + 1, (size_t)A.n_ctx);
    const int n_tiles = (last + KVQ_TILE - 1) / KVQ_TILE;
    const int used = min(P.splits, (n_tiles + P.tiles - 1) / P.tiles);
    for (int c0 = 0; c0 < width / 4; c0 += 32) {
        const int c4 = min(c0 + cq, width / 4 - 1);
        float m = -FLT_MAX, l = 0.0f;
        f4v o = {0, 0, 0, 0};
        for (int s0 = sg; s0 < P.splits; s0 += 8 * 8) {
            float ms[8], ls[8];
            f4v os[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {                         // (read together, ahead of the position:
                const float *p = base + (size_t)min(s0 + 8 * k, P.splits - 1) * rec;   // unused ones are
                ms[k] = p[0];                                     // there and left out below)
                ls[k] = p[1];
                os[k] = *(const f4v *)(p + 4 + 4 * c4);
            }
            if (s0 >= used) break;
            float mn = m;
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (s0 + 8 * k < used) mn = fmaxf(mn, ms[k]);
            const float f = __builtin_amdgcn_exp2f(m - mn);
            l *= f;
            o *= f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (s0 + 8 * k >= used) continue;
                const float g = __builtin_amdgcn_exp2f(ms[k] - mn);
                l += ls[k] * g;
                o += os[k] * g;
            }
            m = mn;
        }
        if (used == 1) return;                                    // (uniform; written whole)
        if (cq == 0) {
            sm[sg] = m;
            sl[sg] = l;
        }
        so[sg][cq] = o;
        __syncthreads();
        if (sg == 0 && c0 + cq < width / 4) {
            float mx = sm[0], sum = 0.0f;
            for (int g = 1; g < 8; g++) mx = fmaxf(mx, sm[g]);
            f4v v = {0, 0, 0, 0};
            for (int g = 0; g < 8; g++) {
                const float f = __builtin_amdgcn_exp2f(sm[g] - mx);
                sum += sl[g] * f;
                v += so[g][cq] * f;
            }
            put_row(A, kvh, row, 4 * c4, v * (0.25f / sum));
        }
        __syncthreads();
    }
}

// The same for up to 16 splits: 32 threads to a row, eight rows to a workgroup,
// a column quad's records read together.
template <bool EITHER>
__global__ __launch_bounds__(256) void kv_merge_rows_k(const uint32_t *pos, AttnArgs A, int width, KvqParts few, KvqParts many)
{
    const int rows = A.M * A.G, row = blockIdx.x * 8 + (threadIdx.x >> 5), kvh = blockIdx.y;
    if (row >= rows) return;
    const KvqParts P = EITHER && seen_of(A, pos[0]) >= A.from ? many : few;
    const int row_last = min(row / P.rows * P.rows + P.rows, rows) - 1;
    const int last = (int)min((size_t)pos[0] + (size_t)token_of(A, row_last) + 1, (size_t)A.n_ctx);
    const int n_tiles = (last + KVQ_TILE - 1) / KVQ_TILE;
    const int used = min(P.splits, (n_tiles + P.tiles - 1) / P.tiles);
    if (used == 1) return;
    const size_t rec = 4 + (size_t)width;
    const float *base = A.part + ((size_t)kvh * rows + row) * P.splits * rec;
    for (int c4 = threadIdx.x & 31; c4 < width / 4; c4 += 32) {
        float m = -FLT_MAX, l = 0.0f;
        f4v o = {0, 0, 0, 0};
        for (int s0 = 0; s0 < used; s0 += 4) {
            float ms[4], ls[4];
            f4v os[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float *p = base + (size_t)min(s0 + k, used - 1) * rec;
                ms[k] = p[0];
                ls[k] = p[1];
                os[k] = *(const f4v *)(p + 4 + 4 * c4);
            }
            const float mn = fmaxf(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), m);
            const float f = __builtin_amdgcn_exp2f(m - mn);
            l *= f;
            o *= f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float g = s0 + k < used ? __builtin_amdgcn_exp2f(ms[k] - mn) : 0.0f;
                if (s0 + k < used) {
                    l += ls[k] * g;
                    o += os[k] * g;
                }
            }
            m = mn;
        }
        put_row(A, kvh, row, 4 * c4, o * (0.25f / l));
    }
}

template <int BITS, bool ONE>
static const void *few_kernel(int ng, int per)
{
#define FOX_FEW(n)                                                                     \
    (per == 8 ? (const void *)kv_attn_few<BITS, n, 8, ONE>                                  \
              : per == 16 ? (const void *)kv_attn_few<BITS, n, 16, ONE> : (const void *)kv_attn_few<BITS, n, 32, ONE>)
    switch (ng) {
    case 1: return FOX_FEW(1);
    case 2: return FOX_FEW(2);
    case 3: return FOX_FEW(3);
    case 4: return FOX_FEW(4);
    case 6: return FOX_FEW(6);
    default: return per == 8 ? (const void *)kv_attn_few<BITS, 8, 8, ONE> : (const void *)kv_attn_few<BITS, 8, 16, ONE>;
    }
#undef FOX_FEW
}

template <int BITS>
static const void *many_kernel(int ng)
{
    switch (ng) {
    case 1: return (const void *)kv_attn_many<BITS, 1, 2>;
    case 2: return (const void *)kv_attn_many<BITS, 2, 2>;
    case 3: return (const void *)kv_attn_many<BITS, 3, 2>;
    case 4: return (const void *)kv_attn_many<BITS, 4, 2>;
    default: return (const void *)kv_attn_many<BITS, 8, 1>;
    }
}

// What a workgroup costs, in microseconds as measured: its way in and out, a step
// (its waves' next tiles), the merge behind it and a split's records; pairs: two share a
// compute unit, in 1.2 times one's way and 1.7 times its steps.
struct Cost {
    double way, step, merge, record;
    bool pairs;
};

// Into how many splits of `most` steps at most each item's positions go: the
// fewest that give the steps that 1..4 workgroups a compute unit can have, or one.  A
// call's time is its longest workgroup's or a compute unit's share, whose
// rows see `share` of the positions on average.
static int split_count(size_t items, size_t most, int n_cu, double share, const Cost &c, double &least)
{
    size_t best = 1;
    for (int w = 0; w <= 4; w++) {                               // (w = 0: one split)
        size_t s = w ? w * (size_t)n_cu / items : 1;
        if (s > most) s = most;
        if (s == 0) continue;
        const size_t steps = (most + s - 1) / s;
        s = (most + steps - 1) / steps;
        const size_t load = (items * s + n_cu - 1) / n_cu;
        const double longest = c.step * (double)steps, mean = longest * share;
        double us = c.pairs ? (double)(load / 2) * (1.2 * c.way + 1.7 * mean) + (double)(load % 2) * (c.way + mean)
                            : (double)load * (c.way + mean);
        if (us < c.way + longest) us = c.way + longest;
        if (s > 1) us += c.merge + c.record * (double)s;
        if (w == 0 || us < least) {
            least = us;
            best = s;
        }
    }
    return (int)best;
}

// Which kernels a call launches, and how it is divided: a choice by sizes alone.
KvqPlan fox_kvq_plan(size_t head_dim, size_t n_head, size_t n_head_kv, size_t M, size_t n_ctx, int n_cu)
{
    KvqPlan p = {};
    const int width = kvq_width((int)head_dim), ng = width / 32;
    const size_t rows = M * (n_head / n_head_kv);
    // Unpacking a tile once for 128 rows costs a long way in and out (a workgroup of
    // one tile 9 us against 2 to 6), so only long work pays for it: from 9e7 pairs
    // of a row and a position on (2e7 of 256 dimensions, where a wave holds 16 rows), and
    // where the last 128 rows are not mostly empty.  In tiles by the wave and unpacked
    // once, kv heads x rows x positions, of 128 dimensions: 8 x 4000 x 1500 47 / 52 us,
    // 8 x 4000 x 2500 80 / 80, 8 x 4000 x 6000 197 / 183, 8 x 3108 x 8777 279 / 224,
    // 8 x 192 x 40000 79 / 88, 8 x 512 x 40000 181 / 164; of 64: 2 x 4000 x 6000 38 / 38,
    // 2 x 4096 x 16000 87 / 79; of 256: 16 x 1024 x 1024 76 / 97, 16 x 512 x 2500
    // 87 / 80, 4 x 384 x 16000 114 / 89.  Of 192, never (4 x 6000 x 16000 675 / 716).
    // Where the position decides, both are launched and the one that it is not for
    // ends at once (2 us).  More rows than 65535 blocks of a wave's (a launch's third
    // dimension) go to kv_attn_many at any position.
    const size_t most_per = ng > 6 ? 16 : 32, turns = ng > 4 ? 1 : 2, many_blocks = (rows + 127) / 128;
    const bool wide = ng != 6 && 2 * ((rows + most_per - 1) / most_per) > (ng > 6 ? 10 : 7) * many_blocks;
    const double from = (ng > 6 ? 2e7 : 9e7) / ((double)rows * (double)n_head_kv);
    const bool fits = (rows + most_per - 1) / most_per <= 65535;
    p.from = !fits ? 0 : wide && from < (double)n_ctx ? (int)from + 1 : INT_MAX;
    p.many = p.from <= (int64_t)n_ctx;
    p.few = p.from > (int64_t)M;                                  // (a call has M positions at least)
    const double record = 1e-6 * (double)(rows * n_head_kv) * (4 + width) * sizeof(float);   // MB of a split's
    double us, least = 0.0;
    if (p.few) {
        // Rows of a workgroup, 8, 16 or 32: more of them share a tile's unpacking, but a
        // short call waits longer for one.  Whole calls, 16 / 32 rows (heads of
        // 128): 12 tokens of 32 heads over 8 at 100 positions 4.9 / 7.0 us, 31 at 1000
        // 11.1 / 13.5, at 9000 24.4 / 22.6, a prompt of 200 7.4 / 9.0, of 500 16.6 / 14.0.
        // Records cost 0.5 us a MB, at any position, where a split gains at long ones only, so
        // they count four times: 200 tokens at 700 of 32768 positions 29.9 -> 22.1 us,
        // of 5000 20.4 -> 16.9; at 9000 of 9100, 100 tokens, 47.0 -> 50.5.  (Not of more
        // dimensions, where a step is longer: 200 at 2000 of 2200 68.7 -> 76.3.)
        const size_t n = p.from < (int64_t)n_ctx ? (size_t)p.from : n_ctx;
        const double share = M < n ? 1.0 - 0.5 * (double)M / (double)n : 0.5;
        for (size_t per = 8; per <= most_per && (per == 8 || rows > per / 2); per *= 2) {
            const Cost c = {per == 32 ? 0.3 + 0.9 * ng : per == 16 ? 0.4 + 0.42 * ng : 0.2 + 0.4 * ng,
                            per == 32 ? 0.35 + 0.19 * ng : 0.2 + 0.18 * ng, 1.9,
                            (ng > 4 ? 0.5 : 2.0) * record, ng <= 4};
            const size_t blocks = (rows + per - 1) / per;
            if (blocks > 65535) continue;                        // (more rows a workgroup fit)
            const int s = split_count(n_head_kv * blocks, (n + KVQ_TILE * KA_WAVES - 1) / (KVQ_TILE * KA_WAVES),
                                      n_cu, share, c, us);
            if (p.few_blocks && us >= least) continue;
            least = us;
            p.few_blocks = blocks;
            p.few_parts = {s, (int)per, KA_WAVES};
        }
    }
    if (p.many) {
        const Cost c = {8.0, 1.65, 5.0, record, false};
        p.many_blocks = many_blocks;
        p.many_parts = {split_count(n_head_kv * many_blocks, (n_ctx + KVQ_TILE * turns - 1) / (KVQ_TILE * turns),
                                    n_cu, 1.0, c, us),
                        128, (int)turns};
    }
    return p;
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
    // (65535 blocks of 32 rows in a launch; of other widths kv_attn_many takes them)
    if (kvq_width((int)head_dim) == 192 && M * (n_head / n_head_kv) > 65535 * 32)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: %zu query rows a kv head", M * (n_head / n_head_kv));
    if (M > 1 && (q_stride < n_head * head_dim || out_stride < n_head * head_dim))
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: a stride below the row's width");
    if ((uintptr_t)cache % 16)
        return fox_fail(FOX_GPU_ERR_ARG, "kvq_attention: the cache must be 16-byte aligned");
    FOX_HIP(hipSetDevice(ctx->device));
    AttnArgs A = {};
    A.out = out;
    A.out_stride = out_stride;
    A.q = q;
    A.q_stride = q_stride;
    A.cache = (const uint8_t *)cache;
    A.n_ctx = (int)n_ctx;
    A.n_head_kv = (int)n_head_kv;
    A.G = (int)(n_head / n_head_kv);
    A.hd = (uint16_t)head_dim;
    while (((uint32_t)1 << A.g_shift) < (uint32_t)A.G) A.g_shift++;
    A.by_g = (uint32_t)((((uint64_t)1 << (30 + A.g_shift)) + (uint32_t)A.G - 1) / (uint32_t)A.G);
    A.score = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
    A.M = (uint16_t)M;
    A.q_wide = head_dim % 4 == 0 && (uintptr_t)q % 16 == 0 && (M == 1 || q_stride % 4 == 0);
    A.out_wide = head_dim % 4 == 0 && (uintptr_t)out % 16 == 0 && (M == 1 || out_stride % 4 == 0);
    const int width = kvq_width((int)head_dim), ng = width / 32;
    const size_t rows = M * (size_t)A.G;
    const bool q4 = kv_type == FOX_GPU_KV_Q4;
    const KvqPlan p = fox_kvq_plan(head_dim, n_head, n_head_kv, M, n_ctx, ctx->n_cu);
    A.from = p.from;
    const int splits = p.few_parts.splits > p.many_parts.splits ? p.few_parts.splits : p.many_parts.splits;
    if (splits > 1) {
        st = fox_ws_reserve(ctx, n_head_kv * rows * splits * (4 + (size_t)width) * sizeof(float));
        if (st) return st;
        A.part = (float *)ctx->ws;
    }
    void *args[] = {(void *)&pos, &A};
    A.splits = p.few_parts.splits;
    if (p.few) {
        const void *k = A.splits == 1 ? q4 ? few_kernel<4, true>(ng, p.few_parts.rows) : few_kernel<8, true>(ng, p.few_parts.rows)
                                      : q4 ? few_kernel<4, false>(ng, p.few_parts.rows) : few_kernel<8, false>(ng, p.few_parts.rows);
        FOX_HIP(hipLaunchKernel(k, dim3((unsigned)p.few_parts.splits, (unsigned)n_head_kv, (unsigned)p.few_blocks),
                                dim3(64 * KA_WAVES), args, 0, ctx->stream));
    }
    if (p.many) {
        A.splits = p.many_parts.splits;
        const void *k = q4 ? many_kernel<4>(ng) : many_kernel<8>(ng);
        const size_t turns = p.many_parts.tiles;
        const size_t tiles_lds = 2 * turns * 4 * ng * 1024, rows_lds = 128 * turns * (width + 4) * sizeof(float);
        const size_t lds = tiles_lds > rows_lds ? tiles_lds : rows_lds;
        FOX_HIP(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        FOX_HIP(hipLaunchKernel(k, dim3((unsigned)(n_head_kv * p.many_blocks * p.many_parts.splits)), dim3(256 * turns),
                                args, lds, ctx->stream));
    }
    if (splits > 1) {
        // a workgroup a row or eight rows: whole calls of 512 rows 18.2 / 19.9 us, of
        // 992 14.0 / 13.5 and 23.0 / 22.5
        const bool by_rows = splits <= 16 && rows * n_head_kv >= 800, either = p.few && p.many;
        KvqParts few = p.few ? p.few_parts : p.many_parts, many = p.many_parts;
        const void *k = by_rows ? either ? (const void *)kv_merge_rows_k<true> : (const void *)kv_merge_rows_k<false>
                                : either ? (const void *)kv_merge_k<true> : (const void *)kv_merge_k<false>;
        void *merge_args[] = {(void *)&pos, &A, (void *)&width, &few, &many};
        FOX_HIP(hipLaunchKernel(k, dim3((unsigned)(by_rows ? (rows + 7) / 8 : rows), (unsigned)n_head_kv), dim3(256),
                                merge_args, 0, ctx->stream));
    }
    return FOX_GPU_OK;
}
