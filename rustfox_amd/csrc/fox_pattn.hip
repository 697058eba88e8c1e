// fox_pattn.hip -- attention of one token a row over a paged cache, on the
// matrix cores.
//
// Arithmetic.  A tile is 16 positions of one kv head, by the (up to 16) query heads that
// share it:
//   S[pos][head] = sum_d K[pos][d] q[head][d]          16x16x32 products of 16 bits
//   O[dim][head] += sum_pos V[pos][dim] P[pos][head]   16x16x4 products of 32 bits
// The cache's values are multiplied as they are.  A query is the sum of two halves (its head's row
// first brought to 2^14 .. 2^15 by a power of two) or of three bfloat16 (exact), each
// its own product into the same float sums.  Weights stay floats: a 16-bit second
// product would need V by columns, eight positions of a dimension to a lane, where pages hold
// rows; of the 32-bit one, a lane of S holds four positions of one head, which are the
// operands of four products as they stand, and a row of V is read whole by 16 lanes.  Its rate is
// enough: a tile of 128 dimensions takes 1100 clocks of one SIMD's matrix unit, and
// 8 KB at the copy's rate 1600 clocks of a SIMD's share.
// The running maximum only follows scores that pass it by 8 (in powers of two), so
// between updates no lane needs another's.
//
// Division.  A row's heads have ceil(length / 64) units of 64 positions, one tile for
// each wave of a workgroup.  All units of a call, in order of row, head, position, are
// cut into equal runs, one a workgroup, whatever the lengths, which only the device knows; a
// head whose units lie in several runs is merged by a second launch.
#include "fox_paged_dev.h"

#include <cfloat>
#include <cmath>

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

#define PA_WAVES 4
#define PA_THREADS (64 * PA_WAVES)
#define PA_TILE 16
#define PA_UNIT (PA_TILE * PA_WAVES)
#define PA_ROOM 8.0f             // how far scores may pass the running maximum
#define PA_CHUNK 2048            // positions that a workgroup weighs

struct PagedAttnArgs {
    PagedDev C;
    const float *q;
    float *out;
    size_t q_stride, out_stride;
    const uint32_t *length, *seq;
    uint32_t G, M;               // query heads of a kv head; rows
    uint32_t per, tiles;         // query heads of a head tile (the last may have fewer); head tiles of a kv head
    uint32_t workers;            // workgroups that share the units
    float score;                 // log2(e) / sqrt(hd)
    // of slot (worker + item): sums [slot][per][hd], maxima and weights' sums [slot][per][2]
    float *part, *stats;
    float *scores;               // [row][head][cap], where rows are weighed
    bool q_wide, out_wide;       // rows take 16-byte accesses
};

// ---------------------------------------------------------------- division

__device__ __forceinline__ uint32_t row_length(const PagedAttnArgs &A, uint32_t t)
{
    const uint32_t s = A.seq ? A.seq[t] : t;
    return s < A.C.n_seqs ? min(A.length[t], A.C.cap) : 0;
}

__device__ __forceinline__ uint32_t units_of(uint32_t n) { return (n + PA_UNIT - 1) / PA_UNIT; }

// Where the units of each row begin, counted for one of its heads (an item): up to 64
// rows by every wave for itself, lane t row t, without LDS or a barrier; more by the
// workgroup, in LDS.
struct PagedWork {
    const uint64_t *start;        // [M + 1], past 64 rows
    uint64_t run, total;          // units of a worker; of the call
    uint32_t items, M, before, units;

    // the row that holds unit u of the call, and its first unit of one item
    __device__ __forceinline__ uint32_t row_of(uint64_t u, uint64_t &first, uint32_t &n) const
    {
        uint32_t t;
        if (M <= 64) {
            const uint32_t lane = threadIdx.x & 63;
            t = 63 - __builtin_clzll(__ballot(lane < M && (uint64_t)before * items <= u));
        } else {
            uint32_t lo = 0, hi = M;                        // the last with start items <= u
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (start[mid] * items <= u) lo = mid;
                else hi = mid;
            }
            t = __builtin_amdgcn_readfirstlane(lo);
        }
        row(t, first, n);
        return t;
    }
    __device__ __forceinline__ void row(uint32_t t, uint64_t &first, uint32_t &n) const
    {
        if (M <= 64) {
            first = (uint32_t)__builtin_amdgcn_readlane((int)before, t);
            n = (uint32_t)__builtin_amdgcn_readlane((int)units, t);
        } else {
            first = start[t];
            n = (uint32_t)(start[t + 1] - first);
        }
    }
    // the workers whose runs hold an item's units: first and last
    __device__ __forceinline__ void runs(uint32_t t, uint32_t item, uint32_t &a, uint32_t &b) const
    {
        uint64_t first;
        uint32_t n;
        row(t, first, n);
        const uint64_t u = first * items + (uint64_t)item * n;
        a = (uint32_t)(u / run);
        b = (uint32_t)((u + n - 1) / run);
    }
};

__device__ __forceinline__ PagedWork divide(const PagedAttnArgs &A, uint64_t *start)
{
    __shared__ uint64_t sums[PA_WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    PagedWork D;
    D.start = start;
    D.M = A.M;
    D.items = A.C.n_kv * A.tiles;
    if (A.M <= 64) {
        D.units = lane < A.M ? units_of(row_length(A, lane)) : 0;   // (64 of at most 2^24)
        const uint32_t x = wave_scan(D.units);
        D.before = x - D.units;
        D.total = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, (int)A.M - 1) * D.items;
    } else {
        const uint32_t each = (A.M + PA_THREADS - 1) / PA_THREADS;  // (at most 4)
        uint64_t mine = 0;
        for (uint32_t i = 0; i < each; i++) {
            const uint32_t t = tid * each + i;
            if (t < A.M) mine += units_of(row_length(A, t));
        }
        uint64_t x = mine;
        for (uint32_t m = 1; m < 64; m <<= 1) {
            const uint64_t y = __shfl_up((unsigned long long)x, m);
            if (lane >= m) x += y;
        }
        if (lane == 63) sums[w] = x;
        __syncthreads();
        uint64_t before = x - mine;
        for (uint32_t i = 0; i < w; i++) before += sums[i];
        for (uint32_t i = 0; i < each; i++) {
            const uint32_t t = tid * each + i;
            if (t >= A.M) break;
            start[t] = before;
            before += units_of(row_length(A, t));
        }
        if (tid == PA_THREADS - 1) start[A.M] = before;
        __syncthreads();
        D.total = start[A.M] * D.items;
    }
    D.run = (D.total + A.workers - 1) / A.workers;
    return D;
}

// ------------------------------------------------------------------- tiles

// eight floats of a query's row from dimension d on (zero past hd)
__device__ __forceinline__ void load_q(float x[8], const float *row, uint32_t d, uint32_t hd, bool on, bool wide)
{
    on = on && d < hd;
    if (wide) {
        *(float4 *)x = on ? *(const float4 *)(row + d) : float4{0, 0, 0, 0};
        *(float4 *)(x + 4) = on ? *(const float4 *)(row + d + 4) : float4{0, 0, 0, 0};
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = on ? row[d + i] : 0.0f;
}

// the parts of eight query values: two halves of x 2^e, or three bfloat16
template <bool BF>
__device__ __forceinline__ void split_q(uint4 part[BF ? 3 : 2], const float x[8], int e)
{
    uint32_t w[3][4] = {};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (BF) {
            float r = x[i];
#pragma unroll
            for (int k = 0; k < 3; k++) {                // (truncated: what is left is exact)
                const uint32_t u = __float_as_uint(r) & 0xFFFF0000u;
                w[k][i / 2] |= i & 1 ? u : u >> 16;
                r -= __uint_as_float(u);
            }
        } else {
            const float y = ldexpf(x[i], e);
            const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
            w[0][i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, hi) << (16 * (i & 1));
            w[1][i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, lo) << (16 * (i & 1));
        }
    }
#pragma unroll
    for (int k = 0; k < (BF ? 3 : 2); k++) part[k] = uint4{w[k][0], w[k][1], w[k][2], w[k][3]};
}

template <bool BF>
__device__ __forceinline__ f4v mfma_16(uint4 a, uint4 b, f4v c)
{
    if (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}

// value 0 or 1 of two
template <bool BF>
__device__ __forceinline__ float value_of(uint32_t w, int i)
{
    if (BF) return __uint_as_float(i ? w & 0xFFFF0000u : w << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i ? w >> 16 : w));
}

__device__ __forceinline__ float max_of_groups(float x)      // over lanes l, l ^ 16, l ^ 32, l ^ 48
{
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_of_groups(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// One tile's keys and values as a wave holds them.  Lane l = i + 16 g: of the
// keys row i, dimensions 32 c + 8 g ..; of the values rows 4 g + r, from dimension
// 8 i on in each 128 dimensions, 4 i in the 64 after those.
template <int W>
struct Tile {
    uint4 k[W / 32];
    uint4 v[W / 128 ? W / 128 : 1][4];
    uint2 u[4];
};

template <int W, bool FULL>
__device__ __forceinline__ void load_tile(Tile<W> &T, const PagedAttnArgs &A, const uint16_t *k, const uint16_t *v)
{
    const uint32_t lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, hd = FULL ? W : A.C.hd;
#pragma unroll
    for (int c = 0; c < W / 32; c++) {
        T.k[c] = uint4{0, 0, 0, 0};
        if (FULL || 32 * c + 8 * g < hd) T.k[c] = *(const uint4 *)(k + (size_t)i * hd + 32 * c + 8 * g);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const uint16_t *row = v + (size_t)(4 * g + r) * hd;
#pragma unroll
        for (int b = 0; b < W / 128; b++) {
            T.v[b][r] = uint4{0, 0, 0, 0};
            if (FULL || 128 * b + 8 * i < hd) T.v[b][r] = *(const uint4 *)(row + 128 * b + 8 * i);
        }
        if (W % 128) {
            constexpr int at = W / 128 * 128;
            T.u[r] = uint2{0, 0};
            if (FULL || at + 4 * i < hd) T.u[r] = *(const uint2 *)(row + at + 4 * i);
        }
    }
}

// W: dimensions, up to the next of 64, 128, 192, 256; FULL: hd is that
template <bool BF, int W, bool FULL, bool WEIGH>
__global__ __launch_bounds__(PA_THREADS, 2) void paged_attn_k(PagedAttnArgs A)
{
    constexpr int NC = W / 32, NP = BF ? 3 : 2, NB = W / 128, NU = W % 128 ? 4 : 0, NA = NB * 8 + NU;
    constexpr bool QLDS = W > 128;           // queries' parts stay in LDS
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float wm[PA_WAVES][16], wl[PA_WAVES][16];
    __shared__ uint4 qlds[QLDS ? NP * NC * 64 : 1];
    uint64_t *start = (uint64_t *)lds;
    float *sums = (float *)(lds + ((size_t)(A.M + 1) * 8 + 15) / 16 * 16);     // [wave][head][hd]
    const uint32_t tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t hd = FULL ? W : A.C.hd, width = A.C.n_kv * A.G * hd;
    const PagedWork D = divide(A, start);
    for (uint32_t t = blockIdx.x; t < A.M; t += gridDim.x) {
        uint64_t first;
        uint32_t n;
        D.row(t, first, n);
        if (n == 0)
            for (uint32_t d = tid; d < width; d += PA_THREADS) A.out[t * A.out_stride + d] = 0.0f;
    }
    uint64_t u = blockIdx.x * D.run;
    const uint64_t end = min(u + D.run, D.total);
    while (u < end) {                                       // (uniform)
        uint64_t first;
        uint32_t units;
        const uint32_t t = D.row_of(u, first, units);
        const uint64_t in_row = u - first * D.items;
        const uint32_t item = __builtin_amdgcn_readfirstlane((uint32_t)(in_row / units));
        const uint32_t k0 = __builtin_amdgcn_readfirstlane((uint32_t)(in_row - (uint64_t)item * units));
        const uint32_t k1 = __builtin_amdgcn_readfirstlane((uint32_t)min((uint64_t)units, k0 + (end - u)));
        const uint32_t h = item / A.tiles, h0 = item % A.tiles * A.per, heads = min(A.per, A.G - h0);
        const uint32_t n = __builtin_amdgcn_readfirstlane(row_length(A, t));
        const uint32_t s = A.seq ? A.seq[t] : t;
        const uint32_t *table = A.C.table + (size_t)s * A.C.max_pages;

        // the queries' rows and the first tile are asked for together
        float x[NC][8], top = 0.0f;
        {
            const float *row = A.q + t * A.q_stride + (size_t)(h * A.G + h0 + (i < heads ? i : 0)) * hd;
#pragma unroll
            for (int c = 0; c < NC; c++) load_q(x[c], row, 32 * c + 8 * g, hd, i < heads, A.q_wide);
        }
        Tile<W> now, next;
        const uint32_t in_page = (1u << A.C.shift) - 1;
        auto load = [&](Tile<W> &T, uint32_t page, uint32_t p) {       // p: a tile's first position
            const size_t at = ((((size_t)page * A.C.n_kv + h) << A.C.shift) + (p & in_page)) * hd;
            load_tile<W, FULL>(T, A, (const uint16_t *)A.C.k + at, (const uint16_t *)A.C.v + at);
        };
        uint32_t p0 = k0 * PA_UNIT + wave * PA_TILE;
        const uint32_t stop = min(n, k1 * PA_UNIT);
        // pages of this tile and the next, read one tile before its rows are
        uint32_t page = p0 < stop ? table[p0 >> A.C.shift] : ~0u;
        uint32_t page_next = p0 + PA_UNIT < stop ? table[(p0 + PA_UNIT) >> A.C.shift] : ~0u;
        if (page < A.C.n_pages) load(now, page, p0);

        uint4 q[QLDS ? 1 : NC][NP];
        float factor;
        {
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[c][j]));
            int e = 0;
            if (!BF) {
                top = max_of_groups(top);
                // (top is in 2^-149 .. 2^128; an infinity stays one)
                e = top > 0.0f && top <= FLT_MAX ? 15 - (ilogbf(top) + 1) : 0;
            }
            factor = ldexpf(A.score, -e);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                uint4 p[NP];
                split_q<BF>(p, x[c], e);
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    if (!QLDS) q[c][k] = p[k];
                    else if (c % PA_WAVES == wave) qlds[(c * NP + k) * 64 + lane] = p[k];
                }
            }
            if (QLDS) __syncthreads();
        }

        f4v acc[NA];
#pragma unroll
        for (int a = 0; a < NA; a++) acc[a] = f4v{0, 0, 0, 0};
        float m = -INFINITY, l = 0.0f;
        while (p0 < stop) {
            const uint32_t p1 = p0 + PA_UNIT, p2 = p1 + PA_UNIT;
            const uint32_t page_after = p2 < stop ? table[p2 >> A.C.shift] : ~0u;
            if (page_next < A.C.n_pages) load(next, page_next, p1);
            if (page < A.C.n_pages) {
                f4v S = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int k = 0; k < NP; k++)
                        S = mfma_16<BF>(now.k[c], QLDS ? qlds[(c * NP + k) * 64 + lane] : q[QLDS ? 0 : c][k], S);
                float sc[4];
                const uint32_t p = p0 + 4 * g;
#pragma unroll
                for (int r = 0; r < 4; r++) sc[r] = S[r] * factor;
                if (p0 + PA_TILE > n) {
                    // the row's last tile: what is behind it may hold anything
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (p + r >= n) {
                            sc[r] = -INFINITY;
#pragma unroll
                            for (int b = 0; b < NB; b++) now.v[b][r] = uint4{0, 0, 0, 0};
                            if (NU) now.u[r] = uint2{0, 0};
                        }
                }
                if (WEIGH && i < heads)
                    *(f4v *)(A.scores + ((size_t)t * A.C.n_kv * A.G + h * A.G + h0 + i) * A.C.cap + p) = *(f4v *)sc;
                const float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                if (__any(top > m + PA_ROOM)) {
                    const float mx = fmaxf(m, max_of_groups(top));
                    const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
                    l *= f;
#pragma unroll
                    for (int a = 0; a < NA; a++) acc[a] *= f;
                    m = mx;
                }
                const float shift = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float w = __builtin_amdgcn_exp2f(sc[r] - shift);
                    l += w;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint32_t v[4] = {now.v[b][r].x, now.v[b][r].y, now.v[b][r].z, now.v[b][r].w};
#pragma unroll
                        for (int a = 0; a < 8; a++)
                            acc[8 * b + a] = __builtin_amdgcn_mfma_f32_16x16x4f32(value_of<BF>(v[a / 2], a & 1), w,
                                                                                  acc[8 * b + a], 0, 0, 0);
                    }
                    if (NU) {
                        const uint32_t v[2] = {now.u[r].x, now.u[r].y};
#pragma unroll
                        for (int a = 0; a < 4; a++)
                            acc[8 * NB + a] = __builtin_amdgcn_mfma_f32_16x16x4f32(value_of<BF>(v[a / 2], a & 1), w,
                                                                                   acc[8 * NB + a], 0, 0, 0);
                    }
                }
            }
            now = next;
            page = page_next;
            page_next = page_after;
            p0 = p1;
        }

        // the waves' sums at one maximum, added
        l = sum_of_groups(l);
        if (g == 0) {
            wm[wave][i] = m;
            wl[wave][i] = l;
        }
        __syncthreads();
        float mx = wm[0][i];
#pragma unroll
        for (int w = 1; w < PA_WAVES; w++) mx = fmaxf(mx, wm[w][i]);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
        if (i < heads) {
            float *to = sums + ((size_t)wave * A.per + i) * hd;
#pragma unroll
            for (int a = 0; a < NA; a++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t d = a < 8 * NB ? a / 8 * 128 + 8 * (4 * g + r) + a % 8 : NB * 128 + 4 * (4 * g + r) + a % 4;
                    // (a wave that saw nothing has no sums, but a NaN maximum must not hide)
                    if (FULL || d < hd) to[d] = m == -INFINITY ? acc[a][r] : acc[a][r] * f;
                }
        }
        __syncthreads();
        const bool whole = k0 == 0 && k1 == units;
        const size_t slot = (size_t)blockIdx.x + (size_t)t * D.items + item;
        for (uint32_t x = tid; x < heads * hd; x += PA_THREADS) {
            const uint32_t j = x / hd, d = x % hd;
            float y = sums[x];
#pragma unroll
            for (int w = 1; w < PA_WAVES; w++) y += sums[(size_t)w * A.per * hd + x];
            float top = wm[0][j], all = 0.0f;
#pragma unroll
            for (int w = 1; w < PA_WAVES; w++) top = fmaxf(top, wm[w][j]);
#pragma unroll
            for (int w = 0; w < PA_WAVES; w++)
                all += wm[w][j] == -INFINITY ? wl[w][j] : wl[w][j] * __builtin_amdgcn_exp2f(wm[w][j] - top);
            if (whole)
                A.out[t * A.out_stride + (size_t)(h * A.G + h0 + j) * hd + d] = all == 0.0f ? 0.0f : y / all;
            else
                A.part[(slot * A.per + j) * hd + d] = y;
            if (d == 0) {
                A.stats[(slot * A.per + j) * 2] = top;
                A.stats[(slot * A.per + j) * 2 + 1] = all;
            }
        }
        __syncthreads();
        u += k1 - k0;
    }
}

// ------------------------------------------------------------------- merge

// A head's maximum and sum over its parts, first .. last, by a wave: a lane a part.
// `stats` of the head in part 0.
__device__ __forceinline__ void all_parts(const float *stats, size_t stride, uint32_t first, uint32_t last, float &top,
                                          float &all)
{
    const uint32_t lane = threadIdx.x & 63;
    top = -INFINITY;
    all = 0.0f;
    for (uint32_t w = first + lane; w <= last; w += 64) {
        const float m = stats[w * stride], l = stats[w * stride + 1], mx = fmaxf(top, m);
        all = (top == -INFINITY ? all : all * __builtin_amdgcn_exp2f(top - mx)) +
              (m == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - mx));
        top = mx;
    }
    float mx = top;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
    if (top != -INFINITY) all *= __builtin_amdgcn_exp2f(top - mx);
    top = mx;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) all += __shfl_xor(all, x);
}

// A workgroup a query head: its parts at one maximum, added.  A wave takes every
// fourth part, a lane four dimensions.
__global__ __launch_bounds__(PA_THREADS) void paged_merge_k(PagedAttnArgs A)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ __attribute__((aligned(16))) float sums[PA_WAVES][256];
    const PagedWork D = divide(A, (uint64_t *)lds);
    const uint32_t t = blockIdx.y, head = blockIdx.x, h = head / A.G, j = head % A.G, tid = threadIdx.x;
    const uint32_t wave = tid >> 6, d = (tid & 63) * 4, hd = A.C.hd;
    const uint32_t item = h * A.tiles + j / A.per;
    uint64_t at;
    uint32_t units, first, last;
    D.row(t, at, units);
    if (units == 0) return;
    D.runs(t, item, first, last);
    if (first == last) return;
    const size_t slot = (size_t)t * D.items + item;
    const float *stats = A.stats + (slot * A.per + j % A.per) * 2;
    const float *part = A.part + (slot * A.per + j % A.per) * hd + d;
    float top, all;
    all_parts(stats, A.per * 2, first, last, top, all);
    float4 y = {0, 0, 0, 0};
    if (d < hd)
#pragma unroll 4
        for (uint32_t w = first + wave; w <= last; w += PA_WAVES) {
            const float m = stats[(size_t)w * A.per * 2], f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
            const float4 x = *(const float4 *)(part + (size_t)w * A.per * hd);
            y.x += x.x * f;
            y.y += x.y * f;
            y.z += x.z * f;
            y.w += x.w * f;
        }
    *(float4 *)(sums[wave] + d) = y;
    __syncthreads();
    if (tid < hd)
        A.out[t * A.out_stride + (size_t)head * hd + tid] =
            all == 0.0f ? 0.0f : (sums[0][tid] + sums[1][tid] + sums[2][tid] + sums[3][tid]) / all;
}

// A workgroup a kv head's PA_CHUNK positions: the group's weights of each, from the scores,
// summed before they are added to what the row has.
__global__ __launch_bounds__(PA_THREADS) void paged_weigh_k(PagedAttnArgs A)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const PagedWork D = divide(A, (uint64_t *)lds);
    const uint32_t t = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const uint32_t n = row_length(A, t), p0 = blockIdx.x * PA_CHUNK;
    if (p0 >= n) return;
    float sum[PA_CHUNK / PA_THREADS] = {};
    for (uint32_t j = 0; j < A.G; j++) {
        const uint32_t item = h * A.tiles + j / A.per;
        uint32_t first, last;
        D.runs(t, item, first, last);
        float top, all;
        all_parts(A.stats + (((size_t)t * D.items + item) * A.per + j % A.per) * 2, A.per * 2, first, last, top, all);
        const float *sc = A.scores + ((size_t)t * A.C.n_kv * A.G + h * A.G + j) * A.C.cap;
        if (all == 0.0f) continue;
#pragma unroll
        for (int x = 0; x < PA_CHUNK / PA_THREADS; x++) {
            const uint32_t p = p0 + x * PA_THREADS + tid;
            if (p < n) sum[x] += __builtin_amdgcn_exp2f(sc[p] - top) / all;
        }
    }
    float *weight = A.C.weight + ((size_t)t * A.C.n_kv + h) * A.C.cap;
#pragma unroll
    for (int x = 0; x < PA_CHUNK / PA_THREADS; x++) {
        const uint32_t p = p0 + x * PA_THREADS + tid;
        if (p < n && A.C.table[(size_t)t * A.C.max_pages + (p >> A.C.shift)] < A.C.n_pages) weight[p] += sum[x];
    }
}

template <bool BF, bool WEIGH>
static const void *attn_kernel(size_t hd)
{
#define FOX_ATTN(w) (hd == w ? (const void *)paged_attn_k<BF, w, true, WEIGH> : (const void *)paged_attn_k<BF, w, false, WEIGH>)
    return hd <= 64 ? FOX_ATTN(64) : hd <= 128 ? FOX_ATTN(128) : hd <= 192 ? FOX_ATTN(192) : FOX_ATTN(256);
#undef FOX_ATTN
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
    A.tiles = (A.G + 15) / 16;
    A.per = (A.G + A.tiles - 1) / A.tiles;
    A.score = (float)(1.4426950408889634 / std::sqrt((double)cache->head_dim));
    A.q_wide = (uintptr_t)q % 16 == 0 && (M == 1 || q_stride % 4 == 0);
    A.out_wide = (uintptr_t)out % 16 == 0 && (M == 1 || out_stride % 4 == 0);
    const size_t items = M * cache->n_head_kv * A.tiles;
    const size_t most = items * ((A.C.cap + PA_UNIT - 1) / PA_UNIT);
    A.workers = (uint32_t)(most < (size_t)2 * ctx->n_cu ? most : (size_t)2 * ctx->n_cu);
    // parts, their maxima and sums, and the scores of rows that are weighed
    const size_t slots = items + A.workers, part = slots * A.per * cache->head_dim, stats = slots * A.per * 2;
    const size_t scores = weigh ? M * n_head * A.C.cap : 0;
    if (scores > (size_t)1 << 34)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: the weights of %zu tokens' %zu heads over %u rows are too "
                        "many", M, n_head, A.C.cap);
    if ((st = fox_ws_reserve(ctx, (scores + part + stats) * sizeof(float)))) return st;
    A.scores = (float *)ctx->ws;
    A.part = A.scores + scores;
    A.stats = A.part + part;
    FOX_HIP(hipSetDevice(ctx->device));
    const bool bf = cache->type == FOX_GPU_BF16;
    const void *k = weigh ? bf ? attn_kernel<true, true>(cache->head_dim) : attn_kernel<false, true>(cache->head_dim)
                          : bf ? attn_kernel<true, false>(cache->head_dim) : attn_kernel<false, false>(cache->head_dim);
    const size_t starts = ((M + 1) * 8 + 15) / 16 * 16;
    const size_t lds = starts + (size_t)PA_WAVES * A.per * cache->head_dim * sizeof(float);
    void *args[] = {&A};
    FOX_HIP(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    FOX_HIP(hipLaunchKernel(k, dim3(A.workers), dim3(PA_THREADS), args, lds, ctx->stream));
    if (A.workers > 1)
        FOX_HIP(hipLaunchKernel((const void *)paged_merge_k, dim3((unsigned)n_head, (unsigned)M), dim3(PA_THREADS),
                                args, starts, ctx->stream));
    if (weigh)
        FOX_HIP(hipLaunchKernel((const void *)paged_weigh_k,
                                dim3((A.C.cap + PA_CHUNK - 1) / PA_CHUNK, (unsigned)cache->n_head_kv, (unsigned)M),
                                dim3(PA_THREADS), args, starts, ctx->stream));
    return FOX_GPU_OK;
}
