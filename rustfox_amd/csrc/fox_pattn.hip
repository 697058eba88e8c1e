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
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

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
    bool whole;                  // no: a workgroup an item
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

// A word that no kernel of the call writes, at an address that is the same for the wave: through the
// scalar cache.  (As vector loads, page numbers would be waited for behind the rows' loads.)
typedef const __attribute__((address_space(4))) uint32_t *Words;
__device__ __forceinline__ uint32_t word(const uint32_t *p, size_t i) { return ((Words)(uintptr_t)p)[i]; }

__device__ __forceinline__ uint32_t units_of(uint32_t n) { return (n + PA_UNIT - 1) / PA_UNIT; }

// Where the units of each row begin, counted for one of its heads (an item): up to 64
// rows by every wave for itself, lane t row t, without LDS or a barrier; more by the
// workgroup, in LDS.
// a / b; most calls' units are below 2^32, where a quotient takes 20 instructions, not 150
__device__ __forceinline__ uint64_t over(uint64_t a, uint32_t b)
{
    return a >> 32 ? a / b : (uint32_t)a / b;
}

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
        if (total >> 32 == 0) {
            a = (uint32_t)u / (uint32_t)run;
            b = (uint32_t)(u + n - 1) / (uint32_t)run;
        } else {
            a = (uint32_t)(u / run);
            b = (uint32_t)((u + n - 1) / run);
        }
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
    D.run = over(D.total + A.workers - 1, A.workers);
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

// x and its row's lanes' at a distance, round the row of 16
template <int BY>
__device__ __forceinline__ float add_around(float x)
{
    return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + BY, 0xF, 0xF, false));
}

template <bool BF>
__device__ __forceinline__ f4v mfma_16(u4v a, uint4 b, f4v c)
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
//
// Rows are read through a descriptor of the tile that ends with the last row that is seen: what
// lies behind reads as zeros and moves no data, and so does a tile without a page or behind
// the run (of no rows at all).  So the loads of a loop are the same in every turn, with no branch
// round them, and each wait leaves the later ones under way.
template <int W>
struct Tile {
    u4v k[W / 32];
    u4v v[W / 128 ? W / 128 : 1][4];
    u2v u[4];
};

#define PA_NOWHERE 0x40000000u   // an offset past any descriptor's end

template <int W, bool FULL>
struct Offsets {
    uint32_t k[FULL ? 1 : W / 32], v[FULL ? 1 : W / 128 + 1], u;
    __device__ __forceinline__ Offsets(uint32_t hd)
    {
        const uint32_t lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int c = 0; c < (FULL ? 1 : W / 32); c++)
            k[c] = FULL || 32 * c + 8 * g < hd ? (i * hd + 32 * c + 8 * g) * 2 : PA_NOWHERE;
#pragma unroll
        for (int b = 0; b < (FULL ? 1 : W / 128 + 1); b++) {
            const uint32_t d = b < W / 128 ? 128 * b + 8 * i : W / 128 * 128 + 4 * i;
            v[b] = FULL || d < hd ? (4 * g * hd + d) * 2 : PA_NOWHERE;
        }
        u = FULL ? (4 * g * hd + W / 128 * 128 + 4 * i) * 2 : v[W / 128];
    }
};

// An offset as it stands here: sums with it are formed where they are used, as part of the load (kept in
// registers from before the loop they would cost eight).  Only in the lane's offset and the
// instruction's own, which are held against the descriptor's end as one; the scalar offset
// is taken from the end first, below zero for few rows.
__device__ __forceinline__ uint32_t here(uint32_t x)
{
    asm volatile("" : "+v"(x));
    return x;
}

template <int W, bool FULL>
__device__ __forceinline__ void load_keys(Tile<W> &T, __amdgpu_buffer_rsrc_t at, const Offsets<W, FULL> &O)
{
    const uint32_t k = here(O.k[0]);
#pragma unroll
    for (int c = 0; c < W / 32; c++)
        T.k[c] = __builtin_amdgcn_raw_buffer_load_b128(at, FULL ? k + 64 * c : O.k[FULL ? 0 : c], 0, 0);
}

template <int W, bool FULL>
__device__ __forceinline__ void load_values(Tile<W> &T, __amdgpu_buffer_rsrc_t at, const Offsets<W, FULL> &O, uint32_t hd)
{
    const uint32_t row = FULL ? W * 2 : hd * 2;
#pragma unroll
    for (int b = 0; b < W / 128; b++) {
        const uint32_t v = here(O.v[FULL ? 0 : b]) + (FULL ? 256 * b : 0);
#pragma unroll
        for (int r = 0; r < 4; r++) T.v[b][r] = __builtin_amdgcn_raw_buffer_load_b128(at, v + r * row, 0, 0);
    }
    if (W % 128) {
        const uint32_t u = here(O.u);
#pragma unroll
        for (int r = 0; r < 4; r++) T.u[r] = __builtin_amdgcn_raw_buffer_load_b64(at, u + r * row, 0, 0);
    }
}

// One worker's run of units (or one item, where `whole`).  W: dimensions, up to the next of
// 64, 128, 192, 256; FULL: hd is that; HG: heads of a tile, up to 4 or 16.
//
// Up to 4 heads leave 12 columns of a 16-column product unused.  The queries' parts take them
// in the first: columns 4 k + head hold part k, and two adds round the row give every
// column its head's whole score.  The second is then sixteen products of 4x4x1 (a quarter of the
// matrix unit's time): block b multiplies what its four lanes hold, V's dimensions of
// one position and the weights of the four heads there.
template <bool BF, int W, bool FULL, int HG>
__global__ __launch_bounds__(PA_THREADS, HG == 4 && W <= 128 ? 3 : 2) void paged_attn_k(PagedAttnArgs A)
{
    constexpr int NC = W / 32, NP = HG == 4 ? 1 : BF ? 3 : 2, NB = W / 128, NU = W % 128 ? 4 : 0, NA = NB * 8 + NU;
    constexpr bool QLDS = W > (HG == 4 ? 192 : 128);     // queries' parts stay in LDS
    constexpr int PARTS = HG == 4 ? 4 * PA_WAVES : PA_WAVES;   // partial sums of a workgroup
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float wm[PA_WAVES][HG], wl[PA_WAVES][HG];
    __shared__ uint4 qlds[QLDS ? NP * NC * 64 : 1];
    float *sums = (float *)(lds + (A.M > 64 && !A.whole ? ((size_t)(A.M + 1) * 8 + 15) / 16 * 16 : 0));     // [part][head][hd]
    const uint32_t tid = threadIdx.x, lane = tid & 63, i = lane & 15, g = lane >> 4, col = HG == 4 ? i & 3 : i;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t hd = FULL ? W : A.C.hd, width = A.C.n_kv * A.G * hd, items = A.C.n_kv * A.tiles;
    PagedWork D;
    uint64_t u = 0, end = 1;
    if (!A.whole) {
        D = divide(A, (uint64_t *)lds);
        for (uint32_t t = blockIdx.x; t < A.M; t += gridDim.x) {
            uint64_t first;
            uint32_t n;
            D.row(t, first, n);
            if (n == 0)
                for (uint32_t d = tid; d < width; d += PA_THREADS) A.out[t * A.out_stride + d] = 0.0f;
        }
        u = blockIdx.x * D.run;
        end = min(u + D.run, D.total);
    }
    while (u < end) {                                       // (uniform)
        uint32_t t, item, k0 = 0, k1, units;
        if (A.whole) {
            t = blockIdx.x / items;
            item = blockIdx.x - t * items;
            units = k1 = units_of(row_length(A, t));
        } else {
            uint64_t first;
            t = D.row_of(u, first, units);
            const uint64_t in_row = u - first * items;
            item = (uint32_t)over(in_row, units);
            k0 = (uint32_t)(in_row - (uint64_t)item * units);
            k1 = (uint32_t)min((uint64_t)units, k0 + (end - u));
        }
        t = __builtin_amdgcn_readfirstlane(t);
        item = __builtin_amdgcn_readfirstlane(item);
        k0 = __builtin_amdgcn_readfirstlane(k0);
        k1 = __builtin_amdgcn_readfirstlane(k1);
        const uint32_t h = item / A.tiles, h0 = item % A.tiles * A.per, heads = min(A.per, A.G - h0);
        const uint32_t sq = A.seq ? word(A.seq, t) : t;
        const uint32_t n = sq < A.C.n_seqs ? min(word(A.length, t), A.C.cap) : 0, s = n ? sq : 0;
        const uint32_t *table = A.C.table + (size_t)s * A.C.max_pages;

        // the queries' rows and the first tile are asked for together
        float x[NC][8];
        {
            const float *row = A.q + t * A.q_stride + (size_t)(h * A.G + h0 + (col < heads ? col : 0)) * hd;
#pragma unroll
            for (int c = 0; c < NC; c++) load_q(x[c], row, 32 * c + 8 * g, hd, col < heads, A.q_wide);
        }
        // Tiles of this wave: p0, p0 + PA_UNIT, ...; two are held, and as soon as one's keys
        // (values) are used, those of the tile after the next are asked for in their place.
        const Offsets<W, FULL> O(hd);
        Tile<W> one, two;
        const uint32_t in_page = (1u << A.C.shift) - 1, stop = min(n, k1 * PA_UNIT);
        uint32_t p0 = k0 * PA_UNIT + wave * PA_TILE;
        auto page_of = [&](uint32_t p) -> uint32_t { return p < stop ? word(table, p >> A.C.shift) : ~0u; };
        auto rows_of = [&](uint32_t p, uint32_t page) -> uint32_t {   // that are seen
            return p < stop && page < A.C.n_pages ? min(n - p, (uint32_t)PA_TILE) : 0;
        };
        auto tile_at = [&](const void *pool, uint32_t p, uint32_t page) -> __amdgpu_buffer_rsrc_t {
            const uint32_t rows = rows_of(p, page);
            const size_t at = rows ? ((((size_t)page * A.C.n_kv + h) << A.C.shift) + (p & in_page)) * hd : 0;
            return __builtin_amdgcn_make_buffer_rsrc((uint16_t *)pool + at, 0, rows * hd * 2, 0x00027000);
        };
        uint32_t pages[4];       // of this tile and the three after it
#pragma unroll
        for (int x = 0; x < 4; x++) pages[x] = page_of(p0 + x * PA_UNIT);
        load_keys<W, FULL>(one, tile_at(A.C.k, p0, pages[0]), O);
        load_values<W, FULL>(one, tile_at(A.C.v, p0, pages[0]), O, hd);
        load_keys<W, FULL>(two, tile_at(A.C.k, p0 + PA_UNIT, pages[1]), O);
        load_values<W, FULL>(two, tile_at(A.C.v, p0 + PA_UNIT, pages[1]), O, hd);

        uint4 q[QLDS ? 1 : NC][NP];
        float factor;
        {
            float top = 0.0f;
            int e = 0;
            if (!BF) {
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[c][j]));
                top = max_of_groups(top);
                // (top is in 2^-149 .. 2^128; an infinity stays one)
                e = top > 0.0f && top <= FLT_MAX ? 15 - (ilogbf(top) + 1) : 0;
            }
            factor = ldexpf(A.score, -e);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                uint4 p[BF ? 3 : 2];
                split_q<BF>(p, x[c], e);
                if (HG == 4) p[0] = i < 4 ? p[0] : i < 8 ? p[1] : BF && i < 12 ? p[2 - !BF] : uint4{0, 0, 0, 0};
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
        auto step = [&](Tile<W> &T) {
            const uint32_t seen = rows_of(p0, pages[0]), after = p0 + 2 * PA_UNIT;
            f4v S = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int k = 0; k < NP; k++)
                    S = mfma_16<BF>(T.k[c], QLDS ? qlds[(c * NP + k) * 64 + lane] : q[QLDS ? 0 : c][k], S);
            load_keys<W, FULL>(T, tile_at(A.C.k, after, pages[2]), O);
            float sc[4];
            const int mine = (int)seen - 4 * (int)g;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                sc[r] = (HG == 4 ? add_around<4>(add_around<8>(S[r])) : S[r]) * factor;
                if (r >= mine) sc[r] = -INFINITY;
            }
            if (A.scores && i < heads && seen)
                *(f4v *)(A.scores + ((size_t)t * A.C.n_kv * A.G + h * A.G + h0 + i) * A.C.cap + p0 + 4 * g) = *(f4v *)sc;
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
                for (int a = 0; a < NA; a++) {
                    const uint32_t pair = a < 8 * NB ? T.v[a / 8][r][a % 8 / 2] : T.u[r][a % 4 / 2];
                    const float v = value_of<BF>(pair, a & 1);
                    acc[a] = HG == 4 ? __builtin_amdgcn_mfma_f32_4x4x1f32(v, w, acc[a], 0, 0, 0)
                                     : __builtin_amdgcn_mfma_f32_16x16x4f32(v, w, acc[a], 0, 0, 0);
                }
            }
            load_values<W, FULL>(T, tile_at(A.C.v, after, pages[2]), O, hd);
            p0 += PA_UNIT;
#pragma unroll
            for (int x = 0; x < 3; x++) pages[x] = pages[x + 1];
            pages[3] = page_of(p0 + 3 * PA_UNIT);
        };
        while (p0 + PA_UNIT < stop) {
            step(one);
            step(two);
        }
        if (p0 < stop) step(one);

        // the waves' sums at one maximum, added
        l = sum_of_groups(l);
        if (lane < HG) {
            wm[wave][i % HG] = m;
            wl[wave][i % HG] = l;
        }
        __syncthreads();
        float mx = wm[0][col];
#pragma unroll
        for (int w = 1; w < PA_WAVES; w++) mx = fmaxf(mx, wm[w][col]);
        // (a wave that saw nothing has no sums, but a NaN among them must not hide)
        const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
        if (col < heads) {
            float *to = sums + ((size_t)(HG == 4 ? wave * 4 + g : wave) * A.per + col) * hd;
#pragma unroll
            for (int b = 0; b < NA / 4; b++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    // a lane's rows of the product: 4 (i / 4) + r of its block, or 4 g + r
                    const uint32_t row = HG == 4 ? (i & 12) + r : 4 * g + r;
                    const uint32_t d = b < 2 * NB ? b / 2 * 128 + 8 * row + b % 2 * 4 : NB * 128 + 4 * row;
                    if (FULL || d < hd)
                        *(f4v *)(to + d) = f4v{acc[4 * b][r], acc[4 * b + 1][r], acc[4 * b + 2][r], acc[4 * b + 3][r]} * f;
                }
        }
        __syncthreads();
        const bool whole = k0 == 0 && k1 == units;
        const size_t slot = (size_t)(A.whole ? 0 : blockIdx.x) + (size_t)t * items + item;
        for (uint32_t x = tid; x < heads * hd; x += PA_THREADS) {
            const uint32_t j = x / hd, d = x - j * hd;
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < PARTS; w++) y += sums[(size_t)w * A.per * hd + x];
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
        if (A.whole) return;
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
    PagedWork D;
    if (!A.whole) D = divide(A, (uint64_t *)lds);
    const uint32_t t = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const uint32_t n = row_length(A, t), p0 = blockIdx.x * PA_CHUNK;
    if (p0 >= n) return;
    float sum[PA_CHUNK / PA_THREADS] = {};
    for (uint32_t j = 0; j < A.G; j++) {
        const uint32_t item = h * A.tiles + j / A.per;
        uint32_t first = 0, last = 0;
        if (!A.whole) D.runs(t, item, first, last);
        float top, all;
        all_parts(A.stats + (((size_t)t * A.C.n_kv * A.tiles + item) * A.per + j % A.per) * 2, A.per * 2, first, last, top, all);
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

template <bool BF, int HG>
static const void *attn_kernel(size_t hd)
{
#define FOX_ATTN(w) (hd == w ? (const void *)paged_attn_k<BF, w, true, HG> : (const void *)paged_attn_k<BF, w, false, HG>)
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
    const bool four = A.per <= 4;
    // Short caches: a workgroup an item, one launch.
    A.whole = A.C.cap <= 512;
    const size_t most = items * ((A.C.cap + PA_UNIT - 1) / PA_UNIT);
    const size_t fit = (size_t)(four && cache->head_dim <= 128 ? 3 : 2) * ctx->n_cu;
    A.workers = (uint32_t)(A.whole ? items : most < fit ? most : fit);
    // parts, their maxima and sums, and the scores of rows that are weighed
    const size_t slots = A.whole ? items : items + A.workers;
    const size_t part = A.whole ? 0 : slots * A.per * cache->head_dim, stats = slots * A.per * 2;
    const size_t scores = weigh ? M * n_head * A.C.cap : 0;
    if (scores > (size_t)1 << 34)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: the weights of %zu tokens' %zu heads over %u rows are too "
                        "many", M, n_head, A.C.cap);
    if ((st = fox_ws_reserve(ctx, (scores + part + stats) * sizeof(float)))) return st;
    A.scores = weigh ? (float *)ctx->ws : nullptr;
    A.part = (float *)ctx->ws + scores;
    A.stats = A.part + part;
    FOX_HIP(hipSetDevice(ctx->device));
    const bool bf = cache->type == FOX_GPU_BF16;
    const void *k = four ? bf ? attn_kernel<true, 4>(cache->head_dim) : attn_kernel<false, 4>(cache->head_dim)
                         : bf ? attn_kernel<true, 16>(cache->head_dim) : attn_kernel<false, 16>(cache->head_dim);
    const size_t starts = M > 64 && !A.whole ? ((M + 1) * 8 + 15) / 16 * 16 : 0;
    const size_t lds = starts + (size_t)(four ? 4 : 1) * PA_WAVES * A.per * cache->head_dim * sizeof(float);
    void *args[] = {&A};
    FOX_HIP(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    FOX_HIP(hipLaunchKernel(k, dim3(A.workers), dim3(PA_THREADS), args, lds, ctx->stream));
    if (!A.whole && A.workers > 1)
        FOX_HIP(hipLaunchKernel((const void *)paged_merge_k, dim3((unsigned)n_head, (unsigned)M), dim3(PA_THREADS),
                                args, starts, ctx->stream));
    if (weigh)
        FOX_HIP(hipLaunchKernel((const void *)paged_weigh_k,
                                dim3((A.C.cap + PA_CHUNK - 1) / PA_CHUNK, (unsigned)cache->n_head_kv, (unsigned)M),
                                dim3(PA_THREADS), args, starts, ctx->stream));
    return FOX_GPU_OK;
}
