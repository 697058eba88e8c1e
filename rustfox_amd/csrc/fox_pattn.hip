// fox_pattn.hip -- attention of one token a row over a paged cache, on the
// matrix cores.
//
// Arithmetic.  A tile is 16 positions of one kv head, by the (up to 16) query heads that
// share it:
//   S[pos][head] = sum_d K[pos][d] q[head][d]          16x16x32 products of 16 bits
//   O[dim][head] += sum_pos V[pos][dim] P[pos][head]   16x16x4 or 4x4x1 products of 32 bits
// The cache's values are multiplied as they are.  A query is the sum of two halves (its head's row
// first brought to 2^14 .. 2^15 by a power of two) or of three bfloat16 (exact), each
// its own product into the same float sums.  Weights stay floats: a 16-bit second
// product would need V by columns, eight positions of a dimension to a lane, where pages hold
// rows; of the 32-bit one, a lane of S holds four positions of one head, which are the
// operands of four products as they stand, and a row of V is read whole by 16 lanes.  Its rate is
// enough: a tile of 128 dimensions and 16 heads takes 1100 clocks of one SIMD's matrix unit, and
// 8 KB at the copy's rate 1600 clocks of a SIMD's share.
// The running maximum only follows scores that pass it by 8 (in powers of two), so
// between updates no lane needs another's.
//
// Division.  A row's heads have ceil(length / 64) units of 64 positions, one tile for
// each wave of a workgroup.  All units of a call, in order of row, head, position, are
// cut into equal runs, one a workgroup (or each head's, where that wastes little), whatever the
// lengths, which only the device knows (short caches, and tokens that share rows and are much
// of a length, are not divided: a workgroup has all of a head); a
// head whose units lie in several runs is merged by a second launch.  (Merged by the last workgroup
// to arrive, one launch less takes four times as long: before it counts itself each must write its
// part past its XCD's cache, and the fence for that empties it.)
//
// Bound by reads: 64 sequences of 8192 rows and fewer, 16 kv heads of 128 (1.64 GB), 266 us, 6.2 TB/s
// (a plain read reaches 6.5); one of 131071, 8 kv heads (537 MB), 86 us; matrix units are
// busy a tenth of the time.  Short calls by their way in and out, straight code
// that each workgroup meets cold: 4097 rows of 8 kv heads (17 MB) 12.8 us, 9 of them the first launch.
#include "fox_paged_dev.h"

#include <cfloat>
#include <cmath>

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // (rows of any alignment)
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));

#define PA_WAVES 4
#define PA_THREADS (64 * PA_WAVES)
#define PA_TILE 16
#define PA_UNIT (PA_TILE * PA_WAVES)
#define PA_ROOM 8.0f             // how far scores may pass the running maximum
#define PA_CHUNK 2048            // positions that a workgroup weighs: four a thread

struct PagedAttnArgs {
    PagedDev C;
    const float *q;
    float *out;
    size_t q_stride, out_stride;
    const uint32_t *length, *seq;
    uint32_t G, M;               // query heads of a kv head; rows
    uint32_t per, tiles;         // query heads of a head tile (the last may have fewer); head tiles of a kv head
    // Workgroups that share the units: one a compute unit; two where a call is long or has many items. (A
    // unit's rows arrive no faster for two, and each item has more parts; more than 48 units each
    // hide what rows' ends cost: attn-27b-64 283 / 273.)
    uint32_t few, workers;
    bool whole;                  // no: a workgroup an item
    bool either;                 // the device decides that: workgroups for both are launched
    float score;                 // log2(e) / sqrt(hd)
    // Parts: sums [part][per][hd], maxima and weights' sums [part][per][2].  A worker has two at most:
    // of the item that its run begins in (2 worker) and of the one that it ends in (2 worker + 1).
    // Behind them, where rows are weighed, the maxima and sums of whole items.
    float *part, *stats;
    float *scores;               // [row][head][cap], where rows are weighed
    uint32_t *bounds;            // of every item its first and its last worker
};

// ---------------------------------------------------------------- division

// A word that no kernel of the call writes, at an address that is the same for the wave: through the
// scalar cache.  (As vector loads, page numbers would be waited for behind the rows' loads.)
typedef const __attribute__((address_space(4))) uint32_t *Words;
__device__ __forceinline__ uint32_t word(const uint32_t *p, size_t i) { return ((Words)(uintptr_t)p)[i]; }

__device__ __forceinline__ uint32_t units_of(uint32_t n) { return (n + PA_UNIT - 1) / PA_UNIT; }

// a / b; most calls' units are below 2^32, where a quotient takes 20 instructions, not 150
__device__ __forceinline__ uint64_t over(uint64_t a, uint32_t b)
{
    return a >> 32 ? a / b : (uint32_t)a / b;
}

// Where the pieces of each row begin, counted for one of its heads (an item): up to 64
// rows by every wave for itself, lane t row t, without LDS or a barrier; more by the
// workgroup, in LDS.  A piece is `size` units, or what an item has left: one unit, or all of a worker's
// where every run can end with its item, so that no worker has two ways in and out.
struct PagedWork {
    const uint64_t *start;        // [M + 1], past 64 rows
    uint64_t run, total;          // pieces of a worker; of the call
    uint32_t size;
    uint32_t items, M, before, pieces, length, seq;
    bool whole;                   // no division: a workgroup an item

    // the row that holds piece u of the call
    __device__ __forceinline__ uint32_t row_of(uint64_t u) const
    {
        if (M == 1) return 0;
        if (M <= 64) {
            const uint32_t lane = threadIdx.x & 63;
            return 63 - __builtin_clzll(__ballot(lane < M && (uint64_t)before * items <= u));
        }
        uint32_t lo = 0, hi = M;                            // the last with start items <= u
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (start[mid] * items <= u) lo = mid;
            else hi = mid;
        }
        return __builtin_amdgcn_readfirstlane(lo);
    }
    // a row's first piece of one item, and how many it has
    __device__ __forceinline__ void row(uint32_t t, uint64_t &first, uint32_t &n) const
    {
        if (M <= 64) {
            first = (uint32_t)__builtin_amdgcn_readlane((int)before, t);
            n = (uint32_t)__builtin_amdgcn_readlane((int)pieces, t);
        } else {
            first = start[t];
            n = (uint32_t)(start[t + 1] - first);
        }
    }
};

// rows that row t sees, and its sequence
__device__ __forceinline__ uint32_t row_length(const PagedAttnArgs &A, uint32_t t, uint32_t &s)
{
    s = A.seq ? A.seq[t] : t;
    const uint32_t n = A.length[t];
    return s < A.C.n_seqs ? min(n, A.C.cap) : 0;
}

// Whether a call whose tokens share rows (`alike` of the M are of the sequence of the one before, with rows) takes
// a workgroup an item all the same.  In the items' order a kv head's rows are read by few XCDs' caches, by
// neighbouring tokens at once, which the runs of a division do not; but an item is no faster for what
// else is done, so the longest may take twice an equal share of all units, no more.  Whole / divided, us, 32 heads
// over 8 kv heads of 128: 512 tokens of one sequence at 9000 rows 1222 / 2080, at 2048 276 / 314, 48 at 9000 164 / 222
// (the longest 1.3 shares), 8 of each of 5 sequences of 4000 79 / 103 (1.6); 1000 tokens from the first on 211 / 725;
// 300 over 2 kv heads at 9000 239 / 214.  30 sequences of 1000, one of 100000 and 16 tokens of a
// prompt 1055 / 106 (43 shares).
__host__ __device__ inline bool paged_whole(uint32_t M, uint32_t alike, uint64_t units, uint32_t longest, uint32_t workers)
{
    return 2 * alike >= M && (uint64_t)longest * workers <= 2 * units;
}

// That of more than 64 rows, by the workgroup
__device__ __forceinline__ bool whole_rows(const PagedAttnArgs &A, uint32_t items)
{
    constexpr int EACH = FOX_GPU_BATCH_TOKENS / PA_THREADS;
    static_assert(EACH * PA_THREADS == FOX_GPU_BATCH_TOKENS, "a thread has EACH rows");
    __shared__ uint32_t units[PA_WAVES], longest[PA_WAVES], alike[PA_WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    uint32_t n[EACH], s[EACH], before[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {                         // (asked for together)
        const uint32_t t = min(tid + i * PA_THREADS, A.M - 1);
        n[i] = A.length[t];
        s[i] = A.seq[t];
        before[i] = A.seq[t ? t - 1 : 0];
    }
    uint32_t all = 0, most = 0, same = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t t = tid + i * PA_THREADS;
        const uint32_t u = t < A.M && s[i] < A.C.n_seqs ? units_of(min(n[i], A.C.cap)) : 0;
        all += min(u, (1u << 24) - 1);                       // (a wave's 256 fit: a row has at most 2^24)
        most = max(most, u);
        same += u && t && s[i] == before[i];
    }
    all = wave_scan(all);
    most = wave_max(most);
    same = wave_scan(same);
    if (lane == 63) {
        units[w] = all;
        longest[w] = most;
        alike[w] = same;
    }
    __syncthreads();
    uint64_t total = 0;
    most = same = 0;
    for (int i = 0; i < PA_WAVES; i++) {
        total += (uint64_t)units[i] * items;
        most = max(most, longest[i]);
        same += alike[i];
    }
    return paged_whole(A.M, same, total, most, A.workers);
}

// SEQ: the tokens' sequences may be given
template <bool SEQ>
__device__ __forceinline__ PagedWork divide(const PagedAttnArgs &A, uint64_t *start)
{
    __shared__ uint64_t sums[PA_WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    PagedWork D;
    D.start = start;
    D.M = A.M;
    D.items = A.C.n_kv * A.tiles;
    D.length = D.seq = 0;
    D.size = 1;
    D.whole = false;
    if (A.M == 1) {                                                 // (by the scalar unit)
        D.seq = A.seq ? word(A.seq, 0) : 0;
        const uint32_t n = word(A.length, 0);
        D.length = D.seq < A.C.n_seqs ? min(n, A.C.cap) : 0;
        D.pieces = units_of(D.length);
        D.before = 0;
        D.total = (uint64_t)D.pieces * D.items;
    } else if (A.M <= 64) {
        if (lane < A.M) D.length = row_length(A, lane, D.seq);
        D.pieces = units_of(D.length);                              // (64 of at most 2^24)
        const uint32_t x = wave_scan(D.pieces);
        D.before = x - D.pieces;
        D.total = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, (int)A.M - 1) * D.items;
        if (SEQ && A.either) {
            const uint32_t ahead = __shfl_up(D.seq, 1);
            const uint32_t alike = __popcll(__ballot(lane > 0 && D.pieces && D.seq == ahead));
            D.whole = paged_whole(A.M, alike, D.total, wave_max(D.pieces), A.workers);
            if (D.whole) return D;
        }
    } else {
        if (SEQ && A.either) {
            D.whole = whole_rows(A, D.items);
            if (D.whole) return D;
        }
        const uint32_t each = (A.M + PA_THREADS - 1) / PA_THREADS;  // (at most 4)
        uint64_t mine = 0;
        uint32_t s;
        for (uint32_t i = 0; i < each; i++) {
            const uint32_t t = tid * each + i;
            if (t < A.M) mine += units_of(row_length(A, t, s));
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
            before += units_of(row_length(A, t, s));
        }
        if (tid == PA_THREADS - 1) start[A.M] = before;
        __syncthreads();
        D.total = start[A.M] * D.items;
    }
    // (more items than workers take twice the workers: 24 rows of 150 to 3000, 16 kv heads, 61 / 54.6 us)
    uint32_t workers = D.total < (uint64_t)48 * A.workers && A.M * D.items <= A.few ? A.few : A.workers;
    D.run = over(D.total + workers - 1, workers);
    // Runs that end with their items, where runs a fifth or three units longer leave workers enough for them; if
    // not, with twice the workers: attn-8b-1 15.2 / 12.8 us, 16 rows of 150 to 3000 28.6 / 22.2,
    // 32 of 125 to 2500 50.3 / 34.1.  (Twice the workers without that: 32 rows of 4000 82.8 / 85.4.)
    if (A.M == 1) {
        const uint32_t units = D.pieces, run = (uint32_t)D.run, most = workers / D.items;
        if (run > 1 && most) {
            const uint32_t size = (units + most - 1) / most;
            if (size <= run + 3 * (1 + run / 16)) {
                D.size = size;
                D.pieces = (units + size - 1) / size;
                D.total = D.pieces * D.items;
                D.run = 1;
            }
        }
    } else if (A.M <= 64 && D.run > 1 && A.M * D.items <= workers) {
        const uint32_t units = D.pieces;
        for (;; workers = A.workers) {
            const uint32_t run = (uint32_t)over(D.total + workers - 1, workers), step = 1 + run / 16;
            // four sizes at once, two sums a word (64 of at most 1023; workers are fewer)
            uint32_t x[2], y[2], all = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t size = run + k * step, n = min((units + size - 1) / size, 1023u);
                if (k & 1) y[k / 2] |= n << 16;
                else y[k / 2] = n;
            }
#pragma unroll
            for (int k = 0; k < 2; k++) x[k] = wave_scan(y[k]);
#pragma unroll
            for (int k = 3; k >= 0; k--) {
                const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)x[k / 2], (int)A.M - 1) >> k % 2 * 16 & 0xFFFFu;
                if (at * D.items <= workers) {
                    D.size = run + k * step;
                    D.pieces = y[k / 2] >> k % 2 * 16 & 0xFFFFu;
                    D.before = (x[k / 2] - y[k / 2]) >> k % 2 * 16 & 0xFFFFu;
                    all = at;
                }
            }
            if (all) {
                D.total = all * D.items;
                D.run = 1;
                return D;
            }
            if (workers == A.workers) break;
        }
    }
    return D;
}

// ------------------------------------------------------------------- tiles

// the parts of eight query values: two halves of x 2^e, or three bfloat16
template <bool BF>
__device__ __forceinline__ void split_q(uint4 part[BF ? 3 : 2], const f4v x[2], int e)
{
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {                        // two values a word
        const float a = x[i / 2][i % 2 * 2], b = x[i / 2][i % 2 * 2 + 1];
        if (BF) {                                        // (truncated: what is left is exact)
            uint32_t u = __float_as_uint(a), v = __float_as_uint(b);
#pragma unroll
            for (int k = 0; k < 3; k++) {
                w[k][i] = __builtin_amdgcn_perm(v, u, 0x07060302);
                u = __float_as_uint(__uint_as_float(u) - __uint_as_float(u & 0xFFFF0000u));
                v = __float_as_uint(__uint_as_float(v) - __uint_as_float(v & 0xFFFF0000u));
            }
        } else {
            const f2v y = {ldexpf(a, e), ldexpf(b, e)};
            const h2v hi = __builtin_convertvector(y, h2v);
            const h2v lo = __builtin_convertvector(y - __builtin_convertvector(hi, f2v), h2v);
            w[0][i] = __builtin_bit_cast(uint32_t, hi);
            w[1][i] = __builtin_bit_cast(uint32_t, lo);
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

// ONCE: every row is read by one workgroup of the call (a token of each sequence, one tile of heads), so it need
// not stay in the caches (the instruction's nt bit): attn-27b-64 298 -> 277 us, attn-4b-1-long 101 -> 90.
// Of 512 tokens of one sequence, which share its rows, 360 -> 546.
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

template <int W, bool FULL, bool ONCE>
__device__ __forceinline__ void load_keys(Tile<W> &T, __amdgpu_buffer_rsrc_t at, const Offsets<W, FULL> &O)
{
    const uint32_t k = here(O.k[0]);
#pragma unroll
    for (int c = 0; c < W / 32; c++)
        T.k[c] = __builtin_amdgcn_raw_buffer_load_b128(at, FULL ? k + 64 * c : O.k[FULL ? 0 : c], 0, ONCE ? 2 : 0);
}

template <int W, bool FULL, bool ONCE>
__device__ __forceinline__ void load_values(Tile<W> &T, __amdgpu_buffer_rsrc_t at, const Offsets<W, FULL> &O, uint32_t hd)
{
    const uint32_t row = FULL ? W * 2 : hd * 2;
#pragma unroll
    for (int b = 0; b < W / 128; b++) {
        const uint32_t v = here(O.v[FULL ? 0 : b]) + (FULL ? 256 * b : 0);
#pragma unroll
        for (int r = 0; r < 4; r++) T.v[b][r] = __builtin_amdgcn_raw_buffer_load_b128(at, v + r * row, 0, ONCE ? 2 : 0);
    }
    if (W % 128) {
        const uint32_t u = here(O.u);
#pragma unroll
        for (int r = 0; r < 4; r++) T.u[r] = __builtin_amdgcn_raw_buffer_load_b64(at, u + r * row, 0, ONCE ? 2 : 0);
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
template <bool BF, int W, bool FULL, int HG, bool ONCE>
__global__ __launch_bounds__(PA_THREADS, 2) void paged_attn_k(const uint32_t *length0, const uint32_t *seq0, uint32_t M0,
                                                             uint32_t n_seqs0, uint32_t cap0, PagedAttnArgs A)
{
    // (what the first reads need comes in registers: the rest is read beside them)
    A.length = length0;
    A.seq = seq0;
    A.M = M0;
    A.C.n_seqs = n_seqs0;
    A.C.cap = cap0;
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
    bool whole_item = A.whole;                              // (a workgroup's item is its number)
    if (!A.whole) {
        D = divide<!ONCE>(A, (uint64_t *)lds);
        if (!ONCE) whole_item = D.whole;
    }
    if (!ONCE && whole_item && blockIdx.x >= A.M * items) return;
    if (!whole_item) {
        for (uint32_t t = blockIdx.x; t < A.M; t += gridDim.x) {
            uint64_t first;
            uint32_t n;
            D.row(t, first, n);
            if (n == 0) {
                for (uint32_t d = tid; d < width; d += PA_THREADS) A.out[t * A.out_stride + d] = 0.0f;
                for (uint32_t i = tid; i < 2 * items; i += PA_THREADS) A.bounds[(size_t)t * items * 2 + i] = 0;
            }
        }
        u = blockIdx.x * D.run;
        end = min(u + D.run, D.total);
    }
    while (u < end) {                                       // (uniform)
        uint32_t t, item, k0 = 0, k1 = 0, part = 0, parts = 1;
        if (whole_item) {
            t = blockIdx.x / items;
            item = blockIdx.x - t * items;
        } else {
            uint64_t first;
            t = D.row_of(u);
            D.row(t, first, parts);
            const uint64_t in_row = u - first * items;
            item = (uint32_t)over(in_row, parts);
            part = (uint32_t)(in_row - (uint64_t)item * parts);
            parts = (uint32_t)min((uint64_t)parts - part, end - u);
        }
        t = __builtin_amdgcn_readfirstlane(t);
        item = __builtin_amdgcn_readfirstlane(item);
        const uint32_t h = A.tiles == 1 ? item : item / A.tiles, h0 = (item - h * A.tiles) * A.per;
        const uint32_t heads = min(A.per, A.G - h0);
        uint32_t n, s;
        if (!A.whole && A.M <= 64) {                        // (divided or not)
            n = (uint32_t)__builtin_amdgcn_readlane((int)D.length, t);
            s = (uint32_t)__builtin_amdgcn_readlane((int)D.seq, t);
        } else {
            s = A.seq ? word(A.seq, t) : t;
            const uint32_t length = word(A.length, t);
            n = s < A.C.n_seqs ? min(length, A.C.cap) : 0;
        }
        if (n == 0) s = 0;                                  // (a sequence that is none has no table)
        const uint32_t units = units_of(n);
        if (whole_item) {
            k1 = units;
        } else {
            k0 = part * D.size;
            k1 = min(units, k0 + parts * D.size);
        }
        k0 = __builtin_amdgcn_readfirstlane(k0);
        k1 = __builtin_amdgcn_readfirstlane(k1);
        const uint32_t *table = A.C.table + (size_t)s * A.C.max_pages;

        // the queries' rows and the first tile are asked for together
        // (heads past the tile's read as zeros behind its end, and so do dimensions past the row's)
        f4v x[NC][2];
        {
            const __amdgpu_buffer_rsrc_t at = __builtin_amdgcn_make_buffer_rsrc(
                (float *)A.q + t * A.q_stride + (size_t)(h * A.G + h0) * hd, 0, heads * hd * 4, 0x00027000);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const uint32_t d = 32 * c + 8 * g, o = FULL || d < hd ? (col * hd + d) * 4 : PA_NOWHERE;
#pragma unroll
                for (int k = 0; k < 2; k++)
                    x[c][k] = __builtin_bit_cast(f4v, __builtin_amdgcn_raw_buffer_load_b128(at, o + 16 * k, 0, 0));
            }
        }
        // Tiles of this wave: p0, p0 + PA_UNIT, ...; two are held, and as soon as one's keys
        // (values) are used, those of the tile after the next are asked for in their place.
        const Offsets<W, FULL> O(hd);
        Tile<W> one, two;
        const uint32_t in_page = (1u << A.C.shift) - 1, stop = min(n, k1 * PA_UNIT);
        uint32_t p0 = k0 * PA_UNIT + wave * PA_TILE;
        // (no branches, so that loads are asked for together: places behind the run give some page of the
        // sequence and no rows, and an address that is none is not used)
        auto page_of = [&](uint32_t p) -> uint32_t { return word(table, min(p, A.C.cap - 1) >> A.C.shift); };
        auto rows_of = [&](uint32_t p, uint32_t page) -> uint32_t {   // that are seen
            return p < stop && page < A.C.n_pages ? min(n - p, (uint32_t)PA_TILE) : 0;
        };
        auto tile_at = [&](const void *pool, uint32_t p, uint32_t page) -> __amdgpu_buffer_rsrc_t {
            const uint32_t rows = rows_of(p, page);
            const size_t at = ((((size_t)page * A.C.n_kv + h) << A.C.shift) + (p & in_page)) * hd;
            return __builtin_amdgcn_make_buffer_rsrc((uint16_t *)pool + at, 0, rows * hd * 2, 0x00027000);
        };
        uint32_t pages[4];       // of this tile and the three after it
#pragma unroll
        for (int x = 0; x < 4; x++) pages[x] = page_of(p0 + x * PA_UNIT);
        load_keys<W, FULL, ONCE>(one, tile_at(A.C.k, p0, pages[0]), O);
        load_values<W, FULL, ONCE>(one, tile_at(A.C.v, p0, pages[0]), O, hd);
        load_keys<W, FULL, ONCE>(two, tile_at(A.C.k, p0 + PA_UNIT, pages[1]), O);
        load_values<W, FULL, ONCE>(two, tile_at(A.C.v, p0 + PA_UNIT, pages[1]), O, hd);

        uint4 q[QLDS ? 1 : NC][NP];
        float factor;
        {
            float top = 0.0f;
            int e = 0;
            if (!BF) {
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[c][j / 4][j % 4]));
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
            load_keys<W, FULL, ONCE>(T, tile_at(A.C.k, after, pages[2]), O);
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
            load_values<W, FULL, ONCE>(T, tile_at(A.C.v, after, pages[2]), O, hd);
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

        // the waves' sums, each at its maximum, then added at the greatest
        l = sum_of_groups(l);
        if (lane < HG) {
            wm[wave][i % HG] = m;
            wl[wave][i % HG] = l;
        }
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
                        *(f4v *)(to + d) = f4v{acc[4 * b][r], acc[4 * b + 1][r], acc[4 * b + 2][r], acc[4 * b + 3][r]};
                }
        }
        __syncthreads();
        const bool whole = k0 == 0 && k1 == units;
        const size_t at = (size_t)t * items + item;
        const size_t slot = !whole ? 2 * (size_t)blockIdx.x + (k0 == 0) : (A.whole ? 0 : 2 * (size_t)A.workers) + at;
        if (tid == 0 && !A.whole) {
            if (k0 == 0) A.bounds[2 * at] = blockIdx.x;
            if (k1 == units) A.bounds[2 * at + 1] = blockIdx.x;
        }
        for (uint32_t x = tid * 4; x < heads * hd; x += PA_THREADS * 4) {
            const uint32_t j = x / hd, d = x - j * hd;
            float top = wm[0][j], all = 0.0f;
#pragma unroll
            for (int w = 1; w < PA_WAVES; w++) top = fmaxf(top, wm[w][j]);
            f4v y = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < PA_WAVES; w++) {
                // (a wave that saw nothing has no sums, but a NaN among them must not hide)
                const float f = wm[w][j] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(wm[w][j] - top);
                f4v part = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < PARTS / PA_WAVES; k++)
                    part += *(const f4v *)(sums + (size_t)(w * (PARTS / PA_WAVES) + k) * A.per * hd + x);
                y += part * f;
                all += wl[w][j] * f;
            }
            if (whole) {
                float *to = A.out + t * A.out_stride + (size_t)(h * A.G + h0 + j) * hd + d;
                if (all == 0.0f) y = f4v{0, 0, 0, 0};
                else y /= all;
                *(f4u *)to = y;
            } else {
                *(f4v *)(A.part + (slot * A.per + j) * hd + d) = y;
            }
            if (d == 0 && (!whole || A.scores)) *(float2 *)(A.stats + (slot * A.per + j) * 2) = float2{top, all};
        }
        if (A.whole) {
            if (!A.scores || A.tiles > 1) return;
            // the rows' weights, from the scores that this workgroup has stored, summed in the heads' order
            // before they are added to what the row has
            __shared__ float tops[HG], by[HG];
            if (tid < heads) {
                float top = wm[0][tid], all = 0.0f;
#pragma unroll
                for (int w = 1; w < PA_WAVES; w++) top = fmaxf(top, wm[w][tid]);
#pragma unroll
                for (int w = 0; w < PA_WAVES; w++)
                    all += wm[w][tid] == -INFINITY ? wl[w][tid] : wl[w][tid] * __builtin_amdgcn_exp2f(wm[w][tid] - top);
                tops[tid] = top == -INFINITY ? 0.0f : top;
                by[tid] = all == 0.0f ? 0.0f : 1.0f / all;
            }
            __syncthreads();
            float *weight = A.C.weight + ((size_t)t * A.C.n_kv + h) * A.C.cap;
            const float *scores = A.scores + ((size_t)t * A.C.n_kv + h) * A.G * A.C.cap;
            for (uint32_t p = tid; p < n; p += PA_THREADS) {
                if (table[p >> A.C.shift] >= A.C.n_pages) continue;
                float sum = 0.0f;
                for (uint32_t j = 0; j < heads; j++)
                    sum += __builtin_amdgcn_exp2f(scores[(size_t)j * A.C.cap + p] - tops[j]) * by[j];
                weight[p] += sum;
            }
            return;
        }
        __syncthreads();
        u += parts;                                         // (one, of a whole item)
    }
}

// ------------------------------------------------------------------- merge

#define PM_THREADS 512
#define PM_DEEP 4                // parts that a thread has on the way

// A workgroup a query head: its parts at one maximum, added.  32 lanes (64 past 128 dimensions)
// take every 16th (8th) part, four dimensions a lane, each at the maximum met so far; then
// those sums are added.  Everything a part has is asked for at once: one wait for 64 parts.
__device__ __forceinline__ void merge_head(const PagedAttnArgs &A, uint32_t t, uint32_t head, float *sums, float *tops,
                                           float *alls)
{
    const uint32_t h = head / A.G, j = head - h * A.G, tid = threadIdx.x;
    const uint32_t tile = A.tiles == 1 ? 0 : j / A.per, in_tile = j - tile * A.per;
    const uint32_t hd = A.C.hd, lanes = hd <= 128 ? 32 : 64, groups = PM_THREADS / lanes, group = tid / lanes;
    const uint32_t d = tid % lanes * 4;
    const size_t item = (size_t)t * A.C.n_kv * A.tiles + h * A.tiles + tile;
    const uint32_t first = word(A.bounds, 2 * item), last = word(A.bounds, 2 * item + 1);
    if (first == last) return;
    const float *stats = A.stats + in_tile * 2;
    const float *part = A.part + in_tile * (size_t)hd + (d < hd ? d : 0);
    float top = -INFINITY, all = 0.0f;
    f4v y = {0, 0, 0, 0};
    for (uint32_t w = first + group; w <= last; w += PM_DEEP * groups) {
        float m[PM_DEEP], l[PM_DEEP], mx = top;
        f4v x[PM_DEEP];
#pragma unroll
        for (int k = 0; k < PM_DEEP; k++) {
            const uint32_t worker = min(w + k * groups, last), at = 2 * worker + (worker == first);
            m[k] = stats[(size_t)at * A.per * 2];
            l[k] = stats[(size_t)at * A.per * 2 + 1];
            x[k] = *(const f4v *)(part + (size_t)at * A.per * hd);
        }
#pragma unroll
        for (int k = 0; k < PM_DEEP; k++)
            if (w + k * groups <= last) mx = fmaxf(mx, m[k]);
        if (top != -INFINITY) {
            const float f = __builtin_amdgcn_exp2f(top - mx);
            all *= f;
            y *= f;
        }
#pragma unroll
        for (int k = 0; k < PM_DEEP; k++)
            if (w + k * groups <= last) {
                const float f = m[k] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[k] - mx);
                all += l[k] * f;
                y += x[k] * f;
            }
        top = mx;
    }
    if (d < hd) *(f4v *)(sums + group * lanes * 4 + d) = y;
    if (d == 0) {
        tops[group] = top;
        alls[group] = all;
    }
    __syncthreads();
    if (tid >= hd) return;
    float mx = tops[0], out = 0.0f, sum = 0.0f;
    for (uint32_t g = 1; g < groups; g++) mx = fmaxf(mx, tops[g]);
    for (uint32_t g = 0; g < groups; g++) {
        const float f = tops[g] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(tops[g] - mx);
        sum += alls[g] * f;
        out += sums[g * lanes * 4 + tid] * f;
    }
    A.out[t * A.out_stride + (size_t)head * hd + tid] = sum == 0.0f ? 0.0f : out / sum;
}

// A workgroup a kv head's PA_CHUNK positions, four a thread: the group's weights of each, from the scores,
// summed in the heads' order before they are added to what the row has.  Eight heads at a time: a wave
// adds up one head's parts while every thread has its eight scores on the way.
__device__ __forceinline__ void weigh_chunk(const PagedAttnArgs &A, uint32_t t, uint32_t h, uint32_t chunk, float *tops,
                                            float *by)
{
    constexpr int WAVES = PM_THREADS / 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = min(word(A.length, t), A.C.cap), p = chunk * PA_CHUNK + tid * 4;
    if (chunk * PA_CHUNK >= n) return;
    const bool on = p < n && A.C.table[(size_t)t * A.C.max_pages + (p >> A.C.shift)] < A.C.n_pages;
    float *weight = A.C.weight + ((size_t)t * A.C.n_kv + h) * A.C.cap + p;
    const float *scores = A.scores + ((size_t)t * A.C.n_kv + h) * A.G * A.C.cap + p;
    f4v sum = {0, 0, 0, 0}, had = sum, sc[WAVES];
    if (on) had = *(const f4v *)weight;
    for (uint32_t j0 = 0; j0 < A.G; j0 += WAVES) {
#pragma unroll
        for (int k = 0; k < WAVES; k++)
            if (on && j0 + k < A.G) sc[k] = *(const f4v *)(scores + (size_t)(j0 + k) * A.C.cap);
        const uint32_t j = j0 + wave;
        if (j < A.G) {
            const size_t item = (size_t)t * A.C.n_kv * A.tiles + h * A.tiles + j / A.per;
            const uint32_t first = A.whole ? 0 : word(A.bounds, 2 * item), last = A.whole ? 0 : word(A.bounds, 2 * item + 1);
            const float *stats = A.stats + j % A.per * 2;
            float top = -INFINITY, all = 0.0f;
            for (uint32_t w = first + lane; w <= last; w += 64) {
                const size_t at = first != last ? 2 * (size_t)w + (w == first) : (A.whole ? 0 : 2 * (size_t)A.workers) + item;
                const float2 ml = *(const float2 *)(stats + at * A.per * 2);
                const float mx = fmaxf(top, ml.x);
                all = (top == -INFINITY ? all : all * __builtin_amdgcn_exp2f(top - mx)) +
                      (ml.x == -INFINITY ? ml.y : ml.y * __builtin_amdgcn_exp2f(ml.x - mx));
                top = mx;
            }
            const float mx = wave_max(top);
            all = wave_sum(top == -INFINITY ? all : all * __builtin_amdgcn_exp2f(top - mx));
            if (lane == 0) {
                tops[wave] = mx;
                by[wave] = all == 0.0f ? 0.0f : 1.0f / all;
            }
        }
        __syncthreads();
        if (on)
#pragma unroll
            for (int k = 0; k < WAVES; k++)
                if (j0 + k < A.G) {
                    const float top = tops[k] == -INFINITY ? 0.0f : tops[k];
#pragma unroll
                    for (int r = 0; r < 4; r++) sum[r] += __builtin_amdgcn_exp2f(sc[k][r] - top) * by[k];
                }
        __syncthreads();
    }
    if (!on) return;
    if (p + 4 <= n) {
        *(f4v *)weight = had + sum;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (p + r < n) weight[r] = had[r] + sum[r];
    }
}

// What follows the attention, in one launch: merges of the row's heads, and its kv heads' chunks weighed.
__global__ __launch_bounds__(PM_THREADS) void paged_after_k(const uint32_t *bounds0, uint32_t merges, uint32_t chunks, uint32_t n_kv0,
                                                            uint32_t G0, uint32_t tiles0, uint32_t per0, uint32_t group, PagedAttnArgs A)
{
    A.bounds = (uint32_t *)bounds0;                          // (in registers from the start, as above)
    A.C.n_kv = n_kv0;
    A.G = G0;
    A.tiles = tiles0;
    A.per = per0;
    __shared__ __attribute__((aligned(16))) float sums[16 * 128], tops[16], alls[16];
    const uint32_t t = blockIdx.y;
    if (blockIdx.x < merges) {
        if (group == 1) return merge_head(A, t, blockIdx.x, sums, tops, alls);
        // those of the group that have parts, found by a lane each
        const uint32_t lane = threadIdx.x & 63, mine = blockIdx.x * group + lane;
        uint2 b = {0, 0};
        if (lane < group && mine < n_kv0 * G0) {
            const uint32_t tile = mine / G0 * tiles0 + mine % G0 / per0;
            b = *(const uint2 *)(bounds0 + 2 * ((size_t)t * n_kv0 * tiles0 + tile));
        }
        for (uint64_t left = __ballot(b.x != b.y); left; left &= left - 1) {
            merge_head(A, t, blockIdx.x * group + (uint32_t)__ffsll((unsigned long long)left) - 1, sums, tops, alls);
            __syncthreads();
        }
    } else {
        const uint32_t x = blockIdx.x - merges;
        weigh_chunk(A, t, x / chunks, x % chunks, tops, alls);
    }
}

template <bool BF, int HG, bool ONCE>
static const void *attn_kernel(size_t hd)
{
#define FOX_ATTN(w) (hd == w ? (const void *)paged_attn_k<BF, w, true, HG, ONCE> : (const void *)paged_attn_k<BF, w, false, HG, ONCE>)
    return hd <= 64 ? FOX_ATTN(64) : hd <= 128 ? FOX_ATTN(128)
         : hd <= 192 ? (const void *)paged_attn_k<BF, 192, false, HG, ONCE> : FOX_ATTN(256);
#undef FOX_ATTN
}

PagedPlan fox_paged_plan(size_t n_head, size_t n_head_kv, size_t M, size_t cap, bool seq, int n_cu)
{
    PagedPlan p = {};
    const size_t G = n_head / n_head_kv;
    p.tiles = (uint32_t)((G + 15) / 16);
    p.per = (uint32_t)((G + p.tiles - 1) / p.tiles);
    p.items = M * n_head_kv * p.tiles;
    // Short caches: a workgroup an item, one launch.  How short depends on the items, since one alone
    // draws rows at 55 GB/s (0.6 us for 64 of them), and many fill the compute units anyway.  Whole / divided, us, all
    // as long as the cache (and of 1/20 of it to all): 8 items of 300 rows 8.9 / 10.3, of 600 13.1 / 10.4; 128 of 300
    // 9.8 / 13.1, of 600 14.4 / 15.6 (13.5 / 13.0), of 1000 20.2 / 19.0 (18.8 / 14.0); 192 of 800 18.2 / 21.2
    // (16.3 / 16.6); 256 of 2000 42.3 / 45.4 (33.8 / 29.7); 512 of 2500 100 / 104 (66 / 71),
    // of 4000 157 / 161 (102 / 84).  Calls of many items whose tokens may share rows are decided on the device.
    const double full = (double)p.items / n_cu;
    p.whole = cap <= (full < 1.0 ? 400.0 + 1648.0 * full * full * full : 1536.0 + 512.0 * (full < 4.0 ? full : 4.0));
    p.either = !p.whole && seq && M > 1 && full >= 1.0;
    const size_t most = p.items * ((cap + PA_UNIT - 1) / PA_UNIT), fit = (size_t)2 * n_cu;
    p.workers = (uint32_t)(p.whole ? p.items : most < fit ? most : fit);
    p.few = p.workers < (uint32_t)n_cu ? p.workers : (uint32_t)n_cu;
    return p;
}

bool fox_paged_plan_whole(const PagedPlan &p, size_t M, size_t cap, size_t n_seqs, const uint32_t *length, const uint32_t *seq)
{
    if (!p.either) return p.whole;
    uint64_t units = 0;
    uint32_t longest = 0, alike = 0;
    for (size_t t = 0; t < M; t++) {
        const uint32_t n = seq[t] < n_seqs ? ((length[t] < cap ? length[t] : (uint32_t)cap) + PA_UNIT - 1) / PA_UNIT : 0;
        units += n;
        if (n > longest) longest = n;
        if (n && t && seq[t] == seq[t - 1]) alike++;
    }
    return paged_whole((uint32_t)M, alike, units * (p.items / M), longest, p.workers);
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
    if (fox_rows_overlap(out, out_stride, width, q, q_stride, width, M))
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: out overlaps q");
    A.q = q;
    A.out = out;
    A.q_stride = q_stride;
    A.out_stride = out_stride;
    A.length = length;
    A.seq = seq;
    const PagedPlan p = fox_paged_plan(n_head, cache->n_head_kv, M, A.C.cap, seq != nullptr, ctx->n_cu);
    A.G = (uint32_t)(n_head / cache->n_head_kv);
    A.M = (uint32_t)M;
    A.tiles = p.tiles;
    A.per = p.per;
    A.score = (float)(1.4426950408889634 / std::sqrt((double)cache->head_dim));
    A.whole = p.whole;
    A.either = p.either;
    A.workers = p.workers;
    A.few = p.few;
    const size_t items = p.items;
    const bool four = A.per <= 4;
    // parts, their maxima and sums, and the scores of rows that are weighed
    const size_t parts = A.whole ? 0 : 2 * (size_t)A.workers;
    const size_t part = parts * A.per * cache->head_dim, stats = (parts + (weigh ? items : 0)) * A.per * 2;
    const size_t scores = weigh ? M * n_head * A.C.cap : 0;
    if (scores > (size_t)1 << 33)
        return fox_fail(FOX_GPU_ERR_ARG, "paged_attention: the weights of %zu tokens' %zu heads over %u rows are too "
                        "many", M, n_head, A.C.cap);
    const size_t bounds = A.whole ? 0 : 2 * items;
    FOX_HIP(hipSetDevice(ctx->device));
    if ((st = fox_ws_reserve(ctx, (scores + part + stats + bounds) * sizeof(float)))) return st;
    A.scores = weigh ? (float *)ctx->ws : nullptr;
    A.part = (float *)ctx->ws + scores;
    A.stats = A.part + part;
    A.bounds = (uint32_t *)(A.stats + stats);
    const bool bf = cache->type == FOX_GPU_BF16;
    const bool once = !seq && A.tiles == 1;
#define FOX_ATTN(hg, o) (bf ? attn_kernel<true, hg, o>(cache->head_dim) : attn_kernel<false, hg, o>(cache->head_dim))
    const void *k = four ? once ? FOX_ATTN(4, true) : FOX_ATTN(4, false) : once ? FOX_ATTN(16, true) : FOX_ATTN(16, false);
#undef FOX_ATTN
    const size_t starts = M > 64 && !A.whole ? ((M + 1) * 8 + 15) / 16 * 16 : 0;
    const size_t lds = starts + (size_t)(four ? 4 : 1) * PA_WAVES * A.per * cache->head_dim * sizeof(float);
    void *args[] = {&A.length, &A.seq, &A.M, &A.C.n_seqs, &A.C.cap, &A};
    FOX_HIP(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    FOX_HIP(hipLaunchKernel(k, dim3((unsigned)(A.either && items > A.workers ? items : A.workers)), dim3(PA_THREADS), args, lds,
                            ctx->stream));
    // (query heads of a workgroup: many that may have nothing to merge are looked through by fewer; 1000 tokens of 32
    // heads 23 us one by one, 4.7 by eight)
    const uint32_t group = A.either && M > 64 ? 8 : 1;
    const uint32_t merges = A.whole || A.workers == 1 ? 0 : ((uint32_t)n_head + group - 1) / group;
    // (a workgroup that has all of an item and its group adds its weights itself: 2 rows of 11, 8 kv heads,
    // 7.8 us, by another launch 9.5)
    uint32_t chunks = weigh && !(A.whole && A.tiles == 1) ? (A.C.cap + PA_CHUNK - 1) / PA_CHUNK : 0;
    if (merges || chunks) {
        void *after[] = {&A.bounds, (void *)&merges, &chunks, &A.C.n_kv, &A.G, &A.tiles, &A.per, (void *)&group, &A};
        FOX_HIP(hipLaunchKernel((const void *)paged_after_k, dim3((unsigned)(merges + chunks * cache->n_head_kv), (unsigned)M),
                                dim3(PM_THREADS), after, 0, ctx->stream));
    }
    return FOX_GPU_OK;
}
