// fox_kvq_dev.h -- the quantised cache: layout and arithmetic shared by the
// kernels that write it (fox_kvq.hip) and the attention over it
// (fox_kvattn.hip).
//
// Values.  A head's dimensions are taken in groups of 32 (padded up to a
// supported width, fox_kvq_width; padding holds the code of zero).  A group
// has one scale d, an 8-bit unsigned number of 5 exponent and 3 mantissa bits,
// stored as bits 14..7 of the half d * 4, and a code per value,
//   x ~ d * c,  c = round_half_even(x / d) in [-h, h - 1],  h = 2^(BITS - 1),
// where d is the least scale with max(x) <= (h - 1/2) d and
// -min(x) <= (h + 1/2) d, so |x - d c| <= d / 2 (up to the largest scale, KVQ_CAP;
// larger values saturate; x = (h - 1/2) d alone, a tie, is clamped to h - 1).  A group holding a NaN
// or an infinity gets the scale byte 0xFF, a NaN half: it reads as NaN.
//
// Why four significant bits: times a 4-bit code that is at most 8 of them,
// times an 8-bit code at most 11, so 4 d c is exactly a half and the matrix
// cores multiply the cache's very values; a scale costs one byte of 32
// (4.25 and 8.25 bits a value) and is at most 1/8 above its least value.
//
// Layout.  A layer's cache is [n_head_kv][tiles of 32 positions] records, each
//   K codes  [32 positions][width BITS / 8 bytes]
//   V codes  [width dims][4 chunks][8 positions: BITS bytes]
//   K scales [width / 32 groups][16][2]       position 16 (r / 8) + 8 i + r % 8 at [g][r][i]
//   V scales [width / 32 groups][4 chunks][8]
// with the eight positions of V chunk c (kvq_v_pos) being those whose scores a
// lane of the matrix cores' result holds, so that the softmax's weights are
// the next product's operand where they are.  Eight values of 4 bits make a dword
// whose nibble e / 2 + 4 (e % 2) holds value e, so that a mask takes values
// 2 i and 2 i + 1 as the halves of one register; 8-bit values are in order.
// Codes are stored as c + h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#define KVQ_TILE 32
#define KVQ_MAXHD 256
// the largest scale byte: 4-bit codes are unpacked as (64 + n) d - 72 d, which
// needs 72 * 4 d within a half (4 d <= 896); 8-bit products need 128 * 4 d
// (4 d <= 480)
#define KVQ_CAP(bits) ((bits) == 4 ? 0xC6 : 0xBF)
#define KVQ_NAN 0xFF

// a head's stored width: the next of 32, 64, 96, 128, 192, 256 (the widths
// the attention kernels are built for)
__host__ __device__ inline int kvq_width(int hd)
{
    return hd <= 128 ? (hd + 31) / 32 * 32 : hd <= 192 ? 192 : 256;
}

// byte offsets inside a record, and its size
struct KvqLayout {
    int width, ng, codes, v, ks, vs, record;
};
__host__ __device__ inline KvqLayout kvq_layout(int bits, int hd)
{
    KvqLayout l;
    l.width = kvq_width(hd);
    l.ng = l.width / 32;
    l.codes = KVQ_TILE * l.width * bits / 8;
    l.v = l.codes;
    l.ks = 2 * l.codes;
    l.vs = l.ks + KVQ_TILE * l.ng;
    l.record = l.vs + KVQ_TILE * l.ng;
    return l;
}

// Position of place e in chunk c of a tile.  A 32x32 result holds, in lane half
// c % 2, rows 8 a + 4 (c % 2) + 0..3 for a = 0..3, and an operand's lane eight of
// 16 summands: chunk c is a = 2 (c / 2) and the next.
__host__ __device__ inline int kvq_v_pos(int c, int e)
{
    return 16 * (c >> 1) + 8 * (e >> 2) + 4 * (c & 1) + (e & 3);
}
// and back: chunk and place of a tile's position r
__device__ __forceinline__ int kvq_v_chunk(int r) { return 2 * (r >> 4) + (r >> 2 & 1); }
__device__ __forceinline__ int kvq_v_place(int r) { return (r & 3) + 4 * (r >> 3 & 1); }
__device__ __forceinline__ int kvq_k_scale(int g, int r)
{
    return g * 32 + (8 * (r >> 4) + (r & 7)) * 2 + (r >> 3 & 1);
}
__device__ __forceinline__ int kvq_v_scale(int g, int r)
{
    return g * 32 + kvq_v_chunk(r) * 8 + kvq_v_place(r);
}

// the scale a byte stands for (NaN from 0xF8 on)
__device__ __forceinline__ float kvq_scale(uint32_t b)
{
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(b << 7)) * 0.25f;
}
