// fox_paged_dev.h -- the paged cache's addresses and 16-bit types, shared by
// the kernels that write it (fox_paged.hip) and the attention over it
// (fox_pattn.hip).
#pragma once

#include "fox_internal.h"

// first element of row r (of all the table's) of kv head h of sequence s, in
// either pool; ~0 where the row has no page.  Pools may pass 2^32 elements.
__device__ __forceinline__ size_t paged_row(const PagedDev &C, uint32_t s, uint32_t h, uint32_t r)
{
    const uint32_t page = C.table[(size_t)s * C.max_pages + (r >> C.shift)];
    if (page >= C.n_pages) return ~(size_t)0;
    return ((((size_t)page * C.n_kv + h) << C.shift) + (r & ((1u << C.shift) - 1))) * C.hd;
}

// A float to the cache's type, to the nearest, ties to even.  Halves saturate: an infinite
// key would make every score of its row NaN or infinite.
template <bool BF>
__device__ __forceinline__ uint16_t paged_round(float x)
{
    if (BF) {
        const uint32_t u = __float_as_uint(x);
        if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)(u >> 16 | 0x40u);
        return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1u)) >> 16);
    }
    // (a comparison with a NaN is false: it passes)
    if (x > 65504.0f) x = 65504.0f;
    if (x < -65504.0f) x = -65504.0f;
    return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// Lane l gets the sum of x over lanes 0 .. l, in six adds between neighbours (row shifts, then a
// row's last lane to the rows after it): a shuffle through LDS takes ten times an add.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x)
{
#define FOX_DPP(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xF, false)
    FOX_DPP(0x111, 0xF);
    FOX_DPP(0x112, 0xF);
    FOX_DPP(0x114, 0xF);
    FOX_DPP(0x118, 0xF);
    FOX_DPP(0x142, 0xA);
    FOX_DPP(0x143, 0xC);
#undef FOX_DPP
    return x;
}

// The greatest x of all lanes, and floats' maximum and sum.
__device__ __forceinline__ uint32_t wave_max(uint32_t x)
{
#define FOX_DPP(ctrl, rows) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xF, false))
    FOX_DPP(0x111, 0xF);
    FOX_DPP(0x112, 0xF);
    FOX_DPP(0x114, 0xF);
    FOX_DPP(0x118, 0xF);
    FOX_DPP(0x142, 0xA);
    FOX_DPP(0x143, 0xC);
#undef FOX_DPP
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ float wave_max(float x)
{
#define FOX_DPP(ctrl, rows) \
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp((int)0xFF800000, __float_as_int(x), ctrl, rows, 0xF, false)))
    FOX_DPP(0x111, 0xF);
    FOX_DPP(0x112, 0xF);
    FOX_DPP(0x114, 0xF);
    FOX_DPP(0x118, 0xF);
    FOX_DPP(0x142, 0xA);
    FOX_DPP(0x143, 0xC);
#undef FOX_DPP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float wave_sum(float x)
{
#define FOX_DPP(ctrl, rows) \
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, rows, 0xF, false))
    FOX_DPP(0x111, 0xF);
    FOX_DPP(0x112, 0xF);
    FOX_DPP(0x114, 0xF);
    FOX_DPP(0x118, 0xF);
    FOX_DPP(0x142, 0xA);
    FOX_DPP(0x143, 0xC);
#undef FOX_DPP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
