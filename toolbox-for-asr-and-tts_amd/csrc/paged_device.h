// Device helpers of the paged cache: which sequence a packed row belongs to, where a position lies.
#pragma once

#include "elem.h"
#include "paged.h"

namespace asrfe {

// Largest b with cu_q[b] <= t, for a wave-uniform t: every step a wave compares 64 entries and keeps the interval behind
// the last one that is not above t, so 65535 sequences take three dependent loads.  -1 if the row belongs to nobody.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ cu_q, int batch, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, span = batch + 1, step = 1;
    while (step * 64 < span) step *= 64;
    for (;; step >>= 6) {
        const int i = lo + lane * step;
        const bool below = i < lo + span && cu_q[i] <= t;
        const int c = __builtin_popcountll(__ballot(below));
        if (c == 0) return -1;
        lo += (c - 1) * step;
        const int left = span - (c - 1) * step;
        span = left < step ? left : step;
        if (step == 1) break;
    }
    return lo < batch ? lo : -1;
}

// Page of position pos of sequence b, -1 where there is none.
__device__ __forceinline__ int page_of(const PagedView& c, int b, int pos) {
    const int i = pos >> c.page_shift;
    if (i >= c.table_stride) return -1;
    const int page = c.block_table[static_cast<int64_t>(b) * c.table_stride + i];
    return page >= 0 && page < c.n_pages ? page : -1;
}

// Row index of (page, head, position in the page) in the cache's [pages][heads][page_size] rows.
__device__ __forceinline__ int64_t cache_row(const PagedView& c, int page, int head, int pos) {
    return ((static_cast<int64_t>(page) * c.n_heads + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}

// Eight e4m3 codes (two dwords) times 2^(exp - 127), rounded to the 16-bit type: exact wherever the type has the value.
template <bool F16>
__device__ __forceinline__ uint4 dequantise8(uint2 codes, uint32_t exp) {
    const float scale = exp ? __uint_as_float(exp << 23) : 0x1p-127f;
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = i ? codes.y : codes.x;
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        r[2 * i] = pack_elem2<F16>(lo[0] * scale, lo[1] * scale);
        r[2 * i + 1] = pack_elem2<F16>(hi[0] * scale, hi[1] * scale);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

inline int32_t launched(asrfe_ctx* ctx, const char* who) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_err(ctx, ASRFE_ERR_HIP, std::string(who) + " launch: " + hipGetErrorString(e));
    return ASRFE_OK;
}

// one instance per head width, 16-bit type and storage
#define PAGED_DISPATCH(KERNEL, grid, block, s, p)                                                     \
    do {                                                                                              \
        const bool f16 = dtype == ASRFE_DT_F16;                                                       \
        if (head_dim == 64) {                                                                         \
            if (f16 && e4m3) hipLaunchKernelGGL((KERNEL<64, true, true>), grid, block, 0, s, p);      \
            else if (f16) hipLaunchKernelGGL((KERNEL<64, true, false>), grid, block, 0, s, p);        \
            else if (e4m3) hipLaunchKernelGGL((KERNEL<64, false, true>), grid, block, 0, s, p);       \
            else hipLaunchKernelGGL((KERNEL<64, false, false>), grid, block, 0, s, p);                \
        } else {                                                                                      \
            if (f16 && e4m3) hipLaunchKernelGGL((KERNEL<128, true, true>), grid, block, 0, s, p);     \
            else if (f16) hipLaunchKernelGGL((KERNEL<128, true, false>), grid, block, 0, s, p);       \
            else if (e4m3) hipLaunchKernelGGL((KERNEL<128, false, true>), grid, block, 0, s, p);      \
            else hipLaunchKernelGGL((KERNEL<128, false, false>), grid, block, 0, s, p);               \
        }                                                                                             \
    } while (0)

}  // namespace asrfe
