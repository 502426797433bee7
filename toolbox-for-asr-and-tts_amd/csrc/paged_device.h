// Device helpers of the paged cache: which sequence a packed row belongs to, where a position lies.
#pragma once

#include "elem.h"
#include "paged.h"

namespace asrfe {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A sequence, its packed rows [cu0, cu1) and its length (the same in every lane).
struct Sequence {
    int b, cu0, cu1, len;
};

// Largest b whose first row cu_q[b] has upto(b, cu_q[b]), for rising ones: every step a wave compares 64 entries and keeps the
// interval behind the last one that has it, so 4096 sequences take two dependent loads.  The last step brings the rest
// along: loading it afterwards would be one more.  False if none has it.
template <class Upto>
__device__ __forceinline__ bool find_sequence(const PagedView& c, Sequence& s, Upto&& upto) {
    const int lane = threadIdx.x & 63;
    int lo = 0, span = c.batch, step = 1;
    while (step * 64 < span) step *= 64;
    for (;; step >>= 6) {
        const int i = lo + lane * step;
        const bool in = i < lo + span;
        int cu0 = 0, cu1 = 0, len = 0;
        if (in) {
            cu0 = c.cu_q[i];
            if (step == 1) {
                cu1 = c.cu_q[i + 1];
                len = c.kv_lens[i];
            }
        }
        const int n = __builtin_popcountll(__ballot(in && upto(i, cu0)));
        if (n == 0) return false;
        lo += (n - 1) * step;
        if (step == 1) {
            s.b = __builtin_amdgcn_readfirstlane(lo);
            s.cu0 = __builtin_amdgcn_readlane(cu0, n - 1);
            s.cu1 = __builtin_amdgcn_readlane(cu1, n - 1);
            s.len = __builtin_amdgcn_readlane(len, n - 1);
            return true;
        }
        const int left = span - (n - 1) * step;
        span = left < step ? left : step;
    }
}

// The sequence of packed row t (the same in every lane); false if the row belongs to nobody.
__device__ __forceinline__ bool sequence_of(const PagedView& c, int t, Sequence& s) {
    return find_sequence(c, s, [&](int, int cu) { return cu <= t; }) && t < s.cu1;
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

// Eight e4m3 codes (two dwords) times 2^(exp - 127), rounded to the 16-bit type: exact wherever the type has the value, which
// bf16 has and fp16 from 2^-24 times the code's last place on, up to 65504.
// LARGE: the scale may lead out of fp16's range; what does becomes its largest value.
template <bool F16, bool LARGE>
__device__ __forceinline__ u32x4 dequantise8(uint32_t c0, uint32_t c1, uint32_t exp) {
    const float scale = exp ? __uint_as_float(exp << 23) : 0x1p-127f;
    auto two = [&](uint32_t w, auto high) -> uint32_t {
        constexpr bool H = decltype(high)::value;
        if constexpr (F16 && LARGE) {
            const auto f = __builtin_amdgcn_cvt_pk_f32_fp8(w, H);
            auto in = [&](float v) { return v != v ? v : __builtin_amdgcn_fmed3f(v * scale, -65504.0f, 65504.0f); };
            return pack_elem2<F16>(in(f[0]), in(f[1]));
        }
        if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, H));
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, H));
    };
    return u32x4{two(c0, std::false_type{}), two(c0, std::true_type{}), two(c1, std::false_type{}), two(c1, std::true_type{})};
}

inline int32_t launched(asrfe_ctx* ctx, const char* who) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_err(ctx, ASRFE_ERR_HIP, std::string(who) + " launch: " + hipGetErrorString(e));
    return ASRFE_OK;
}

// one instance per head width, 16-bit type and storage (ONE: the kernel's last argument)
#define PAGED_DISPATCH(KERNEL, ONE, grid, block, s, p)                                                \
    do {                                                                                              \
        const bool f16 = dtype == ASRFE_DT_F16;                                                       \
        if (head_dim == 64) {                                                                         \
            if (f16 && e4m3) hipLaunchKernelGGL((KERNEL<64, true, true, ONE>), grid, block, 0, s, p); \
            else if (f16) hipLaunchKernelGGL((KERNEL<64, true, false, ONE>), grid, block, 0, s, p);   \
            else if (e4m3) hipLaunchKernelGGL((KERNEL<64, false, true, ONE>), grid, block, 0, s, p);  \
            else hipLaunchKernelGGL((KERNEL<64, false, false, ONE>), grid, block, 0, s, p);           \
        } else {                                                                                      \
            if (f16 && e4m3) hipLaunchKernelGGL((KERNEL<128, true, true, ONE>), grid, block, 0, s, p);\
            else if (f16) hipLaunchKernelGGL((KERNEL<128, true, false, ONE>), grid, block, 0, s, p);  \
            else if (e4m3) hipLaunchKernelGGL((KERNEL<128, false, true, ONE>), grid, block, 0, s, p); \
            else hipLaunchKernelGGL((KERNEL<128, false, false, ONE>), grid, block, 0, s, p);          \
        }                                                                                             \
    } while (0)

}  // namespace asrfe
