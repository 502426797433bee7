// Writing new keys and values into the pages of a cache, and reading pages back.
//
//   Both move rows of head_dim elements between a dense array and the pages and are bound by memory.  A row is 8 or 16
//   lanes of 16 bytes (16-bit elements); a wave takes one token (one position) and walks its heads, four or eight rows at
//   a time, so that the search for the token's sequence and the look-up of its page are wave-uniform.
//
//   e4m3: the largest finite magnitude of a row is found across its lanes, e = the least integer >= -126 with
//   max <= 448 * 2^e comes from its exponent and mantissa fields (448 = 1.75 * 2^8: a mantissa above 1.75 needs one more),
//   and the codes are the conversion instruction's round-to-nearest-even of x * 2^-e.  With a power of two as the scale
//   the multiplication rounds nothing, and reading back is exact in both 16-bit types.
//
//   Eight heads of 128: 8 prompts of up to 4096 tokens into an e4m3 cache 31 us (4.9 TB/s), 16 sequences of up to 8192
//   positions out of one 147 us (5.1 TB/s, what a copy reaches).  Eight single tokens 4.4 us: a launch and the chain from
//   cu_q over the length to the page.
#include "paged_device.h"

namespace asrfe {

constexpr int kPagedThreads = 256;

// maximum over the 8 or 16 neighbours that hold a row: pairs, fours, eights (a mirrored half row), sixteens
template <int N>
__device__ __forceinline__ float max_of_row(float v) {
    auto with = [&](auto ctrl) { v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true))); };
    with(std::integral_constant<int, 0xb1>{});
    with(std::integral_constant<int, 0x4e>{});
    with(std::integral_constant<int, 0x141>{});
    if constexpr (N == 16) with(std::integral_constant<int, 0x140>{});
    return v;
}

template <int D, bool F16, bool E4M3>
__global__ __launch_bounds__(kPagedThreads) void kv_append_kernel(const KvAppendParams p) {
    constexpr int kLanes = D / 8;           // lanes of a row
    constexpr int kRows = 64 / kLanes;      // rows of a wave
    const int t = blockIdx.x * (kPagedThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= p.n_tokens) return;
    const int lane = threadIdx.x & 63, sub = lane / kLanes, col = lane % kLanes;
    Sequence seq;
    if (!sequence_of(p.c, t, seq)) return;
    const int64_t pos64 = static_cast<int64_t>(seq.len) - seq.cu1 + t;
    if (pos64 < 0 || pos64 >= seq.len) return;  // (more new rows than positions)
    const int pos = static_cast<int>(pos64);
    const int page = page_of(p.c, seq.b, pos);
    if (page < 0) return;
    for (int h0 = 0; h0 < p.c.n_heads; h0 += kRows) {
        const int h = h0 + sub;
        const bool on = h < p.c.n_heads;
        const int64_t row = cache_row(p.c, page, h, pos);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint16_t* src = kv ? p.v + t * p.v_ts + h * p.v_hs : p.k + t * p.k_ts + h * p.k_hs;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (on) x = *reinterpret_cast<const uint4*>(src + 8 * col);
            char* dst = kv ? p.c.v : p.c.k;
            if constexpr (!E4M3) {
                if (on) *reinterpret_cast<uint4*>(dst + row * (2 * D) + 16 * col) = x;
            } else {
                float f[8];
                unpack_elem2<F16>(x.x, f[0], f[1]);
                unpack_elem2<F16>(x.y, f[2], f[3]);
                unpack_elem2<F16>(x.z, f[4], f[5]);
                unpack_elem2<F16>(x.w, f[6], f[7]);
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = __builtin_fabsf(f[i]);
                    top = fmaxf(top, a < INFINITY ? a : 0.0f);  // (infinities and NaN take no part)
                }
                top = max_of_row<kLanes>(top);
                const uint32_t bits = __float_as_uint(top);
                int e = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7fffffu) > 0x600000u ? 7 : 8);
                e = top > 0.0f ? (e > -126 ? e : -126) : 0;
                const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e, -126 <= e <= 120
                uint32_t w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float s = f[4 * i + j] * inv;
                        const float c = __builtin_amdgcn_fmed3f(s, -448.0f, 448.0f);  // an infinity becomes the largest code
                        y[j] = s != s ? s : c;
                    }
                    int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
                    v = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], v, true);
                    w[i] = static_cast<uint32_t>(v);
                }
                if (on) {
                    *reinterpret_cast<uint2*>(dst + row * D + 8 * col) = make_uint2(w[0], w[1]);
                    if (col == 0) (kv ? p.c.v_exp : p.c.k_exp)[row] = static_cast<uint8_t>(e + 127);
                }
            }
        }
    }
}

template <int D, bool F16, bool E4M3>
__global__ __launch_bounds__(kPagedThreads) void kv_read_kernel(const KvReadParams p) {
    constexpr int kLanes = D / 8;
    constexpr int kRows = 64 / kLanes;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (kPagedThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= static_cast<int64_t>(p.c.batch) * p.t_max) return;
    const int lane = threadIdx.x & 63, sub = lane / kLanes, col = lane % kLanes;
    const int b = static_cast<int>(w / p.t_max), pos = static_cast<int>(w % p.t_max);
    const int page = pos < p.c.kv_lens[b] ? page_of(p.c, b, pos) : -1;
    for (int h0 = 0; h0 < p.c.n_heads; h0 += kRows) {
        const int h = h0 + sub;
        if (h >= p.c.n_heads) break;
        const int64_t row = cache_row(p.c, page, h, pos);
        const int64_t to = (w * p.c.n_heads + h) * D + 8 * col;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            u32x4 x = {0, 0, 0, 0};
            if (page >= 0) {
                const char* src = kv ? p.c.v : p.c.k;
                if constexpr (E4M3) {
                    const uint2 codes = *reinterpret_cast<const uint2*>(src + row * D + 8 * col);
                    x = dequantise8<F16, true>(codes.x, codes.y, (kv ? p.c.v_exp : p.c.k_exp)[row]);
                } else {
                    x = *reinterpret_cast<const u32x4*>(src + row * (2 * D) + 16 * col);
                }
            }
            *reinterpret_cast<u32x4*>((kv ? p.v : p.k) + to) = x;
        }
    }
}

int32_t launch_kv_append(asrfe_ctx* ctx, const KvAppendParams& p, int head_dim, int dtype, bool e4m3, hipStream_t s) {
    const dim3 grid((p.n_tokens + 3) / 4), block(kPagedThreads);
    PAGED_DISPATCH(kv_append_kernel, grid, block, s, p);
    return launched(ctx, "kv_append");
}

int32_t launch_kv_read(asrfe_ctx* ctx, const KvReadParams& p, int head_dim, int dtype, bool e4m3, hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(p.c.batch) * p.t_max + 3) / 4)), block(kPagedThreads);
    PAGED_DISPATCH(kv_read_kernel, grid, block, s, p);
    return launched(ctx, "kv_read");
}

}  // namespace asrfe
