// Writing new keys and values into the pages of a cache, and reading pages back.
//
//   Both move rows of head_dim elements between a dense array and the pages and are bound by memory.  A row is 8 or 16
//   lanes of 16 bytes (16-bit elements); a wave takes one token (one position) and walks its heads, four or eight rows at
//   a time, so that the search for the token's sequence and the look-up of its page are wave-uniform.  Where there are at
//   most half as many heads, it takes as many neighbouring tokens as fill it (2^18 positions of one head of 64 out of an
//   e4m3 cache 57.6 us with one token a wave, 16.8 us this way; into one 84 and 18.6 us).
//
//   e4m3: the largest finite magnitude of a row is found across its lanes, e = the least integer >= -126 with
//   max <= 448 * 2^e comes from its exponent and mantissa fields (448 = 1.75 * 2^8: a mantissa above 1.75 needs one more),
//   and the codes are the conversion instruction's round-to-nearest-even of x * 2^-e.  With a power of two as the scale
//   the multiplication rounds nothing, and reading a row back in the type it came in rounds nothing more (in fp16, what became 65536 is 65504).
//
//   Eight heads of 128: 8 prompts of up to 4096 tokens into an e4m3 cache 30 us (5.0 TB/s), 16 sequences of up to 8192
//   positions out of one 145 us (5.1 TB/s, what a copy reaches).  Eight single tokens 4.0 us: a launch and the chain from
//   cu_q over the length to the page.
#include "paged_device.h"

namespace asrfe {

constexpr int kPagedThreads = 256;

// neighbouring tokens of a wave that holds the rows of `rows` heads at a time
__host__ __device__ __forceinline__ int tokens_of(int n_heads, int rows) { return n_heads < rows ? rows / n_heads : 1; }

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

template <int D, bool F16, bool E4M3, bool ONE>
__global__ __launch_bounds__(kPagedThreads) void kv_append_kernel(const KvAppendParams p) {
    constexpr int kLanes = D / 8;           // lanes of a row
    constexpr int kRows = 64 / kLanes;      // rows of a wave
    const int tokens = ONE ? 1 : tokens_of(p.c.n_heads, kRows);  // of this wave
    const int t0 = (blockIdx.x * (kPagedThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * tokens;
    if (t0 >= p.n_tokens) return;
    const int lane = threadIdx.x & 63, sub = lane / kLanes, col = lane % kLanes;
    Sequence seq;
    if (!sequence_of(p.c, t0, seq)) return;
    const int q = ONE ? 0 : sub / p.c.n_heads, t = t0 + q;
    bool mine = q < tokens && t < p.n_tokens;
    if (!ONE && mine && t >= seq.cu1) {  // (of a later sequence: the last one that begins up to it)
        int lo = seq.b + 1, hi = p.c.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.c.cu_q[mid] <= t) lo = mid;
            else hi = mid;
        }
        mine = lo < p.c.batch;
        if (mine) {
            seq.b = lo;
            seq.cu1 = p.c.cu_q[lo + 1];
            seq.len = p.c.kv_lens[lo];
            mine = t < seq.cu1;
        }
    }
    const int64_t pos64 = static_cast<int64_t>(seq.len) - seq.cu1 + t;
    mine = mine && pos64 >= 0 && pos64 < seq.len;  // (else more new rows than positions)
    const int pos = static_cast<int>(pos64);
    const int page = mine ? page_of(p.c, seq.b, pos) : -1;
    if (__ballot(page >= 0) == 0) return;
    for (int h0 = 0; h0 < p.c.n_heads; h0 += ONE ? kRows : p.c.n_heads) {
        const int h = h0 + sub - q * p.c.n_heads;
        const bool on = page >= 0 && h < p.c.n_heads;
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

template <int D, bool F16, bool E4M3, bool ONE>
__global__ __launch_bounds__(kPagedThreads) void kv_read_kernel(const KvReadParams p) {
    constexpr int kLanes = D / 8;
    constexpr int kRows = 64 / kLanes;
    const int tokens = ONE ? 1 : tokens_of(p.c.n_heads, kRows);  // of this wave
    const int n = p.c.batch * p.t_max;  // (below 2^26)
    const int w0 = (blockIdx.x * (kPagedThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * tokens;
    if (w0 >= n) return;
    const int lane = threadIdx.x & 63, sub = lane / kLanes, col = lane % kLanes;
    const int q = ONE ? 0 : sub / p.c.n_heads, w = w0 + q;
    int b = w0 / p.t_max, pos = w0 % p.t_max + q;
    while (!ONE && pos >= p.t_max) {
        pos -= p.t_max;
        ++b;
    }
    if (q >= tokens || w >= n) return;
    const int page = pos < p.c.kv_lens[b] ? page_of(p.c, b, pos) : -1;
    for (int h0 = 0; h0 < p.c.n_heads; h0 += ONE ? kRows : p.c.n_heads) {
        const int h = h0 + sub - q * p.c.n_heads;
        if (h >= p.c.n_heads) break;
        const int64_t row = cache_row(p.c, page, h, pos);
        const int64_t to = (static_cast<int64_t>(w) * p.c.n_heads + h) * D + 8 * col;
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
    const int tokens = tokens_of(p.c.n_heads, 512 / head_dim), per = tokens * (kPagedThreads / 64);
    const dim3 grid((p.n_tokens + per - 1) / per), block(kPagedThreads);
    if (tokens == 1) PAGED_DISPATCH(kv_append_kernel, true, grid, block, s, p);
    else PAGED_DISPATCH(kv_append_kernel, false, grid, block, s, p);
    return launched(ctx, "kv_append");
}

int32_t launch_kv_read(asrfe_ctx* ctx, const KvReadParams& p, int head_dim, int dtype, bool e4m3, hipStream_t s) {
    const int tokens = tokens_of(p.c.n_heads, 512 / head_dim), per = tokens * (kPagedThreads / 64);
    const dim3 grid((p.c.batch * p.t_max + per - 1) / per), block(kPagedThreads);  // (batch * t_max below 2^26)
    if (tokens == 1) PAGED_DISPATCH(kv_read_kernel, true, grid, block, s, p);
    else PAGED_DISPATCH(kv_read_kernel, false, grid, block, s, p);
    return launched(ctx, "kv_read");
}

}  // namespace asrfe
