// Attention of new rows over a paged cache.
//
//   o_i = sum_j p_ij v_j with p_i = softmax over the visible j of scale * q_i . k_j.  One wave per (row, head) walks the
//   keys 64 at a time with a running maximum and sum: a lane scores one key, then owns head_dim / 64 channels of the sum.
#include "paged_device.h"

namespace asrfe {

template <int D, bool F16, bool E4M3>
__device__ __forceinline__ void load8(const char* base, const uint8_t* exps, int64_t row, int chunk, float* f) {
    uint4 x;
    if constexpr (E4M3) x = dequantise8<F16>(*reinterpret_cast<const uint2*>(base + row * D + 8 * chunk), exps[row]);
    else x = *reinterpret_cast<const uint4*>(base + row * (2 * D) + 16 * chunk);
    unpack_elem2<F16>(x.x, f[0], f[1]);
    unpack_elem2<F16>(x.y, f[2], f[3]);
    unpack_elem2<F16>(x.z, f[4], f[5]);
    unpack_elem2<F16>(x.w, f[6], f[7]);
}

template <int D, bool F16, bool E4M3>
__global__ __launch_bounds__(256) void paged_attn_kernel(const PagedAttnParams p) {
    constexpr int kOwn = D / 64;
    saturate_fp16_conversions<F16>();
    const int lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= static_cast<int64_t>(p.n_tokens) * p.n_q_heads) return;
    const int t = static_cast<int>(item / p.n_q_heads), hq = static_cast<int>(item % p.n_q_heads), h = hq / p.group;
    const int b = find_sequence(p.c.cu_q, p.c.batch, t);
    if (b < 0) return;
    int len = p.c.kv_lens[b];
    const int64_t pos = static_cast<int64_t>(len) - p.c.cu_q[b + 1] + t;
    len = len < p.max_kv ? len : p.max_kv;
    int64_t hi = p.causal ? (pos + 1 < len ? pos + 1 : len) : (pos >= 0 ? len : 0);
    int64_t lo = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
    const uint16_t* q = p.q + t * p.q_ts + hq * p.q_hs;
    float m = -INFINITY, l = 0.0f, o[kOwn] = {};
    for (int64_t j0 = 0; j0 < hi; j0 += 64) {
        if (j0 >= p.sinks && j0 + 64 <= lo) { j0 = (lo & ~63ll) - 64; continue; }
        const int64_t j = j0 + lane;
        int page = j < hi && (j >= lo || j < p.sinks) ? page_of(p.c, b, static_cast<int>(j)) : -1;
        float s = -INFINITY;
        if (page >= 0) {
            const int64_t row = cache_row(p.c, page, h, static_cast<int>(j));
            float acc = 0.0f;
            for (int c = 0; c < D / 8; ++c) {
                float kf[8], qf[8];
                load8<D, F16, E4M3>(p.c.k, p.c.k_exp, row, c, kf);
                load8<D, F16, false>(reinterpret_cast<const char*>(q), nullptr, 0, c, qf);
                for (int i = 0; i < 8; ++i) acc = fmaf(kf[i], qf[i], acc);
            }
            s = acc * p.scale_log2;
        }
        float top = s;
        for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const uint64_t seen = __ballot(page >= 0);
        if (seen == 0) continue;
        const float mn = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float w = page >= 0 ? __builtin_amdgcn_exp2f(s - mn) : 0.0f;
        float sum = w;
        for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * alpha + sum;
        m = mn;
        for (int i = 0; i < kOwn; ++i) o[i] *= alpha;
        for (int k = 0; k < 64; ++k) {
            if (!((seen >> k) & 1)) continue;
            const float wk = __shfl(w, k);
            const int pk = __shfl(page, k);
            const int64_t row = cache_row(p.c, pk, h, static_cast<int>(j0 + k));
            for (int i = 0; i < kOwn; ++i) {
                const int d = lane * kOwn + i;
                float vf[8];
                load8<D, F16, E4M3>(p.c.v, p.c.v_exp, row, d >> 3, vf);
                float v = vf[0];
                for (int e = 1; e < 8; ++e) v = (d & 7) == e ? vf[e] : v;
                o[i] = fmaf(wk, v, o[i]);
            }
        }
    }
    uint16_t* out = p.out + t * p.o_ts + hq * p.o_hs;
    for (int i = 0; i < kOwn; ++i) out[lane * kOwn + i] = to_elem<F16>(l > 0.0f || l != l ? o[i] / l : 0.0f);
}

int64_t paged_attention_workspace(const asrfe_ctx*, int, int, int, int, int, int) { return 0; }

int32_t launch_paged_attention(asrfe_ctx* ctx, const PagedAttnParams& p, int head_dim, int dtype, bool e4m3, void*, hipStream_t s) {
    const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(p.n_tokens) * p.n_q_heads + 3) / 4)), block(256);
    PAGED_DISPATCH(paged_attn_kernel, grid, block, s, p);
    return launched(ctx, "paged_attention");
}

}  // namespace asrfe
