// Choice of a token per row of logits: temperature, top-k, top-p, min-p and one random number.
//
//   One workgroup per row.  Weights w_i = exp((l_i - max) / T) are formed in double precision and summed as integers of
//   2^-44, so that sums are the same in any order.  The order of the vocabulary (falling logit, rising index) is the
//   order of a 32-bit key per logit; what is kept is a prefix of it, described by the key of its last element and the
//   number of elements with that key (ties are taken in rising index).  Each filter's cut is found by bisection of the key.
#include "elem.h"
#include "paged_device.h"

namespace asrfe {

constexpr int kSampleThreads = 1024;

template <int DT>
__device__ __forceinline__ float logit_at(const void* row, int i) {
    float v;
    if constexpr (DT == ASRFE_DT_F32) v = static_cast<const float*>(row)[i];
    else if constexpr (DT == ASRFE_DT_F16) v = static_cast<float>(static_cast<const _Float16*>(row)[i]);
    else v = __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[i]) << 16);
    return v != v ? -INFINITY : v;
}

// a larger logit has the larger key; -0 and +0 have the same; -inf is the least
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
constexpr uint32_t kKeyNone = 0x007fffffu;  // key of -inf

template <class T>
__device__ __forceinline__ T block_sum(T v, T* buf) {
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = 0;
    for (int i = 0; i < kSampleThreads / 64; ++i) s += buf[i];
    return s;
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleParams p) {
    __shared__ unsigned long long buf[kSampleThreads / 64];
    __shared__ unsigned long long upto[kSampleThreads];
    __shared__ int chosen;
    const int r = blockIdx.x, tid = threadIdx.x;
    if (p.token_num && r % p.rows_per >= p.token_num[r / p.rows_per]) {
        if (tid == 0) {
            p.ids[r] = -1;
            if (p.logprobs) p.logprobs[r] = 0.0f;
        }
        return;
    }
    const void* row = static_cast<const char*>(p.logits) + static_cast<int64_t>(r) * p.ld * (DT == ASRFE_DT_F32 ? 4 : 2);
    float top = -INFINITY;
    for (int i = tid; i < p.vocab; i += kSampleThreads) top = fmaxf(top, logit_at<DT>(row, i));
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) buf[tid >> 6] = __float_as_uint(top);
    if (tid == 0) chosen = 0x7fffffff;
    __syncthreads();
    for (int i = 0; i < kSampleThreads / 64; ++i) top = fmaxf(top, __uint_as_float(static_cast<uint32_t>(buf[i])));
    if (top == -INFINITY) {
        if (tid == 0) {
            p.ids[r] = 0;
            if (p.logprobs) p.logprobs[r] = -INFINITY;
        }
        return;
    }
    const float temp = p.temperature ? p.temperature[r] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    const double inv_t = greedy ? 1.0 : 1.0 / static_cast<double>(temp);
    auto weight = [&](float v) -> double {
        if (v == top) return 1.0;
        return v == -INFINITY ? 0.0 : exp((static_cast<double>(v) - static_cast<double>(top)) * inv_t);
    };
    auto fixed = [](double w) { return static_cast<unsigned long long>(w * 0x1p44 + 0.5); };
    // what is kept: keys above `cut`, and the first `ties` elements with that key
    uint32_t cut = key_of(top);
    unsigned long long ties = 1;
    auto count = [&](uint32_t k, bool above) {  // elements with a key at or above (above) k
        unsigned long long n = 0;
        for (int i = tid; i < p.vocab; i += kSampleThreads) {
            const uint32_t x = key_of(logit_at<DT>(row, i));
            n += above ? x > k : x >= k;
        }
        return block_sum(n, buf);
    };
    if (!greedy) {
        const int k = p.top_k ? p.top_k[r] : 0;
        cut = kKeyNone;
        ties = 0;  // (nothing at -inf is ever kept)
        if (k > 0 && k < p.vocab && count(kKeyNone, true) > static_cast<unsigned long long>(k)) {
            uint32_t lo = kKeyNone + 1, hi = key_of(top);  // largest key with at least k elements at or above it
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                if (count(mid, false) >= static_cast<unsigned long long>(k)) lo = mid;
                else hi = mid - 1;
            }
            cut = lo;
            ties = k - count(cut, true);
        }
        auto mass = [&](uint32_t kk) {  // weight of the elements with a key above kk
            unsigned long long n = 0;
            for (int i = tid; i < p.vocab; i += kSampleThreads) {
                const float v = logit_at<DT>(row, i);
                if (key_of(v) > kk) n += fixed(weight(v));
            }
            return block_sum(n, buf);
        };
        auto value_of = [](uint32_t kk) { return __uint_as_float((kk & 0x80000000u) ? (kk & 0x7fffffffu) : ~kk); };
        const float top_p = p.top_p ? p.top_p[r] : 1.0f;
        if (top_p < 1.0f) {
            const unsigned long long all = mass(cut) + ties * fixed(weight(value_of(cut)));
            const double want = static_cast<double>(top_p) * static_cast<double>(all);
            // an element is kept while what lies before it in the order is below `want`: the least key whose elements
            // have less than that before them
            uint32_t lo = cut, hi = key_of(top);
            if (lo == kKeyNone) ++lo;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                if (static_cast<double>(mass(mid)) < want) hi = mid;
                else lo = mid + 1;
            }
            // (an empty key has the next larger element's mass before it: raise to the key of an element)
            const double before = static_cast<double>(mass(lo));
            const double each = static_cast<double>(fixed(weight(value_of(lo))));
            unsigned long long n = each > 0.0 ? static_cast<unsigned long long>(fmax(1.0, ceil((want - before) / each))) : ~0ull;
            if (lo > cut || n < ties) ties = lo > cut ? n : (n < ties ? n : ties);
            cut = lo;
            if (!(want > 0.0)) { cut = key_of(top); ties = 1; }
        }
        const float min_p = p.min_p ? p.min_p[r] : 0.0f;
        if (min_p > 0.0f) {
            uint32_t lo = cut > kKeyNone ? cut : kKeyNone + 1, hi = key_of(top);  // least key whose weight is at least min_p
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo) / 2;
                if (weight(value_of(mid)) >= static_cast<double>(min_p)) hi = mid;
                else lo = mid + 1;
            }
            if (static_cast<double>(min_p) > 1.0) ties = 1;
            else if (lo > cut) ties = ~0ull;
            cut = lo;
        }
    }
    // ---- the kept weights in the order of the vocabulary: every thread a run of elements
    const int run = (p.vocab + kSampleThreads - 1) / kSampleThreads;
    const int i0 = min(p.vocab, tid * run), i1 = min(p.vocab, i0 + run);
    unsigned long long same = 0;
    for (int i = i0; i < i1; ++i) same += key_of(logit_at<DT>(row, i)) == cut;
    auto scan = [&](unsigned long long v) {  // sum over the threads before this one
        __syncthreads();
        upto[tid] = v;
        __syncthreads();
        for (int o = 1; o < kSampleThreads; o <<= 1) {
            const unsigned long long x = tid >= o ? upto[tid - o] : 0;
            __syncthreads();
            upto[tid] += x;
            __syncthreads();
        }
        return upto[tid] - v;
    };
    const unsigned long long same_before = scan(same);
    auto walk = [&](auto&& f) {
        unsigned long long n = same_before;
        for (int i = i0; i < i1; ++i) {
            const float v = logit_at<DT>(row, i);
            const uint32_t x = key_of(v);
            if (x > cut || (x == cut && n < ties)) f(i, weight(v));
            n += x == cut;
        }
    };
    unsigned long long mine = 0;
    walk([&](int, double w) { mine += fixed(w); });
    const unsigned long long before = scan(mine);
    const unsigned long long total = upto[kSampleThreads - 1];
    // sums are whole, so a sum exceeds u * total where it exceeds its whole part; a number outside [0, 1) takes an end
    const double at = fmax(0.0, static_cast<double>(p.u[r])) * static_cast<double>(total);
    const unsigned long long target = at < static_cast<double>(total) ? min(static_cast<unsigned long long>(at), total - 1) : total - 1;
    unsigned long long sum = before;
    if (before + mine > target && before <= target) {
        walk([&](int i, double w) {
            sum += fixed(w);
            if (sum > target) atomicMin(&chosen, i);
        });
    }
    __syncthreads();
    if (tid == 0) {
        p.ids[r] = chosen;
        if (p.logprobs) p.logprobs[r] = static_cast<float>(log(weight(logit_at<DT>(row, chosen)) * 0x1p44 / static_cast<double>(total)));
    }
}

int32_t launch_sample(asrfe_ctx* ctx, const SampleParams& p, int dtype, hipStream_t s) {
    const dim3 grid(p.rows), block(kSampleThreads);
    if (dtype == ASRFE_DT_F32) hipLaunchKernelGGL(sample_kernel<ASRFE_DT_F32>, grid, block, 0, s, p);
    else if (dtype == ASRFE_DT_F16) hipLaunchKernelGGL(sample_kernel<ASRFE_DT_F16>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(sample_kernel<ASRFE_DT_BF16>, grid, block, 0, s, p);
    return launched(ctx, "sample_tokens");
}

}  // namespace asrfe
