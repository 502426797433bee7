// Choice of a token per row of logits: temperature, top-k, top-p, min-p and one random number.
//
//   One workgroup per row (256 threads for small vocabularies, else 1024).  Weights w = 2^((l - max) log2(e) / T) are formed
//   in double precision (a table of 2^(j / 32) and a polynomial: relative error below 1e-11; double FMAs issue at the rate
//   of single ones here) and summed as whole multiples of 2^-44, so a sum is the same in any order and atomics may form
//   it.  What is kept is a prefix of the order (falling logit, rising index), described by the value of its last element,
//   `cut`, and the number of elements of that value that belong to it, `ties`.
//
//   The row is read from memory once for its maximum and, from the caches, once or a few times more:
//     * few candidates (a small top_k, or min_p): the k-th largest of 1024 partial maxima is a lower bound of the k-th
//       largest logit; what is at or above it goes into a list in the LDS, in the order of the vocabulary, and every
//       filter is settled there by counting (256 entries at most; more take the way below);
//     * else a cut is found by histograms in the LDS, first over (max - l) / T, then over the keys of the values left in
//       the bin where the cut lies, 2048 bins at a time, until one value is left;
//     * the number is then looked up in the running sum over the vocabulary: per wave, per step of that wave, per lane.
#include "elem.h"
#include "paged_device.h"

namespace asrfe {

typedef unsigned long long u64;

constexpr int kBins = 2048;
constexpr int kList = 256;        // candidates the list path takes
constexpr int kTopKList = 200;    // largest top_k that tries it: the list holds ties and near misses too
constexpr double kOctaves = 46.0; // weights below 2^-45 are zero in multiples of 2^-44

// an order-preserving whole number per value (16 bits for 16-bit logits); -0 and +0 have the same
template <int DT>
__device__ __forceinline__ uint32_t key_of(float v) {
    v += 0.0f;
    uint32_t b;
    if constexpr (DT == ASRFE_DT_F16) b = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v))) << 16;
    else b = __float_as_uint(v);
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return DT == ASRFE_DT_F32 ? b : b >> 16;
}
template <int DT>
__device__ __forceinline__ float value_of(uint32_t k) {
    uint32_t b = DT == ASRFE_DT_F32 ? k : k << 16;
    b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
    if constexpr (DT == ASRFE_DT_F32) return __uint_as_float(b);
    else if constexpr (DT == ASRFE_DT_BF16) return __uint_as_float(b & 0xffff0000u);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(b >> 16)));
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {  // sum up to and with this lane
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 x = __shfl_up(v, o);
        v += (threadIdx.x & 63) >= static_cast<unsigned>(o) ? x : 0;
    }
    return v;
}

template <int NT>
struct SampleLds {
    static constexpr int kWaves = NT / 64;
    double table[32];
    u64 a[kWaves], b[kWaves];
    union {
        u64 hist[kBins];
        uint32_t maxima[1024];
        struct {
            float value[kWaves][kList];
            int index[kWaves][kList];
        } found;
    };
    struct {
        float value[kList];
        int index[kList];
        u64 weight[kList];
    } list;
    u64 res[4];
    int n[kWaves];
    int total;
};

template <int DT, int NT>
struct Sampler {
    static constexpr int kWaves = NT / 64;
    static constexpr int kVec = DT == ASRFE_DT_F32 ? 4 : 8;
    static constexpr int kSub = 1024 / NT;  // partial maxima of a thread

    const SampleParams& p;
    SampleLds<NT>& s;
    const int tid, lane, wave;
    const char* row;
    int head, n_vec, n_steps;  // elements before the first 16-byte boundary, 16-byte pieces, steps of 64 of them
    float top, low;            // largest logit, least logit with a weight
    double a;                  // log2(e) / T

    __device__ Sampler(const SampleParams& p_, SampleLds<NT>& s_, int r)
        : p(p_), s(s_), tid(threadIdx.x), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
        constexpr int kSize = DT == ASRFE_DT_F32 ? 4 : 2;
        row = static_cast<const char*>(p.logits) + static_cast<int64_t>(r) * p.ld * kSize;
        head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / kSize;
        head = head < p.vocab ? head : p.vocab;
        n_vec = (p.vocab - head) / kVec;
        n_steps = (n_vec + 63) / 64;
    }

    __device__ float one(int i) const {
        if constexpr (DT == ASRFE_DT_F32) return reinterpret_cast<const float*>(row)[i];
        else if constexpr (DT == ASRFE_DT_F16) return static_cast<float>(reinterpret_cast<const _Float16*>(row)[i]);
        else return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[i]) << 16);
    }
    __device__ static void widen(const uint4 w, float (&x)[kVec]) {
        if constexpr (DT == ASRFE_DT_F32) {
            x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
        } else {
            constexpr bool kF16 = DT == ASRFE_DT_F16;
            unpack_elem2<kF16>(w.x, x[0], x[1]);
            unpack_elem2<kF16>(w.y, x[2], x[3]);
            unpack_elem2<kF16>(w.z, x[4], x[5]);
            unpack_elem2<kF16>(w.w, x[6], x[7]);
        }
    }
    // The row in steps: step 0 is the head (one element per lane), then the pieces, then what is left behind the last one.
    // f(x, i0): this lane's elements i0, i0 + 1, ... (NaN where it has none: no comparison holds for them).
    template <class F>
    __device__ void step(int t, F&& f) const {
        float x[kVec];
        if (t > 0 && t <= n_steps) {
            const int v = (t - 1) * 64 + lane;
            const int i0 = head + v * kVec;
            if (v < n_vec) {
                widen(*reinterpret_cast<const uint4*>(row + static_cast<int64_t>(i0) * (DT == ASRFE_DT_F32 ? 4 : 2)), x);
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) x[e] = __builtin_nanf("");
            }
            f(x, i0);
        } else {
            const int i0 = t == 0 ? lane : head + n_vec * kVec + lane, end = t == 0 ? head : p.vocab;
#pragma unroll
            for (int e = 1; e < kVec; ++e) x[e] = __builtin_nanf("");
            x[0] = i0 < end ? one(i0) : __builtin_nanf("");
            f(x, i0);
        }
    }
    __device__ int steps() const { return n_steps + 2; }
    template <class F>
    __device__ void steps_of(int t0, int t1, int by, F&& f) const {
        for (int t = t0; t < t1; t += by) {
            if (t + 3 * by < t1 && t > 0 && t + 3 * by < n_steps) {  // four full steps at once: four loads in flight
                uint4 w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i0 = head + ((t + k * by - 1) * 64 + lane) * kVec;
                    w[k] = *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(i0) * (DT == ASRFE_DT_F32 ? 4 : 2));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float x[kVec];
                    widen(w[k], x);
                    f(x, head + ((t + k * by - 1) * 64 + lane) * kVec);
                }
                t += 3 * by;
            } else {
                step(t, f);
            }
        }
    }
    // this wave's run of steps: runs follow each other in the order of the vocabulary
    __device__ int run_of(int w) const {
        const int per = (steps() + kWaves - 1) / kWaves, t = w * per;
        return t < steps() ? t : steps();
    }
    template <class F>
    __device__ void walk(F&& f) const { steps_of(run_of(wave), run_of(wave + 1), 1, f); }

    // weight in multiples of 2^-44; v is at least `low`
    __device__ u64 fixed(float v) const {
        const double t = fmax((static_cast<double>(fminf(v, 3.402823466e38f)) - static_cast<double>(fminf(top, 3.402823466e38f))) * a, -200.0);
        constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
        const double d = t * 32.0 + kMagic;
        const int k = static_cast<int>(__builtin_bit_cast(u64, d));
        const double f = fma(d - kMagic, -1.0 / 32.0, t);  // |f| <= 1 / 64
        // 2^f = sum (f ln 2)^n / n!, up to n = 4: the next term is below 2e-12
        double y = fma(f, 0.009618129107628477, 0.05550410866482158);
        y = fma(f, y, 0.2402265069591007);
        y = fma(f, y, 0.6931471805599453);
        y = fma(f, y, 1.0) * s.table[k & 31];
        const double scale = __builtin_bit_cast(double, static_cast<u64>(1023 + 44 + (k >> 5)) << 52);
        return __builtin_bit_cast(u64, fma(y, scale, 0x1p52)) & 0xfffffffffffffull;
    }
    __device__ u64 weight(float v) const { return v >= low ? fixed(v) : 0; }

    __device__ u64 block_sum(u64 v) {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) s.a[wave] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) t += s.a[i];
        return t;
    }

    // Finds the value at which a running sum over falling values first reaches `want` (1 <= want <= the sum of all):
    // the sum over larger values is below `want`, the sum with that value's elements is not.  MASS: sums of weights, else of
    // elements.
    template <bool MASS>
    __device__ float reach(u64 want, u64& before) {
        const float least = MASS ? low : -3.402823466e38f;
        const float span = static_cast<float>(kOctaves / a);  // logits per kOctaves octaves of weight
        const float scale = fminf(static_cast<float>(kBins) / span, 3e38f);
        auto bin1 = [&](float v) {
            const float d = (top - v) * scale;
            return static_cast<int>(d < kBins - 1 ? d : (d == d ? kBins - 1.0f : 0.0f));  // (inf - inf: the top itself)
        };
        before = 0;
        uint32_t lo = 0, hi = 0;  // keys among which the value is, after the first pass
        int shift = -1;
        for (;;) {
            __syncthreads();
            for (int i = tid; i < kBins; i += NT) s.hist[i] = 0;
            __syncthreads();
            walk([&](const float (&x)[kVec], int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (!(x[e] >= least)) continue;
                    int b;
                    if (shift < 0) {
                        b = bin1(x[e]);
                    } else {
                        const uint32_t k = key_of<DT>(x[e]);
                        if (k < lo || k > hi) continue;
                        b = static_cast<int>((hi - k) >> shift);
                    }
                    atomicAdd(&s.hist[b], MASS ? fixed(x[e]) : u64{1});
                }
            });
            __syncthreads();
            // the bin where `want` is reached: every thread a run of bins
            constexpr int kPer = kBins / NT;
            u64 mine = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) mine += s.hist[tid * kPer + i];
            u64 sum = wave_scan(mine);
            if (lane == 63) s.a[wave] = sum;
            __syncthreads();
            for (int i = 0; i < wave; ++i) sum += s.a[i];
            sum += before - mine;
            if (sum < want && want <= sum + mine) {
                int b = tid * kPer;
                while (sum + s.hist[b] < want) sum += s.hist[b++];
                s.res[0] = sum;
                s.res[1] = b;
            }
            __syncthreads();
            before = s.res[0];
            const int b = static_cast<int>(s.res[1]);
            if (shift < 0) {
                // keys of the bin's values: the ends are found by trying 64 keys at a time (bins fall as keys rise)
                const uint32_t k0 = key_of<DT>(least), k1 = key_of<DT>(top);
                auto first = [&](int bin) {  // least key whose bin is at most `bin`
                    uint32_t l = k0, h = k1;
                    while (l < h) {
                        const uint32_t w = (h - l) / 64 + 1;
                        const u64 at = static_cast<u64>(l) + static_cast<u64>(w) * lane;
                        const bool yes = at >= h || bin1(value_of<DT>(static_cast<uint32_t>(at))) <= bin;
                        const u64 m = __ballot(yes);
                        const int c = m ? __builtin_ctzll(m) : 64;  // lanes before c: a higher bin
                        if (c == 0) return l;
                        const u64 nl = static_cast<u64>(l) + static_cast<u64>(w) * (c - 1) + 1, nh = c < 64 ? static_cast<u64>(l) + static_cast<u64>(w) * c : h;
                        l = static_cast<uint32_t>(nl);
                        h = static_cast<uint32_t>(nh < h ? nh : h);
                    }
                    return l;
                };
                lo = first(b);
                hi = b > 0 ? first(b - 1) - 1 : k1;
            } else {
                hi -= static_cast<uint32_t>(b) << shift;
                const uint32_t width = (1u << shift) - 1;
                lo = hi - lo > width ? hi - width : lo;
            }
            lo = __builtin_amdgcn_readfirstlane(lo);
            hi = __builtin_amdgcn_readfirstlane(hi);
            if (lo >= hi) return value_of<DT>(hi);
            shift = 0;
            while (((hi - lo) >> shift) >= static_cast<uint32_t>(kBins)) ++shift;
        }
    }

    // id and log-probability: v its logit, total the kept weight
    __device__ void put(int r, int id, float v, u64 total) const {
        p.ids[r] = id;
        if (p.logprobs) {
            const double t = (static_cast<double>(fminf(v, 3.402823466e38f)) - static_cast<double>(fminf(top, 3.402823466e38f))) * a;
            p.logprobs[r] = static_cast<float>(t * 0.6931471805599453 - log(static_cast<double>(total) * 0x1p-44));
        }
    }
    // sums are whole, so a sum exceeds u * total where it exceeds its whole part; a number outside [0, 1) takes an end
    __device__ u64 target_of(int r, u64 total) const {
        const double at = fmax(0.0, static_cast<double>(p.u[r])) * static_cast<double>(total);
        if (!(at < static_cast<double>(total))) return total - 1;
        const u64 t = static_cast<u64>(at);
        return t < total ? t : total - 1;
    }

    // ---- few candidates: those at or above `bound`; false if there are too many
    __device__ bool from_list(int r, float bound, int top_k, float top_p, float min_p, bool need_all) {
        __syncthreads();
        int n = 0;  // of this wave
        u64 all = 0;
        walk([&](const float (&x)[kVec], int i0) {
            uint32_t take = 0;
#pragma unroll
            for (int e = 0; e < kVec; ++e) take |= x[e] >= bound ? 1u << e : 0u;
            if (need_all) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) all += weight(x[e]);
            }
            if (__any(take != 0)) {
                const int c = __builtin_popcount(take);
                int upto = c;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int y = __shfl_up(upto, o);
                    upto += lane >= o ? y : 0;
                }
                int at = n + upto - c;
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if ((take >> e) & 1) {
                        if (at < kList) {
                            s.found.value[wave][at] = x[e];
                            s.found.index[wave][at] = i0 + e;
                        }
                        ++at;
                    }
                n += __shfl(upto, 63);
            }
        });
        if (need_all) all = block_sum(all);
        if (lane == 0) s.n[wave] = n;
        __syncthreads();
        int start = 0, total_n = 0;
        for (int i = 0; i < kWaves; ++i) {
            start += i < wave ? s.n[i] : 0;
            total_n += s.n[i];
        }
        if (total_n > kList) return false;
        for (int i = lane; i < n; i += 64) {
            const float v = s.found.value[wave][i];
            s.list.value[start + i] = v;
            s.list.index[start + i] = s.found.index[wave][i];
            s.list.weight[start + i] = weight(v);
        }
        __syncthreads();
        // every candidate counts what comes before it in the order
        const bool on = tid < total_n;
        const float v = on ? s.list.value[tid] : 0.0f;
        const u64 w = on ? s.list.weight[tid] : 0;
        int rank = 0;
        u64 before = 0;
        if (wave * 64 < total_n) {
            for (int j = 0; j < total_n; ++j) {
                const float vj = s.list.value[j];
                const bool ahead = vj > v || (vj == v && j < tid);
                rank += ahead;
                before += ahead ? s.list.weight[j] : 0;
            }
        }
        const bool in_k = on && (top_k <= 0 || rank < top_k);
        if (!need_all) all = block_sum(in_k ? w : 0);
        bool keep = in_k;
        if (top_p < 1.0f) keep = keep && static_cast<double>(before) < static_cast<double>(top_p) * static_cast<double>(all);
        if (min_p > 0.0f) keep = keep && static_cast<double>(w) >= static_cast<double>(min_p) * 0x1p44;
        keep = keep || (on && rank == 0);
        const u64 mine = keep ? w : 0;
        u64 sum = wave_scan(mine);
        __syncthreads();
        if (lane == 63) s.a[wave] = sum;
        __syncthreads();
        u64 total = 0;
        for (int i = 0; i < kWaves; ++i) {
            sum += i < wave ? s.a[i] : 0;
            total += s.a[i];
        }
        const u64 target = target_of(r, total);
        if (keep && sum > target && sum - mine <= target) put(r, s.list.index[tid], v, total);
        return true;
    }

    // ---- the number in the running sum over the vocabulary of what the cut keeps
    __device__ void from_cut(int r, float cut, u64 ties) {
        const u64 each = weight(cut);
        int t0 = 0, t1 = steps();
        u64 target = 0, total = 0, ties_left = ties;
        // the run of steps in which the sum is reached, first of the whole row, then inside that run
        for (int level = 0; level < 2; ++level) {
            const int per = (t1 - t0 + kWaves - 1) / kWaves;
            const int w0 = t0 + wave * per < t1 ? t0 + wave * per : t1, w1 = w0 + per < t1 ? w0 + per : t1;
            u64 above = 0, same = 0;
            steps_of(w0, w1, 1, [&](const float (&x)[kVec], int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (x[e] > cut) above += weight(x[e]);
                    same += x[e] == cut;
                }
            });
            above = wave_sum(above);
            same = wave_sum(same);
            __syncthreads();
            if (lane == 0) {
                s.a[wave] = above;
                s.b[wave] = same;
            }
            __syncthreads();
            if (level == 0) {
                u64 left = ties;
                for (int i = 0; i < kWaves; ++i) {
                    const u64 n = s.b[i] < left ? s.b[i] : left;
                    total += s.a[i] + n * each;
                    left -= n;
                }
                target = target_of(r, total);
            }
            int found = kWaves - 1;
            for (int i = 0; i < kWaves; ++i) {
                const u64 n = s.b[i] < ties_left ? s.b[i] : ties_left, sum = s.a[i] + n * each;
                if (sum > target) {
                    found = i;
                    break;
                }
                target -= sum;
                ties_left -= n;
            }
            const int f0 = t0 + found * per;
            t1 = f0 + per < t1 ? f0 + per : t1;
            t0 = f0;
        }
        if (wave != 0) return;
        for (int t = t0; t < t1; ++t) {
            bool done = false;
            step(t, [&](const float (&x)[kVec], int i0) {
                u64 above = 0, same = 0;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (x[e] > cut) above += weight(x[e]);
                    same += x[e] == cut;
                }
                const u64 same_to = wave_scan(same), same_before = same_to - same;
                const u64 taken = same_before >= ties_left ? 0 : (same < ties_left - same_before ? same : ties_left - same_before);
                const u64 mine = above + taken * each, upto = wave_scan(mine);
                const u64 sum = __shfl(upto, 63);
                if (sum > target) {
                    done = true;
                    if (upto > target && upto - mine <= target) {
                        u64 run = upto - mine, left = taken;
                        int at = -1;
                        float val = 0.0f;
#pragma unroll
                        for (int e = 0; e < kVec; ++e) {
                            u64 w = 0;
                            if (x[e] > cut) w = weight(x[e]);
                            else if (x[e] == cut && left > 0) { w = each; --left; }
                            run += w;
                            if (at < 0 && run > target) { at = i0 + e; val = x[e]; }
                        }
                        put(r, at, val, total);
                    }
                } else {
                    target -= sum;
                    const u64 n = __shfl(same_to, 63);
                    ties_left -= n < ties_left ? n : ties_left;
                }
            });
            if (done) return;
        }
    }

    __device__ void run(int r) {
        if (tid < 32) s.table[tid] = exp2(tid / 32.0);
        const float temp = p.temperature ? p.temperature[r] : 1.0f;
        const bool greedy = !(temp > 0.0f);
        const int top_k = p.top_k ? p.top_k[r] : 0;
        const float top_p = p.top_p ? p.top_p[r] : 1.0f, min_p = p.min_p ? p.min_p[r] : 0.0f;
        // ---- the maximum, and partial maxima of kSub places per thread; for the arg-max its first index, too
        float part[kSub];
#pragma unroll
        for (int i = 0; i < kSub; ++i) part[i] = -INFINITY;
        int where = 0x7fffffff;
        if (greedy) {
            steps_of(wave, steps(), kWaves, [&](const float (&x)[kVec], int i0) {
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (x[e] > part[0]) { part[0] = x[e]; where = i0 + e; }
            });
        } else {
            steps_of(wave, steps(), kWaves, [&](const float (&x)[kVec], int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) part[e % kSub] = fmaxf(part[e % kSub], x[e]);
            });
        }
        top = part[0];
#pragma unroll
        for (int i = 1; i < kSub; ++i) top = fmaxf(top, part[i]);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (lane == 0) s.a[wave] = __float_as_uint(top);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = fmaxf(top, __uint_as_float(static_cast<uint32_t>(s.a[i])));
        if (top == -INFINITY) {  // nothing to choose from
            if (tid == 0) {
                p.ids[r] = 0;
                if (p.logprobs) p.logprobs[r] = -INFINITY;
            }
            return;
        }
        if (greedy) {
            int first = part[0] == top ? where : 0x7fffffff;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) first = min(first, __shfl_xor(first, o));
            if (lane == 0) s.n[wave] = first;
            __syncthreads();
            for (int i = 0; i < kWaves; ++i) first = min(first, s.n[i]);
            if (tid == 0) {
                p.ids[r] = first;
                if (p.logprobs) p.logprobs[r] = 0.0f;
            }
            return;
        }
        a = 1.4426950408889634 / static_cast<double>(temp);
        const float reachable = static_cast<float>(kOctaves / a);
        low = top == INFINITY ? INFINITY : fmaxf(top - reachable, -3.402823466e38f);
        // ---- a bound that all that can be kept lies at or above
        float bound = -INFINITY;
        if (top_k > 0 && top_k <= kTopKList) {
            // the top_k-th largest partial maximum, to within a few parts in 10^5 of their range: every round tries 64 keys
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSub; ++i) s.maxima[tid * kSub + i] = key_of<ASRFE_DT_F32>(part[i]);
            __syncthreads();
            uint32_t mine[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) mine[i] = s.maxima[i * 64 + lane];
            uint32_t l = key_of<ASRFE_DT_F32>(-3.402823466e38f), h = key_of<ASRFE_DT_F32>(top);  // at least top_k at or above l?
            auto count = [&](uint32_t k) {
                int c = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) c += __builtin_popcountll(__ballot(mine[i] >= k));
                return c;
            };
            if (count(l) >= top_k) {
                while (l < h) {
                    const uint32_t mid = l + (h - l) / 2 + 1;
                    if (count(mid) >= top_k) l = mid;
                    else h = mid - 1;
                }
                bound = value_of<ASRFE_DT_F32>(l);
            }
        }
        // (top_p measures against all that top_k leaves: the list has to hold that, whatever min_p drops afterwards)
        const bool some_k = top_k > 0 && top_k < p.vocab;
        if (min_p > 0.0f && !(some_k && top_p < 1.0f)) {
            // l >= max + log2(min_p) / a, and a little below: the candidates' own weights decide
            const double edge = static_cast<double>(top) + log2(fmin(static_cast<double>(min_p), 1.0)) / a;
            if (top < INFINITY) bound = fmaxf(bound, static_cast<float>(edge - 1e-6 * (fabs(edge) + fabs(static_cast<double>(top))) - 1e-30));
        }
        if (bound > -INFINITY) {
            bound = fminf(bound, top);
            if (from_list(r, bound, top_k, top_p, min_p, top_p < 1.0f && !some_k)) return;
        }
        // ---- the general way
        float cut = low;   // without a filter all that has a weight is kept
        u64 ties = ~0ull >> 1, before = 0;
        u64 all = 0;
        if (some_k) {
            u64 n = 0;
            walk([&](const float (&x)[kVec], int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) n += x[e] >= -3.402823466e38f;
            });
            n = block_sum(n);
            if (n > static_cast<u64>(top_k)) {
                cut = reach<false>(static_cast<u64>(top_k), before);
                ties = static_cast<u64>(top_k) - before;
            }
        }
        if (top_p < 1.0f) {
            u64 n = 0, same = 0;
            walk([&](const float (&x)[kVec], int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (x[e] > cut) n += weight(x[e]);
                    same += x[e] == cut;
                }
            });
            all = block_sum(n);
            same = block_sum(same);
            all += (same < ties ? same : ties) * weight(cut);
            const double want = static_cast<double>(top_p) * static_cast<double>(all);
            u64 want_n = want > 0.0 ? static_cast<u64>(ceil(want)) : 1;
            want_n = want_n < 1 ? 1 : (want_n > all ? all : want_n);
            cut = reach<true>(want_n, before);
            const u64 each = weight(cut);
            ties = (want_n - before + each - 1) / each;
        }
        if (min_p > 0.0f) {
            // the least value whose weight is at least min_p
            uint32_t l = key_of<DT>(cut), h = key_of<DT>(top);
            const double need = static_cast<double>(min_p) * 0x1p44;
            while (l < h) {
                const uint32_t mid = l + (h - l) / 2;
                if (static_cast<double>(weight(value_of<DT>(mid))) >= need) h = mid;
                else l = mid + 1;
            }
            const float c = value_of<DT>(l);
            if (c > cut) {
                cut = c;
                ties = min_p > 1.0f ? 1 : ~0ull >> 1;
            }
        }
        from_cut(r, cut, ties);
    }
};

template <int DT, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(const SampleParams p) {
    __shared__ SampleLds<NT> s;
    const int r = blockIdx.x;
    if (p.token_num && r % p.rows_per >= p.token_num[r / p.rows_per]) {
        if (threadIdx.x == 0) {
            p.ids[r] = -1;
            if (p.logprobs) p.logprobs[r] = 0.0f;
        }
        return;
    }
    Sampler<DT, NT> sampler(p, s, r);
    sampler.run(r);
}

int32_t launch_sample(asrfe_ctx* ctx, const SampleParams& p, int dtype, hipStream_t s) {
    const dim3 grid(p.rows);
    // small vocabularies: eight rows of a compute unit at once instead of two
    const bool small = p.vocab <= 16384;
#define SAMPLE(DT)                                                                                 \
    do {                                                                                           \
        if (small) hipLaunchKernelGGL((sample_kernel<DT, 256>), grid, dim3(256), 0, s, p);         \
        else hipLaunchKernelGGL((sample_kernel<DT, 1024>), grid, dim3(1024), 0, s, p);             \
    } while (0)
    if (dtype == ASRFE_DT_F32) SAMPLE(ASRFE_DT_F32);
    else if (dtype == ASRFE_DT_F16) SAMPLE(ASRFE_DT_F16);
    else SAMPLE(ASRFE_DT_BF16);
#undef SAMPLE
    return launched(ctx, "sample_tokens");
}

}  // namespace asrfe
