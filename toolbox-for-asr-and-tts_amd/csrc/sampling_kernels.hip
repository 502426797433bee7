// Choice of a token per row of logits: temperature, top-k, top-p, min-p and one random number.
//
//   One workgroup per row (256 threads for small vocabularies, else 1024).  Weights w = 2^((l - max) log2(e) / T) are formed
//   in double precision (a table of 2^(j / 1024) and a polynomial: relative error below 1e-11; double FMAs issue at the
//   rate of single ones here) and summed as whole multiples of 2^-44, so a sum is the same in any order and atomics may form
//   it.  What is kept is a prefix of the order (falling logit, rising index), described by the value of its last element,
//   `cut`, and the number of elements of that value that belong to it, `ties`.
//
//   The row is read from memory once for its maximum and, from the caches, once or a few times more:
//     * few candidates (a small top_k, or min_p): the k-th largest of 4096 (2048) partial maxima is a lower bound of the k-th
//       largest logit; what is at or above it goes into a list in the LDS, in the order of the vocabulary, and every
//       filter is settled there by counting (256 entries at most; more take the way below);
//     * else a cut is found by histograms in the LDS, one a wave, first over the logarithm of the weight, then over the keys of
//       the values left in the bin where the cut lies, until one value is left (or few: they go into a list, too);
//     * the number is then looked up in the running sum over the vocabulary: per wave, per step of that wave, per lane.
//   A row's time is its compute unit's arithmetic (some 25 instructions a weight, 3 a maximum): 256 rows of 131072 16-bit logits
//   take 14 us for the arg-max (4.9 TB/s), 34 us under top_k, 47 us without a filter, 75 us under a top_p that keeps
//   thousands, 68 us each with filters of its own; one row of 8404 in 32 bits takes 10.5 us with all filters, 4.1 us for the
//   arg-max; 4000 rows of 8404 in 32 bits 68 us.
#include "elem.h"
#include "paged_device.h"

namespace asrfe {

typedef unsigned long long u64;
typedef u64 u64x2 __attribute__((ext_vector_type(2)));

constexpr int kList = 256;        // candidates the list path takes
// Largest top_k that tries it.  The bound is the top_k-th of the partial maxima, and some maxima hide a second value above it:
// with 2048 of them a list holds 216 values of a row in the mean under top_k = 200 (230 at most in 200 rows), 250 under 230,
// where one row in five finds it too short, 263 under 240.  Past it the general way takes its time: top_k = 200 and 201 of one
// row of 8404 in 32 bits 12.8 and 25.7 us, of 131072 in 16 bits 24.5 and 65.8 us, of 256 such rows 34 and 83 us.
constexpr int kTopKList = 200;
constexpr double kOctaves = 46.0; // weights below 2^-45 are zero in multiples of 2^-44

// an order-preserving whole number per value (16 bits for 16-bit logits); -0 and +0 have the same, kMinusZero + 1
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

// Sums over the lanes up to and with this one, by moves inside and between rows of 16 lanes (shuffles go through the LDS, six
// round trips each: one row of 8404 with all filters 12.6 us, this way 10.8 us).
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T moved(T v, T none) {  // `none` where no lane has a value for this one
    if constexpr (sizeof(T) == 8) {
        const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(v), CTRL, ROWS, 0xf, false));
        const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(none >> 32), static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false));
        return static_cast<u64>(hi) << 32 | lo;
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    }
}
template <class T, class Join>
__device__ __forceinline__ T wave_scan(T v, T none, Join&& join) {
    v = join(v, moved<0x111, 0xf>(v, none));  // from 1, 2, 4 and 8 lanes below in the row,
    v = join(v, moved<0x112, 0xf>(v, none));
    v = join(v, moved<0x114, 0xf>(v, none));
    v = join(v, moved<0x118, 0xf>(v, none));
    v = join(v, moved<0x142, 0xa>(v, none));  // from the last lane of the row below,
    return join(v, moved<0x143, 0xc>(v, none));  // and of the lower half
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
    return wave_scan(v, u64{0}, [](u64 x, u64 y) { return x + y; });
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    return static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ u64 wave_sum(u64 v) { return last_lane(wave_scan(v)); }

// 2^(44 + j / 1024), for weight()
struct Powers {
    double v[1024];
    constexpr Powers() : v() {
        for (int j = 0; j < 1024; ++j) {
            const double x = j * (0.6931471805599453 / 1024.0);  // e^x: 20 terms, the last below 1e-20
            double sum = 0.0;
            for (int i = 20; i >= 1; --i) sum = (1.0 + sum) * x / i;
            v[j] = (1.0 + sum) * 17592186044416.0;
        }
    }
};
__device__ constexpr Powers kPowers;

template <int NT>
struct SampleLds {
    static constexpr int kWaves = NT / 64;
    // A histogram of its own per wave, so that the mass a cut leaves to every wave's run of the vocabulary is known with the
    // cut.  Their bins of weights are 2^kBinBits / 1024 octaves wide.
    static constexpr int kBinBits = NT == 1024 ? 6 : 7, kBins = static_cast<int>(kOctaves * 1024) >> kBinBits;
    static constexpr int kNear = NT == 1024 ? 4096 : 2048;  // bins of the search for a bound
    double table[1024];  // 2^(44 + j / 1024)
    u64 a[kWaves], b[kWaves];
    union {
        u64 hist[kWaves * kBins];
        uint32_t near[kNear];
        struct {
            float value[kWaves][kList];
            int index[kWaves][kList];
        } found;
    };
    struct {
        struct alignas(16) {
            u64 order;   // key, then the place in the list from behind: unique, larger ones come first
            u64 weight;
        } entry[kList];
        float value[kList];
        int index[kList], rank[kList];
        u64 before[kList];
    } list;
    u64 res[4];
    int n[kWaves];
    int total;
};

// (a function's own variable, so that every access is known to be one of the LDS: through a reference kept in an object
// they would be flat ones)
template <int NT>
__device__ __forceinline__ SampleLds<NT>& sample_lds() {
    __shared__ SampleLds<NT> s;
    return s;
}

template <int DT, int NT>
struct Sampler {
    static constexpr int kWaves = NT / 64;
    static constexpr int kBins = SampleLds<NT>::kBins, kNear = SampleLds<NT>::kNear;
    static constexpr int kVec = DT == ASRFE_DT_F32 ? 4 : 8;
    static constexpr int kSub = NT == 1024 ? 4 : 8;  // partial maxima of a thread
    static constexpr uint32_t kMinusZero = DT == ASRFE_DT_F32 ? 0x7fffffffu : 0x7fffu;

    const SampleParams& p;
    const int tid, lane, wave;
    typedef __attribute__((address_space(1))) const char Global;  // (flat loads would wait for every access of the LDS, and it for them)
    Global* row;
    int lead, last, n_steps;   // elements of the first 16-byte piece before the row, last piece, steps of 64 pieces
    bool flat;                 // all that counts has the same logit, one without a scale (+inf, or the least there is)
    float top, low;            // largest logit, least logit with a weight
    double a, a_units;         // log2(e) / T, and 1024 times as much, for weight()

    __device__ __forceinline__ Sampler(const SampleParams& p_, int r)
        : p(p_), tid(threadIdx.x), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), flat(false) {
        constexpr int kSize = DT == ASRFE_DT_F32 ? 4 : 2;
        row = (Global*)p.logits + static_cast<int64_t>(r) * p.ld * kSize;
        lead = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / kSize;
        row -= lead * kSize;
        last = (lead + p.vocab - 1) / kVec;
        n_steps = last / 64 + 1;
    }

    // The row in steps of 64 aligned pieces of 16 bytes.  The first and the last piece may hold elements that are not the row's (a
    // piece with one of the row's lies inside its allocation's granule), and lanes behind the last piece read that one again:
    // at() makes them all NaN, for which no comparison holds, and which has no weight.  Loads take no branch, so they stay in
    // flight while other pieces are worked on.
    __device__ __forceinline__ int steps() const { return n_steps; }
    __device__ __forceinline__ int first_of(int t) const { return (t * 64 + lane) * kVec - lead; }  // this lane's first element
    __device__ __forceinline__ u32x4 load(int t) const {
        const uint32_t piece = static_cast<uint32_t>(min(t * 64 + lane, last));
        return *reinterpret_cast<__attribute__((address_space(1))) const u32x4*>(row + piece * 16);
    }
    __device__ __forceinline__ void at(int t, const u32x4 w, float (&x)[kVec]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == ASRFE_DT_F32) x[i] = __uint_as_float(w[i]);
            else unpack_elem2<DT == ASRFE_DT_F16>(w[i], x[2 * i], x[2 * i + 1]);
        }
        if (t == 0 || t == n_steps - 1) {
            const int i0 = first_of(t);
#pragma unroll
            for (int e = 0; e < kVec; ++e) x[e] = static_cast<unsigned>(i0 + e) < static_cast<unsigned>(p.vocab) ? x[e] : __builtin_nanf("");
        }
    }
    // f(x, i0, t) for the n steps t0, t0 + by, ..., from the one of number `from` around to the one before it: this lane's
    // elements i0, i0 + 1, ...  AHEAD loads are in flight (each in registers of its own: moving them would wait for them).
    template <int AHEAD, class F>
    __device__ __forceinline__ void steps_of(int t0, int n, int by, int from, F&& f) const {
        if (n <= 0) return;
        u32x4 w[AHEAD];
        int next = from, now = from;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            w[j] = load(t0 + next * by);
            next = next + 1 < n ? next + 1 : 0;
        }
        for (int k = 0; k < n; k += AHEAD) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (k + j >= n) break;
                float x[kVec];
                const int t = t0 + now * by;
                at(t, w[j], x);
                w[j] = load(t0 + next * by);
                f(x, first_of(t), t);
                now = now + 1 < n ? now + 1 : 0;
                next = next + 1 < n ? next + 1 : 0;
            }
        }
    }
    // this wave's run of steps: runs follow each other in the order of the vocabulary
    __device__ __forceinline__ int run_of(int w) const {
        const int per = (steps() + kWaves - 1) / kWaves, t = w * per;
        return t < steps() ? t : steps();
    }
    template <int AHEAD, class F>
    __device__ __forceinline__ void walk(F&& f) const {
        // (every wave begins elsewhere in its run: all at the same distance from their runs' starts ask the same few memory
        // channels at once: 256 rows of 131072 in 32 bits under top_k 59 us, this way 53 us)
        const int t0 = run_of(wave), n = run_of(wave + 1) - t0;
        steps_of<AHEAD>(t0, n, 1, n > 0 ? wave % n : 0, f);
    }

    // Weight in multiples of 2^-44, with kOffset added (a sum over n values takes it off n times; whole numbers may wrap).
    // Below `low`, and for NaN, the median of three takes `low`, whose weight is zero.
    static constexpr u64 kOffset = 0x4330000000000000ull;  // bits of 2^52, whose unit is one
    __device__ __forceinline__ u64 weight_bits(float v) const {
        int k;
        return weight_bits(v, k);
    }
    // and k, its logarithm in units of 1 / 1024 octave (zero or below)
    static constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: a sum's low bits are the nearest whole number
    __device__ __forceinline__ double below_top(float v) const {
        return static_cast<double>(__builtin_amdgcn_fmed3f(v, low, top)) - static_cast<double>(top);
    }
    __device__ __forceinline__ int log_weight(float v) const { return static_cast<int>(__builtin_bit_cast(u64, __builtin_fma(below_top(v), a_units, kMagic))); }
    __device__ __forceinline__ u64 weight_bits(float v, int& k) const {
        const double x = below_top(v), d = __builtin_fma(x, a_units, kMagic);
        k = static_cast<int>(__builtin_bit_cast(u64, d));
        const double f = __builtin_fma(x, a_units, kMagic - d);  // |f| <= 1 / 2, in units of 1 / 1024
        // 2^(f / 1024) = 1 + f ln 2 / 1024 + (f ln 2 / 1024)^2 / 2: the next term is below 7e-12.  (A table of 32 entries, which
        // meets no bank conflicts, and two terms more: 5 % slower.)
        const double e = f * __builtin_fma(f, 2.2909787910375658e-07, 0.0006769015435155716);
        const u64 tab = __builtin_bit_cast(u64, sample_lds<NT>().table[k & 1023]);  // 2^44 times the power
        // (its exponent moved by k / 1024)
        const uint32_t high = static_cast<uint32_t>(tab >> 32) + (static_cast<uint32_t>(k & ~1023) << 10);
        const double w = __builtin_bit_cast(double, static_cast<u64>(high) << 32 | static_cast<uint32_t>(tab));
        return __builtin_bit_cast(u64, __builtin_fma(w, e, w + 0x1p52));
    }
    __device__ __forceinline__ u64 weight(float v) const { return weight_bits(v) - kOffset; }

    __device__ __forceinline__ u64 block_sum(u64 v) {
        SampleLds<NT>& s = sample_lds<NT>();
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) s.a[wave] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) t += s.a[i];
        return t;
    }

    // The bin at which a sum over bins that starts at `before` reaches `want`, in s.res[1] (left as it is where none does), and
    // the sum before it in `before`.  Every thread takes a run of N / NT bins, each the sum of ROWS.
    template <int ROWS, int N, class T>
    __device__ __forceinline__ void find_bin(const T* hist, u64 want, u64& before) {
        SampleLds<NT>& s = sample_lds<NT>();
        constexpr int kPer = (N + NT - 1) / NT;
        u64 bin[kPer], mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            bin[i] = 0;
            const int at = tid * kPer + i;
            if (at < N) {
#pragma unroll
                for (int j = 0; j < ROWS; ++j) bin[i] += hist[j * N + at];
            }
            mine += bin[i];
        }
        u64 sum = wave_scan(mine);
        if (lane == 63) s.b[wave] = sum;
        __syncthreads();
        for (int i = 0; i < wave; ++i) sum += s.b[i];
        sum += before - mine;
        if (sum < want && want <= sum + mine) {
            int b = 0;
#pragma unroll
            for (int i = 0; i + 1 < kPer; ++i)
                if (b == i && sum + bin[i] < want) {
                    sum += bin[i];
                    ++b;
                }
            s.res[0] = sum;
            s.res[1] = tid * kPer + b;
        }
        __syncthreads();
        before = s.res[0];
    }

    // Finds the value at which a running sum over falling values first reaches `want` (1 <= want <= the sum of all):
    // the sum over larger values is below `want`, the sum with that value's elements is not.  MASS: sums of weights, else of
    // elements.  want = 0: `share` of the sum of all, rounded up.  `settle(from, all)` may end the search when a bin of values
    // not below `from` is known to hold the end: it says whether it did (all: zero, or that sum).  mine: what this wave's
    // run of the vocabulary has above the value, and of it.
    struct Mine {
        u64 above, same;
    };
    template <bool MASS, class F>
    __device__ __forceinline__ float reach(u64& want, float share, u64& before, Mine& mine_run, bool& settled, F&& settle) {
        SampleLds<NT>& s = sample_lds<NT>();
        const float least = MASS ? low : -3.402823466e38f;
        const float span = static_cast<float>(kOctaves / a);  // logits per kOctaves octaves of weight
        const float scale = fminf(static_cast<float>(kBins) / span, 3e38f);
        auto bin1 = [&](float v) {
            if (MASS) return -log_weight(v) >> SampleLds<NT>::kBinBits;
            const float d = fmaxf((top - v) * scale, 0.0f);  // (0 * inf: the top itself)
            return static_cast<int>(fminf(d, kBins - 1.0f));
        };
        before = 0;
        u64 all = 0;
        float from = least, to = top;  // the value lies among these
        uint32_t lo = 0, hi = 0;       // and, after the first pass, among these keys
        int shift = -1;
        for (;;) {
            __syncthreads();
            for (int i = tid; i < kWaves * kBins; i += NT) s.hist[i] = 0;
            __syncthreads();
            if (shift < 0) {
                walk<2>([&](const float (&x)[kVec], int, int) {
                    u64 w[kVec];
                    int at[kVec];
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        if (MASS) {
                            w[e] = weight_bits(x[e], at[e]) - kOffset;
                            at[e] = -at[e] >> SampleLds<NT>::kBinBits;
                        } else {
                            w[e] = x[e] >= least;
                            at[e] = bin1(x[e]);
                        }
                        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int e = 0; e < kVec; ++e)
                        if (MASS ? at[e] < kBins : w[e] != 0) atomicAdd(&s.hist[wave * kBins + at[e]], w[e]);
                });
            } else {
                // few lanes have one and fewer have two: one of each lane at a time
                walk<2>([&](const float (&x)[kVec], int, int) {
                    uint32_t take = 0;
#pragma unroll
                    for (int e = 0; e < kVec; ++e) take |= x[e] >= from && x[e] <= to ? 1u << e : 0u;
                    while (__any(take != 0)) {
                        const int e = __builtin_ctz(take | 1u << kVec);
                        float v = x[0];
#pragma unroll
                        for (int i = 1; i < kVec; ++i) v = e == i ? x[i] : v;
                        if (take != 0) atomicAdd(&s.hist[wave * kBins + ((hi - key_of<DT>(v)) >> shift)], MASS ? weight(v) : u64{1});
                        take &= take - 1;
                    }
                });
            }
            __syncthreads();
            if (want == 0) {
                u64 mine = 0;
                for (int i = tid; i < kWaves * kBins; i += NT) mine += s.hist[i];
                all = block_sum(mine);
                const double x = ceil(static_cast<double>(share) * static_cast<double>(all));
                want = x >= 1.0 ? static_cast<u64>(x) : 1;
                want = want > all ? all : want;
            }
            find_bin<kWaves, kBins>(s.hist, want, before);
            const int b = static_cast<int>(s.res[1]);
            if (MASS) {
                u64 mine = 0;
                for (int i = lane; i < b; i += 64) mine += s.hist[wave * kBins + i];
                mine_run.above += wave_sum(mine);
                mine_run.same = s.hist[wave * kBins + b];
            }
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
            // No element has the key of -0.  As the upper end it would let zeros in, whose key lies above it: their place in the
            // next histogram would be far outside of it.  (The bin holds an element, so a key below remains.)
            if (hi == kMinusZero) --hi;
            from = value_of<DT>(lo);
            if (shift < 0 && settle(from, all)) {
                settled = true;
                return from;
            }
            if (lo >= hi) return value_of<DT>(hi);
            to = value_of<DT>(hi);
            shift = 0;
            while (((hi - lo) >> shift) >= static_cast<uint32_t>(kBins)) ++shift;
        }
    }

    // id and log-probability: v its logit, total the kept weight
    __device__ __forceinline__ void put(int r, int id, float v, u64 total) const {
        p.ids[r] = id;
        if (p.logprobs) {
            const double t = flat ? 0.0 : (static_cast<double>(v) - static_cast<double>(top)) * a;
            p.logprobs[r] = static_cast<float>(t * 0.6931471805599453 - log(static_cast<double>(total) * 0x1p-44));
        }
    }
    // sums are whole, so a sum exceeds u * total where it exceeds its whole part; a number outside [0, 1) takes an end
    __device__ __forceinline__ u64 target_of(int r, u64 total) const {
        const double at = fmax(0.0, static_cast<double>(p.u[r])) * static_cast<double>(total);
        if (!(at < static_cast<double>(total))) return total - 1;
        const u64 t = static_cast<u64>(at);
        return t < total ? t : total - 1;
    }

    // ---- few candidates: those at or above `bound`; false if there are too many.  top_p is measured against `all`, or, where
    // that is zero, against what top_k leaves.
    __device__ __forceinline__ bool from_list(int r, float bound, int top_k, float top_p, float min_p, u64 all) {
        SampleLds<NT>& s = sample_lds<NT>();
        __syncthreads();
        int n = 0, early = 0;  // of this wave; those found before its run began anew at its first step
        const int first_step = run_of(wave);
        walk<3>([&](const float (&x)[kVec], int i0, int t) {
            if (t == first_step) early = n;
            u64 who[kVec], any = 0;  // the lanes whose element e is one
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                who[e] = __ballot(x[e] >= bound);
                any |= who[e];
            }
            if (any != 0) {
                int at = n;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    at = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who[e] >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who[e]), at));
                    n += __builtin_popcountll(who[e]);
                }
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (x[e] >= bound) {
                        if (at < kList) {
                            s.found.value[wave][at] = x[e];
                            s.found.index[wave][at] = i0 + e;
                        }
                        ++at;
                    }
            }
        });
        if (lane == 0) s.n[wave] = n;
        __syncthreads();
        int start = 0, total_n = 0;
        for (int i = 0; i < kWaves; ++i) {
            start += i < wave ? s.n[i] : 0;
            total_n += s.n[i];
        }
        if (total_n > kList) return false;
        for (int i = lane; i < n; i += 64) {  // (what was found early lies behind the rest in the order of the vocabulary)
            const float v = s.found.value[wave][i];
            const int at = start + (i < early ? i + n - early : i - early);
            s.list.value[at] = v;
            s.list.index[at] = s.found.index[wave][i];
            s.list.entry[at].order = static_cast<u64>(key_of<ASRFE_DT_F32>(v)) << 32 | static_cast<uint32_t>(kList - at);
            s.list.entry[at].weight = weight(v);
            s.list.rank[at] = 0;
            s.list.before[at] = 0;
        }
        __syncthreads();
        // every candidate counts what comes before it in the order
        const bool on = tid < total_n;
        const float v = on ? s.list.value[tid] : 0.0f;
        const u64 w = on ? s.list.entry[tid].weight : 0;
        // (64 candidates a wave, and the list cut among the waves that have the same ones)
        const int blocks = total_n <= 64 ? 1 : total_n <= 128 ? 2 : 4, cuts = kWaves / blocks, per = (total_n + cuts - 1) / cuts;
        {
            const int i = wave % blocks * 64 + lane, j0 = wave / blocks * per, j1 = min(total_n, j0 + per);
            const u64 order = s.list.entry[i].order;  // (behind the end: what is there, for nobody)
            int rank = 0;
            u64 before = 0;
#pragma unroll 8
            for (int j = j0; j < j1; ++j) {
                const u64x2 at = *reinterpret_cast<const u64x2*>(&s.list.entry[j]);
                const bool ahead = at[0] > order;
                rank += ahead;
                before += ahead ? at[1] : 0;
            }
            if (i < total_n && rank) {
                atomicAdd(&s.list.rank[i], rank);
                atomicAdd(&s.list.before[i], before);
            }
        }
        __syncthreads();
        const int rank = on ? s.list.rank[tid] : 0;
        const u64 before = on ? s.list.before[tid] : 0;
        const bool in_k = on && (top_k <= 0 || rank < top_k);
        if (all == 0) all = block_sum(in_k ? w : 0);
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

    // ---- the number in the running sum over the vocabulary of what the cut keeps; each: the weight at the cut
    __device__ __forceinline__ void from_cut(int r, float cut, u64 ties, u64 each, const Mine& mine_run, bool known) {
        SampleLds<NT>& s = sample_lds<NT>();
        int t0 = 0, t1 = steps();
        u64 target = 0, total = 0, ties_left = ties;
        // the run of steps in which the sum is reached, first of the whole row, then inside that run
        for (int level = 0; level < 2; ++level) {
            const int per = (t1 - t0 + kWaves - 1) / kWaves;
            const int w0 = t0 + wave * per < t1 ? t0 + wave * per : t1, w1 = w0 + per < t1 ? w0 + per : t1;
            u64 above = mine_run.above, same = mine_run.same;
            if (level > 0 || !known) {
                above = 0;
                int equal = 0;
                steps_of<2>(w0, w1 - w0, 1, w1 > w0 ? wave % (w1 - w0) : 0, [&](const float (&x)[kVec], int, int) {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        above += weight_bits(x[e] > cut ? x[e] : low);
                        equal += x[e] == cut;
                        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
                });
                above = wave_sum(above - kOffset * static_cast<u64>((w1 - w0) * kVec));
                same = wave_sum(static_cast<u64>(equal));
            }
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
            float x[kVec];
            at(t, load(t), x);
            const int i0 = first_of(t);
            {
                u64 above = 0, same = 0;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    above += weight_bits(x[e] > cut ? x[e] : low);
                    same += x[e] == cut;
                    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
                above -= kOffset * kVec;
                const u64 same_to = wave_scan(same), same_before = same_to - same;
                const u64 taken = same_before >= ties_left ? 0 : (same < ties_left - same_before ? same : ties_left - same_before);
                const u64 mine = above + taken * each, upto = wave_scan(mine);
                const u64 sum = last_lane(upto);
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
                    const u64 n = last_lane(same_to);
                    ties_left -= n < ties_left ? n : ties_left;
                }
            }
            if (done) return;
        }
    }

    __device__ __forceinline__ void run(int r) {
        SampleLds<NT>& s = sample_lds<NT>();
        const float given = p.temperature ? p.temperature[r] : 1.0f, temp = fminf(given, 1e30f);  // (as documented; only logits past 1e20 would see a difference)
        const bool greedy = !(given > 0.0f);  // (NaN, too)
        double power[1024 / NT];  // on their way while the maximum is found
#pragma unroll
        for (int i = 0; i < 1024 / NT; ++i) power[i] = kPowers.v[i * NT + tid];
        const int top_k = p.top_k ? p.top_k[r] : 0;
        const float top_p = p.top_p ? p.top_p[r] : 1.0f, min_p = p.min_p ? p.min_p[r] : 0.0f;
        // ---- the maximum, and partial maxima of kSub places per thread; for the arg-max its first index, too
        float part[kSub];
#pragma unroll
        for (int i = 0; i < kSub; ++i) part[i] = -INFINITY;
        int where = 0x7fffffff;
        if (greedy) {
            steps_of<4>(wave, (steps() - wave + kWaves - 1) / kWaves, kWaves, 0, [&](const float (&x)[kVec], int i0, int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const bool up = x[e] > part[0];
                    part[0] = up ? x[e] : part[0];
                    where = up ? i0 + e : where;
                }
            });
        } else {
            steps_of<4>(wave, (steps() - wave + kWaves - 1) / kWaves, kWaves, 0, [&](const float (&x)[kVec], int, int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) part[e % kSub] = x[e] > part[e % kSub] ? x[e] : part[e % kSub];
                if constexpr (kVec < kSub) {  // the other half's turn
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        const float y = part[e];
                        part[e] = part[e + kVec];
                        part[e + kVec] = y;
                    }
                }
            });
        }
#pragma unroll
        for (int i = 0; i < 1024 / NT; ++i) s.table[i * NT + tid] = power[i];
        top = part[0];
#pragma unroll
        for (int i = 1; i < kSub; ++i) top = fmaxf(top, part[i]);
        top = wave_scan(top, -INFINITY, [](float x, float y) { return fmaxf(x, y); });
        top = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), 63));
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
            first = __builtin_amdgcn_readlane(wave_scan(first, 0x7fffffff, [](int x, int y) { return min(x, y); }), 63);
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
        // far enough below the top for no weight even after its rounding, and below the top in any case
        const uint32_t tb = __float_as_uint(top);
        const float below = __uint_as_float(tb == 0 || tb == 0x80000000u ? 0x80000001u : (tb & 0x80000000u) ? tb + 1 : tb - 1);
        low = fminf(top - static_cast<float>(2.0 * kOctaves / a), below);
        // (where logits are so large that nothing lies between `low` and the top, a power the exponent can hold will do)
        a_units = 1024.0 * fmin(a, 4.0 * kOctaves / (static_cast<double>(top) - static_cast<double>(low)));
        float cut;
        u64 ties = ~0ull >> 1, each = 0;
        Mine mine{};
        bool known = false;  // `mine` is
        const bool some_k = top_k > 0 && top_k < p.vocab;
        if (low < -3.402823466e38f || top == INFINITY) {
            // a share by number, from the lowest index
            u64 n = 0;
            walk<2>([&](const float (&x)[kVec], int, int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) n += x[e] == top;
            });
            n = block_sum(n);
            if (some_k && n > static_cast<u64>(top_k)) n = static_cast<u64>(top_k);
            if (top_p < 1.0f) n = static_cast<u64>(fmax(1.0, ceil(static_cast<double>(top_p) * static_cast<double>(n))));
            cut = top;
            ties = min_p > 1.0f ? 1 : n;
            each = 1ull << 44;
            flat = true;
            top = 0.0f;  // (for the weights of what is not chosen: none)
            low = -1.0f;
            a_units = 1024.0 * 2.0 * kOctaves;
        } else if (!filtered(r, top_k, top_p, min_p, part, cut, ties, each, mine, known)) {
            return;  // chosen from a list
        }
        from_cut(r, cut, ties, each, mine, known);
    }

    // The cut of the three filters; false if the token was chosen from a list of candidates instead.
    __device__ __forceinline__ bool filtered(int r, int top_k, float top_p, float min_p, const float (&part)[kSub], float& cut, u64& ties, u64& each,
                                             Mine& mine, bool& known) {
        SampleLds<NT>& s = sample_lds<NT>();
        const bool some_k = top_k > 0 && top_k < p.vocab;
        u64 before = 0;
        // ---- a bound that all that can be kept lies at or above
        float bound = -INFINITY;
        if (top_k > 0 && top_k <= kTopKList) {
            // The top_k-th largest partial maximum, or a little below it: by number, over the distance from the top, in
            // bins of a hundredth of it or so (its upper bits, from 2^-16 on).  d < e is l > top - e, exactly: e has few bits,
            // and roundings keep the order.  (Bins reach down to 2^16.)
            constexpr int kFine = 23 - (kNear == 4096 ? 7 : 6);
            constexpr uint32_t kLeast = 111u << 23;  // 2^-16
            for (int i = tid; i < kNear; i += NT) s.near[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
                const uint32_t d = __float_as_uint(fmaxf(top - part[i], 0.0f)), b = d < kLeast ? 0 : (d - kLeast) >> kFine;
                if (b < static_cast<uint32_t>(kNear) && part[i] >= -3.402823466e38f) atomicAdd(&s.near[b], 1u);
            }
            if (tid == 0) s.res[1] = kNear;
            __syncthreads();
            u64 sum = 0;
            find_bin<1, kNear>(s.near, static_cast<u64>(top_k), sum);
            const uint32_t b = static_cast<uint32_t>(s.res[1]);
            if (b < static_cast<uint32_t>(kNear)) bound = fmaxf(top - __uint_as_float(kLeast + ((b + 1) << kFine)), -3.402823466e38f);
            // fewer than top_k are so near (a mask of -inf or of the type's least value hides the others): they may be all
            // that has a weight
            else if (a * 65536.0 >= 2.0 * kOctaves) bound = fmaxf(top - 65536.0f, -3.402823466e38f);
        }
        // (top_p measures against all that top_k leaves: the list has to hold that, whatever min_p drops afterwards)
        if (min_p > 0.0f && !(some_k && top_p < 1.0f)) {
            // l >= max + log2(min_p) / a, and a little below: the candidates' own weights decide
            const double edge = static_cast<double>(top) + log2(fmin(static_cast<double>(min_p), 1.0)) / a;
            bound = fmaxf(bound, static_cast<float>(edge - 1e-6 * (fabs(edge) + fabs(static_cast<double>(top))) - 1e-30));
        }
        // (top_p alone measures against all of the row, whose sum comes with a histogram: then the list has its turn behind that)
        bool few = bound > -INFINITY && (some_k || !(top_p < 1.0f));
        if (few && !(top_k > 0 && top_k <= kTopKList)) {  // (where the partial maxima alone are too many, so are the values)
            int many = 0;
#pragma unroll
            for (int i = 0; i < kSub; ++i) many += part[i] >= bound;
            few = block_sum(static_cast<u64>(many)) <= kList;
        }
        bound = fminf(bound, top);
        if (few && from_list(r, bound, top_k, top_p, min_p, 0)) return false;
        float most[kSub / 4];
#pragma unroll
        for (int i = 0; i < kSub / 4; ++i) most[i] = fmaxf(fmaxf(part[4 * i], part[4 * i + 1]), fmaxf(part[4 * i + 2], part[4 * i + 3]));
        // ---- the general way
        cut = low;  // without a filter all that has a weight is kept
        if (some_k) {
            u64 n = 0;
            walk<2>([&](const float (&x)[kVec], int, int) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) n += x[e] >= -3.402823466e38f;
            });
            n = block_sum(n);
            if (n > static_cast<u64>(top_k)) {
                u64 want = static_cast<u64>(top_k);
                bool never = false;
                Mine none{};
                cut = reach<false>(want, 0.0f, before, none, never, [](float, u64) { return false; });
                ties = want - before;
            }
        }
        if (top_p < 1.0f) {
            u64 want = 0, left = 0;
            if (some_k) {  // a share of what top_k leaves
                u64 n = 0, same = 0;
                walk<2>([&](const float (&x)[kVec], int, int) {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        const u64 w = weight(x[e]);
                        n += x[e] > cut ? w : 0;
                        same += x[e] == cut;
                    }
                });
                n = block_sum(n);
                same = block_sum(same);
                n += (same < ties ? same : ties) * weight(cut);
                const double x = ceil(static_cast<double>(top_p) * static_cast<double>(n));
                want = x >= 1.0 ? static_cast<u64>(x) : 1;
                want = want > n ? n : want;
                left = n;
            }
            bool settled = false;
            cut = reach<true>(want, top_p, before, mine, settled, [&](float least, u64 all) {
                const float from = fmaxf(least, bound);
                // Few values go into a list.  How many there are is not known, but most of few are maxima of a thread: 256 are
                // 226 of 1024 maxima, or 201 of 512, where they lie anywhere.
                int many = 0;
#pragma unroll
                for (int i = 0; i < kSub / 4; ++i) many += most[i] >= from;
                return block_sum(static_cast<u64>(many)) <= kList / 8 * 7 && from_list(r, from, top_k, top_p, min_p, some_k ? left : all);
            });
            if (settled) return false;
            each = weight(cut);
            ties = (want - before + each - 1) / each;
            mine.same /= each;
            known = true;
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
            if (c > cut || min_p > 1.0f) {  // (above one: only the first of the order stays, also of ties that are the cut already)
                known = false;
                cut = c;
                ties = min_p > 1.0f ? 1 : ~0ull >> 1;
            }
        }
        each = weight(cut);
        return true;
    }
};

template <int DT, int NT>
__global__ __launch_bounds__(NT, 4) void sample_kernel(const SampleParams p) {
    const int r = blockIdx.x;
    if (p.token_num && r % p.rows_per >= p.token_num[r / p.rows_per]) {
        if (threadIdx.x == 0) {
            p.ids[r] = -1;
            if (p.logprobs) p.logprobs[r] = 0.0f;
        }
        return;
    }
    Sampler<DT, NT>(p, r).run(r);
}

int32_t launch_sample(asrfe_ctx* ctx, const SampleParams& p, int dtype, hipStream_t s) {
    const dim3 grid(p.rows);
    // Four rows of a compute unit at once where there are more rows than compute units, one row of 1024 threads else (16-bit
    // logits, rows of mixed filters, 256 against 1024 threads: 4000 rows of 8404 75 and 198 us, 1000 of 65536 93 and 102 us;
    // 300 of 32768 40 and 37 us, 300 of 65536 59 and 49 us: the second round of a few rows of a large vocabulary costs more
    // than it gives).
    const bool small = p.rows > ctx->num_cus && (p.vocab <= 32768 || p.rows >= 3 * ctx->num_cus);
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
