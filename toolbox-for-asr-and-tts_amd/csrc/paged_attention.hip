// Attention of new rows over a paged cache, on the matrix cores.
//
//   o_i = sum_j p_ij v_j, p_i = softmax over the visible j of scale * q_i . k_j.
//
//   Rows.  The query heads that share a cache head read the same keys, so the rows of a product are (token, head of the
//   group) pairs: row r of a sequence is token r / group, head r % group.  A workgroup takes a tile of 128 rows (prompts:
//   four waves with 32 rows each share every key tile) or of 16 or 32 (single tokens, short chunks, and all calls of little
//   work: every wave has the same rows and key tiles of its own, so that four tiles are in flight and no barrier stands
//   between them).
//
//   Keys.  One pass with a running maximum and sum.  Scores are formed transposed, S^T = K Q^T (v_mfma_f32_32x32x16), so a
//   lane holds the scores of one row; the weights are then already laid out as the operand of O^T = V^T P^T, V being read
//   transposed from the LDS.  Tiles arrive by 16-byte global -> LDS loads (16-bit caches) with the bank swizzle applied to
//   the source address, or through registers, where e4m3 codes become 16-bit values (their scales are powers of two: exact
//   but for fp16 below 2^-14 and past 65504, see dequantise8).  A tile is made of 16-position pieces, each inside one page,
//   so pages may end anywhere in a tile.
//
//   Masks.  Only the tiles a mask's edge crosses (the causal diagonal, either end of the window, the end of the sequence,
//   a page that does not exist) look at positions; there, too, values that are infinite or NaN are kept out of the product
//   (0 * inf) and added to the rows that see them.  Other tiles multiply them as they are; where a weight that became zero made
//   NaN of one, the tiles are gone through again, all of them as edge tiles.  Tiles no row of the workgroup sees are not
//   loaded: a window's walk skips from the sinks to it.
//
//   Long caches with few rows are cut along the keys into parts, whose sums a second kernel joins.
//
//   Scores, maxima, sums and outputs are fp32.  The weights are rounded to the 16 bits of the product's other operand (the sum they
//   are divided by takes them before that): half a step of each weight, at random, so an output is off by at most as much
//   as its own rounding adds (of sum p |v|), and less the more weights there are.  See Raised for small ones.
#include <algorithm>

#include "lds_dma.h"
#include "paged_device.h"

namespace asrfe {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) int32_t* const_i32;

// The same address in scalar registers, for a value that is the same in every lane.  (In the global address space: loads
// through a pointer made of a number would be flat ones, which the LDS counter waits for, too.)
typedef const __attribute__((address_space(1))) char* global_ptr;
__device__ __forceinline__ global_ptr uniform(const char* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
    return (global_ptr)(static_cast<uint64_t>(hi) << 32 | lo);
}

// Two results in 16 bits.  A mean of fp16 values can leave their range by its rounding errors only: it stays inside;
// infinities and NaN stay what they are.
template <bool F16>
__device__ __forceinline__ uint32_t pack_result(float a, float b) {
    auto in = [](float v) { return F16 && __builtin_fabsf(v) < INFINITY ? __builtin_amdgcn_fmed3f(v, -65504.0f, 65504.0f) : v; };
    return pack_elem2<F16>(in(a), in(b));
}

template <class T>
__device__ __forceinline__ __attribute__((address_space(3))) T* lds(uint32_t addr) {
    return (__attribute__((address_space(3))) T*)addr;
}

// Weights are 2^(score - reference), scores in base 2.  The reference is the largest score seen less kRaise, brought up to
// that when a tile exceeds it by more than kLag: a weight is at most 2^(kLag + kRaise), the largest one seen at least 2^kRaise.
// fp16 has little range below one: raised by 2^9, weights down to 2^-23 of the largest keep all bits of their rounding and
// those below 2^-34 become zero in the product (without it 2^-14 and 2^-25, and such weights of 131072 positions can hold
// 0.4 % of the sum).  Six and nine cost nothing; with four and eleven prompts under a window take 2 % longer.
template <bool F16>
struct Raised {
    static constexpr float kLag = F16 ? 6.0f : 8.0f, kRaise = F16 ? 9.0f : 0.0f;
};

// What brings sums from one reference to another.  Never zero: an infinite sum stays infinite.  (2^-149, the least there is, of a
// finite one: at most 5e-7, from values at the end of bf16's range; 2^-126 would leave 4.)
__device__ __forceinline__ float factor(float from, float to) { return fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-149f); }

// 1 / a sum of weights; 0 where there were none, NaN where a score was
__device__ __forceinline__ float inverse(float sum) { return sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum); }

// Workgroups are dealt round-robin over the 8 XCDs: a contiguous range for each, so that those that share keys share an L2.
__device__ __forceinline__ int xcd_contiguous(int bid, int n) {
    const int xcd = bid & 7, q = n >> 3, r = n & 7;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
}

// Place k of n -> the k-th of a sequence that takes every s-th place first, then the ones behind those, ...
__device__ __forceinline__ int strided(int k, int n, int s) {
    const int q = n / s, r = n % s, big = r * (q + 1);
    return k < big ? k % (q + 1) * s + k / (q + 1) : (k - big) % q * s + r + (k - big) / q;
}

// bytes of 135 or more, a scale of 2^8 or more, which can lead out of fp16's range: bit 7, and 7 in the rest
__device__ __forceinline__ uint32_t large_scales(uint32_t x) { return x & 0x80808080u & ((x & 0x7f7f7f7fu) + 0x79797979u); }

// Infinities and NaN among pairs of 16-bit elements.  An element whose exponent field is all ones carries into its sign bit
// when one is added below the field.
//
// A product meets them where a weight of zero (a hidden key, or one far below the row's largest) would make NaN of them: there
// the finite part is multiplied as usual, and for each kind of the others a product of indicators tells which (channel, row)
// pairs meet one under a score that is not -inf.
template <bool F16>
struct OddValues {
    static constexpr uint32_t kExp = (F16 ? 0x7c00u : 0x7f80u) * 0x10001u, kUnit = (F16 ? 0x0400u : 0x0080u) * 0x10001u;
    static constexpr uint32_t kMant = kUnit - 0x10001u, kSign = 0x80008000u, kRest = 0x7fff7fffu, kOne = F16 ? 0x3c00u : 0x3f80u;
    __device__ static uint32_t any(const u32x4 w) {  // its sign bits
        const u32x4 t = (w & kExp) + kUnit;
        return t[0] | t[1] | t[2] | t[3];
    }
    __device__ static u32x4 odd(const u32x4 w) { return ((w & kExp) + kUnit) & kSign; }
    __device__ static u32x4 finite(const u32x4 w) { return w & ~((odd(w) >> 15) * 0xffffu); }
    __device__ static u32x4 kind(const u32x4 w, int t) {  // ones in the place of +inf, -inf, NaN
        const u32x4 o = odd(w), nan = ((w & kMant) + kRest) & o;
        return ((t == 0 ? (o & ~nan & ~w) : t == 1 ? (o & ~nan & w) : nan) >> 15) * kOne;
    }
    __device__ static u32x4 ones(uint32_t bits) {  // in the places of the set ones of eight bits
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = ((bits >> (2 * i) & 1) | (bits >> (2 * i + 1) & 1) << 16) * kOne;
        return r;
    }
    __device__ static float value(int t) { return t == 0 ? INFINITY : t == 1 ? -INFINITY : __builtin_nanf(""); }
};

// How a call is cut into workgroups.
struct AttnPlan {
    int row_tile;    // 16, 32 or 128 rows
    int n_tiles;     // upper bound of the row tiles of all sequences
    int n_split;     // parts a tile's keys may be cut into
    int chunk;       // key tiles of a part
    int key_tile;    // 32 or 64 positions
    int most_split;  // parts the workspace has room for: a window only lessens them
    bool one_wave;   // so few key tiles that a single wave takes a row tile
};

struct AttnJob {
    PagedAttnParams p;
    int n_tiles, n_split, chunk;
    float* part_o;   // [head, row tile][part][row][D]
    float* part_ml;  // [head, row tile][part][row][2]: reference (see Raised) and sum
};

// How a row tile's n_vt key tiles are cut: never into more parts than the launch has places for, whatever the host took for
// the number of tiles.
struct Parts {
    int chunk, n;
    __device__ Parts(const AttnJob& job, int n_vt) {
        const int least = (n_vt + job.n_split - 1) / job.n_split;
        chunk = job.chunk > least ? job.chunk : least;
        n = n_vt <= chunk ? 1 : (n_vt + chunk - 1) / chunk;
    }
};

// What a row tile covers.
struct TileSpan {
    int b, row0, n_rows, tok0, pos0, len;
    int sink_tiles, first, n_vt;  // key tiles: 0 .. sink_tiles - 1, then first ..; n_vt of them
};

// Sequence b's row tiles begin at cu_q[b] * group / row_tile + b: never fewer places than it needs.
template <int RT>
__device__ __forceinline__ int first_tile(const PagedAttnParams& p, int b, int cu) {
    return static_cast<int>(static_cast<int64_t>(cu) * p.group / RT) + b;
}

// What row tile `tile` covers of a sequence; false if none of its rows.
template <int RT, int TK>
__device__ __forceinline__ bool span_of(const PagedAttnParams& p, const Sequence& seq, int tile, TileSpan& s) {
    s.b = seq.b;
    const int cu0 = seq.cu0, cu1 = seq.cu1, kv = seq.len;
    const int64_t n_rows = static_cast<int64_t>((cu1 < p.n_tokens ? cu1 : p.n_tokens) - cu0) * p.group;
    const int64_t row0 = (static_cast<int64_t>(tile) - first_tile<RT>(p, s.b, cu0)) * RT;
    if (cu0 < 0 || row0 < 0 || row0 >= n_rows) return false;
    s.n_rows = static_cast<int>(n_rows);
    s.row0 = static_cast<int>(row0);
    s.tok0 = cu0;
    s.len = kv < 0 ? 0 : (kv < p.max_kv ? kv : p.max_kv);
    const int64_t pos0 = static_cast<int64_t>(kv) - cu1 + cu0;
    s.pos0 = static_cast<int>(pos0 < -(1 << 30) ? -(1 << 30) : pos0);
    const int last = s.row0 + RT - 1 < s.n_rows ? s.row0 + RT - 1 : s.n_rows - 1;
    const int pmin = s.pos0 + s.row0 / p.group, pmax = s.pos0 + last / p.group;
    int hi = pmax < 0 ? 0 : (p.causal && pmax + 1 < s.len ? pmax + 1 : s.len);
    int low = p.window > 0 ? pmin - p.window + 1 : 0;
    low = low < 0 ? 0 : low;
    s.first = low / TK;
    const int sink = p.sinks < hi ? p.sinks : hi;
    const int sink_tiles = (sink + TK - 1) / TK;
    s.sink_tiles = sink_tiles < s.first ? sink_tiles : s.first;
    const int end = (hi + TK - 1) / TK;
    s.n_vt = s.sink_tiles + (end > s.first ? end - s.first : 0);
    return true;
}

template <int RT, int TK>
__device__ __forceinline__ bool tile_span(const PagedAttnParams& p, int tile, TileSpan& s) {
    Sequence seq;
    return find_sequence(p.c, seq, [&](int i, int cu) { return first_tile<RT>(p, i, cu) <= tile; }) && span_of<RT, TK>(p, seq, tile, s);
}

template <int D>
__device__ __forceinline__ int swz_k(int r) {
    return D == 128 ? (r & 15) : ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int swz_v(int r) {
    return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

// Where the 16-position pieces of a key tile lie: rows of the cache, and which of them exist.  (Row numbers fit 32 bits: checked
// at the entry.)  Pages that hold whole tiles take one look-up, smaller ones one per piece.
template <int N>
struct Pieces {
    uint32_t row[N];
    uint32_t valid;
};

struct PageWalk {
    const_i32 table;
    int stride, n_pages, shift;
    uint32_t page_rows, head;  // rows of a page (all heads), first row of this head in it
    __device__ PageWalk(const PagedView& c, int b, int kvh)
        : table((const_i32)(c.block_table + static_cast<int64_t>(b) * c.table_stride)), stride(c.table_stride), n_pages(c.n_pages),
          shift(c.page_shift), page_rows(static_cast<uint32_t>(c.n_heads) << c.page_shift), head(static_cast<uint32_t>(kvh) << c.page_shift) {}
    __device__ __forceinline__ uint32_t find(int key, bool& ok) const {
        const int i = key >> shift;
        const int page = table[i < stride ? i : stride - 1];
        ok = (i < stride) & (static_cast<uint32_t>(page) < static_cast<uint32_t>(n_pages));
        return (ok ? page : 0) * page_rows + head + (key & ((1 << shift) - 1));
    }
    template <int N>
    __device__ __forceinline__ Pieces<N> tile(int key0) const {
        Pieces<N> r;
        bool ok;
        if (16 * N <= (1 << shift)) {
            const uint32_t row = find(key0, ok);
#pragma unroll
            for (int g = 0; g < N; ++g) r.row[g] = row + 16 * g;
            r.valid = ok ? (1u << N) - 1 : 0;
        } else {
            r.valid = 0;
#pragma unroll
            for (int g = 0; g < N; ++g) {
                r.row[g] = find(key0 + 16 * g, ok);
                r.valid |= ok ? 1u << g : 0u;
            }
        }
        return r;
    }
};

// What one row sees: positions [lo, hi) and the first `sinks`, of pieces that exist.  N scores of a lane in runs of four
// positions, run e / 4 of them at first(e / 4), in the piece of the same number that piece(e / 4) gives.
struct RowMask {
    int lo, hi, sinks;
    template <int N, class First, class Piece, class Score>
    __device__ __forceinline__ void hide(int key0, uint32_t valid, uint32_t all, First&& first, Piece&& piece, Score&& score) const {
        const uint32_t n = static_cast<uint32_t>(hi > lo ? hi - lo : 0);
        const int base = key0 - lo;
        const bool sink_tile = key0 < sinks;  // (the same in every lane)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int at = first(e / 4) + (e & 3);
            bool see = static_cast<uint32_t>(base + at) < n;
            if (sink_tile) see = see | ((key0 + at < sinks) & (key0 + at < hi));
            score(e) = see ? score(e) : -INFINITY;
        }
        if (valid != all) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (!((valid >> piece(e / 4)) & 1)) score(e) = -INFINITY;
        }
    }
};

// ---- many rows: prompts ------------------------------------------------------------------------------------------------
// Four waves with 32 rows each share key tiles of 64 positions in the LDS: tile t + 1 arrives while tile t is used.
//
// Bound by instruction issue: 64 scores cost 32 cycles of matrix instructions at 128 channels (16 at 64), an exponential of 16
// and some 20 cycles of other vector work.  Two chunks of 2048 tokens over 16 k positions, 16 heads of 128 on 4: 441 us, 970
// TFLOP/s (an 8192-cubed library product: 1296), 539 us from an 8-bit cache, whose tiles every workgroup converts; heads of
// 64: 261 us and 717 TFLOP/s for 4 prompts of up to 4096 over 6000, 113 us under a window of 1024; 64 sequences of up to 8192
// positions with 16 new tokens each, 32 heads on 8 of 128, 273 us.  (Cards differ: 474, 562, 276, 117 and 289 us on the slowest.)
template <int D, bool E4M3>
struct ManyShape {
    static constexpr int kKeys = 64, kRowTile = 128;
    static constexpr int kRowBytes = 2 * D;               // of a position in the LDS
    static constexpr int kTile = kKeys * kRowBytes;       // one of K, V
    static constexpr int kRpi = 1024 / kRowBytes;         // rows one wave brings in with one load
    static constexpr int kLoads = kKeys / (4 * kRpi);     // loads per wave for one of K, V
    static constexpr int kPieces = kKeys / 16;
};

template <int D, bool F16, bool E4M3>
__global__ __launch_bounds__(256, (D == 64 && !E4M3 ? 3 : 2)) void paged_attn_many_kernel(const AttnJob job) {
    using S = ManyShape<D, E4M3>;
    constexpr int kKeys = S::kKeys, kRowBytes = S::kRowBytes, kTile = S::kTile, kChunks = kRowBytes / 16, kMt = D / 32;
    constexpr uint32_t kAll = (1u << S::kPieces) - 1;
    using O = OddValues<F16>;
    __shared__ __attribute__((aligned(1024))) char smem[4 * kTile];
    __shared__ int odd_tile;   // the last edge tile in whose V an infinity or NaN was found
    __shared__ int once_more;  // whether the tiles are to be gone through again
    // (no saturate_fp16_conversions here: in that mode the matrix instructions lose infinities and NaN in their accumulators)
    const PagedAttnParams& p = job.p;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int logical = xcd_contiguous(blockIdx.x, gridDim.x);
    const int part = logical % job.n_split, item = logical / job.n_split;
    // Where XCDs share a head, each takes row tiles from all over the sequences: of contiguous halves one would have the long
    // sequence, or the rows that see most.  The last tiles, which see most, begin.  (Two prompts of 16 k and 13 k positions on
    // four heads: 463 us with contiguous shares, 443 us this way.)
    const int kvh = item / job.n_tiles;
    const int ways = 8 / (p.c.n_heads & 7 ? p.c.n_heads & -p.c.n_heads : 8);
    const int tile = job.n_tiles - 1 - strided(item % job.n_tiles, job.n_tiles, ways);
    TileSpan ts;
    if (!tile_span<S::kRowTile, kKeys>(p, tile, ts)) return;
    const Parts parts(job, ts.n_vt);
    const int n_parts = parts.n;
    if (part >= n_parts) return;
    const int vt0 = part * parts.chunk, vt1 = vt0 + parts.chunk < ts.n_vt ? vt0 + parts.chunk : ts.n_vt;

    // ---- this wave's rows, this lane's row
    const int rbase = ts.row0 + wave * 32;
    const bool has_rows = rbase < ts.n_rows;
    const int row = rbase + l31 < ts.n_rows ? rbase + l31 : ts.n_rows - 1;
    const int tok = row / p.group, hq = kvh * p.group + row % p.group;
    const int pos = ts.pos0 + tok;
    const int wlast = rbase + 31 < ts.n_rows ? rbase + 31 : ts.n_rows - 1;
    const int pmin = __builtin_amdgcn_readfirstlane(ts.pos0 + rbase / p.group), pmax = __builtin_amdgcn_readfirstlane(ts.pos0 + wlast / p.group);
    auto hi_of = [&](int i) { return i < 0 ? 0 : (p.causal && i + 1 < ts.len ? i + 1 : ts.len); };
    auto lo_of = [&](int i) { return p.window > 0 && i - p.window + 1 > 0 ? i - p.window + 1 : 0; };
    const int hi = hi_of(pos), lo = lo_of(pos);
    const int w_hi_max = hi_of(pmax), w_lo_min = lo_of(pmin);

    // ---- key tiles: where their pieces lie
    const PageWalk pages(p.c, ts.b, kvh);
    auto key0_of = [&](int vt) { return (vt < ts.sink_tiles ? vt : ts.first + vt - ts.sink_tiles) * kKeys; };

    // LDS addresses.  A row's 16-byte pieces are swizzled by functions of the row that are linear over its bits, so every
    // address below is one base per lane, an exclusive or with a constant and a constant offset.  The bases are hidden from
    // the compiler where they are used: it would keep each sum in a register of its own through the loop, and spill.
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr_of(smem));
    // 16-bit caches, straight into the LDS: load i of this wave covers rows (4 i + wave) * kRpi .. + kRpi - 1 of the tile, a
    // lane 16 bytes; the place in the LDS follows the lane, so the swizzle is applied to the source (K and V differ)
    const int lrow = (wave * S::kRpi & 15) + lane / kChunks, lchunk = lane % kChunks;
    const uint32_t voff_k = lrow * kRowBytes + (lchunk ^ swz_k<D>(lrow)) * 16, voff_v = lrow * kRowBytes + (lchunk ^ swz_v<D>(lrow)) * 16;
    auto issue16 = [&](const Pieces<S::kPieces>& pc, int buf) __attribute__((always_inline)) {
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + buf * 2 * kTile + wave * 1024);
        static_for<S::kLoads>([&](auto ic) {
            constexpr int I = decltype(ic)::value;
            int64_t at;
            if constexpr (S::kRpi == 8) {
                const uint32_t even = pc.row[2 * I], odd = pc.row[2 * I + 1];
                at = wave & 2 ? odd : even;
            } else {
                at = pc.row[I];
            }
            lds_dma16((const void*)uniform(p.c.k + at * kRowBytes), voff_k, dst + I * 4096);
            lds_dma16((const void*)uniform(p.c.v + at * kRowBytes), voff_v, dst + kTile + I * 4096);
        });
    };
    // e4m3, through registers: a wave takes a piece, a lane 16 codes of each of kLoads8 consecutive rows, so that their
    // exponents lie side by side
    constexpr int kLpr = D / 16, kLoads8 = 16 * kLpr / 64;
    const int r8 = (lane / kLpr) * kLoads8, c8 = lane % kLpr;  // first row (of the wave's), pair of 16-byte pieces
    u32x4 k8[E4M3 ? kLoads8 : 1], v8[E4M3 ? kLoads8 : 1];
    uint32_t ke8 = 0, ve8 = 0;
    auto issue8 = [&](const Pieces<S::kPieces>& pc) __attribute__((always_inline)) {
        if constexpr (E4M3) {
            int64_t at = pc.row[0];
#pragma unroll
            for (int g = 1; g < S::kPieces; ++g) {
                const uint32_t x = pc.row[g];
                at = wave == g ? x : at;
            }
            const char* kp = p.c.k + (at + r8) * D + 16 * c8;
            const char* vp = p.c.v + (at + r8) * D + 16 * c8;
#pragma unroll
            for (int i = 0; i < kLoads8; ++i) {
                k8[i] = *reinterpret_cast<const u32x4*>(kp + i * D);
                v8[i] = *reinterpret_cast<const u32x4*>(vp + i * D);
            }
            using E = std::conditional_t<kLoads8 == 2, uint16_t, uint8_t>;
            ke8 = *reinterpret_cast<const E*>(p.c.k_exp + at + r8);
            ve8 = *reinterpret_cast<const E*>(p.c.v_exp + at + r8);
        }
    };
    const int r8w = wave * 16 + r8;
    const uint32_t put_k = r8w * kRowBytes + ((2 * c8) ^ swz_k<D>(r8w)) * 16, put_v = r8w * kRowBytes + ((2 * c8) ^ swz_v<D>(r8w)) * 16;
    auto put8 = [&](uint32_t tile_base) __attribute__((always_inline)) {
        if constexpr (E4M3) {
            uint32_t kb = tile_base + put_k, vb = tile_base + kTile + put_v;
            asm volatile("" : "+v"(kb), "+v"(vb));
            auto put = [&](auto large) __attribute__((always_inline)) {
                constexpr bool kLarge = decltype(large)::value;
#pragma unroll
                for (int i = 0; i < kLoads8; ++i) {
                    const uint32_t ke = (ke8 >> (8 * i)) & 255u, ve = (ve8 >> (8 * i)) & 255u;
                    *lds<u32x4>((kb ^ (swz_k<D>(i) * 16)) + i * kRowBytes) = dequantise8<F16, kLarge>(k8[i][0], k8[i][1], ke);
                    *lds<u32x4>((kb ^ ((swz_k<D>(i) ^ 1) * 16)) + i * kRowBytes) = dequantise8<F16, kLarge>(k8[i][2], k8[i][3], ke);
                    *lds<u32x4>((vb ^ (swz_v<D>(i) * 16)) + i * kRowBytes) = dequantise8<F16, kLarge>(v8[i][0], v8[i][1], ve);
                    *lds<u32x4>((vb ^ ((swz_v<D>(i) ^ 1) * 16)) + i * kRowBytes) = dequantise8<F16, kLarge>(v8[i][2], v8[i][3], ve);
                }
            };
            if (F16 && __any((large_scales(ke8) | large_scales(ve8)) != 0)) put(std::true_type{});
            else put(std::false_type{});
        }
    };

    // ---- first tile, queries
    uint32_t valid = 0;  // of the tile that is about to be used: which of its pieces exist
    auto first_tile_of_walk = [&]() __attribute__((always_inline)) {
        if (vt0 >= vt1) return;
        const Pieces<S::kPieces> pc = pages.tile<S::kPieces>(key0_of(vt0));
        valid = pc.valid;
        if constexpr (E4M3) issue8(pc);
        else issue16(pc, 0);
    };
    first_tile_of_walk();
    const float c = fmaxf(__builtin_fabsf(p.scale_log2), 1e-37f);  // (a scale of zero weighs all positions the same)
    u16x8 qf[D / 16];
    {
        const uint16_t* qp = p.q + (ts.tok0 + tok) * p.q_ts + hq * p.q_hs + 8 * h;
        const uint16_t flip = p.scale_log2 < 0.0f ? 0x8000 : 0;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qp + 16 * s) ^ flip;
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) asm volatile("" : "+v"(qf[s]));  // waited for here, not behind the next tile's loads

    const uint32_t get_k = l31 * kRowBytes + ((h ^ swz_k<D>(l31)) << 4);  // piece 2 s + h of key row l31
    uint32_t get_v;  // V read transposed: lane 4 q + pp of 16 fetches key row q, channels 4 pp ..; it receives 4 keys of a channel
    {
        const int q = (lane >> 2) & 3, pp = lane & 3, g1 = (lane >> 4) & 1, r = 4 * h + q;
        get_v = r * kRowBytes + ((2 * g1 + (pp >> 1)) ^ swz_v<D>(r)) * 16 + 8 * (pp & 1);
    }

    f32x16 oacc[kMt];
    float mc, l_run;  // reference (see Raised) and sum of this lane's half of the keys
    int buf, vt;
    auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[mt][e] = 0.0f;
        mc = -INFINITY;
        l_run = 0.0f;
        buf = 0;
        vt = vt0;
        if (tid == 0) odd_tile = -1;  // (every use of it lies behind a barrier)
    };
    begin();
    if (tid == 0) once_more = 0;

    auto compute = [&](uint32_t tile_base, int key0, uint32_t exist, bool special, auto edge_c) __attribute__((always_inline)) {
        constexpr bool edge = decltype(edge_c)::value;
        f32x16 sacc[2];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int e = 0; e < 16; ++e) sacc[kk][e] = 0.0f;
        uint32_t kb = tile_base + get_k;
        asm volatile("" : "+v"(kb));
        // (fragments three steps ahead of their use; consecutive products alternate between the two accumulators)
        auto k_frag = [&](int s, int kk) { return *lds<const u16x8>((kb ^ (s << 5)) + kk * 32 * kRowBytes); };
        u16x8 kf[3][2];
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            kf[s][0] = k_frag(s, 0);
            kf[s][1] = k_frag(s, 1);
        }
        static_for<D / 16>([&](auto sc) {
            constexpr int T = decltype(sc)::value;
            sacc[0] = mfma32<F16>(kf[T % 3][0], qf[T], sacc[0]);
            sacc[1] = mfma32<F16>(kf[T % 3][1], qf[T], sacc[1]);
            if constexpr (T + 3 < D / 16) {
                kf[T % 3][0] = k_frag(T + 3, 0);
                kf[T % 3][1] = k_frag(T + 3, 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        uint32_t vb = tile_base + kTile + get_v;
        asm volatile("" : "+v"(vb));
        auto v_frag = [&](int kk, int s2, int mt) {  // rows 8 x + 4 h + q of the 16: the swizzle turns by 2 x, the channels by 4 mt
            const uint32_t at = vb ^ (mt * 64);
            const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<v4s>(at + (kk * 32 + s2 * 16) * kRowBytes));
            const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<v4s>((at ^ 32) + (kk * 32 + s2 * 16 + 8) * kRowBytes));
            return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // the products' steps: 32-position half kk, 16 positions s2 of it, 32 channels mt; fragments are read four steps ahead
        constexpr int kSteps = 4 * kMt, kRing = 4;
        u32x4 vf[kRing];
        auto v_step = [&](auto tc) __attribute__((always_inline)) {
            constexpr int T = decltype(tc)::value;
            vf[T % kRing] = v_frag(T / (2 * kMt), (T / kMt) & 1, T % kMt);
        };
        if constexpr (!edge) static_for<kRing>([&](auto tc) { v_step(tc); });
        uint32_t seen = 0;  // of this lane's 32 scores, where that is asked for
        if constexpr (edge) {
            const RowMask mask{lo, hi, p.sinks};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
                mask.hide<16>(key0, exist, kAll, [&](int r) { return kk * 32 + 8 * r + 4 * h; }, [&](int r) { return 2 * kk + (r >> 1); },
                              [&](int e) -> float& { return reinterpret_cast<float*>(&sacc[kk])[e]; });
            if (special) {
#pragma unroll
                for (int e = 0; e < 32; ++e) seen |= sacc[e / 16][e % 16] == -INFINITY ? 0u : 1u << e;
            }
        }
        float rmax = sacc[0][0];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int e = 0; e < 16; ++e) rmax = fmaxf(rmax, sacc[kk][e]);
        {   // the row's other keys sit in lane ^ 32
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(rmax), __float_as_uint(rmax), false, false);
            rmax = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        }
        // the maximum only has to keep the weights in range
        const float most = fmaf(rmax, c, -Raised<F16>::kRaise);
        const bool grew = most > mc + Raised<F16>::kLag;
        const float m_new = grew ? most : mc;
        const float alpha = grew ? factor(mc, m_new) : 1.0f;
        mc = m_new;
        const float sub = mc == -INFINITY ? 0.0f : mc;  // (nothing seen yet: every weight below is exp2(-inf))
        if (__any(grew)) {
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[mt][e] *= alpha;
        }
        float psum = 0.0f;
        u32x4 pf[2][2];
        auto weigh = [&](auto qc) __attribute__((always_inline)) {  // two scores: pair Q of the 16 of a lane
            constexpr int Q = decltype(qc)::value, kk = Q / 8, e = 2 * (Q % 8);
            const float a = __builtin_amdgcn_exp2f(fmaf(sacc[kk][e], c, -sub));
            const float b = __builtin_amdgcn_exp2f(fmaf(sacc[kk][e + 1], c, -sub));
            psum += a + b;
            pf[kk][e / 8][(e % 8) / 2] = pack_elem2<F16>(a, b);
        };
        auto times = [&](const u32x4 v, const u32x4 w, const f32x16 acc) { return mfma32<F16>(__builtin_bit_cast(u16x8, v), __builtin_bit_cast(u16x8, w), acc); };
        if constexpr (edge) {
            static_for<16>([&](auto qc) { weigh(qc); });
            l_run = l_run * alpha + psum;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) asm volatile("" : "+v"(pf[kk][s2]));  // (packed here: not in 32 bits up to their use)
        }
        if (!special) {
            if constexpr (edge) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                        for (int mt = 0; mt < kMt; ++mt) oacc[mt] = times(v_frag(kk, s2, mt), pf[kk][s2], oacc[mt]);
            } else {
                // the products of the first half of the keys have the exponentials of the second between them
                static_for<8>([&](auto qc) { weigh(qc); });
                static_for<kSteps>([&](auto tc) {
                    constexpr int T = decltype(tc)::value, kk = T / (2 * kMt), s2 = (T / kMt) & 1, mt = T % kMt;
                    const u32x4 v = vf[T % kRing];
                    if constexpr (T + kRing < kSteps) v_step(IC<T + kRing>{});
                    oacc[mt] = times(v, pf[kk][s2], oacc[mt]);
                    if constexpr (kk == 0) static_for<4 / kMt>([&](auto xc) { weigh(IC<8 + T * (4 / kMt) + decltype(xc)::value>{}); });
                    __builtin_amdgcn_sched_barrier(0);
                });
                l_run = l_run * alpha + psum;
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                    for (int mt = 0; mt < kMt; ++mt) {
                        const u32x4 v = v_frag(kk, s2, mt);
                        oacc[mt] = times(O::finite(v), pf[kk][s2], oacc[mt]);
#pragma unroll
                        for (int t = 0; t < 3; ++t) {
                            f32x16 hit;
#pragma unroll
                            for (int e = 0; e < 16; ++e) hit[e] = 0.0f;
                            hit = times(O::kind(v, t), O::ones(seen >> (16 * kk + 8 * s2)), hit);
#pragma unroll
                            for (int e = 0; e < 16; ++e) oacc[mt][e] += hit[e] > 0.0f ? O::value(t) : 0.0f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
        }
    };

    // Tiles [inner0, inner1) lie inside every row's mask.  They run in a loop of their own: with both kinds in one loop the
    // accumulators would be copied between them, 64 registers a tile.  (The way back, for infinities, costs heads of 64 some 1 %
    // even if none takes it; a second copy of the edge loop instead of it costs 8-bit caches 11 %.)
    const int first_row = ts.row0 / p.group, last_row = (ts.row0 + S::kRowTile - 1 < ts.n_rows ? ts.row0 + S::kRowTile - 1 : ts.n_rows - 1) / p.group;
    const int all_lo = lo_of(ts.pos0 + last_row), from = (all_lo + kKeys - 1) / kKeys - ts.first;
    const int inner0 = ts.sink_tiles + (from > 0 ? from : 0), to = ts.sink_tiles + hi_of(ts.pos0 + first_row) / kKeys - ts.first;
    int inner1 = to < vt1 ? to : vt1;
    auto turn = [&](auto edge_c) __attribute__((always_inline)) {
        constexpr bool edge = decltype(edge_c)::value;
        if constexpr (E4M3) put8(lds0 + buf * 2 * kTile);
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the tile are in
        __syncthreads();  // and all others'; and no wave reads the other buffer any more
        const uint32_t now = valid;
        if (vt + 1 < vt1) {
            const Pieces<S::kPieces> pc = pages.tile<S::kPieces>(key0_of(vt + 1));
            valid = pc.valid;
            if constexpr (E4M3) issue8(pc);
            else issue16(pc, buf ^ 1);
        }
        const int key0 = key0_of(vt);
        // In an edge tile a hidden value may meet a weight of zero: every wave looks through 16 of its rows of V.
        bool special = false;
        if constexpr (edge) {
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < 16 * kRowBytes / 1024; ++i) any |= O::any(*lds<const u32x4>(lds0 + (2 * buf + 1) * kTile + (wave * 16 * kRowBytes + i * 1024) + lane * 16));
            if (__any((any & O::kSign) != 0)) odd_tile = vt;
            __syncthreads();
            special = __builtin_amdgcn_readfirstlane(odd_tile) == vt;
        }
        // (an edge tile may be hidden from every row of a wave: the keys behind a prompt's first rows, the window of its last)
        if (!edge || (has_rows && key0 < w_hi_max && (key0 + kKeys > w_lo_min || key0 < p.sinks))) compute(lds0 + buf * 2 * kTile, key0, now, special, edge_c);
        buf ^= 1;
        ++vt;
    };
    for (;;) {
        bool plain = false;  // an inner tile was met
        while (vt < vt1) {
            if (vt >= inner0 && vt < inner1 && valid == kAll) {
                plain = true;
                do turn(std::false_type{});
                while (vt < inner1 && valid == kAll);
            } else {
                turn(std::true_type{});
            }
        }
        if (!plain) break;
        // a sum that is NaN though no score was: an infinity may have met a weight of zero in an inner tile
        bool nan = false;
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
            for (int e = 0; e < 16; e += 2) nan |= __builtin_isunordered(oacc[mt][e], oacc[mt][e + 1]);
        if (__any(nan && l_run == l_run)) once_more = 1;
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(once_more) == 0) break;
        inner1 = vt0;  // none is
        begin();
        first_tile_of_walk();
    }

    // ---- results: lane (l31, h) holds of its row the channels 32 mt + 8 (e >> 2) + 4 h + (e & 3)
    if (!has_rows || rbase + l31 >= ts.n_rows) return;
    const float l_tot = l_run + __shfl_xor(l_run, 32);
    const float inv = inverse(l_tot);
    const int64_t part_row = ((static_cast<int64_t>(kvh) * job.n_tiles + tile) * job.n_split + part) * S::kRowTile + wave * 32 + l31;
    int t = ts.tok0 + tok, head = hq;
    asm volatile("" : "+v"(t), "+v"(head));  // (addresses are formed here: not kept through the loop)
    uint16_t* out = p.out + t * p.o_ts + head * p.o_hs + 4 * h;
    float* po = job.part_o + part_row * D + 4 * h;
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 o = make_float4(oacc[mt][e], oacc[mt][e + 1], oacc[mt][e + 2], oacc[mt][e + 3]);
            const int ch = 32 * mt + 2 * e;
            if (n_parts == 1) *reinterpret_cast<uint2*>(out + ch) = make_uint2(pack_result<F16>(o.x * inv, o.y * inv), pack_result<F16>(o.z * inv, o.w * inv));
            else *reinterpret_cast<float4*>(po + ch) = o;
        }
    if (n_parts > 1 && h == 0) *reinterpret_cast<float2*>(job.part_ml + part_row * 2) = make_float2(mc, l_tot);
}

// ---- few rows: single tokens, short chunks ---------------------------------------------------------------------------
// A wave has the 16 * NQ rows of the tile and key tiles of 32 positions of its own.  With v_mfma_f32_16x16x32 the first
// operand is 16 keys by 32 channels, 8 consecutive channels per lane: K goes from memory straight to registers, one tile
// ahead; V goes to the LDS and is read transposed.  The scores of a lane are those of keys 4 g .. 4 g + 3 (g = lane / 16) of
// either half of the tile, for row lane % 16: taken in this order they are the second operand of O^T = V^T P^T as they are.
//
// Bound by memory: 64 sequences of up to 8192 positions, 32 heads on 8 of 128: 219 us and 5.4 TB/s in 16 bits, 132 us in 8
// (4.5 TB/s); 8 sequences of up to 131072 in 8 bits 95 us, 4.5 TB/s; 256 chunks of 10 frames under a window of 50 13.5 us in 16
// bits, 12.5 us in 8.
template <int D, bool E4M3, int NQ, int KW>
struct FewShape {
    static constexpr int kRowBytes = 2 * D;
    static constexpr int kTile = 32 * kRowBytes;                   // V of a key tile
    static constexpr int kBufs = E4M3 ? 1 : 2;                     // (e4m3: the next one waits in registers)
    static constexpr int kAcc = NQ * (D / 16) * 4;                 // accumulators of a lane
    static constexpr int kJoin = KW > 1 ? KW * kAcc * 256 + KW * NQ * 128 : 0;
    static constexpr int kLds = KW * kBufs * kTile > kJoin ? KW * kBufs * kTile : kJoin;
    static constexpr int kRpi = 1024 / kRowBytes, kLoads = 32 / kRpi, kVar = 16 / kRpi;
    static constexpr int kKs = E4M3 ? D / 64 : D / 32;             // 16-byte loads of K per lane and 16 keys
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool F16>
__device__ __forceinline__ f32x4 mfma16(const u32x4 a, const u32x4 b, const f32x4 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// maximum and sum over the four lanes that hold one row
__device__ __forceinline__ float max_of_row(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_of_row(float v) {
    v += __shfl_xor(v, 32);
    return v + __shfl_xor(v, 16);
}

template <int D, bool F16, bool E4M3, int NQ, int KW>
__global__ __launch_bounds__(64 * KW, (NQ == 1 ? 2 : 1)) void paged_attn_few_kernel(const AttnJob job) {
    using S = FewShape<D, E4M3, NQ, KW>;
    constexpr int kRowBytes = S::kRowBytes, kTile = S::kTile, kChunks = kRowBytes / 16, kMb = D / 16, kRt = 16 * NQ, kKeys = 32, kKs = S::kKs;
    __shared__ __attribute__((aligned(1024))) char smem[S::kLds];
    const PagedAttnParams& p = job.p;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int logical = xcd_contiguous(blockIdx.x, gridDim.x);
    const int part = logical % job.n_split, item = logical / job.n_split;
    const int tile = item % job.n_tiles, kvh = item / job.n_tiles;
    TileSpan ts;
    if (!tile_span<kRt, kKeys>(p, tile, ts)) return;
    const Parts parts(job, ts.n_vt);
    const int n_parts = parts.n;
    if (part >= n_parts) return;
    const int vt0 = part * parts.chunk, vt1 = vt0 + parts.chunk < ts.n_vt ? vt0 + parts.chunk : ts.n_vt;

    // ---- rows
    const int last = ts.row0 + kRt - 1 < ts.n_rows ? ts.row0 + kRt - 1 : ts.n_rows - 1;
    const int pmin = __builtin_amdgcn_readfirstlane(ts.pos0 + ts.row0 / p.group), pmax = __builtin_amdgcn_readfirstlane(ts.pos0 + last / p.group);
    auto hi_of = [&](int i) { return i < 0 ? 0 : (p.causal && i + 1 < ts.len ? i + 1 : ts.len); };
    auto lo_of = [&](int i) { return p.window > 0 && i - p.window + 1 > 0 ? i - p.window + 1 : 0; };
    int w_hi_min = hi_of(pmin);
    const int w_lo_max = lo_of(pmax);
    int hi[NQ], lo[NQ];
    int64_t out_at[NQ];
    u32x4 qf[NQ][D / 32];
    const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
    const float c = fmaxf(__builtin_fabsf(p.scale_log2), 1e-37f);  // (a scale of zero weighs all positions the same)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = ts.row0 + 16 * n + col, row = r < ts.n_rows ? r : ts.n_rows - 1;
        const int tok = row / p.group, hq = kvh * p.group + row % p.group;
        hi[n] = hi_of(ts.pos0 + tok);
        lo[n] = lo_of(ts.pos0 + tok);
        out_at[n] = (ts.tok0 + tok) * p.o_ts + hq * p.o_hs;
        const uint16_t* qp = p.q + (ts.tok0 + tok) * p.q_ts + hq * p.q_hs;
        // the channels of step s, in the order in which this lane has those of its keys
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const int d = E4M3 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
            qf[n][s] = *reinterpret_cast<const u32x4*>(qp + d) ^ flip;
        }
    }

    // ---- key tiles
    const PageWalk pages(p.c, ts.b, kvh);
    auto key0_of = [&](int vt) { return (vt < ts.sink_tiles ? vt : ts.first + vt - ts.sink_tiles) * kKeys; };
    const uint32_t own_base = __builtin_amdgcn_readfirstlane(lds_addr_of(smem + wave * S::kBufs * kTile));
    const int lrow = lane / kChunks, lchunk = lane % kChunks;
    uint32_t voff_v[E4M3 ? 1 : S::kVar];
    if constexpr (!E4M3) {
#pragma unroll
        for (int i = 0; i < S::kVar; ++i) {
            const int r = i * S::kRpi + lrow;
            voff_v[i] = r * kRowBytes + (lchunk ^ swz_v<D>(r)) * 16;
        }
    }
    constexpr int kStored = E4M3 ? D : 2 * D;
    const uint32_t voff_k = col * kStored + 16 * g;
    constexpr int kLpr = D / 16, kLoads8 = 32 * kLpr / 64;
    const int r8 = (lane / kLpr) * kLoads8, c8 = lane % kLpr;
    u32x4 v8[E4M3 ? kLoads8 : 1];
    uint32_t ve8 = 0;
    struct Keys {
        u32x4 w[2][kKs];
        uint32_t exp[2];
    };
    auto issue = [&](const Pieces<2>& pc, Keys& k, int buf) __attribute__((always_inline)) {
        if constexpr (E4M3) {
            const uint32_t even = pc.row[0], odd = pc.row[1];
            const int64_t at = static_cast<int64_t>(r8 & 16 ? odd : even) + (r8 & 15);
            const char* vp = p.c.v + at * D + 16 * c8;
#pragma unroll
            for (int i = 0; i < kLoads8; ++i) v8[i] = *reinterpret_cast<const u32x4*>(vp + i * D);
            using E = std::conditional_t<kLoads8 == 4, uint32_t, uint16_t>;
            ve8 = *reinterpret_cast<const E*>(p.c.v_exp + at);
        } else {
            const uint32_t dst = __builtin_amdgcn_readfirstlane(own_base + buf * kTile);
            static_for<S::kLoads>([&](auto ic) {
                constexpr int I = decltype(ic)::value;
                lds_dma16((const void*)uniform(p.c.v + static_cast<int64_t>(pc.row[I * S::kRpi / 16]) * kRowBytes), voff_v[I % S::kVar], dst + I * 1024);
            });
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const global_ptr kp = uniform(p.c.k + static_cast<int64_t>(pc.row[u]) * kStored);
#pragma unroll
            for (int s = 0; s < kKs; ++s) k.w[u][s] = *(const __attribute__((address_space(1))) u32x4*)(kp + voff_k + 64 * s);
            if constexpr (E4M3) k.exp[u] = (uint8_t)uniform(reinterpret_cast<const char*>(p.c.k_exp) + pc.row[u])[static_cast<uint32_t>(col)];
        }
    };
    const uint32_t put_v = r8 * kRowBytes + ((2 * c8) ^ swz_v<D>(r8)) * 16;
    uint32_t get_v;  // V read transposed: lane 4 q + pp of 16 fetches key row 4 g + q, channels 4 pp ..; it receives 4 keys of a channel
    {
        const int q = col >> 2, pp = col & 3, r = 4 * g + q;
        get_v = r * kRowBytes + ((pp >> 1) ^ swz_v<D>(r)) * 16 + 8 * (pp & 1);
    }

    f32x4 oacc[NQ][kMb];
    float mc[NQ], l_run[NQ];

    auto compute = [&](const Keys& k, uint32_t tile_base, int key0, uint32_t valid, auto edge_c) __attribute__((always_inline)) {
        constexpr bool edge = decltype(edge_c)::value;
        f32x4 sacc[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) sacc[n][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const bool large = F16 && E4M3 && __any((k.exp[0] >= 135) | (k.exp[1] >= 135));
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u32x4 kf;
                if constexpr (E4M3) {
                    const uint32_t a = k.w[u][s >> 1][2 * (s & 1)], b = k.w[u][s >> 1][2 * (s & 1) + 1];
                    kf = large ? dequantise8<F16, true>(a, b, k.exp[u]) : dequantise8<F16, false>(a, b, k.exp[u]);
                } else {
                    kf = k.w[u][s];
                }
#pragma unroll
                for (int n = 0; n < NQ; ++n) sacc[n][u] = mfma16<F16>(kf, qf[n][s], sacc[n][u]);
            }
        u32x4 pf[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            if constexpr (edge) {
                const RowMask mask{lo[n], hi[n], p.sinks};
                mask.hide<8>(key0, valid, 3, [&](int u) { return 16 * u + 4 * g; }, [&](int u) { return u; },
                             [&](int e) -> float& { return reinterpret_cast<float*>(&sacc[n][e >> 2])[e & 3]; });
            }
            float rmax = sacc[n][0][0];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) rmax = fmaxf(rmax, sacc[n][u][i]);
            rmax = max_of_row(rmax);
            // the maximum only has to keep the weights in range
            const float most = fmaf(rmax, c, -Raised<F16>::kRaise);
            const bool grew = most > mc[n] + Raised<F16>::kLag;
            const float m_new = grew ? most : mc[n];
            const float alpha = grew ? factor(mc[n], m_new) : 1.0f;
            mc[n] = m_new;
            const float sub = m_new == -INFINITY ? 0.0f : m_new;  // (nothing seen yet: every weight below is exp2(-inf))
            if (__any(grew)) {
#pragma unroll
                for (int m = 0; m < kMb; ++m) oacc[n][m] *= alpha;
            }
            float psum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float a = __builtin_amdgcn_exp2f(fmaf(sacc[n][u][i], c, -sub));
                    const float b = __builtin_amdgcn_exp2f(fmaf(sacc[n][u][i + 1], c, -sub));
                    psum += a + b;
                    pf[n][2 * u + i / 2] = pack_elem2<F16>(a, b);
                }
            l_run[n] = l_run[n] * alpha + psum;
        }
        uint32_t vb = tile_base + get_v;
        asm volatile("" : "+v"(vb));
        auto v_frag = [&](int m) {
            const uint32_t at = vb ^ (m * 32);
            const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<v4s>(at));
            const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<v4s>(at + 16 * kRowBytes));
            return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        using O = OddValues<F16>;
        bool special = false;
        if constexpr (edge) {
            uint32_t any = 0;
#pragma unroll
            for (int m = 0; m < kMb; ++m) any |= O::any(v_frag(m));
            special = __any((any & O::kSign) != 0);
        }
        if (!special) {
#pragma unroll
            for (int m = 0; m < kMb; ++m) {
                const u32x4 v = v_frag(m);
#pragma unroll
                for (int n = 0; n < NQ; ++n) oacc[n][m] = mfma16<F16>(v, pf[n], oacc[n][m]);
            }
        } else {
            uint32_t seen[NQ];  // of this lane's eight scores of a row
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                seen[n] = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) seen[n] |= sacc[n][e >> 2][e & 3] == -INFINITY ? 0u : 1u << e;
            }
#pragma unroll
            for (int m = 0; m < kMb; ++m) {
                const u32x4 v = v_frag(m);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    oacc[n][m] = mfma16<F16>(O::finite(v), pf[n], oacc[n][m]);
#pragma unroll
                    for (int t = 0; t < 3; ++t) {
                        const f32x4 hit = mfma16<F16>(O::kind(v, t), O::ones(seen[n]), f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int i = 0; i < 4; ++i) oacc[n][m][i] += hit[i] > 0.0f ? O::value(t) : 0.0f;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };

    int vt;
    uint32_t valid = 0;  // of the tile that is about to be used: which of its pieces exist
    bool plain = false;  // an inner tile was met
    Keys ka, kb;
    auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            mc[n] = -INFINITY;
            l_run[n] = 0.0f;
#pragma unroll
            for (int m = 0; m < kMb; ++m) oacc[n][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        vt = vt0 + wave;
        if (vt < vt1) {
            const Pieces<2> pc = pages.tile<2>(key0_of(vt));
            valid = pc.valid;
            issue(pc, ka, 0);
        }
    };
    auto turn = [&](Keys& now_k, Keys& next_k, int buf) __attribute__((always_inline)) {
        // everything of this tile is in, and the reads of the tile before are done with the other buffer
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
        asm volatile("" ::: "memory");
        if constexpr (E4M3) {
            uint32_t vb = own_base + put_v;
            asm volatile("" : "+v"(vb));
            auto put = [&](auto big) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < kLoads8; ++i) {
                    const uint32_t e = (ve8 >> (8 * i)) & 255u;
                    *lds<u32x4>((vb ^ (swz_v<D>(i) * 16)) + i * kRowBytes) = dequantise8<F16, decltype(big)::value>(v8[i][0], v8[i][1], e);
                    *lds<u32x4>((vb ^ ((swz_v<D>(i) ^ 1) * 16)) + i * kRowBytes) = dequantise8<F16, decltype(big)::value>(v8[i][2], v8[i][3], e);
                }
            };
            if (F16 && __any(large_scales(ve8) != 0)) put(std::true_type{});
            else put(std::false_type{});
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        const uint32_t now = valid;
        const int next = vt + KW, key0 = key0_of(vt);
        if (next < vt1) {
            const Pieces<2> pc = pages.tile<2>(key0_of(next));
            valid = pc.valid;
            issue(pc, next_k, E4M3 ? 0 : buf ^ 1);
        }
        const uint32_t base = own_base + (E4M3 ? 0 : buf * kTile);
        if (key0 + kKeys <= w_hi_min && (key0 >= w_lo_max || key0 + kKeys <= p.sinks) && now == 3) {
            plain = true;
            compute(now_k, base, key0, now, std::false_type{});
        } else {
            compute(now_k, base, key0, now, std::true_type{});
        }
        vt = next;
    };
    begin();
    for (;;) {
        while (vt < vt1) {
            turn(ka, kb, 0);
            if (vt >= vt1) break;
            turn(kb, ka, 1);
        }
        if (!plain) break;
        // a sum that is NaN though no score was: an infinity may have met a weight of zero in an inner tile
        bool nan = false;
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int m = 0; m < kMb; ++m)
                nan |= (__builtin_isunordered(oacc[n][m][0], oacc[n][m][1]) | __builtin_isunordered(oacc[n][m][2], oacc[n][m][3])) & (l_run[n] == l_run[n]);
        if (!__any(nan)) break;
        w_hi_min = -1;  // none is
        plain = false;
        begin();
    }

    // ---- results: lane (col, g) holds of row col the channels 16 m + 4 g .. + 3
    const int64_t part_row = (static_cast<int64_t>(item) * job.n_split + part) * kRt;
    auto store = [&](int n, int m, float4 o, float inv) {
        if (ts.row0 + 16 * n + col >= ts.n_rows) return;
        const int ch = 16 * m + 4 * g;
        if (n_parts == 1) *reinterpret_cast<uint2*>(p.out + out_at[n] + ch) = make_uint2(pack_result<F16>(o.x * inv, o.y * inv), pack_result<F16>(o.z * inv, o.w * inv));
        else *reinterpret_cast<float4*>(job.part_o + (part_row + 16 * n + col) * D + ch) = o;
    };
    auto store_ml = [&](int n, float m, float l) {
        if (n_parts > 1 && g == 0 && ts.row0 + 16 * n + col < ts.n_rows) *reinterpret_cast<float2*>(job.part_ml + (part_row + 16 * n + col) * 2) = make_float2(m, l);
    };
#pragma unroll
    for (int n = 0; n < NQ; ++n) l_run[n] = sum_of_row(l_run[n]);
    if constexpr (KW == 1) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int m = 0; m < kMb; ++m) store(n, m, make_float4(oacc[n][m][0], oacc[n][m][1], oacc[n][m][2], oacc[n][m][3]), inverse(l_run[n]));
            store_ml(n, mc[n], l_run[n]);
        }
    } else {
        // the waves' sums are brought to one maximum and added through the LDS
        float* ml = reinterpret_cast<float*>(smem);  // [wave][n][maximum of 16 rows, sum of 16 rows]
        float* os = ml + KW * NQ * 32;
        __syncthreads();  // all waves are done with their tiles
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            if (g == 0) {
                ml[(wave * NQ + n) * 32 + col] = mc[n];
                ml[(wave * NQ + n) * 32 + 16 + col] = l_run[n];
            }
        __syncthreads();
        float inv[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float top = mc[n], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < KW; ++i) top = fmaxf(top, ml[(i * NQ + n) * 32 + col]);
            const float sub = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < KW; ++i) sum += ml[(i * NQ + n) * 32 + 16 + col] * __builtin_amdgcn_exp2f(ml[(i * NQ + n) * 32 + col] - sub);
            const float f = factor(mc[n], sub);
#pragma unroll
            for (int m = 0; m < kMb; ++m)
                *reinterpret_cast<float4*>(os + (((wave * NQ + n) * kMb + m) * 64 + lane) * 4) = make_float4(oacc[n][m][0] * f, oacc[n][m][1] * f, oacc[n][m][2] * f, oacc[n][m][3] * f);
            inv[n] = inverse(sum);
            if (wave == 0) store_ml(n, top, sum);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            for (int m = wave; m < kMb; m += KW) {
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    const float4 t = *reinterpret_cast<const float4*>(os + (((i * NQ + n) * kMb + m) * 64 + lane) * 4);
                    a.x += t.x; a.y += t.y; a.z += t.z; a.w += t.w;
                }
                store(n, m, a, inv[n]);
            }
    }
}

// ---- joining parts -----------------------------------------------------------------------------------------------------
// Row (t, hq): where its parts begin (place `at` of n, RT places apart); false if there is nothing to join.
template <int RT, int TK>
__device__ __forceinline__ bool parts_of(const AttnJob& job, int t, int hq, int& n, int64_t& at) {
    const PagedAttnParams& p = job.p;
    Sequence seq;
    if (!sequence_of(p.c, t, seq)) return false;
    const int row = (t - seq.cu0) * p.group + hq % p.group, tile = first_tile<RT>(p, seq.b, seq.cu0) + row / RT;
    TileSpan ts;
    if (tile >= job.n_tiles || !span_of<RT, TK>(p, seq, tile, ts)) return false;
    n = Parts(job, ts.n_vt).n;
    at = (static_cast<int64_t>(hq / p.group) * job.n_tiles + tile) * job.n_split * RT + row % RT;
    return n > 1;
}

__device__ __forceinline__ void add(float4& a, const float4 o, float w) {
    a.x = fmaf(o.x, w, a.x);
    a.y = fmaf(o.y, w, a.y);
    a.z = fmaf(o.z, w, a.z);
    a.w = fmaf(o.w, w, a.w);
}

template <bool F16>
__device__ __forceinline__ void put_row(const PagedAttnParams& p, int t, int hq, int ch, const float4 a, float inv) {
    uint16_t* out = p.out + t * p.o_ts + hq * p.o_hs + ch;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_result<F16>(a.x * inv, a.y * inv), pack_result<F16>(a.z * inv, a.w * inv));
}

// A wave joins a row of few parts: lane i weighs part i, then D / 4 lanes add four channels of a part, two or four parts at a
// time.  (2048 rows of 128 channels in 4 parts 5.3 us, with a workgroup a row 8.3 us; of 7700 rows of 64 channels in 4 parts the
// whole call 35 and 47 us.)
constexpr int kFewParts = 16;

template <int D, bool F16, int RT, int TK>
__global__ __launch_bounds__(256) void paged_join_few_kernel(const AttnJob job) {
    constexpr int kT = D / 4, kSlices = 64 / kT;
    const PagedAttnParams& p = job.p;
    const int i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = i / p.n_q_heads, hq = i % p.n_q_heads;
    if (t >= p.n_tokens) return;
    int n;
    int64_t at;
    if (!parts_of<RT, TK>(job, t, hq, n, at)) return;
    const int lane = threadIdx.x & 63, slice = lane / kT, ch = 4 * (lane % kT);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(job.part_ml + (at + static_cast<int64_t>(lane) * RT) * 2);
    const float* part = job.part_o + at * D + ch;
    constexpr int kEarly = 4;  // on their way while the weights are found
    float4 early[kEarly];
#pragma unroll
    for (int k = 0; k < kEarly; ++k) {
        const int j = slice + k * kSlices;
        early[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j < n) early[k] = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(j) * RT * D);
    }
    float top = ml.x;
#pragma unroll
    for (int o = kFewParts / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float f = factor(ml.x, top == -INFINITY ? 0.0f : top);
    float sum = ml.y * f;
#pragma unroll
    for (int o = kFewParts / 2; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    sum = __shfl(sum, 0);
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < kFewParts / kSlices; ++k) {
        if (k * kSlices >= n) break;
        const int j = slice + k * kSlices;
        const float w = __shfl(f, j);
        if (j < n) add(a, k < kEarly ? early[k < kEarly ? k : 0] : *reinterpret_cast<const float4*>(part + static_cast<int64_t>(j) * RT * D), w);
    }
#pragma unroll
    for (int o = kT; o < 64; o <<= 1) {
        a.x += __shfl_xor(a.x, o);
        a.y += __shfl_xor(a.y, o);
        a.z += __shfl_xor(a.z, o);
        a.w += __shfl_xor(a.w, o);
    }
    if (slice == 0) put_row<F16>(p, t, hq, ch, a, inverse(sum));
}

// A workgroup joins a row of many (at most kMostParts): a thread adds four channels over every eighth part or so, the sums meet
// in the LDS.  A chain of dependent loads: 6.3 us for 128 rows of up to 128 parts (first loads of the parts ahead of their
// weights do not change it).
constexpr int kMostParts = 256;

template <int D, bool F16, int RT, int TK>
__global__ __launch_bounds__(256) void paged_join_kernel(const AttnJob job) {
    constexpr int kT = D / 4, kSlices = 256 / kT;
    __shared__ float weight[kMostParts];
    __shared__ float4 sums[kSlices][kT];
    __shared__ float red[8];
    const PagedAttnParams& p = job.p;
    const int t = blockIdx.x / p.n_q_heads, hq = blockIdx.x % p.n_q_heads, tid = threadIdx.x;
    int n;
    int64_t at;
    if (!parts_of<RT, TK>(job, t, hq, n, at)) return;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (tid < n) ml = *reinterpret_cast<const float2*>(job.part_ml + (at + static_cast<int64_t>(tid) * RT) * 2);
    float top = ml.x;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float f = factor(ml.x, top == -INFINITY ? 0.0f : top);
    weight[tid] = f;
    float sum = ml.y * f;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
    __syncthreads();
    const int ch = 4 * (tid % kT), slice = tid / kT;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = slice; i < n; i += kSlices) add(a, *reinterpret_cast<const float4*>(job.part_o + (at + static_cast<int64_t>(i) * RT) * D + ch), weight[i]);
    sums[slice][tid % kT] = a;
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int i = 1; i < kSlices; ++i) add(a, sums[i][tid % kT], 1.0f);
    put_row<F16>(p, t, hq, ch, a, inverse((red[4] + red[5]) + (red[6] + red[7])));
}

namespace {
// Key tiles a part has at least: below this a part costs more than the time its neighbours save (one stream of 500 positions:
// 9.3 us whole, 10.3 us as two parts and their join).
constexpr int kMinChunk = 16;
// The same for 128 rows of many tiles, which a workgroup alone on its compute unit takes slowly (4 chunks of 61 tokens over 1609
// positions 28 us with parts of 16, 21 us with parts of 8 or 4; of fewer than 24 tiles the join takes what the parts give: 8
// chunks of 50 over 331 13 us whole, 20 us in parts of 4).
constexpr int kManyTiles = 24, kMinChunkMany = 6;
// Key tiles up to which one wave takes a row tile by itself (256 chunks of 10 frames under a window of 50: 13.5 us, with
// four waves 19.9 us).
constexpr int kOneWave = 4;

// More rows than 32 a sequence and head are taken in tiles of 128, a workgroup's four waves sharing the keys, or, where that
// leaves little for every compute unit, in tiles of 32: four times as many workgroups, whose waves have keys of their own and
// no barriers, at half the rate where the chip is full.  Little: so many products of 128 rows by 64 keys per compute unit.
// (70 rows of 8 sequences, 1.5 products a unit: 20.2 us in tiles of 128, 17.2 us in tiles of 32; 250 rows over 2700 positions, 8
// a unit: 35 and 61 us; 150 calls of 33 rows and more, most of them of some 20 us, are 14 % faster by this rule in the mean.)
constexpr int kLittle = 3, kLittle8 = 6;  // in halves of a product; 8-bit caches take a tile longer, which all rows wait for

int64_t little(const asrfe_ctx* ctx, bool e4m3) { return int64_t{64} * (e4m3 ? kLittle8 : kLittle) * ctx->num_cus; }

// row_tile 0: by the rules
AttnPlan plan_of(const asrfe_ctx* ctx, int n_heads, int n_tokens, int n_q_heads, int batch, int max_kv, int window, int sinks, bool e4m3, int row_tile) {
    AttnPlan a;
    const int64_t rows = static_cast<int64_t>(n_tokens) * (n_q_heads / n_heads), seqs = std::max(batch, 1);
    auto tiles_of = [&](int keys, bool masked) {
        const int64_t all = std::max<int64_t>(1, (static_cast<int64_t>(max_kv) + keys - 1) / keys);
        // what a row tile can see of a window: its keys, the tokens of the tile, and an end of a tile on either side
        const int64_t seen = static_cast<int64_t>(window) + sinks + n_tokens / seqs;
        return masked && window > 0 ? std::min(all, seen / keys + 3) : all;
    };
    a.row_tile = row_tile;
    if (row_tile == 0) {
        const double work = static_cast<double>(rows) * n_heads * static_cast<double>(tiles_of(64, true));
        a.row_tile = rows <= seqs * 16 ? 16 : rows <= seqs * 32 || work < static_cast<double>(little(ctx, e4m3)) ? 32 : 128;
    }
    a.key_tile = a.row_tile == 128 ? 64 : 32;
    a.n_tiles = static_cast<int>(rows / a.row_tile) + batch;
    const int64_t items = static_cast<int64_t>(a.n_tiles) * n_heads;
    const int64_t all = tiles_of(a.key_tile, false), tiles = tiles_of(a.key_tile, true);
    // enough parts for every compute unit to have several, so that sequences of different lengths even out
    const int64_t want = (a.row_tile == 128 ? 2 : 8) * ctx->num_cus;
    auto most_of = [&](int64_t n) {  // (not falling as n rises: the workspace is that of all tiles)
        const int least = a.row_tile == 128 && n >= kManyTiles ? kMinChunkMany : kMinChunk;
        return std::max<int64_t>(1, std::min<int64_t>({want / std::max<int64_t>(1, items), (n + least - 1) / least, kMostParts}));
    };
    a.most_split = static_cast<int>(most_of(all));
    a.chunk = static_cast<int>((tiles + most_of(tiles) - 1) / most_of(tiles));
    a.n_split = static_cast<int>((tiles + a.chunk - 1) / a.chunk);
    a.one_wave = a.row_tile != 128 && a.chunk <= kOneWave;
    return a;
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
}  // namespace

int64_t paged_attention_workspace(const asrfe_ctx* ctx, int head_dim, bool e4m3, int n_heads, int n_tokens, int n_q_heads, int batch, int max_kv) {
    auto bytes = [&](int row_tile) -> int64_t {
        const AttnPlan a = plan_of(ctx, n_heads, n_tokens, n_q_heads, batch, max_kv, 0, 0, e4m3, row_tile);
        if (a.most_split == 1) return 0;
        const int64_t rows = static_cast<int64_t>(a.n_tiles) * n_heads * a.most_split * a.row_tile;
        return align256(rows * head_dim * 4) + align256(rows * 8);
    };
    // (a call's window may turn tiles of 128 rows into tiles of 32)
    const int64_t rows = static_cast<int64_t>(n_tokens) * (n_q_heads / n_heads);
    const bool either = rows > static_cast<int64_t>(std::max(batch, 1)) * 32 && rows * n_heads < little(ctx, e4m3);
    return either ? std::max(bytes(32), bytes(128)) : bytes(0);
}

template <int D, bool F16, bool E4M3>
static int32_t launch_attn(asrfe_ctx* ctx, const AttnJob& job, const AttnPlan& a, hipStream_t s) {
    const int64_t items = static_cast<int64_t>(a.n_tiles) * job.p.c.n_heads, wgs = items * a.n_split;
    if (wgs * 256 > UINT32_MAX) return set_err(ctx, ASRFE_ERR_SHAPE, "paged_attention: too many rows and heads for one launch");
    const dim3 grid(static_cast<uint32_t>(wgs));
    if (a.row_tile == 16 && a.one_wave) hipLaunchKernelGGL((paged_attn_few_kernel<D, F16, E4M3, 1, 1>), grid, dim3(64), 0, s, job);
    else if (a.row_tile == 16) hipLaunchKernelGGL((paged_attn_few_kernel<D, F16, E4M3, 1, 4>), grid, dim3(256), 0, s, job);
    else if (a.row_tile == 32 && a.one_wave) hipLaunchKernelGGL((paged_attn_few_kernel<D, F16, E4M3, 2, 1>), grid, dim3(64), 0, s, job);
    else if (a.row_tile == 32) hipLaunchKernelGGL((paged_attn_few_kernel<D, F16, E4M3, 2, 4>), grid, dim3(256), 0, s, job);
    else hipLaunchKernelGGL((paged_attn_many_kernel<D, F16, E4M3>), grid, dim3(256), 0, s, job);
    if (int32_t rc = launched(ctx, "paged_attention")) return rc;
    if (a.n_split == 1) return ASRFE_OK;
    const int64_t rows = static_cast<int64_t>(job.p.n_tokens) * job.p.n_q_heads;  // (at most 2^30: checked at the entry)
    const bool few = a.n_split <= kFewParts;
    const dim3 jg(static_cast<uint32_t>(few ? (rows + 3) / 4 : rows));
#define JOIN(RT, TK)                                                                                              \
    do {                                                                                                          \
        if (few) hipLaunchKernelGGL((paged_join_few_kernel<D, F16, RT, TK>), jg, dim3(256), 0, s, job);           \
        else hipLaunchKernelGGL((paged_join_kernel<D, F16, RT, TK>), jg, dim3(256), 0, s, job);                   \
    } while (0)
    if (a.row_tile == 16) JOIN(16, 32);
    else if (a.row_tile == 32) JOIN(32, 32);
    else JOIN(128, 64);
#undef JOIN
    return launched(ctx, "paged_attention join");
}

int32_t launch_paged_attention(asrfe_ctx* ctx, const PagedAttnParams& p, int head_dim, int dtype, bool e4m3, void* ws, int max_kv,
                               hipStream_t s) {
    const AttnPlan a = plan_of(ctx, p.c.n_heads, p.n_tokens, p.n_q_heads, p.c.batch, max_kv, p.window, p.sinks, e4m3, 0);
    AttnJob job{};
    job.p = p;
    job.n_tiles = a.n_tiles;
    job.n_split = a.n_split;
    job.chunk = a.chunk;
    if (a.n_split > 1) {
        const int64_t rows = static_cast<int64_t>(a.n_tiles) * p.c.n_heads * a.n_split * a.row_tile;
        job.part_o = static_cast<float*>(ws);
        job.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + align256(rows * head_dim * 4));
    }
    const bool f16 = dtype == ASRFE_DT_F16;
    if (head_dim == 64) {
        if (f16) return e4m3 ? launch_attn<64, true, true>(ctx, job, a, s) : launch_attn<64, true, false>(ctx, job, a, s);
        return e4m3 ? launch_attn<64, false, true>(ctx, job, a, s) : launch_attn<64, false, false>(ctx, job, a, s);
    }
    if (f16) return e4m3 ? launch_attn<128, true, true>(ctx, job, a, s) : launch_attn<128, true, false>(ctx, job, a, s);
    return e4m3 ? launch_attn<128, false, true>(ctx, job, a, s) : launch_attn<128, false, false>(ctx, job, a, s);
}

}  // namespace asrfe
