// Attention of new rows over a paged cache, on the matrix cores.
//
//   o_i = sum_j p_ij v_j, p_i = softmax over the visible j of scale * q_i . k_j.
//
//   Rows.  The query heads that share a cache head read the same keys, so the rows of a product are (token, head of the
//   group) pairs: row r of a sequence is token r / group, head r % group.  A workgroup takes a tile of 128 rows (prompts:
//   four waves with 32 rows each share every key tile) or of 32 rows (single tokens and short chunks: every wave has the
//   same rows and key tiles of its own, so that four tiles are in flight and no barrier stands between them).
//
//   Keys.  One pass with a running maximum and sum.  Scores are formed transposed, S^T = K Q^T (v_mfma_f32_32x32x16), so a
//   lane holds the scores of one row; the weights are then already laid out as the operand of O^T = V^T P^T, V being read
//   transposed from the LDS.  Tiles arrive by 16-byte global -> LDS loads (16-bit caches) with the bank swizzle applied to
//   the source address, or through registers, where e4m3 codes become 16-bit values (exactly: the scales are powers of
//   two).  A tile is made of 16-position pieces, each inside one page, so pages may end anywhere in a tile.
//
//   Masks.  Only the tiles a mask's edge crosses (the causal diagonal, either end of the window, the end of the sequence,
//   a page that does not exist) look at positions; there, too, hidden values that are infinite or NaN are kept out of the
//   product (0 * inf).  Tiles no row of the workgroup sees are not loaded: a window's walk skips from the sinks to it.
//
//   Long caches with few rows are cut along the keys into parts, whose sums a second kernel joins.
#include <algorithm>

#include "lds_dma.h"
#include "paged_device.h"

namespace asrfe {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) int32_t* const_i32;

// The same address in scalar registers, for a value that is the same in every lane.
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
    return reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
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

// How a call is cut into workgroups.
struct AttnPlan {
    int row_tile;    // 32 or 128 rows
    int n_tiles;     // upper bound of the row tiles of all sequences
    int n_split;     // parts a tile's keys may be cut into
    int chunk;       // key tiles of a part
    int key_tile;    // 32 or 64 positions
};

struct AttnJob {
    PagedAttnParams p;
    int n_tiles, n_split, chunk;
    float* part_o;   // [item][part][row][D]
    float* part_ml;  // [item][part][row][2]: running maximum (scaled, base 2) and sum
};

// What a row tile covers.
struct TileSpan {
    int b, row0, n_rows, tok0, pos0, len;
    int sink_tiles, first, n_vt;  // key tiles: 0 .. sink_tiles - 1, then first ..; n_vt of them
};

// Row tile `tile` -> its sequence.  Sequence b's tiles start at cu_q[b] * group / row_tile + b: never fewer places than it
// needs, and the search for them is one comparison of 64 sequences per step.
template <int RT, int TK>
__device__ __forceinline__ bool tile_span(const PagedAttnParams& p, int tile, TileSpan& s) {
    const int lane = threadIdx.x & 63;
    int lo = 0, span = p.c.batch, step = 1;
    while (step * 64 < span) step *= 64;
    auto start = [&](int i) { return static_cast<int>(static_cast<int64_t>(p.c.cu_q[i]) * p.group / RT) + i; };
    for (;; step >>= 6) {
        const int i = lo + lane * step;
        const bool below = i < lo + span && start(i) <= tile;
        const int c = __builtin_popcountll(__ballot(below));
        if (c == 0) return false;
        lo += (c - 1) * step;
        const int left = span - (c - 1) * step;
        span = left < step ? left : step;
        if (step == 1) break;
    }
    s.b = __builtin_amdgcn_readfirstlane(lo);
    const int cu0 = __builtin_amdgcn_readfirstlane(p.c.cu_q[s.b]), cu1 = __builtin_amdgcn_readfirstlane(p.c.cu_q[s.b + 1]);
    const int kv = __builtin_amdgcn_readfirstlane(p.c.kv_lens[s.b]);
    const int64_t n_rows = static_cast<int64_t>((cu1 < p.n_tokens ? cu1 : p.n_tokens) - cu0) * p.group;
    const int64_t row0 = (static_cast<int64_t>(tile) - (static_cast<int64_t>(cu0) * p.group / RT + s.b)) * RT;
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

template <int D>
__device__ __forceinline__ int swz_k(int r) {
    return D == 128 ? (r & 15) : ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int swz_v(int r) {
    return D == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
}

template <int D, bool E4M3, int RW, int KW>
struct AttnShape {
    static constexpr int kWaves = RW * KW;
    static constexpr int kRowTile = 32 * RW;
    static constexpr int kKeys = RW == 1 ? 32 : 64;                // positions of a key tile
    static constexpr int kRowBytes = 2 * D;                        // of a position in the LDS
    static constexpr int kTile = kKeys * kRowBytes;                // one of K, V
    static constexpr int kBufs = E4M3 && RW == 1 ? 1 : 2;          // (e4m3, own tiles: the next one waits in registers)
    static constexpr int kGroupLds = kBufs * 2 * kTile;            // of the waves that share tiles
    static constexpr int kJoin = KW > 1 ? KW * (D / 2) * 256 + KW * 256 : 0;
    static constexpr int kLds = KW * kGroupLds > kJoin ? KW * kGroupLds : kJoin;
    static constexpr int kRpi = 1024 / kRowBytes;                  // rows one wave brings in with one load
    static constexpr int kLoads = kKeys / (RW * kRpi);             // loads per wave for one of K, V
    static constexpr int kVar = RW == 1 ? 16 / kRpi : 1;           // different places of a load inside its 16 rows
    static constexpr int kPieces = kKeys / 16;
    static constexpr int kPerCu = 160 * 1024 / kLds >= 2 ? 2 : 1;  // workgroups of a compute unit
    static constexpr int kWavesPerSimd = kPerCu * kWaves >= 8 ? 2 : 1;
};

template <int D, bool F16, bool E4M3, int RW, int KW>
__global__ __launch_bounds__(64 * RW * KW, (AttnShape<D, E4M3, RW, KW>::kWavesPerSimd)) void paged_attn_kernel(const AttnJob job) {
    using S = AttnShape<D, E4M3, RW, KW>;
    constexpr int kKeys = S::kKeys, kRowBytes = S::kRowBytes, kTile = S::kTile, kChunks = kRowBytes / 16, kMt = D / 32, kKk = kKeys / 32;
    __shared__ __attribute__((aligned(1024))) char smem[S::kLds];
    // (no saturate_fp16_conversions here: in that mode the matrix instructions lose infinities and NaN in their accumulators)
    const PagedAttnParams& p = job.p;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = RW == 1 ? 0 : wave, kw = RW == 1 ? wave : 0;
    // workgroups are dealt round-robin over the 8 XCDs: give each a contiguous range, row tiles of one head together
    const int nwg = gridDim.x, bid = blockIdx.x;
    const int xcd = bid & 7, xq = nwg >> 3, xr = nwg & 7;
    const int logical = (xcd < xr ? xcd * (xq + 1) : xr * (xq + 1) + (xcd - xr) * xq) + (bid >> 3);
    const int part = logical % job.n_split, item = logical / job.n_split;
    const int tile = item % job.n_tiles, kvh = item / job.n_tiles;
    TileSpan ts;
    if (!tile_span<32 * RW, kKeys>(p, tile, ts)) return;
    const int n_parts = ts.n_vt <= job.chunk ? 1 : (ts.n_vt + job.chunk - 1) / job.chunk;
    if (part >= n_parts) return;
    const int vt0 = part * job.chunk, vt1 = vt0 + job.chunk < ts.n_vt ? vt0 + job.chunk : ts.n_vt;

    // ---- this wave's rows, this lane's row
    const int rbase = ts.row0 + rw * 32;
    const bool has_rows = rbase < ts.n_rows;
    const int row = rbase + l31 < ts.n_rows ? rbase + l31 : ts.n_rows - 1;
    const int tok = row / p.group, hq = kvh * p.group + row % p.group;
    const int pos = ts.pos0 + tok;
    const int wlast = rbase + 31 < ts.n_rows ? rbase + 31 : ts.n_rows - 1;
    const int pmin = __builtin_amdgcn_readfirstlane(ts.pos0 + rbase / p.group), pmax = __builtin_amdgcn_readfirstlane(ts.pos0 + wlast / p.group);
    auto hi_of = [&](int i) { return i < 0 ? 0 : (p.causal && i + 1 < ts.len ? i + 1 : ts.len); };
    auto lo_of = [&](int i) { return p.window > 0 && i - p.window + 1 > 0 ? i - p.window + 1 : 0; };
    const int hi = hi_of(pos), lo = lo_of(pos);
    const int w_hi_min = hi_of(pmin), w_hi_max = hi_of(pmax), w_lo_min = lo_of(pmin), w_lo_max = lo_of(pmax);

    // ---- key tiles: where their pieces lie
    const const_i32 table = (const_i32)(p.c.block_table + static_cast<int64_t>(ts.b) * p.c.table_stride);
    const int page_mask = (1 << p.c.page_shift) - 1;
    struct Pieces {
        int64_t row[S::kPieces];
        uint32_t valid;
    };
    auto key0_of = [&](int vt) { return (vt < ts.sink_tiles ? vt : ts.first + vt - ts.sink_tiles) * kKeys; };
    auto pieces_of = [&](int vt) {
        Pieces r;
        r.valid = 0;
        const int key0 = key0_of(vt);
#pragma unroll
        for (int g = 0; g < S::kPieces; ++g) {
            const int key = key0 + 16 * g, i = key >> p.c.page_shift;
            const int page = table[i < p.c.table_stride ? i : p.c.table_stride - 1];
            const bool ok = i < p.c.table_stride && page >= 0 && page < p.c.n_pages;
            r.valid |= ok ? 1u << g : 0u;
            r.row[g] = ((static_cast<int64_t>(ok ? page : 0) * p.c.n_heads + kvh) << p.c.page_shift) + (key & page_mask);
        }
        return r;
    };

    // LDS addresses.  A row's 16-byte pieces are swizzled by functions of the row that are linear over its bits, so every
    // address below is one base per lane, an exclusive or with a constant and a constant offset.  The bases are hidden from
    // the compiler where they are used: it would keep each sum in a register of its own through the loop, and spill.
    const uint32_t own_base = __builtin_amdgcn_readfirstlane(lds_addr_of(smem + kw * S::kGroupLds));
    // 16-bit caches, straight into the LDS: load i of this wave covers rows (i * RW + rw) * kRpi .. + kRpi - 1 of the tile,
    // a lane 16 bytes; the place in the LDS follows the lane, so the swizzle is applied to the source (K and V differ)
    const int lrow = lane / kChunks, lchunk = lane % kChunks;
    uint32_t voff_k[S::kVar], voff_v[S::kVar];
#pragma unroll
    for (int i = 0; i < S::kVar; ++i) {
        const int r = ((RW == 1 ? i : rw) * S::kRpi & 15) + lrow;
        voff_k[i] = r * kRowBytes + (lchunk ^ swz_k<D>(r)) * 16;
        voff_v[i] = r * kRowBytes + (lchunk ^ swz_v<D>(r)) * 16;
    }
    auto issue16 = [&](const Pieces& pc, int buf) {
        const uint32_t dst = __builtin_amdgcn_readfirstlane(own_base + buf * 2 * kTile + rw * 1024);
        static_for<S::kLoads>([&](auto ic) {
            constexpr int I = decltype(ic)::value;
            int64_t at;
            if constexpr (RW * S::kRpi == 32) {
                const int64_t even = pc.row[2 * I], odd = pc.row[2 * I + 1];
                at = rw & 2 ? odd : even;
            } else {
                at = pc.row[I * RW * S::kRpi / 16];
            }
            lds_dma16(uniform(p.c.k + at * kRowBytes), voff_k[I % S::kVar], dst + I * RW * 1024);
            lds_dma16(uniform(p.c.v + at * kRowBytes), voff_v[I % S::kVar], dst + kTile + I * RW * 1024);
        });
    };
    // e4m3, through registers: a lane takes 16 codes of each of kLoads8 consecutive rows, so their exponents lie side by side
    constexpr int kLpr = D / 16, kLoads8 = kKeys / RW * kLpr / 64;
    const int r8 = (lane / kLpr) * kLoads8, c8 = lane % kLpr;  // first row (of the wave's), pair of 16-byte pieces
    u32x4 k8[E4M3 ? kLoads8 : 1], v8[E4M3 ? kLoads8 : 1];
    uint32_t ke8 = 0, ve8 = 0;
    auto issue8 = [&](const Pieces& pc) {
        if constexpr (E4M3) {
            int64_t at = pc.row[0];
            const int piece = RW == 1 ? r8 >> 4 : rw;
#pragma unroll
            for (int g = 1; g < S::kPieces; ++g) {
                const int64_t x = pc.row[g];
                at = piece == g ? x : at;
            }
            at += r8 & 15;
            const char* kp = p.c.k + at * D + 16 * c8;
            const char* vp = p.c.v + at * D + 16 * c8;
#pragma unroll
            for (int i = 0; i < kLoads8; ++i) {
                k8[i] = *reinterpret_cast<const u32x4*>(kp + i * D);
                v8[i] = *reinterpret_cast<const u32x4*>(vp + i * D);
            }
            using E = std::conditional_t<kLoads8 == 4, uint32_t, std::conditional_t<kLoads8 == 2, uint16_t, uint8_t>>;
            ke8 = *reinterpret_cast<const E*>(p.c.k_exp + at);
            ve8 = *reinterpret_cast<const E*>(p.c.v_exp + at);
        }
    };
    const int r8w = (RW == 1 ? 0 : rw * 16) + r8;
    const uint32_t put_k = r8w * kRowBytes + ((2 * c8) ^ swz_k<D>(r8w)) * 16, put_v = r8w * kRowBytes + ((2 * c8) ^ swz_v<D>(r8w)) * 16;
    auto put8 = [&](uint32_t tile_base) {
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
            // a scale of 2^8 or more can lead out of fp16's range (bytes of 135 or more: bit 7, and 7 in the rest)
            auto big = [](uint32_t x) { return x & 0x80808080u & ((x & 0x7f7f7f7fu) + 0x79797979u); };
            if (F16 && __any((big(ke8) | big(ve8)) != 0)) put(std::true_type{});
            else put(std::false_type{});
        }
    };

    // ---- first tile, queries
    constexpr int kStep = KW;
    int vt = vt0 + kw;
    uint32_t valid = 0;  // of the tile that is about to be used: which of its pieces exist
    if (vt < vt1) {
        const Pieces pc = pieces_of(vt);
        valid = pc.valid;
        if constexpr (E4M3) issue8(pc);
        else issue16(pc, 0);
    }
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
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[mt][e] = 0.0f;
    float mc = -INFINITY, l_run = 0.0f;  // running maximum (scaled, base 2) and sum of this lane's half of the keys

    auto compute = [&](uint32_t tile_base, int key0, uint32_t valid, auto edge_c) __attribute__((always_inline)) {
        constexpr bool edge = decltype(edge_c)::value;
        f32x16 sacc[kKk];
#pragma unroll
        for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
            for (int e = 0; e < 16; ++e) sacc[kk][e] = 0.0f;
        uint32_t kb = tile_base + get_k;
        asm volatile("" : "+v"(kb));
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int kk = 0; kk < kKk; ++kk) {
                const u16x8 kf = *lds<const u16x8>((kb ^ (s << 5)) + kk * 32 * kRowBytes);
                sacc[kk] = mfma32<F16>(kf, qf[s], sacc[kk]);
            }
        if constexpr (edge) {
#pragma unroll
            for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = key0 + kk * 32 + (e & 3) + 8 * (e >> 2) + 4 * h;
                    const bool see = (j < hi) & ((j >= lo) | (j < p.sinks)) & (((valid >> (kk * 2 + (e >> 3))) & 1) != 0);
                    sacc[kk][e] = see ? sacc[kk][e] : -INFINITY;
                }
        }
        float rmax = sacc[0][0];
#pragma unroll
        for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
            for (int e = 0; e < 16; ++e) rmax = fmaxf(rmax, sacc[kk][e]);
        {   // the row's other keys sit in lane ^ 32
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(rmax), __float_as_uint(rmax), false, false);
            rmax = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        }
        // the maximum only has to keep exp2 in range: it is raised when a tile exceeds it by more than 2^8
        const bool grew = rmax * c > mc + 8.0f;
        const float m_new = grew ? rmax * c : mc;
        const float alpha = grew ? __builtin_amdgcn_exp2f(mc - m_new) : 1.0f;
        mc = m_new;
        const float sub = mc == -INFINITY ? 0.0f : mc;  // (nothing seen yet: every weight below is exp2(-inf))
        if (__any(grew)) {
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[mt][e] *= alpha;
        }
        float psum = 0.0f;
        u32x4 pf[kKk][2];
#pragma unroll
        for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float a = __builtin_amdgcn_exp2f(fmaf(sacc[kk][8 * s2 + j], c, -sub));
                    const float b = __builtin_amdgcn_exp2f(fmaf(sacc[kk][8 * s2 + j + 1], c, -sub));
                    psum += a + b;
                    pf[kk][s2][j / 2] = pack_elem2<F16>(a, b);
                }
        l_run = l_run * alpha + psum;
#pragma unroll
        for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) asm volatile("" : "+v"(pf[kk][s2]));  // (packed here: not in 32 bits up to their use)
        uint32_t vb = tile_base + kTile + get_v;
        asm volatile("" : "+v"(vb));
        auto v_frag = [&](int kk, int s2, int mt) {  // rows 8 x + 4 h + q of the 16: the swizzle turns by 2 x, the channels by 4 mt
            const uint32_t at = vb ^ (mt * 64);
            const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<v4s>(at + (kk * 32 + s2 * 16) * kRowBytes));
            const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<v4s>((at ^ 32) + (kk * 32 + s2 * 16 + 8) * kRowBytes));
            return __builtin_bit_cast(u16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // A 16-bit element whose exponent field is all ones carries into its sign bit when one is added below the field.
        constexpr uint32_t kExp = (F16 ? 0x7c00u : 0x7f80u) * 0x10001u, kUnit = (F16 ? 0x0400u : 0x0080u) * 0x10001u;
        constexpr uint32_t kMant = kUnit - 0x10001u, kSign = 0x80008000u, kRest = 0x7fff7fffu, kOne = F16 ? 0x3c00u : 0x3f80u;
        bool special = false;
        if constexpr (edge) {
            uint32_t any = 0;
#pragma unroll
            for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
#pragma unroll
                    for (int mt = 0; mt < kMt; ++mt) {
                        const u32x4 w = __builtin_bit_cast(u32x4, v_frag(kk, s2, mt));
                        const u32x4 t = (w & kExp) + kUnit;
                        any |= t[0] | t[1] | t[2] | t[3];
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            special = __any((any & kSign) != 0);
        }
        if (!special) {
#pragma unroll
            for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                    for (int mt = 0; mt < kMt; ++mt) oacc[mt] = mfma32<F16>(v_frag(kk, s2, mt), __builtin_bit_cast(u16x8, pf[kk][s2]), oacc[mt]);
        } else {
            // Infinities and NaN in V: the finite part as usual, then, for each kind of the others, a product of
            // indicators tells which (channel, row) pairs meet one under a weight that is not zero.
#pragma unroll
            for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const u32x4 on = ((((pf[kk][s2] & kRest) + kRest) & kSign) >> 15) * kOne;
#pragma unroll
                    for (int mt = 0; mt < kMt; ++mt) {
                        const u32x4 v = __builtin_bit_cast(u32x4, v_frag(kk, s2, mt));
                        const u32x4 odd = ((v & kExp) + kUnit) & kSign, nan = ((v & kMant) + kRest) & odd;
                        oacc[mt] = mfma32<F16>(__builtin_bit_cast(u16x8, v & ~((odd >> 15) * 0xffffu)), __builtin_bit_cast(u16x8, pf[kk][s2]), oacc[mt]);
#pragma unroll
                        for (int t = 0; t < 3; ++t) {
                            const u32x4 is = t == 0 ? (odd & ~nan & ~v) : t == 1 ? (odd & ~nan & v) : nan;
                            f32x16 n;
#pragma unroll
                            for (int e = 0; e < 16; ++e) n[e] = 0.0f;
                            n = mfma32<F16>(__builtin_bit_cast(u16x8, (is >> 15) * kOne), __builtin_bit_cast(u16x8, on), n);
                            const float add = t == 0 ? INFINITY : t == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
                            for (int e = 0; e < 16; ++e) oacc[mt][e] += n[e] > 0.0f ? add : 0.0f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
        }
    };

    int buf = 0;
    while (vt < vt1) {
        const int next = vt + kStep;
        const bool more = next < vt1;
        if constexpr (E4M3) {
            put8(own_base + buf * 2 * kTile);
            if (RW > 1) __syncthreads();
            else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
            // this wave's loads of the tile are in, and its reads of the tile before are done with the other buffer
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            if (RW > 1) __syncthreads();
        }
        const uint32_t now = valid;
        if (more) {
            const Pieces pc = pieces_of(next);
            valid = pc.valid;
            if constexpr (E4M3) issue8(pc);
            else issue16(pc, buf ^ 1);
        }
        const int key0 = key0_of(vt);
        // (hidden from every row of the wave: the end of a prompt's shorter rows)
        if (has_rows && key0 < w_hi_max && (key0 + kKeys > w_lo_min || key0 < p.sinks)) {
            const bool inside = key0 + kKeys <= w_hi_min && (key0 >= w_lo_max || key0 + kKeys <= p.sinks) && now == (1u << S::kPieces) - 1;
            if (inside) compute(own_base + buf * 2 * kTile, key0, now, std::false_type{});
            else compute(own_base + buf * 2 * kTile, key0, now, std::true_type{});
        }
        if (S::kBufs == 2) buf ^= 1;
        vt = next;
    }

    // ---- results: lane (l31, h) holds of its row the channels 32 mt + 8 (e >> 2) + 4 h + (e & 3)
    float l_tot = l_run + __shfl_xor(l_run, 32);
    float* po = job.part_o + ((static_cast<int64_t>(item) * job.n_split + part) * S::kRowTile + rw * 32 + l31) * D;
    float* pml = job.part_ml + ((static_cast<int64_t>(item) * job.n_split + part) * S::kRowTile + rw * 32 + l31) * 2;
    uint16_t* out = p.out + (ts.tok0 + tok) * p.o_ts + hq * p.o_hs;
    const bool mine = has_rows && rbase + l31 < ts.n_rows;
    auto store = [&](int f, float a, float b, float cc, float d, float inv) {  // channels of flat accumulator index f .. f + 3
        const int ch = 32 * (f >> 4) + 8 * ((f & 15) >> 2) + 4 * h;
        if (n_parts == 1) {
            const uint2 w = make_uint2(pack_result<F16>(a * inv, b * inv), pack_result<F16>(cc * inv, d * inv));
            if (mine) *reinterpret_cast<uint2*>(out + ch) = w;
        } else if (mine) {
            *reinterpret_cast<float4*>(po + ch) = make_float4(a, b, cc, d);
        }
    };
    if constexpr (KW == 1) {
        const float inv = l_tot > 0.0f ? 1.0f / l_tot : (l_tot == 0.0f ? 0.0f : l_tot);
#pragma unroll
        for (int f = 0; f < 16 * kMt; f += 4) store(f, oacc[f >> 4][f & 15], oacc[f >> 4][(f & 15) + 1], oacc[f >> 4][(f & 15) + 2], oacc[f >> 4][(f & 15) + 3], inv);
        if (n_parts > 1 && mine && h == 0) *reinterpret_cast<float2*>(pml) = make_float2(mc, l_tot);
    } else {
        // the waves' sums are brought to one maximum and added through the LDS
        constexpr int kN = 16 * kMt, kOwn = kN / KW;
        float* ml = reinterpret_cast<float*>(smem);
        float* os = ml + KW * 64;
        __syncthreads();  // all waves are done with their tiles
        if (h == 0) {
            ml[wave * 64 + l31] = mc;
            ml[wave * 64 + 32 + l31] = l_tot;
        }
        __syncthreads();
        float top = mc, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < KW; ++i) top = fmaxf(top, ml[i * 64 + l31]);
        const float sub = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int i = 0; i < KW; ++i) sum += ml[i * 64 + 32 + l31] * __builtin_amdgcn_exp2f(ml[i * 64 + l31] - sub);
        const float f0 = __builtin_amdgcn_exp2f(mc - sub);
#pragma unroll
        for (int f = 0; f < kN; f += 4)
            *reinterpret_cast<float4*>(os + ((wave * (kN / 4) + f / 4) * 64 + lane) * 4) =
                make_float4(oacc[f >> 4][f & 15] * f0, oacc[f >> 4][(f & 15) + 1] * f0, oacc[f >> 4][(f & 15) + 2] * f0, oacc[f >> 4][(f & 15) + 3] * f0);
        __syncthreads();
        const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
        for (int x = 0; x < kOwn; x += 4) {
            const int f = wave * kOwn + x;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const float4 t = *reinterpret_cast<const float4*>(os + ((i * (kN / 4) + f / 4) * 64 + lane) * 4);
                a.x += t.x; a.y += t.y; a.z += t.z; a.w += t.w;
            }
            store(f, a.x, a.y, a.z, a.w, inv);
        }
        if (n_parts > 1 && mine && h == 0 && wave == 0) *reinterpret_cast<float2*>(pml) = make_float2(top, sum);
    }
}

// Joins the parts of a row tile: a thread has 4 channels of a row.
template <int D, bool F16, int RT, int TK>
__global__ __launch_bounds__(256) void paged_join_kernel(const AttnJob job) {
    const PagedAttnParams& p = job.p;
    const int item = blockIdx.x, tile = item % job.n_tiles, kvh = item / job.n_tiles;
    TileSpan ts;
    if (!tile_span<RT, TK>(p, tile, ts)) return;
    const int n_parts = (ts.n_vt + job.chunk - 1) / job.chunk;
    if (ts.n_vt <= job.chunk) return;
    constexpr int kT = D / 4;
    const int d = 4 * (threadIdx.x % kT);
    for (int r = threadIdx.x / kT; r < RT && ts.row0 + r < ts.n_rows; r += 256 / kT) {
        const int64_t base = static_cast<int64_t>(item) * job.n_split * RT + r;
        float top = -INFINITY;
        for (int i = 0; i < n_parts; ++i) top = fmaxf(top, job.part_ml[(base + static_cast<int64_t>(i) * RT) * 2]);
        const float sub = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int i = 0; i < n_parts; ++i) {
            const int64_t at = base + static_cast<int64_t>(i) * RT;
            const float2 ml = *reinterpret_cast<const float2*>(job.part_ml + at * 2);
            const float4 o = *reinterpret_cast<const float4*>(job.part_o + at * D + d);
            const float f = __builtin_amdgcn_exp2f(ml.x - sub);
            sum = fmaf(ml.y, f, sum);
            a.x = fmaf(o.x, f, a.x);
            a.y = fmaf(o.y, f, a.y);
            a.z = fmaf(o.z, f, a.z);
            a.w = fmaf(o.w, f, a.w);
        }
        const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
        const int row = ts.row0 + r, tok = row / p.group, hq = kvh * p.group + row % p.group;
        uint16_t* out = p.out + (ts.tok0 + tok) * p.o_ts + hq * p.o_hs + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_result<F16>(a.x * inv, a.y * inv), pack_result<F16>(a.z * inv, a.w * inv));
    }
}

namespace {
// Key tiles a part has at least: below this a part costs more than the time its neighbours save.
constexpr int kMinChunk = 8;

AttnPlan plan_of(const asrfe_ctx* ctx, int n_heads, int n_tokens, int n_q_heads, int batch, int max_kv) {
    AttnPlan a;
    const int64_t rows = static_cast<int64_t>(n_tokens) * (n_q_heads / n_heads);
    // up to 32 rows per sequence and head: the waves of a workgroup share the rows instead of the keys
    a.row_tile = batch > 0 && rows <= static_cast<int64_t>(batch) * 32 ? 32 : 128;
    a.key_tile = a.row_tile == 32 ? 32 : 64;
    a.n_tiles = static_cast<int>(rows / a.row_tile) + batch;
    const int64_t items = static_cast<int64_t>(a.n_tiles) * n_heads;
    const int64_t tiles = std::max<int64_t>(1, (static_cast<int64_t>(max_kv) + a.key_tile - 1) / a.key_tile);
    // enough parts for every compute unit to have several, so that sequences of different lengths even out
    const int64_t want = a.row_tile == 32 ? 16 * ctx->num_cus : 2 * ctx->num_cus;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>({want / std::max<int64_t>(1, items), (tiles + kMinChunk - 1) / kMinChunk, 256}));
    a.chunk = static_cast<int>((tiles + most - 1) / most);
    a.n_split = static_cast<int>((tiles + a.chunk - 1) / a.chunk);
    return a;
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
}  // namespace

int64_t paged_attention_workspace(const asrfe_ctx* ctx, int head_dim, int n_heads, int n_tokens, int n_q_heads, int batch, int max_kv) {
    const AttnPlan a = plan_of(ctx, n_heads, n_tokens, n_q_heads, batch, max_kv);
    if (a.n_split == 1) return 0;
    const int64_t rows = static_cast<int64_t>(a.n_tiles) * n_heads * a.n_split * a.row_tile;
    return align256(rows * head_dim * 4) + align256(rows * 8);
}

template <int D, bool F16, bool E4M3>
static int32_t launch_attn(asrfe_ctx* ctx, const AttnJob& job, const AttnPlan& a, hipStream_t s) {
    const int64_t items = static_cast<int64_t>(a.n_tiles) * job.p.c.n_heads, wgs = items * a.n_split;
    if (wgs > INT32_MAX) return set_err(ctx, ASRFE_ERR_SHAPE, "paged_attention: too many rows and heads for one launch");
    const dim3 grid(static_cast<uint32_t>(wgs));
    if (a.row_tile == 32) hipLaunchKernelGGL((paged_attn_kernel<D, F16, E4M3, 1, 4>), grid, dim3(256), 0, s, job);
    else hipLaunchKernelGGL((paged_attn_kernel<D, F16, E4M3, 4, 1>), grid, dim3(256), 0, s, job);
    if (int32_t rc = launched(ctx, "paged_attention")) return rc;
    if (a.n_split == 1) return ASRFE_OK;
    const dim3 jg(static_cast<uint32_t>(items));
    if (a.row_tile == 32) hipLaunchKernelGGL((paged_join_kernel<D, F16, 32, 32>), jg, dim3(256), 0, s, job);
    else hipLaunchKernelGGL((paged_join_kernel<D, F16, 128, 64>), jg, dim3(256), 0, s, job);
    return launched(ctx, "paged_attention join");
}

int32_t launch_paged_attention(asrfe_ctx* ctx, const PagedAttnParams& p, int head_dim, int dtype, bool e4m3, void* ws, int max_kv,
                               hipStream_t s) {
    const AttnPlan a = plan_of(ctx, p.c.n_heads, p.n_tokens, p.n_q_heads, p.c.batch, max_kv);
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
