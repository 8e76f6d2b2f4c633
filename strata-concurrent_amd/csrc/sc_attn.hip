// sc_attn.hip - attention of one new token a sequence over its paged cache (sc_attn_decode_async).
//
// With scores x_j = scale * q . k_j * log2(e) over the cells left by the length, the window and the page table, a part of
// them gives l = sum 2^(x_j - m) and o = sum 2^(x_j - m) v_j for a reference m near its largest score; parts join by
// bringing them to one m, and out = o / l.  A kv head's query heads share its cells, so both products are matrix products:
// scores [cells] x [16 heads], outputs [values] x [16 heads].  What bounds a call is reading the cache once.
//
// A wave takes 32 cells a turn, its rows straight from memory into the matrix instructions' operands, nothing through LDS:
//   scores   A = keys (row = cell, 8 consecutive values a lane), B = queries; a lane ends with the scores of one head
//            (lane % 16) for cells 4 g + i and 16 + 4 g + i, g = lane / 16, i < 4;
//   outputs  A = values transposed (row = value index, 8 cells a lane), B = probabilities.  The products' cells may come
//            in any order that both agree on, so the lane's eight cells are the ones whose scores it already holds, and its
//            A operand is an 8 x 8 block of the cache that it loads as 16-byte rows and transposes in its registers.
// The head is the lane's column in both results, so the running statistics are the lane's own: only the largest score of a
// turn crosses lanes (two swaps), and bringing o to a new m is a product by the lane's own factor.
//
// Rows that are read once go past the caches' keeping: values that are loaded by 16 bytes (262 us for 1.5 GB of eight
// sequences where they do not, 236 where they do), keys in int8 (42.3 and 38.8 us for 135 MB), but not in f16, where a row's
// 512 bytes are read by instructions of 64 of them (245 us where they do, 236).  Measured, 2 kv heads of 256 and 24 query
// heads: 1.5 GB of f16 rows in 236 us, 6.4 TB/s where reading alone reaches 6.9; 135 MB of int8 rows in 39 us, where a call
// whose workgroups take one turn each takes 12.5.
//
// Accuracy: weights and f32 queries enter the matrix instructions as two f16 parts, each rounded to nearest; keys, values and
// f16 queries are exact, int8 codes are exact in f16 and their scales are applied in f32; sums are in 32 bits.  f16 is a fixed
// point below 2^-14, so the reference m follows the turn's weights (the constants below): a cell that outweighs the rest by
// 2^80 takes no bit from them.  Infinities: an infinite value may meet a weight's part that is 0, an infinite key a query's
// second part of the other sign, and make a NaN where the formula has an infinity.  A wave whose sums are no finite numbers goes
// over its turns again with weights as they are, by 32-bit products; no weight is 0 there, unless it is below 2^-126 of the
// part's largest.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "sc_attn_split.hpp"
#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();
constexpr int kAttnThreads = kAttnWaves * 64;
// Log2 of a turn's weights, relative to m: at most kMost, at least kLeast.  Two f16 parts keep a weight to 2^-23 of itself from
// 2^-2 on, and to 2^-17 from 2^kLeast on.  Where a turn's leave that range m moves, up or down by whole numbers, so that the
// largest is about kTop, or kDeep where the least would be too small; but it is never more than kFar below the largest of all:
// what is summed stays below 2^125.  Cells that are too small even then, and below kWait (an int8 cell's weights differ by its
// blocks' scales), wait for another go at the same turn, with an m of their own: each go takes its largest, so there is an end.
constexpr float kTop = 11.0f, kDeep = 14.0f, kMost = 15.0f, kLeast = -8.0f, kWait = 5.0f, kFar = 76.0f;
constexpr float kNear = 12.0f, kNearBy = 0x1p12f;
constexpr float kTiny = 0x1p-126f;

// 2^x by the hardware's instruction (1 unit in the last place; results below the normal range are 0).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool rarely(bool x) { return __builtin_expect(x, false); }
// 2^(a - b), at least the smallest normal number, which changes no sum but leaves infinities what they are; nothing weighs
// nothing.
__device__ __forceinline__ float weight(float a, float b) { return a == -kInf ? 0.0f : fmaxf(exp2_fast(a - b), kTiny); }
// Log of a sum of 2^(x - m), natural.  The sum's exponent goes to m, a whole number as well: added to the logarithm, which can
// be 20 from m's other sign, it would take the bits of a result near 0.
__device__ __forceinline__ float log_of_sum(float m, float sum) {
    float e = float(__builtin_amdgcn_frexp_expf(sum)), f = __builtin_amdgcn_frexp_mantf(sum);
    if (f < 0.70710678f) f *= 2, e -= 1;
    return sum == 0 ? -kInf : ((m + e) + __builtin_log2f(f)) * kLn2;
}
__device__ __forceinline__ float min_of(float a, float b) { return fminf(a, b); }

// ---- which cells a workgroup takes ------------------------------------------------------------------------------------

__device__ __forceinline__ Span span_of(const AttnArgs& a, int64_t n) { return cells_of(n, a.max_len, a.window); }

// The workgroups of a sequence are its parts times its tiles (kv heads and tiles of query heads), the tiles of a part next
// to each other: they read the same pages.
struct Place {
    uint32_t s, parts;    // sequence, how many parts its units are in
    uint32_t wg0, ws0;    // its first workgroup, and the first one's place in the workspace (parts > 1)
    Span span;
};
// The units of all sequences are shared out among about `slots` workgroups: a part takes `per` units at most, `per` being
// what one of them would get, so long and short sequences of a ragged batch give parts of like size.  Every workgroup
// finds its place from the lengths alone: one load a lane and a few scans for 64 sequences.
__device__ __forceinline__ bool place_of(const AttnArgs& a, uint32_t lane, uint32_t wg, Place& p) {
    auto length = [&](uint32_t s) { return s < a.n_seqs ? ld_global<int64_t>(a.lens + s) : int64_t(0); };
    const int64_t mine = length(lane);   // kept for batches of 64
    const uint32_t my_units = span_of(a, mine).units;
    uint32_t sum = my_units;             // at most 2^24 units a sequence and 16 sequences a lane
    for (uint32_t base = 64; base < a.n_seqs; base += 64) sum += span_of(a, length(base + lane)).units;
    const uint64_t total = uint64_t(last_lane(scan_add(sum & 0xFFFFFFu))) + (uint64_t(last_lane(scan_add(sum >> 24))) << 24);
    uint32_t per = units_of_part(total, a.tiles, a.slots, a.least);
    auto parts_of = [&](uint32_t s, uint32_t units) { return s >= a.n_seqs ? 0u : parts_of_units(units, per); };
    if (parts_fit(a.n_seqs, a.tiles, a.slots))
        while (last_lane(scan_add(parts_of(lane, my_units))) * a.tiles > a.slots) per = wider_part(per);
    uint32_t wgs = 0, ids = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 64) {
        const int64_t n = base ? length(base + lane) : mine;
        const uint32_t parts = parts_of(base + lane, base ? span_of(a, n).units : my_units), more = parts > 1 ? parts : 0u;
        const uint32_t w = scan_add(parts), d = scan_add(more);
        const uint32_t lo = wgs + (w - parts) * a.tiles, hi = wgs + w * a.tiles;
        const uint64_t here = __ballot(wg >= lo && wg < hi);
        if (here) {
            const int at = __builtin_ctzll(here);
            p.s = __builtin_amdgcn_readfirstlane(base + at);
            p.parts = __builtin_amdgcn_readlane(parts, at);
            p.wg0 = __builtin_amdgcn_readlane(lo, at);
            p.ws0 = ids + __builtin_amdgcn_readlane(d - more, at) * a.tiles;
            p.span = span_of(a, int64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(n)), at)) |
                                        uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(uint64_t(n) >> 32)), at))) << 32));
            return true;
        }
        wgs += last_lane(w) * a.tiles;
        ids += last_lane(d) * a.tiles;
    }
    return false;
}

// ---- a wave's turn ------------------------------------------------------------------------------------------------------

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ f16x2 two(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
__device__ __forceinline__ uint32_t bits(f16x2 h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ f16x8 eight(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(f16x8, ops_u32x4{a, b, c, d});
}
// Two f16 parts of eight values: the value rounded to nearest, and what that left out rounded likewise.
__device__ __forceinline__ void split8(const float (&p)[8], f16x8& hi, f16x8& lo) {
    uint32_t h[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = bits(f16x2{_Float16(p[2 * i]), _Float16(p[2 * i + 1])});
        asm("" : "+v"(h[i]));   // what is left out is of this, not of a product that the compiler would round once more
        const f16x2 t = two(h[i]);
        r[i] = bits(f16x2{_Float16(p[2 * i] - float(t.x)), _Float16(p[2 * i + 1] - float(t.y))});
    }
    hi = eight(h[0], h[1], h[2], h[3]);
    lo = eight(r[0], r[1], r[2], r[3]);
}
// The largest of a cell's f16 scales, which are not negative, and the least but one less; and their exponents, as bounds.
template <int kBlocks>
__device__ __forceinline__ void scales_of(const uint32_t (&s)[2], u16x2& hi, u16x2& lo) {
#pragma unroll
    for (int i = 0; i < (kBlocks > 2 ? 2 : 1); ++i) {
        const uint32_t w = (kBlocks == 1 ? s[i] | s[i] << 16 : s[i]) & 0x7FFF7FFFu;
        const u16x2 a = __builtin_bit_cast(u16x2, w);
        hi = __builtin_elementwise_max(hi, a);
        lo = __builtin_elementwise_min(lo, u16x2(a - u16x2{1, 1}));
    }
}
__device__ __forceinline__ float exponent_most(u16x2 hi) { return float(int(max(uint32_t(hi.x), uint32_t(hi.y)) >> 10) - 14); }
__device__ __forceinline__ float exponent_least(u16x2 lo) {
    const uint32_t e = min(uint32_t(lo.x), uint32_t(lo.y)) >> 10;
    return e ? float(int(e) - 15) : -24.0f;
}
// A tile of values by eight cells' weights, in two parts; or as they are, by 32-bit products at a quarter of the rate, where no
// weight is 0, so that an infinite value of little weight is infinite.
template <bool kAsIs>
__device__ __forceinline__ void add_values(f32x4& o, f16x8 v, const float (&p)[8], f16x8 hi, f16x8 lo) {
    if constexpr (kAsIs) {
#pragma unroll
        for (int n = 0; n < 8; ++n) o = mfma_f32(float(v[n]), fmaxf(p[n], kTiny), o);
    } else {
        o = mfma(v, hi, o);
        o = mfma(v, lo, o);
    }
}

// Four int8 codes with 128 added (one exclusive or) as f16: 0x64 above a byte is 1024 + the byte, exactly.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& a, uint32_t& b) {
    const f16x2 off = two(0xE480E480u);   // -1152
    a = bits(two(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off);
    b = bits(two(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off);
}

template <int D, bool kInt8>
struct Rows {
    // f16: 16 bytes of 32 values a step; int8: 16 bytes of 64 values a step
    static constexpr int kKeySteps = kInt8 ? D / 64 : D / 32;
    // f16: D / 16 consecutive values a lane in pieces of 16 bytes; int8: 4 values of every block of 64
    static constexpr int kValWords = kInt8 ? 1 : D >= 128 ? 4 : 2, kValPieces = kInt8 ? D / 64 : D >= 128 ? D / 128 : 1;
    ops_u32x4 k[2][kKeySteps];
    uint32_t v[8][kValPieces][kValWords];
    uint32_t ks[kInt8 ? 8 : 1][2], vs[kInt8 ? 8 : 1][2];   // f16 scales of the lane's eight cells, a block each
};

// The value index of row r of output product j: what lane r loaded at its place j.
template <int D, bool kInt8>
__device__ __forceinline__ uint32_t value_of(uint32_t j, uint32_t r) {
    if constexpr (kInt8) return j / 4 * 64 + r * 4 + j % 4;
    constexpr uint32_t each = D >= 128 ? 8 : 4;
    return j / each * 128 + r * each + j % each;
}

template <int D>
__device__ __forceinline__ void ld_scales(uint32_t (&s)[2], const uint16_t* scales, uint64_t row) {
    if constexpr (D == 256) {
        const ops_u32x2 w = ld_global<ops_u32x2>(scales + row * 4);
        s[0] = w.x, s[1] = w.y;
    } else if constexpr (D == 128) {
        s[0] = ld_global<uint32_t>(scales + row * 2);
    } else {
        s[0] = ld_global<uint16_t>(scales + row);
    }
}
__device__ __forceinline__ float scale_of(const uint32_t (&s)[2], int block) {
    const f16x2 t = two(s[block / 2]);
    return float(block & 1 ? t.y : t.x);
}

// The page table's entry for cell base + l % 32 of a sequence in lane l; a cell past the table reads the last entry.  The
// load is only waited for where the entry becomes a row.
__device__ __forceinline__ int32_t entry_of(const AttnArgs& a, uint32_t s, uint32_t base, uint32_t lane) {
    const uint32_t cell = base + (lane & 31), page = ops_div(cell < a.c.cells ? cell : a.c.cells - 1, a.c.ps);
    const int64_t at = int64_t(s) * a.c.table_ld + page;
    return a.c.table ? ld_global<int32_t>(a.c.table + at) : int32_t(at);
}
// The pool row of that cell, or -1 where it is outside the span or not resident.
__device__ __forceinline__ int32_t row_of(const AttnArgs& a, const Span& p, int32_t entry, uint32_t h, uint32_t base, uint32_t lane) {
    const uint32_t cell = base + (lane & 31), page = ops_div(cell, a.c.ps);
    const bool in = cell >= p.first && cell < p.len && uint32_t(entry) < a.c.n_pages;
    return in ? int32_t((uint32_t(entry) * a.c.H + h) * a.c.ps.d + (cell - page * a.c.ps.d)) : -1;
}

template <int D, bool kInt8>
__device__ __forceinline__ void load_keys(Rows<D, kInt8>& r, const AttnArgs& a, int32_t row, uint32_t lane) {
    using R = Rows<D, kInt8>;
    constexpr uint64_t bytes = kInt8 ? D : D * 2;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint32_t at = uint32_t(__shfl(row, int(t * 16 + (lane & 15))));
        const uint8_t* p = a.c.k + at * bytes + (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < R::kKeySteps; ++i) r.k[t][i] = kInt8 ? ld_once<ops_u32x4>(p + i * 64) : ld_global<ops_u32x4>(p + i * 64);
    }
}

template <int D, bool kInt8>
__device__ __forceinline__ void load_values(Rows<D, kInt8>& r, const AttnArgs& a, int32_t row, uint32_t lane) {
    using R = Rows<D, kInt8>;
    constexpr uint64_t bytes = kInt8 ? D : D * 2;
    const uint32_t g4 = (lane >> 4) * 4;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const uint32_t at = uint32_t(__shfl(row, int((n & 3) + g4 + (n >> 2) * 16)));
        const uint8_t* p = a.c.v + at * bytes + (lane & 15) * (R::kValWords * 4);
#pragma unroll
        for (int i = 0; i < R::kValPieces; ++i) {
            if constexpr (R::kValWords == 4) {
                const ops_u32x4 w = ld_once<ops_u32x4>(p + i * 256);
                r.v[n][i][0] = w.x, r.v[n][i][1] = w.y, r.v[n][i][2] = w.z, r.v[n][i][3] = w.w;
            } else if constexpr (R::kValWords == 2) {
                const ops_u32x2 w = ld_global<ops_u32x2>(p);
                r.v[n][i][0] = w.x, r.v[n][i][1] = w.y;
            } else {
                r.v[n][i][0] = ld_global<uint32_t>(p + i * 64);
            }
        }
        if constexpr (kInt8) {
            ld_scales<D>(r.ks[n], a.c.k_scale, at);
            ld_scales<D>(r.vs[n], a.c.v_scale, at);
        }
    }
}

// A query part's operand for value step i (lane = head % 16 + 16 * group).
template <int D, int kParts>
struct Queries {
    ops_u32x4 q[kParts][D / 32][64];
};

// ---- the kernel -----------------------------------------------------------------------------------------------------------

template <int D, bool kInt8, bool kF16>
__global__ void __launch_bounds__(kAttnThreads, 2) attn_part_kernel(AttnArgs a) {
    using R = Rows<D, kInt8>;
    constexpr int kParts = kF16 ? 1 : 2;        // f16 queries are exact
    constexpr int kOut = D / 16, kBlocks = D / 64;
    constexpr int kRowF = D + 4;                // floats of a head's row in LDS
    // the queries' place is taken by the waves' outputs at the end
    __shared__ union {
        Queries<D, kParts> q;
        float o[kAttnWaves][16 * kRowF];
    } s;
    __shared__ float s_c[16], s_m[kAttnWaves][16], s_l[kAttnWaves][16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;

    // In the direct form a workgroup takes one unit, and which one does not depend on the lengths: the first loads need
    // not wait for them
    Place p;
    uint32_t within;
    int64_t n = 0;
    if (a.direct) {
        const uint32_t wgs = a.direct * a.tiles;
        p.s = blockIdx.x / wgs;
        within = blockIdx.x - p.s * wgs;
        n = ld_global<int64_t>(a.lens + p.s);
        p.ws0 = p.s * wgs;
    } else {
        if (!place_of(a, lane, blockIdx.x, p)) return;
        within = blockIdx.x - p.wg0;
    }
    const uint32_t part = within / a.tiles, ht = within - part * a.tiles;
    const uint32_t per_head = a.tiles / a.c.H, h = ht / per_head, G = a.n_head / a.c.H;
    const uint32_t head0 = h * G + (ht - h * per_head) * 16;
    const uint32_t heads = (h + 1) * G - head0 < 16 ? (h + 1) * G - head0 : 16;
    uint32_t u0 = part, u1 = part + 1;
    if (!a.direct) {
        const uint32_t each = (p.span.units + p.parts - 1) / p.parts;
        u0 = part * each;
        u1 = u0 + each < p.span.units ? u0 + each : p.span.units;
    }
    uint32_t base0 = (a.direct ? 0u : p.span.begin) + wave * kTurn;
    // loads return in the order they are asked for: the first turn's table entries, the queries, then that turn's rows
    int32_t entry = entry_of(a, p.s, base0 + u0 * kUnit, lane);
    float xq[4][D / 64];   // heads wave, wave + 4, ...: values lane, lane + 64, ...
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            const uint32_t at = (head0 + (i * 4 + wave < heads ? i * 4 + wave : 0)) * D + k * 64 + lane;
            const uint8_t* q = a.q + int64_t(p.s) * a.q_ld;
            if constexpr (kF16) xq[i][k] = float(__builtin_bit_cast(_Float16, ld_global<uint16_t>(q + at * 2)));
            else xq[i][k] = ld_global<float>(q + at * 4);
        }
    if (a.direct) {
        p.span = span_of(a, n);
        p.parts = p.span.units ? p.span.units : 1;
        if (part >= p.parts) return;
        u1 = u1 < p.span.units ? u1 : p.span.units;
    }
    const Span& span = p.span;
    // where the joining kernel finds the sequence's parts
    if (a.join && within == 0 && threadIdx.x == 0) a.where[p.s] = ops_u32x2{p.parts, p.ws0};

    // the first turn's rows are on their way while the queries are laid out
    R r;
    int32_t row = row_of(a, span, entry, h, base0 + u0 * kUnit, lane);
    uint32_t there = uint32_t(__ballot(row >= 0));
    row = row < 0 ? 0 : row;
    if (u0 < u1) {
        entry = entry_of(a, p.s, base0 + (u0 + 1) * kUnit, lane);
        load_keys<D, kInt8>(r, a, row, lane);
        load_values<D, kInt8>(r, a, row, lane);
    }
#pragma unroll
    for (uint32_t i4 = 0; i4 < 4; ++i4) {
        // an f32 head is scaled by a power of two to a largest value of 2^14 .. 2^15, so that the two parts of values down to
        // 2^-16 of that keep all bits: a key can be as much larger there
        const uint32_t i = i4 * 4 + wave;
        float x[D / 64], top = 0;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            x[k] = i < heads ? xq[i4][k] : 0.0f;
            top = fmaxf(top, fabsf(x[k]));
        }
        float by = 1.0f, back = 1.0f;
        if constexpr (!kF16) {
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
            if (top > 0) {
                // within what a power of two and its inverse can be; infinite for an infinite value, which stays one
                const int e = int(__float_as_uint(top) >> 23) - 127, f = e > 127 ? 127 : e < -112 ? -112 : e;
                by = __uint_as_float(uint32_t(127 + 14 - f) << 23);
                back = __uint_as_float(uint32_t(127 - 14 + f) << 23);
            }
        }
        if (lane == 0) s_c[i] = a.scale * kLog2e * back;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            const uint32_t d = k * 64 + lane;
            // f16 rows: step d / 32, group (d % 32) / 8.  int8 rows: half u of 64-value step, group (d % 64) / 16
            const uint32_t step = kInt8 ? d / 64 * 2 + (d % 16) / 8 : d / 32, grp = kInt8 ? (d % 64) / 16 : (d % 32) / 8;
            const _Float16 hi = _Float16(x[k] * by);
            reinterpret_cast<_Float16*>(&s.q.q[0][step][grp * 16 + i])[d % 8] = hi;
            if constexpr (!kF16)
                reinterpret_cast<_Float16*>(&s.q.q[kParts - 1][step][grp * 16 + i])[d % 8] = _Float16(x[k] * by - float(hi));
        }
    }
    __syncthreads();
    const float c = s_c[col];

    f32x4 o[kOut];
    float m, l;
    // the rows of turn u, by way of the table's entries
    auto load_row = [&](uint32_t u) {
        row = row_of(a, span, entry_of(a, p.s, base0 + u * kUnit, lane), h, base0 + u * kUnit, lane);
        there = uint32_t(__ballot(row >= 0));
        row = row < 0 ? 0 : row;
        entry = entry_of(a, p.s, base0 + (u + 1) * kUnit, lane);
    };
    // The part's turns: weights in two parts, or as they are.
    auto turns = [&](auto form) {
        constexpr bool kAsIs = decltype(form)::value;
#pragma unroll
        for (int j = 0; j < kOut; ++j) o[j] = f32x4{};
        m = -kInf, l = 0;
        // the largest weight of all; of a turn that is gone at again, the m of the cells that waited
        float high = -kInf, waited = 0;
        bool again = false;
        // a turn's table entries are asked for before the rows of the turn before it: asked for after them, they would only
        // come when all of those have
        for (uint32_t u = u0; u < u1;) {
            // scores: x[t * 4 + i] of cell 16 t + 4 g + i.  The queries are read from LDS every turn, two steps at a time (the
            // barriers to the compiler): kept in registers they would take the place of rows in flight
            float x[8];
            f32x4 hi[2]{}, lo[2]{};   // the low part's products apart only where infinities are looked for
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                asm volatile("" ::: "memory");
                f16x8 q[kParts][2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < kParts; ++i) q[i][k] = __builtin_bit_cast(f16x8, s.q.q[i][2 * b + k][lane]);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if constexpr (kInt8) {
                        f32x4 bh{}, bl{};
                        uint32_t w[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) codes4(r.k[t][b][k] ^ 0x80808080u, w[2 * k], w[2 * k + 1]);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const f16x8 key = eight(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                            bh = mfma(key, q[0][k], bh);
                            if constexpr (!kF16) (kAsIs ? bl : bh) = mfma(key, q[kParts - 1][k], kAsIs ? bl : bh);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float ks = scale_of(r.ks[t * 4 + i], b);
                            hi[t][i] += ks * bh[i];
                            if constexpr (!kF16 && kAsIs) lo[t][i] += ks * bl[i];
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const f16x8 key = __builtin_bit_cast(f16x8, r.k[t][2 * b + k]);
                            hi[t] = mfma(key, q[0][k], hi[t]);
                            if constexpr (!kF16) (kAsIs ? lo[t] : hi[t]) = mfma(key, q[kParts - 1][k], kAsIs ? lo[t] : hi[t]);
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                // an infinite key makes the low part's product NaN: the high part has the score
                const float high = hi[n / 4][n % 4], sum = kF16 || !kAsIs || !(fabsf(high) < kInf) ? high : high + lo[n / 4][n % 4];
                x[n] = sum * c;
            }
            // the next turn's keys take the place of this one's
            const uint32_t seen = there;
            const bool more = u + 1 < u1;
            if (more) {
                row = row_of(a, span, entry, h, base0 + (u + 1) * kUnit, lane);
                there = uint32_t(__ballot(row >= 0));
                row = row < 0 ? 0 : row;
                entry = entry_of(a, p.s, base0 + (u + 2) * kUnit, lane);
                load_keys<D, kInt8>(r, a, row, lane);
            }
            uint32_t gone[8];   // all ones where a cell is not there
            const bool whole = seen == 0xFFFFFFFFu;
            if (!whole) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    gone[n] = (seen >> ((n & 3) + g * 4 + (n >> 2) * 16)) & 1u ? 0u : ~0u;
                    if (gone[n]) x[n] = -kInf;
#pragma unroll
                    for (int i = 0; i < R::kValPieces; ++i)
#pragma unroll
                        for (int k = 0; k < R::kValWords; ++k) r.v[n][i][k] = gone[n] ? 0u : r.v[n][i][k];
                    if constexpr (kInt8) r.vs[n][0] = gone[n] ? 0u : r.vs[n][0], r.vs[n][1] = gone[n] ? 0u : r.vs[n][1];
                }
            }
            // Where the turn's weights lie: the largest of the column, the least of the lane's own cells.  An int8 weight is
            // multiplied with its blocks' scales before it becomes f16: their exponents count, bounds over the lane's cells, or
            // cell by cell where cells wait.
            float top = -kInf, low = kInf;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                top = fmaxf(top, x[n]);
                low = fminf(low, x[n] == -kInf ? kInf : x[n]);
            }
            if constexpr (kInt8) {
                u16x2 hi{}, lo{0xFFFF, 0xFFFF};   // one less for the least, so that scales that are 0 do not count
#pragma unroll
                for (int n = 0; n < 8; ++n) scales_of<kBlocks>(r.vs[n], hi, lo);
                top += exponent_most(hi);
                low += exponent_least(lo);
            }
            auto waits = [&](int n, float m, float& y) {
                float z = y = x[n];
                if constexpr (kInt8) {
                    u16x2 hi{}, lo{0xFFFF, 0xFFFF};
                    scales_of<kBlocks>(r.vs[n], hi, lo);
                    y += exponent_most(hi);
                    z += exponent_least(lo);
                }
                return z < m + kLeast && y < m + kWait;
            };
            if (rarely(again)) {
                top = -kInf, low = kInf;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    float y;
                    x[n] = waits(n, waited, y) ? x[n] : -kInf;
                    top = fmaxf(top, x[n] == -kInf ? -kInf : y);
                    low = x[n] == -kInf ? low : -kInf;   // it will be looked for
                }
            }
            top = over_rows(top, max_of);
            if (const bool out = top > m + kMost || low < m + kLeast; rarely(__any(out))) {
                const float f = floorf(top), least = over_rows(low, min_of);
                high = fmaxf(high, f);
                const bool moves = over_rows(out ? 1.0f : 0.0f, max_of) > 0 && top > -kInf;
                const float to = moves ? fmaxf(f - (least < f - kTop + kLeast ? kDeep : kTop), high - kFar) : m;
                const float w = m == -kInf ? 0.0f : fmaxf(__builtin_amdgcn_ldexpf(1.0f, min(int(m - to), 100)), kTiny);
                m = to;
                l *= w;
#pragma unroll
                for (int j = 0; j < kOut; ++j) o[j] *= w;
            }
            // by way of a reference near the largest: a difference from m itself would round the exponents of weights near 1
            const float ref = m == -kInf ? 0.0f : m + kNear;
            float pr[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) pr[n] = exp2_fast(x[n] - ref) * kNearBy;
            again = false;
            if (!kAsIs && rarely(__any(low < m + kLeast))) {
                bool left = false;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    float y;
                    const bool w = m > high - kFar && x[n] > -kInf && waits(n, m, y);
                    pr[n] = w ? 0.0f : pr[n];
                    left |= w;
                }
                waited = over_rows(left ? 1.0f : 0.0f, max_of) > 0 ? m : -kInf;
                again = __any(left);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) l += pr[n];
            if constexpr (kInt8) {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    float pb[8];
#pragma unroll
                    for (int n = 0; n < 8; ++n) pb[n] = pr[n] * scale_of(r.vs[n], b);
                    f16x8 hi{}, lo{};
                    if constexpr (!kAsIs) split8(pb, hi, lo);
                    uint32_t w[8];
#pragma unroll
                    for (int n = 0; n < 8; ++n) w[n] = r.v[n][b][0] ^ 0x80808080u;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t e0[4], e1[4];   // the pair of places 2 k, 2 k + 1 of cells 2 i, 2 i + 1
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            codes4(__builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], k ? 0x07030602u : 0x05010400u), e0[i], e1[i]);
                        add_values<kAsIs>(o[b * 4 + 2 * k], eight(e0[0], e0[1], e0[2], e0[3]), pb, hi, lo);
                        add_values<kAsIs>(o[b * 4 + 2 * k + 1], eight(e1[0], e1[1], e1[2], e1[3]), pb, hi, lo);
                    }
                }
            } else {
                f16x8 hi{}, lo{};
                if constexpr (!kAsIs) split8(pr, hi, lo);
#pragma unroll
                for (int i = 0; i < R::kValPieces; ++i)
#pragma unroll
                    for (int k = 0; k < R::kValWords; ++k) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t sel = e ? 0x07060302u : 0x05040100u;
                            uint32_t w[4];
#pragma unroll
                            for (int n = 0; n < 4; ++n) w[n] = __builtin_amdgcn_perm(r.v[2 * n + 1][i][k], r.v[2 * n][i][k], sel);
                            add_values<kAsIs>(o[(i * R::kValWords + k) * 2 + e], eight(w[0], w[1], w[2], w[3]), pr, hi, lo);
                        }
                    }
            }
            if (rarely(again)) load_row(u), load_keys<D, kInt8>(r, a, row, lane);
            else ++u;
            if (again || more) load_values<D, kInt8>(r, a, row, lane);
        }
    };
    turns(std::false_type{});
    // an infinite value may have met a part that is 0 (a value that is no number shows either way)
    bool odd = false;
#pragma unroll
    for (int j = 0; j < kOut; ++j) odd |= !(fabsf((o[j].x + o[j].y) + (o[j].z + o[j].w)) < kInf);
    if (rarely(__any(odd))) {
        load_row(u0);
        load_keys<D, kInt8>(r, a, row, lane);
        load_values<D, kInt8>(r, a, row, lane);
        turns(std::true_type{});
    }

    // the waves' results to one m, summed through LDS
    l = over_rows(l, [](float p, float q) { return p + q; });
    if (g == 0) s_m[wave][col] = m, s_l[wave][col] = l;
    __syncthreads();
    float M = s_m[0][col];
#pragma unroll
    for (int w = 1; w < kAttnWaves; ++w) M = fmaxf(M, s_m[w][col]);
    const float w = weight(m, M);
#pragma unroll
    for (int j = 0; j < kOut; j += 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 four{o[j][i] * w, o[j + 1][i] * w, o[j + 2][i] * w, o[j + 3][i] * w};
            *reinterpret_cast<f32x4*>(&s.o[wave][col * kRowF + value_of<D, kInt8>(j, g * 4 + i)]) = four;
        }
    __syncthreads();
    constexpr uint32_t kQuads = D / 4;
    for (uint32_t at = threadIdx.x; at < heads * kQuads; at += kAttnThreads) {
        const uint32_t i = at / kQuads, d = at % kQuads * 4;
        float top = s_m[0][i], sum = 0;
#pragma unroll
        for (int k = 1; k < kAttnWaves; ++k) top = fmaxf(top, s_m[k][i]);
        f32x4 acc{};
#pragma unroll
        for (int k = 0; k < kAttnWaves; ++k) {
            acc += *reinterpret_cast<const f32x4*>(&s.o[k][i * kRowF + d]);
            sum += s_l[k][i] * weight(s_m[k][i], top);
        }
        if (p.parts == 1) {
            st_act4<kF16>(a.out + int64_t(p.s) * a.out_ld, (head0 + i) * D + d, sum == 0 ? f32x4{} : acc / sum);
            if (d == 0 && a.lse) a.lse[uint64_t(p.s) * a.n_head + head0 + i] = log_of_sum(top, sum);
        } else {
            float* part = a.ws + uint64_t(p.ws0 + within) * (16 * kRowF) + i * kRowF;
            if (d == 0) *reinterpret_cast<f32x4*>(part) = f32x4{top, sum, 0, 0};
            *reinterpret_cast<f32x4*>(part + 4 + d) = acc;
        }
    }
}

// Joins the parts of kCols values of one query head: sets of lanes share the parts, then add up through LDS.
template <int D, int kCols, bool kF16>
__global__ void __launch_bounds__(kAttnThreads) attn_join_kernel(AttnArgs a) {
    constexpr uint32_t kRowF = D + 4, kLanes = kCols / 4, kSets = kAttnThreads / kLanes;
    __shared__ f32x4 s_acc[kSets][kLanes];
    __shared__ float s_w[kAttnSlots + 1], s_m[kAttnWaves], s_l[kAttnWaves];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t s = blockIdx.x / a.n_head, head = blockIdx.x - s * a.n_head;
    const ops_u32x2 where = a.where[s];
    const uint32_t parts = where.x;
    if (parts <= 1) return;
    const uint32_t G = a.n_head / a.c.H, h = head / G, tile = (head - h * G) / 16;
    const uint32_t ht = h * (a.tiles / a.c.H) + tile, i = head - h * G - tile * 16;
    const uint64_t step = uint64_t(a.tiles) * (16 * kRowF);   // from part to part
    const float* first = a.ws + (uint64_t(where.y) + ht) * (16 * kRowF) + i * kRowF;
    constexpr uint32_t kMine = (kAttnSlots + 1 + kAttnThreads - 1) / kAttnThreads;   // parts whose statistics a thread reads
    constexpr uint32_t kAhead = 8;                                                   // its parts that are read meanwhile
    const uint32_t set = threadIdx.x / kLanes, d = blockIdx.y * kCols + threadIdx.x % kLanes * 4;
    float pm[kMine], pl[kMine], m = -kInf, l = 0;
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        const uint32_t at = threadIdx.x + k * kAttnThreads;
        const ops_u32x2 ml = ld_global<ops_u32x2>(first + (at < parts ? at : 0) * step);
        pm[k] = at < parts ? __uint_as_float(ml.x) : -kInf;
        pl[k] = at < parts ? __uint_as_float(ml.y) : 0.0f;
    }
    f32x4 ahead[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) ahead[k] = ld_global<f32x4>(first + (set + k * kSets < parts ? set + k * kSets : 0) * step + 4 + d);
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) m = fmaxf(m, pm[k]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    if (lane == 0) s_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        const uint32_t at = threadIdx.x + k * kAttnThreads;
        const float w = weight(pm[k], m);
        l += pl[k] * w;
        if (at < parts) s_w[at] = w;
    }
    l = wave_sum(l);
    if (lane == 0) s_l[wave] = l;
    __syncthreads();
    f32x4 acc{};
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k)
        if (set + k * kSets < parts) acc += ahead[k] * s_w[set + k * kSets];
#pragma unroll 8
    for (uint32_t k = set + kAhead * kSets; k < parts; k += kSets) acc += ld_global<f32x4>(first + k * step + 4 + d) * s_w[k];
    s_acc[set][threadIdx.x % kLanes] = acc;
    __syncthreads();
    if (set) return;
#pragma unroll
    for (uint32_t k = 1; k < kSets; ++k) acc += s_acc[k][threadIdx.x];
    l = s_l[0] + s_l[1] + s_l[2] + s_l[3];
    st_act4<kF16>(a.out + int64_t(s) * a.out_ld, head * D + d, l == 0 ? f32x4{} : acc / l);
    if (d == 0 && a.lse) a.lse[uint64_t(s) * a.n_head + head] = log_of_sum(m, l);
}

template <int D, bool kInt8, bool kF16>
hipError_t launch_of(const AttnArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((attn_part_kernel<D, kInt8, kF16>), dim3(a.grid), dim3(kAttnThreads), 0, stream, a);
    // A head's parts by one workgroup where the heads fill the chip or its threads have all the parts in flight at once, else by
    // one for 64 values each: with 24 heads 12.5 us against 12.8 for 1 K cells (both kernels), but 53.3 against 51.8 for
    // 128 K; with 768 heads 38.8 against 42.0
    const uint32_t rows = a.n_seqs * a.n_head;
    if (a.join && (rows >= 128 || a.parts <= 32)) hipLaunchKernelGGL((attn_join_kernel<D, D, kF16>), dim3(rows), dim3(kAttnThreads), 0, stream, a);
    else if (a.join) hipLaunchKernelGGL((attn_join_kernel<D, 64, kF16>), dim3(rows, D / 64), dim3(kAttnThreads), 0, stream, a);
    return hipGetLastError();
}
template <int D>
hipError_t launch_of(const AttnArgs& a, int format, bool f16, hipStream_t stream) {
    if (format == 1) return f16 ? launch_of<D, true, true>(a, stream) : launch_of<D, true, false>(a, stream);
    return f16 ? launch_of<D, false, true>(a, stream) : launch_of<D, false, false>(a, stream);
}

}  // namespace

uint64_t plan_attn(AttnArgs& a, int head_dim) {
    a.tiles = a.c.H * ((a.n_head / a.c.H + 15) / 16);
    a.slots = kAttnSlots;
    a.least = 1;
    const SplitPlan p = plan_split(a.n_seqs, a.tiles, a.max_len, a.window, a.slots);
    a.join = p.join;
    a.direct = p.direct;
    a.parts = p.parts;
    a.grid = uint32_t(p.grid);
    return a.join ? p.places * 16 * uint64_t(head_dim + 4) * 4 + (uint64_t(a.n_seqs) * 8 + 15) / 16 * 16 : 16;
}

void place_attn(AttnArgs& a, void* workspace, uint64_t bytes) {
    a.ws = static_cast<float*>(workspace);
    if (a.join) a.where = reinterpret_cast<ops_u32x2*>(static_cast<uint8_t*>(workspace) + bytes - (uint64_t(a.n_seqs) * 8 + 15) / 16 * 16);
}

hipError_t launch_attn(const AttnArgs& a, int head_dim, int format, bool f16, hipStream_t stream) {
    if (head_dim == 64) return launch_of<64>(a, format, f16, stream);
    if (head_dim == 128) return launch_of<128>(a, format, f16, stream);
    if (head_dim == 256) return launch_of<256>(a, format, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
