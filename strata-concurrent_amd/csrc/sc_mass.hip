// sc_mass.hip - the attention weights that a sequence's latest queries give its cells, added to what each cell has had before
// (sc_attn_mass_async).
//
// With scores x = scale * q . k * log2(e), a cell's weight from a query is 2^(x - m) / l for the query's reference m and the sum
// l of 2^(x - m) over its cells.  Where the attention has left the log of that sum, one pass over the keys gives the weights;
// else one pass before it gives the sums, parts of the cells by workgroups, and a small kernel joins the parts: the product is
// formed twice, which is less than writing the scores down and reading them again (rows * heads of 4 bytes a cell against a row
// of keys).
//
// Keys are the left operands of matrix products, row = cell, and stay in a wave's registers; the kv head's queries of all rows are the
// columns of the right ones, 16 at a time, which the workgroup lays out in LDS.  A lane ends with the scores of one column for
// some cells, and adds their weights up over the columns by itself; the 16 lanes of a row of lanes are summed once at the end,
// always in the same order.
//   Up to 16 columns (a new token a sequence): the queries are laid out once, a wave takes 32 cells a turn and has its next turn's
//   keys on the way while it forms weights.  Reading the keys bounds it, and for short calls the chain of latencies to the first
//   weights.  2 kv heads of 256 and 24 query heads: 1021 cells 5.8 us; 24 sequences up to 8190 cells in int8, 57 MB, 17.7 us (24
//   where a lane loads the scales of its eight cells itself and keys go past the caches); 128 K cells in f16, 135 MB, 34 us.
//   More columns: a workgroup's waves share 128 cells' keys and go over the tiles of columns, the next tiles' queries on their way to
//   LDS meanwhile, and what the sets of waves have summed up is added at the end.  Half of a call is the products and the weights,
//   half the way to the first of them.  32 queries of two prompts up to 16 381 cells without their sums, 11.5 GFLOP a pass: 57 us (26 a
//   pass, the join 5).  Tried: 64 cells a wave, which needs all registers of a SIMD for two waves (80 us), one tile of columns at
//   a time for three waves a SIMD (65), the weights of cells that are all seen in a branch of their own (65).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_attn_split.hpp"
#include "sc_attn_tiles.hpp"
#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr uint32_t kMassThreads = kAttnWaves * 64;
constexpr uint32_t kMostColumns = 1024;         // rows times query heads of a kv head
// Workgroups that the cells are shared out among where columns are few.  One long f16 sequence likes fewer (128 K cells: 30.5 us with
// 256, 33.4 with 512, 34.3 with 1024; int8 18.9, 16.0, 16.0), a batch more (24 int8 sequences up to 8190 cells 28, 22.7 and 17.7, f16
// 47, 40 and 28; eight f16 ones up to 16 000 cells 20.5, 18.7 and 13.3, with f32 queries 21.8, 14.9 and 15.7).
constexpr uint32_t kFewSlots = 1024;
constexpr float kLog2eRest = 1.92596299e-8f;    // log2(e) - kLog2e

// x and the same of the 16 lanes of its row of lanes, in every one of them (row_ror by 8, 4, 2, 1).
template <class F>
__device__ __forceinline__ float over_lanes(float x, F f) {
    x = f(x, __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), 0x128, 0xF, 0xF, false))));
    x = f(x, __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), 0x124, 0xF, 0xF, false))));
    x = f(x, __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), 0x122, 0xF, 0xF, false))));
    return f(x, __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), 0x121, 0xF, 0xF, false))));
}
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }

__device__ __forceinline__ uint32_t length_of(const MassArgs& a, uint32_t s) {
    const int64_t n = ld_global<int64_t>(a.lens + s);
    return n < 0 ? 0u : n > int64_t(a.max_len) ? a.max_len : uint32_t(n);
}

// The row and the query head of a column of kv head h, as an index [sequence's rows][n_head].
__device__ __forceinline__ uint64_t query_of(const MassArgs& a, uint32_t s, uint32_t h, uint32_t col) {
    const uint32_t r = ops_div(col, a.G);
    return (uint64_t(s) * a.rows + r) * a.n_head + h * a.G.d + (col - r * a.G.d);
}
__device__ __forceinline__ const uint8_t* values_of(const MassArgs& a, uint32_t s, uint32_t h, uint32_t col, uint32_t bytes) {
    const uint32_t r = ops_div(col, a.G);
    return a.q + (int64_t(s) * a.rows + r) * a.q_ld + uint64_t(h * a.G.d + (col - r * a.G.d)) * bytes;
}
// What a weight is formed with: 2^(x - m) * by, from the log of the sum or from what the parts' sums gave.  Nothing past the
// columns.
__device__ __forceinline__ f32x2 norm_of(const MassArgs& a, uint32_t s, uint32_t h, uint32_t col) {
    f32x2 v{kInf, 0};
    if (col >= a.cols) return v;
    if (!a.lse) return ld_global<f32x2>(a.norm + (uint64_t(s) * a.c.H + h) * a.cols + col);
    // in base 2, a whole number of it apart: differences from that keep their bits
    const float lse = ld_global<float>(a.lse + query_of(a, s, h, col));
    const float t = lse * kLog2e, rest = fmaf(lse, kLog2e, -t) + lse * kLog2eRest;
    if (fabsf(lse) == kInf) return f32x2{kInf, lse > 0 ? 1.0f : 0.0f};
    return f32x2{rintf(t), exp2_fast((rintf(t) - t) - rest)};
}
// Right operands' places in LDS: value d of a column, 8 at a time, is in step d / 32, group (d % 32) / 8 where keys are f16; where
// they are int8, of which a lane has 16 of a step of 64, in step d / 64 * 2 + (d % 16) / 8, group (d % 64) / 16.
template <bool kInt8>
__device__ __forceinline__ uint32_t place_of(uint32_t d) {
    return kInt8 ? (d / 64 * 2 + d % 16 / 8) * 64 + d % 64 / 16 * 16 : d / 32 * 64 + d % 32 / 8 * 16;
}
// And back: the values that operand `at` of a column holds.
template <bool kInt8>
__device__ __forceinline__ uint32_t value_at(uint32_t at) {
    const uint32_t step = at / 64, group = at % 64 / 16;
    return kInt8 ? step / 2 * 64 + group * 16 + step % 2 * 8 : step * 32 + group * 8;
}
// Eight values as two f16 parts.
__device__ __forceinline__ void parts_of(const float (&x)[8], ops_u32x4& hi, ops_u32x4& lo) {
    f16x8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = _Float16(x[i]);
        l[i] = _Float16(x[i] - float(h[i]));
    }
    hi = __builtin_bit_cast(ops_u32x4, h), lo = __builtin_bit_cast(ops_u32x4, l);
}
// An f32 query is scaled by a power of two to a largest value of 2^14 .. 2^15, so that the two parts of values down to 2^-16 of
// that keep 22 bits or more: a key can be as much larger there.  They do not keep all 24: the first part leaves up to 12 bits, and
// the second has 11, so one value in four is a unit in its last place off.  A third part would be half as many products again, for an
// error that is small beside the others: of 1021 weights by queries of 256 values 1.4e-8 is the parts', 4.6e-8 the rounding of
// x - m, 3.2e-8 the products' sums.
__device__ __forceinline__ void scaling(float top, float& by, float& back) {
    by = back = 1.0f;
    if (top > 0) {
        const int e = int(__float_as_uint(top) >> 23) - 127, f = e > 127 ? 127 : e < -112 ? -112 : e;
        by = __uint_as_float(uint32_t(127 + 14 - f) << 23);
        back = __uint_as_float(uint32_t(127 - 14 + f) << 23);
    }
}

// Keys of 32 cells as left operands: of row lane % 16, 8 values a step of 32 by lane / 16 (f16), or 16 of 64 (int8).
template <int D, bool kInt8>
struct KeyRows {
    static constexpr int kLoads = kInt8 ? D / 64 : D / 32;
    static constexpr uint32_t kScaleWords = D == 256 ? 2 : 1;   // f16 scales of a cell, a block of 64 each
    ops_u32x4 w[2][kLoads];
    uint32_t own[2];                    // scales of cell lane % 32
    uint32_t scale[kInt8 ? 8 : 1][2];   // and of the cells of the lane's results

    // `row`: the cells' pool rows, in lanes 0 .. 31 and again in the others
    __device__ __forceinline__ void load(const CacheArgs& c, uint32_t row, uint32_t lane) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t at = uint32_t(__shfl(int(row), int(t * 16 + (lane & 15))));
            const uint8_t* p = c.k + uint64_t(at) * (kInt8 ? D : D * 2) + (lane >> 4) * 16;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) w[t][i] = ld_global<ops_u32x4>(p + i * 64);
        }
        if constexpr (kInt8) ld_scales<D>(own, c.k_scale, row);
    }
    // The scales to the lanes whose results they multiply, by way of the wave's own part of LDS: one load a cell, not one a lane.
    __device__ __forceinline__ void spread(uint32_t* s, uint32_t lane) {
        if constexpr (kInt8) {
#pragma unroll
            for (uint32_t i = 0; i < kScaleWords; ++i) s[(lane & 31) * kScaleWords + i] = own[i];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
#pragma unroll
                for (uint32_t k = 0; k < kScaleWords; ++k) scale[i][k] = s[(i / 4 * 16 + (lane >> 4) * 4 + i % 4) * kScaleWords + k];
            __builtin_amdgcn_wave_barrier();
        }
    }
};
// The operand of step i.
template <int D>
__device__ __forceinline__ f16x8 operand(const KeyRows<D, false>& k, int t, int i) { return __builtin_bit_cast(f16x8, k.w[t][i]); }
template <int D>
__device__ __forceinline__ f16x8 operand(const KeyRows<D, true>& k, int t, int i) {
    uint32_t x[4];
    codes4(k.w[t][i / 2][i % 2 * 2] ^ 0x80808080u, x[0], x[1]);
    codes4(k.w[t][i / 2][i % 2 * 2 + 1] ^ 0x80808080u, x[2], x[3]);
    return eight(x[0], x[1], x[2], x[3]);
}

// Products with 16 columns: x[t * 4 + i] of the lane's column and cell 16 t + 4 (lane / 16) + i.  An infinite key makes the second
// part's product NaN: the first part has the score.
template <int D, bool kInt8, int kParts>
__device__ __forceinline__ void products_of(float (&x)[8], const KeyRows<D, kInt8>& key, const ops_u32x4* q, uint32_t part, uint32_t lane) {
    f32x4 hi[2]{}, lo[2]{};
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
        f16x8 v[kParts][2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < kParts; ++i) v[i][k] = __builtin_bit_cast(f16x8, q[i * part + (2 * b + k) * 64 + lane]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 bh{}, bl{};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f16x8 w = operand(key, t, 2 * b + k);
                if constexpr (kInt8) {
                    bh = mfma(w, v[0][k], bh);
                    if constexpr (kParts > 1) bl = mfma(w, v[kParts - 1][k], bl);
                } else {
                    hi[t] = mfma(w, v[0][k], hi[t]);
                    if constexpr (kParts > 1) lo[t] = mfma(w, v[kParts - 1][k], lo[t]);
                }
            }
            if constexpr (kInt8)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float scale = scale_of(key.scale[t * 4 + i], b);
                    hi[t][i] += scale * bh[i];
                    if constexpr (kParts > 1) lo[t][i] += scale * bl[i];
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float first = hi[i / 4][i % 4];
        x[i] = kParts == 1 || !(fabsf(first) < kInf) ? first : first + lo[i / 4][i % 4];
    }
}

// Which of the lane's cells its column sees, where `there` has a bit for each of 32 cells from `base` on (the first of them cell 0).
__device__ __forceinline__ uint32_t seen_of(const MassArgs& a, uint32_t n, uint32_t col, uint32_t there, uint32_t base, uint32_t lane) {
    const uint32_t r = ops_div(col < a.cols ? col : a.cols - 1, a.G), own = (lane >> 4) * 4;
    const int32_t ends = row_ends(n, a.rows, r, base + own);
    uint32_t sees = 0;
#pragma unroll
    for (int32_t i = 0; i < 8; ++i) {
        const int32_t cell = i / 4 * 16 + i % 4;
        sees |= uint32_t((there >> (uint32_t(cell) + own) & 1) && row_sees(ends, a.window, cell)) << i;
    }
    return sees;
}
// Whether every row sees 32 cells from `base` on, where they are there.
__device__ __forceinline__ bool all_see(const MassArgs& a, uint32_t n, uint32_t base) {
    return int64_t(base) + kTurn <= int64_t(n) - a.rows + 1 && (!a.window || int64_t(base) >= int64_t(n) - a.window);
}
// Cells below this are seen by no row.
__device__ __forceinline__ int64_t first_seen(const MassArgs& a, uint32_t n) {
    return a.window ? int64_t(n) - a.rows + 1 - a.window : 0;
}

// A column's reference and sum go on over more scores, those of -inf adding nothing; the reference is a whole number.
__device__ __forceinline__ f32x2 summed(f32x2 old, const float (&x)[8]) {
    float top = x[0], sum = 0;
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    const float M = fmaxf(old.x, floorf(over_rows(top, max_of))), ref = M == -kInf ? 0.0f : M;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += exp2_fast(x[i] - ref);
    return f32x2{M, old.y * exp2_fast(old.x - ref) + over_rows(sum, sum_of)};
}
__device__ __forceinline__ f32x2 joined(f32x2 p, f32x2 q) {
    const float M = fmaxf(p.x, q.x), ref = M == -kInf ? 0.0f : M;
    return f32x2{M, p.y * exp2_fast(p.x - ref) + q.y * exp2_fast(q.x - ref)};
}
// A weight by its exponent.  Exponents of some classes have none: -inf, a cell that the column does not see, also where the column's
// sum is no number; all of them where the column has no weight (its query saw nothing, or it is past the last one), also where an
// infinite key or the query itself has made NaN.
__device__ __forceinline__ int none_of(float by) { return by == 0 ? 0x3FF : 0x004; }
__device__ __forceinline__ float weight_of(float x, float by, int none) { return __builtin_amdgcn_classf(x, none) ? 0.0f : exp2_fast(x) * by; }
// The exponents of the weights of scores c * x of the cells that the column sees, -inf of the others.
__device__ __forceinline__ void exponents_of(float (&x)[8], float c, float m, bool all, uint32_t sees) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], c, -m);
    if (!all)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sees >> i & 1 ? x[i] : -kInf;
}

// ---- up to 16 columns ---------------------------------------------------------------------------------------------------------

template <int D, bool kInt8, bool kF16, bool kSums>
__global__ void __launch_bounds__(kMassThreads, 2) mass_few_kernel(MassArgs a) {
    constexpr int kParts = kF16 ? 1 : 2, kOps = D / 32 * 64;
    __shared__ ops_u32x4 s_q[kParts][kOps];
    __shared__ float s_back[16];
    __shared__ f32x2 s_ml[kAttnWaves][16];
    __shared__ uint32_t s_scale[kInt8 ? kAttnWaves : 1][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15, h = blockIdx.y, s = blockIdx.z;
    const uint32_t n = length_of(a, s), units = (n + kUnit - 1) / kUnit;
    uint32_t u = blockIdx.x;
    if (u >= units) return;
    const Span span{0, n, 0, 0};
    const int64_t seen = first_seen(a, n);
    if constexpr (kSums)   // what no row sees needs no sum
        while (u < units && int64_t(u + 1) * kUnit <= seen) u += a.parts;

    // the first turn's table entries, the queries, then that turn's rows, in the order that they are needed
    const uint32_t base0 = wave * kTurn;
    int32_t entry = entry_of(a.c, s, base0 + u * kUnit, lane);
    float q[4][D / 64];   // columns wave, wave + 4, ...: values lane, lane + 64, ...
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t c = i * 4 + wave;
        const uint8_t* p = values_of(a, s, h, c < a.cols ? c : 0, D * (kF16 ? 2 : 4));
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
            if constexpr (kF16) q[i][k] = float(__builtin_bit_cast(_Float16, ld_global<uint16_t>(p + (k * 64 + lane) * 2)));
            else q[i][k] = ld_global<float>(p + (k * 64 + lane) * 4);
    }
    f32x2 norm{};
    if constexpr (!kSums) norm = norm_of(a, s, h, col);
    KeyRows<D, kInt8> key;
    int32_t row = row_of(a.c, span, entry, h, base0 + u * kUnit, lane);
    uint32_t there = uint32_t(__ballot(row >= 0));
    if (u < units) {
        entry = entry_of(a.c, s, base0 + (u + a.parts < units ? u + a.parts : u) * kUnit, lane);
        key.load(a.c, row < 0 ? 0u : uint32_t(row), lane);
    }
#pragma unroll
    for (uint32_t i4 = 0; i4 < 4; ++i4) {
        const uint32_t i = i4 * 4 + wave;
        float top = 0, by = 1.0f, back = 1.0f;
        if constexpr (!kF16) {
#pragma unroll
            for (int k = 0; k < D / 64; ++k) top = fmaxf(top, fabsf(q[i4][k]));
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
            scaling(top, by, back);
        }
        if (lane == 0) s_back[i] = back;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            const uint32_t d = k * 64 + lane;
            const float x = i < a.cols ? q[i4][k] * by : 0.0f;
            const _Float16 hi = _Float16(x);
            reinterpret_cast<_Float16*>(&s_q[0][place_of<kInt8>(d) + i])[d % 8] = hi;
            if constexpr (!kF16) reinterpret_cast<_Float16*>(&s_q[kParts - 1][place_of<kInt8>(d) + i])[d % 8] = _Float16(x - float(hi));
        }
    }
    __syncthreads();
    const float c = a.scale * kLog2e * s_back[col];
    f32x2 ml{-kInf, 0};
    for (; u < units; u += a.parts) {
        const uint32_t base = base0 + u * kUnit;
        // the mass that a lane will write, as it was
        const uint32_t cell = base + col / 4 * 16 + g * 4 + col % 4;
        float* mass = nullptr;
        float old = 0;
        if constexpr (!kSums) {
            mass = a.mass + (uint64_t(s) * a.c.H + h) * a.mass_ld + cell;
            if (col < 8 && cell < n && a.decay != 0) old = a.decay * ld_global<float>(mass);
        }
        float x[8];
        key.spread(s_scale[kInt8 ? wave : 0], lane);
        products_of<D, kInt8, kParts>(x, key, s_q[0], kOps, lane);
        const uint32_t now = there;
        if (u + a.parts < units) {   // the next turn's keys take the place of this one's
            const uint32_t next = u + a.parts;
            row = row_of(a.c, span, entry, h, base0 + next * kUnit, lane);
            there = uint32_t(__ballot(row >= 0));
            entry = entry_of(a.c, s, base0 + (next + a.parts < units ? next + a.parts : next) * kUnit, lane);
            key.load(a.c, row < 0 ? 0u : uint32_t(row), lane);
        }
        const uint32_t sees = now == 0xFFFFFFFFu && all_see(a, n, base) ? 0xFFu : seen_of(a, n, col, now, base, lane);
        if constexpr (kSums) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = sees >> i & 1 ? x[i] * c : -kInf;
            ml = summed(ml, x);
        } else {
            float mine = 0;
            exponents_of(x, c, norm.x, false, sees);
            const int none = none_of(norm.y);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float sum = over_lanes(weight_of(x[i], norm.y, none), sum_of);
                mine = int(col) == i ? sum : mine;
            }
            if (col < 8 && cell < n) st_global<float>(mass, old + mine);
        }
    }
    if constexpr (kSums) {
        if (g == 0) s_ml[wave][col] = ml;
        __syncthreads();
        if (wave == 0 && g == 0 && col < a.cols) {
            for (int w = 1; w < kAttnWaves; ++w) ml = joined(ml, s_ml[w][col]);
            st_global<f32x2>(a.sums + ((uint64_t(s) * a.c.H + h) * a.parts + blockIdx.x) * a.cols + col, ml);
        }
    }
}

// ---- more columns -------------------------------------------------------------------------------------------------------------

// f32 queries as two f16 parts [query][2][D], and what their products are scaled back by; a wave a query.
template <int D>
__global__ void __launch_bounds__(256) mass_parts_kernel(MassArgs a) {
    const uint32_t lane = threadIdx.x & 63, h = blockIdx.y, s = blockIdx.z, c = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (c >= a.cols) return;
    const uint8_t* p = values_of(a, s, h, c, D * 4);
    float x[8] = {}, top = 0, by, back;
    if (lane < D / 8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 v = ld_global<f32x4>(p + lane * 32 + i * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i * 4 + j] = v[j], top = fmaxf(top, fabsf(v[j]));
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    scaling(top, by, back);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= by;
    ops_u32x4 hi, lo;
    parts_of(x, hi, lo);
    const uint64_t at = (uint64_t(s) * a.c.H + h) * a.cols + c;
    if (lane < D / 8) {
        st_global<ops_u32x4>(a.split + at * (D / 4) + lane, hi);
        st_global<ops_u32x4>(a.split + at * (D / 4) + D / 8 + lane, lo);
    }
    if (lane == 0) st_global<float>(a.back + at, back);
}

// The sets of four waves of a workgroup: each has all of its 128 cells, 32 a wave, and takes every kSets-th tile of columns.  Two for
// f16 keys of 256 and f16 queries, whose workgroups are few enough to a unit for a wave's products to hide behind another's weights
// (58 us and 62, 32 queries of 16 K cells); else one (16 queries of four sequences up to 8000 cells, 4 kv heads of 128: f16 12.4 us
// and 16, f32 queries 19 and 25, int8 12.6 and 15.5).
template <int D, bool kInt8, bool kF16>
struct Many {
    static constexpr int kParts = kF16 ? 1 : 2;
    static constexpr uint32_t kSets = D == 256 && kF16 && !kInt8 ? 2 : 1, kThreads = kSets * kMassThreads;
};

// A launch has less than 2^32 threads across a sequence's cells: beyond 2^29 cells there are several, from cell a.first_part * kUnit on.
constexpr uint32_t kMostParts = 1u << 22;

template <int D, bool kInt8, bool kF16, bool kSums>
__global__ void __launch_bounds__((Many<D, kInt8, kF16>::kThreads), 2) mass_many_kernel(MassArgs a) {
    using M = Many<D, kInt8, kF16>;
    constexpr int kParts = M::kParts, kOps = D / 32 * 64;
    constexpr uint32_t kEach = (M::kSets * kParts * kOps + M::kThreads - 1) / M::kThreads;   // operands that a thread brings of a tile a set
    __shared__ ops_u32x4 s_q[2][M::kSets][kParts * kOps];
    // sums: the references and sums of a wave's cells; weights: what they are formed with, at the end the sets' sums
    __shared__ f32x2 s_ml[kSums ? kAttnWaves : 1][kMostColumns];
    __shared__ float s_back[kF16 ? 1 : kMostColumns];
    __shared__ uint32_t s_scale[kInt8 ? M::kSets * kAttnWaves : 1][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15, h = blockIdx.y, s = blockIdx.z;
    const uint32_t quarter = wave % kAttnWaves, set = wave / kAttnWaves;
    const uint32_t n = length_of(a, s), unit = a.first_part + blockIdx.x, first = unit * kUnit, base = first + quarter * kTurn;
    if (first >= n) return;
    const uint64_t sh = uint64_t(s) * a.c.H + h;
    const uint32_t tiles = (a.cols + 15) / 16, stages = (tiles + M::kSets - 1) / M::kSets;
    const bool none = int64_t(first) + kUnit <= first_seen(a, n);
    const Span span{0, n, 0, 0};

    const uint8_t* q0 = a.q + int64_t(s) * a.rows * a.q_ld;
    const uint32_t q_ld16 = uint32_t(a.q_ld / 16);
    ops_u32x4 next[kEach];
    auto load = [&](uint32_t stage) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            // operand `at` of a part of a tile; past the columns the last one's, whose results are left out
            const uint32_t e = threadIdx.x + i * M::kThreads, at = e % kOps, part = e / kOps % kParts, tile = stage * M::kSets + e / (kOps * kParts);
            const uint32_t j = tile * 16 + at % 16, c = j < a.cols ? j : a.cols - 1, d = value_at<kInt8>(at);
            if constexpr (kF16) {
                // in pieces of 16 bytes, of which a sequence's rows have less than 2^32
                const uint32_t r = ops_div(c, a.G), at16 = r * q_ld16 + (h * a.G.d + (c - r * a.G.d)) * (D / 8) + d / 8;
                next[i] = ld_global<ops_u32x4>(q0 + uint64_t(at16) * 16);
            }
            if constexpr (!kF16) next[i] = ld_global<ops_u32x4>(a.split + (sh * a.cols + c) * (D / 4) + part * (D / 8) + d / 8);
        }
    };
    auto lay_out = [&](uint32_t half) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t e = threadIdx.x + i * M::kThreads;
            if (M::kSets * kParts * kOps % M::kThreads == 0 || e < M::kSets * kParts * kOps) s_q[half][0][e] = next[i];
        }
    };
    KeyRows<D, kInt8> key;
    float acc[8] = {};
    if (!none) {
        const int32_t row = row_of(a.c, span, entry_of(a.c, s, base, lane), h, base, lane);
        const uint32_t there = uint32_t(__ballot(row >= 0));
        key.load(a.c, row < 0 ? 0u : uint32_t(row), lane);
        const bool whole = there == 0xFFFFFFFFu && all_see(a, n, base);
        load(0);
        key.spread(s_scale[kInt8 ? wave : 0], lane);
        for (uint32_t c = threadIdx.x; c < tiles * 16; c += M::kThreads) {
            if constexpr (!kSums) s_ml[0][c] = norm_of(a, s, h, c);
            if constexpr (!kF16) s_back[c] = ld_global<float>(a.back + sh * a.cols + (c < a.cols ? c : 0));
        }
        lay_out(0);
        __syncthreads();
        for (uint32_t stage = 0; stage < stages; ++stage) {
            if (stage + 1 < stages) load(stage + 1);
            const uint32_t tile = stage * M::kSets + set, j = tile * 16 + col;
            if (tile < tiles) {
                float x[8];
                products_of<D, kInt8, kParts>(x, key, s_q[stage & 1][set], kOps, lane);
                const float c = a.scale * kLog2e * (kF16 ? 1.0f : s_back[j]);
                const uint32_t sees = whole ? 0xFFu : seen_of(a, n, j, there, base, lane);
                if constexpr (kSums) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = sees >> i & 1 ? x[i] * c : -kInf;
                    const f32x2 v = summed(f32x2{-kInf, 0}, x);
                    if (g == 0) s_ml[quarter][j] = v;
                } else {
                    // past the columns the last one's queries, of no weight
                    const f32x2 norm = s_ml[0][j];
                    exponents_of(x, c, norm.x, whole, sees);
                    const int none = none_of(norm.y);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] += weight_of(x[i], norm.y, none);
                }
            }
            if (stage + 1 < stages) lay_out((stage + 1) & 1);
            __syncthreads();
        }
    }
    if constexpr (kSums) {
        f32x2* part = a.sums + (sh * a.parts + unit) * a.cols;
        for (uint32_t c = threadIdx.x; c < a.cols; c += M::kThreads) {
            f32x2 v{-kInf, 0};
            if (!none)
                for (int w = 0; w < kAttnWaves; ++w) v = joined(v, s_ml[w][c]);
            st_global<f32x2>(part + c, v);
        }
    } else {
        float* sums = reinterpret_cast<float*>(s_q);   // [set][cell]
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sum = over_lanes(acc[i], sum_of);
            if (int(col) == i) sums[set * kUnit + quarter * kTurn + i / 4 * 16 + g * 4 + i % 4] = sum;
        }
        __syncthreads();
        const uint32_t cell = first + threadIdx.x;
        if (threadIdx.x < kUnit && cell < n) {
            float mine = 0;
#pragma unroll
            for (uint32_t w = 0; w < M::kSets; ++w) mine += sums[w * kUnit + threadIdx.x];
            float* p = a.mass + sh * a.mass_ld + cell;
            st_global<float>(p, a.decay == 0 ? mine : a.decay * ld_global<float>(p) + mine);
        }
    }
}

// The reference and the inverse of the sum of 64 columns, from the parts that the cells were in.
constexpr uint32_t kJoinSets = 16;
__global__ void __launch_bounds__(64 * kJoinSets) mass_join_kernel(MassArgs a) {
    __shared__ f32x2 s_ml[kJoinSets][64];
    const uint32_t lane = threadIdx.x & 63, set = threadIdx.x >> 6, h = blockIdx.y, s = blockIdx.z;
    const uint32_t c = blockIdx.x * 64 + lane;
    const uint64_t sh = uint64_t(s) * a.c.H + h;
    const uint32_t all = (length_of(a, s) + kUnit - 1) / kUnit, parts = all < a.parts ? all : a.parts;
    const f32x2* first = a.sums + sh * a.parts * a.cols + (c < a.cols ? c : a.cols - 1);
    f32x2 v{-kInf, 0};
#pragma unroll 8
    for (uint32_t p = set; p < parts; p += kJoinSets) v = joined(v, ld_global<f32x2>(first + uint64_t(p) * a.cols));
    s_ml[set][lane] = v;
    __syncthreads();
    if (set) return;
    for (uint32_t k = 1; k < kJoinSets; ++k) v = joined(v, s_ml[k][lane]);
    // nothing seen, or nothing but scores of -inf: no weight; a sum that is no number makes every weight none
    if (c < a.cols) st_global<f32x2>(a.norm + sh * a.cols + c, v.y == 0 ? f32x2{kInf, 0} : f32x2{v.y == v.y ? v.x : v.y, 1.0f / v.y});
}

template <int D, bool kInt8, bool kF16>
hipError_t launch_of(const MassArgs& a, hipStream_t stream) {
    const dim3 block(kMassThreads), many(Many<D, kInt8, kF16>::kThreads), join((a.cols + 63) / 64, a.c.H, a.n_seqs), few(a.parts, a.c.H, a.n_seqs);
    if (a.cols <= 16) {
        if (!a.lse) {
            hipLaunchKernelGGL((mass_few_kernel<D, kInt8, kF16, true>), few, block, 0, stream, a);
            hipLaunchKernelGGL(mass_join_kernel, join, dim3(64 * kJoinSets), 0, stream, a);
        }
        hipLaunchKernelGGL((mass_few_kernel<D, kInt8, kF16, false>), few, block, 0, stream, a);
        return hipGetLastError();
    }
    if constexpr (!kF16) hipLaunchKernelGGL(mass_parts_kernel<D>, dim3((a.cols + 3) / 4, a.c.H, a.n_seqs), dim3(256), 0, stream, a);
    auto pass = [&](auto kernel) {
        MassArgs b = a;
        for (b.first_part = 0; b.first_part < a.parts; b.first_part += kMostParts) {
            const uint32_t left = a.parts - b.first_part;
            hipLaunchKernelGGL(kernel, dim3(left < kMostParts ? left : kMostParts, a.c.H, a.n_seqs), many, 0, stream, b);
        }
    };
    if (!a.lse) {
        pass(mass_many_kernel<D, kInt8, kF16, true>);
        hipLaunchKernelGGL(mass_join_kernel, join, dim3(64 * kJoinSets), 0, stream, a);
    }
    pass(mass_many_kernel<D, kInt8, kF16, false>);
    return hipGetLastError();
}
template <int D>
hipError_t launch_of(const MassArgs& a, int format, bool f16, hipStream_t stream) {
    if (format == 1) return f16 ? launch_of<D, true, true>(a, stream) : launch_of<D, true, false>(a, stream);
    return f16 ? launch_of<D, false, true>(a, stream) : launch_of<D, false, false>(a, stream);
}

uint64_t whole(uint64_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

uint64_t plan_mass(MassArgs& a, int head_dim, bool f16, void* workspace) {
    const uint64_t heads = uint64_t(a.n_seqs) * a.c.H;
    const uint64_t units = (uint64_t(a.max_len) + kUnit - 1) / kUnit, turns = a.cols > 16 ? 1 : units * heads / kFewSlots;
    a.parts = uint32_t(turns > 1 ? (units + turns - 1) / turns : units);   // turns that a sequence of max_len takes, alike for its parts
    uint8_t* p = static_cast<uint8_t*>(workspace);
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) { return at += whole(bytes), p ? p + at - whole(bytes) : nullptr; };
    if (!a.lse) {
        a.sums = reinterpret_cast<f32x2*>(take(heads * a.parts * a.cols * sizeof(f32x2)));
        a.norm = reinterpret_cast<f32x2*>(take(heads * a.cols * sizeof(f32x2)));
    }
    if (a.cols > 16 && !f16) {
        a.split = reinterpret_cast<ops_u32x4*>(take(heads * a.cols * uint64_t(head_dim) * 4));
        a.back = reinterpret_cast<float*>(take(heads * a.cols * 4));
    }
    return at < 16 ? 16 : at;
}

hipError_t launch_mass(const MassArgs& a, int head_dim, int format, bool f16, hipStream_t stream) {
    if (head_dim == 64) return launch_of<64>(a, format, f16, stream);
    if (head_dim == 128) return launch_of<128>(a, format, f16, stream);
    if (head_dim == 256) return launch_of<256>(a, format, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
