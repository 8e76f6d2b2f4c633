// sc_mass.hip - the attention weights that a sequence's latest queries give its cells, added to what each cell has had before
// (sc_attn_mass_async).
//
// With scores x = scale * q . k * log2(e), a cell's weight from a query is 2^(x - m) / l for the query's reference m and the sum
// l of 2^(x - m) over its cells.  Where the attention has left the log of that sum, one pass over the keys gives the weights;
// else one pass before it gives the sums, parts of the cells by workgroups, and a small kernel joins the parts: the product is
// formed twice, which is less than writing the scores down and reading them again (rows * heads of 4 bytes a cell against a row
// of keys).
//
// A wave has 32 cells' keys in registers as the left operands of matrix products, row = cell, and goes over the kv head's queries
// of all rows, 16 columns at a time, which the workgroup lays out in LDS as right operands, the next ones while these are
// multiplied.  A lane ends with the scores of one column for eight cells, and adds their weights up over the columns by itself;
// the 16 lanes of a row of lanes are summed once at the end, always in the same order.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_attn_split.hpp"
#include "sc_attn_tiles.hpp"
#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr uint32_t kMassThreads = kAttnWaves * 64;
constexpr uint32_t kMostColumns = 1024;         // rows times query heads of a kv head
constexpr uint32_t kSumSlots = 1024;            // workgroups that the cells' parts are shared out among
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

// 16 columns' queries on their way: a wave has four of them, 16 lanes each, eight values at a time.
template <int D, bool kF16>
struct Held {
    static constexpr int kEach = D >= 128 ? D / 128 : 1;
    ops_u32x4 w[kEach][kF16 ? 1 : 2];
    float m, by;   // of the lane's column
};

// The queries' values as right operands: step d / 32, group (d % 32) / 8 where keys are f16; where they are int8, of which a lane
// has 16 of a step of 64, step d / 64 * 2 + (d % 16) / 8, group (d % 64) / 16.
template <bool kInt8>
__device__ __forceinline__ uint32_t place_of(uint32_t d) {
    return kInt8 ? (d / 64 * 2 + d % 16 / 8) * 64 + d % 64 / 16 * 16 : d / 32 * 64 + d % 32 / 8 * 16;
}

template <int D, bool kInt8, bool kF16, bool kSums>
__global__ void __launch_bounds__(kMassThreads) mass_kernel(MassArgs a) {
    using H = Held<D, kF16>;
    constexpr int kParts = kF16 ? 1 : 2, kSteps = D / 32, kBlocks = D / 64;
    __shared__ ops_u32x4 s_q[2][kParts][kSteps * 64];
    __shared__ float s_back[2][16];
    __shared__ f32x2 s_ml[kSums ? kAttnWaves : 1][kSums ? kMostColumns : 1];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15, h = blockIdx.y, s = blockIdx.z;
    const uint32_t n = length_of(a, s), units = (n + kUnit - 1) / kUnit;
    const uint32_t u0 = blockIdx.x * (kSums ? a.per : 1), u1 = u0 + (kSums ? a.per : 1) < units ? u0 + (kSums ? a.per : 1) : units;
    if (u0 >= u1) return;
    const uint32_t tiles = (a.cols + 15) / 16;
    // Row r sees cells [ends - window, ends) with ends = n - rows + 1 + r: all rows see those below `all` and from `late` on, none
    // one below `seen`.
    const int64_t all = int64_t(n) - a.rows + 1;
    const int64_t late = a.window ? int64_t(n) - a.window : 0, seen = a.window ? all - a.window : 0;

    auto load = [&](H& q, uint32_t tile) {
        const uint32_t c4 = tile * 16 + wave * 4 + g, c = c4 < a.cols ? c4 : a.cols - 1, r = ops_div(c, a.G);
        const uint8_t* p = a.q + (int64_t(s) * a.rows + r) * a.q_ld + int64_t(h * a.G.d + (c - r * a.G.d)) * D * (kF16 ? 2 : 4);
#pragma unroll
        for (int k = 0; k < H::kEach; ++k) {
            const uint32_t e = D >= 128 ? col + 16 * k : col % 8;
            q.w[k][0] = ld_global<ops_u32x4>(p + e * (kF16 ? 16 : 32));
            if constexpr (!kF16) q.w[k][1] = ld_global<ops_u32x4>(p + e * 32 + 16);
        }
        if constexpr (!kSums) {
            const uint32_t mine = tile * 16 + col, j = mine < a.cols ? mine : a.cols - 1, row = ops_div(j, a.G);
            if (a.lse) {
                // the log of the sum in base 2, a whole number of it apart: differences from that keep their bits
                const float lse = ld_global<float>(a.lse + (int64_t(s) * a.rows + row) * a.n_head + h * a.G.d + (j - row * a.G.d));
                const float t = lse * kLog2e, rest = fmaf(lse, kLog2e, -t) + lse * kLog2eRest;
                q.m = rintf(t);
                q.by = exp2_fast((q.m - t) - rest);
                if (fabsf(lse) == kInf) q.m = kInf, q.by = lse > 0 ? 1.0f : 0.0f;
            } else {
                const f32x2 v = ld_global<f32x2>(a.norm + (uint64_t(s) * a.c.H + h) * a.cols + j);
                q.m = v.x, q.by = v.y;
            }
            if (mine >= a.cols) q.m = kInf, q.by = 0;
        }
    };
    auto lay_out = [&](const H& q, uint32_t tile, uint32_t half) {
        const uint32_t c4 = wave * 4 + g;
        const bool real = tile * 16 + c4 < a.cols;
        if constexpr (kF16) {
#pragma unroll
            for (int k = 0; k < H::kEach; ++k) {
                const uint32_t e = D >= 128 ? col + 16 * k : col % 8;
                if (D >= 128 || col < 8) s_q[half][0][place_of<kInt8>(e * 8) + c4] = real ? q.w[k][0] : ops_u32x4{};
            }
        } else {
            // scaled by a power of two to a largest value of 2^14 .. 2^15, so that the two f16 parts of values down to 2^-16 of
            // that keep all bits: a key can be as much larger there
            float top = 0;
#pragma unroll
            for (int k = 0; k < H::kEach; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(__uint_as_float(q.w[k][i / 4][i % 4])));
            top = over_lanes(top, max_of);
            float by = 1.0f, back = 1.0f;
            if (top > 0) {
                const int e = int(__float_as_uint(top) >> 23) - 127, f = e > 127 ? 127 : e < -112 ? -112 : e;
                by = __uint_as_float(uint32_t(127 + 14 - f) << 23);
                back = __uint_as_float(uint32_t(127 - 14 + f) << 23);
            }
            if (col == 0) s_back[half][c4] = back;
#pragma unroll
            for (int k = 0; k < H::kEach; ++k) {
                const uint32_t e = D >= 128 ? col + 16 * k : col % 8;
                f16x8 hi, lo;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = real ? __uint_as_float(q.w[k][i / 4][i % 4]) * by : 0.0f;
                    hi[i] = _Float16(x);
                    lo[i] = _Float16(x - float(hi[i]));
                }
                if (D >= 128 || col < 8) {
                    s_q[half][0][place_of<kInt8>(e * 8) + c4] = __builtin_bit_cast(ops_u32x4, hi);
                    s_q[half][kParts - 1][place_of<kInt8>(e * 8) + c4] = __builtin_bit_cast(ops_u32x4, lo);
                }
            }
        }
    };
    if constexpr (kSums)
        for (uint32_t c = lane; c < tiles * 16; c += 64) s_ml[wave][c] = f32x2{-kInf, 0};

    float acc[8] = {};
    H next;
    for (uint32_t u = u0; u < u1; ++u) {
        if (int64_t(u + 1) * kUnit <= seen) continue;
        // this wave's 32 cells; where they are none it goes through the columns all the same, for the barriers
        const uint32_t base = u * kUnit + wave * kTurn;
        const Span span{0, n, 0, 0};
        int32_t row = row_of(a.c, span, entry_of(a.c, s, base, lane), h, base, lane);
        const uint32_t there = uint32_t(__ballot(row >= 0));
        row = row < 0 ? 0 : row;
        ops_u32x4 key[2][kSteps];
        uint32_t ks[kInt8 ? 8 : 1][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t at = uint32_t(__shfl(row, int(t * 16 + col)));
            const uint8_t* p = a.c.k + uint64_t(at) * (kInt8 ? D : D * 2) + g * 16;
            if constexpr (kInt8) {
#pragma unroll
                for (int i = 0; i < kBlocks; ++i) {
                    const ops_u32x4 w = ld_once<ops_u32x4>(p + i * 64) ^ 0x80808080u;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t x[4];
                        codes4(w[2 * k], x[0], x[1]);
                        codes4(w[2 * k + 1], x[2], x[3]);
                        key[t][2 * i + k] = ops_u32x4{x[0], x[1], x[2], x[3]};
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) key[t][i] = ld_global<ops_u32x4>(p + i * 64);
            }
        }
        if constexpr (kInt8)
#pragma unroll
            for (int i = 0; i < 8; ++i) ld_scales<D>(ks[i], a.c.k_scale, uint32_t(__shfl(row, int(i / 4 * 16 + g * 4 + i % 4))));
        const bool whole = there == 0xFFFFFFFFu && int64_t(base) + kTurn <= all && int64_t(base) >= late;

        load(next, 0);
        if (kSums) __syncthreads();   // the last cells' products have read what is written now
        lay_out(next, 0, 0);
        float m = next.m, by = next.by;
        for (uint32_t tile = 0; tile < tiles; ++tile) {
            const uint32_t half = tile & 1;
            __syncthreads();
            if (tile + 1 < tiles) load(next, tile + 1);
            f32x4 hi[2]{}, lo[2]{};   // products with the queries' first part, and with their second
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                f16x8 q[kParts][2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < kParts; ++i) q[i][k] = __builtin_bit_cast(f16x8, s_q[half][i][(2 * b + k) * 64 + lane]);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    f32x4 bh{}, bl{};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const f16x8 x = __builtin_bit_cast(f16x8, key[t][2 * b + k]);
                        (kInt8 ? bh : hi[t]) = mfma(x, q[0][k], kInt8 ? bh : hi[t]);
                        if constexpr (!kF16) (kInt8 ? bl : lo[t]) = mfma(x, q[kParts - 1][k], kInt8 ? bl : lo[t]);
                    }
                    if constexpr (kInt8)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float scale = scale_of(ks[t * 4 + i], b);
                            hi[t][i] += scale * bh[i];
                            if constexpr (!kF16) lo[t][i] += scale * bl[i];
                        }
                }
            }
            const float c = a.scale * kLog2e * (kF16 ? 1.0f : s_back[half][col]);
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // an infinite key makes the second part's product NaN: the first part has the score
                const float first = hi[i / 4][i % 4];
                x[i] = c * (kF16 || !(fabsf(first) < kInf) ? first : first + lo[i / 4][i % 4]);
            }
            uint32_t sees = 0xFF;   // of the lane's eight cells, those that its column sees
            if (!whole) {
                const uint32_t j = tile * 16 + col, r = ops_div(j < a.cols ? j : a.cols - 1, a.G);
                const int64_t ends = all + r, begins = a.window ? ends - a.window : 0;
                sees = 0;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t in = i / 4 * 16 + g * 4 + i % 4;
                    const int64_t cell = int64_t(base) + in;
                    sees |= uint32_t((there >> in & 1) && cell < ends && cell >= begins) << i;
                }
            }
            if constexpr (kSums) {
                float top = -kInf, sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = sees >> i & 1 ? x[i] : -kInf;
                    top = fmaxf(top, x[i]);
                }
                const f32x2 old = s_ml[wave][tile * 16 + col];
                const float M = fmaxf(old.x, floorf(over_rows(top, max_of))), ref = M == -kInf ? 0.0f : M;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += exp2_fast(x[i] - ref);
                sum = over_rows(sum, sum_of);
                if (g == 0) s_ml[wave][tile * 16 + col] = f32x2{M, old.y * exp2_fast(old.x - ref) + sum};
            } else {
                sees = by == 0 ? 0u : sees;   // nor past the columns, where an infinite key has made NaN with a query of zeros
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float w = exp2_fast(x[i] - m) * by;
                    acc[i] += sees >> i & 1 ? w : 0.0f;
                }
            }
            if (tile + 1 < tiles) lay_out(next, tile + 1, half ^ 1);
            m = next.m, by = next.by;
        }
    }

    if constexpr (kSums) {
        __syncthreads();
        f32x2* part = a.sums + ((uint64_t(s) * a.c.H + h) * a.parts + blockIdx.x) * a.cols;
        for (uint32_t c = threadIdx.x; c < a.cols; c += kMassThreads) {
            float M = -kInf, l = 0;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) M = fmaxf(M, s_ml[w][c].x);
            const float ref = M == -kInf ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) l += s_ml[w][c].y * exp2_fast(s_ml[w][c].x - ref);
            st_global<f32x2>(part + c, f32x2{M, l});
        }
    } else {
        float mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sum = over_lanes(acc[i], sum_of);
            mine = int(col) == i ? sum : mine;
        }
        const uint32_t cell = u0 * kUnit + wave * kTurn + col / 4 * 16 + g * 4 + col % 4;
        if (col < 8 && cell < n) {
            float* p = a.mass + (uint64_t(s) * a.c.H + h) * a.mass_ld + cell;
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
    const uint32_t units = (length_of(a, s) + kUnit - 1) / kUnit, parts = (units + a.per - 1) / a.per;
    const f32x2* first = a.sums + sh * a.parts * a.cols + (c < a.cols ? c : a.cols - 1);
    auto add = [](float& M, float& l, f32x2 v) {
        const float to = fmaxf(M, v.x), ref = to == -kInf ? 0.0f : to;
        l = l * exp2_fast(M - ref) + v.y * exp2_fast(v.x - ref);
        M = to;
    };
    float M = -kInf, l = 0;
#pragma unroll 8
    for (uint32_t p = set; p < parts; p += kJoinSets) add(M, l, ld_global<f32x2>(first + uint64_t(p) * a.cols));
    s_ml[set][lane] = f32x2{M, l};
    __syncthreads();
    if (set) return;
    for (uint32_t k = 1; k < kJoinSets; ++k) add(M, l, s_ml[k][lane]);
    // nothing seen, or nothing but scores of -inf: no weight
    if (c < a.cols) st_global<f32x2>(a.norm + sh * a.cols + c, l == 0 ? f32x2{kInf, 0} : f32x2{M, 1.0f / l});
}

template <int D, bool kInt8, bool kF16>
hipError_t launch_of(const MassArgs& a, hipStream_t stream) {
    const dim3 block(kMassThreads);
    if (!a.lse) {
        hipLaunchKernelGGL((mass_kernel<D, kInt8, kF16, true>), dim3(a.parts, a.c.H, a.n_seqs), block, 0, stream, a);
        hipLaunchKernelGGL(mass_join_kernel, dim3((a.cols + 63) / 64, a.c.H, a.n_seqs), dim3(64 * kJoinSets), 0, stream, a);
    }
    hipLaunchKernelGGL((mass_kernel<D, kInt8, kF16, false>), dim3((a.max_len + kUnit - 1) / kUnit, a.c.H, a.n_seqs), block, 0, stream, a);
    return hipGetLastError();
}
template <int D>
hipError_t launch_of(const MassArgs& a, int format, bool f16, hipStream_t stream) {
    if (format == 1) return f16 ? launch_of<D, true, true>(a, stream) : launch_of<D, true, false>(a, stream);
    return f16 ? launch_of<D, false, true>(a, stream) : launch_of<D, false, false>(a, stream);
}

}  // namespace

uint64_t plan_mass(MassArgs& a, void* workspace) {
    if (a.lse || a.max_len == 0) return 16;
    const uint64_t units = (uint64_t(a.max_len) + kUnit - 1) / kUnit, heads = uint64_t(a.n_seqs) * a.c.H;
    a.per = uint32_t((units * heads + kSumSlots - 1) / kSumSlots);
    a.parts = uint32_t((units + a.per - 1) / a.per);
    a.sums = static_cast<f32x2*>(workspace);
    a.norm = a.sums + heads * a.parts * a.cols;
    return heads * (a.parts + 1) * a.cols * sizeof(f32x2);
}

hipError_t launch_mass(const MassArgs& a, int head_dim, int format, bool f16, hipStream_t stream) {
    if (head_dim == 64) return launch_of<64>(a, format, f16, stream);
    if (head_dim == 128) return launch_of<128>(a, format, f16, stream);
    if (head_dim == 256) return launch_of<256>(a, format, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
