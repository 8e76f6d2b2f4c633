// sc_rope.hip - new tokens' keys and values into a paged cache, the position rotation applied on the way, and the
// queries rotated (sc_rope_append_async).
//
// A pair (a, b) of a head at position p turns by p * inv_freq[i]: a cos - b sin, a sin + b cos.  It is data movement: every
// value is read and written once, and the few operations a value hide behind that.  A workgroup takes one token (and, when
// tokens are few, a share of its rows): the token's cosines and sines are formed once in 64 bits, where the angle at
// position 10^5 still has its low digits, and its rows of queries, keys and values are then taken a wave each, four values
// a lane.  A pair's other value is in the lane itself (neighbours) or rot / 8 lanes away (halves: one lane exchange).
// 10 854 tokens of 24 + 2 x 2 heads of 256 (f32 into an f16 cache): 600 MB in 109 us, 5.5 TB/s where this library's plain copy
// reaches 5.7.  Rows asked for several at a time, before they are turned, made it slower (119 us by twos, 127 by fours): many
// waves with a row each keep memory busier than fewer with more.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"
#include "sc_quant_rows.hpp"

namespace sc {
namespace {

constexpr int kRopeThreads = 256;
// Calls with as many tokens fill the chip with a workgroup a token, and their queries do not stay in the caches until they
// are read: they are stored past them (10 K tokens of 24 heads of 256, f32: 118 us by plain stores, 109 past the caches).
// With fewer, a token's rows are shared by workgroups and the queries left in the caches for the attention that follows
// (one token of 28 rows: 3.6 us in shares, 4.5 by one workgroup).
constexpr uint32_t kManyTokens = 512;
constexpr double kTwoPi = 6.283185307179586476925286766559;

// Writes four values of a pool row at `d` in the cache's format; `row` is the pool row.
template <int D, bool kInt8>
__device__ __forceinline__ void st_cache4(uint8_t* pool, uint16_t* scales, uint64_t row, uint32_t d, f32x4 x, bool keep) {
    if constexpr (kInt8) {
        uint32_t sb;
        const uint32_t codes = q8_quad(x.x, x.y, x.z, x.w, sb);   // every lane takes part: 16 lanes share a scale
        if (keep) {
            st_global<uint32_t>(pool + row * D + d, codes);
            if (d % 64 == 0) st_global<uint16_t>(scales + row * (D / 64) + d / 64, uint16_t(sb));
        }
    } else if (keep) {
        const uint32_t lo = f16_bits_rne(__float_as_uint(x.x)) | (f16_bits_rne(__float_as_uint(x.y)) << 16);
        const uint32_t hi = f16_bits_rne(__float_as_uint(x.z)) | (f16_bits_rne(__float_as_uint(x.w)) << 16);
        st_global<ops_u32x2>(pool + (row * D + d) * 2, ops_u32x2{lo, hi});
    }
}

template <int D, bool kInt8, bool kF16, bool kMany>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(RopeArgs a) {
    constexpr uint32_t kLanes = D / 4, kRows = 64 / kLanes;   // lanes of a row, rows of a wave
    __shared__ float s_cos[D / 2], s_sin[D / 2];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = t;
    int64_t local = 0;
    if (a.cu) {
        s = seq_of_row(a.cu, a.n_seqs, t, lane);
        if (s >= a.n_seqs) return;                            // uniform: the row belongs to no sequence
        local = int64_t(t) - ld_global<int64_t>(a.cu + s);
        if (local < 0) return;
    }
    const int64_t pos = ld_global<int64_t>(a.pos0 + s) + local;
    for (uint32_t i = threadIdx.x; i < a.rot / 2; i += kRopeThreads) {
        const double angle = double(pos) * double(ld_global<float>(a.inv_freq + i));
        const float r = float(angle - rint(angle / kTwoPi) * kTwoPi);
        sincosf(r, &s_sin[i], &s_cos[i]);
    }
    __syncthreads();
    int64_t row0 = -1;                                        // pool row of kv head 0, or no row to write
    if (pos >= 0 && pos < int64_t(a.c.cells)) {
        const uint32_t cell = uint32_t(pos), page = ops_div(cell, a.c.ps);
        const int32_t phys = cache_page(a.c, s, page);
        if (phys >= 0) row0 = int64_t(phys) * a.c.H * a.c.ps.d + (cell - page * a.c.ps.d);
    }
    const uint32_t d = (lane % kLanes) * 4, total = a.n_head + 2 * a.c.H, half = a.rot / 2;
    const uint32_t stride = gridDim.y * (kRopeThreads / 64) * kRows;
    for (uint32_t base = (blockIdx.y * (kRopeThreads / 64) + wave) * kRows; base < total; base += stride) {
        const uint32_t r = base + lane / kLanes;
        const bool there = r < total, is_q = r < a.n_head, is_k = !is_q && r < a.n_head + a.c.H;
        const uint32_t h = !there ? 0 : is_q ? r : is_k ? r - a.n_head : r - a.n_head - a.c.H;
        const uint8_t* src = is_q ? a.q + t * a.q_ld : is_k ? a.k + t * a.k_ld : a.v + t * a.v_ld;
        f32x4 x = ld_act4<kF16, true>(src, h * D + d);
        if (a.rot) {
            f32x4 o{};
            uint32_t i[4];
            float sign[4];
            if (a.neighbours) {
                o = f32x4{x.y, x.x, x.w, x.z};
                for (int j = 0; j < 4; ++j) i[j] = (d + j) / 2, sign[j] = j & 1 ? 1.0f : -1.0f;
            } else {
                const uint32_t from = d < half ? lane + half / 4 : d < a.rot ? lane - half / 4 : lane;
                for (int j = 0; j < 4; ++j) {
                    o[j] = __shfl(x[j], int(from));
                    i[j] = d + j < half ? d + j : d + j - half;
                    sign[j] = d < half ? -1.0f : 1.0f;
                }
            }
            if (d < a.rot && (is_q || is_k))
                for (int j = 0; j < 4; ++j) x[j] = x[j] * s_cos[i[j]] + sign[j] * o[j] * s_sin[i[j]];
        }
        if (there && is_q) st_act4<kF16, kMany>(a.q_out + t * a.q_out_ld, h * D + d, x);
        const bool keep = there && !is_q && row0 >= 0;
        const uint64_t row = keep ? uint64_t(row0) + uint64_t(h) * a.c.ps.d : 0;
        st_cache4<D, kInt8>(is_k ? a.c.k : a.c.v, is_k ? a.c.k_scale : a.c.v_scale, row, d, x, keep);
    }
}

template <int D, bool kInt8>
hipError_t launch_of(const RopeArgs& a, bool f16, hipStream_t stream) {
    constexpr uint32_t per_wg = kRopeThreads / 64 * (64 / (D / 4));
    const uint32_t total = a.n_head + 2 * a.c.H, most = (total + per_wg - 1) / per_wg;
    const uint32_t shares = (kManyTokens + a.tokens - 1) / a.tokens, y = most < shares ? most : shares;
    const bool many = a.tokens >= kManyTokens;
    const dim3 grid(a.tokens, y), block(kRopeThreads);
    if (f16 && many) hipLaunchKernelGGL((rope_append_kernel<D, kInt8, true, true>), grid, block, 0, stream, a);
    else if (f16) hipLaunchKernelGGL((rope_append_kernel<D, kInt8, true, false>), grid, block, 0, stream, a);
    else if (many) hipLaunchKernelGGL((rope_append_kernel<D, kInt8, false, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((rope_append_kernel<D, kInt8, false, false>), grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, int head_dim, int format, bool f16, hipStream_t stream) {
    const bool q8 = format == 1;
    if (head_dim == 64) return q8 ? launch_of<64, true>(a, f16, stream) : launch_of<64, false>(a, f16, stream);
    if (head_dim == 128) return q8 ? launch_of<128, true>(a, f16, stream) : launch_of<128, false>(a, f16, stream);
    if (head_dim == 256) return q8 ? launch_of<256, true>(a, f16, stream) : launch_of<256, false>(a, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
