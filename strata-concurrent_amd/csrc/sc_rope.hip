// sc_rope.hip - new tokens' keys and values into a paged cache, the position rotation applied on the way, and the
// queries rotated (sc_rope_append_async, sc_rope_axes_append_async).
//
// A pair (a, b) of a head at position p turns by p * inv_freq[i]: a cos - b sin, a sin + b cos.  It is data movement: every
// value is read and written once, and the few operations a value hide behind that.  A workgroup takes one token (and, when
// tokens are few, a share of its rows): the token's cosines and sines are formed once in 64 bits, where the angle at
// position 10^5 still has its low digits, and its rows of queries, keys and values are then taken a wave each, four values
// a lane.  A pair's other value is in the lane itself (neighbours) or rot / 8 lanes away (halves: one lane exchange).  With positions
// of several axes a pair's angle is formed of the position on its axis, which two bits of the arguments name.
//
// 10 854 tokens of 24 + 2 x 2 heads of 256: f32 into an f16 cache, 600 MB, in 101 us, f16, 311 MB, in 54 us, where this library's
// plain copy's 5.7 TB/s would take 105 and 55.  Four rows of a wave are asked for together, into registers that outlive the loop (its
// own are copied where it ends early: 107 and 66 us), where a row belongs is decided once a wave, and the sines are read once, not a row.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"
#include "sc_quant_rows.hpp"

namespace sc {
namespace {

constexpr int kRopeThreads = 256;
// How a call's rows are shared out.  A small one is a chain of latencies, of which fetching the kernel's instructions is one: where up
// to kOneRowWgs workgroups have a row a wave the kernel has no loop and asks for its row before it forms the sines, and positions of
// one axis or several (kAxes) are kernels of their own.  One token of 28 rows 3.4 us (3.9 by the loop with both), 61 tokens 3.9 (4.4),
// 100 4.1 (4.5); 200 tokens would be 1400 workgroups and 5.0 us, 4.8 by the loop.  From kManyTokens on a workgroup a token fills the chip,
// and the queries do not stay in the caches until they are read: they are stored past them (10 K tokens of 24 heads of 256, f32:
// 118 us by plain stores, 109 past the caches).  Between the two workgroups share a token's rows, up to kAhead a wave (256 tokens of 80
// rows of 128: 7.4 us, 7.9 where waves have five), and the queries are left in the caches for the attention that follows.
enum class Form { one_row, shared, many };
constexpr uint32_t kOneRowWgs = 1024, kManyTokens = 512;
constexpr uint32_t kAhead = 4;    // rows of a wave that are asked for together
constexpr double kTwoPi = 6.283185307179586476925286766559;

// Writes four values of a pool row at `d` in the cache's format; `row` is the pool row.
template <int D, bool kInt8>
__device__ __forceinline__ void st_cache4(uint8_t* pool, uint16_t* scales, uint64_t row, uint32_t d, f32x4 x) {
    if constexpr (kInt8) {
        uint32_t sb;
        const uint32_t codes = q8_quad(x.x, x.y, x.z, x.w, sb);   // 16 lanes share a scale, and a row's lanes are here together
        st_global<uint32_t>(pool + row * D + d, codes);
        if (d % 64 == 0) st_global<uint16_t>(scales + row * (D / 64) + d / 64, uint16_t(sb));
    } else {
        const uint32_t lo = f16_bits_rne(__float_as_uint(x.x)) | (f16_bits_rne(__float_as_uint(x.y)) << 16);
        const uint32_t hi = f16_bits_rne(__float_as_uint(x.z)) | (f16_bits_rne(__float_as_uint(x.w)) << 16);
        st_global<ops_u32x2>(pool + (row * D + d) * 2, ops_u32x2{lo, hi});
    }
}

template <int D, bool kInt8, bool kF16, Form kForm, bool kAxes>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(RopeArgs a) {
    constexpr uint32_t kLanes = D / 4, kRows = 64 / kLanes;   // lanes of a row, rows of a wave
    __shared__ float s_cos[D / 2], s_sin[D / 2];
    const uint32_t t = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t s = t;
    int64_t local = 0;
    if (a.cu) {
        s = seq_of_row(a.cu, a.n_seqs, t, lane);
        if (s >= a.n_seqs) return;                            // uniform: the row belongs to no sequence
        local = int64_t(t) - ld_global<int64_t>(a.cu + s);
        if (local < 0) return;
    }
    const int64_t pos = ld_global<int64_t>(a.pos0 + s) + local;
    const uint32_t d = (lane % kLanes) * 4, total = a.n_head + 2 * a.c.H, half = a.rot / 2;
    // the rows of queries, then of keys and of values: for heads of 256 a wave has one row, and where it belongs is the same for its lanes
    const uint32_t stride = gridDim.y * (kRopeThreads / 64) * kRows, first = (blockIdx.y * (kRopeThreads / 64) + wave) * kRows;
    constexpr uint32_t kHeld = kForm == Form::one_row ? 1 : kAhead;
    f32x4 rows[kHeld];
    auto ask = [&](uint32_t base) {
#pragma unroll
        for (uint32_t u = 0; u < kHeld; ++u) {
            if (base + u * stride >= total) break;
            const uint32_t r = base + u * stride + lane / kLanes, k = r - a.n_head, v = k - a.c.H;
            if (r < a.n_head) rows[u] = ld_act4<kF16, true>(a.q + t * a.q_ld, r * D + d);
            else if (k < a.c.H) rows[u] = ld_act4<kF16, true>(a.k + t * a.k_ld, k * D + d);
            else if (r < total) rows[u] = ld_act4<kF16, true>(a.v + t * a.v_ld, v * D + d);
        }
    };
    const bool in = pos >= 0 && pos < int64_t(a.c.cells);
    const uint32_t cell = in ? uint32_t(pos) : 0u, page = ops_div(cell, a.c.ps);
    auto entry_of = [&] {
        const int64_t at = int64_t(s) * a.c.table_ld + page;
        return a.c.table ? ld_global<int32_t>(a.c.table + at) : int32_t(at);
    };
    int32_t entry;
    if constexpr (kForm == Form::one_row) ask(first), entry = entry_of();   // on their way while the sines are formed
    for (uint32_t i = threadIdx.x; i < a.rot / 2; i += kRopeThreads) {
        int64_t at = pos;
        if constexpr (kAxes) {
            uint32_t word = 0;
#pragma unroll
            for (uint32_t j = 0; j < D / 32; ++j) word = i / 16 == j ? a.axis[j] : word;
            at = ld_global<int64_t>(a.pos + (word >> i % 16 * 2 & 3) * a.pos_ld + t);
        }
        const double angle = double(at) * double(ld_global<float>(a.inv_freq + i));
        const float r = float(angle - rint(angle / kTwoPi) * kTwoPi);
        sincosf(r, &s_sin[i], &s_cos[i]);
    }
    __syncthreads();
    if constexpr (kForm != Form::one_row) entry = entry_of();
    // pool row of kv head 0, or no row to write
    const int64_t row0 = in && uint32_t(entry) < a.c.n_pages ? int64_t(entry) * a.c.H * a.c.ps.d + (cell - page * a.c.ps.d) : -1;
    // the lane's turn is that of all its rows: of its value j, x cos[j] + (the pair's other value) sin[j], with the sine's sign
    const bool turns = d < a.rot;
    f32x4 cos{}, sin{};
    if (turns)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t i = a.neighbours ? (d + j) / 2 : d + j < half ? d + j : d + j - half;
            cos[j] = s_cos[i];
            sin[j] = (a.neighbours ? j % 2 == 0 : d < half) ? -s_sin[i] : s_sin[i];
        }
    const uint32_t from = d < half ? lane + half / 4 : turns ? lane - half / 4 : lane;
    auto turned = [&](f32x4 x) {
        f32x4 o{};
        if (a.neighbours) o = f32x4{x.y, x.x, x.w, x.z};
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __shfl(x[j], int(from));
        if (turns)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = fmaf(x[j], cos[j], o[j] * sin[j]);   // the same bits in every form
        return x;
    };
    for (uint32_t base = first; base < total; base += kForm == Form::one_row ? total : stride * kAhead) {
        if constexpr (kForm != Form::one_row) ask(base);
#pragma unroll
        for (uint32_t u = 0; u < kHeld; ++u) {
            if (base + u * stride >= total) break;
            const uint32_t r = base + u * stride + lane / kLanes, k = r - a.n_head, v = k - a.c.H;
            f32x4 x = rows[u];
            if (r < a.n_head) {
                st_act4<kF16, kForm == Form::many>(a.q_out + t * a.q_out_ld, r * D + d, a.rot ? turned(x) : x);
            } else if (r < total && row0 >= 0) {
                const bool is_k = k < a.c.H;
                if (is_k && a.rot) x = turned(x);
                st_cache4<D, kInt8>(is_k ? a.c.k : a.c.v, is_k ? a.c.k_scale : a.c.v_scale, uint64_t(row0) + uint64_t(is_k ? k : v) * a.c.ps.d, d, x);
            }
        }
    }
}

template <int D, bool kInt8, bool kF16, bool kAxes>
hipError_t launch_of(const RopeArgs& a, hipStream_t stream) {
    constexpr uint32_t per_wg = kRopeThreads / 64 * (64 / (D / 4));
    const uint32_t total = a.n_head + 2 * a.c.H, most = (total + per_wg - 1) / per_wg;
    // so many that a wave of a shared token asks for all of its rows at once, and the launch has kManyTokens
    const uint32_t least = a.tokens < kManyTokens ? (most + kAhead - 1) / kAhead : 1, fill = (kManyTokens + a.tokens - 1) / a.tokens;
    const uint32_t shares = least > fill ? least : fill, y = most < shares ? most : shares;
    const dim3 block(kRopeThreads);
    if (uint64_t(a.tokens) * most <= kOneRowWgs)
        hipLaunchKernelGGL((rope_append_kernel<D, kInt8, kF16, Form::one_row, kAxes>), dim3(a.tokens, most), block, 0, stream, a);
    else if (a.tokens < kManyTokens)
        hipLaunchKernelGGL((rope_append_kernel<D, kInt8, kF16, Form::shared, kAxes>), dim3(a.tokens, y), block, 0, stream, a);
    else
        hipLaunchKernelGGL((rope_append_kernel<D, kInt8, kF16, Form::many, kAxes>), dim3(a.tokens, y), block, 0, stream, a);
    return hipGetLastError();
}
template <int D, bool kInt8>
hipError_t launch_of(const RopeArgs& a, bool f16, hipStream_t stream) {
    if (a.axes) return f16 ? launch_of<D, kInt8, true, true>(a, stream) : launch_of<D, kInt8, false, true>(a, stream);
    return f16 ? launch_of<D, kInt8, true, false>(a, stream) : launch_of<D, kInt8, false, false>(a, stream);
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
