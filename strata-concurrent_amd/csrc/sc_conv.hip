// sc_conv.hip - the short causal convolution before a recurrent layer (sc_conv_async).
//
// out[t][c] = f(bias[c] + sum_j weight[c][j] x[t - (W - 1) + j][c]): a channel meets no other, and a row is needed by W - 1 rows
// after it.  It is data movement: a lane has four channels, their taps in registers, and goes down its rows with the last W - 1
// of them in registers too, so a row is read once, but for the W - 1 before a tile's first.  Those the caches have: a tile's
// workgroups across the channels are next to each other, so where they are 8 the tiles of the same channels are on one XCD.
//
// Measured, 10 854 rows of 8192 channels: f32 120 us, 5.9 TB/s where this library's plain copy reaches 5.7, f16 66 us, 5.4 TB/s.
// Tiles of 16 rows 123 us in f32 and of 8 rows 69 us in f16; the tiles of the same channels next to each other 158 us; outputs
// through the caches 125 us.  New tokens are a launch and a chain of loads: one of 8192 channels 3.1 us, 61 of them 4.6 us.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr uint32_t kConvThreads = 256;
// Rows of a prompt's tile, which are all asked for at once: 128 bytes a lane.
constexpr uint32_t tile_rows(bool f16) { return f16 ? 16 : 8; }

// v / (1 + e^-v) by the hardware's exponential and reciprocal, 1 unit in the last place each; 0 where e^-v is beyond 2^126.  The
// exponent t = -v log2(e) is rounded to 2^-24 of itself, which is 2^-24 |v| of e^-v: little beside a unit of an f16 result, and of an f32
// one down to kNear (3e-7), not below (4e-6 at v = -87).
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f, kLn2Rest = -1.90465421e-9f;   // kLn2Rest: ln 2 - kLn2
constexpr float kNear = -5.5f;
__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -kLog2e)); }
// Below kNear what the rounding left out, r = -v - t ln 2, is taken along, e^r being 1 + r: 2e-7 at any v.  The others get the bits
// that they get without: a wave comes here only if one of its values is far.
__device__ __forceinline__ float silu_far(float v) {
    const float x = __builtin_amdgcn_fmed3f(v, -88.0f, 200.0f);   // finite, where the result is v or 0 or no number beyond
    const float t = x * -kLog2e, e = __builtin_amdgcn_exp2f(t), r = fmaf(t, -kLn2Rest, fmaf(t, -kLn2, -x));
    return v * __builtin_amdgcn_rcpf(1.0f + fmaf(e, v < kNear ? r : 0.0f, e));
}

// Four channels of a history, a row a vector, from channel c on.
template <int W, bool kSlot>
__device__ __forceinline__ void ld_history(f32x4 (&h)[W - 1], const float* state, int64_t ld, uint32_t c) {
    if constexpr (kSlot) {
        f32x4 w[W - 1];   // [channel][row]
#pragma unroll
        for (int i = 0; i < W - 1; ++i) w[i] = ld_global<f32x4>(state + uint64_t(c) * (W - 1) + 4 * i);
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) h[k][j] = w[(j * (W - 1) + k) / 4][(j * (W - 1) + k) % 4];
    } else {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) h[k] = ld_global<f32x4>(state + k * ld + c);
    }
}
template <int W, bool kSlot>
__device__ __forceinline__ void st_history(const f32x4 (&h)[W - 1], float* state, int64_t ld, uint32_t c) {
    if constexpr (kSlot) {
        f32x4 w[W - 1];
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[(j * (W - 1) + k) / 4][(j * (W - 1) + k) % 4] = h[k][j];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) st_global<f32x4>(state + uint64_t(c) * (W - 1) + 4 * i, w[i]);
    } else {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) st_global<f32x4>(state + k * ld + c, h[k]);
    }
}

// The taps of four channels, a tap a vector.
template <int W>
__device__ __forceinline__ void ld_taps(f32x4 (&w)[W], const float* weight, uint32_t c) {
    f32x4 v[W];   // [channel][tap]
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = ld_global<f32x4>(weight + uint64_t(c) * W + 4 * i);
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) w[k][j] = v[(j * W + k) / 4][(j * W + k) % 4];
}

template <int W, bool kF16>
__device__ __forceinline__ f32x4 sum_of(const f32x4 (&before)[W - 1], f32x4 x, const f32x4 (&w)[W], f32x4 bias, bool act) {
    f32x4 y = bias;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) y += w[k] * before[k];
    y += w[W - 1] * x;
    if (!act) return y;
    if (!kF16 && __any(fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) < kNear)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = silu_far(y[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = silu(y[j]);
    }
    return y;
}

// One new token of a sequence, four channels a lane.
template <int W, bool kF16, bool kSlot>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(ConvArgs a) {
    const uint32_t c = (blockIdx.x * kConvThreads + threadIdx.x) * 4, s = blockIdx.y;
    if (c >= a.channels) return;
    uint8_t* out = a.out + int64_t(s) * a.out_ld;
    float* base = a.state[s];
    if (!base) {
        st_act4<kF16>(out, c, f32x4{});
        return;
    }
    float* state = base + a.state_offset;
    f32x4 h[W - 1], w[W];
    ld_history<W, kSlot>(h, state, a.state_ld, c);
    ld_taps<W>(w, a.weight, c);
    const f32x4 x = ld_act4<kF16>(a.x + int64_t(s) * a.x_ld, c), bias = a.bias ? ld_global<f32x4>(a.bias + c) : f32x4{};
    st_act4<kF16>(out, c, sum_of<W, kF16>(h, x, w, bias, a.silu));
#pragma unroll
    for (int k = 0; k + 1 < W - 1; ++k) h[k] = h[k + 1];
    h[W - 2] = x;
    st_history<W, kSlot>(h, state, a.state_ld, c);
}

// Where tile `tile` of a packed batch lies, the sequences' tiles in order: its sequence, the sequence's rows and which of its
// tiles it is.  One load a lane and a scan for 64 sequences.
struct Tile {
    uint32_t s, first, rows, at;
};
template <uint32_t kRows>
__device__ __forceinline__ bool tile_of(const ConvArgs& a, uint32_t tile, uint32_t lane, Tile& p) {
    uint32_t before = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 64) {
        const bool in = base + lane < a.n_seqs;
        int64_t b = in ? ld_global<int64_t>(a.cu + base + lane) : 0, e = in ? ld_global<int64_t>(a.cu + base + lane + 1) : 0;
        b = b < 0 ? 0 : b;
        e = e > int64_t(a.tokens) ? int64_t(a.tokens) : e;
        const uint32_t rows = e > b ? uint32_t(e - b) : 0u, tiles = (rows + kRows - 1) / kRows;
        const uint32_t hi = before + scan_add(tiles), lo = hi - tiles;
        const uint64_t here = __ballot(tile >= lo && tile < hi);
        if (here) {
            const int l = __builtin_ctzll(here);
            p.s = base + uint32_t(l);
            p.first = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), l));
            p.rows = uint32_t(__builtin_amdgcn_readlane(int(rows), l));
            p.at = tile - uint32_t(__builtin_amdgcn_readlane(int(lo), l));
            return true;
        }
        before = last_lane(hi);
    }
    return false;
}

// A tile of a sequence's rows.  The first tile's workgroup reads the old history and, when it has, writes the new one: no other
// one touches it.
template <int W, bool kF16, bool kSlot>
__global__ void __launch_bounds__(kConvThreads) conv_prompt_kernel(ConvArgs a) {
    constexpr uint32_t kRows = tile_rows(kF16);
    static_assert(kRows >= W - 1);
    const uint32_t tile = ops_div(blockIdx.x, a.blocks), c = ((blockIdx.x - tile * a.blocks.d) * blockDim.x + threadIdx.x) * 4;
    Tile p;
    if (!tile_of<kRows>(a, tile, threadIdx.x & 63, p)) return;
    if (c >= a.channels) return;
    const uint32_t r0 = p.at * kRows, n = p.rows - r0 < kRows ? p.rows - r0 : kRows;
    const uint8_t* x = a.x + int64_t(p.first) * a.x_ld;
    uint8_t* out = a.out + int64_t(p.first) * a.out_ld;
    float* base = a.state[p.s];
    if (!base) {
        for (uint32_t r = r0; r < r0 + n; ++r) st_act4<kF16>(out + int64_t(r) * a.out_ld, c, f32x4{});
        return;
    }
    float* state = base + a.state_offset;
    f32x4 h[W - 1], w[W], rows[kRows];
    if (r0) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) h[k] = ld_act4<kF16>(x + int64_t(r0 - (W - 1) + k) * a.x_ld, c);
    } else {
        ld_history<W, kSlot>(h, state, a.state_ld, c);
    }
    ld_taps<W>(w, a.weight, c);
    const f32x4 bias = a.bias ? ld_global<f32x4>(a.bias + c) : f32x4{};
    if (r0 == 0) {   // the new history: the last rows of the old one and the sequence's
        f32x4 next[W - 1];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            const int64_t r = int64_t(p.rows) - (W - 1) + k;
            next[k] = h[W - 2];
#pragma unroll
            for (int i = 0; i < W - 1; ++i) next[k] = r + (W - 1) == i ? h[i] : next[k];
            if (r >= 0) next[k] = ld_act4<kF16>(x + r * a.x_ld, c);
        }
        st_history<W, kSlot>(next, state, a.state_ld, c);
    }
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
        const uint32_t at = r0 + (i < n ? i : n - 1);   // past the tile's last row that row again
        rows[i] = ld_act4<kF16>(x + int64_t(at) * a.x_ld, c);
    }
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
        if (i < n) st_act4<kF16, true>(out + int64_t(r0 + i) * a.out_ld, c, sum_of<W, kF16>(h, rows[i], w, bias, a.silu));
#pragma unroll
        for (int k = 0; k + 1 < W - 1; ++k) h[k] = h[k + 1];
        h[W - 2] = rows[i];
    }
}

template <int W, bool kF16, bool kSlot>
hipError_t launch_of(ConvArgs a, hipStream_t stream) {
    const uint32_t lanes = a.channels / 4;
    if (!a.cu) {
        hipLaunchKernelGGL((conv_step_kernel<W, kF16, kSlot>), dim3((lanes + kConvThreads - 1) / kConvThreads, a.n_seqs),
                           dim3(kConvThreads), 0, stream, a);
    } else {
        // a sequence has at most one tile that is not whole
        const uint32_t tiles = a.tokens / tile_rows(kF16) + (a.n_seqs < a.tokens ? a.n_seqs : a.tokens);
        const uint32_t threads = lanes >= kConvThreads ? kConvThreads : (lanes + 63) / 64 * 64;
        a.blocks = make_fastdiv((lanes + threads - 1) / threads);
        hipLaunchKernelGGL((conv_prompt_kernel<W, kF16, kSlot>), dim3(tiles * a.blocks.d), dim3(threads), 0, stream, a);
    }
    return hipGetLastError();
}
template <int W>
hipError_t launch_of(const ConvArgs& a, bool f16, bool slot, hipStream_t stream) {
    if (slot) return f16 ? launch_of<W, true, true>(a, stream) : launch_of<W, false, true>(a, stream);
    return f16 ? launch_of<W, true, false>(a, stream) : launch_of<W, false, false>(a, stream);
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, int taps, bool f16, bool slot, hipStream_t stream) {
    if (taps == 2) return launch_of<2>(a, f16, slot, stream);
    if (taps == 3) return launch_of<3>(a, f16, slot, stream);
    if (taps == 4) return launch_of<4>(a, f16, slot, stream);
    if (taps == 5) return launch_of<5>(a, f16, slot, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
