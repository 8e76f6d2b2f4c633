// sc_attn.hip - attention of one new token a sequence over its paged cache (sc_attn_decode_async).
//
// With scores s_j = scale * q . k_j over the cells left by the length, the window and the page table, a part of them gives
// m = max s_j, l = sum exp(s_j - m) and acc = sum exp(s_j - m) v_j; two parts join by bringing both to the larger m.  A wave
// takes a part of one query head's cells, a few lanes a cell, and a second kernel joins the parts of a head.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// Four values of a pool row.
template <int D, bool kInt8>
__device__ __forceinline__ f32x4 ld_cache4(const uint8_t* pool, const uint16_t* scales, uint64_t row, uint32_t d) {
    if constexpr (kInt8) {
        const uint32_t c = ld_global<uint32_t>(pool + row * D + d);
        const float s = float(__builtin_bit_cast(_Float16, ld_global<uint16_t>(scales + row * (D / 64) + d / 64)));
        return f32x4{float(int8_t(c)) * s, float(int8_t(c >> 8)) * s, float(int8_t(c >> 16)) * s, float(int8_t(c >> 24)) * s};
    } else {
        return ld_act4<true>(pool + row * (D * 2), d);
    }
}

// exp2(a - b) where either may be -inf: nothing weighs nothing.
__device__ __forceinline__ float weight(float a, float b) { return a == -__builtin_inff() ? 0.0f : __builtin_exp2f(a - b); }

template <int D, bool kInt8, bool kF16>
__global__ void __launch_bounds__(64) attn_part_kernel(AttnArgs a) {
    constexpr uint32_t kLanes = D / 4, kRows = 64 / kLanes;
    const uint32_t lane = threadIdx.x, s = blockIdx.x / a.n_head, head = blockIdx.x % a.n_head;
    const uint32_t h = head / (a.n_head / a.c.H), d = (lane % kLanes) * 4;
    int64_t len = ld_global<int64_t>(a.lens + s);
    len = len < 0 ? 0 : len > int64_t(a.max_len) ? int64_t(a.max_len) : len;
    const int64_t first = a.window && len > int64_t(a.window) ? len - a.window : 0;
    const int64_t lo = first > int64_t(blockIdx.y) * a.chunk ? first : int64_t(blockIdx.y) * a.chunk;
    const int64_t hi = len < int64_t(blockIdx.y + 1) * a.chunk ? len : int64_t(blockIdx.y + 1) * a.chunk;
    f32x4 q = ld_act4<kF16>(a.q + s * a.q_ld, head * D + d) * (a.scale * kLog2e), acc{};
    float m = -__builtin_inff(), l = 0;
    for (int64_t j = lo + lane / kLanes; j < hi; j += kRows) {
        const uint32_t page = ops_div(uint32_t(j), a.c.ps);
        const int32_t phys = cache_page(a.c, s, page);
        if (phys < 0) continue;
        const uint64_t row = (uint64_t(phys) * a.c.H + h) * a.c.ps.d + (uint32_t(j) - page * a.c.ps.d);
        const f32x4 k = ld_cache4<D, kInt8>(a.c.k, a.c.k_scale, row, d), v = ld_cache4<D, kInt8>(a.c.v, a.c.v_scale, row, d);
        float x = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
        for (uint32_t i = 1; i < kLanes; i <<= 1) x += __shfl_xor(x, int(i));
        if (x == -__builtin_inff()) continue;
        const float top = x > m || x != x ? x : m, w = weight(m, top), p = __builtin_exp2f(x - top);
        l = l * w + p;
        acc = acc * w + p * v;
        m = top;
    }
    for (uint32_t i = kLanes; i < 64; i <<= 1) {
        const float om = __shfl_xor(m, int(i)), ol = __shfl_xor(l, int(i));
        f32x4 oa;
        for (int j = 0; j < 4; ++j) oa[j] = __shfl_xor(acc[j], int(i));
        const float top = m > om || m != m ? m : om, w = weight(m, top), ow = weight(om, top);
        l = l * w + ol * ow;
        acc = acc * w + oa * ow;
        m = top;
    }
    float* part = a.ws + (uint64_t(blockIdx.x) * a.parts + blockIdx.y) * (D + 4);
    if (lane < kLanes) *reinterpret_cast<f32x4*>(part + 4 + d) = acc;
    if (lane == 0) part[0] = m, part[1] = l;
}

template <int D, bool kF16>
__global__ void __launch_bounds__(64) attn_join_kernel(AttnArgs a) {
    const uint32_t lane = threadIdx.x, s = blockIdx.x / a.n_head, head = blockIdx.x % a.n_head;
    const float* part = a.ws + uint64_t(blockIdx.x) * a.parts * (D + 4);
    float m = -__builtin_inff(), l = 0;
    f32x4 acc{};
    for (uint32_t i = 0; i < a.parts; ++i, part += D + 4) {
        const float om = part[0], ol = part[1], top = m > om || m != m ? m : om, w = weight(m, top), ow = weight(om, top);
        l = l * w + ol * ow;
        if (lane < D / 4) acc = acc * w + *reinterpret_cast<const f32x4*>(part + 4 + lane * 4) * ow;
        m = top;
    }
    const bool none = m == -__builtin_inff();
    if (lane < D / 4) st_act4<kF16>(a.out + s * a.out_ld, head * D + lane * 4, none ? f32x4{} : acc / l);
    if (lane == 0 && a.lse) a.lse[uint64_t(s) * a.n_head + head] = none ? m : (m + __builtin_log2f(l)) * kLn2;
}

template <int D, bool kInt8>
hipError_t launch_of(const AttnArgs& a, bool f16, hipStream_t stream) {
    const dim3 grid(a.n_seqs * a.n_head, a.parts), join(a.n_seqs * a.n_head);
    if (f16) {
        hipLaunchKernelGGL((attn_part_kernel<D, kInt8, true>), grid, dim3(64), 0, stream, a);
        hipLaunchKernelGGL((attn_join_kernel<D, true>), join, dim3(64), 0, stream, a);
    } else {
        hipLaunchKernelGGL((attn_part_kernel<D, kInt8, false>), grid, dim3(64), 0, stream, a);
        hipLaunchKernelGGL((attn_join_kernel<D, false>), join, dim3(64), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attn(const AttnArgs& a, int head_dim, int format, bool f16, hipStream_t stream) {
    const bool q8 = format == 1;
    if (head_dim == 64) return q8 ? launch_of<64, true>(a, f16, stream) : launch_of<64, false>(a, f16, stream);
    if (head_dim == 128) return q8 ? launch_of<128, true>(a, f16, stream) : launch_of<128, false>(a, f16, stream);
    if (head_dim == 256) return q8 ? launch_of<256, true>(a, f16, stream) : launch_of<256, false>(a, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
