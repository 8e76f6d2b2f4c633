// sc_gdn.hip - the gated delta rule by single tokens (sc_gdn_step_async).
//
// A head's state M [key][value] takes one token as u = beta (v - e^g M^T k), M <- e^g M + k u^T, out = scale M^T q.  With
// both products taken of the state as it was, x = M^T k and y = M^T q, the token needs one pass over it:
//     u = beta (v - e^g x),   out = scale (e^g y + (q . k) u),   M <- e^g M + k u^T.
// Columns of the state (values) do not meet, so a workgroup takes a head's columns, or some of them, and keeps them in
// registers: four columns a lane, the keys spread over the lanes and waves and summed over them.  Reading and writing the
// state bounds it, past the caches' keeping (53 us; 58 through them): 64 sequences of 32 heads of 128, 270 MB in 48 us, 5.6 TB/s
// where this library's plain copy reaches 5.7.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr int kGdnThreads = 256;
// A decay of e^-200 is 0 in f32, and a bounded g keeps sums of decays finite.
constexpr float kLeastG = -200.0f;

// kCols columns of one head's state over one token of a sequence.
template <int S, int kCols, bool kF16>
__global__ void __launch_bounds__(kGdnThreads) gdn_step_kernel(GdnArgs a) {
    constexpr int kLanes = kCols / 4;                  // lanes across the columns
    constexpr int kGroups = kGdnThreads / kLanes;      // key groups: a thread holds keys group + i * kGroups
    constexpr int kKeys = S / kGroups;
    constexpr int kWaves = kGdnThreads / 64, kEach = (S + 63) / 64;
    static_assert(S % kGroups == 0);
    __shared__ float s_k[S], s_q[S], s_qk;
    __shared__ f32x4 s_x[kWaves][kLanes], s_y[kWaves][kLanes];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t h = blockIdx.x / (S / kCols), col = blockIdx.x % (S / kCols) * kCols, s = blockIdx.y;
    const uint32_t kh = ops_div(h, a.share), c = col + tid % kLanes * 4, group = tid / kLanes;
    const int64_t t = s;
    float* base = a.state[s];
    if (!base) {
        if (tid < kLanes) st_act4<kF16>(a.out + t * a.out_ld, h * S + c, f32x4{});
        return;
    }
    float* state = base + a.state_offset + h * a.head_ld + c;
    f32x4 m[kKeys];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) m[i] = ld_once<f32x4>(state + (group + i * kGroups) * a.key_ld);
    const float g = ld_global<float>(a.g + t * a.gate_ld + h), beta = ld_global<float>(a.beta + t * a.gate_ld + h);
    const f32x4 v = ld_act4<kF16>(a.v + t * a.v_ld, h * S + c);
    if (wave == 0) {
        float k[kEach], q[kEach], kk = 0, qq = 0, qk = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t at = lane + i * 64;
            const bool in = S >= 64 || at < S;
            if constexpr (kF16) {
                k[i] = in ? float(__builtin_bit_cast(_Float16, ld_global<uint16_t>(a.k + t * a.k_ld + (kh * S + at) * 2))) : 0.0f;
                q[i] = in ? float(__builtin_bit_cast(_Float16, ld_global<uint16_t>(a.q + t * a.q_ld + (kh * S + at) * 2))) : 0.0f;
            } else {
                k[i] = in ? ld_global<float>(a.k + t * a.k_ld + (kh * S + at) * 4) : 0.0f;
                q[i] = in ? ld_global<float>(a.q + t * a.q_ld + (kh * S + at) * 4) : 0.0f;
            }
            kk += k[i] * k[i];
            qq += q[i] * q[i];
        }
        if (a.l2norm) {
            const float rk = 1.0f / sqrtf(wave_sum(kk) + a.eps), rq = 1.0f / sqrtf(wave_sum(qq) + a.eps);
            for (int i = 0; i < kEach; ++i) k[i] *= rk, q[i] *= rq;
        }
        for (int i = 0; i < kEach; ++i) {
            qk += q[i] * k[i];
            if (S >= 64 || lane < S) s_k[(lane + i * 64) % S] = k[i], s_q[(lane + i * 64) % S] = q[i];
        }
        qk = wave_sum(qk);
        if (lane == 0) s_qk = qk;
    }
    __syncthreads();
    f32x4 x{}, y{};
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
        x += s_k[group + i * kGroups] * m[i];
        y += s_q[group + i * kGroups] * m[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = kLanes; d < 64; d <<= 1) x[j] += __shfl_xor(x[j], d), y[j] += __shfl_xor(y[j], d);
    if (lane < kLanes) s_x[wave][lane] = x, s_y[wave][lane] = y;
    __syncthreads();
    x = s_x[0][tid % kLanes], y = s_y[0][tid % kLanes];
    for (int w = 1; w < kWaves; ++w) x += s_x[w][tid % kLanes], y += s_y[w][tid % kLanes];
    const float decay = expf(g < kLeastG ? kLeastG : g);
    const f32x4 u = beta * (v - decay * x);
    if (tid < kLanes) st_act4<kF16>(a.out + t * a.out_ld, h * S + c, a.scale * (decay * y + s_qk * u));
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
        st_once<f32x4>(state + (group + i * kGroups) * a.key_ld, decay * m[i] + s_k[group + i * kGroups] * u);
}

template <int S, int kCols>
hipError_t launch_cols(const GdnArgs& a, bool f16, hipStream_t stream) {
    const dim3 grid(a.v_heads * (S / kCols), a.n_seqs), block(kGdnThreads);
    if (f16) hipLaunchKernelGGL((gdn_step_kernel<S, kCols, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((gdn_step_kernel<S, kCols, false>), grid, block, 0, stream, a);
    return hipGetLastError();
}
// The columns of a workgroup: 64, whose rows are whole lines of two, where there are workgroups of them for every unit of
// the chip twice over (64 sequences of 32 heads of 128: 47.8 us, 52.8 with 32 columns); else 32, which spreads a few heads
// wider (one sequence of 32 heads: 4.4 us, 4.8 with 64 columns).
template <int S>
hipError_t launch_of(const GdnArgs& a, bool f16, hipStream_t stream) {
    if constexpr (S >= 64)
        if (uint64_t(a.n_seqs) * a.v_heads * (S / 64) >= 512) return launch_cols<S, 64>(a, f16, stream);
    return launch_cols<S, 32>(a, f16, stream);
}

}  // namespace

hipError_t launch_gdn_step(const GdnArgs& a, int size, bool f16, hipStream_t stream) {
    if (size == 32) return launch_of<32>(a, f16, stream);
    if (size == 64) return launch_of<64>(a, f16, stream);
    if (size == 128) return launch_of<128>(a, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
