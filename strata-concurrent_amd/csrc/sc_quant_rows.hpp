// sc_quant_rows.hpp - the int8 rule of the K/V rows, as the lanes of a 16-lane DPP row hold a group of 64 values.
//
// Included by every kernel that writes int8 rows, so that an appended row and a carved one hold the same codes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_arith.hpp"
#include "sc_convert.hpp"

namespace sc {

// The int8 code rint(x / sf) clamped to [-127, 127], with x / sf the correctly rounded quotient, formed from y, the
// correctly rounded 1 / sf computed once per group: q0 = x * y, then one correction q = q0 + (x - q0 * sf) * y with
// the residual exact in an fma (Markstein's method: P. Markstein, "Computation of elementary functions on the IBM
// RISC System/6000 processor", IBM J. Res. Dev. 34(1), 1990).  That q equals the IEEE quotient for every f32
// significand over every f16 significand is checked exhaustively by the test suite; the operations scale exactly
// with the exponents, and where they would not (a residual below the normal range) |x / sf| < 2^-78 codes 0 both
// ways.  sf = +inf gives y = 0 and a NaN q, which codes 0 as x / inf does.  A NaN quotient (x NaN, or x infinite
// over an infinite scale) codes 0, as a NaN converts to integer 0.  Written as selects: every lane forms its
// quotient and discards it where the code is 0.
__device__ __forceinline__ uint32_t q8_code(float x, float sf, float y) {
#pragma clang fp contract(off)
    const float q0 = x * y;
    const float q = __builtin_fmaf(__builtin_fmaf(-q0, sf, x), y, q0);
    const float r = __builtin_rintf(q);
    const float c = __builtin_fminf(__builtin_fmaxf(r, -127.0f), 127.0f);
    const bool coded = sf > 0.0f && r == r;
    return coded ? uint32_t(int(c)) & 0xFFu : 0u;
}

// Cross-lane moves inside a 16-lane DPP row (VALU operations, no LDS round trip).  A row of 16 lanes holds one
// int8 group of 64 values; half a row holds one q4_0 block of 32.
constexpr int kDppXor1 = 0xB1;         // quad_perm [1,0,3,2]
constexpr int kDppXor2 = 0x4E;         // quad_perm [2,3,0,1]
constexpr int kDppHalfMirror = 0x141;  // lane i <-> 7 - i within each half row (pairs the two quads of a half)
constexpr int kDppMirror = 0x140;      // lane i <-> 15 - i within the row (pairs the two halves)
constexpr int kDppRowShl4 = 0x104;     // lane i reads lane i + 4 of its row (lanes 12..15 keep their own value)
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), kCtrl, 0xF, 0xF, false));
}
template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(dpp<kCtrl>(__float_as_uint(v)));
}

// The maximum over a 16-lane DPP row of non-negative, non-NaN floats, as unsigned integers: for such values the bit
// patterns order as the numbers do, so the comparison needs no NaN handling and each step folds into one DPP max.
__device__ __forceinline__ float row16_max_nonneg(float a) {
    uint32_t u = __float_as_uint(a);
    u = max(u, uint32_t(__builtin_amdgcn_update_dpp(0, int(u), kDppXor1, 0xF, 0xF, true)));
    u = max(u, uint32_t(__builtin_amdgcn_update_dpp(0, int(u), kDppXor2, 0xF, 0xF, true)));
    u = max(u, uint32_t(__builtin_amdgcn_update_dpp(0, int(u), kDppHalfMirror, 0xF, 0xF, true)));
    u = max(u, uint32_t(__builtin_amdgcn_update_dpp(0, int(u), kDppMirror, 0xF, 0xF, true)));
    return __uint_as_float(u);
}

// The int8 codes of this lane's four values x0 .. x3 (packed), and the f16 scale (bits) of its group: the 64 values of the
// 16 lanes of its DPP row.  Max |x| is over the group (fmax is exact, so any order gives the same).  It starts from 0, so
// NaNs never count; a group of NaNs only (which the reference's fmaxf reduction leaves NaN) gets the f16 NaN 0x7E00 as
// its scale, and codes 0.
__device__ __forceinline__ uint32_t q8_quad(float x0, float x1, float x2, float x3, uint32_t& sb) {
    const float a = row16_max_nonneg(fmaxf(fmaxf(fmaxf(fabsf(x0), fabsf(x1)), fmaxf(fabsf(x2), fabsf(x3))), 0.0f));
    const uint32_t real = uint32_t((x0 == x0) | (x1 == x1) | (x2 == x2) | (x3 == x3));
    const bool any_real = __float_as_uint(row16_max_nonneg(__uint_as_float(real))) != 0u;
    sb = any_real ? f16_bits_rne_not_nan(div127(a)) : 0x7E00u;   // a is never NaN, nor a / 127
    const float sf = f32_of_f16(sb);
    const float y = recip_normal(sf);   // sf is a binary16 value: 2^-24 <= sf <= 65504 wherever it codes
    return q8_code(x0, sf, y) | (q8_code(x1, sf, y) << 8) | (q8_code(x2, sf, y) << 16) | (q8_code(x3, sf, y) << 24);
}

}  // namespace sc
