// sc_attn_tiles.hpp - what the kernels share that multiply queries with the rows of a paged cache (sc_attn.hip, sc_mass.hip):
// operands of the matrix instructions, int8 rows as f16, where a turn's cells lie.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_attn_split.hpp"
#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();

// 2^x by the hardware's instruction (1 unit in the last place; results below the normal range are 0).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ f16x2 two(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
__device__ __forceinline__ uint32_t bits(f16x2 h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ f16x8 eight(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(f16x8, ops_u32x4{a, b, c, d});
}

// Four int8 codes with 128 added (one exclusive or) as f16: 0x64 above a byte is 1024 + the byte, exactly.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& a, uint32_t& b) {
    const f16x2 off = two(0xE480E480u);   // -1152
    a = bits(two(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off);
    b = bits(two(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off);
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
__device__ __forceinline__ int32_t entry_of(const CacheArgs& c, uint32_t s, uint32_t base, uint32_t lane) {
    const uint32_t cell = base + (lane & 31), page = ops_div(cell < c.cells ? cell : c.cells - 1, c.ps);
    const int64_t at = int64_t(s) * c.table_ld + page;
    return c.table ? ld_global<int32_t>(c.table + at) : int32_t(at);
}
// The pool row of that cell, or -1 where it is outside the span or not resident.
__device__ __forceinline__ int32_t row_of(const CacheArgs& c, const Span& p, int32_t entry, uint32_t h, uint32_t base, uint32_t lane) {
    const uint32_t cell = base + (lane & 31), page = ops_div(cell, c.ps);
    const bool in = cell >= p.first && cell < p.len && uint32_t(entry) < c.n_pages;
    return in ? int32_t((uint32_t(entry) * c.H + h) * c.ps.d + (cell - page * c.ps.d)) : -1;
}

}  // namespace
}  // namespace sc
