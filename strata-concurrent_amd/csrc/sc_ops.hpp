// sc_ops.hpp - the arguments of the operators' kernels (include/sc_ops.h), shared by their host layer (sc_ops_capi.cpp)
// and the kernels (sc_rope.hip, sc_attn.hip, sc_gdn.hip).  Everything travels in the kernel arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_internal.hpp"

namespace sc {

using ops_u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using ops_u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

// A paged cache (sc_kv_cache) as the kernels see it.
struct CacheArgs {
    uint8_t *k, *v;
    uint16_t *k_scale, *v_scale;
    const int32_t* table;
    int64_t table_ld;
    uint32_t cells;       // table_ld * page_size: cells of a sequence
    uint32_t n_pages;
    uint32_t H;
    FastDiv ps;
};

struct RopeArgs {
    CacheArgs c;
    const uint8_t *k, *v, *q;
    uint8_t* q_out;
    int64_t k_ld, v_ld, q_ld, q_out_ld;   // bytes from token to token
    const int64_t *cu, *pos0;
    const float* inv_freq;
    uint32_t tokens, n_seqs, n_head, rot, neighbours;
};

struct AttnArgs {
    CacheArgs c;
    const int64_t* lens;
    const uint8_t* q;
    uint8_t* out;
    float* lse;
    int64_t q_ld, out_ld;                 // bytes from sequence to sequence
    uint32_t n_seqs, n_head, max_len, window;
    float scale;
    // how the length is split, by plan_attn
    uint32_t tiles;                       // kv heads times the tiles of 16 query heads of each
    uint32_t slots, least;                // workgroups the units are shared out among, units of a part at least
    uint32_t grid, join;                  // workgroups of the launch, whether a sequence can have more than one part
    uint32_t direct;                      // units a sequence can have, where each is a workgroup of its own; else 0
    uint32_t parts;                       // parts a sequence can have
    float* ws;                            // the parts' results
    ops_u32x2* where;                     // [n_seqs] parts of a sequence and its first one's place
};

struct GdnArgs {
    const uint8_t *q, *k, *v;
    uint8_t* out;
    int64_t q_ld, k_ld, v_ld, out_ld;     // bytes from token to token
    const float *g, *beta;
    int64_t gate_ld;
    float* const* state;
    int64_t state_offset, head_ld, key_ld;
    const int64_t* cu;
    uint32_t n_seqs, tokens, v_heads, l2norm;
    FastDiv share;                        // value heads of a key head
    float scale, eps;
};

// The chunks of one pair of launches of the chunk form.
struct ChunkArgs {
    uint32_t first, count, total;         // chunks [first, first + count) of at most `total`, of all sequences in order
    uint32_t k_heads;
    uint64_t rows_at;                     // 16-byte words before `rows`
    ops_u32x4 *chunks, *rows;             // the workspace: operands and factors of each chunk and value head; f32 rows' parts
};

hipError_t launch_rope(const RopeArgs& a, int head_dim, int format, bool f16, hipStream_t stream);
// Fills the split of a call and returns the bytes of its workspace.
uint64_t plan_attn(AttnArgs& a, int head_dim);
// Places its parts in a workspace of those bytes.
void place_attn(AttnArgs& a, void* workspace, uint64_t bytes);
hipError_t launch_attn(const AttnArgs& a, int head_dim, int format, bool f16, hipStream_t stream);
hipError_t launch_gdn_step(const GdnArgs& a, int size, bool f16, hipStream_t stream);
// Fills the pieces that a call goes in and returns the bytes of its workspace.
uint64_t plan_gdn_chunks(const GdnArgs& a, int size, bool f16, ChunkArgs& c);
hipError_t launch_gdn_chunk(const GdnArgs& a, int size, bool f16, void* workspace, hipStream_t stream);

#if defined(__HIPCC__)
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using u16x2 = __attribute__((ext_vector_type(2))) uint16_t;

__device__ __forceinline__ uint32_t ops_div(uint32_t n, const FastDiv& f) {
    return uint32_t((uint64_t(__umulhi(n, f.m)) + uint64_t(n)) >> f.s);
}

// Global memory said to be such, so that accesses are not flat ones.
template <class T>
__device__ __forceinline__ T ld_global(const void* p) {
    return *(const __attribute__((address_space(1))) T*) (p);
}
template <class T>
__device__ __forceinline__ void st_global(void* p, T v) {
    *(__attribute__((address_space(1))) T*) (p) = v;
}
// What is read or written once, past the caches' keeping.
template <class T>
__device__ __forceinline__ T ld_once(const void* p) {
    return __builtin_nontemporal_load((const __attribute__((address_space(1))) T*) (p));
}
template <class T>
__device__ __forceinline__ void st_once(void* p, T v) {
    __builtin_nontemporal_store(v, (__attribute__((address_space(1))) T*) (p));
}

// Four consecutive values of an activation row, in f32; kOnce: past the caches' keeping.
template <bool kF16, bool kOnce = false>
__device__ __forceinline__ f32x4 ld_act4(const uint8_t* row, uint32_t at) {
    if constexpr (kF16) {
        const uint8_t* p = row + uint64_t(at) * 2;
        const f16x4 h = __builtin_bit_cast(f16x4, kOnce ? ld_once<ops_u32x2>(p) : ld_global<ops_u32x2>(p));
        return f32x4{float(h.x), float(h.y), float(h.z), float(h.w)};
    } else {
        const uint8_t* p = row + uint64_t(at) * 4;
        return __builtin_bit_cast(f32x4, kOnce ? ld_once<ops_u32x4>(p) : ld_global<ops_u32x4>(p));
    }
}
template <bool kF16, bool kOnce = false>
__device__ __forceinline__ void st_act4(uint8_t* row, uint32_t at, f32x4 v) {
    if constexpr (kF16) {
        // round to nearest even: the results' type holds 11 bits
        const f16x4 h{_Float16(v.x), _Float16(v.y), _Float16(v.z), _Float16(v.w)};
        const ops_u32x2 bits = __builtin_bit_cast(ops_u32x2, h);
        uint8_t* p = row + uint64_t(at) * 2;
        if constexpr (kOnce) st_once<ops_u32x2>(p, bits);
        else st_global<ops_u32x2>(p, bits);
    } else {
        const ops_u32x4 bits = __builtin_bit_cast(ops_u32x4, v);
        uint8_t* p = row + uint64_t(at) * 4;
        if constexpr (kOnce) st_once<ops_u32x4>(p, bits);
        else st_global<ops_u32x4>(p, bits);
    }
}

// Products of matrix tiles of 32-bit numbers: a lane has one value of a row of the left and a column of the right one.
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// The maximum and the sum (or another function) over the four lanes that share lane % 16, the 16-lane rows of the wave, in
// every one of them.
template <class F>
__device__ __forceinline__ float over_rows(float x, F f) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }

// The physical page of a sequence's cell, or -1 where it is not resident.  `cell` is below c.cells.
__device__ __forceinline__ int32_t cache_page(const CacheArgs& c, uint32_t seq, uint32_t page) {
    const int64_t at = int64_t(seq) * c.table_ld + page;
    const int64_t p = c.table ? int64_t(ld_global<int32_t>(c.table + at)) : at;
    return p >= 0 && p < int64_t(c.n_pages) ? int32_t(p) : -1;
}

// The sequence of row t of a packed batch by its first rows cu[0 .. n], or n when it is past them all; every lane of the
// wave gives the same t.  One load a lane and a vote for 64 sequences.
__device__ __forceinline__ uint32_t seq_of_row(const int64_t* cu, uint32_t n, int64_t t, uint32_t lane) {
    uint32_t s = 0;
    for (uint32_t base = 0; base < n; base += 64) {
        const int64_t end = base + lane < n ? ld_global<int64_t>(cu + base + lane + 1) : INT64_MAX;
        const uint64_t before = __ballot(end <= t);
        s += uint32_t(__popcll(before));
        if (before != ~0ull) break;
    }
    return s;
}

// Inclusive sums over the wave's lanes, by row shifts and row broadcasts (no trip through LDS).
__device__ __forceinline__ uint32_t scan_add(uint32_t x) {
    x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x111, 0xF, 0xF, false));   // row_shr 1, 2, 4, 8
    x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x112, 0xF, 0xF, false));
    x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x114, 0xF, 0xF, false));
    x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x118, 0xF, 0xF, false));
    x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x142, 0xA, 0xF, false));   // lane 15 of a row to the next one
    x += uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x143, 0xC, 0xF, false));   // lane 31 to the upper half
    return x;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return uint32_t(__builtin_amdgcn_readlane(int(x), 63)); }

// Sum over a wave, the same in every lane and in the same order every time.
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
    return x;
}
#endif

}  // namespace sc
