// sc_evict.hip - the cells with the most accumulated attention weight kept and moved to the front of a paged cache
// (sc_kv_evict_async).
//
// A cell's key is its mass in an order of whole numbers, the largest of all for tokens that are kept whatever their mass.  Of
// the n cells of a kv head `keep` are kept: those above the keep-th largest key T, and as many of those equal to it, from the
// lowest cell on, as there is room for.  T is found by its bytes from the highest on: the counts of a byte's values among the
// keys that share the bytes found so far.  In one more pass over the cells a prefix count gives each cell the number of kept
// ones before it, and with that the place in the list of kept cells at or past `keep` or of free places below it: the i-th of
// one goes to the i-th of the other.  No source is a destination, so rows move in any order.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr uint32_t kCopies = 32;        // counts of a byte's values, for as many lanes, so that equal keys do not meet
constexpr uint32_t kSteps = 4;          // cells of a thread between two barriers of the last pass
constexpr uint32_t kMoveThreads = 256, kMoveWaves = kMoveThreads / 64, kMoveAhead = 4;

// Masses as whole numbers in the same order: NaN below all, -0 with 0.
__device__ __forceinline__ uint32_t key_of(float mass) {
    const float m = mass + 0.0f;
    const uint32_t b = __float_as_uint(m);
    return m != m ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}
constexpr uint32_t kAlways = 0xFFFFFFFFu;   // above the key of every mass

// The cells of one kv head of one sequence.
struct Cells {
    const float* mass;
    const int32_t* born;
    uint32_t n, known;
    int64_t total, sinks, latest;   // numbers below `sinks` and from `latest` on are kept

    __device__ __forceinline__ int64_t number(uint32_t c) const {
        return c < known ? int64_t(ld_global<int32_t>(born + c)) : total - n + c;
    }
    __device__ __forceinline__ bool always(int64_t number) const { return number < sinks || number >= latest; }
};
__device__ __forceinline__ int64_t clamped(int64_t x, int64_t most) { return x < 0 ? 0 : x > most ? most : x; }
// What a sequence's entries of lens, known and total say, within their bounds.
__device__ __forceinline__ EvictSeq seq_of(const EvictArgs& a, uint32_t s) {
    EvictSeq q;
    q.n = uint32_t(clamped(ld_global<int64_t>(a.lens + s), a.max_len));
    q.known = a.born && a.known ? uint32_t(clamped(ld_global<int64_t>(a.known + s), q.n)) : 0;
    q.total = a.total ? uint32_t(clamped(ld_global<int64_t>(a.total + s), INT32_MAX)) : q.n;
    q.kept = q.n < a.keep ? q.n : a.keep;
    return q;
}
__device__ __forceinline__ Cells cells_of(const EvictArgs& a, const EvictSeq& q, uint64_t at) {
    return {a.mass + at, a.born ? a.born + at : nullptr, q.n, q.known, q.total, a.sinks, int64_t(q.total) - a.recent};
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t s_count[256 * kCopies], s_bin[256], s_found[2], s_step[2][kSteps * kSelectWaves];
    static_assert(kSteps * kSelectWaves == 64, "a wave scans a step's counts");
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.x, s = blockIdx.y;
    const uint64_t sh = uint64_t(s) * a.c.H + h, at = sh * a.ld;
    const EvictSeq seq = seq_of(a, s);
    const Cells cells = cells_of(a, seq, at);
    float* mass_out = a.mass_out + at;
    int32_t* born_out = a.born_out ? a.born_out + at : nullptr;
    if (tid == 0 && h == 0) a.seqs[s] = seq;   // lens_out may be what they came from
    if (cells.n <= a.keep) {
        for (uint32_t c = tid; c < cells.n; c += kSelectThreads) {
            if (mass_out != cells.mass) st_global<float>(mass_out + c, ld_global<float>(cells.mass + c));
            if (born_out) st_global<int32_t>(born_out + c, int32_t(cells.number(c)));
        }
        if (tid == 0) a.moved[sh] = 0;
        return;
    }
    auto key_at = [&](uint32_t c) { return cells.always(cells.number(c)) ? kAlways : key_of(ld_global<float>(cells.mass + c)); };

    uint32_t T = 0, need = a.keep;   // the bytes found, and how many of the keys that have them are kept
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (uint32_t i = tid; i < 256 * kCopies; i += kSelectThreads) s_count[i] = 0;
        __syncthreads();
        for (uint32_t c = tid; c < cells.n; c += kSelectThreads) {
            const uint32_t k = key_at(c);
            if (shift == 24 || k >> (shift + 8) == T >> (shift + 8)) atomicAdd(&s_count[(k >> shift & 255) * kCopies + lane % kCopies], 1u);
        }
        __syncthreads();
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < kCopies / 4; ++i) sum += s_count[tid / 4 * kCopies + tid % 4 * (kCopies / 4) + i];
        sum += __shfl_xor(sum, 1);
        sum += __shfl_xor(sum, 2);
        if (tid % 4 == 0) s_bin[tid / 4] = sum;
        __syncthreads();
        if (wave == 0) {   // from the largest byte down, four a lane, to where the counts reach `need`
            uint32_t v[4], mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[i] = s_bin[255 - lane * 4 - i], mine += v[i];
            const uint32_t upto = scan_add(mine);
            if (int(lane) == __builtin_ctzll(__ballot(upto >= need))) {
                uint32_t left = need - (upto - mine), byte = 255 - lane * 4;
                bool past = true;
#pragma unroll
                for (uint32_t i = 0; i < 3; ++i) {
                    past = past && left > v[i];
                    if (past) left -= v[i], --byte;
                }
                s_found[0] = byte;
                s_found[1] = left;
            }
        }
        __syncthreads();
        T |= s_found[0] << shift;
        need = s_found[1];
    }

    // The lists: cells and places in ascending order.
    uint32_t *dst = a.dst + sh * a.cap, *src = a.src + sh * a.cap;
    uint32_t above = 0, equal = 0;   // before this step's cells
    for (uint32_t first = 0, half = 0; first < cells.n; first += kSteps * kSelectThreads, half ^= 1) {
        uint64_t gt[kSteps], eq[kSteps];
        float mass[kSteps];
        int64_t number[kSteps];
#pragma unroll
        for (uint32_t i = 0; i < kSteps; ++i) {
            const uint32_t c = first + i * kSelectThreads + tid;
            const bool in = c < cells.n;
            number[i] = cells.number(in ? c : 0);
            mass[i] = ld_global<float>(cells.mass + (in ? c : 0));
            const uint32_t k = cells.always(number[i]) ? kAlways : key_of(mass[i]);
            gt[i] = __ballot(in && k > T);
            eq[i] = __ballot(in && k == T);
            if (lane == 0) s_step[half][i * kSelectWaves + wave] = uint32_t(__popcll(gt[i])) | uint32_t(__popcll(eq[i])) << 16;
        }
        __syncthreads();
        const uint32_t mine = s_step[half][lane], upto = scan_add(mine);   // at most 4096 each
#pragma unroll
        for (uint32_t i = 0; i < kSteps; ++i) {
            const uint32_t c = first + i * kSelectThreads + tid;
            const uint32_t before = uint32_t(__builtin_amdgcn_readlane(int(upto - mine), int(i * kSelectWaves + __builtin_amdgcn_readfirstlane(wave))));
            const uint64_t lower = (uint64_t(1) << lane) - 1;
            const uint32_t e = equal + (before >> 16) + uint32_t(__popcll(eq[i] & lower));
            const uint32_t rank = above + (before & 0xFFFF) + uint32_t(__popcll(gt[i] & lower)) + (e < need ? e : need);
            if (c >= cells.n) break;
            const bool kept = (gt[i] >> lane & 1) || ((eq[i] >> lane & 1) && e < need);
            if (c == a.keep) a.moved[sh] = a.keep - rank;
            if (c < a.keep) {
                if (!kept) {
                    st_global<uint32_t>(dst + (c - rank), c);
                } else {
                    if (mass_out != cells.mass) st_global<float>(mass_out + c, mass[i]);
                    if (born_out) st_global<int32_t>(born_out + c, int32_t(number[i]));
                }
            } else if (kept) {
                st_global<uint32_t>(src + (rank + a.cap - a.keep), c);
            } else {
                st_global<float>(mass_out + c, 0.0f);
            }
        }
        const uint32_t all = last_lane(upto);
        above += all & 0xFFFF;
        equal += all >> 16;
    }
}

__device__ __forceinline__ int64_t row_of(const EvictArgs& a, uint32_t s, uint32_t h, uint32_t cell) {
    const uint32_t page = ops_div(cell, a.c.ps);
    const int32_t phys = cache_page(a.c, s, page);
    return phys < 0 ? -1 : (int64_t(phys) * a.c.H + h) * a.c.ps.d + (cell - page * a.c.ps.d);
}

// Rows of kBytes from place to place, a key's and a value's by as many lanes as they have 16 bytes.
template <int kBytes, int kBlocks, bool kInt8>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(EvictArgs a) {
    constexpr uint32_t kLanes = kBytes / 16, kPairs = 64 / (2 * kLanes);   // lanes of a row, pairs of rows of a wave
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, s = blockIdx.z;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.lens_out[s] = a.seqs[s].kept;
    const uint64_t sh = uint64_t(s) * a.c.H + h;
    const uint32_t moved = a.moved[sh];
    if (moved == 0) return;
    const uint32_t *dst = a.dst + sh * a.cap, *src = a.src + sh * a.cap + (a.cap - moved);
    const uint32_t piece = lane % kLanes, value = lane / kLanes % 2;
    uint8_t* pool = value ? a.c.v : a.c.k;
    uint16_t* scales = value ? a.c.v_scale : a.c.k_scale;
    const Cells cells = cells_of(a, a.seqs[s], sh * a.ld);
    const bool first_lane = piece == 0 && value == 0;   // of a pair: it takes the mass and the number along
    for (uint32_t first = (blockIdx.x * kMoveWaves + wave) * kPairs * kMoveAhead; first < moved; first += gridDim.x * kMoveWaves * kPairs * kMoveAhead) {
        ops_u32x4 x[kMoveAhead];
        uint64_t scale[kMoveAhead];
        float mass[kMoveAhead];
        int32_t number[kMoveAhead];
        uint32_t from[kMoveAhead], to[kMoveAhead];
        int64_t r_to[kMoveAhead];
        bool there[kMoveAhead];
#pragma unroll
        for (uint32_t u = 0; u < kMoveAhead; ++u) {
            const uint32_t i = first + u * kPairs + lane / (2 * kLanes);
            there[u] = i < moved;
            from[u] = ld_global<uint32_t>(src + (there[u] ? i : 0));
            to[u] = ld_global<uint32_t>(dst + (there[u] ? i : 0));
        }
#pragma unroll
        for (uint32_t u = 0; u < kMoveAhead; ++u) {
            const int64_t r = row_of(a, s, h, from[u]);
            r_to[u] = r < 0 || !there[u] ? -1 : row_of(a, s, h, to[u]);
            const uint64_t row = r < 0 ? 0 : uint64_t(r);
            x[u] = ld_once<ops_u32x4>(pool + row * kBytes + piece * 16);
            if constexpr (kInt8) {
                const uint16_t* p = scales + row * kBlocks;
                if constexpr (kBlocks == 4) scale[u] = ld_global<uint64_t>(p);
                else if constexpr (kBlocks == 2) scale[u] = ld_global<uint32_t>(p);
                else scale[u] = ld_global<uint16_t>(p);
            }
            if (first_lane) {
                mass[u] = ld_global<float>(cells.mass + from[u]);
                if (a.born_out) number[u] = int32_t(cells.number(from[u]));
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kMoveAhead; ++u) {
            if (!there[u]) continue;
            if (r_to[u] >= 0) {
                st_global<ops_u32x4>(pool + uint64_t(r_to[u]) * kBytes + piece * 16, x[u]);
                if (kInt8 && piece == 0) {
                    uint16_t* p = scales + uint64_t(r_to[u]) * kBlocks;
                    if constexpr (kBlocks == 4) st_global<uint64_t>(p, scale[u]);
                    else if constexpr (kBlocks == 2) st_global<uint32_t>(p, uint32_t(scale[u]));
                    else st_global<uint16_t>(p, uint16_t(scale[u]));
                }
            }
            if (first_lane) {
                st_global<float>(a.mass_out + sh * a.ld + to[u], mass[u]);
                st_global<float>(a.mass_out + sh * a.ld + from[u], 0.0f);
                if (a.born_out) st_global<int32_t>(a.born_out + sh * a.ld + to[u], number[u]);
            }
        }
    }
}

template <int kBytes, int kBlocks, bool kInt8>
hipError_t launch_of(const EvictArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(a.c.H, a.n_seqs), dim3(kSelectThreads), 0, stream, a);
    constexpr uint32_t each = kMoveWaves * (64 / (2 * (kBytes / 16))) * kMoveAhead;
    const uint32_t blocks = a.cap / each + 1;
    hipLaunchKernelGGL((evict_move_kernel<kBytes, kBlocks, kInt8>), dim3(blocks < 4096 ? blocks : 4096, a.c.H, a.n_seqs), dim3(kMoveThreads), 0,
                       stream, a);
    return hipGetLastError();
}

uint64_t whole(uint64_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

uint64_t plan_evict(EvictArgs& a, void* workspace) {
    a.cap = a.max_len <= a.keep ? 0 : a.keep < a.max_len - a.keep ? a.keep : a.max_len - a.keep;
    const uint64_t heads = uint64_t(a.n_seqs) * a.c.H, list = whole(heads * a.cap * 4);
    uint8_t* p = static_cast<uint8_t*>(workspace);
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) { return at += whole(bytes), p ? p + at - whole(bytes) : nullptr; };
    a.seqs = reinterpret_cast<EvictSeq*>(take(a.n_seqs * sizeof(EvictSeq)));
    a.moved = reinterpret_cast<uint32_t*>(take(heads * 4));
    a.dst = reinterpret_cast<uint32_t*>(take(list));
    a.src = reinterpret_cast<uint32_t*>(take(list));
    return at;
}

hipError_t launch_evict(const EvictArgs& a, int head_dim, int format, hipStream_t stream) {
    const bool q8 = format == 1;
    if (head_dim == 64) return q8 ? launch_of<64, 1, true>(a, stream) : launch_of<128, 1, false>(a, stream);
    if (head_dim == 128) return q8 ? launch_of<128, 2, true>(a, stream) : launch_of<256, 2, false>(a, stream);
    if (head_dim == 256) return q8 ? launch_of<256, 4, true>(a, stream) : launch_of<512, 4, false>(a, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
