// sc_evict.hip - the cells with the most accumulated attention weight kept and moved to the front of a paged cache
// (sc_kv_evict_async).
//
// A cell's key is its mass in an order of whole numbers, the largest of all for tokens that are kept whatever their mass.  Of
// the n cells of a kv head `keep` are kept: those above the keep-th largest key T, and as many of those equal to it, from the
// lowest cell on, as there is room for.  T is found by parts of 11, 11 and 10 bits from the highest on: the counts of a part's
// values among the keys that share the parts found so far.  In one more pass over the cells a prefix count gives each cell the
// number of kept ones before it, and with that the place in the list of kept cells at or past `keep` or of free places below it:
// the i-th of one goes to the i-th of the other.  No source is a destination, so rows move in any order.
//
// A workgroup chooses for a head; its keys stay in registers where it has them all, and a thread asks for all of its cells at
// once (asked for one by one 131 072 cells took it 210 us).  What bounds it is a chain of latencies and barriers: 9 us for 4 K
// cells.  Where a head can move few rows the workgroup moves them itself (32 caches of 2064 cells to 2048: 10 us in all, 14
// with a launch for the moves).  One workgroup is bound by its unit's instructions for many cells, so from three chunks on, if
// heads are few, several share a head and a launch ends each part: 131 072 cells 35 us (134 by one), 16 K cells 33 us in all
// where one workgroup takes 29.  The moves are bound by rows of 512 bytes at places all over the pool: 57 MB in 16 us, 3.6 TB/s;
// two pairs of a wave on their way (four 18 us, and 15 us against 13.4 for 8 short caches), through the caches (past them 18).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr uint32_t kHold = 8, kChunk = kHold * kSelectThreads;   // cells that a thread, and the workgroup, has in registers
constexpr uint32_t kCopies = 4;         // counts of each value, for as many lanes, so that equal ones seldom meet
constexpr uint32_t kValues = 2048;      // of a part of a key
constexpr uint32_t kCopy = kValues + 2; // from copy to copy: another bank
constexpr uint32_t kFewMoves = 128;     // moves of a head at most that are made where they are chosen
constexpr uint32_t kShares = 256;       // workgroups that heads of more than a chunk are shared out among, a chunk each at least
constexpr uint32_t kLeastShares = 3;    // that a head is shared out among
constexpr uint32_t kMoveThreads = 256, kMoveWaves = kMoveThreads / 64, kMoveAhead = 2;
constexpr int kParts = 3, kShift[kParts] = {21, 10, 0};   // the parts of a key, from the highest on

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
    int32_t before, sinks, latest;   // tokens that have no cell any more; numbers below `sinks` and from `latest` on are kept

    __device__ __forceinline__ int32_t number(uint32_t c) const {
        return c < known ? ld_global<int32_t>(born + c) : before + int32_t(c);
    }
    __device__ __forceinline__ bool always(int32_t number) const { return number < sinks || number >= latest; }
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
    return {a.mass + at, a.born ? a.born + at : nullptr, q.n, q.known, int32_t(q.total) - int32_t(q.n), int32_t(a.sinks),
            int32_t(q.total) - int32_t(a.recent)};
}

__device__ __forceinline__ int64_t row_of(const EvictArgs& a, uint32_t s, uint32_t h, uint32_t cell) {
    const uint32_t page = ops_div(cell, a.c.ps);
    const int32_t phys = cache_page(a.c, s, page);
    return phys < 0 ? -1 : (int64_t(phys) * a.c.H + h) * a.c.ps.d + (cell - page * a.c.ps.d);
}

// A row of a cache: its bytes, its blocks' scales where it is int8.
template <int kBytes_, int kBlocks_, bool kInt8_>
struct Row {
    static constexpr int kBytes = kBytes_, kBlocks = kBlocks_;
    static constexpr bool kInt8 = kInt8_;
    static constexpr uint32_t kLanes = kBytes / 16, kPairs = 64 / (2 * kLanes);   // lanes of a row, pairs of rows of a wave
};

// Moves number `wave`, `wave` + `waves`, ... of `moved`, kMoveAhead times kPairs at a time: a key's and a value's row by as many lanes
// as they have 16 bytes, the mass and the number along with the key.
template <class R, class Dst, class Src>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const Cells& cells, uint32_t s, uint32_t h, uint32_t moved, uint32_t wave,
                                          uint32_t waves, uint32_t lane, Dst dst, Src src) {
    const uint64_t at = (uint64_t(s) * a.c.H + h) * a.ld;
    const uint32_t piece = lane % R::kLanes, value = lane / R::kLanes % 2;
    uint8_t* pool = value ? a.c.v : a.c.k;
    uint16_t* scales = value ? a.c.v_scale : a.c.k_scale;
    const bool first_lane = piece == 0 && value == 0;
    for (uint32_t first = wave * R::kPairs * kMoveAhead; first < moved; first += waves * R::kPairs * kMoveAhead) {
        ops_u32x4 x[kMoveAhead];
        uint64_t scale[kMoveAhead];
        float mass[kMoveAhead];
        int32_t number[kMoveAhead];
        uint32_t from[kMoveAhead], to[kMoveAhead];
        int64_t r_to[kMoveAhead];
        bool there[kMoveAhead];
#pragma unroll
        for (uint32_t u = 0; u < kMoveAhead; ++u) {
            const uint32_t i = first + u * R::kPairs + lane / (2 * R::kLanes);
            there[u] = i < moved;
            from[u] = src(there[u] ? i : 0);
            to[u] = dst(there[u] ? i : 0);
        }
#pragma unroll
        for (uint32_t u = 0; u < kMoveAhead; ++u) {
            const int64_t r = row_of(a, s, h, from[u]), t = row_of(a, s, h, to[u]);
            r_to[u] = r < 0 || !there[u] ? -1 : t;
            const uint64_t row = r < 0 ? 0 : uint64_t(r);
            x[u] = ld_global<ops_u32x4>(pool + row * R::kBytes + piece * 16);
            if constexpr (R::kInt8) {
                const uint16_t* p = scales + row * R::kBlocks;
                if constexpr (R::kBlocks == 4) scale[u] = ld_global<uint64_t>(p);
                else if constexpr (R::kBlocks == 2) scale[u] = ld_global<uint32_t>(p);
                else scale[u] = ld_global<uint16_t>(p);
            }
            if (first_lane) {
                mass[u] = ld_global<float>(cells.mass + from[u]);
                if (a.born_out) number[u] = cells.number(from[u]);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kMoveAhead; ++u) {
            if (!there[u]) continue;
            if (r_to[u] >= 0) {
                st_global<ops_u32x4>(pool + uint64_t(r_to[u]) * R::kBytes + piece * 16, x[u]);
                if (R::kInt8 && piece == 0) {
                    uint16_t* p = scales + uint64_t(r_to[u]) * R::kBlocks;
                    if constexpr (R::kBlocks == 4) st_global<uint64_t>(p, scale[u]);
                    else if constexpr (R::kBlocks == 2) st_global<uint32_t>(p, uint32_t(scale[u]));
                    else st_global<uint16_t>(p, uint16_t(scale[u]));
                }
            }
            if (first_lane) {
                st_global<float>(a.mass_out + at + to[u], mass[u]);
                st_global<float>(a.mass_out + at + from[u], 0.0f);
                if (a.born_out) st_global<int32_t>(a.born_out + at + to[u], number[u]);
            }
        }
    }
}

// ---- the choice -----------------------------------------------------------------------------------------------------------

struct Shared {
    alignas(16) uint32_t count[kCopy * kCopies];
    alignas(16) uint32_t step[2][kHold * kSelectWaves];
    uint32_t wave[kSelectWaves], found[2], moved;
};

// Keys of cells first + i * kSelectThreads + tid: asked for together, since latency is what a few take.
struct Keys {
    uint32_t k[kHold];
    __device__ __forceinline__ void load(const Cells& cells, uint32_t first, uint32_t end) {
        float m[kHold];
        int32_t number[kHold];
#pragma unroll
        for (uint32_t i = 0; i < kHold; ++i) {
            if (first + i * kSelectThreads >= end) break;
            const uint32_t c = first + i * kSelectThreads + threadIdx.x;
            m[i] = ld_global<float>(cells.mass + (c < end ? c : first));
            number[i] = cells.number(c < end ? c : first);
        }
#pragma unroll
        for (uint32_t i = 0; i < kHold; ++i) {
            if (first + i * kSelectThreads >= end) break;
            k[i] = cells.always(number[i]) ? kAlways : key_of(m[i]);
        }
    }
};

// Counts the values of part kPart among the keys of cells [begin, end) that share T's parts before it.  Keys that the workgroup
// has (`held`) are those of its cells.
template <int kPart>
__device__ __forceinline__ void count_keys(Shared& s, Keys& keys, bool held, const Cells& cells, uint32_t begin, uint32_t end, uint32_t T) {
    constexpr uint32_t shift = kShift[kPart], values = kPart == kParts - 1 ? 1u << kShift[kPart - 1] : kValues;
    constexpr uint32_t above = kPart == 0 ? 0u : ~0u << kShift[kPart ? kPart - 1 : 0];
    uint32_t* mine = s.count + threadIdx.x % kCopies * kCopy;
    for (uint32_t first = begin; first < end; first += kChunk) {
        if (!held) keys.load(cells, first, end);
#pragma unroll
        for (uint32_t i = 0; i < kHold; ++i) {
            if (first + i * kSelectThreads >= end) break;
            const uint32_t k = keys.k[i];
            if (first + i * kSelectThreads + threadIdx.x < end && ((k ^ T) & above) == 0) atomicAdd(&mine[k >> shift & (values - 1)], 1u);
        }
    }
}

// A thread's two values, the largest first, and their counts in shared memory, which it leaves 0.
__device__ __forceinline__ uint32_t value_of(uint32_t j) { return kValues - 1 - 2 * threadIdx.x - j; }
__device__ __forceinline__ void take_counts(Shared& s, uint32_t (&v)[2]) {
    ops_u32x2* pair = reinterpret_cast<ops_u32x2*>(&s.count[value_of(1)]);
    v[0] = v[1] = 0;
#pragma unroll
    for (uint32_t i = 0; i < kCopies; ++i) {
        v[0] += pair[i * (kCopy / 2)].y;
        v[1] += pair[i * (kCopy / 2)].x;
        pair[i * (kCopy / 2)] = ops_u32x2{};
    }
}
// Sums over the workgroup's threads up to this one's; barriers on both sides of what it shares.
__device__ __forceinline__ uint32_t sum_upto(Shared& s, uint32_t x, uint32_t wave, uint32_t lane) {
    uint32_t upto = scan_add(x);
    if (lane == 63) s.wave[wave] = upto;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w + 1 < kSelectWaves; ++w) upto += w < wave ? s.wave[w] : 0u;
    return upto;
}
// The value at which the counts of all from the largest on reach `need`: it goes to T, what is left of need to `need`.
__device__ __forceinline__ void find(Shared& s, const uint32_t (&v)[2], int shift, uint32_t wave, uint32_t lane, uint32_t& T, uint32_t& need) {
    const uint32_t mine = v[0] + v[1], upto = sum_upto(s, mine, wave, lane);
    if (upto >= need && upto - mine < need) {   // one thread
        const uint32_t left = need - (upto - mine), second = left > v[0];
        s.found[0] = value_of(second);
        s.found[1] = second ? left - v[0] : left;
    }
    __syncthreads();
    T |= s.found[0] << shift;
    need = s.found[1];
}

// The lists of the moves, cells and places in ascending order, from cells [begin, end), with `above` keys above T and `equal` equal ones
// before them; what stays where it is goes to the outputs.
template <bool kFew>
__device__ __forceinline__ void list_moves(Shared& s, Keys& keys, bool held, const EvictArgs& a, const Cells& cells, uint64_t sh, uint32_t begin,
                                           uint32_t end, uint32_t T, uint32_t need, uint32_t above, uint32_t equal, uint32_t wave, uint32_t lane) {
    float* mass_out = a.mass_out + sh * a.ld;
    int32_t* born_out = a.born_out ? a.born_out + sh * a.ld : nullptr;
    uint32_t half = 0;
    for (uint32_t first = begin; first < end; first += kChunk, half ^= 1) {
        if (!held) keys.load(cells, first, end);
        uint64_t gt[kHold], eq[kHold];
#pragma unroll
        for (uint32_t i = 0; i < kHold; ++i) {
            const bool in = first + i * kSelectThreads + threadIdx.x < end;
            gt[i] = __ballot(in && keys.k[i] > T);
            eq[i] = __ballot(in && keys.k[i] == T);
            if (lane == 0) s.step[half][i * kSelectWaves + wave] = uint32_t(__popcll(gt[i])) | uint32_t(__popcll(eq[i])) << 16;
        }
        __syncthreads();
        // a lane sums up two of the 128 counts, in the cells' order; a total is at most 2^13
        static_assert(kHold * kSelectWaves == 128);
        const ops_u32x2 two = reinterpret_cast<const ops_u32x2*>(s.step[half])[lane];
        const uint32_t sum = two.x + two.y, upto = scan_add(sum), mine = upto - sum + (wave % 2 ? two.x : 0u);
#pragma unroll
        for (uint32_t i = 0; i < kHold; ++i) {
            if (first + i * kSelectThreads >= end) break;
            const uint32_t c = first + i * kSelectThreads + threadIdx.x;
            const uint32_t before = uint32_t(__builtin_amdgcn_readlane(int(mine), int(i * (kSelectWaves / 2) + wave / 2)));
            const uint64_t lower = (uint64_t(1) << lane) - 1;
            const uint32_t e = equal + (before >> 16) + uint32_t(__popcll(eq[i] & lower));
            const uint32_t rank = above + (before & 0xFFFF) + uint32_t(__popcll(gt[i] & lower)) + (e < need ? e : need);
            const bool kept = (gt[i] >> lane & 1) || ((eq[i] >> lane & 1) && e < need);
            if (c >= end) continue;
            if (c == a.keep) (kFew ? s.moved : a.moved[sh]) = a.keep - rank;
            if (c < a.keep) {
                if (!kept) {
                    (kFew ? s.count : a.dst + sh * a.cap)[c - rank] = c;
                } else {
                    if (mass_out != cells.mass) st_global<float>(mass_out + c, ld_global<float>(cells.mass + c));
                    if (born_out && (born_out != cells.born || c >= cells.known)) st_global<int32_t>(born_out + c, cells.number(c));
                }
            } else if (kept) {
                (kFew ? s.count + kFewMoves : a.src + sh * a.cap)[rank + a.cap - a.keep] = c;
            } else {
                st_global<float>(mass_out + c, 0.0f);
            }
        }
        const uint32_t all = last_lane(upto);
        above += all & 0xFFFF;
        equal += all >> 16;
    }
}

// What a sequence that has no more than it may keep leaves, cells c, c + by, ...
__device__ __forceinline__ void pass_on(const EvictArgs& a, const Cells& cells, uint64_t sh, uint32_t c, uint32_t by) {
    float* mass_out = a.mass_out + sh * a.ld;
    int32_t* born_out = a.born_out ? a.born_out + sh * a.ld : nullptr;
    for (; c < cells.n; c += by) {
        if (mass_out != cells.mass) st_global<float>(mass_out + c, ld_global<float>(cells.mass + c));
        if (born_out) st_global<int32_t>(born_out + c, cells.number(c));
    }
}

// The choice for one kv head of one sequence by a workgroup, and where few rows can move (kFew) their moves.
template <class R, bool kFew>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(EvictArgs a) {
    __shared__ Shared shared;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.x, s = blockIdx.y;
    const uint64_t sh = uint64_t(s) * a.c.H + h;
    const EvictSeq seq = seq_of(a, s);
    const Cells cells = cells_of(a, seq, sh * a.ld);
    if (threadIdx.x == 0 && h == 0) {
        if constexpr (kFew) a.lens_out[s] = seq.kept;
        else a.seqs[s] = seq;   // lens_out may be what they came from
    }
    if (cells.n <= a.keep) {
        pass_on(a, cells, sh, threadIdx.x, kSelectThreads);
        if (!kFew && threadIdx.x == 0) a.moved[sh] = 0;
        return;
    }
    Keys keys;
    const bool held = cells.n <= kChunk;
    if (held) keys.load(cells, 0, cells.n);
    for (uint32_t i = threadIdx.x; i < kCopy * kCopies; i += kSelectThreads) shared.count[i] = 0;
    __syncthreads();
    uint32_t T = 0, need = a.keep, v[2];
    auto part = [&](auto p) {
        constexpr int kPart = decltype(p)::value;
        count_keys<kPart>(shared, keys, held, cells, 0, cells.n, T);
        __syncthreads();
        take_counts(shared, v);
        find(shared, v, kShift[kPart], wave, lane, T, need);
    };
    part(std::integral_constant<int, 0>{});
    part(std::integral_constant<int, 1>{});
    part(std::integral_constant<int, 2>{});
    list_moves<kFew>(shared, keys, held, a, cells, sh, 0, cells.n, T, need, 0, 0, wave, lane);
    if constexpr (kFew) {
        __syncthreads();
        const uint32_t moved = shared.moved;
        move_rows<R>(a, cells, s, h, moved, wave, kSelectWaves, lane, [&](uint32_t i) { return shared.count[i]; },
                     [&](uint32_t i) { return shared.count[kFewMoves + a.cap - moved + i]; });
    }
}

// The same by a.shares workgroups a head, a launch for each part of the key and one for the lists.  A launch begins with what the
// workgroups counted in the one before.
template <int kPart>
__global__ void __launch_bounds__(kSelectThreads) evict_share_kernel(EvictArgs a) {
    __shared__ Shared shared;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t share = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    const uint64_t sh = uint64_t(s) * a.c.H + h;
    const EvictSeq seq = kPart == 0 ? seq_of(a, s) : a.seqs[s];
    const Cells cells = cells_of(a, seq, sh * a.ld);
    const uint64_t each = (uint64_t(cells.n) + uint64_t(a.shares) * kSelectThreads - 1) / (uint64_t(a.shares) * kSelectThreads) * kSelectThreads;
    const uint32_t begin = uint32_t(share * each < cells.n ? share * each : cells.n), end = uint32_t((share + 1) * each < cells.n ? (share + 1) * each : cells.n);
    if (kPart == 0 && threadIdx.x == 0 && share == 0 && h == 0) a.seqs[s] = seq;
    if (cells.n <= a.keep) {
        if (kPart < kParts) return;
        pass_on(a, cells, sh, share * kSelectThreads + threadIdx.x, a.shares * kSelectThreads);
        if (threadIdx.x == 0 && share == 0) a.moved[sh] = 0;
        return;
    }
    Keys keys;
    const bool held = end - begin <= kChunk;
    if (held && begin < end) keys.load(cells, begin, end);
    EvictFound found{0, a.keep};   // the parts found so far, and how many of the keys that have them are kept
    uint32_t above = 0, equal = 0;
    uint32_t* own = a.counts + (sh * a.shares + share) * kParts * kValues;
    if constexpr (kPart > 0) {
        constexpr int kLast = kPart - 1;
        if constexpr (kLast > 0) found = a.found[sh * kParts + kLast - 1];
        // the counts of this thread's two values by all workgroups, by those before this one, and by this one
        const uint32_t* p = a.counts + sh * a.shares * kParts * kValues + kLast * kValues + value_of(1);
        uint32_t v[2] = {}, before[2] = {}, mine[2] = {};
#pragma unroll 8
        for (uint32_t q = 0; q < a.shares; ++q) {
            const ops_u32x2 c = ld_global<ops_u32x2>(p + uint64_t(q) * kParts * kValues);
            v[0] += c.y, v[1] += c.x;
            before[0] += q < share ? c.y : 0u, before[1] += q < share ? c.x : 0u;
            if (q == share) mine[0] = c.y, mine[1] = c.x;
        }
        find(shared, v, kShift[kLast], wave, lane, found.T, found.need);
        if (threadIdx.x == 0 && share == 0) a.found[sh * kParts + kLast] = found;
        // keys above T in this part: of the last part, those of the workgroups before this one; of the others this one's own, which
        // the last launch sums up
        const uint32_t value = found.T >> kShift[kLast] & (kLast == kParts - 1 ? (1u << kShift[kParts - 2]) - 1 : kValues - 1);
        uint32_t more = 0, same = 0;
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t c = kPart == kParts ? before[j] : mine[j];
            more += value_of(j) > value ? c : 0u;
            same += value_of(j) == value ? c : 0u;
        }
        if constexpr (kPart == kParts)   // and what they had above T in the parts before
            for (uint32_t q = threadIdx.x; q < share * (kParts - 1); q += kSelectThreads)
                more += ld_global<uint32_t>(a.above + sh * a.shares * (kParts - 1) + q);
        __syncthreads();
        above = sum_upto(shared, more, wave, lane);
        if (threadIdx.x == kSelectThreads - 1) shared.found[0] = above;
        if (value_of(0) == value || value_of(1) == value) shared.found[1] = same;
        __syncthreads();
        above = shared.found[0], equal = shared.found[1];
        if (kPart < kParts && threadIdx.x == 0) a.above[(sh * a.shares + share) * (kParts - 1) + kLast] = above;
        __syncthreads();
    }
    if constexpr (kPart < kParts) {
        for (uint32_t i = threadIdx.x; i < kCopy * kCopies; i += kSelectThreads) shared.count[i] = 0;
        __syncthreads();
        count_keys<kPart>(shared, keys, held, cells, begin, end, found.T);
        __syncthreads();
        uint32_t v[2];
        take_counts(shared, v);
        st_global<ops_u32x2>(own + kPart * kValues + value_of(1), ops_u32x2{v[1], v[0]});
    } else {
        list_moves<false>(shared, keys, held, a, cells, sh, begin, end, found.T, found.need, above, equal, wave, lane);
    }
}

template <class R>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(EvictArgs a) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, s = blockIdx.z;
    const EvictSeq seq = a.seqs[s];
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.lens_out[s] = seq.kept;
    const uint64_t sh = uint64_t(s) * a.c.H + h;
    const uint32_t moved = a.moved[sh];
    const uint32_t *dst = a.dst + sh * a.cap, *src = a.src + sh * a.cap + (a.cap - moved);
    move_rows<R>(a, cells_of(a, seq, sh * a.ld), s, h, moved, blockIdx.x * kMoveWaves + wave, gridDim.x * kMoveWaves, lane,
                 [&](uint32_t i) { return ld_global<uint32_t>(dst + i); }, [&](uint32_t i) { return ld_global<uint32_t>(src + i); });
}

// Whether the array that an eviction leaves may be written while another head's workgroup reads the ones that it was given.
bool apart(const EvictArgs& a) {
    auto clear = [&](const int64_t* p) { return !p || a.lens_out + a.n_seqs <= p || p + a.n_seqs <= a.lens_out; };
    return clear(a.lens) && clear(a.known) && clear(a.total);
}

template <class R>
hipError_t launch_of(const EvictArgs& a, hipStream_t stream) {
    const dim3 heads(a.c.H, a.n_seqs), block(kSelectThreads);
    if (a.shares == 1 && a.cap <= kFewMoves && apart(a)) {
        hipLaunchKernelGGL((evict_select_kernel<R, true>), heads, block, 0, stream, a);
        return hipGetLastError();
    }
    if (a.shares == 1) {
        hipLaunchKernelGGL((evict_select_kernel<Row<64, 1, true>, false>), heads, block, 0, stream, a);   // of any rows
    } else {
        const dim3 shares(a.shares, a.c.H, a.n_seqs);
        hipLaunchKernelGGL(evict_share_kernel<0>, shares, block, 0, stream, a);
        hipLaunchKernelGGL(evict_share_kernel<1>, shares, block, 0, stream, a);
        hipLaunchKernelGGL(evict_share_kernel<2>, shares, block, 0, stream, a);
        hipLaunchKernelGGL(evict_share_kernel<3>, shares, block, 0, stream, a);
    }
    constexpr uint32_t each = kMoveWaves * R::kPairs * kMoveAhead;
    const uint32_t blocks = a.cap / each + 1;
    hipLaunchKernelGGL(evict_move_kernel<R>, dim3(blocks < 4096 ? blocks : 4096, a.c.H, a.n_seqs), dim3(kMoveThreads), 0, stream, a);
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
    const uint64_t chunks = (uint64_t(a.max_len) + kChunk - 1) / kChunk, most = kShares / heads;
    a.shares = uint32_t(chunks < most ? chunks : most);
    if (a.cap == 0 || a.shares < kLeastShares) {
        a.shares = 1;
    } else {
        a.counts = reinterpret_cast<uint32_t*>(take(heads * a.shares * kParts * kValues * 4));
        a.above = reinterpret_cast<uint32_t*>(take(heads * a.shares * (kParts - 1) * 4));
        a.found = reinterpret_cast<EvictFound*>(take(heads * kParts * sizeof(EvictFound)));
    }
    return at;
}

hipError_t launch_evict(const EvictArgs& a, int head_dim, int format, hipStream_t stream) {
    const bool q8 = format == 1;
    if (head_dim == 64) return q8 ? launch_of<Row<64, 1, true>>(a, stream) : launch_of<Row<128, 1, false>>(a, stream);
    if (head_dim == 128) return q8 ? launch_of<Row<128, 2, true>>(a, stream) : launch_of<Row<256, 2, false>>(a, stream);
    if (head_dim == 256) return q8 ? launch_of<Row<256, 4, true>>(a, stream) : launch_of<Row<512, 4, false>>(a, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
