// sc_attn_split.hpp - how attention's cells are shared out among workgroups (sc_attn.hip): arithmetic that holds on a host
// as on the device, compiled into the plan, the kernels and, by the CPU tests, into a host program.
#pragma once

#include <cstdint>

namespace sc {

constexpr int kAttnWaves = 4;
constexpr int kTurn = 32;                       // cells of a wave's turn
constexpr uint32_t kUnit = kTurn * kAttnWaves;  // cells of a workgroup's turn
// Workgroups that the units are shared out among, one to each of the chip's 256 units, whose next turn's rows are in flight
// while this one's are worked on.  Two to each have more in flight, but give twice the parts to write and to join; between
// the two some run alone at the end.  Eight sequences of 1 K to 128 K cells: 236 us with 256, 270 with 384, 239 with 512; one
// of 128 K 52, 62, 54; 32 of up to 8 K in int8 39, 43, 40.
constexpr uint32_t kAttnSlots = 256;

// Cells [first, len) of a sequence, counted in units from `begin`, a multiple of a turn.
struct Span {
    uint32_t first, len, begin, units;
};
constexpr Span cells_of(int64_t n, uint32_t max_len, uint32_t window) {
    const uint32_t len = n < 0 ? 0u : n > int64_t(max_len) ? max_len : uint32_t(n);
    const uint32_t first = window && len > window ? len - window : 0u, begin = first & ~uint32_t(kTurn - 1);
    return {first, len, begin, (len - begin + kUnit - 1) / kUnit};
}

// Units of a part at most, where all sequences have `total` and each is taken by `tiles` workgroups a part.  No sequence has
// more than 2^24 units; the share of one of the slots can be beyond that, and beyond 32 bits, in a batch of many (pages can
// be shared, so lengths are not bounded by memory).
constexpr uint32_t kMostUnits = 1u << 24;
constexpr uint32_t units_of_part(uint64_t total, uint32_t tiles, uint32_t slots, uint32_t least) {
    const uint64_t share = (total * tiles + slots - 1) / slots;
    return share < least ? least : share > kMostUnits ? kMostUnits : uint32_t(share);
}
constexpr uint32_t parts_of_units(uint32_t units, uint32_t per) { return units <= per ? 1u : (units + per - 1) / per; }
// A few workgroups more than run at once would run alone at the end; where this holds, twice the share is always enough for
// no more than the slots.
constexpr bool parts_fit(uint32_t n_seqs, uint32_t tiles, uint32_t slots) { return n_seqs <= 64 && n_seqs * tiles * 2 <= slots; }
constexpr uint32_t wider_part(uint32_t per) { return per + per / 32 + 1; }

// What the host plans from the bounds alone.
struct SplitPlan {
    uint64_t grid, places;    // workgroups of the launch; results of parts that the workspace has room for
    uint32_t parts;           // parts a sequence can have
    uint32_t direct;          // units a sequence can have, where each is a workgroup of its own; else 0
    bool join;                // whether a sequence can have more than one part
};
constexpr SplitPlan plan_split(uint32_t n_seqs, uint32_t tiles, uint32_t max_len, uint32_t window, uint32_t slots) {
    const uint64_t rows = uint64_t(n_seqs) * tiles;
    // a window may begin anywhere in a turn, so it can touch a unit more
    const uint64_t most = ((window ? uint64_t(window) + kTurn : uint64_t(max_len)) + kUnit - 1) / kUnit;
    SplitPlan p{};
    p.join = most > 1;
    // With a workgroup for every unit that there can be, none has to find its place: 12.5 us for 1 K cells, 13.4 without.
    p.direct = p.join && !window && rows * most <= slots ? uint32_t(most) : 0;
    p.parts = uint32_t(most < slots ? most : slots + 1);
    // parts of all sequences: at most a slot's share each, and one more a sequence
    const uint64_t shares = slots < rows * most ? slots : rows * most;
    p.grid = p.direct ? rows * most : rows + (p.join ? shares : 0);
    p.places = p.join ? 2 * shares : 0;
    return p;
}

}  // namespace sc
