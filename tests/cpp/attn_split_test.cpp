// How attention's cells are shared out (csrc/sc_attn_split.hpp, the header the kernels are compiled from): whatever the
// lengths, every workgroup that has cells is in the launch and every part's result has a place in the workspace.
// `attn_split_test <name>` runs one test; it prints the first difference and returns 1, or returns 0.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "sc_attn_split.hpp"

namespace {

// The places that the kernels take, by a plain loop over the sequences; 1 and a line where one is not there.
int fits(const std::vector<int64_t>& lens, uint32_t tiles, uint32_t max_len, uint32_t window) {
    const uint32_t n = uint32_t(lens.size()), slots = sc::kAttnSlots;
    const sc::SplitPlan p = sc::plan_split(n, tiles, max_len, window, slots);
    uint64_t total = 0, wgs = 0, places = 0;
    std::vector<uint32_t> units;
    for (int64_t len : lens) units.push_back(sc::cells_of(len, max_len, window).units), total += units.back();
    auto count = [&](uint32_t per) {
        uint64_t all = 0;
        for (uint32_t u : units) all += sc::parts_of_units(u, per);
        return all * tiles;
    };
    uint32_t per = sc::units_of_part(total, tiles, slots, 1);
    if (p.direct) per = 1;
    else if (sc::parts_fit(n, tiles, slots))
        while (count(per) > slots) per = sc::wider_part(per);
    uint64_t most = 0, covered = 0;
    for (uint32_t u : units) {
        const uint64_t parts = sc::parts_of_units(u, per), each = (u + parts - 1) / parts;
        most = std::max(most, parts);
        covered += std::min(parts * each, uint64_t(u));
        if (parts > 1) places += parts * tiles;
    }
    wgs = count(per);
    if (p.direct) places = uint64_t(n) * p.direct * tiles;   // places are kept for units that a sequence does not have
    const char* what = wgs > p.grid ? "workgroups past the launch" : places > p.places ? "places past the workspace"
                       : p.join && most > p.parts ? "parts past the plan's" : most > 1 && !p.join ? "parts without a join"
                       : covered != total ? "units left out" : nullptr;
    if (!what) return 0;
    std::printf("%s: %u sequences, %u tiles, max_len %u, window %u: %llu of %llu workgroups, %llu of %llu places, %llu of %u parts\n", what,
                n, tiles, max_len, window, (unsigned long long)wgs, (unsigned long long)p.grid, (unsigned long long)places,
                (unsigned long long)p.places, (unsigned long long)most, p.parts);
    return 1;
}

constexpr uint32_t kTiles[] = {1, 2, 4, 7, 64, 255, 256, 257, 480, 512};

// The longest sequences that a request may have, as many as it may have.
int longest() {
    for (uint32_t n : {1u, 2u, 63u, 64u, 65u, 300u, 1024u})
        for (uint32_t tiles : kTiles)
            for (uint32_t window : {0u, 1u << 30}) {
                std::vector<int64_t> lens(n, INT64_MAX);
                if (fits(lens, tiles, 0x7FFFFFFFu, window)) return 1;
                for (uint32_t i = 0; i < n; i += 3) lens[i] = i % 2 ? -1 : 1000 + i;
                if (fits(lens, tiles, 0x7FFFFFFFu, window)) return 1;
            }
    return 0;
}

int ragged() {
    std::mt19937_64 rng(1);
    for (int t = 0; t < 20000; ++t) {
        const uint32_t n = 1 + uint32_t(rng() % (t % 3 ? 70 : 1024)), tiles = kTiles[rng() % 10];
        const uint32_t max_len = uint32_t(rng() % (uint64_t(1) << (1 + rng() % 31))), window = rng() % 2 ? uint32_t(rng() % (max_len + 1ull)) : 0;
        std::vector<int64_t> lens(n);
        for (int64_t& len : lens) len = int64_t(rng() % (uint64_t(1) << (1 + rng() % 33))) - 3;
        if (fits(lens, tiles, max_len, window >= max_len ? 0 : window)) return 1;
    }
    return 0;
}

}  // namespace

int main(int argc, char** argv) {
    const struct { const char* name; int (*run)(); } tests[] = {{"longest", longest}, {"ragged", ragged}};
    for (const auto& t : tests)
        if (argc == 2 && !std::strcmp(argv[1], t.name)) return t.run();
    std::printf("usage: attn_split_test <test>\n");
    return 2;
}
