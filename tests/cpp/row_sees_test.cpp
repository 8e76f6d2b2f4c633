// Which cells a sequence's latest queries see (csrc/sc_attn_split.hpp, the header the kernels are compiled from), against the same in
// 64 bits: around every border that a length, a window and a lane's first cell can have, up to the longest of them.
// Prints the first difference and returns 1, or returns 0.
#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "sc_attn_split.hpp"

namespace {

constexpr uint32_t kLongest = 0x7FFFFFFF, kRows = 1024;

// What passes 32 bits is no constant: the farthest that a cell can lie on either side of a row's last one.
static_assert(!sc::row_sees(sc::row_ends(kLongest, kRows, 0, kLongest - 1 + sc::kUnit), kLongest - 1, 19));
static_assert(!sc::row_sees(sc::row_ends(1, kRows, 0, sc::kUnit), kLongest - 1, 19));
static_assert(!sc::row_sees(sc::row_ends(kLongest, 1, 0, 0), 1, 0) && sc::row_sees(sc::row_ends(kLongest, 1, 0, 0), 0, 0));
static_assert(sc::row_sees(sc::row_ends(kLongest, kRows, kRows - 1, 0), kLongest, 0));

int check(uint32_t n, uint32_t rows, uint32_t r, uint32_t window, uint32_t from) {
    const int32_t ends = sc::row_ends(n, rows, r, from);
    for (int32_t cell = 0; cell < 20; ++cell) {
        const int64_t at = int64_t(from) + cell, end = int64_t(n) - rows + 1 + r;
        const bool sees = at < end && (!window || at >= end - window);
        if (sc::row_sees(ends, window, cell) == sees) continue;
        std::printf("n %u rows %u row %u window %u from %u cell %d: %d\n", n, rows, r, window, from, cell, int(!sees));
        return 1;
    }
    return 0;
}

}  // namespace

int main() {
    for (uint32_t n : {1u, 2u, 31u, 33u, 1023u, 1024u, 1025u, 100000u, kLongest - 33, kLongest - 1, kLongest})
        for (uint32_t rows : {1u, 2u, 100u, kRows})
            for (uint32_t r : {0u, 1u, rows / 2, rows - 1})
                for (uint32_t window : {0u, 1u, 2u, 40u, 1000u, n / 2, n - 1, n, kLongest - 1, kLongest}) {
                    if (r >= rows) continue;
                    const int64_t end = int64_t(n) - rows + 1 + r, last = int64_t(n) - 1 + sc::kUnit;
                    for (int64_t border : {int64_t(0), end, end - int64_t(window), last})
                        for (int64_t d = -24; d <= 24; ++d)
                            if (check(n, rows, r, window, uint32_t(std::clamp(border + d, int64_t(0), last)))) return 1;
                }
    return 0;
}
