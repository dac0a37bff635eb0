// How attention over a paged cache deals a request's positions to workgroups,
// for host and device alike.
#pragma once

#include <stdint.h>

constexpr uint32_t STEP = 64;         // positions of a value product
constexpr uint32_t MAX_CHUNK = 1024;  // positions of a workgroup
constexpr uint32_t CHUNK_PAGES = MAX_CHUNK / 4 + 1;

// Positions of a chunk (whole steps) where (request, key head) pairs `pairs`
// look at up to `span` positions each. About 1024 workgroups, of at most 1024
// positions: each begins with some microseconds of dependent loads, and its
// sums are written and read again. us, at most 512 / 1024 / 2048 positions: 4
// tokens at up to 32700 145 / 127 / 127, 32 trees of 25 at up to 8000 563 / 520
// / 582, 16 tokens at up to 20000 280 / 290 / 357, 64 at up to 2000 122 / 128 /
// 129.
constexpr uint32_t chunk_positions(uint64_t span, uint64_t pairs) {
    const uint64_t want = 1024 / pairs > 1 ? 1024 / pairs : 1;
    const uint64_t each = ((span + want - 1) / want + STEP - 1) / STEP * STEP;
    return (uint32_t)(each < STEP ? STEP : each > MAX_CHUNK ? MAX_CHUNK : each);
}

// The most pages of 2^log positions that `count` positions in a row meet: the
// first and the last may lie anywhere in theirs.
constexpr uint32_t most_pages(uint32_t count, uint32_t log) { return ((count - 1) >> log) + 2; }
