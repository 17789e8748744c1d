// lookup_grid.h - launch shapes of the lookup channel (host only, no device code).
#pragma once
#include <stddef.h>

// workgroups along the first axis of a grid: fewer than 2^32 work-items there, 256 in each workgroup
constexpr size_t kLkMaxGrid = ((size_t)1 << 24) - 1;

// Instances by XCD (lk_place): for what is read out of order in elements or rows, while it stays in an L2 of 4 MiB - the table of
// an instance for a lookup or a message by position (up to twice that: 8 x 20000 x 64 f32 18.2 -> 14.3 us; 64 x 200000 f64 82 ->
// 53 us), its positions for the sums (64 x 100000 f64, gradient 102 -> 92 us; 8 x 17 MB would be 169 -> 178 us) - and while the
// last round of eight leaves few XCDs idle and the first axis holds all instances.
static inline int lk_spread(size_t batch, size_t blocks, size_t bytes, size_t most) {
    return batch > 1 && bytes <= most && (batch + 7) / 8 * 8 * 7 <= batch * 8 && (batch + 7) / 8 * 8 * blocks <= kLkMaxGrid;
}
