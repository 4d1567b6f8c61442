// The grid of a launch of more workgroups than one dimension holds.
#pragma once
#include <stdint.h>

namespace catcoc {

// Workgroups of a row of a launch's second dimension: with 1024 threads each, the most there are, 2^30 threads.
constexpr uint32_t kGridRowLog = 20, kGridRow = 1u << kGridRowLog;

struct LaunchGrid {
    uint32_t x, y;
};

// For fewer than 2^36 workgroups (2^16 rows).
constexpr LaunchGrid launch_grid(uint64_t wgs, uint32_t threads)
{
    if (wgs * threads < (1ull << 32)) return {(uint32_t)wgs, 1u};
    return {kGridRow, (uint32_t)((wgs + kGridRow - 1u) >> kGridRowLog)};
}

}  // namespace catcoc
