// attn_lines.h — the lines by distance (key place - query place) that the attention kernels keep in LDS: their lengths and the
// indexes into them.  Plain C++, for the kernels, the launches and a check of all indexes on the host.
//
// Tiles are 32 x 32 and begin at multiples of 32, so a tile's e0 = first key - first query is a multiple of 32 too.  R, the reach, is
// the first distance of the last bucket: a tile wholly at R or beyond is far and touches no line.
#pragma once

namespace vdbk {

constexpr int kMargin = 64;     // what the tiles that are not far meet beyond R

constexpr bool tile_is_far(int e0, int reach) { return e0 - 31 >= reach || e0 + 31 <= -reach; }

// start values of a tile's sums: distance e at start_zero + e, |e| <= R + margin
constexpr int start_zero(int reach) { return reach + kMargin; }
constexpr int start_span(int reach) { return 2 * (reach + kMargin) + 1; }
constexpr int start_at(int reach, int e) { return start_zero(reach) + e; }

// sums of ds by distance: distance e at sums_zero + e.  Each lane l of a wave's half adds to two places: sums_at, and 32 behind it (a zero
// where that is no distance of the tile).  e0 reaches R + 30, half 4 and 32 more: R + 66, three behind the margin.
constexpr int sums_zero(int reach) { return reach + kMargin; }
constexpr int sums_span(int reach) { return 2 * (reach + kMargin) + 3; }
constexpr int sums_at(int reach, int e0, int half, int l) { return sums_zero(reach) + e0 + 4 * half - l; }

}  // namespace vdbk
