// Which expert's rows a workgroup multiplies: rows sorted by expert, expert e's from
// offsets[e] to offsets[e + 1], are cut into tiles of bm rows that never span two experts.
// How many there are only the device knows; a grid is launched for the most there can be
// and its workgroups past the last tile end at once.
#pragma once

#include <algorithm>

#include "common.h"

namespace mj {

struct ExpertTile {
  int expert, row0, rows;  // of the whole expert; expert == experts: the rows behind the last
  int m, n;                // tile
};

// An entry of the sort's results, kept inside the rows: a plan that is none (a caller's own
// or overwritten) gives meaningless results, but no access outside the arrays.
__device__ __forceinline__ int within(int at, int rows) { return std::min(std::max(at, 0), rows); }

// An inclusive sum over a wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
#define MJ_SCAN(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false)
  MJ_SCAN(0x111, 0xF);  // row_shr:1, 2, 4, 8
  MJ_SCAN(0x112, 0xF);
  MJ_SCAN(0x114, 0xF);
  MJ_SCAN(0x118, 0xF);
  MJ_SCAN(0x142, 0xA);  // row_bcast:15 into rows 1 and 3
  MJ_SCAN(0x143, 0xC);  // row_bcast:31 into rows 2 and 3
#undef MJ_SCAN
  return v;
}

// Which of the tiles a launch takes.  Large tiles leave most CUs idle in a last round of a few,
// and how many there are the host cannot know: with at most half a round over (CUT_REST_MOST)
// one launch takes the whole rounds and a second one those tiles in quarters (twice as many
// rows and columns of tiles of half the sides); with more, the first takes all and the
// second ends at once.
enum : int { CUT_NONE = 0, CUT_ROUNDS, CUT_REST };
constexpr int kTileRound = 256, CUT_REST_MOST = kTileRound / 2;

// The tile of workgroup bid.  tail: the rows from offsets[experts] to `rows` are a group
// too.  Each wave scans the experts' tile counts, 64 experts at a time.  XCD: neighbouring
// tiles of one expert go to one XCD (they share its operand panels in its L2), 4 tile rows
// at a time; without, tiles go column by column in launch order.  CUT_REST: bm and tiles_n are
// the large tiles', t.m and t.n the quarter's.
template <bool XCD>
__device__ __forceinline__ bool expert_tile(const int *offsets, int experts, int rows, bool tail, int bm,
                                            int tiles_n, int bid, ExpertTile &t, int cut = CUT_NONE) {
  const int lane = threadIdx.x & 63, groups = experts + (tail ? 1 : 0);
  auto counts = [&](int g0, int &start, int &n) __attribute__((always_inline)) {
    const int g = g0 + lane;
    start = g < groups ? within(offsets[g], rows) : 0;
    n = g < groups ? std::max((g < experts ? within(offsets[g + 1], rows) : rows) - start, 0) : 0;
    return (n + bm - 1) / bm;
  };
  int start, n, total_m = 0;
  for (int g0 = 0; g0 < groups; g0 += 64)
    total_m += __builtin_amdgcn_readlane(wave_scan(counts(g0, start, n)), 63);
  int total = total_m * tiles_n, first_tile = 0;
  if (cut != CUT_NONE) {
    const int rest = total % kTileRound;
    const bool split = rest <= CUT_REST_MOST;
    if (cut == CUT_ROUNDS && split) total -= rest;
    if (cut == CUT_REST) first_tile = total - rest, total = split ? 4 * rest : 0;
  }
  if (bid >= total) return false;
  int logical = bid;
  if constexpr (XCD) {
    const int x = bid & 7, q = total >> 3, r = total & 7;
    logical = x * q + (x < r ? x : r) + (bid >> 3);
  }
  const int quarter = logical & 3;
  if (cut == CUT_REST) logical = first_tile + (logical >> 2);
  const int lm = logical / tiles_n;
  for (int g0 = 0, before = 0; g0 < groups; g0 += 64) {
    const int c = counts(g0, start, n), sum = wave_scan(c) + before;
    const uint64_t past = __ballot(sum > lm);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int tiles_m = __builtin_amdgcn_readlane(c, at);
      const int first = __builtin_amdgcn_readlane(sum, at) - tiles_m;
      t.expert = g0 + at;
      t.row0 = __builtin_amdgcn_readlane(start, at);
      t.rows = __builtin_amdgcn_readlane(n, at);
      logical -= first * tiles_n;
      if constexpr (XCD) {
        group_coords(logical, tiles_m, tiles_n, 4, t.m, t.n);
      } else {
        t.m = logical / tiles_n;
        t.n = logical - t.m * tiles_n;
      }
      if ((uint32_t)t.m >= (uint32_t)tiles_m || (uint32_t)t.n >= (uint32_t)tiles_n) return false;
      if (cut == CUT_REST) t.m = 2 * t.m + (quarter >> 1), t.n = 2 * t.n + (quarter & 1);
      return true;
    }
    before = __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// The most tiles of bm rows that `rows` rows of `groups` groups can make.
inline int64_t expert_tiles_most(int64_t rows, int64_t groups, int64_t bm) {
  const int64_t full = rows < groups ? rows : groups;  // groups that can have a part of a tile
  return (rows + full * (bm - 1)) / bm;
}

}  // namespace mj
