// How attention with shared starts of prompts is cut into work (sp_shared_prefix.hip): arithmetic that its launches share with each other and
// that a plain C++ compiler takes as well.
//
// Rows are (token, query head of the kv group) pairs, the heads of a token side by side, 64 of them a tile.  Items are the groups, over their
// shared keys, and behind them the requests, over their own.  An item has as many units as its tiles have steps of 32 keys, and SH_OVERHEAD beside them a
// tile, for its queries, its first loads and the waves' meeting; the items lie on a line that is cut into equal parts, one workgroup of a kv head each.
// Single tokens whose heads fit 16 rows are no matter of the workgroup's but of its waves: four of them have a quarter each of what of the requests falls to
// it, go through it step by step and count one unit beside an item's steps (SH_STREAM_OVERHEAD).
#pragma once
#include "sp_paged_plan.h"

#define SH_TILE 64
#define SH_KEYS 32       // of a step
#define SH_MAX_SEQS 1024
#define SH_OVERHEAD 6
#define SH_STREAM_OVERHEAD 1
#define SH_MIN_SHARE 8   // units of a part at least
#define SH_WAVES 4       // that share a workgroup's keys

// Where a cut `off` units into an item stands whose tiles have n steps each: in front of a step of a tile (the n-th: behind the tile).
PG_FN void sh_place(int64_t off, int n, int near, int* tile, int* step) {
  const int64_t each = n + SH_OVERHEAD, at = off < PG_SHORT_LINE ? (int64_t)((unsigned)off / (unsigned)each) : off / each;
  *tile = (int)at;
  *step = pg_snap(off - at * each, n, SH_OVERHEAD, near);
}
// The same of a request's steps among those of a wave.
PG_FN int sh_stream_step(int64_t off, int n) { return pg_snap(off, n, SH_STREAM_OVERHEAD, 1); }
PG_FN int64_t sh_units(int n, int rows, int streams) {
  return n <= 0 ? 0 : streams ? n + SH_STREAM_OVERHEAD : (int64_t)(n + SH_OVERHEAD) * ((rows + SH_TILE - 1) / SH_TILE);
}
// A request whose first new token stands behind its group's shared keys takes part in the group; any other sees to all of its keys by itself.
PG_FN int sh_first_own(int len, int q_len, int shared) { return len - q_len >= shared ? shared : 0; }
// Numbers of row tiles: every sequence has room for its last, partly filled one (pg_first_slot); single tokens whose heads fit a tile have one each.
PG_FN int64_t sh_own_slot(int64_t start, int g, int b, int dense) { return dense ? b : pg_first_slot(start, g, b, SH_TILE); }
// Groups of many rows are left to the kernel that has matrix products' rate (sp_chunk.hip, tiles of 256 rows) and a launch of its own.
PG_FN bool sh_apart(int64_t tokens, int64_t groups, int64_t g) { return groups > 0 && tokens * g > 128 * groups; }
