// How attention with shared starts of prompts is cut into work (sp_shared_prefix.hip): arithmetic that its launches share with each other and
// that a plain C++ compiler takes as well.
//
// Rows are (token, query head of the kv group) pairs, the heads of a token side by side, 64 or 128 of them a tile.  Items are the groups, over their
// shared keys, and behind them the requests, over their own.  An item has as many units as its tiles have steps of 32 keys, and SH_OVERHEAD (SH_OWN_OVERHEAD) beside them a
// tile, for its queries, its first loads and the waves' meeting; the items lie on a line that is cut into equal parts, one workgroup of a kv head each.
// Single tokens whose heads fit 16 rows are no matter of the workgroup's but of its waves: four of them have a quarter each of what of the requests falls to
// it, go through it step by step and count one unit beside an item's steps (SH_STREAM_OVERHEAD).
#pragma once
#include "sp_paged_plan.h"

#define SH_UNIT 64       // rows that tiles are numbered by
#define SH_ROWS 128      // of a tile at most
#define SH_KEYS 32       // of a step
#define SH_MAX_SEQS 1024
enum { SH_GROUP, SH_OWN, SH_STREAM };  // items: a group's shared keys, a request's own, the same as a matter of waves
// Units of a tile beside its steps.  (us, 32 heads over 8, 6 / 10 / 14 / 20 of a request's: nine tokens each of 20 requests behind 2000 shared keys 65 / 51 / 51 / 49, two of 37
// over 1336 own ones 49 / 50 / 50 / 50, of 14 heads over 2 22 / 22 / 22 / 24; 6 / 7 / 8 of a group's: eight tokens each of 8 requests behind 1024 keys 30 / 33 / 33.)
#define SH_OVERHEAD 6
#define SH_OWN_OVERHEAD 10
#define SH_STREAM_OVERHEAD 1
#define SH_MIN_SHARE 8   // units of a part at least
#define SH_WAVES 4       // that share a workgroup's keys

// Rows of a tile where there are `rows` of them: with more than 64 keys are read half as often for a step's work twice as long or more, which its steps count.
// (us, 2 / 3 / 4 units: 64 single tokens of 32 heads over 8 behind 8192 keys 95 / 86 / 95, four groups of 16 of 28 over 4 behind 4000 42 / 42 / 40.)
PG_FN int sh_tile(int rows) { return rows <= SH_UNIT ? SH_UNIT : SH_ROWS; }
PG_FN int sh_step_units(int rows) { return rows <= SH_UNIT ? 1 : 3; }
// Where a cut `off` units into an item stands whose tiles have n steps each: in front of a step of a tile (the n-th: behind the tile).
PG_FN int sh_overhead(int kind) { return kind == SH_GROUP ? SH_OVERHEAD : kind == SH_OWN ? SH_OWN_OVERHEAD : SH_STREAM_OVERHEAD; }
PG_FN void sh_place(int64_t off, int n, int rows, int kind, int near, int* tile, int* step) {
  const int of_step = sh_step_units(rows), overhead = sh_overhead(kind);
  const int64_t each = (int64_t)n * of_step + overhead, at = off < PG_SHORT_LINE ? (int64_t)((unsigned)off / (unsigned)each) : off / each;
  const int64_t in = off - at * each;
  *tile = (int)at;
  *step = pg_snap(in < overhead ? 0 : overhead + (in - overhead) / of_step, n, overhead, near);
}
// The same of a request's steps among those of a wave.
PG_FN int sh_stream_step(int64_t off, int n) { return pg_snap(off, n, SH_STREAM_OVERHEAD, 1); }
PG_FN int64_t sh_units(int n, int rows, int kind) {
  return n <= 0 ? 0 : kind == SH_STREAM ? n + SH_STREAM_OVERHEAD : ((int64_t)n * sh_step_units(rows) + sh_overhead(kind)) * ((rows + sh_tile(rows) - 1) / sh_tile(rows));
}
// A request whose first new token stands behind its group's shared keys takes part in the group; any other sees to all of its keys by itself.
PG_FN int sh_first_own(int len, int q_len, int shared) { return len - q_len >= shared ? shared : 0; }
// Numbers of row tiles, by 64 rows (a larger one has that of its first): every sequence has room for its last, partly filled one (pg_first_slot); single tokens whose heads fit a tile have one each.
PG_FN int64_t sh_own_slot(int64_t start, int g, int b, int dense) { return dense ? b : pg_first_slot(start, g, b, SH_UNIT); }
// Groups of many rows are left to the kernel that has matrix products' rate (sp_chunk.hip, tiles of 256 rows) where the table has room for enough keys to pay
// for two launches more, but not where keys are weighed: its sums are those of probabilities rounded to two bf16 values.  By rows x keys of all kv heads, in millions, us
// within one launch / apart: 32 heads over 8 of 128 channels 6 37 / 58, 26 68 / 75, 34 78 / 79, 49 100 / 91, 66 128 / 103, 132 202 / 131, 526 714 / 379; 28 over 4 9
// 39 / 52, 36 87 / 77, 57 121 / 97; of 64 channels 26 56 / 58, 49 85 / 72, 58 99 / 77, 66 107 / 81, 132 169 / 96.  At 256 rows and fewer tiles of 256 are not full.
PG_FN bool sh_may_be_apart(int64_t tokens, int64_t groups, int64_t g, bool weighed) { return !weighed && groups > 0 && tokens * g > 256 * groups; }
PG_FN bool sh_apart(int64_t tokens, int64_t groups, int64_t hq, int64_t hkv, int64_t room, bool weighed) {
  return sh_may_be_apart(tokens, groups, hq / hkv, weighed) && (double)(tokens * hq) * (double)room > 3e7;
}
