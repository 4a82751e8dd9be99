// How attention with shared starts of prompts is cut into work (sp_shared_prefix.hip): arithmetic that its launches share with each other and
// that a plain C++ compiler takes as well.
//
// Items are row tiles of SH_TILE rows, (token, query head of the kv group) pairs with the heads of a token side by side: first those of the groups over
// their shared keys, then those of the requests over their own.  An item's steps of 32 keys and SH_OVERHEAD units beside them, for its queries,
// its first loads and the waves' meeting, lie on a line that is cut into equal parts, one workgroup of a kv head each.
#pragma once
#include "sp_paged_plan.h"

#define SH_TILE 64       // rows of an item
#define SH_KEYS 32       // keys of a step
#define SH_MAX_SEQS 1024
#define SH_OVERHEAD 6
#define SH_MIN_SHARE 6   // units of a part at least

// the steps of an item of n steps at unit `start` of the line that fall to the part between two cuts
PG_FN void sh_steps(int64_t start, int n, int64_t cut0, int64_t cut1, int near, int* begin, int* end) {
  *begin = cut0 <= start ? 0 : pg_snap(cut0 - start, n, SH_OVERHEAD, near);
  *end = cut1 >= start + n + SH_OVERHEAD ? n : cut1 <= start ? 0 : pg_snap(cut1 - start, n, SH_OVERHEAD, near);
}
// the part that unit x of the line lies in
PG_FN int64_t sh_part(int64_t x, int64_t total, int64_t parts) {
  int64_t p = total < PG_SHORT_LINE ? (int64_t)((uint64_t)(unsigned)x * (unsigned)parts / (unsigned)total) : (int64_t)((double)x / (double)total * (double)parts);
  if (p >= parts) p = parts - 1;
  while (p > 0 && pg_cut(total, parts, p) > x) --p;
  while (p + 1 < parts && pg_cut(total, parts, p + 1) <= x) ++p;
  return p;
}
// A request whose first new token stands behind its group's shared keys takes part in the group; any other sees to all of its keys by itself.
PG_FN int sh_first_own(int len, int q_len, int shared) { return len - q_len >= shared ? shared : 0; }
// Row tiles are numbered as pg_first_slot says; single tokens whose heads fit a tile have one each.
PG_FN int64_t sh_own_slot(int64_t start, int g, int b, int dense) { return dense ? b : pg_first_slot(start, g, b, SH_TILE); }
