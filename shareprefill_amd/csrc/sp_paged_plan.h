// How attention over pages and windows is cut into work (sp_chunk.hip, sp_paged_decode.hip): arithmetic on positions and lengths that the
// kernels and the host share and a plain C++ compiler takes as well.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define PG_FN __host__ __device__ static inline
#else
#define PG_FN static inline
#endif

#define PG_MAX_SEQS 4096           // sequences of a call
#define PG_MAX_KEYS (1 << 30)      // keys of a sequence: positions and their differences have 31 bits
#define PG_NO_WINDOW PG_MAX_KEYS   // every key in front of a query lies inside it

// (A row tile has `tile` rows: (token, query head of the kv group) pairs, the heads of a token side by side.)

PG_FN int pg_min(int a, int b) { return a < b ? a : b; }
PG_FN int pg_max(int a, int b) { return a > b ? a : b; }

// Lengths as the device finds them, and sums of them that hold at 2^30 instead of growing past it: 32 bits wide, sorted, and the same whatever the
// order of adding.  (Two sums at 2^30 make 2^31, which only unsigned numbers hold.)
PG_FN int pg_length(int n) { return pg_max(0, pg_min(n, PG_MAX_KEYS - 1)); }
PG_FN int pg_held_sum(int x, int y) {
  const unsigned sum = (unsigned)x + (unsigned)y;
  return sum < (unsigned)PG_MAX_KEYS ? (int)sum : PG_MAX_KEYS;
}
PG_FN int pg_holder(const int* sums, int n, int x) {  // the last of n entries that starts at or in front of x: sums[i] <= x < sums[i + 1]
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// A stride as the kernels take it: that of an axis of length one says nothing, and may be anything.
PG_FN int64_t pg_used_stride(int64_t stride, int64_t length) { return length == 1 ? 0 : stride; }

// The query at position p sees key j: causal, inside its window or among the first `sinks`.
PG_FN bool pg_sees(int p, int j, int window, int sinks) { return j <= p && (j > p - window || j < sinks); }

// Units of `unit` keys that queries at positions p0 .. p1 see something of, as two runs: [0, front) holds sinks, [lo, hi) the windows.
struct PgSpan {
  int front, lo, hi;
};
PG_FN int pg_span_units(const PgSpan& s) { return s.front + s.hi - s.lo; }
PG_FN int pg_span_unit(const PgSpan& s, int i) { return i < s.front ? i : s.lo + (i - s.front); }
PG_FN PgSpan pg_span(int p0, int p1, int window, int sinks, int unit) {
  PgSpan s = {0, 0, 0};
  if (p1 < 0) return s;
  s.hi = p1 / unit + 1;
  const int first = p0 - window + 1;  // of the windows
  s.lo = first > 0 ? first / unit : 0;
  const int k = pg_min(sinks, p1 + 1);
  s.front = pg_min((k + unit - 1) / unit, s.lo);
  return s;
}

// Row tiles are numbered so that a workgroup finds its own without a scan: those of sequence b, whose tokens start at `start`, begin at
// floor(start * g / tile) + b.  Every sequence has room for its last, partly filled tile; numbers left over stand for nothing.
PG_FN int64_t pg_first_slot(int64_t start, int g, int b, int tile) { return start * g / tile + b; }
PG_FN int64_t pg_slots(int64_t tokens, int g, int batch, int tile) { return tokens * g / tile + batch; }
PG_FN int64_t pg_row_tiles(int64_t q_len, int g, int tile) { return (q_len * g + tile - 1) / tile; }

// Quotients by a launch's one divisor: the division takes a wave some 35 instructions, and a row tile needs a dozen.  With 2^l the power of two
// at or above the divisor, x * ceil(2^(31 + l) / by) / 2^(31 + l) has the quotient for x below 2^31: the multiplier is too large by less than
// one part in 2^31.
struct PgDivisor {
  unsigned by, mul, shift;
};
PG_FN PgDivisor pg_divisor(unsigned by) {  // 1 <= by < 2^31
  PgDivisor d = {by, 0u, 0u};
  while ((1u << d.shift) < by) ++d.shift;
  d.mul = (unsigned)((((uint64_t)1 << (31 + d.shift)) + by - 1) / by);
  return d;
}
PG_FN unsigned pg_div(unsigned x, const PgDivisor& d) { return (unsigned)((uint64_t)(x << 1) * d.mul >> 32) >> d.shift; }

// Positions of a row tile's first and last row: row r of a sequence, fewer than 2^31 of them, is token r / g.
PG_FN void pg_tile_positions(int rt, int q_len, int len, const PgDivisor& g, int tile, int* p0, int* p1) {
  const unsigned rows = (unsigned)q_len * g.by, r0 = (unsigned)rt * (unsigned)tile, r1 = rows - r0 < (unsigned)tile ? rows : r0 + (unsigned)tile;
  *p0 = len - q_len + (int)pg_div(r0, g);
  *p1 = len - q_len + (int)pg_div(r1 - 1u, g);
}

// A launch cuts the line of all its row tiles' blocks, one line per kv head, into equal parts: part p of `parts` starts at unit
// total * p / parts.  A row tile counts its blocks and PG_OVERHEAD units for its queries, its first loads and its output; a cut near a row
// tile's start or end goes there (pg_near).
// (us, 1 / 2 / 3 / 4 units: 512 tokens over 8192 keys 88.6 / 88.3 / 86.5 / 86.7, 16 chunks of 200 over 1000 78.1 / 75.2 / 73.5 / 73.2, one of 900
// beside three tokens over 4000 80.6 / 83.0 / 85.6 / 88.8, a mixed batch of 64 channels 133.1 / 132.7 / 132.6 / 135.3.)
#define PG_OVERHEAD 3
#define PG_MIN_SHARE 3  // units of a part at least
// The same of single tokens, whose line is made of sequences and their steps of 32 keys: queries, first loads, the waves' meeting.  (us, 8 and 8 /
// 4 and 4: one token over 1025 keys 11.5 / 9.9, 64 over 500 27.0 / 23.5, 64 over 8192 128.7 either way.)
#define PD_OVERHEAD 4
#define PD_MIN_SHARE 4
// (Quotients of 64 bits take the device a hundred instructions each, and every workgroup forms them: lines that fit 31 bits do without.)
#define PG_SHORT_LINE (1ll << 31)
PG_FN int64_t pg_parts(int64_t total, int64_t room, int share) {
  const int64_t parts = total < PG_SHORT_LINE ? (int64_t)(((unsigned)total + (unsigned)share - 1u) / (unsigned)share) : room;
  return parts < room ? (parts < 1 ? 1 : parts) : room;
}
// (at most 2^15 parts)
PG_FN int64_t pg_cut(int64_t total, int64_t parts, int64_t p) {
  if (total < PG_SHORT_LINE) {
    const unsigned t = (unsigned)total, n = (unsigned)parts, at = (unsigned)p, each = t / n;
    return (int64_t)(each * at + (t - each * n) * at / n);
  }
  return total / parts * p + total % parts * p / parts;
}
// How near: a cut leaves partials behind that are written, read and merged, some four units' worth, and is not worth a quarter of a part.
PG_FN int pg_near(int64_t total, int64_t parts) {
  const int64_t four = 16 * parts;
  return total >= four ? 4 : total >= 12 * parts ? 3 : total >= 8 * parts ? 2 : 1;
}
// Where a cut `off` units into a row tile of n blocks stands: block 0 .. n - 1 of it, or n: the start of what follows.
PG_FN int pg_snap(int64_t off, int n, int overhead, int near) {
  const int64_t t = off - overhead;
  return t < near ? 0 : t > n - near ? n : (int)t;
}

// Sequences of as many rows and keys each may keep their row tiles whole: a kv head's workgroups are dealt them turn by turn, there and back,
// the longest first.  The tiles of `together` sequences, four turns of them, are dealt before the next ones', so that workgroups that run at a
// time read the same keys.  (32 prompts of 1024 tokens, us, two turns / four / all at once: 32 heads over 8 346 / 351 / 368, in a window of
// 256 280 / 267 / 272, 28 over 4 336 / 328 / 313, 14 over 2 of 64 channels 123 / 110 / 104.)  false: nothing falls to the workgroup in this turn.
PG_FN int pg_together(int tiles, int workgroups, int batch) { return pg_min(pg_max(1, (4 * workgroups + tiles - 1) / tiles), batch); }
PG_FN bool pg_deal(int turn, int part, int workgroups, int batch, int tiles, int together, int* b, int* rt) {
  const int place = turn * workgroups + (turn & 1 ? workgroups - 1 - part : part);
  if (place >= tiles * batch) return false;
  if (batch == 1) {
    *b = 0;
    *rt = tiles - 1 - place;
    return true;
  }
  const int deal = place / (together * tiles), at = place - deal * (together * tiles), n = pg_min(together, batch - deal * together);
  *rt = tiles - 1 - at / n;
  *b = deal * together + at % n;
  return true;
}
