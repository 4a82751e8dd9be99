// Eviction from a paged cache by accumulated attention weight (sp_paged_evict_bf16): of every kv head of a request the first keys, the last ones and
// the `budget` heaviest of those between stay, moved to the front of the request's pages in the order they stood in.
//
// The heaviest are those above the budget-th largest weight T and as many of those equal to it as there is room for, lowest place first.  Finite
// floats without a sign are ordered as their patterns are: a histogram of the patterns' upper 11 bits says which of its bins T lies in; the keys of that
// bin and of those above it are listed in order, some hundredths more than stay; and two histograms of 10 bits over the list find T and what of it goes.
// So the weights are read twice, by as many workgroups as a kv head's keys are shared out to, and the list by one.  Moving is a gather in place: a kept key
// comes from its place or further back, so that a row may be written once the rows in front of it have been read.  Chunks of rows are read all at a time, by a
// workgroup each, and written behind a wait for the chunks in front (sp_evict_move_kernel).
// Moving is HBM-bound where there are many kv heads in all, kept rows once in and out; one request's is latency: chains of three loads.
//
// Measured, 128 channels, on rows that have not been moved before: 16 requests of up to 8001 keys, 4 kv heads, 2064 rows left, 133 MB: choosing 14 us, moving 35, 3.8 TB/s;
// one of 131072 keys, 8 kv heads, 8192 left: two reads of the weights 7 and 10, choosing 21, moving 27; one of 2000, 320 left: choosing 13, moving 6.
#include "sp_common.h"
#include "sp_paged_plan.h"

#define EV_THREADS 1024
#define EV_WAVES (EV_THREADS / SP_WAVE)
#define EV_MAX_SEQS 4096
#define EV_BINS 2048        // of the first histogram: bits 20 .. 30 of a weight's pattern
#define EV_RUN 16           // keys of a thread, which lie in one page
#define EV_CHUNK (EV_THREADS * EV_RUN)
#define EV_MAX_SHARES 16    // workgroups that share a kv head's keys
#define EV_ONE 49152        // keys that one workgroup goes through at least
#define EV_TURN 10          // entries of a lane on their way
#define EV_SLICE 512        // channels of a row that a workgroup moves
#define EV_AHEAD 6          // rows of a thread
#define EV_POLLS (1 << 20)  // looks that a lane of a workgroup that waits has for all of its wait: a second or more
#define EV_FEW 256          // workgroups that move: one a CU
#define EV_MOST 8192        // workgroups that move at most, but for one a stream: 16 times as many as the card holds

typedef uint32_t ev_u32x4 __attribute__((ext_vector_type(4)));
typedef float ev_floatx4 __attribute__((ext_vector_type(4)));

struct EvArgs {
  sp_bf16 *k, *v;
  float* weights;
  const int32_t *table, *lens, *first;
  int32_t* new_lens;
  int64_t table_stride, sk_p, sk_n, sk_h, sv_p, sv_n, sv_h, sw_p, sw_h;
  int batch, hkv, d, width, num_pages, shift, budget, recent, shares, by_four, slices, chunks, polls;
  // By place in the pages, [num_pages][kv head][page]: entry i of a request's list stands at the place of its i-th key behind the first ones.  First
  // pattern << 32 | place of what is listed, then the place that a kept key comes from; a place is page << shift + place in it.
  uint64_t* list;
  uint32_t* hists;  // [request][kv head][share][EV_BINS]
  int32_t* counts;  // [request][kv head][share]: entries of the list
  int2* bins;       // [request][kv head]: what ev_find says of the first histogram
  int32_t *tickets, *done;  // [stream] chunks that were taken, [stream][chunk] those that are read; a stream: a kv head's K, V (by EV_SLICE channels) or weights
};

// What becomes of a request: keys first .. first + mid - 1 may go, `keep` of them stay (keep == mid: nothing moves).
struct EvRequest {
  int len, first, mid, keep;
};
__device__ __forceinline__ EvRequest ev_request(const EvArgs& a, int b) {
  EvRequest r;
  r.len = pg_max(0, pg_min(a.lens[b], PG_MAX_KEYS));
  r.first = a.first != nullptr ? pg_max(0, pg_min(a.first[b], r.len)) : 0;
  r.mid = pg_max(0, r.len - r.first - a.recent);
  r.keep = pg_min(r.mid, a.budget);
  return r;
}
// every key behind the first ones has a page; asked by all threads of a workgroup, which meet
__device__ __forceinline__ bool ev_has_pages(const EvArgs& a, int b, const EvRequest& r) {
  int missing = r.len > (a.width << a.shift);
  if (!missing)
    for (int i = (r.first >> a.shift) + (int)threadIdx.x; i <= (r.len - 1) >> a.shift; i += EV_THREADS)
      missing |= (unsigned)a.table[b * a.table_stride + i] >= (unsigned)a.num_pages;
  return __syncthreads_or(missing) == 0;
}
// A kv head whose keys a workgroup's registers hold is done by the choosing launch alone.
__device__ __forceinline__ bool ev_in_registers(const EvRequest& r) { return ((r.first + r.mid + EV_RUN - 1) & -EV_RUN) - (r.first & -EV_RUN) <= EV_CHUNK; }
// A request's kv head, one of a.batch * a.hkv.
struct EvPair {
  const EvArgs& a;
  const int32_t* table;
  int kvh;
  EvRequest r;
  int each, more;  // keys of a share; so many shares have one more
  __device__ __forceinline__ int64_t place(int j) const {  // of key j in the pages: of a kv head, of all of them where there are a.hkv side by side
    return ((int64_t)table[j >> a.shift] << a.shift) + (j & ((1 << a.shift) - 1));
  }
  __device__ __forceinline__ uint64_t* entry(int page, int j) const { return a.list + ((((int64_t)page * a.hkv + kvh) << a.shift) + (j & ((1 << a.shift) - 1))); }
  __device__ __forceinline__ uint64_t* entry(int i) const { return entry(table[(r.first + i) >> a.shift], r.first + i); }
  // Patterns of keys j .. j + EV_RUN - 1 (j a multiple of EV_RUN); those outside lo .. hi - 1 are left as they are.  -> place of key j
  __device__ __forceinline__ uint32_t load(int j, int lo, int hi, uint32_t (&key)[EV_RUN]) const {
    if (j + EV_RUN <= lo || j >= hi) return 0u;
    const float* const w = a.weights + (int64_t)table[j >> a.shift] * a.sw_p + kvh * a.sw_h + (j & ((1 << a.shift) - 1));
    float x[EV_RUN];
    if (a.by_four) {
#pragma unroll
      for (int e = 0; e < EV_RUN; e += 4) {
        const ev_floatx4 y = *reinterpret_cast<const ev_floatx4*>(w + e);
#pragma unroll
        for (int u = 0; u < 4; ++u) x[e + u] = y[u];
      }
    } else {
#pragma unroll
      for (int e = 0; e < EV_RUN; ++e) x[e] = w[e];
    }
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e)
      if (j + e >= lo && j + e < hi) key[e] = sp_sort_key(x[e]);
    return (uint32_t)place(j);
  }
  // keys of a share, from .. to
  __device__ __forceinline__ int share_start(int s) const {
    return r.first + each * s + pg_min(s, more);
  }
};

// bins of a histogram in LDS from above: the one that holds the left-th largest, and which of it that is
struct EvBin {
  int bin, left;
};
template <int BINS>
__device__ __forceinline__ EvBin ev_find(const uint32_t* hist, int left, int* wave_s, int* found_s) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  constexpr int EACH = BINS / EV_THREADS;
  int mine = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) mine += hist[BINS - 1 - (t * EACH + e)];
  int at = mine;
#pragma unroll
  for (int o = 1; o < SP_WAVE; o <<= 1) {
    const int y = __shfl_up(at, o, SP_WAVE);
    if (lane >= o) at += y;
  }
  if (lane == SP_WAVE - 1) wave_s[wave] = at;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < EV_WAVES; ++x) at += x < wave ? wave_s[x] : 0;
  at -= mine;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int bin = BINS - 1 - (t * EACH + e), n = hist[bin];
    if (at < left && left <= at + n) found_s[0] = bin, found_s[1] = left - at;
    at += n;
  }
  __syncthreads();
  const EvBin f = {found_s[0], found_s[1]};
  __syncthreads();
  return f;
}
// the histogram of a share, in LDS
__device__ __forceinline__ void ev_hist(const EvPair& p, int from, int to, uint32_t* hist) {
  for (int i = threadIdx.x; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
  __syncthreads();
  for (int j = (from & -EV_RUN) + (int)threadIdx.x * EV_RUN; j < to; j += EV_THREADS * EV_RUN) {
    uint32_t key[EV_RUN];
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e) key[e] = ~0u;
    p.load(j, from, to, key);
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e)
      if (key[e] != ~0u) atomicAdd(&hist[key[e] >> 20], 1u);
  }
  __syncthreads();
}
// sums of the threads in front, and over all of them (two barriers)
__device__ __forceinline__ int ev_scan(int mine, int* wave_s, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int at = mine;
#pragma unroll
  for (int o = 1; o < SP_WAVE; o <<= 1) {
    const int y = __shfl_up(at, o, SP_WAVE);
    if (lane >= o) at += y;
  }
  if (lane == SP_WAVE - 1) wave_s[wave] = at;
  __syncthreads();
  *all = 0;
#pragma unroll
  for (int x = 0; x < EV_WAVES; ++x) {
    if (x == wave) at += *all;
    *all += wave_s[x];
  }
  __syncthreads();
  return at - mine;
}
// Lists the keys of a share that lie in bin `bin` or above, in order; -> how many.  stage: EV_CHUNK entries of LDS, so that threads side by side write them.
__device__ __forceinline__ int ev_gather(const EvPair& p, int from, int to, uint32_t bin, int* wave_s, uint64_t* stage) {
  int listed = 0;
  for (int j0 = from & -EV_RUN; j0 < to; j0 += EV_CHUNK) {
    const int j = j0 + (int)threadIdx.x * EV_RUN;
    uint32_t key[EV_RUN];
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e) key[e] = ~0u;
    const uint32_t place = p.load(j, from, to, key);
    int mine = 0, all;
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e) mine += key[e] != ~0u && key[e] >> 20 >= bin;
    int at = ev_scan(mine, wave_s, &all);
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e)
      if (key[e] != ~0u && key[e] >> 20 >= bin) stage[at++] = (uint64_t)key[e] << 32 | (place + e);
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += EV_THREADS) *p.entry(from - p.r.first + listed + i) = stage[i];
    listed += all;
    __syncthreads();
  }
  return listed;
}

__device__ __forceinline__ EvPair ev_pair(const EvArgs& a, int pair) {
  const int b = pair / a.hkv;
  const EvRequest r = ev_request(a, b);
  const int each = a.shares > 1 ? (int)((unsigned)r.mid / (unsigned)a.shares) : r.mid;
  return EvPair{a, a.table + b * a.table_stride, pair % a.hkv, r, each, r.mid - each * a.shares};
}

__global__ __launch_bounds__(EV_THREADS) void sp_evict_hist_kernel(const EvArgs a) {
  __shared__ uint32_t hist[EV_BINS];
  const int pair = blockIdx.x / a.shares, share = blockIdx.x % a.shares;
  const EvPair p = ev_pair(a, pair);
  if (p.r.keep == p.r.mid || p.r.keep == 0 || ev_in_registers(p.r) || !ev_has_pages(a, pair / a.hkv, p.r)) return;
  ev_hist(p, p.share_start(share), p.share_start(share + 1), hist);
  for (int i = threadIdx.x; i < EV_BINS; i += EV_THREADS) a.hists[(int64_t)blockIdx.x * EV_BINS + i] = hist[i];
}
// (a kv head's shares find the same bin)
__device__ __forceinline__ EvBin ev_first_bin(const EvArgs& a, int pair, int keep, uint32_t* hist, int* wave_s, int* found_s) {
  for (int i = threadIdx.x; i < EV_BINS; i += EV_THREADS) {
    uint32_t part[EV_MAX_SHARES], n = 0;
#pragma unroll
    for (int x = 0; x < EV_MAX_SHARES; ++x) part[x] = a.hists[((int64_t)pair * a.shares + pg_min(x, a.shares - 1)) * EV_BINS + i];
    __builtin_amdgcn_sched_barrier(0);  // (all on their way at once)
#pragma unroll
    for (int x = 0; x < EV_MAX_SHARES; ++x) n += x < a.shares ? part[x] : 0;
    hist[i] = n;
  }
  __syncthreads();
  return ev_find<EV_BINS>(hist, keep, wave_s, found_s);
}
__global__ __launch_bounds__(EV_THREADS) void sp_evict_gather_kernel(const EvArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint64_t stage[];
  __shared__ uint32_t hist[EV_BINS];
  __shared__ int wave_s[EV_WAVES], found_s[2];
  const int pair = blockIdx.x / a.shares, share = blockIdx.x % a.shares;
  const EvPair p = ev_pair(a, pair);
  if (p.r.keep == p.r.mid || p.r.keep == 0 || ev_in_registers(p.r) || !ev_has_pages(a, pair / a.hkv, p.r)) return;
  const EvBin f = ev_first_bin(a, pair, p.r.keep, hist, wave_s, found_s);
  const int n = ev_gather(p, p.share_start(share), p.share_start(share + 1), (uint32_t)f.bin, wave_s, stage);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
  if (threadIdx.x == 0 && share == 0) a.bins[pair] = make_int2(f.bin, f.left);
}

// One workgroup a kv head: T, and the list of what stays.  Up to EV_CHUNK keys, a kv head's own or those that are listed, stay in registers for all of it.
__global__ __launch_bounds__(EV_THREADS) void sp_evict_choose_kernel(const EvArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint64_t stage[];
  __shared__ uint32_t hist[EV_BINS];
  __shared__ int wave_s[2 * EV_WAVES], found_s[2], count_s[EV_MAX_SHARES], start_s[EV_MAX_SHARES];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, pair = blockIdx.x, b = pair / a.hkv;
  const EvPair p = ev_pair(a, pair);
  for (int part = 0; part <= 2 * a.slices; ++part) {
    const int stream = part * a.batch * a.hkv + pair;
    if (t == 0) a.tickets[stream] = 0;
    for (int i = t; i < a.chunks; i += EV_THREADS) a.done[(int64_t)stream * a.chunks + i] = 0;
  }
  const bool goes = p.r.keep < p.r.mid && ev_has_pages(a, b, p.r);
  if (p.kvh == 0 && t == 0) a.new_lens[b] = goes ? p.r.len - p.r.mid + p.r.keep : p.r.len;
  if (!goes || p.r.keep == 0) return;
  EvBin f;
  const bool whole = ev_in_registers(p.r);
  int listed = 0;  // (uniform)
  if (!whole) {
    if (a.shares == 1) {
      ev_hist(p, p.r.first, p.r.first + p.r.mid, hist);
      f = ev_find<EV_BINS>(hist, p.r.keep, wave_s, found_s);
      const int n = ev_gather(p, p.r.first, p.r.first + p.r.mid, (uint32_t)f.bin, wave_s, stage);
      if (t == 0) count_s[0] = n;
    } else {
      const int2 bin = a.bins[pair];
      f = {bin.x, bin.y};
      if (t < a.shares) count_s[t] = a.counts[pair * a.shares + t];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < EV_MAX_SHARES; ++s) {
      const int n = s < a.shares ? count_s[s] : 0;
      if (t == s) start_s[s] = listed;
      listed += n;
    }
    __syncthreads();
  }
  if (whole || listed <= EV_CHUNK) {
    uint32_t key[EV_RUN], place[EV_RUN];
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e) key[e] = ~0u, place[e] = 0u;
    if (whole) {
      const int j = (p.r.first & -EV_RUN) + t * EV_RUN;
      const uint32_t first = p.load(j, p.r.first, p.r.first + p.r.mid, key);
#pragma unroll
      for (int e = 0; e < EV_RUN; ++e) place[e] = first + e;
    } else {
      // A wave has as many entries as any, of one share or of several, and lanes side by side read entries side by side; then every thread its own out of LDS.
      // (Pages, then entries: asked for one after the other each waits for the last.)
      const int r0 = listed * wave / EV_WAVES, r1 = listed * (wave + 1) / EV_WAVES;
      const int starts = lane < a.shares ? start_s[lane] : 0, ends = lane < a.shares ? starts + count_s[lane] : 0;
      for (uint64_t of = __ballot(starts < r1 && ends > r0); of != 0ull; of &= of - 1ull) {
        const int s = __builtin_ctzll(of), start = __builtin_amdgcn_readlane(starts, s), base = p.share_start(s) - start;
        const int lo = pg_max(r0, start), hi = pg_min(r1, __builtin_amdgcn_readlane(ends, s));
        for (int i0 = lo; i0 < hi; i0 += EV_TURN * SP_WAVE) {
          int page[EV_TURN];
          uint64_t x[EV_TURN];
#pragma unroll
          for (int e = 0; e < EV_TURN; ++e) page[e] = p.table[(base + pg_min(i0 + e * SP_WAVE + lane, hi - 1)) >> a.shift];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < EV_TURN; ++e) x[e] = *p.entry(page[e], base + pg_min(i0 + e * SP_WAVE + lane, hi - 1));
#pragma unroll
          for (int e = 0; e < EV_TURN; ++e)
            if (i0 + e * SP_WAVE + lane < hi) stage[i0 + e * SP_WAVE + lane] = x[e];
        }
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EV_RUN; ++e)
        if (t * EV_RUN + e < listed) key[e] = (uint32_t)(stage[t * EV_RUN + e] >> 32), place[e] = (uint32_t)stage[t * EV_RUN + e];
    }
    uint32_t top = whole ? 0 : (uint32_t)f.bin;
    int left = whole ? p.r.keep : f.left;
    for (int shift = whole ? 20 : 10; shift >= 0; shift -= 10) {
      for (int i = t; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EV_RUN; ++e)
        if (key[e] != ~0u && (shift == 20 || key[e] >> (shift + 10) == top)) atomicAdd(&hist[(key[e] >> shift) & (shift == 20 ? 2047u : 1023u)], 1u);
      __syncthreads();
      f = ev_find<EV_BINS>(hist, left, wave_s, found_s);
      top = top << 10 | (uint32_t)f.bin;
      left = f.left;
    }
    // `left` of those equal to T stay, the first
    int overs = 0, sames = 0, all;
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e) overs += key[e] != ~0u && key[e] > top, sames += key[e] == top;
    const int in_front = ev_scan(overs | sames << 16, wave_s, &all);  // (neither reaches 2^16: EV_CHUNK is 2^14)
    int over_at = in_front & 0xffff, same_at = in_front >> 16;
#pragma unroll
    for (int e = 0; e < EV_RUN; ++e) {
      const bool over = key[e] != ~0u && key[e] > top, same = key[e] == top;
      if (over || (same && same_at < left)) stage[over_at + pg_min(same_at, left)] = place[e];
      over_at += over, same_at += same;
    }
    __syncthreads();
#pragma unroll 8
    for (int i = t; i < p.r.keep; i += EV_THREADS) *p.entry(i) = stage[i];
    return;
  }
  uint32_t top = (uint32_t)f.bin;  // bits of T that are known
  int left = f.left;               // the left-th largest of those that share them is T
  for (int shift = 10; shift >= 0; shift -= 10) {
    for (int i = t; i < 1024; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int s = 0; s < a.shares; ++s) {
      const int base = p.share_start(s) - p.r.first;
      for (int i = t; i < count_s[s]; i += EV_THREADS) {
        const uint32_t key = (uint32_t)(*p.entry(base + i) >> 32);
        if (key >> (shift + 10) == top) atomicAdd(&hist[(key >> shift) & 1023u], 1u);
      }
    }
    __syncthreads();
    f = ev_find<1024>(hist, left, wave_s, found_s);
    top = top << 10 | (uint32_t)f.bin;
    left = f.left;
  }
  // `left` of those equal to T stay.  The list becomes where they come from, in place: an entry is written at or in front of where it was read.
  int kept = 0, equal = 0;  // in front of this turn
  for (int s = 0; s < a.shares; ++s) {
    const int base = p.share_start(s) - p.r.first;
    for (int i0 = 0; i0 < count_s[s]; i0 += EV_THREADS) {
      const int i = i0 + t;
      const bool there = i < count_s[s];
      const uint64_t x = there ? *p.entry(base + i) : 0ull;
      const uint32_t key = (uint32_t)(x >> 32);
      const bool over = there && key > top, same = there && key == top;
      const uint64_t overs = __ballot(over), sames = __ballot(same), below = (1ull << lane) - 1ull;
      if (lane == 0) wave_s[wave] = __builtin_popcountll(overs), wave_s[EV_WAVES + wave] = __builtin_popcountll(sames);
      __syncthreads();  // (the turn's entries are read)
      int over_at = 0, same_at = equal, overs_all = 0, sames_all = 0;
#pragma unroll
      for (int y = 0; y < EV_WAVES; ++y) {
        const int n = wave_s[y], m = wave_s[EV_WAVES + y];
        if (y < wave) over_at += n, same_at += m;
        overs_all += n, sames_all += m;
      }
      over_at += __builtin_popcountll(overs & below);
      same_at += __builtin_popcountll(sames & below);
      if (over || (same && same_at < left)) *p.entry(kept + over_at + pg_min(same_at, left) - pg_min(equal, left)) = (uint32_t)x;
      kept += overs_all + pg_min(equal + sames_all, left) - pg_min(equal, left);
      equal += sames_all;
      __syncthreads();
    }
  }
}

// A workgroup moves a chunk of a kv head's kept rows: reads them all, waits until the chunks in front of it have read theirs, which alone may need what it
// writes over, and writes.  A chunk is taken when its workgroup has begun, so that whoever is waited for runs, and waits for nobody before it has read: a wait
// of some microseconds.  It is bounded all the same; a workgroup that has waited in vain does not write, and the request's length is -1.
template <int AHEAD, bool MORE>  // MORE: a stream has more chunks than workgroups, which take another behind each (it costs those that have had their own 6 us of 46)
__global__ __launch_bounds__(EV_THREADS) void sp_evict_move_kernel(const EvArgs a) {
  __shared__ int chunk_s, in_vain_s;
  const int t = threadIdx.x, pair = blockIdx.x, part = blockIdx.y, stream = part * gridDim.x + pair, b = pair / a.hkv;
  const EvPair p = ev_pair(a, pair);
  const EvRequest& r = p.r;
  if (r.keep >= r.mid) return;
  // (the look at the table brings its entries near while the ticket is on its way: 30 us for 44 where the launch before this one had told what it says)
  auto take = [&] {
    if (t == 0) chunk_s = __hip_atomic_fetch_add(a.tickets + stream, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  take();
  if (!ev_has_pages(a, b, r)) return;
  const int rows = r.keep + r.len - r.first - r.mid, in = (1 << a.shift) - 1;
  auto move_chunk = [&](auto type, int lanes, auto at) {  // elements of a row side by side, one a thread.  -> there may be another chunk
    const int per = EV_THREADS / lanes, row = t / lanes, chunk = chunk_s;
    const int64_t i0 = (int64_t)chunk * (per * AHEAD);
    if (i0 >= rows) return false;
    // (a thread without a row reads the last one's.  Every row's page, then every row's source, then every row: asked for row by row each waits for the last)
    decltype(type) y[AHEAD];
    uint32_t to[AHEAD], come[AHEAD];
    int last[AHEAD];  // page that a last key comes from
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = pg_min((int)i0 + u * per + row, rows - 1);
      to[u] = (uint32_t)p.place(r.first + i);
      last[u] = p.table[pg_min(r.first + r.mid + pg_max(i - r.keep, 0), r.len - 1) >> a.shift];  // (there may be no last keys)
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) come[u] = (uint32_t)a.list[(((int64_t)(to[u] >> a.shift) * a.hkv + p.kvh) << a.shift) + (to[u] & in)];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = pg_min((int)i0 + u * per + row, rows - 1);
      y[u] = *at(i < r.keep ? come[u] : ((uint32_t)last[u] << a.shift) + ((r.first + r.mid + (i - r.keep)) & in));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the chunk is read
    int32_t* const done = a.done + (int64_t)stream * a.chunks;
    if (t == 0) __hip_atomic_store(done + chunk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (t < SP_WAVE) {
      int polls = a.polls;
      bool in_vain = false;
      for (int i = t; i < chunk; i += SP_WAVE) {
        bool read = false;
        while (!read && polls > 0) {
          read = __hip_atomic_load(done + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
          if (!read) --polls, __builtin_amdgcn_s_sleep(1);
        }
        in_vain |= !read;
      }
      const bool any = __ballot(in_vain) != 0ull;
      if (t == 0) in_vain_s = any;
    }
    asm volatile("" ::: "memory");
    __syncthreads();
    if (in_vain_s) {
      if (t == 0) a.new_lens[b] = -1;
      return false;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (row < per && i0 + u * per + row < rows) *at(to[u]) = y[u];
    return MORE && i0 + per * AHEAD < rows;
  };
  auto move = [&](auto type, int lanes, auto at) {
    while (move_chunk(type, lanes, at)) {
      take();
      __syncthreads();
    }
  };
  if (part == 2 * a.slices) {
    float* const w = a.weights + p.kvh * a.sw_h;
    move(0.f, 1, [&](int64_t x) { return w + (x >> a.shift) * a.sw_p + (x & in); });
  } else {
    const bool is_v = part >= a.slices;
    const int c = part % a.slices * EV_SLICE, lanes = pg_min(a.d - c, EV_SLICE) / 8;
    const int64_t page_at = is_v ? a.sv_p : a.sk_p, slot_at = is_v ? a.sv_n : a.sk_n;
    sp_bf16* const x = (is_v ? a.v + p.kvh * a.sv_h : a.k + p.kvh * a.sk_h) + c + t % lanes * 8;
    move(ev_u32x4{}, lanes, [&](int64_t y) { return reinterpret_cast<ev_u32x4*>(x + (y >> a.shift) * page_at + (y & in) * slot_at); });
  }
}

// ---- host -------------------------------------------------------------------------------------------------
// Workgroups that share a kv head's keys, by what the table has room for: as many as fill the card, of some 8192 keys at least, where they pay for the two launches
// more.  us for the whole call, one / shared, eight kv heads' 8000 keys 22 / 26, 20000 33 / 37, 32000 37 / 40, 65000 53 / 47, 131072 87 / 70; 64 kv heads' 20000
// 43 / 50.
static int ev_shares(int64_t pairs, int64_t room) {
  const int64_t by_keys = room < EV_ONE ? 1 : room / 8192, by_card = 256 / pairs;
  const int64_t n = by_keys < by_card ? by_keys : by_card;
  return n < 1 ? 1 : n > EV_MAX_SHARES ? EV_MAX_SHARES : (int)n;
}
struct EvMove {
  int64_t slices, streams, ahead, chunks;
};
// Chunks of `kept` rows at most, as many as the widest stream needs.  A thread has EV_AHEAD rows in flight, or one where few workgroups are enough all the same: us,
// one / 2 / 4 / 6 / 8, eight kv heads' 320 rows of 128 channels 7 / 9 / 10 / 11 / 11, their 8192 rows 45 / 34 / 31 / 29 / 30, 64 kv heads' 2000 rows 67 / 45 / 37 /
// 36 / 38.
static EvMove ev_move(int64_t pairs, int64_t d, int64_t kept) {
  EvMove m;
  m.slices = (d + EV_SLICE - 1) / EV_SLICE, m.streams = pairs * (2 * m.slices + 1);
  const int64_t rows = EV_THREADS / ((d < EV_SLICE ? d : EV_SLICE) / 8);
  m.ahead = m.streams * ((kept + rows - 1) / rows) <= EV_FEW ? 1 : EV_AHEAD;
  m.chunks = (kept + rows * m.ahead - 1) / (rows * m.ahead);
  return m;
}
struct EvSizes {
  size_t list, hists, counts, bins, tickets, done, bytes;
};
static EvSizes ev_sizes(int64_t batch, int64_t hkv, int64_t pool_keys, int shares, const EvMove& m) {
  EvSizes s;
  const int64_t pairs = batch * hkv;
  s.list = 0;
  s.hists = (size_t)(hkv * pool_keys) * sizeof(uint64_t);
  s.counts = s.hists + (shares > 1 ? (size_t)(pairs * shares) * EV_BINS * sizeof(uint32_t) : 0);
  s.bins = s.counts + (shares > 1 ? ((size_t)(pairs * shares) * sizeof(int32_t) + 15) / 16 * 16 : 0);
  s.tickets = s.bins + (shares > 1 ? ((size_t)pairs * sizeof(int2) + 15) / 16 * 16 : 0);
  s.done = s.tickets + ((size_t)m.streams * sizeof(int32_t) + 15) / 16 * 16;
  const int64_t chunks = m.streams * m.chunks;
  s.bytes = s.done + ((size_t)(chunks > EV_FEW ? chunks : EV_FEW) * sizeof(int32_t) + 15) / 16 * 16;  // (those of fewer rows than the most may be more)
  return s;
}
extern "C" size_t sp_paged_evict_workspace_bytes(int32_t batch, int32_t hkv, int32_t d, int64_t num_pages, int64_t page_size, int64_t table_width) {
  if (batch <= 0 || hkv <= 0 || d <= 0 || d % 8 || d > 65536 || num_pages <= 0 || page_size <= 0 || table_width <= 0 || num_pages > 0x7fffffffll || page_size > 1024 || table_width > PG_MAX_KEYS)
    return 0;
  const int64_t pairs = (int64_t)batch * hkv;
  const int64_t room = table_width * page_size;
  return ev_sizes(batch, hkv, num_pages * page_size, ev_shares(pairs, room), ev_move(pairs, d, room)).bytes;
}

extern "C" int sp_paged_evict_bf16(const sp_paged_evict_args* x) { return sp_paged_evict_bounded_bf16(x, EV_POLLS); }

extern "C" int sp_paged_evict_bounded_bf16(const sp_paged_evict_args* x, int32_t polls) {
  const char* who = "sp_paged_evict_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->batch > 0 && x->hkv > 0 && x->table_width > 0 && x->num_pages > 0, SP_ERR_INVALID_ARGUMENT,
             "%s: batch=%lld hkv=%lld table_width=%lld num_pages=%lld", who, (long long)x->batch, (long long)x->hkv, (long long)x->table_width,
             (long long)x->num_pages);
  SP_REQUIRE(x->budget >= 0 && x->recent >= 0, SP_ERR_INVALID_ARGUMENT, "%s: budget=%lld recent=%lld", who, (long long)x->budget, (long long)x->recent);
  SP_REQUIRE(polls >= 0, SP_ERR_INVALID_ARGUMENT, "%s: polls %d", who, (int)polls);
  SP_REQUIRE(x->d > 0 && x->d % 8 == 0 && x->d <= 65536, SP_ERR_UNSUPPORTED, "%s: head_dim %lld (a multiple of 8)", who, (long long)x->d);
  int shift = 4;
  while (shift <= 10 && x->page_size != 1ll << shift) ++shift;
  SP_REQUIRE(shift <= 10, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  SP_REQUIRE(x->batch <= EV_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, EV_MAX_SEQS);
  const int64_t pairs = x->batch * x->hkv;
  SP_REQUIRE(x->hkv <= 65536 && x->num_pages <= 0x7fffffffll && x->table_width <= PG_MAX_KEYS && x->table_width << shift <= PG_MAX_KEYS &&
                 x->num_pages << shift <= 0xffffffffll && pairs * EV_THREADS < (1ll << 32),
             SP_ERR_UNSUPPORTED, "%s: hkv=%lld num_pages=%lld table_width=%lld too large", who, (long long)x->hkv, (long long)x->num_pages,
             (long long)x->table_width);
  const int64_t k_p = pg_used_stride(x->k_stride_page, x->num_pages), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  const int64_t v_p = pg_used_stride(x->v_stride_page, x->num_pages), v_h = pg_used_stride(x->v_stride_h, x->hkv);
  SP_REQUIRE(x->k_pages && x->v_pages && x->weights && x->block_table && x->seq_lens && x->new_lens, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->new_lens != x->seq_lens && x->new_lens != x->first, SP_ERR_INVALID_ARGUMENT, "%s: an output is an input", who);
  SP_REQUIRE(((uintptr_t)x->k_pages | (uintptr_t)x->v_pages) % 16 == 0 && (k_p | k_h | x->k_stride_slot | v_p | v_h | x->v_stride_slot) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  const int shares = ev_shares(pairs, x->table_width << shift);
  const int64_t room = x->table_width << shift, most = x->budget > room || x->recent > room || x->budget + x->recent > room ? room : x->budget + x->recent;
  const EvMove move = ev_move(pairs, x->d, most);  // (rows that are kept beside the first ones, at most)
  SP_REQUIRE(move.streams * move.chunks <= 0x7fffffffll, SP_ERR_UNSUPPORTED, "%s: %lld rows of %lld kv heads are too many", who, (long long)most,
             (long long)pairs);
  const EvSizes sizes = ev_sizes(x->batch, x->hkv, x->num_pages << shift, shares, move);
  SP_REQUIRE(x->workspace != nullptr && x->workspace_bytes >= sizes.bytes && (uintptr_t)x->workspace % 16 == 0, SP_ERR_WORKSPACE,
             "%s: workspace missing, too small or misaligned", who);
  EvArgs a = {};
  a.k = (sp_bf16*)x->k_pages, a.v = (sp_bf16*)x->v_pages, a.weights = x->weights;
  a.table = x->block_table, a.lens = x->seq_lens, a.first = x->first, a.new_lens = x->new_lens, a.table_stride = x->table_stride;
  a.sk_p = k_p, a.sk_n = x->k_stride_slot, a.sk_h = k_h, a.sv_p = v_p, a.sv_n = x->v_stride_slot, a.sv_h = v_h;
  a.sw_p = pg_used_stride(x->w_stride_page, x->num_pages), a.sw_h = pg_used_stride(x->w_stride_h, x->hkv);
  a.batch = (int)x->batch, a.hkv = (int)x->hkv, a.d = (int)x->d, a.width = (int)x->table_width, a.num_pages = (int)x->num_pages, a.shift = shift;
  a.budget = (int)(x->budget < PG_MAX_KEYS ? x->budget : PG_MAX_KEYS), a.recent = (int)(x->recent < PG_MAX_KEYS ? x->recent : PG_MAX_KEYS);
  a.shares = shares, a.slices = (int)move.slices, a.chunks = (int)move.chunks, a.polls = polls;
  a.by_four = (uintptr_t)x->weights % 16 == 0 && (a.sw_p | a.sw_h) % 4 == 0;
  char* const ws = (char*)x->workspace;
  a.list = (uint64_t*)(ws + sizes.list), a.hists = (uint32_t*)(ws + sizes.hists), a.counts = (int32_t*)(ws + sizes.counts);
  a.bins = (int2*)(ws + sizes.bins), a.tickets = (int32_t*)(ws + sizes.tickets), a.done = (int32_t*)(ws + sizes.done);
  const hipStream_t stream = (hipStream_t)x->stream;
  constexpr int lds = EV_CHUNK * (int)sizeof(uint64_t);
  static bool attr_set[64] = {false};  // per device, once (idempotent)
  int dev = 0;
  SP_HIP(hipGetDevice(&dev));
  SP_REQUIRE(dev >= 0 && dev < 64, SP_ERR_UNSUPPORTED, "%s: device index %d", who, dev);
  if (!attr_set[dev]) {
    for (const void* f : {(const void*)sp_evict_gather_kernel, (const void*)sp_evict_choose_kernel})
      SP_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    attr_set[dev] = true;
  }
  if (shares > 1) {
    hipLaunchKernelGGL(sp_evict_hist_kernel, dim3((unsigned)(pairs * shares)), dim3(EV_THREADS), 0, stream, a);
    hipLaunchKernelGGL(sp_evict_gather_kernel, dim3((unsigned)(pairs * shares)), dim3(EV_THREADS), lds, stream, a);
  }
  hipLaunchKernelGGL(sp_evict_choose_kernel, dim3((unsigned)pairs), dim3(EV_THREADS), lds, stream, a);
  if (move.chunks > 0) {
    const int64_t each = EV_MOST / move.streams, of_stream = move.chunks < each ? move.chunks : each < 1 ? 1 : each;
    const auto kernel = of_stream < move.chunks ? sp_evict_move_kernel<EV_AHEAD, true> : move.ahead == 1 ? sp_evict_move_kernel<1, false> : sp_evict_move_kernel<EV_AHEAD, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)pairs, (unsigned)(move.streams / pairs), (unsigned)of_stream), dim3(EV_THREADS), 0, stream, a);
  }
  SP_LAUNCH_CHECK();
  return SP_OK;
}
