// Attention of new tokens over a paged cache in which groups of requests have their first keys in common (sp_shared_attn_bf16):
//   out = sum_j exp(scale q . k_j) v_j / sum_j exp(scale q . k_j) over the keys j <= p of the row's request,
// the sum over the shared keys formed once for all rows of the group and joined with that over the request's own: with running maxima m and
// sums l of either side, out = (2^(m1 - m) o1 + 2^(m2 - m) o2) / (2^(m1 - m) l1 + 2^(m2 - m) l2).
//
// HBM-bound as long as a group has fewer than some 250 rows a kv head, (token, query head) pairs: shared keys are read once per tile of up to 128
// rows, a request's own once.  Two loops over steps of 32 keys, whose operands direct loads bring to rings in LDS:
//   * single tokens of up to 16 heads over their own keys: a wave goes by itself through the steps of one request after the other, the next one's
//     first keys on their way under the end of the one in front; no barrier, and nobody waits for a request to end;
//   * tiles of up to 128 rows: eight waves share blocks of four steps and meet twice in each; a wave has 32 rows, and the waves of the same rows
//     share out the steps.  Two waves share a SIMD, where the matrix instructions of one run under the exponentials of the other.
// Groups of many rows over many keys go to sp_chunk.hip's loop first, in a launch of its own (sh_apart).
//
// Measured, 32 heads over 8 of 128 channels, this launch and the joining one: 64 single tokens behind 8192 shared keys and up to 2000 own, 365 MB, 79 + 6.9 us,
// 4.3 TB/s (a copy 5.05); 8 behind 1024 and up to 200 15.3 + 4.3 us, of which 3.5 are the line, 2 the launch, 9 a part of the group: its queries and first keys,
// two blocks, its end; 128 behind 32768, 55 us for the requests and 117 + 11 for the group (69 GFLOP and half as many for the probabilities' second parts, 880 TFLOP/s).  Without groups 64 single tokens over
// 500 to 2000 keys take 67 us, sp_paged_decode.hip's kernels 70; 8 over 50 to 200 keys 14 and 7, 32 of 64 channels over 250 to 1000
// 23 and 12: the line, and a joining launch whether anything was cut or not.
#include "sp_chunk.h"
#include "sp_ring.h"
#include "sp_shared_plan.h"

#define SH_THREADS (2 * SH_WAVES * SP_WAVE)
// Octaves by which a row's logits may pass its running maximum before that is moved and what has been summed is scaled: nearly all steps go without.
// (Probabilities up to 2^7 are as exact in bf16 as those below 1.)
#define SH_SLACK 7.f

struct ShRequest {
  int first_own;            // its first key that no group sees to
  int group, start0, end0;  // its group, that group's first token and the one behind its last
  int start;                // its own first token
  int pad[3];
};
struct ShArgs {
  const sp_bf16 *q, *k, *v;
  const int32_t *table, *lens, *cu, *shared, *groups, *joined;  // shared: keys of a group, [n_groups]; groups: first requests, [n_groups + 1]
  sp_bf16* out;
  int64_t table_stride, sq_n, sq_h, sk_p, sk_n, sk_h, sv_p, sv_n, sv_h, sw_p, sw_h;  // elements; _p between pages
  int batch, tokens, width, num_pages, shift, n_groups;
  int hkv, group, dense;      // dense: single tokens, a row tile each
  PgDivisor by_group;
  int shared_slots;           // numbers of the groups' row tiles
  int parts;                  // of the line at most, and workgroups of a kv head
  int apart;                  // groups have been seen to (o_row, ml_row)
  int streams;                // single tokens of up to 16 heads: a request's parts are waves', four a workgroup
  float scale_log2;
  float* o_part;              // [part][kv head][2][SH_ROWS][D]: a row tile that began in an earlier part, one that goes on in the next
  float2* ml_part;            // [part][kv head][2][SH_ROWS]
  float* o_stream;            // [part of a wave][kv head][2][16][D]
  float2* ml_stream;
  float* o_row;               // [2][token][query head][D]: row tiles that lie in one part, of groups and of requests
  float2* ml_row;
  int2* parts_of;             // by row tile number: first and last part that hold steps of it
  int4* cuts;                 // [part of a wave]: request and step that it begins with, those that it ends in front of
  ShRequest* of_request;      // [batch + 1]
  float* weights;             // null, or [num_pages][kv head][page]
  const int32_t* weigh_from;  // null, or [batch]: a request's keys in front of that are not weighed
  int weights_by_four;        // four places side by side are one access
  float* logits;              // [num_pages][query head][page]: scaled logits of own keys, in octaves
};

template <int D>
using ShShape = DsShape<D, D / 16, SH_WAVES, 128>;
// LDS: the rings, where the waves meet afterwards; their maxima and sums; what is known of the requests and groups
#define SH_RING 131072
#define SH_MEET (2 * SH_WAVES * 32)  // rows that the waves bring together
#define SH_ML (SH_RING)              // [2][SH_MEET] floats
#define SH_SUMS (SH_ML + 2 * SH_MEET * 4)  // [2 SH_WAVES + 1] int64
#define SH_SEEN (SH_SUMS + 80)                        // [SH_WAVES][4] words
#define SH_ARRAYS (SH_SEEN + 64)
static size_t sh_lds_bytes(int batch, int groups) { return SH_ARRAYS + (3 * ((size_t)batch + 1) + 2 * ((size_t)groups + 1)) * sizeof(int); }
static_assert(ShShape<128>::LDS_BYTES <= SH_RING && ShShape<64>::LDS_BYTES <= SH_RING && SH_MEET * 128 * 4 <= SH_RING && (2 * SH_MAX_SEQS + 1) * 8 <= SH_RING, "");

template <int IMM>
__device__ static __forceinline__ dc_u32x4 sh_read_k(uint32_t addr) {  // (as ds_read_k)
  dc_u32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(IMM));
  return r;
}

struct ShItem {
  int table_row;    // of the block table
  int start, rows;  // first token; rows from there on
  int key0, key1;   // keys that some row sees
  int pos;          // position of token `start`: its row and the following ones see keys up to pos, pos + 1, ..; groups: far behind the last key
  int lo, n;        // first step, steps of a tile
  int slot;         // number of its first row tile
  int row0;         // first row of a tile
};

template <int D>
__global__ __launch_bounds__(SH_THREADS, 1) void sp_shared_kernel(const ShArgs a) {
  using Shape = ShShape<D>;
  constexpr int CT = Shape::CT, KS = D / 32, WAVES = SH_WAVES, NB = Shape::NB;
  constexpr int CHUNKS = D / 8, ROWS = SP_WAVE / CHUNKS;  // of a row; rows of a load instruction
  constexpr int HALF = 16 / ROWS;                         // instructions of 16 keys
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lq = lane & 15, gr = lane >> 4;  // head (or key row, channel) in a 16-wide tile, lane group
  const int g = a.group, kvh = blockIdx.x % a.hkv, part = blockIdx.x / a.hkv;
  const int slot = wave % SH_WAVES, half = wave / SH_WAVES;  // the wave's keys of a block, and its rows where two waves share them
  const int room = a.width << a.shift, n_groups = a.apart ? 0 : a.n_groups, items = n_groups + a.batch;

  // ---- requests and groups ----
  int* const start_s = reinterpret_cast<int*>(lds + SH_ARRAYS);  // [batch + 1] first tokens
  int* const len_s = start_s + a.batch + 1;                      // [batch]
  int* const first_s = len_s + a.batch + 1;                      // [batch] first own keys
  int* const group_s = first_s + a.batch + 1;                    // [n_groups + 1] first requests
  int* const shared_s = group_s + a.n_groups + 1;                // [n_groups] shared keys
  int back = 0;
  for (int i = t; i <= a.batch; i += SH_THREADS) {
    auto start = [&](int j) { return a.cu != nullptr ? pg_max(0, pg_min(a.cu[j], a.tokens)) : j; };
    start_s[i] = start(i);
    if (i < a.batch) {
      len_s[i] = pg_max(0, pg_min(a.lens[i], PG_MAX_KEYS)), back |= start(i + 1) < start(i);
      first_s[i] = a.joined != nullptr ? a.joined[i] : PG_MAX_KEYS;  // (until the line is formed)
    }
  }
  for (int i = a.n_groups > 0 ? t : 1; i <= a.n_groups; i += SH_THREADS) {
    auto first = [&](int j) { return pg_max(0, pg_min(a.groups[j], a.batch)); };
    group_s[i] = first(i);
    if (i < a.n_groups) shared_s[i] = pg_max(0, pg_min(a.shared[i], room)), back |= first(i + 1) < first(i);
  }
  // (offsets that go back count as the largest in front of them: searches need them in order)
  if (__syncthreads_or(back)) {
    if (t == 0) {
      for (int i = 1; i <= a.batch; ++i) start_s[i] = pg_max(start_s[i], start_s[i - 1]);
      for (int i = 1; i <= a.n_groups; ++i) group_s[i] = pg_max(group_s[i], group_s[i - 1]);
    }
    __syncthreads();
  }
  auto request = [&](int b) {
    ShRequest r = {0, 0, 0, 0, start_s[b], {0, 0, 0}};
    if (a.n_groups > 0) {
      const int i = pg_holder(group_s, a.n_groups, b);
      if (group_s[i] <= b && b < group_s[i + 1]) {
        r.first_own = first_s[b] >= shared_s[i] ? sh_first_own(len_s[b], start_s[b + 1] - r.start, shared_s[i]) : 0;
        r.group = i, r.start0 = start_s[group_s[i]], r.end0 = start_s[group_s[i + 1]];
      }
    }
    return r;
  };
  auto item = [&](int x) {
    ShItem p;
    p.row0 = 0;
    if (x < n_groups) {
      p.table_row = pg_min(group_s[x], a.batch - 1);
      p.start = start_s[group_s[x]];
      p.rows = (start_s[group_s[x + 1]] - p.start) * g;
      p.key0 = 0, p.key1 = shared_s[x], p.pos = PG_MAX_KEYS;
      p.slot = (int)pg_first_slot(p.start, g, x, SH_UNIT);
    } else {
      const int b = x - n_groups, q_len = start_s[b + 1] - start_s[b];
      p.table_row = b;
      p.start = start_s[b];
      p.rows = q_len * g;
      p.key0 = first_s[b], p.key1 = pg_min(len_s[b], room), p.pos = len_s[b] - q_len;
      p.slot = a.shared_slots + (int)sh_own_slot(p.start, g, b, a.dense);
    }
    p.lo = p.key0 / SH_KEYS;
    p.n = p.rows > 0 && p.key1 > p.key0 ? (p.key1 + SH_KEYS - 1) / SH_KEYS - p.lo : 0;
    return p;
  };

  // ---- the line: where every item starts, in the place of the rings ----
  int64_t* const line_s = reinterpret_cast<int64_t*>(lds);  // [items + 1]
  int64_t total = 0;
  {
    int64_t* const sums_s = reinterpret_cast<int64_t*>(lds + SH_SUMS);
    const int per = (items + SH_THREADS - 1) / SH_THREADS, x0 = t * per, x1 = pg_min(x0 + per, items);
    int64_t at = 0;
    for (int x = x0; x < x1; ++x) {
      if (x >= n_groups) {
        const ShRequest r = request(x - n_groups);
        first_s[x - n_groups] = r.first_own;
        if (blockIdx.x == 0) a.of_request[x - n_groups] = r;
      }
      const ShItem p = item(x);
      const int64_t units = sh_units(p.n, p.rows, x < n_groups ? SH_GROUP : a.streams ? SH_STREAM : SH_OWN);
      line_s[x] = at;  // (of the thread's; completed below)
      at += units;
    }
    const int64_t mine = at;
#pragma unroll
    for (int o = 1; o < SP_WAVE; o <<= 1) {
      const int64_t y = __shfl_up(at, o, SP_WAVE);
      if (lane >= o) at += y;
    }
    if (lane == SP_WAVE - 1) sums_s[wave] = at;
    if (blockIdx.x == 0 && t == 0) a.of_request[a.batch] = ShRequest{0, 0, 0, 0, start_s[a.batch], {0, 0, 0}};
    __syncthreads();
    at -= mine;
#pragma unroll
    for (int w = 0; w < 2 * WAVES; ++w) {
      if (w == wave) at += total;
      total += sums_s[w];
    }
    for (int x = x0; x < x1; ++x) line_s[x] += at;
    if (t == 0) line_s[items] = total;
    __syncthreads();
  }
  auto uniform64 = [](int64_t x) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
  };
  total = uniform64(total);
  const int64_t full = (total + SH_MIN_SHARE - 1) / SH_MIN_SHARE;
  const int parts = full < a.parts ? pg_max((int)full, 1) : a.parts, near = pg_near(total, parts);
  // Of the streams the groups alone are the workgroup's matter, else all items are.
  const int shared_items = a.streams ? n_groups : items;
  const int64_t shared_units = uniform64(line_s[shared_items]);
  // Where a unit of the line is: item, tile and step; behind the last one: items.
  struct Place {
    int item, tile, step;
  };
  // What the workgroup begins with and ends in front of, and the same of a wave of the streams: four cuts, sixteen lanes each.  (One after the other
  // they took a wave 1.5 us more.)
  Place places[4];
  {
    const PgCuts cuts = pg_cuts(total, parts);
    int64_t cut = pg_cut_at(cuts, part + (gr & 1));
    const int64_t cut0 = ds_lane64(cut, 0), cut1 = ds_lane64(cut, 16);
    const int64_t own0 = cut0 > shared_units ? cut0 : shared_units, own1 = cut1 > shared_units ? cut1 : shared_units;
    if (gr >= 2) cut = own0 + (own1 - own0) * (slot + gr - 2) / WAVES;
    Place f = {gr < 2 ? shared_items : items, 0, 0};
    const bool wanted = gr < 2 ? cut < shared_units : a.streams && cut < total;
    int lo = 0;  // the item is the last that starts at or in front of the cut, by 16 candidates at a time
    for (int span = items; span > 1;) {
      const int step = (span + 15) / 16, x = lo + lq * step;
      const int n = __builtin_popcount((unsigned)(__ballot(lq * step < span && x < items && line_s[pg_min(x, items)] <= cut) >> (16 * gr)) & 0xffffu);
      lo += pg_max(n - 1, 0) * step;
      span = step;
    }
    const ShItem p = item(lo);
    const int64_t off = cut - line_s[lo];
    if (wanted) {
      f.item = lo;
      if (gr < 2)
        sh_place(off, p.n, p.rows, lo < n_groups ? SH_GROUP : SH_OWN, near, &f.tile, &f.step);
      else
        f.step = sh_stream_step(off, p.n);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      places[e] = {__builtin_amdgcn_readlane(f.item, 16 * e), __builtin_amdgcn_readlane(f.tile, 16 * e), __builtin_amdgcn_readlane(f.step, 16 * e)};
  }
  const Place &from = places[0], &to_place = places[1];
  if (a.streams && half == 0 && kvh == 0 && lane == 0)
    a.cuts[part * WAVES + slot] = make_int4(places[2].item - n_groups, places[2].step, places[3].item - n_groups, places[3].step);

  // Arguments of what is done once an item are read where they are used: scalar registers do not suffice to keep them.
  const auto kernel_args = (const __attribute__((address_space(4))) ShArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  auto args = [&] {
    auto p = kernel_args;
    asm volatile("" : "+s"(p));
    return p;
  };
  const uint32_t k_row = (uint32_t)a.sk_n * 2u, v_row = (uint32_t)a.sv_n * 2u;  // bytes
  const uint32_t rings = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds, ring = rings + slot * NB * Shape::STEP_BYTES;
  const uint32_t k_at = rings + lq * (D * 2);
  const int v_key = 4 * gr + (lq >> 2);  // row of the transposing read; 16 rows further the swizzle is the same
  const uint32_t v_at = rings + Shape::K_BYTES + v_key * (CT * 32) + 8 * (lq & 3);
  float* const m_s = reinterpret_cast<float*>(lds + SH_ML);
  float* const l_s = m_s + SH_MEET;

  const char* const kh = (const char*)(a.k + kvh * a.sk_h);
  const char* const vh = (const char*)(a.v + kvh * a.sv_h);
  struct Ids {
    int id[2];
  };
  auto entries = [&](auto table, int key) {  // pages of a step's halves
    Ids e;
#pragma unroll
    for (int h = 0; h < 2; ++h) e.id[h] = table[pg_min((key + 16 * h) >> a.shift, a.width - 1)];
    return e;
  };
  // The loads of the step at `key`, K's or V's or both, and which of its keys are any: those from key0 to key1 with a page.  The others are zeros, without a
  // read, whatever stands there.
  auto fetch = [&](uint32_t at, int key, int key0, int key1, Ids ids, bool with_k, bool with_v) {
    auto low = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
    uint32_t seen = low(key1 - key) & ~low(key0 - key);
    int64_t id[2];
    int in[2], there[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int first = key + 16 * h;
      const int page = first >> a.shift < a.width && (unsigned)ids.id[h] < (unsigned)a.num_pages ? ids.id[h] : -1;
      in[h] = first & ((1 << a.shift) - 1);
      there[h] = page < 0 ? 0 : pg_max(0, pg_min(key1 - first, 16));
      if (page < 0) seen &= h == 0 ? 0xffff0000u : 0x0000ffffu;
      id[h] = pg_max(page, 0);
    }
    // (formed anew for every step: kept in registers they would crowd out what the loop needs)
    int lane_here = lane;
    asm volatile("" : "+v"(lane_here));
    auto load = [&](const char* from, int64_t page_bytes, uint32_t row_bytes, uint32_t to, auto&& chunk) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(from + id[h] * page_bytes + (uint64_t)(uint32_t)in[h] * row_bytes), 0,
            there[h] > 0 ? (int)((uint32_t)(there[h] - 1) * row_bytes + 2u * D) : 0, 0x00027000);
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
          const int row = i * ROWS + lane_here / CHUNKS;
          uint32_t off = (uint32_t)row * row_bytes + 16u * (uint32_t)chunk(16 * h + row);
          off = (seen >> (16 * h + row)) & 1u ? off : 0x7ffffff0u;  // (past the buffer's end: zeros)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ds_lds_ptr)(uintptr_t)(to + (h * HALF + i) * 1024), 16, (int)off, 0, 0, 0);
        }
      }
    };
    if (with_k) load(kh, a.sk_p * 2, k_row, at, [&](int row) { return (lane_here % CHUNKS) ^ ds_swz_k<D>(row); });
    if (with_v) load(vh, a.sv_p * 2, v_row, at + Shape::K_BYTES, [&](int row) { return (lane_here % CHUNKS) ^ (2 * ds_swz_v<CT>(row)); });
    return seen;
  };
  // One step of a wave's rows, RT tiles of 16: its operands lie at `off` of the rings, its first key is `key`, `mine` says which are seen; partly: some rows
  // do not see some of them, those behind pos.  m, l: the rows' maxima, and the sums of this lane group's keys.  logits(sc) is called with the logits.
  auto attend = [&](auto tiles, uint32_t off, int key, uint32_t mine, auto& qb, auto& pos, bool partly, auto& o, auto& m, auto& l, auto&& logits) {
    constexpr int RT = decltype(tiles)::value;
    dc_u32x4 kr[2][KS];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t at = k_at + off + (((4 * ks + gr) ^ ds_swz_k<D>(lq)) << 4);  // (16 rows further the swizzle is the same)
        kr[i][ks] = i == 0 ? sh_read_k<0>(at) : sh_read_k<16 * D * 2>(at);
      }
    if constexpr (KS == 4)
      asm volatile("s_waitcnt lgkmcnt(0)"
                   : "+v"(kr[0][0]), "+v"(kr[0][1]), "+v"(kr[0][2]), "+v"(kr[0][3]), "+v"(kr[1][0]), "+v"(kr[1][1]), "+v"(kr[1][2]), "+v"(kr[1][3]));
    else
      asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(kr[0][0]), "+v"(kr[0][1]), "+v"(kr[1][0]), "+v"(kr[1][1]));
    ds_floatx4 sc[RT][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        sc[rt][i] = (ds_floatx4){0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          sc[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, kr[i][ks]), qb[rt][ks], sc[rt][i], 0, 0, 0);
      }
    const uint32_t bits = mine >> (4 * gr);  // the lane's keys: 16 i + 4 gr + j
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[rt][i][j] *= a.scale_log2;
    if (mine != ~0u) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[rt][i][j] = bits & (1u << (16 * i + j)) ? sc[rt][i][j] : -INFINITY;
    }
    if (partly) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[rt][i][j] = key + 4 * gr + 16 * i + j <= pos[rt] ? sc[rt][i][j] : -INFINITY;
    }
    logits(sc);
    float mx[RT];
    bool moves = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      mx[rt] = fmaxf(fmaxf(fmaxf(sc[rt][0][0], sc[rt][0][1]), fmaxf(sc[rt][0][2], sc[rt][0][3])),
                     fmaxf(fmaxf(sc[rt][1][0], sc[rt][1][1]), fmaxf(sc[rt][1][2], sc[rt][1][3])));
      moves |= mx[rt] > m[rt] + SH_SLACK;
    }
    // (the lanes of a row need its maximum only where one of them finds that it moves; a row that has seen no finite logit: m is -inf, every weight
    // exp2(-inf) = 0)
    if (__ballot(moves) != 0ull) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float to = fmaxf(m[rt], ds_quad_max(mx[rt])), alpha = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[rt] - to);
        m[rt] = to;
        l[rt] *= alpha;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[rt][ct] *= alpha;
      }
    }
    // V is asked for here, under the exponentials: no branch lies between these reads and the wait for them
    ds_u32x2 vr[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const uint32_t at = v_at + off + ((ct ^ ds_swz_v<CT>(v_key)) << 5);
      vr[ct][0] = ds_read_v<0>(at);
      vr[ct][1] = ds_read_v<16 * CT * 32>(at);
    }
    // Probabilities enter the product as two bf16 values: what truncation leaves of them, and the rest, of at least 2^-23 of the probability: an infinite value
    // has met its weight in the first product, and zero or a negative number times infinity would make a NaN of the sum.
    dc_bf16x8 ph[RT], pl[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float base = m[rt] == -INFINITY ? 0.f : m[rt];
      uint32_t hi[4], lw[4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const float p0 = __builtin_amdgcn_exp2f(sc[rt][i][j] - base), p1 = __builtin_amdgcn_exp2f(sc[rt][i][j + 1] - base);
          const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
          hi[2 * i + j / 2] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
          l[rt] += p0 + p1;
          lw[2 * i + j / 2] = dc_pack2(fmaf(p0, 0x1.000002p0f, -__uint_as_float(b0 & 0xffff0000u)), fmaf(p1, 0x1.000002p0f, -__uint_as_float(b1 & 0xffff0000u)));
        }
      ph[rt] = __builtin_bit_cast(dc_bf16x8, (dc_u32x4){hi[0], hi[1], hi[2], hi[3]});
      pl[rt] = __builtin_bit_cast(dc_bf16x8, (dc_u32x4){lw[0], lw[1], lw[2], lw[3]});
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(vr[ct][0]), "+v"(vr[ct][1]));
    // Where a row does not see a key, 0 times a value that is no number would make a NaN of its sum: the product takes zeros in such places, and rows
    // that do see such a key have a sum of weights that is none.
    if (partly) {
      uint32_t odd[2] = {0u, 0u};  // exponents of ones, of the lane's keys 16 h + 4 gr + 0 .. 3: bits 15, 31 of words 0 and 1
      uint32_t any = 0u;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) any |= ((vr[ct][h][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      if (__ballot(any != 0u) != 0ull) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t here = 0u;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              const uint32_t ones = ((vr[ct][h][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
              here |= ones;
              vr[ct][h][e] &= ~((ones >> 15) * 0xffffu);
            }
            odd[h] |= here >> (15 * e);  // (keys 2 e and 2 e + 1: bits 15 - 15 e and 31 - 15 e)
          }
        uint32_t met = 0u;  // the lane's rows see such a key (bits)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int by = 1; by < 16; by <<= 1) odd[h] |= __shfl_xor(odd[h], by, SP_WAVE);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((odd[h] >> (15 - 15 * (j >> 1) + 16 * (j & 1))) & 1u) {
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                if (key + 16 * h + 4 * gr + j <= pos[rt]) met |= 1u << rt;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          if ((met >> rt) & 1u) l[rt] *= __builtin_nanf("");
      }
    }
    auto weigh = [&](const dc_bf16x8 (&p)[RT]) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          o[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, __builtin_shufflevector(vr[ct][0], vr[ct][1], 0, 1, 2, 3)),
                                                              p[rt], o[rt][ct], 0, 0, 0);
    };
    weigh(ph), weigh(pl);
  };

  // A tile's steps: wave w has rows 32 (w / share) .. of the tile and of a block's four steps w % share, + share, ..; it fills K's or V's half of ring
  // w % 4, and all meet twice in a block.
  auto run = [&](const ShItem& p, int begin, int s_end, bool of_group) {
    constexpr int RT = 2;
    const int tile = sh_tile(p.rows - p.row0), share = SH_MEET / tile;  // (as few rows as there are: waves without any would only wait)
    const int mine_of = wave & (share - 1), tile_row = 32 * (wave / share);
    auto row_of = [&](int in_tile, int* token, int* head) {
      const int r = pg_min(p.row0 + in_tile, p.rows - 1);
      *token = (int)pg_div((unsigned)r, a.by_group);
      *head = kvh * g + (r - *token * g);
    };
    dc_bf16x8 qb[RT][KS];
    int pos[RT];  // last key that the lane's rows see
    {
      const auto r = args();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        int token, head;
        row_of(tile_row + 16 * rt + lq, &token, &head);
        pos[rt] = p.pos + token;
        const sp_bf16* src = r->q + (int64_t)(p.start + token) * r->sq_n + (int64_t)head * r->sq_h + 8 * gr;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qb[rt][ks] = *reinterpret_cast<const dc_bf16x8*>(src + 32 * ks);
      }
    }
    const int pos0 = p.pos + (int)pg_div((unsigned)p.row0, a.by_group);  // of the tile's first row
    // (scalar loads: nothing writes the table during the launch)
    const auto table = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(a.table + (int64_t)p.table_row * a.table_stride);
    auto key_of = [&](int step) { return (p.lo + step) * SH_KEYS; };
    ds_floatx4 o[RT][CT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[rt][ct] = (ds_floatx4){0, 0, 0, 0};
      m[rt] = -INFINITY, l[rt] = 0.f;
    }

    __syncthreads();  // the rings are free
    // The ring holds NB steps; a step's place is filled again when its operands have been read.  The first NB rounds do nothing but fill.
    constexpr int MINE = Shape::LOADS / 2;  // loads of the wave for a step
    const int s0 = begin + slot;
    const bool has_rows = p.row0 + tile_row < p.rows;
    // which keys of a step are any: the wave that fetches it leaves a word for all (LDS accesses of its own: the compiler would wait for all loads in flight
    // in front of them)
    const uint32_t seen_at = rings + SH_SEEN;
    auto any_of = [&](int j, int of_buf) {
      uint32_t v;
      asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(v) : "v"(seen_at + 4u * (uint32_t)(j * NB + of_buf)));
      return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
    };
    Ids next[NB];  // pages of the wave's step of the blocks to come
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (s0 + i * WAVES < s_end) next[i] = entries(table, key_of(s0 + i * WAVES));
    int buf = 0;
    for (int s = s0 - NB * WAVES; s - slot < s_end; s += WAVES) {
      if (s >= begin) {
        // the block's loads have landed, those of the NB - 1 behind it stay in flight (what is asked for returns in order)
        if (s + (NB - 1) * WAVES < s_end)
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 1) * MINE) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (has_rows) {
          for (int j = mine_of; j < WAVES && s - slot + j < s_end; j += share) {
            const int key = key_of(s - slot + j);
            // (uniform: some row does not see a key that others see)
            attend(std::integral_constant<int, RT>{}, (j * NB + buf) * Shape::STEP_BYTES, key, any_of(j, buf), qb, pos, pg_min(key + SH_KEYS, p.key1) - 1 > pos0,
                   o, m, l, [](ds_floatx4 (&)[RT][2]) {});
          }
        }
        asm volatile("s_barrier" ::: "memory");  // the others have read them too
      }
      const int ahead = s + NB * WAVES;
      if (ahead < s_end) {
        const uint32_t seen = fetch(ring + buf * Shape::STEP_BYTES, key_of(ahead), p.key0, p.key1, next[0], half == 0, half == 1);
        if (half == 0) asm volatile("ds_write_b32 %0, %1" ::"v"(seen_at + 4u * (uint32_t)(slot * NB + buf)), "v"(seen) : "memory");
      }
#pragma unroll
      for (int i = 0; i + 1 < NB; ++i) next[i] = next[i + 1];
      if (ahead + NB * WAVES < s_end) next[NB - 1] = entries(table, key_of(ahead + NB * WAVES));
      buf = buf + 1 == NB ? 0 : buf + 1;
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = ds_quad_sum(l[rt]);
    __syncthreads();  // the rings are free
    // [share][tile][D] floats, 16-byte pieces swizzled by the row
    float* const o_s = reinterpret_cast<float*>(lds);
    {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = mine_of * tile + tile_row + 16 * rt + lq;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<ds_floatx4*>(o_s + r * D + ((4 * ct + gr) ^ lq) * 4) = o[rt][ct];
        if (gr == 0) m_s[r] = m[rt], l_s[r] = l[rt];
      }
    }
    __syncthreads();
    const auto to_args = args();
    const bool whole = begin == 0 && s_end == p.n;
    const int rows = pg_min(p.rows - p.row0, tile);
    const int64_t slab = ((int64_t)(part * a.hkv + kvh) * 2 + (begin == 0 ? 1 : 0)) * SH_ROWS;
    const bool final = whole && p.key0 == 0 && !of_group;
    for (int i = t; i < rows * (D / 4); i += SH_THREADS) {
      const int r = i / (D / 4), c = i % (D / 4);
      float top = -INFINITY, sum = 0.f;
      for (int w = 0; w < share; ++w) top = fmaxf(top, m_s[w * tile + r]);
      ds_floatx4 acc = {0, 0, 0, 0};
      for (int w = 0; w < share; ++w) {
        const float mw = m_s[w * tile + r];
        const float f = mw == -INFINITY && l_s[w * tile + r] == 0.f ? 0.f : __builtin_amdgcn_exp2f(mw - top);  // (a wave without keys: 0)
        sum += l_s[w * tile + r] * f;
        acc += *reinterpret_cast<const ds_floatx4*>(o_s + (w * tile + r) * D + (c ^ (r & 15)) * 4) * f;
      }
      int token, head;
      row_of(r, &token, &head);
      const int64_t row = (int64_t)(p.start + token) * (a.hkv * g) + head;
      if (final) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // (a row without keys: zeros)
        *reinterpret_cast<uint2*>(to_args->out + row * D + 4 * c) = make_uint2(dc_pack2(acc[0] * inv, acc[1] * inv), dc_pack2(acc[2] * inv, acc[3] * inv));
      }
      if (!final || a.weights != nullptr) {
        const int64_t to = whole ? (of_group ? 0 : (int64_t)a.tokens * (a.hkv * g)) + row : slab + r;
        if (!final) *reinterpret_cast<ds_floatx4*>((whole ? to_args->o_row : to_args->o_part) + to * D + 4 * c) = acc;
        if (c == 0) (whole ? to_args->ml_row : to_args->ml_part)[to] = make_float2(fmaxf(top, CK_NO_MAX), sum);
      }
    }
  };

  for (int x = from.item, first_tile = from.tile, begin = from.step; x < shared_items && x <= to_place.item; ++x, first_tile = 0, begin = 0) {
    ShItem p = item(x);
    if (p.n == 0) continue;
    // (uniform: out of vector registers)
    p.table_row = __builtin_amdgcn_readfirstlane(p.table_row), p.start = __builtin_amdgcn_readfirstlane(p.start);
    p.rows = __builtin_amdgcn_readfirstlane(p.rows), p.key0 = __builtin_amdgcn_readfirstlane(p.key0);
    p.pos = __builtin_amdgcn_readfirstlane(p.pos), p.lo = __builtin_amdgcn_readfirstlane(p.lo), p.n = __builtin_amdgcn_readfirstlane(p.n);
    p.slot = __builtin_amdgcn_readfirstlane(p.slot);
    const int key1 = __builtin_amdgcn_readfirstlane(p.key1);
    const int tile = sh_tile(p.rows);
    for (int at = first_tile; at * tile < p.rows; ++at, begin = 0) {
      if (x == to_place.item && at > to_place.tile) break;
      const int end = x == to_place.item && at == to_place.tile ? pg_min(to_place.step, p.n) : p.n;
      if (begin >= end) continue;
      p.row0 = at * tile;
      // (of a request's tile: up to its last row's position)
      p.key1 = x < n_groups ? key1 : pg_min(key1, p.pos + (int)pg_div((unsigned)(pg_min(p.row0 + tile, p.rows) - 1), a.by_group) + 1);
      if (kvh == 0 && t == 0) {
        if (begin == 0) a.parts_of[p.slot + p.row0 / SH_UNIT].x = part;
        if (end == p.n) a.parts_of[p.slot + p.row0 / SH_UNIT].y = part;
      }
      run(p, begin, end, x < n_groups);
    }
  }
  if (!a.streams) return;

  // ---- single tokens over their own keys, a wave by itself ----
  __syncthreads();  // the rings are free
  if (half != 0) return;
  const int b0 = places[2].item - n_groups, b1 = places[3].item - n_groups, step0 = places[2].step, step1 = places[3].step, wave_part = part * WAVES + slot;
  struct At {  // a step of request b (b = batch: none is left): steps up to `end` of its n fall to the wave
    int b, s, end, n, lo, key0, key1, weigh0;
  };
  auto settle = [&](At& x) {
    for (;; ++x.b, x.s = 0) {
      if (x.b >= a.batch || x.b > b1 || (x.b == b1 && step1 == 0)) {
        x.b = a.batch;
        return;
      }
      x.key0 = __builtin_amdgcn_readfirstlane(first_s[x.b]), x.key1 = pg_min(__builtin_amdgcn_readfirstlane(len_s[x.b]), room);
      x.lo = x.key0 / SH_KEYS, x.n = x.key1 > x.key0 ? (x.key1 + SH_KEYS - 1) / SH_KEYS - x.lo : 0;  // (as in item)
      x.end = x.b == b1 ? pg_min(step1, x.n) : x.n;
      const auto weigh_from = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)args()->weigh_from;
      x.weigh0 = weigh_from != nullptr ? weigh_from[x.b] : 0;
      if (x.s < x.end) return;
    }
  };
  auto key_of = [](const At& x) { return (x.lo + x.s) * SH_KEYS; };
  auto table_of = [&](int b) { return (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(a.table + (int64_t)b * a.table_stride); };
  struct Step {  // on its way, or about to be computed on
    int b, key;
    uint32_t seen;
    Ids ids;  // pages of halves that hold keys to be weighed, else -1
    bool first, last, from_start, to_end, alone;  // of the wave's steps of the request; they begin with its first, end with its last; no shared keys
  };
  At ahead = {b0, step0, 0, 0, 0, 0, 0, 0};
  settle(ahead);
  Ids ids = {{0, 0}};
  if (ahead.b < a.batch) ids = entries(table_of(ahead.b), key_of(ahead));
  auto push = [&](int buf) {
    Step x = {a.batch, 0, 0u, {{0, 0}}, false, false, false, false, false};
    if (ahead.b < a.batch) {
      const int key = key_of(ahead);
      const bool from_start = ahead.b != b0 || step0 == 0;
      x = {ahead.b, key, fetch(ring + buf * Shape::STEP_BYTES, key, ahead.key0, ahead.key1, ids, true, true), ids,
           ahead.s == (from_start ? 0 : step0), ahead.s + 1 == ahead.end, from_start, ahead.end == ahead.n, ahead.key0 == 0};
      // (no page: no key is seen.  The logits' scratch goes by places in the pages: what lies in front of the weighed keys may be several requests')
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (((x.seen >> (16 * i)) & 0xffffu) == 0u || key + 16 * i + 16 <= ahead.weigh0) x.ids.id[i] = -1;
      if (++ahead.s >= ahead.end) {
        ++ahead.b, ahead.s = 0;
        settle(ahead);
      }
      if (ahead.b < a.batch) ids = entries(table_of(ahead.b), key_of(ahead));
    }
    return x;
  };
  dc_bf16x8 qb[1][KS], q_next[KS];
  auto load_q = [&](int b) {
    const auto r = args();
    const sp_bf16* src = r->q + (int64_t)b * r->sq_n + (int64_t)(kvh * g + pg_min(lq, g - 1)) * r->sq_h + 8 * gr;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q_next[ks] = *reinterpret_cast<const dc_bf16x8*>(src + 32 * ks);
  };
  if (ahead.b < a.batch) load_q(ahead.b);
  Step queue[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) queue[i] = {-1, 0, 0u, {{0, 0}}, false, false, false, false, false};  // (the first NB rounds do nothing but fill)
  ds_floatx4 o[1][CT];
  float m[1], l[1];
  int pos[1] = {0};
  int buf = 0;
  bool wrote = false;  // at least CT stores are younger than all loads
  while (queue[0].b < a.batch) {
    const Step now = queue[0];
    if (now.b >= 0) {
      // the step's loads have landed, those of the NB - 1 behind it stay in flight (what is asked for returns in order)
      if (queue[NB - 1].b >= a.batch)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if (wrote)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 1) * Shape::LOADS + CT) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 1) * Shape::LOADS) : "memory");
      if (now.first) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qb[0][ks] = q_next[ks];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[0][ct] = (ds_floatx4){0, 0, 0, 0};
        m[0] = -INFINITY, l[0] = 0.f;
      }
        if (queue[1].b < a.batch && queue[1].first) load_q(queue[1].b);
      attend(
          std::integral_constant<int, 1>{}, (slot * NB + buf) * Shape::STEP_BYTES, now.key, now.seen, qb, pos, false, o, m, l,
          [&](ds_floatx4 (&sc)[1][2]) {
            if (a.weights == nullptr || lq >= g) return;  // the logits themselves, for the keys' weights
            float* const to = args()->logits;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (now.ids.id[i] >= 0)
                *reinterpret_cast<ds_floatx4*>(to + ((((int64_t)now.ids.id[i] * a.hkv + kvh) * g + lq) << a.shift) + ((now.key + 16 * i + 4 * gr) & ((1 << a.shift) - 1))) = sc[0][i];
          });
    }
#pragma unroll
    for (int i = 0; i + 1 < NB; ++i) queue[i] = queue[i + 1];
    queue[NB - 1] = push(buf);
    wrote = now.b >= 0 && now.last;
    if (wrote) {
      const auto r = args();
      const float sum = ds_quad_sum(l[0]);
      const int64_t row = (int64_t)now.b * (a.hkv * g) + kvh * g + lq;
      const bool whole = now.from_start && now.to_end, final = whole && now.alone;
      if (lq < g) {
        if (final) {
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            *reinterpret_cast<uint2*>(r->out + row * D + 16 * ct + 4 * gr) =
                make_uint2(dc_pack2(o[0][ct][0] * inv, o[0][ct][1] * inv), dc_pack2(o[0][ct][2] * inv, o[0][ct][3] * inv));
        }
        if (!final || a.weights != nullptr) {
          const int64_t to = whole ? (int64_t)a.tokens * (a.hkv * g) + row : ((int64_t)(wave_part * a.hkv + kvh) * 2 + (now.from_start ? 1 : 0)) * 16 + lq;
          if (!final) {
            float* const dst = (whole ? r->o_row : r->o_stream) + to * D + 4 * gr;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<ds_floatx4*>(dst + 16 * ct) = o[0][ct];
          }
          if (gr == 0) (whole ? r->ml_row : r->ml_stream)[to] = make_float2(fmaxf(m[0], CK_NO_MAX), sum);
        }
      }
      if (kvh == 0 && lane == 0) {
        if (now.from_start) r->parts_of[a.shared_slots + now.b].x = wave_part;
        if (now.to_end) r->parts_of[a.shared_slots + now.b].y = wave_part;
      }
    }
    buf = buf + 1 == NB ? 0 : buf + 1;
  }
}

// ---- joining ----------------------------------------------------------------------------------------------------
// The number of a row's tile (group, or request), and the row's place in it.
struct ShRow {
  int slot, in_tile;
};
__device__ __forceinline__ ShRow sh_group_row(const ShArgs& a, const ShRequest& r, int token, int h) {
  const int row = (token - r.start0) * a.group + h, first = row & -sh_tile((r.end0 - r.start0) * a.group);
  return ShRow{(int)pg_first_slot(r.start0, a.group, r.group, SH_UNIT) + first / SH_UNIT, row - first};
}
__device__ __forceinline__ ShRow sh_own_row(const ShArgs& a, const ShRequest& r, int end, int b, int token, int h) {
  const int row = (token - r.start) * a.group + h, first = row & -sh_tile((end - r.start) * a.group);
  return ShRow{a.shared_slots + (int)sh_own_slot(r.start, a.group, b, a.dense) + first / SH_UNIT, row - first};
}
// Parts that hold some of it: (0, -1) where there are no keys.
__device__ __forceinline__ int2 sh_group_parts(const ShArgs& a, const ShRequest& r, const ShRow& row) {
  return r.first_own == 0 ? make_int2(0, -1) : a.apart ? make_int2(0, 0) : a.parts_of[row.slot];
}
__device__ __forceinline__ int2 sh_own_parts(const ShArgs& a, const ShRequest& r, int b, const ShRow& row) {
  return pg_min(a.lens[b], a.width << a.shift) > r.first_own ? a.parts_of[row.slot] : make_int2(0, -1);
}
// Where part i of a tile that parts.x .. parts.y hold stands: in o_row and ml_row where there is but one, else in o_part and ml_part.
__device__ __forceinline__ int64_t sh_slab(const ShArgs& a, int2 parts, int i, int kvh, int in_tile, int rows) {
  return ((int64_t)((parts.x + i) * a.hkv + kvh) * 2 + (i == 0 ? 1 : 0)) * rows + in_tile;
}

#define SM_THREADS 256
// A row's parts joined: D / 4 threads a row, SETS of them that take every so many parts, on a running maximum of their own, and meet in LDS.
template <int D, int SETS>
__device__ __forceinline__ void sh_join(const ShArgs& a) {
  constexpr int WIDTH = D / 4, PER = SM_THREADS / (WIDTH * SETS), AHEAD = 4;
  __shared__ float2 ml_s[SETS][PER];
  __shared__ __attribute__((aligned(16))) float o_s[SETS > 1 ? SETS : 1][SETS > 1 ? PER : 1][D];
  const int t = threadIdx.x, hq = a.hkv * a.group, c = t % WIDTH * 4, in_block = t / WIDTH % PER, set = t / (WIDTH * PER);
  const unsigned row = blockIdx.x * PER + in_block;
  const unsigned rows = (unsigned)a.tokens * (unsigned)hq;
  const int token = (int)(pg_min((int)row, (int)rows - 1) / hq), head = pg_min((int)row, (int)rows - 1) - token * hq, kvh = (int)pg_div((unsigned)head, a.by_group);
  int b = token;
  if (a.cu != nullptr) {
    b = 0;
    int hi = a.batch;
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (a.of_request[mid].start <= token)
        b = mid;
      else
        hi = mid;
    }
  }
  const ShRequest r = a.of_request[b];
  const int end = a.of_request[b + 1].start, h = head - kvh * a.group;
  const ShRow own = sh_own_row(a, r, end, b, token, h), group = sh_group_row(a, r, token, h);
  bool wanted = row < rows && token >= r.start && token < end;  // (a row outside every request)
  int2 own_parts = make_int2(0, -1), group_parts = own_parts;
  if (wanted) own_parts = sh_own_parts(a, r, b, own), group_parts = sh_group_parts(a, r, group);
  if (r.first_own == 0 && own_parts.x == own_parts.y) wanted = false, own_parts.y = own_parts.x - 1;  // (the row is done)
  float top = CK_NO_MAX, sum = 0.f;
  ds_floatx4 acc = {0, 0, 0, 0};
  auto add = [&](const ShRow& it, int2 parts, bool of_group) {
    const int count = parts.y - parts.x + 1;
    const bool stream = !of_group && a.streams;
    const float2* const ml_from = count == 1 ? a.ml_row : stream ? a.ml_stream : a.ml_part;
    const float* const o_from = count == 1 ? a.o_row : stream ? a.o_stream : a.o_part;
    for (int i0 = set; i0 < count; i0 += SETS * AHEAD) {
      float2 ml[AHEAD];
      ds_floatx4 o[AHEAD];
      float to = top;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = pg_min(i0 + u * SETS, count - 1);
        const int64_t at = count > 1 ? sh_slab(a, parts, i, kvh, it.in_tile, stream ? 16 : SH_ROWS) : (of_group ? 0 : (int64_t)a.tokens * hq) + row;
        ml[u] = ml_from[at];
        o[u] = *reinterpret_cast<const ds_floatx4*>(o_from + at * D + c);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) to = fmaxf(to, ml[u].x);
      const float before = __builtin_amdgcn_exp2f(top - to);
      top = to;
      sum *= before;
      acc *= before;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (i0 + u * SETS < count) {
          const float f = __builtin_amdgcn_exp2f(ml[u].x - top);
          sum += ml[u].y * f;
          acc += o[u] * f;
        }
    }
  };
  add(group, group_parts, true);
  add(own, own_parts, false);
  if constexpr (SETS > 1) {
    *reinterpret_cast<ds_floatx4*>(&o_s[set][in_block][c]) = acc;
    if (c == 0) ml_s[set][in_block] = make_float2(top, sum);
    __syncthreads();
    if (set > 0) return;
    for (int i = 0; i < SETS; ++i) top = fmaxf(top, ml_s[i][in_block].x);
    sum = 0.f, acc = (ds_floatx4){0, 0, 0, 0};
    for (int i = 0; i < SETS; ++i) {
      const float f = __builtin_amdgcn_exp2f(ml_s[i][in_block].x - top);
      sum += ml_s[i][in_block].y * f;
      acc += *reinterpret_cast<const ds_floatx4*>(&o_s[i][in_block][c]) * f;
    }
  }
  if (!wanted) return;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  *reinterpret_cast<uint2*>(a.out + (int64_t)row * D + c) = make_uint2(dc_pack2(acc[0] * inv, acc[1] * inv), dc_pack2(acc[2] * inv, acc[3] * inv));
}

// Weights of the own keys that fell to wave's part w / hkv of kv head w % hkv (single tokens):
//   weight[j] += sum over the group's heads of 2^(logit - m) / l.
__device__ __forceinline__ void sh_weigh(const ShArgs& a, int w) {
  const int t = threadIdx.x, lane = t & 63, hq = a.hkv * a.group, kvh = w % a.hkv, part = w / a.hkv;
  const int4 cut = a.cuts[part];
  const int room = a.width << a.shift;
  // the part's requests side by side: for each all waves, two or one (each is a chain of six loads: 12 us one after the other)
  const int b0 = pg_max(cut.x, 0), span = pg_min(cut.w > 0 ? cut.z : cut.z - 1, a.batch - 1) - b0 + 1;
  const int waves = span <= 1 ? SM_THREADS / SP_WAVE : span == 2 ? SM_THREADS / SP_WAVE / 2 : 1, threads = waves * SP_WAVE;
  for (int i = __builtin_amdgcn_readfirstlane(t / threads); i < span; i += SM_THREADS / threads) {
    const int b = b0 + i;
    const ShRequest r = a.of_request[b];
    const int len = pg_max(0, pg_min(a.lens[b], PG_MAX_KEYS));
    const int lo = r.first_own / SH_KEYS, keys = pg_min(len, room);
    const int begin = b == cut.x ? cut.y : 0, end = b == cut.z ? cut.w : PG_MAX_KEYS / SH_KEYS;
    const int weigh0 = a.weigh_from != nullptr ? pg_max(a.weigh_from[b], r.first_own) : r.first_own;
    if (keys <= weigh0 || begin >= end) continue;
    // Maxima and sums of the group's heads, by every wave for itself: lane 16 q + h takes every fourth part of head h from q on.
    float top = CK_NO_MAX, inv = 0.f;
    {
      const int h = pg_min(lane & 15, a.group - 1);
      const ShRow own = sh_own_row(a, r, r.start + 1, b, b, h), group = sh_group_row(a, r, b, h);
      const int2 own_parts = sh_own_parts(a, r, b, own), group_parts = sh_group_parts(a, r, group);
      float sum = 0.f;
      auto add = [&](int in_tile, int2 held, bool of_group) {
        const int count = held.y - held.x + 1;
        for (int i0 = lane >> 4; i0 < count; i0 += 16) {
          float2 ml[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            ml[u] = count > 1 ? (of_group ? a.ml_part : a.ml_stream)[sh_slab(a, held, pg_min(i0 + 4 * u, count - 1), kvh, in_tile, of_group ? SH_ROWS : 16)]
                              : a.ml_row[(of_group ? 0 : (int64_t)a.tokens * hq) + (int64_t)b * hq + kvh * a.group + h];
          float to = top;
#pragma unroll
          for (int u = 0; u < 4; ++u) to = fmaxf(to, ml[u].x);
          sum *= __builtin_amdgcn_exp2f(top - to);
          top = to;
#pragma unroll
          for (int u = 0; u < 4; ++u) sum += i0 + 4 * u < count ? ml[u].y * __builtin_amdgcn_exp2f(ml[u].x - top) : 0.f;
        }
      };
      add(group.in_tile, group_parts, true);
      add(own.in_tile, own_parts, false);
#pragma unroll
      for (int by = 16; by < SP_WAVE; by <<= 1) {
        const float top1 = __shfl_xor(top, by, SP_WAVE), sum1 = __shfl_xor(sum, by, SP_WAVE), to = fmaxf(top, top1);
        sum = sum * __builtin_amdgcn_exp2f(top - to) + sum1 * __builtin_amdgcn_exp2f(top1 - to);
        top = to;
      }
      inv = sum == 0.f ? 0.f : 1.0f / sum;
    }
    const int first = pg_max((lo + begin) * SH_KEYS, weigh0 / SH_KEYS * SH_KEYS), last = (int)pg_min((int)(lo + end < keys / SH_KEYS + 1 ? (lo + end) * SH_KEYS : keys), keys);
    // (all lanes go through the loop together: they hold the heads' maxima and sums for each other)
    for (int at = first; at < last; at += 4 * threads) {
      const int key = at + 4 * (t % threads), in = key & ((1 << a.shift) - 1), page = pg_min(key >> a.shift, a.width - 1);
      int id = a.table[b * a.table_stride + page];
      const bool there = key < last && (unsigned)id < (unsigned)a.num_pages;
      id = there ? id : 0;
      const float* const from = a.logits + ((((int64_t)id * a.hkv + kvh) * a.group) << a.shift) + in;
      ds_floatx4 sum = {0, 0, 0, 0};
      for (int h0 = 0; h0 < a.group; h0 += 4) {
        ds_floatx4 s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = *reinterpret_cast<const ds_floatx4*>(from + ((int64_t)pg_min(h0 + u, a.group - 1) << a.shift));
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (h0 + u < a.group) {
            const float m = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), h0 + u));
            const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inv), h0 + u));
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += __builtin_amdgcn_exp2f(s[u][j] - m) * f;
          }
      }
      if (!there) continue;
      float* const to = a.weights + id * a.sw_p + kvh * a.sw_h + in;
      if (a.weights_by_four && key >= weigh0 && key + 4 < len && key + 4 <= last) {
        *reinterpret_cast<ds_floatx4*>(to) += sum;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key + j >= weigh0 && key + j < last) to[j] = (key + j == len - 1 ? 0.f : to[j]) + sum[j];  // (the newest key's starts here)
      }
    }
  }
}

// The workgroups behind the joining ones, where weights are kept: one for every wave's part of the line.
template <int D, int SETS>
__global__ __launch_bounds__(SM_THREADS) void sp_shared_join_kernel(const ShArgs a, int join_blocks) {
  if ((int)blockIdx.x < join_blocks)
    sh_join<D, SETS>(a);
  else
    sh_weigh(a, (int)blockIdx.x - join_blocks);
}

// ---- host -------------------------------------------------------------------------------------------------
#define SH_PLACES 256  // workgroups that are resident at once: one a CU
static int sh_workgroups(int64_t hkv) { return hkv < SH_PLACES ? SH_PLACES / (int)hkv : 1; }  // of a kv head

struct ShSizes {
  int64_t shared_slots, slots, logits;
  size_t o_part, ml_part, o_stream, ml_stream, o_row, ml_row, parts_of, cuts, of_request, bytes;
};
static ShSizes sh_sizes(int64_t tokens, int64_t batch, int64_t groups, int64_t hq, int64_t hkv, int64_t d, bool single, int64_t pool_keys, bool apart) {
  ShSizes s;
  const int64_t g = hq / hkv;
  s.shared_slots = groups > 0 && !apart ? tokens * g / SH_UNIT + groups : 0;
  s.slots = s.shared_slots + (single && g <= SH_UNIT ? batch : tokens * g / SH_UNIT + batch);
  const int64_t rows = (int64_t)sh_workgroups(hkv) * hkv * 2 * SH_ROWS;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  // (the groups' partials are joined before those of the requests are written)
  s.o_part = take(apart ? ck_groups_workspace_bytes((int)hkv, (int)d) : (size_t)rows * d * sizeof(float));
  s.ml_part = take((size_t)rows * sizeof(float2));
  const bool streams = single && g <= PD_MAX_GROUP;
  const int64_t stream_rows = streams ? (int64_t)sh_workgroups(hkv) * hkv * SH_WAVES * 2 * PD_MAX_GROUP : 0;
  s.o_stream = take((size_t)stream_rows * d * sizeof(float));
  s.ml_stream = take((size_t)stream_rows * sizeof(float2));
  s.o_row = take(groups > 0 ? (size_t)(2 * tokens * hq) * d * sizeof(float) : 0);
  s.ml_row = take((size_t)(2 * tokens * hq) * sizeof(float2));
  s.parts_of = take((size_t)s.slots * sizeof(int2));
  s.cuts = take((size_t)sh_workgroups(hkv) * SH_WAVES * sizeof(int4));
  s.of_request = take((size_t)(batch + 1) * sizeof(ShRequest));
  s.logits = (int64_t)take((size_t)pool_keys * hq * sizeof(float));
  s.bytes = at;
  return s;
}
static bool sh_shape_ok(int64_t tokens, int64_t batch, int64_t groups, int64_t hq, int64_t hkv, int64_t d) {
  return tokens > 0 && batch > 0 && batch <= SH_MAX_SEQS && groups >= 0 && groups <= batch && hq > 0 && hkv > 0 && hq % hkv == 0 && (d == 64 || d == 128) &&
         tokens <= PG_MAX_KEYS && hq <= 65536 && tokens * hq < (1ll << 31);
}

extern "C" size_t sp_shared_attn_workspace_bytes(int64_t tokens, int32_t batch, int32_t groups, int32_t hq, int32_t hkv, int32_t d, int32_t single_tokens,
                                                 int64_t pool_keys) {
  if (!sh_shape_ok(tokens, batch, groups, hq, hkv, d) || pool_keys < 0 || pool_keys > (1ll << 40)) return 0;
  const size_t one = sh_sizes(tokens, batch, groups, hq, hkv, d, single_tokens != 0, pool_keys, false).bytes;
  if (!sh_may_be_apart(tokens, groups, hq / hkv, pool_keys > 0)) return one;
  const size_t apart = sh_sizes(tokens, batch, groups, hq, hkv, d, single_tokens != 0, pool_keys, true).bytes;
  return one > apart ? one : apart;
}

extern "C" int sp_shared_attn_bf16(const sp_shared_attn_args* x) { return sp_shared_attn_from_bf16(x, nullptr); }

extern "C" int sp_shared_attn_from_bf16(const sp_shared_attn_args* x, const int32_t* first) {
  const char* who = "sp_shared_attn_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->hq > 0 && x->hkv > 0 && x->hq % x->hkv == 0, SP_ERR_INVALID_ARGUMENT, "%s: bad shape hq=%lld hkv=%lld", who, (long long)x->hq,
             (long long)x->hkv);
  SP_REQUIRE(x->d == 64 || x->d == 128, SP_ERR_UNSUPPORTED, "%s: head_dim %lld unsupported (64 or 128)", who, (long long)x->d);
  SP_REQUIRE((float)x->softmax_scale > 0.f, SP_ERR_INVALID_ARGUMENT, "%s: softmax_scale must be > 0", who);
  SP_REQUIRE(x->batch > 0 && x->tokens >= 0 && x->table_width > 0 && x->num_pages > 0 && x->groups >= 0, SP_ERR_INVALID_ARGUMENT,
             "%s: batch=%lld tokens=%lld table_width=%lld num_pages=%lld groups=%lld", who, (long long)x->batch, (long long)x->tokens,
             (long long)x->table_width, (long long)x->num_pages, (long long)x->groups);
  SP_REQUIRE(x->groups <= x->batch, SP_ERR_INVALID_ARGUMENT, "%s: %lld groups of %lld requests", who, (long long)x->groups, (long long)x->batch);
  SP_REQUIRE(x->batch <= SH_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, SH_MAX_SEQS);
  int shift = 4;
  while (shift <= 10 && x->page_size != 1ll << shift) ++shift;
  SP_REQUIRE(shift <= 10, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  SP_REQUIRE(x->tokens <= PG_MAX_KEYS && x->num_pages <= 0x7fffffffll && x->table_width <= PG_MAX_KEYS && x->table_width << shift <= PG_MAX_KEYS,
             SP_ERR_UNSUPPORTED, "%s: tokens=%lld num_pages=%lld table_width=%lld too large", who, (long long)x->tokens, (long long)x->num_pages,
             (long long)x->table_width);
  SP_REQUIRE(x->cu_q != nullptr || x->tokens == x->batch, SP_ERR_INVALID_ARGUMENT, "%s: without cu_q every sequence has one token (%lld for %lld)",
             who, (long long)x->tokens, (long long)x->batch);
  const int64_t g = x->hq / x->hkv;
  SP_REQUIRE(x->weights == nullptr || (x->cu_q == nullptr && g <= PD_MAX_GROUP), SP_ERR_UNSUPPORTED,
             "%s: weights go with single tokens of up to %d query heads a kv head", who, PD_MAX_GROUP);
  if (x->tokens == 0) return SP_OK;
  SP_REQUIRE(sh_shape_ok(x->tokens, x->batch, x->groups, x->hq, x->hkv, x->d), SP_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads are too many", who,
             (long long)x->tokens, (long long)x->hq);
  const int64_t q_n = pg_used_stride(x->q_stride_n, x->tokens), q_h = pg_used_stride(x->q_stride_h, x->hq);
  const int64_t k_p = pg_used_stride(x->k_stride_page, x->num_pages), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  const int64_t v_p = pg_used_stride(x->v_stride_page, x->num_pages), v_h = pg_used_stride(x->v_stride_h, x->hkv);
  const int64_t w_p = pg_used_stride(x->w_stride_page, x->num_pages), w_h = pg_used_stride(x->w_stride_h, x->hkv);
  SP_REQUIRE(x->q && x->k_pages && x->v_pages && x->block_table && x->seq_lens && x->out && ((x->shared_lens && x->cu_groups) || x->groups == 0),
             SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->q | (uintptr_t)x->k_pages | (uintptr_t)x->v_pages | (uintptr_t)x->out) % 16 == 0 &&
                 (q_n | q_h | k_p | k_h | v_p | v_h) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  for (const int64_t n : {x->k_stride_slot, x->v_stride_slot})
    SP_REQUIRE(n >= 0 && n < (1ll << 24) && n * x->page_size < (1ll << 30) && n % 8 == 0, SP_ERR_UNSUPPORTED, "%s: slot stride %lld unsupported", who,
               (long long)n);
  const bool apart = sh_apart(x->tokens, x->groups, x->hq, x->hkv, x->table_width << shift, x->weights != nullptr);
  const ShSizes s = sh_sizes(x->tokens, x->batch, x->groups, x->hq, x->hkv, x->d, x->cu_q == nullptr,
                             x->weights != nullptr ? x->num_pages << shift : 0, apart);
  SP_REQUIRE(s.slots <= 0x7ffffff0ll, SP_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads are too many", who, (long long)x->tokens, (long long)x->hq);
  SP_REQUIRE(x->workspace != nullptr && x->workspace_bytes >= s.bytes && (uintptr_t)x->workspace % 16 == 0, SP_ERR_WORKSPACE,
             "%s: workspace missing, too small or misaligned", who);
  char* const ws = (char*)x->workspace;
  ShArgs a = {};
  a.q = (const sp_bf16*)x->q, a.k = (const sp_bf16*)x->k_pages, a.v = (const sp_bf16*)x->v_pages;
  a.table = x->block_table, a.lens = x->seq_lens, a.cu = x->cu_q, a.shared = x->shared_lens, a.groups = x->cu_groups, a.joined = x->joined;
  a.out = (sp_bf16*)x->out;
  a.table_stride = x->table_stride, a.sq_n = q_n, a.sq_h = q_h;
  a.sk_p = k_p, a.sk_n = x->k_stride_slot, a.sk_h = k_h, a.sv_p = v_p, a.sv_n = x->v_stride_slot, a.sv_h = v_h, a.sw_p = w_p, a.sw_h = w_h;
  a.batch = (int)x->batch, a.tokens = (int)x->tokens, a.width = (int)x->table_width, a.num_pages = (int)x->num_pages, a.shift = shift;
  a.n_groups = (int)x->groups;
  a.hkv = (int)x->hkv, a.group = (int)g, a.dense = x->cu_q == nullptr && g <= SH_UNIT;
  a.by_group = pg_divisor((unsigned)g);
  a.shared_slots = (int)s.shared_slots;
  a.parts = sh_workgroups(x->hkv);
  a.scale_log2 = (float)x->softmax_scale * 1.4426950408889634f;
  a.o_part = (float*)(ws + s.o_part), a.ml_part = (float2*)(ws + s.ml_part), a.o_row = (float*)(ws + s.o_row), a.ml_row = (float2*)(ws + s.ml_row);
  a.parts_of = (int2*)(ws + s.parts_of), a.cuts = (int4*)(ws + s.cuts), a.of_request = (ShRequest*)(ws + s.of_request);
  a.o_stream = (float*)(ws + s.o_stream), a.ml_stream = (float2*)(ws + s.ml_stream);
  a.streams = x->cu_q == nullptr && g <= PD_MAX_GROUP;
  a.weights_by_four = (uintptr_t)x->weights % 16 == 0 && (w_p | w_h) % 4 == 0;
  a.weights = x->weights, a.weigh_from = x->weights != nullptr ? first : nullptr, a.logits = (float*)(ws + s.logits);
  const int grid = a.parts * a.hkv;
  // few rows may have many parts each: a workgroup a row
  const int sets = x->tokens * x->hq <= 512 ? SM_THREADS / ((int)x->d / 4) : 1;
  const int64_t join = sp_ceil_div(x->tokens * x->hq * sets, SM_THREADS / (x->d / 4));
  const int64_t joins = join + (x->weights != nullptr ? (int64_t)grid * SH_WAVES : 0);
  SP_REQUIRE(joins * SM_THREADS < (1ll << 32), SP_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads are too many", who, (long long)x->tokens,
             (long long)x->hq);  // (a launch has fewer threads than that)
  static bool attr_set[64] = {false};  // per device, once (idempotent)
  int dev = 0;
  SP_HIP(hipGetDevice(&dev));
  SP_REQUIRE(dev >= 0 && dev < 64, SP_ERR_UNSUPPORTED, "%s: device index %d", who, dev);
  if (!attr_set[dev]) {
    for (const void* f : {(const void*)sp_shared_kernel<64>, (const void*)sp_shared_kernel<128>})
      SP_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sh_lds_bytes(SH_MAX_SEQS, SH_MAX_SEQS)));
    attr_set[dev] = true;
  }
  const hipStream_t stream = (hipStream_t)x->stream;
  a.apart = apart;
  if (a.apart) {
    CkArgs c = {};
    c.q = a.q, c.k = a.k, c.v = a.v, c.table = a.table, c.lens = a.shared, c.cu = a.cu, c.groups = a.groups, c.o_row = a.o_row, c.ml_row = a.ml_row;
    c.table_stride = a.table_stride, c.sq_n = a.sq_n, c.sq_h = a.sq_h;
    c.sk_p = a.sk_p, c.sk_n = a.sk_n, c.sk_h = a.sk_h, c.sv_p = a.sv_p, c.sv_n = a.sv_n, c.sv_h = a.sv_h;
    c.batch = a.n_groups, c.n_seqs = a.batch, c.tokens = a.tokens, c.width = a.width, c.num_pages = a.num_pages, c.shift = a.shift, c.n_queries = 1;
    c.hkv = a.hkv, c.group = a.group, c.scale_log2 = a.scale_log2;
    const int rc = ck_groups_launch(c, (int)x->d, ws + s.o_part, stream);
    if (rc) return rc;
  }
  const size_t lds = sh_lds_bytes(a.batch, a.n_groups);
  auto go = [&](auto kernel, auto many, auto few) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(SH_THREADS), lds, stream, a);
    hipLaunchKernelGGL(sets == 1 ? many : few, dim3((unsigned)joins), dim3(SM_THREADS), 0, stream, a, (int)join);
  };
  if (x->d == 64)
    go(sp_shared_kernel<64>, sp_shared_join_kernel<64, 1>, sp_shared_join_kernel<64, SM_THREADS / 16>);
  else
    go(sp_shared_kernel<128>, sp_shared_join_kernel<128, 1>, sp_shared_join_kernel<128, SM_THREADS / 32>);
  SP_LAUNCH_CHECK();
  return SP_OK;
}
