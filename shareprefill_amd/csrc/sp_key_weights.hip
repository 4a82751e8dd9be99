// How much attention every cached key receives from a request's last queries (sp_paged_key_weights):
//   weight[j] = sum over the rows r, (token, query head of the kv group) pairs, that see key j, of exp(scale q_r . k_j) / sum_j' exp(scale q_r . k_j').
// A row's maximum and sum have to be known before its weights can be summed over the rows, so the keys are walked twice: once for
// the rows' maxima and sums, once for the weights, S = K . Q^T formed anew (a second product costs less than 4 bytes a logit written and read
// back once there are more than a few rows; the second walk of a cache that fits the 256 MB behind the L2 is read from there).
// What bounds it: HBM for few rows (2 D bytes a key and kv head), else the vector unit: an exponential, four other instructions and half a product's 16 cycles a
// logit and walk, where the matrix cores take D / 8 cycles for sixteen rows' product with sixteen keys.
//
// A wave has 32 keys, its K operands in registers, those of its next 32 keys on their way; the rows' queries lie in LDS, up to 256 of them, and serve all
// keys of the workgroup's part; two row tiles are on their way at a time, one's products under the other's exponentials.  Two workgroups a CU: with one of eight
// waves the queries would be staged half as often, which took as long.  Every key's sum is formed by one wave in one order: results do not depend on timing.
// Requests' blocks of 128 keys lie on a line per kv head that is cut into equal parts, a workgroup each.
//
// Measured (first walk, rows' parts joined, second walk): 32 queries of 28 heads over 4 of 128 channels over 32768 keys 23.9 + 4.8 + 19.6 us, 15 GFLOP in both
// products; of a walk 3 us are the line, 5 the queries and first keys, 4 a block of 224 rows.  64 queries each of 8 requests of 32 heads over 8 of 64 channels over up
// to 8001 keys 31.2 + 5.9 + 26.1; 16 over 1025 keys of 32 heads over 8 10.6 + 10.4, all of it latency.
#include "sp_ring.h"
#include "sp_paged_plan.h"

#define KW_WAVES 4
#define KW_THREADS (KW_WAVES * SP_WAVE)
#define KW_KEYS 32                       // of a wave
#define KW_BLOCK (KW_WAVES * KW_KEYS)
#define KW_TILES 16                      // row tiles of 16 in LDS
#define KW_SLACK 7.f
// The exponent takes a logit's exact product with the scale and the row's maximum rounded, half a step of the maximum apart for all of its keys alike: 8 octaves
// below 2^28, more than an exponential holds from 2^31 on.  Rows that lie further out take rounded products.
#define KW_FAR 0x1p28f
#define KW_ROWS (16 * KW_TILES)
#define KW_OVERHEAD 2                    // blocks' worth of a request beside its blocks: its queries, the rows' meeting
#define KW_UNITS(rows) (((rows) + 31) / 32 + 1)  // of a block: pairs of row tiles, and its keys
#define KW_SHARE 4                       // units of a part at least
#define KW_MAX_SEQS 1024
#define KW_FEW 16                        // parts that the second walk joins by itself
#define KW_PLACES 512                    // workgroups: two a CU

typedef const __attribute__((address_space(1))) void* kw_gbl_ptr;

struct KwArgs {
  const sp_bf16 *q, *k;
  const int32_t *table, *lens, *cu, *first;
  float* weights;
  int64_t table_stride, sq_n, sq_h, sk_p, sk_n, sk_h, sw_p, sw_h;
  int batch, tokens, width, num_pages, shift;
  int hkv, group, accumulate, parts, few;
  PgDivisor by_group;
  float scale_log2;
  float2* part_ml;   // [token][query head][part]: of the keys that fell to a part, counted from the request's first
  float2* row_ml;    // [token][query head]: maximum, 1 / sum
  int2* of_request;  // [batch + 1]: parts that the request's keys fell to, its first token
};

// ---- the line ----
// Blocks of 128 keys of every request with new tokens, from block `from` on (the walk for the weights leaves out what lies in front of the
// request's first wanted key).

// (a NaN passes, and makes the lane's sum one: no other logit of the row counts then)
__device__ static __forceinline__ float kw_max(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
__device__ static __forceinline__ float kw_max(ds_floatx4 v) { return __builtin_elementwise_maximum(kw_max(v[0], v[1], v[2]), v[3]); }

// x / by with 1 / by to 2^-24 at least, quotients below 2^24
__device__ static __forceinline__ int64_t kw_quotient(int64_t x, int by, double inverse) {
  int64_t q = (int64_t)((double)x * inverse);
  const int64_t left = x - q * by;
  return q + (left >= by) - (left < 0);
}

__device__ static __forceinline__ bool kw_far(float m) { return __builtin_fabsf(m) >= KW_FAR && __builtin_fabsf(m) < INFINITY; }

__device__ static __forceinline__ float kw_octaves(float x, float scale, float m) {  // (the product is rounded)
#pragma clang fp contract(off)
  const float p = x * scale;
  return p - m;
}

// over the 16 lanes of a row, each in an order of its own
__device__ static __forceinline__ float kw_row_sum(float v) {
#define KW_ROTATED(n) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x120 + n, 0xf, 0xf, true))
  v += KW_ROTATED(8), v += KW_ROTATED(4), v += KW_ROTATED(2), v += KW_ROTATED(1);
#undef KW_ROTATED
  return v;
}

// A row's parts joined where there are KW_FEW at most: maximum and 1 / sum, infinity and 0 of a row that sees no key.
__device__ static __forceinline__ float2 kw_joined(float top, float sum) { return make_float2(top == -INFINITY ? INFINITY : top, sum == 0.f ? 0.f : 1.0f / sum); }
__device__ static __forceinline__ float2 kw_join(const float2* parts, int count) {
  float2 p[KW_FEW];
#pragma unroll
  for (int i = 0; i < KW_FEW; ++i) p[i] = i < count ? parts[i] : make_float2(-INFINITY, 0.f);
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < KW_FEW; ++i) top = fmaxf(top, p[i].x);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < KW_FEW; ++i) sum += p[i].y * __builtin_amdgcn_exp2f(p[i].x - base);
  return kw_joined(top, sum);
}

template <int D, bool SUMS>
__global__ __launch_bounds__(KW_THREADS, 2) void sp_key_weights_kernel(const KwArgs a) {
  constexpr int KS = D / 32, CHUNKS = D / 8;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // queries [KW_ROWS][D], swizzled; rows' maxima and sums; offsets and lengths
  char* const q_lds = lds;
  float2* const ml_s = reinterpret_cast<float2*>(lds + KW_ROWS * D * 2);  // [KW_WAVES][KW_ROWS]
  int* const start_s = reinterpret_cast<int*>(ml_s + KW_WAVES * KW_ROWS);
  int* const len_s = start_s + a.batch + 1;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lq = lane & 15, gr = lane >> 4;
  const int kvh = blockIdx.x % a.hkv, part = blockIdx.x / a.hkv, g = a.group, room = a.width << a.shift;
  const int hq = a.hkv * g;

  int back = 0;
  for (int i = t; i <= a.batch; i += KW_THREADS) {
    auto start = [&](int j) { return a.cu != nullptr ? pg_max(0, pg_min(a.cu[j], a.tokens)) : j; };
    start_s[i] = start(i);
    if (i < a.batch) len_s[i] = pg_max(0, pg_min(a.lens[i], PG_MAX_KEYS)), back |= start(i + 1) < start(i);
  }
  if (__syncthreads_or(back)) {  // (offsets that go back count as the largest in front of them)
    if (t == 0)
      for (int i = 1; i <= a.batch; ++i) start_s[i] = pg_max(start_s[i], start_s[i - 1]);
    __syncthreads();
  }
  auto blocks = [&](int b, int* from) {
    const int keys = pg_min(len_s[b], room);
    *from = SUMS && a.first != nullptr ? pg_max(0, pg_min(a.first[b], keys)) / KW_BLOCK : 0;
    return start_s[b + 1] > start_s[b] && keys > 0 ? (keys + KW_BLOCK - 1) / KW_BLOCK - *from : 0;
  };
  auto units_of = [&](int b, int n) { return n > 0 ? (int64_t)(n + KW_OVERHEAD) * KW_UNITS((start_s[b + 1] - start_s[b]) * g) : 0; };
  // the line, by every wave for itself: a lane has some requests side by side
  const int per = (a.batch + SP_WAVE - 1) / SP_WAVE, b0 = lane * per, b1 = pg_min(b0 + per, a.batch);
  int64_t mine = 0, lead = 0;
  int from;
  for (int b = b0; b < b1; ++b) {
    const int n = blocks(b, &from);
    const int64_t units = units_of(b, n);
    if (mine == 0 && n > 0) lead = (int64_t)KW_OVERHEAD * KW_UNITS((start_s[b + 1] - start_s[b]) * g);
    mine += units;
  }
  int64_t at = mine;
  for (int o = 1; o < a.batch && o < SP_WAVE; o <<= 1) {
    const int64_t y = __shfl_up(at, o, SP_WAVE);
    if (lane >= o) at += y;
  }
  const int64_t total = ds_lane64(at, pg_min(a.batch, SP_WAVE) - 1);
  at -= mine;
  // what the line's first request has beside its blocks every part has: the parts begin behind it
  const uint64_t some = __ballot(mine > 0);
  lead = some != 0ull ? ds_lane64(lead, __builtin_ctzll(some)) : 0;
  const int64_t shared = total - lead, full = (shared + KW_SHARE - 1) / KW_SHARE;
  const int parts = full < a.parts ? pg_max((int)full, 1) : a.parts;
  const PgCuts cuts = pg_cuts(shared, parts);
  auto cut = [&](int p) { return lead + pg_cut_at(cuts, p); };
  const int64_t cut0 = cut(part), cut1 = cut(part + 1);
  // of a request whose blocks have `each` units: KW_OVERHEAD blocks' worth, then its blocks; a part may fall between two cuts of one block and hold none
  auto steps = [&](int64_t start, int n, int each, int64_t c0, int64_t c1, int* begin, int* end) {
    const double by = __builtin_amdgcn_rcp((double)each);
    auto block = [&](int64_t c) {
      const int64_t off = c - start, at = off > 0 ? kw_quotient(off, each, by) : 0;
      return (int)(at <= KW_OVERHEAD ? 0 : at - KW_OVERHEAD < n ? at - KW_OVERHEAD : n);
    };
    *begin = block(c0);
    *end = block(c1);
  };
  // the part that unit x lies in, and the one that a request's first block ends in
  auto part_of = [&](int64_t x) {
    int p = (int)((float)(x - lead) * (float)parts * __builtin_amdgcn_rcpf((float)shared));  // within one: parts are KW_PLACES at most
    p = pg_min(p, parts - 1);
    while (p > 0 && cut(p) > x) --p;
    while (p + 1 < parts && cut(p + 1) <= x) ++p;
    return p;
  };
  auto first_part = [&](int64_t start, int each) { return part_of(start + (int64_t)(KW_OVERHEAD + 1) * each - 1); };
  const bool holds = cut0 < cut1 && cut0 >= at && cut0 < at + mine;
  const bool tell = !SUMS && blockIdx.x == gridDim.x - 1;  // (the one that small calls leave idle)
  int b = a.batch;
  int64_t unit = at;
  if (holds || tell) {
    int64_t u = at;
    for (int i = b0; i < b1; ++i) {
      const int n = blocks(i, &from);
      const int64_t units = units_of(i, n);
      if (tell && wave == 0)
        a.of_request[i] = make_int2(n > 0 ? part_of(u + units - 1) - first_part(u, KW_UNITS((start_s[i + 1] - start_s[i]) * g)) + 1 : 0, start_s[i]);
      if (holds && cut0 >= u && cut0 < u + units) b = i, unit = u;
      u += units;
    }
  }
  if (tell && t == 0) a.of_request[a.batch] = make_int2(0, start_s[a.batch]);
  const uint64_t holder = __ballot(holds);
  const int held = holder != 0ull ? __builtin_ctzll(holder) : 0;  // (the lanes' b is the batch where none holds)
  b = __builtin_amdgcn_readlane(b, held);
  unit = ds_lane64(unit, held);

  for (; b < a.batch && unit < cut1; ++b) {
    const int n = blocks(b, &from);
    if (n == 0) continue;
    const int start = start_s[b], q_len = start_s[b + 1] - start, len = len_s[b], rows = q_len * g, keys = pg_min(len, room), each = KW_UNITS(rows);
    const int64_t start_unit = unit;
    unit += units_of(b, n);
    int begin, end;
    steps(start_unit, n, each, cut0, cut1, &begin, &end);
    const int rel = SUMS ? 0 : part - first_part(start_unit, each);
    if (begin >= end) {
      if (!SUMS && rel >= 0)  // (a part between the others' that holds nothing)
        for (int r = t; r < rows; r += KW_THREADS) {
          const int token = (int)pg_div((unsigned)r, a.by_group);
          a.part_ml[((int64_t)(start + token) * hq + kvh * g + (r - token * g)) * a.parts + rel] = make_float2(-INFINITY, 0.f);
        }
      continue;
    }
    const int first_key = SUMS && a.first != nullptr ? pg_max(0, pg_min(a.first[b], keys)) : 0;
    const int pos0 = len - q_len;  // of the first row
    const sp_bf16* const kh = a.k + kvh * a.sk_h;
    // (scalar loads: nothing writes the table during the launch)
    const auto table = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(a.table + (int64_t)__builtin_amdgcn_readfirstlane(b) * a.table_stride);
    struct Ids {
      int id[2];  // pages of the wave's 16-key halves of a block, in Keys -1: none
    };
    struct Keys {  // K operands of the wave's 32 keys of a block
      dc_u32x4 r[2][KS];
      Ids ids;
    };
    auto entries = [&](int block) {
      Ids x;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int page = ((from + block) * KW_BLOCK + wave * KW_KEYS + 16 * i) >> a.shift;
        x.id[i] = table[pg_min(page, a.width - 1)];
      }
      return x;
    };
    auto fetch = [&](int block, Ids ids, Keys& x) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = (from + block) * KW_BLOCK + wave * KW_KEYS + 16 * i;
        x.ids.id[i] = key >> a.shift < a.width && (unsigned)ids.id[i] < (unsigned)a.num_pages ? ids.id[i] : -1;
        const sp_bf16* src = kh + (int64_t)pg_max(x.ids.id[i], 0) * a.sk_p + (int64_t)((key & ((1 << a.shift) - 1)) + lq) * a.sk_n + 8 * gr;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x.r[i][ks] = *reinterpret_cast<const dc_u32x4*>(src + 32 * ks);
      }
    };
    for (int row0 = 0; row0 < rows; row0 += KW_ROWS) {
      const int here = pg_min(rows - row0, KW_ROWS), tiles = (here + 31) / 32 * 2;  // (an even number)
      Keys cur, nxt;
      Ids ids = entries(begin);
      __syncthreads();  // (the rows before are done with)
      // (workgroups side by side begin at rows of their own: all of them ask for the same ones)
      const int runs = tiles * 16 * CHUNKS / KW_THREADS;
      for (int j = 0, at = part % runs; j < runs; ++j, at = at + 1 < runs ? at + 1 : 0) {
        const int i = at * KW_THREADS + t, r = i / CHUNKS, row = row0 + pg_min(r, here - 1), token = (int)pg_div((unsigned)row, a.by_group);
        __builtin_amdgcn_global_load_lds((kw_gbl_ptr)(a.q + (int64_t)(start + token) * a.sq_n + (int64_t)(kvh * g + (row - token * g)) * a.sq_h +
                                                      8 * ((i % CHUNKS) ^ ds_swz_k<D>(r & 15))),
                                         (ds_lds_ptr)(q_lds + (i - lane) * 16), 16, 0, 0);
      }
      fetch(begin, ids, cur);
      ids = entries(pg_min(begin + 1, end - 1));
      if constexpr (SUMS) {
        const int count = a.few ? a.of_request[b].x : 0;
        for (int r = t; r < tiles * 16; r += KW_THREADS) {  // (rows that are none weigh nothing)
          float2 ml = make_float2(INFINITY, 0.f);
          if (r < here) {
            const int row = row0 + r, token = (int)pg_div((unsigned)row, a.by_group);
            const int64_t at = (int64_t)(start + token) * hq + kvh * g + (row - token * g);
            ml = a.few ? kw_join(a.part_ml + at * a.parts, count) : a.row_ml[at];
          }
          ml_s[r] = ml;
        }
      }
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the queries
      __syncthreads();
      float m[SUMS ? 1 : KW_TILES], l[SUMS ? 1 : KW_TILES];
      // (uniform) some row of the wave lies far out; in the walk for the weights: or is no number
      bool odd = false;
      if constexpr (!SUMS) {
#pragma unroll
        for (int i = 0; i < KW_TILES; ++i) m[i] = -INFINITY, l[i] = 0.f;
      } else {
        for (int r = lane; r < tiles * 16; r += SP_WAVE) odd |= kw_far(ml_s[r].x) || ml_s[r].y != ml_s[r].y;
        odd = __ballot(odd) != 0ull;
      }
      for (int block = begin; block < end; ++block) {
        // (the last block asks for itself again: were it not to ask, the wait for this block's keys would be one for the next one's too)
        fetch(pg_min(block + 1, end - 1), ids, nxt);
        ids = entries(pg_min(block + 2, end - 1));
        const int key0 = (from + block) * KW_BLOCK + wave * KW_KEYS;
        const bool edge = key0 + KW_KEYS - 1 > pos0 + (int)pg_div((unsigned)row0, a.by_group) || (cur.ids.id[0] | cur.ids.id[1]) < 0;  // some row does not see some key
        float acc[2][4] = {{0.f}};
        // the products of row tiles i and i + 1: keys 16 h + 4 gr + j of row lq.  -> where `edge`: bit 8 u + 4 h + j says that row lq of tile i + u sees that key
        auto pair = [&](int i, ds_floatx4 (&sc)[2][2]) {
          uint32_t seen = 0u;
          dc_bf16x8 qb[2][KS];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
              qb[u][ks] = *reinterpret_cast<const dc_bf16x8*>(q_lds + (16 * (i + u) + lq) * (D * 2) + (((4 * ks + gr) ^ ds_swz_k<D>(lq)) << 4));
          __builtin_amdgcn_sched_barrier(0);  // (all on their way at once)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[u][h] = (ds_floatx4){0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                sc[u][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, cur.r[h][ks]), qb[u][ks], sc[u][h], 0, 0, 0);
          if (edge) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int pos = pos0 + (int)pg_div((unsigned)pg_min(row0 + 16 * (i + u) + lq, rows - 1), a.by_group);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const bool sees = key0 + 16 * h + 4 * gr + j <= pos && cur.ids.id[h] >= 0;
                  sc[u][h][j] = sees ? sc[u][h][j] : -INFINITY;
                  seen |= (uint32_t)sees << (8 * u + 4 * h + j);
                }
            }
          }
          return seen;
        };
        if constexpr (!SUMS) {
#pragma unroll
          for (int i = 0; i < KW_TILES; i += 2) {
            if (i < tiles) {
              ds_floatx4 sc[2][2];
              pair(i, sc);
              float mx[2];
#pragma unroll
              for (int u = 0; u < 2; ++u)
                mx[u] = a.scale_log2 * kw_max(kw_max(kw_max(sc[u][0]), sc[u][1][0], sc[u][1][1]), sc[u][1][2], sc[u][1][3]);
              // (a lane's maximum moves when a logit passes it by seven octaves, which few do: sums of 2^7 are as exact)
              if (__ballot(mx[0] > m[i] + KW_SLACK || mx[1] > m[i + 1] + KW_SLACK) != 0ull) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const float to = fmaxf(m[i + u], mx[u]);
                  l[i + u] *= to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[i + u] - to);
                  m[i + u] = to;
                  odd |= __ballot(kw_far(to)) != 0ull;
                }
              }
              auto add = [&](auto far_out) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const float base = m[i + u] == -INFINITY ? 0.f : m[i + u];
                  const bool far = decltype(far_out)::value && kw_far(base);
                  auto octaves = [&](float x) { return far ? kw_octaves(x, a.scale_log2, base) : fmaf(x, a.scale_log2, -base); };
                  float more = 0.f;
#pragma unroll
                  for (int j = 0; j < 4; ++j) more += __builtin_amdgcn_exp2f(octaves(sc[u][0][j])) + __builtin_amdgcn_exp2f(octaves(sc[u][1][j]));
                  l[i + u] += more;
                }
              };
              if (__builtin_expect(odd, false))
                add(std::true_type{});
              else
                add(std::false_type{});
            }
          }
        } else {
          auto walk = [&](auto any) {
            for (int i = 0; i < tiles; i += 2) {
              ds_floatx4 sc[2][2];
              const uint32_t seen = pair(i, sc);
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const float2 ml = ml_s[16 * (i + u) + lq];
                const bool far = decltype(any)::value && kw_far(ml.x);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    const float x = far ? kw_octaves(sc[u][h][j], a.scale_log2, ml.x) : fmaf(sc[u][h][j], a.scale_log2, -ml.x);
                    const float w = __builtin_amdgcn_exp2f(x) * ml.y;
                    // (a row that is no number makes none of the keys it sees, and of no others: 0 times its sum's reciprocal would be none too)
                    acc[h][j] += decltype(any)::value && edge && !((seen >> (8 * u + 4 * h + j)) & 1u) ? 0.f : w;
                  }
              }
            }
          };
          if (__builtin_expect(odd, false)) walk(std::true_type{}); else walk(std::false_type{});
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[h][j] = kw_row_sum(acc[h][j]);
          // lanes 0 .. 7 of a group have a key each: 16 (lq / 4) + 4 gr + lq % 4
          float sum = acc[0][0];
#pragma unroll
          for (int i = 1; i < 8; ++i) sum = lq == i ? acc[i >> 2][i & 3] : sum;
          const int key = key0 + 16 * (lq >> 2) + 4 * gr + (lq & 3);
          const int id = lq < 4 ? cur.ids.id[0] : cur.ids.id[1];
          if (lq < 8 && id >= 0 && key >= first_key && key < keys) {
            float* const to = a.weights + (int64_t)id * a.sw_p + kvh * a.sw_h + (key & ((1 << a.shift) - 1));
            const bool adds = row0 > 0 || (a.accumulate && key < pos0);
            *to = (adds ? *to : 0.f) + sum;
          }
        }
        cur = nxt;
      }
      if constexpr (!SUMS) {
#pragma unroll
        for (int i = 0; i < KW_TILES; ++i) {
          if (i < tiles) {
            const float top = ds_quad_max(m[i]), sum = ds_quad_sum(l[i] * __builtin_amdgcn_exp2f(m[i] - (top == -INFINITY ? 0.f : top)));
            if (gr == 0) ml_s[wave * KW_ROWS + 16 * i + lq] = make_float2(top, sum);
          }
        }
        __syncthreads();
        for (int r = t; r < here; r += KW_THREADS) {
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int w = 0; w < KW_WAVES; ++w) top = fmaxf(top, ml_s[w * KW_ROWS + r].x);
          const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int w = 0; w < KW_WAVES; ++w) sum += ml_s[w * KW_ROWS + r].y * __builtin_amdgcn_exp2f(ml_s[w * KW_ROWS + r].x - base);
          const int row = row0 + r, token = (int)pg_div((unsigned)row, a.by_group);
          a.part_ml[((int64_t)(start + token) * hq + kvh * g + (row - token * g)) * a.parts + rel] = make_float2(top, sum);
        }
      }
    }
  }
}

// A row's parts joined, a wave each: its maximum and 1 / sum (infinity and 0: it sees no key).
__global__ __launch_bounds__(KW_THREADS) void sp_key_weights_join_kernel(const KwArgs a) {
  const int lane = threadIdx.x & 63, hq = a.hkv * a.group;
  const int64_t row = (int64_t)blockIdx.x * KW_WAVES + (threadIdx.x >> 6);
  if (row >= (int64_t)a.tokens * hq) return;
  const int token = (int)(row / hq);
  int b = token;
  if (a.cu != nullptr) {
    b = 0;
    int hi = a.batch;
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (a.of_request[mid].y <= token)
        b = mid;
      else
        hi = mid;
    }
  }
  const int count = token >= a.of_request[b].y && token < a.of_request[b + 1].y ? a.of_request[b].x : 0;
  float top = -INFINITY, sum = 0.f;
  for (int i0 = 0; i0 < count; i0 += SP_WAVE) {
    const float2 ml = i0 + lane < count ? a.part_ml[row * a.parts + i0 + lane] : make_float2(-INFINITY, 0.f);
    const float to = fmaxf(top, sp_wave_max(ml.x)), base = to == -INFINITY ? 0.f : to;
    sum = sum * __builtin_amdgcn_exp2f(top - base) + sp_wave_sum(ml.y * __builtin_amdgcn_exp2f(ml.x - base));
    top = to;
  }
  if (lane == 0) a.row_ml[row] = kw_joined(top, sum);
}

// ---- host -------------------------------------------------------------------------------------------------
static int kw_parts(int64_t hkv) { return hkv < KW_PLACES ? KW_PLACES / (int)hkv : 1; }
struct KwSizes {
  size_t part_ml, row_ml, of_request, bytes;
};
static KwSizes kw_sizes(int64_t tokens, int64_t batch, int64_t hq, int64_t hkv) {
  KwSizes s;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  s.part_ml = take((size_t)(tokens * hq) * kw_parts(hkv) * sizeof(float2));
  s.row_ml = take((size_t)(tokens * hq) * sizeof(float2));
  s.of_request = take((size_t)(batch + 1) * sizeof(int2));
  s.bytes = at;
  return s;
}
static bool kw_shape_ok(int64_t tokens, int64_t batch, int64_t hq, int64_t hkv) {
  return tokens > 0 && tokens <= PG_MAX_KEYS && batch > 0 && batch <= KW_MAX_SEQS && hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 65536 &&
         tokens * hq < (1ll << 31);
}

extern "C" size_t sp_paged_key_weights_workspace_bytes(int64_t tokens, int32_t batch, int32_t hq, int32_t hkv) {
  return kw_shape_ok(tokens, batch, hq, hkv) ? kw_sizes(tokens, batch, hq, hkv).bytes : 0;
}

extern "C" int sp_paged_key_weights_bf16(const sp_paged_key_weights_args* x) {
  const char* who = "sp_paged_key_weights_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->hq > 0 && x->hkv > 0 && x->hq % x->hkv == 0, SP_ERR_INVALID_ARGUMENT, "%s: bad shape hq=%lld hkv=%lld", who, (long long)x->hq,
             (long long)x->hkv);
  SP_REQUIRE(x->d == 64 || x->d == 128, SP_ERR_UNSUPPORTED, "%s: head_dim %lld unsupported (64 or 128)", who, (long long)x->d);
  SP_REQUIRE((float)x->softmax_scale > 0.f, SP_ERR_INVALID_ARGUMENT, "%s: softmax_scale must be > 0", who);
  SP_REQUIRE(x->batch > 0 && x->tokens >= 0 && x->table_width > 0 && x->num_pages > 0, SP_ERR_INVALID_ARGUMENT,
             "%s: batch=%lld tokens=%lld table_width=%lld num_pages=%lld", who, (long long)x->batch, (long long)x->tokens, (long long)x->table_width,
             (long long)x->num_pages);
  SP_REQUIRE(x->batch <= KW_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, KW_MAX_SEQS);
  int shift = 4;
  while (shift <= 10 && x->page_size != 1ll << shift) ++shift;
  SP_REQUIRE(shift <= 10, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  SP_REQUIRE(x->tokens <= PG_MAX_KEYS && x->num_pages <= 0x7fffffffll && x->table_width <= PG_MAX_KEYS && x->table_width << shift <= PG_MAX_KEYS,
             SP_ERR_UNSUPPORTED, "%s: tokens=%lld num_pages=%lld table_width=%lld too large", who, (long long)x->tokens, (long long)x->num_pages,
             (long long)x->table_width);
  SP_REQUIRE(x->cu_q != nullptr || x->tokens == x->batch, SP_ERR_INVALID_ARGUMENT, "%s: without cu_q every sequence has one token (%lld for %lld)",
             who, (long long)x->tokens, (long long)x->batch);
  if (x->tokens == 0) return SP_OK;
  SP_REQUIRE(kw_shape_ok(x->tokens, x->batch, x->hq, x->hkv) && (x->tokens * x->hq + KW_WAVES - 1) * SP_WAVE < (1ll << 32), SP_ERR_UNSUPPORTED,  // (the joining launch)
             "%s: %lld tokens of %lld heads are too many", who,
             (long long)x->tokens, (long long)x->hq);
  const int64_t q_n = pg_used_stride(x->q_stride_n, x->tokens), q_h = pg_used_stride(x->q_stride_h, x->hq);
  const int64_t k_p = pg_used_stride(x->k_stride_page, x->num_pages), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  SP_REQUIRE(x->q && x->k_pages && x->block_table && x->seq_lens && x->weights, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->q | (uintptr_t)x->k_pages) % 16 == 0 && (q_n | q_h | k_p | k_h | x->k_stride_slot) % 8 == 0, SP_ERR_UNSUPPORTED,
             "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  const KwSizes s = kw_sizes(x->tokens, x->batch, x->hq, x->hkv);
  SP_REQUIRE(x->workspace != nullptr && x->workspace_bytes >= s.bytes && (uintptr_t)x->workspace % 16 == 0, SP_ERR_WORKSPACE,
             "%s: workspace missing, too small or misaligned", who);
  char* const ws = (char*)x->workspace;
  KwArgs a = {};
  a.q = (const sp_bf16*)x->q, a.k = (const sp_bf16*)x->k_pages;
  a.table = x->block_table, a.lens = x->seq_lens, a.cu = x->cu_q, a.first = x->first, a.weights = x->weights;
  a.table_stride = x->table_stride, a.sq_n = q_n, a.sq_h = q_h, a.sk_p = k_p, a.sk_n = x->k_stride_slot, a.sk_h = k_h;
  a.sw_p = pg_used_stride(x->w_stride_page, x->num_pages), a.sw_h = pg_used_stride(x->w_stride_h, x->hkv);
  a.batch = (int)x->batch, a.tokens = (int)x->tokens, a.width = (int)x->table_width, a.num_pages = (int)x->num_pages, a.shift = shift;
  a.hkv = (int)x->hkv, a.group = (int)(x->hq / x->hkv), a.accumulate = x->accumulate != 0, a.parts = kw_parts(x->hkv);
  a.by_group = pg_divisor((unsigned)a.group);
  a.scale_log2 = (float)x->softmax_scale * 1.4426950408889634f;
  a.part_ml = (float2*)(ws + s.part_ml), a.row_ml = (float2*)(ws + s.row_ml), a.of_request = (int2*)(ws + s.of_request);
  // parts of a request: two ends and what lies between them, of KW_SHARE - 1 units at least (n units make ceil(n / KW_SHARE) parts: three parts of 9)
  const int64_t blocks = ((x->table_width << shift) + KW_BLOCK - 1) / KW_BLOCK + KW_OVERHEAD;
  a.few = blocks * KW_UNITS(x->tokens * a.group) / (KW_SHARE - 1) + 2 <= KW_FEW;
  auto lds = [](int d, int batch) { return (size_t)KW_ROWS * d * 2 + KW_WAVES * KW_ROWS * sizeof(float2) + (2 * (size_t)batch + 1) * sizeof(int); };
  static bool attr_set[64] = {false};  // per device, once (idempotent)
  int dev = 0;
  SP_HIP(hipGetDevice(&dev));
  SP_REQUIRE(dev >= 0 && dev < 64, SP_ERR_UNSUPPORTED, "%s: device index %d", who, dev);
  if (!attr_set[dev]) {
    for (const void* f : {(const void*)sp_key_weights_kernel<64, false>, (const void*)sp_key_weights_kernel<64, true>,
                          (const void*)sp_key_weights_kernel<128, false>, (const void*)sp_key_weights_kernel<128, true>})
      SP_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds(128, KW_MAX_SEQS)));
    attr_set[dev] = true;
  }
  const hipStream_t stream = (hipStream_t)x->stream;
  const unsigned grid = (unsigned)(a.parts * a.hkv), joins = (unsigned)sp_ceil_div(x->tokens * x->hq, KW_WAVES);
  auto go = [&](auto stats, auto sums) {
    hipLaunchKernelGGL(stats, dim3(grid), dim3(KW_THREADS), lds((int)x->d, a.batch), stream, a);
    if (!a.few) hipLaunchKernelGGL(sp_key_weights_join_kernel, dim3(joins), dim3(KW_THREADS), 0, stream, a);
    hipLaunchKernelGGL(sums, dim3(grid), dim3(KW_THREADS), lds((int)x->d, a.batch), stream, a);
  };
  x->d == 64 ? go(sp_key_weights_kernel<64, false>, sp_key_weights_kernel<64, true>) : go(sp_key_weights_kernel<128, false>, sp_key_weights_kernel<128, true>);
  SP_LAUNCH_CHECK();
  return SP_OK;
}
