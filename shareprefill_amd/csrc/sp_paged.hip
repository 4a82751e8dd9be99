// The bookkeeping of a key / value cache in pages: which pages a step's new tokens open and where each of them goes
// (sp_paged_tables), and the copy of their keys and values there (sp_paged_cache_write_bf16).
#include "sp_common.h"
#include "sp_paged_plan.h"

#define PT_THREADS 256

struct TablesArgs {
  const int32_t *lens, *new_lens;
  int32_t* table;
  int64_t table_stride;
  const int32_t *free_pages, *free_count;
  int batch, shift, width, num_pages, free_room, max_tokens;
  int32_t *seq_lens, *cu_new;
  int64_t* slots;
  int32_t *positions, *free_left;
};

// With len, new >= 0 of a request and pages of P tokens, W of them in its row of the table:
//   have = min(ceil(len / P), W), need = min(ceil((len + new) / P), W) - have;
// the pages of all requests in order come off the top of the stack, token t of the step belongs to the request whose prefix sum of `new`
// it lies behind.  Latency is all there is to it (some 130 KB for 256 requests): one launch, and every workgroup forms the two prefix sums over the
// requests for itself, which costs less than a launch that hands them over.  Sums hold at 2^30 (pg_held_sum); what the requests bring is
// read once and kept in LDS, the stack's height is asked for first.
// A new token's slot is taken from the stack itself, not from the table's entry, so nothing that another workgroup of the launch writes is read.
// TRUNCATE: tokens from max_tokens on are none.  What a request keeps of `new` follows from the prefix sums, which are formed first then: offsets
// held at max_tokens, and their differences.
template <bool TRUNCATE>
__global__ __launch_bounds__(PT_THREADS) void sp_paged_tables_kernel(TablesArgs a) {
  extern __shared__ int sh[];  // of the requests: tokens [batch + 1] and pages [batch + 1], then their prefix sums; lengths [batch]
  __shared__ int wave_sums[2][PT_THREADS / SP_WAVE];
  int* const tok = sh;
  int* const pgs = tok + a.batch + 1;
  int* const len_of = pgs + a.batch + 1;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, P = 1 << a.shift;
  const int count = pg_max(0, pg_min(a.free_count[0], a.free_room));
  const int per = (a.batch + PT_THREADS - 1) / PT_THREADS;
  auto pages = [&](int n) { return pg_min((int)(((unsigned)n + (unsigned)P - 1u) >> a.shift), a.width); };
  if constexpr (TRUNCATE) {
    int sum = 0;
    for (int i = t * per; i < (t + 1) * per && i < a.batch; ++i) tok[i] = pg_length(a.new_lens[i]), sum = pg_held_sum(sum, tok[i]);
    int at = sum;
#pragma unroll
    for (int o = 1; o < SP_WAVE; o <<= 1) {
      const int x = __shfl_up(at, o, SP_WAVE);
      if (lane >= o) at = pg_held_sum(at, x);
    }
    if (lane == SP_WAVE - 1) wave_sums[0][wave] = at;
    at = __shfl_up(at, 1, SP_WAVE);
    if (lane == 0) at = 0;
    __syncthreads();
    for (int w = 0; w < wave; ++w) at = pg_held_sum(at, wave_sums[0][w]);
    for (int i = t * per; i < (t + 1) * per && i < a.batch; ++i) {
      const int end = pg_held_sum(at, tok[i]);
      tok[i] = pg_min(end, a.max_tokens) - pg_min(at, a.max_tokens);
      at = end;
    }
    __syncthreads();  // the waves' sums are free
  }
  int tokens = 0, opened = 0;
  for (int i = t * per; i < (t + 1) * per && i < a.batch; ++i) {
    const int len = pg_length(a.lens[i]), n = TRUNCATE ? tok[i] : pg_length(a.new_lens[i]), p = pages(len + n) - pages(len);
    len_of[i] = len, tok[i] = n, pgs[i] = p;
    tokens = pg_held_sum(tokens, n), opened = pg_held_sum(opened, p);
  }
  int tok_at = tokens, page_at = opened;  // inclusive sums over the wave's lanes, then what lies in front of the thread
#pragma unroll
  for (int o = 1; o < SP_WAVE; o <<= 1) {
    const int x = __shfl_up(tok_at, o, SP_WAVE), y = __shfl_up(page_at, o, SP_WAVE);
    if (lane >= o) tok_at = pg_held_sum(tok_at, x), page_at = pg_held_sum(page_at, y);
  }
  if (lane == SP_WAVE - 1) wave_sums[0][wave] = tok_at, wave_sums[1][wave] = page_at;
  tok_at = __shfl_up(tok_at, 1, SP_WAVE), page_at = __shfl_up(page_at, 1, SP_WAVE);
  if (lane == 0) tok_at = page_at = 0;
  __syncthreads();
  for (int w = 0; w < wave; ++w) tok_at = pg_held_sum(tok_at, wave_sums[0][w]), page_at = pg_held_sum(page_at, wave_sums[1][w]);
  for (int i = t * per; i < (t + 1) * per && i < a.batch; ++i) {
    const int n = tok[i], p = pgs[i];
    tok[i] = tok_at, pgs[i] = page_at;
    if (blockIdx.x == 0) a.seq_lens[i] = len_of[i] + n;
    tok_at = pg_held_sum(tok_at, n), page_at = pg_held_sum(page_at, p);
  }
  if (t == PT_THREADS - 1) tok[a.batch] = tok_at, pgs[a.batch] = page_at;
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = t; i <= a.batch; i += PT_THREADS) a.cu_new[i] = tok[i];
    if (t == 0) a.free_left[0] = count - pgs[a.batch];  // (below zero: as many pages were missing)
  }
  auto from_stack = [&](int i) {  // the i-th page that the step opens
    const int id = i < count ? a.free_pages[count - 1 - i] : -1;
    return (unsigned)id < (unsigned)a.num_pages ? id : -1;
  };
  const int gid = blockIdx.x * PT_THREADS + t;
  for (int i = gid; i < pgs[a.batch]; i += gridDim.x * PT_THREADS) {  // (as many as tokens at most, unless those are capped)
    const int b = pg_holder(pgs, a.batch, i);
    a.table[b * a.table_stride + pages(len_of[b]) + (i - pgs[b])] = from_stack(i);
  }
  if (gid >= a.max_tokens) return;
  int64_t slot = -1;
  int pos = 0;
  if (gid < tok[a.batch]) {
    const int b = pg_holder(tok, a.batch, gid), len = len_of[b];
    pos = len + (gid - tok[b]);
    const int page = pos >> a.shift, have = pages(len);
    if (page < a.width) {
      int id = page < have ? a.table[b * a.table_stride + page] : from_stack(pgs[b] + page - have);
      if ((unsigned)id < (unsigned)a.num_pages) slot = ((int64_t)id << a.shift) + (pos & (P - 1));
    }
  }
  a.slots[gid] = slot;
  a.positions[gid] = pos;
}

static int page_shift(int64_t page_size) {  // -1: not a page size
  for (int s = 4; s <= 10; ++s)
    if (page_size == 1ll << s) return s;
  return -1;
}

static int tables_launch(const char* who, const sp_paged_tables_args* x, bool truncate) {
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->batch > 0 && x->table_width > 0 && x->num_pages >= 0 && x->free_room >= 0 && x->max_tokens >= 0, SP_ERR_INVALID_ARGUMENT,
             "%s: batch=%lld table_width=%lld num_pages=%lld free_room=%lld max_tokens=%lld", who, (long long)x->batch, (long long)x->table_width,
             (long long)x->num_pages, (long long)x->free_room, (long long)x->max_tokens);
  SP_REQUIRE(x->lens && x->new_lens && x->block_table && (x->free_pages || x->free_room == 0) && x->free_count && x->seq_lens && x->cu_new &&
                 x->free_left && ((x->slots && x->positions) || x->max_tokens == 0),
             SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  const int32_t* const in[3] = {x->lens, x->new_lens, x->free_count};
  for (const int32_t* p : in)
    SP_REQUIRE(p != x->seq_lens && p != x->cu_new && p != x->free_left, SP_ERR_INVALID_ARGUMENT, "%s: an output is an input", who);
  SP_REQUIRE(x->table_stride >= x->table_width || x->batch == 1, SP_ERR_INVALID_ARGUMENT, "%s: rows of %lld entries overlap at a stride of %lld", who,
             (long long)x->table_width, (long long)x->table_stride);
  SP_REQUIRE(x->batch <= PG_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, PG_MAX_SEQS);
  const int shift = page_shift(x->page_size);
  SP_REQUIRE(shift >= 0, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  SP_REQUIRE(x->table_width <= PG_MAX_KEYS && x->table_width << shift <= PG_MAX_KEYS && x->max_tokens <= PG_MAX_KEYS && x->num_pages <= 0x7fffffffll &&
                 x->free_room <= 0x7fffffffll,
             SP_ERR_UNSUPPORTED, "%s: table_width=%lld max_tokens=%lld num_pages=%lld free_room=%lld too large", who, (long long)x->table_width,
             (long long)x->max_tokens, (long long)x->num_pages, (long long)x->free_room);
  const TablesArgs a = {x->lens, x->new_lens, x->block_table, x->table_stride, x->free_pages, x->free_count, (int)x->batch, shift,
                        (int)x->table_width, (int)x->num_pages, (int)x->free_room, (int)x->max_tokens, x->seq_lens, x->cu_new, x->slots,
                        x->positions, x->free_left};
  const unsigned grid = x->max_tokens > 0 ? (unsigned)sp_ceil_div(x->max_tokens, PT_THREADS) : 1u;
  hipLaunchKernelGGL(truncate ? sp_paged_tables_kernel<true> : sp_paged_tables_kernel<false>, dim3(grid), dim3(PT_THREADS),
                     (3 * x->batch + 2) * sizeof(int), (hipStream_t)x->stream, a);
  SP_LAUNCH_CHECK();
  return SP_OK;
}

extern "C" int sp_paged_tables(const sp_paged_tables_args* x) { return tables_launch("sp_paged_tables", x, false); }
extern "C" int sp_paged_tables_truncated(const sp_paged_tables_args* x) { return tables_launch("sp_paged_tables_truncated", x, true); }

// ---- new keys and values into their pages ---------------------------------------------------------------------------------
#define PW_THREADS 256
#define PW_MAX_ITEMS (1ll << 30)  // of a launch: items and their numbers past the end stay below 2^31

typedef uint32_t pw_u32x4 __attribute__((ext_vector_type(4)));

struct WriteArgs {
  const sp_bf16 *k, *v;
  sp_bf16 *k_pages, *v_pages;
  const int64_t* slots;
  int64_t room;               // tokens of the pool
  int items, shift;           // 16-byte chunks of k, below 2^31
  PgDivisor chunks, hkv;      // of a row, rows of a token
  int64_t k_n, k_h, v_n, v_h;
  int64_t kp_p, kp_n, kp_h, vp_p, vp_n, vp_h;
};

// pages[slot / P][h][slot % P] = x[t][h] for k and v: a copy, HBM-bound.  A thread moves 16 bytes of either; the chunks of a token's heads
// lie side by side over the lanes, as projections leave them.  us for 16384 tokens of 8 heads of 128 channels, 4 / 2 / 1 chunks a thread 29.8 /
// 28.5 / 27.4 (4.9 TB/s), for 8 tokens 3.1 / 2.2 / 1.9 (quotients of 64 bits: 3.9).  Stores past the caches would take 25.6 alone, but attention
// reads the pages next: of both together 4096 tokens 169 / 170.5, 16384 the same.
__global__ __launch_bounds__(PW_THREADS) void sp_paged_write_kernel(WriteArgs a) {
  const unsigned item = blockIdx.x * PW_THREADS + threadIdx.x;
  if (item >= (unsigned)a.items) return;
  const unsigned row = pg_div(item, a.chunks);
  const int64_t t = pg_div(row, a.hkv);  // (token, head)
  const int c = (int)(item - row * a.chunks.by) * 8, h = (int)(row - (unsigned)t * a.hkv.by);
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.room) return;
  const int64_t page = slot >> a.shift, in = slot & ((1 << a.shift) - 1);
  const pw_u32x4 kx = *reinterpret_cast<const pw_u32x4*>(a.k + t * a.k_n + h * a.k_h + c);
  const pw_u32x4 vx = *reinterpret_cast<const pw_u32x4*>(a.v + t * a.v_n + h * a.v_h + c);
  *reinterpret_cast<pw_u32x4*>(a.k_pages + page * a.kp_p + in * a.kp_n + h * a.kp_h + c) = kx;
  *reinterpret_cast<pw_u32x4*>(a.v_pages + page * a.vp_p + in * a.vp_n + h * a.vp_h + c) = vx;
}

extern "C" int sp_paged_cache_write_bf16(const sp_paged_write_args* x) {
  const char* who = "sp_paged_cache_write_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->tokens >= 0 && x->hkv > 0 && x->num_pages >= 0, SP_ERR_INVALID_ARGUMENT, "%s: tokens=%lld hkv=%lld num_pages=%lld", who,
             (long long)x->tokens, (long long)x->hkv, (long long)x->num_pages);
  SP_REQUIRE(x->d > 0 && x->d % 8 == 0 && x->d <= 65536, SP_ERR_UNSUPPORTED, "%s: head_dim %lld (a multiple of 8)", who, (long long)x->d);
  const int shift = page_shift(x->page_size);
  SP_REQUIRE(shift >= 0, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  if (x->tokens == 0 || x->num_pages == 0) return SP_OK;
  const int64_t k_n = pg_used_stride(x->k_stride_n, x->tokens), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  const int64_t v_n = pg_used_stride(x->v_stride_n, x->tokens), v_h = pg_used_stride(x->v_stride_h, x->hkv);
  const int64_t kp_p = pg_used_stride(x->k_stride_page, x->num_pages), kp_h = pg_used_stride(x->k_stride_page_h, x->hkv);
  const int64_t vp_p = pg_used_stride(x->v_stride_page, x->num_pages), vp_h = pg_used_stride(x->v_stride_page_h, x->hkv);
  SP_REQUIRE(x->k && x->v && x->k_pages && x->v_pages && x->slots, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->k | (uintptr_t)x->v | (uintptr_t)x->k_pages | (uintptr_t)x->v_pages) % 16 == 0 &&
                 (k_n | k_h | v_n | v_h | kp_p | x->k_stride_slot | kp_h | vp_p | x->v_stride_slot | vp_h) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  SP_REQUIRE(x->tokens <= (1ll << 40) && x->hkv <= 65536 && x->num_pages <= 0x7fffffffll, SP_ERR_UNSUPPORTED,
             "%s: tokens=%lld hkv=%lld num_pages=%lld too many", who, (long long)x->tokens, (long long)x->hkv, (long long)x->num_pages);
  const int64_t of_token = x->hkv * (x->d / 8), most = PW_MAX_ITEMS / of_token;
  SP_REQUIRE(most > 0, SP_ERR_UNSUPPORTED, "%s: hkv=%lld head_dim=%lld too large", who, (long long)x->hkv, (long long)x->d);
  for (int64_t t = 0; t < x->tokens; t += most) {
    const int items = (int)((x->tokens - t < most ? x->tokens - t : most) * of_token);
    const WriteArgs a = {(const sp_bf16*)x->k + t * k_n, (const sp_bf16*)x->v + t * v_n, (sp_bf16*)x->k_pages, (sp_bf16*)x->v_pages,
                         x->slots + t, x->num_pages << shift, items, shift, pg_divisor((unsigned)(x->d / 8)), pg_divisor((unsigned)x->hkv),
                         k_n, k_h, v_n, v_h, kp_p, x->k_stride_slot, kp_h, vp_p, x->v_stride_slot, vp_h};
    hipLaunchKernelGGL(sp_paged_write_kernel, dim3((unsigned)sp_ceil_div(items, PW_THREADS)), dim3(PW_THREADS), 0, (hipStream_t)x->stream, a);
  }
  SP_LAUNCH_CHECK();
  return SP_OK;
}

// ---- new keys' weights ------------------------------------------------------------------------------------------------------
struct ClearArgs {
  float* weights;
  const int64_t* slots;
  int64_t room, w_p, w_h;
  int items, shift;
  PgDivisor hkv;
};

// weights[slot / P][h][slot % P] = 0, a thread for every token and head.  Latency: 2 us for 1024 tokens of 8 heads, 4 for 16384.
__global__ __launch_bounds__(PW_THREADS) void sp_paged_weights_clear_kernel(ClearArgs a) {
  const unsigned item = blockIdx.x * PW_THREADS + threadIdx.x;
  if (item >= (unsigned)a.items) return;
  const unsigned t = pg_div(item, a.hkv);
  const int64_t slot = a.slots[t], h = item - t * a.hkv.by;
  if (slot < 0 || slot >= a.room) return;
  a.weights[(slot >> a.shift) * a.w_p + h * a.w_h + (slot & ((1 << a.shift) - 1))] = 0.f;
}

extern "C" int sp_paged_weights_clear(float* weights, const int64_t* slots, int64_t tokens, int64_t hkv, int64_t num_pages, int64_t page_size, int64_t w_stride_page,
                                      int64_t w_stride_h, sp_stream_t stream) {
  const char* who = "sp_paged_weights_clear";
  SP_REQUIRE(tokens >= 0 && hkv > 0 && num_pages >= 0, SP_ERR_INVALID_ARGUMENT, "%s: tokens=%lld hkv=%lld num_pages=%lld", who, (long long)tokens, (long long)hkv,
             (long long)num_pages);
  const int shift = page_shift(page_size);
  SP_REQUIRE(shift >= 0, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)page_size);
  if (tokens == 0 || num_pages == 0) return SP_OK;
  SP_REQUIRE(weights && slots, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(hkv <= 65536 && num_pages <= 0x7fffffffll && tokens <= PW_MAX_ITEMS / hkv, SP_ERR_UNSUPPORTED, "%s: tokens=%lld hkv=%lld num_pages=%lld too many", who,
             (long long)tokens, (long long)hkv, (long long)num_pages);
  const ClearArgs a = {weights, slots, num_pages << shift, pg_used_stride(w_stride_page, num_pages), pg_used_stride(w_stride_h, hkv), (int)(tokens * hkv), shift,
                       pg_divisor((unsigned)hkv)};
  hipLaunchKernelGGL(sp_paged_weights_clear_kernel, dim3((unsigned)sp_ceil_div(a.items, PW_THREADS)), dim3(PW_THREADS), 0, (hipStream_t)stream, a);
  SP_LAUNCH_CHECK();
  return SP_OK;
}
