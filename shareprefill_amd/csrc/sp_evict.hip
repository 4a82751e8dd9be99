// Eviction from a paged cache by accumulated attention weight (sp_paged_evict_bf16): of every kv head of a request the first keys, the last ones and
// the `budget` heaviest of those between stay, moved to the front of the request's pages in the order they stood in.
//
// The heaviest are those above the budget-th largest weight T and as many of those equal to it as there is room for, lowest place first.  T is
// found by its bits from above, 11, 10 and 10 of the weight's pattern (finite floats without a sign are ordered as their patterns are), a
// histogram each.  Moving is a gather in place: a kept key comes from its place or further back, so rows are moved front to
// back in tiles that are read before they are written, by one workgroup, and what other rows still need is never overwritten.
// Rows are cut across instead: 64 channels of K or V are a workgroup's.  HBM-bound: kept rows once in and out, weights once in.
#include "sp_common.h"
#include "sp_paged_plan.h"

#define EV_THREADS 1024
#define EV_WAVES (EV_THREADS / SP_WAVE)
#define EV_MAX_SEQS 4096

typedef uint32_t ev_u32x4 __attribute__((ext_vector_type(4)));

struct EvArgs {
  sp_bf16 *k, *v;
  float* weights;
  const int32_t *table, *lens, *first;
  int32_t* new_lens;
  int64_t table_stride, sk_p, sk_n, sk_h, sv_p, sv_n, sv_h, sw_p, sw_h;
  int batch, hkv, d, width, num_pages, shift, budget, recent;
  int32_t* list;  // [request][kv head][budget]: places of the heaviest, behind the first keys
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

__global__ __launch_bounds__(EV_THREADS) void sp_evict_select_kernel(const EvArgs a) {
  __shared__ int hist[2048];
  __shared__ int wave_s[2][EV_WAVES];
  __shared__ int found_s[2];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int b = blockIdx.x / a.hkv, kvh = blockIdx.x % a.hkv;
  const EvRequest r = ev_request(a, b);
  const bool goes = r.keep < r.mid && ev_has_pages(a, b, r);
  if (kvh == 0 && t == 0) a.new_lens[b] = goes ? r.len - r.mid + r.keep : r.len;
  if (!goes || r.keep == 0) return;
  const int32_t* const table = a.table + b * a.table_stride;
  const float* const w = a.weights + kvh * a.sw_h;
  auto key_at = [&](int i) {  // pattern of the weight at place i behind the first keys
    const int j = r.first + i;
    return sp_sort_key(w[(int64_t)table[j >> a.shift] * a.sw_p + (j & ((1 << a.shift) - 1))]);
  };
  uint32_t top = 0;     // bits of T that are known
  int left = r.keep;    // the left-th largest of those that share them is T
  int shift = 20;
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass == 0 ? 11 : 10;
    for (int i = t; i < 1 << bits; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = t; i < r.mid; i += EV_THREADS) {
      const uint32_t key = key_at(i);
      if (pass == 0 || key >> (shift + bits) == top) atomicAdd(&hist[(key >> shift) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // bins from above, two a thread in the first pass
    const int each = pass == 0 ? 2 : 1, bins = 1 << bits;
    int mine = 0;
    for (int e = 0; e < each; ++e) mine += hist[bins - 1 - (t * each + e)];
    int at = mine;
#pragma unroll
    for (int o = 1; o < SP_WAVE; o <<= 1) {
      const int y = __shfl_up(at, o, SP_WAVE);
      if (lane >= o) at += y;
    }
    if (lane == SP_WAVE - 1) wave_s[0][wave] = at;
    __syncthreads();
    for (int x = 0; x < wave; ++x) at += wave_s[0][x];
    at -= mine;
    for (int e = 0; e < each; ++e) {
      const int bin = bins - 1 - (t * each + e), n = hist[bin];
      if (at < left && left <= at + n) found_s[0] = bin, found_s[1] = left - at;
      at += n;
    }
    __syncthreads();
    top = pass == 0 ? (uint32_t)found_s[0] : top << bits | (uint32_t)found_s[0];
    left = found_s[1];
    shift -= 10;
    __syncthreads();
  }
  // `left` of those equal to T stay
  int32_t* const list = a.list + (int64_t)blockIdx.x * a.budget;
  int kept = 0, equal = 0;  // in front of this chunk
  for (int i0 = 0; i0 < r.mid; i0 += EV_THREADS) {
    const int i = i0 + t;
    const uint32_t key = i < r.mid ? key_at(i) : 0u;
    const bool over = i < r.mid && key > top, same = i < r.mid && key == top;
    const uint64_t overs = __ballot(over), sames = __ballot(same), below = (1ull << lane) - 1ull;
    if (lane == 0) wave_s[0][wave] = __builtin_popcountll(overs), wave_s[1][wave] = __builtin_popcountll(sames);
    __syncthreads();
    int over_at = 0, same_at = equal, overs_all = 0, sames_all = 0;
#pragma unroll
    for (int x = 0; x < EV_WAVES; ++x) {
      const int n = wave_s[0][x], m = wave_s[1][x];
      if (x < wave) over_at += n, same_at += m;
      overs_all += n, sames_all += m;
    }
    // (those equal to T that stay, in front of the lane)
    over_at += __builtin_popcountll(overs & below);
    same_at += __builtin_popcountll(sames & below);
    const int place = kept + over_at + pg_min(same_at, left) - pg_min(equal, left);
    if (over || (same && same_at < left)) list[place] = i;
    kept += overs_all + pg_min(equal + sames_all, left) - pg_min(equal, left);
    equal += sames_all;
    __syncthreads();
  }
}

#define EV_AHEAD 8  // rows of a thread in flight
__global__ __launch_bounds__(EV_THREADS) void sp_evict_move_kernel(const EvArgs a) {
  const int t = threadIdx.x, slices = (a.d + 63) / 64, per = 2 * slices + 1;  // K's, V's, the weights
  const int pair = blockIdx.x / per, part = blockIdx.x % per, b = pair / a.hkv, kvh = pair % a.hkv;
  const EvRequest r = ev_request(a, b);
  if (!(r.keep < r.mid && ev_has_pages(a, b, r))) return;
  const int32_t* const table = a.table + b * a.table_stride;
  const int32_t* const list = a.list + (int64_t)pair * a.budget;
  const int rows = r.keep + r.len - r.first - r.mid, in = (1 << a.shift) - 1;
  auto from = [&](int i) { return r.first + (i < r.keep ? list[i] : r.mid + (i - r.keep)); };
  if (part == per - 1) {
    float* const w = a.weights + kvh * a.sw_h;
    auto at = [&](int j) { return (int64_t)table[j >> a.shift] * a.sw_p + (j & in); };
    for (int i0 = 0; i0 < rows; i0 += EV_THREADS * EV_AHEAD) {
      float x[EV_AHEAD];
#pragma unroll
      for (int u = 0; u < EV_AHEAD; ++u) {
        const int i = i0 + u * EV_THREADS + t;
        if (i < rows) x[u] = w[at(from(i))];
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tile is read
      __syncthreads();
#pragma unroll
      for (int u = 0; u < EV_AHEAD; ++u) {
        const int i = i0 + u * EV_THREADS + t;
        if (i < rows) w[at(r.first + i)] = x[u];
      }
    }
    return;
  }
  const bool is_v = part >= slices;
  const int c = (part % slices) * 64 + (t & 7) * 8;
  const int64_t page_at = is_v ? a.sv_p : a.sk_p, slot_at = is_v ? a.sv_n : a.sk_n;
  sp_bf16* const x = (is_v ? a.v + kvh * a.sv_h : a.k + kvh * a.sk_h) + c;
  auto at = [&](int j) { return x + (int64_t)table[j >> a.shift] * page_at + (int64_t)(j & in) * slot_at; };
  constexpr int ROWS = EV_THREADS / 8;
  for (int i0 = 0; i0 < rows; i0 += ROWS * EV_AHEAD) {
    ev_u32x4 y[EV_AHEAD];
#pragma unroll
    for (int u = 0; u < EV_AHEAD; ++u) {
      const int i = i0 + u * ROWS + (t >> 3);
      if (i < rows && c < a.d) y[u] = *reinterpret_cast<const ev_u32x4*>(at(from(i)));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tile is read
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EV_AHEAD; ++u) {
      const int i = i0 + u * ROWS + (t >> 3);
      if (i < rows && c < a.d) *reinterpret_cast<ev_u32x4*>(at(r.first + i)) = y[u];
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------
extern "C" size_t sp_paged_evict_workspace_bytes(int32_t batch, int32_t hkv, int64_t budget) {
  return batch <= 0 || hkv <= 0 || budget <= 0 ? 0 : (size_t)batch * hkv * (size_t)budget * sizeof(int32_t);
}

extern "C" int sp_paged_evict_bf16(const sp_paged_evict_args* x) {
  const char* who = "sp_paged_evict_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->batch > 0 && x->hkv > 0 && x->table_width > 0 && x->num_pages > 0, SP_ERR_INVALID_ARGUMENT,
             "%s: batch=%lld hkv=%lld table_width=%lld num_pages=%lld", who, (long long)x->batch, (long long)x->hkv, (long long)x->table_width,
             (long long)x->num_pages);
  SP_REQUIRE(x->budget >= 0 && x->recent >= 0, SP_ERR_INVALID_ARGUMENT, "%s: budget=%lld recent=%lld", who, (long long)x->budget, (long long)x->recent);
  SP_REQUIRE(x->d > 0 && x->d % 8 == 0 && x->d <= 65536, SP_ERR_UNSUPPORTED, "%s: head_dim %lld (a multiple of 8)", who, (long long)x->d);
  int shift = 4;
  while (shift <= 10 && x->page_size != 1ll << shift) ++shift;
  SP_REQUIRE(shift <= 10, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  SP_REQUIRE(x->batch <= EV_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, EV_MAX_SEQS);
  const int64_t pairs = x->batch * x->hkv, per = 2 * ((x->d + 63) / 64) + 1;
  SP_REQUIRE(x->hkv <= 65536 && x->num_pages <= 0x7fffffffll && x->table_width <= PG_MAX_KEYS && x->table_width << shift <= PG_MAX_KEYS &&
                 pairs * per <= 0x7fffffffll,
             SP_ERR_UNSUPPORTED, "%s: hkv=%lld num_pages=%lld table_width=%lld too large", who, (long long)x->hkv, (long long)x->num_pages,
             (long long)x->table_width);
  const int64_t k_p = pg_used_stride(x->k_stride_page, x->num_pages), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  const int64_t v_p = pg_used_stride(x->v_stride_page, x->num_pages), v_h = pg_used_stride(x->v_stride_h, x->hkv);
  SP_REQUIRE(x->k_pages && x->v_pages && x->weights && x->block_table && x->seq_lens && x->new_lens, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(x->new_lens != x->seq_lens && x->new_lens != x->first, SP_ERR_INVALID_ARGUMENT, "%s: an output is an input", who);
  SP_REQUIRE(((uintptr_t)x->k_pages | (uintptr_t)x->v_pages) % 16 == 0 && (k_p | k_h | x->k_stride_slot | v_p | v_h | x->v_stride_slot) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  // (a table cannot hold more keys than its width, so no list is longer)
  const int64_t budget = x->budget < x->table_width << shift ? x->budget : x->table_width << shift;
  const size_t need = sp_paged_evict_workspace_bytes((int)x->batch, (int)x->hkv, budget);
  SP_REQUIRE(need == 0 || (x->workspace != nullptr && x->workspace_bytes >= need && (uintptr_t)x->workspace % 16 == 0), SP_ERR_WORKSPACE,
             "%s: workspace missing, too small or misaligned", who);
  EvArgs a = {};
  a.k = (sp_bf16*)x->k_pages, a.v = (sp_bf16*)x->v_pages, a.weights = x->weights;
  a.table = x->block_table, a.lens = x->seq_lens, a.first = x->first, a.new_lens = x->new_lens, a.table_stride = x->table_stride;
  a.sk_p = k_p, a.sk_n = x->k_stride_slot, a.sk_h = k_h, a.sv_p = v_p, a.sv_n = x->v_stride_slot, a.sv_h = v_h;
  a.sw_p = pg_used_stride(x->w_stride_page, x->num_pages), a.sw_h = pg_used_stride(x->w_stride_h, x->hkv);
  a.batch = (int)x->batch, a.hkv = (int)x->hkv, a.d = (int)x->d, a.width = (int)x->table_width, a.num_pages = (int)x->num_pages, a.shift = shift;
  a.budget = (int)budget, a.recent = (int)(x->recent < PG_MAX_KEYS ? x->recent : PG_MAX_KEYS);
  a.list = (int32_t*)x->workspace;
  hipLaunchKernelGGL(sp_evict_select_kernel, dim3((unsigned)pairs), dim3(EV_THREADS), 0, (hipStream_t)x->stream, a);
  hipLaunchKernelGGL(sp_evict_move_kernel, dim3((unsigned)(pairs * per)), dim3(EV_THREADS), 0, (hipStream_t)x->stream, a);
  SP_LAUNCH_CHECK();
  return SP_OK;
}
