// Arguments, lengths and the merging launch that the kernels for many new tokens (sp_chunk.hip) and for single ones
// (sp_paged_decode.hip) share.
#pragma once
#include "sp_common.h"
#include "sp_paged_plan.h"

#define CK_NO_MAX (-1.0e30f)  // running maximum of a row without keys: finite, so its partial weighs 0 beside others and nothing is NaN

struct CkArgs {
  const sp_bf16 *q, *k, *v;
  const int32_t* table;     // [batch][width] pages of 1 << shift keys; null: page i of a sequence is its keys i << shift ..
  const int32_t *lens, *cu;  // per sequence, or null: n_keys keys and n_queries queries each
  sp_bf16* out;             // [tokens][hq][D]
  int64_t table_stride;
  int64_t sq_b, sq_n, sq_h, sk_b, sk_p, sk_n, sk_h, sv_b, sv_p, sv_n, sv_h;  // elements; _b between sequences, _p between pages
  int batch, tokens, width, num_pages, shift, n_keys, n_queries;
  int hkv, group, window, sinks;
  int slots, parts;         // row tiles per kv head; parts of their line at most, or 0: a workgroup per row tile
  float scale_log2;
  float* o_part;            // [workgroup][2][128][D]: its first row tile where that began in an earlier part, its last where that goes on
  float2* ml_part;          // [workgroup][2][128]
  int4* notes;              // [workgroup]
};
// notes of a workgroup: x: its first row tile's part is 0 no partial, 1 the last of the row tile, 2 one in the middle;
// y: >= 0: its last row tile starts here and goes on in the next part: sequence y, row tile z
#define CK_NONE 0
#define CK_LAST 1
#define CK_MIDDLE 2

__device__ __forceinline__ int ck_start(const CkArgs& a, int b) {
  return a.cu != nullptr ? pg_max(0, pg_min(a.cu[b], a.tokens)) : b * a.n_queries;
}
__device__ __forceinline__ int ck_len(const CkArgs& a, int b) { return a.lens != nullptr ? pg_max(0, pg_min(a.lens[b], PG_MAX_KEYS)) : a.n_keys; }

// units of `unit` keys that positions p0 .. p1 see something of; none behind the table's last page
__device__ __forceinline__ PgSpan ck_span(const CkArgs& a, int p0, int p1, int unit) {
  PgSpan s = pg_span(p0, p1, a.window, a.sinks, unit);
  if (a.table != nullptr) {
    s.hi = pg_min(s.hi, ((a.width << a.shift) + unit - 1) / unit);
    s.lo = pg_min(s.lo, s.hi);
    s.front = pg_min(s.front, s.lo);
  }
  return s;
}

// Row tiles that cuts went through: the workgroup whose part such a row tile starts in has noted it, those of the following parts that they
// hold a middle or the last of it.  grid (workgroups of the main launch, bands of 16 rows); sixteen threads a row, the parts in order.
#define CM_ROWS 16
typedef float cm_floatx4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t cm_pack2(float a, float b) { return (uint32_t)sp_f32_to_bf16(a) | (uint32_t)sp_f32_to_bf16(b) << 16; }
// ROWS: of a row tile
#define CM_THREADS 256
template <int D, int ROWS>
__global__ __launch_bounds__(CM_THREADS) void sp_chunk_merge_kernel(const CkArgs a, int workgroups) {
  const int4 note = a.notes[blockIdx.x];
  if (note.y < 0) return;
  const int b = note.y, rt = note.z, t = threadIdx.x, lane = t & 63;
  const int kvh = blockIdx.x % a.hkv;
  const int start = ck_start(a, b), q_len = pg_max(0, ck_start(a, b + 1) - start);
  const int rows = pg_min(q_len * a.group - rt * ROWS, ROWS), row0 = blockIdx.y * CM_ROWS;
  if (row0 >= rows) return;
  int more = 0;  // parts behind the first
  for (;;) {
    const int64_t w = blockIdx.x + (int64_t)(more + 1 + lane) * a.hkv;
    const uint64_t ends = __ballot(w >= workgroups || a.notes[w < workgroups ? w : 0].x != CK_MIDDLE);
    if (ends != 0ull) {
      more += __builtin_ctzll(ends) + 1;
      break;
    }
    more += SP_WAVE;
  }
  const int row = row0 + (t >> 4), c0 = (t & 15) * 4;
  if (row >= rows) return;
  auto slab = [&](int i) { return i == 0 ? (int64_t)blockIdx.x * 2 + 1 : ((int64_t)blockIdx.x + (int64_t)i * a.hkv) * 2; };
  float top = CK_NO_MAX;
  for (int i = 0; i <= more; ++i) top = fmaxf(top, a.ml_part[slab(i) * ROWS + row].x);
  cm_floatx4 acc[D / 64];
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) acc[c] = (cm_floatx4){0, 0, 0, 0};
#pragma unroll 4
  for (int i = 0; i <= more; ++i) {
    const float2 ml = a.ml_part[slab(i) * ROWS + row];
    const float w = __builtin_amdgcn_exp2f(ml.x - top);
    sum += ml.y * w;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      acc[c] += *reinterpret_cast<const cm_floatx4*>(a.o_part + (slab(i) * ROWS + row) * D + 64 * c + c0) * w;
  }
  const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
  const int r = rt * ROWS + row, token = (int)((unsigned)r / (unsigned)a.group), head = kvh * a.group + (r - token * a.group);
  sp_bf16* dst = a.out + ((int64_t)(start + token) * (a.hkv * a.group) + head) * D + c0;
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    *reinterpret_cast<uint2*>(dst + 64 * c) = make_uint2(cm_pack2(acc[c][0] * inv, acc[c][1] * inv), cm_pack2(acc[c][2] * inv, acc[c][3] * inv));
}

// single tokens (sp_paged_decode.hip): groups of up to 16 heads
#define PD_MAX_GROUP 16
bool pd_takes(const CkArgs& a);
size_t pd_workspace_bytes(int32_t hkv, int32_t d);
int pd_launch(const char* who, CkArgs& a, int64_t max_keys, int32_t d, void* workspace, size_t workspace_bytes, hipStream_t s);
