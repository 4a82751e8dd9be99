// Arguments, lengths and the merging launch that the kernels for many new tokens (sp_chunk.hip) and for single ones
// (sp_paged_decode.hip) share.
#pragma once
#include "sp_common.h"
#include "sp_paged_plan.h"

// Running maximum of a row without keys: finite, so its partial weighs 0 beside others and nothing is NaN, and below every logit there is, so that the
// first keys move it and a part's weight is that of its own largest logit.
#define CK_NO_MAX (-0x1.fffffep127f)

struct CkArgs {
  const sp_bf16 *q, *k, *v;
  const int32_t* table;     // [batch][width] pages of 1 << shift keys; null: page i of a sequence is its keys i << shift ..
  const int32_t *lens, *cu;  // per sequence, or null: n_keys keys and n_queries queries each
  sp_bf16* out;             // [tokens][hq][D]
  int64_t table_stride;
  int64_t sq_b, sq_n, sq_h, sk_b, sk_p, sk_n, sk_h, sv_b, sv_p, sv_n, sv_h;  // elements; _b between sequences, _p between pages
  int batch, tokens, width, num_pages, shift, n_keys, n_queries;
  int hkv, group, window, sinks;
  PgDivisor by_group;
  int workgroups;           // of a kv head
  int slots, parts;         // row tile numbers per kv head; parts of their line at most, or 0: row tiles stay whole
  int tiles, together;      // whole ones (pg_deal): of a sequence, sequences dealt at a time
  float scale_log2;
  float* o_part;            // [workgroup][2][rows of a tile][D]: its first row tile where that began in an earlier part, its last where that goes on
  float2* ml_part;          // [workgroup][2][rows of a tile]
  int4* notes;              // [workgroup], and where by_slot is not null [row tile number][kv head]
  int4* by_slot;
  // Groups of sequences over the keys that they share (sp_shared_prefix.hip): what is a sequence above is a group then, its rows' sums are left as they are
  const int32_t* groups;    // first sequences, of n_seqs; a group's pages are those of its first
  float* o_row;             // [token][hq][D], sums of the weights' values
  float2* ml_row;           // [token][hq], maxima and sums of the weights
  int n_seqs;
};
// Notes of a workgroup.  x: the part of its first row tile is no partial, the last of the row tile, or one in the middle; y: rows of the row
// tile that starts here and goes on in the next part, 0: there is none; z: its first row in the sequence, w: the sequence's first token.
// By row tile: x the workgroup that it starts in, the others the same.
#define CK_NONE 0
#define CK_LAST 1
#define CK_MIDDLE 2

__device__ __forceinline__ int ck_start(const CkArgs& a, int b) {
  return a.cu != nullptr ? pg_max(0, pg_min(a.cu[b], a.tokens)) : b * a.n_queries;
}
__device__ __forceinline__ int ck_len(const CkArgs& a, int b) { return a.lens != nullptr ? pg_max(0, pg_min(a.lens[b], PG_MAX_KEYS)) : a.n_keys; }

// units of `unit` keys that positions p0 .. p1 see something of; none behind the table's last page
template <bool WINDOWED = true>
__device__ __forceinline__ PgSpan ck_span(const CkArgs& a, int p0, int p1, int unit) {
  PgSpan s = {0, 0, p1 < 0 ? 0 : p1 / unit + 1};
  if constexpr (WINDOWED) s = pg_span(p0, p1, a.window, a.sinks, unit);
  if (a.table != nullptr) {
    s.hi = pg_min(s.hi, ((a.width << a.shift) + unit - 1) / unit);
    s.lo = pg_min(s.lo, s.hi);
    s.front = pg_min(s.front, s.lo);
  }
  return s;
}

// Row tiles that cuts went through: the workgroup whose part such a row tile starts in has noted it, those of the following parts that they
// hold a middle or the last of it.  grid (row tile numbers, or workgroups of the main launch where those are fewer; bands of BAND rows); 16
// threads a row, sets of them that take every so many parts on a running maximum of their own and meet in LDS.  Latency is what it takes, a
// chain of loads and as many workgroups as there are to place, so one load has the notes of 64 workgroups, the partials are asked for with
// the maxima that they are weighed by, and few row tiles, each of many parts, are spread over more workgroups than many.
// ROWS: of a row tile
#define CM_THREADS 1024
#define CM_AHEAD 4  // parts of a set in flight
typedef float cm_floatx4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t cm_pack2(float a, float b) { return (uint32_t)sp_f32_to_bf16(a) | (uint32_t)sp_f32_to_bf16(b) << 16; }
// parts of a row tile that starts in workgroup w0, 0: none is cut; note: the workgroup's
__device__ __forceinline__ int cm_parts(const CkArgs& a, int workgroups, int lane, int64_t w0, int4* note) {
  for (int first = 0;; first += SP_WAVE) {
    const int64_t w = w0 + (int64_t)(first + lane) * a.hkv;
    const int4 there = a.notes[w < workgroups ? w : w0];
    if (first == 0) {
      note->y = __builtin_amdgcn_readfirstlane(there.y);
      note->z = __builtin_amdgcn_readfirstlane(there.z);
      note->w = __builtin_amdgcn_readfirstlane(there.w);
      if (note->y == 0) return 0;
    }
    const uint64_t ends = __ballot(first + lane > 0 && (w >= workgroups || there.x != CK_MIDDLE));
    if (ends != 0ull) return first + __builtin_ctzll(ends) + 1;
  }
}
template <int D, int ROWS, int BAND, bool RAW = false>  // RAW: sums as they are, into o_row and ml_row
__global__ __launch_bounds__(CM_THREADS) void sp_chunk_merge_kernel(const CkArgs a, int workgroups) {
  constexpr int C4 = D / 64, SETS = CM_THREADS / (16 * BAND);  // 16-byte pieces of a thread
  __shared__ __attribute__((aligned(16))) float o_s[SETS > 1 ? SETS - 1 : 1][BAND][D];
  __shared__ float2 ml_s[SETS][BAND];
  const int t = threadIdx.x, row0 = blockIdx.y * BAND;
  int64_t w0 = blockIdx.x;
  if (a.by_slot != nullptr) {
    const int4 x = a.by_slot[blockIdx.x];
    if (row0 >= x.y) return;
    w0 = x.x;
  }
  int4 note;
  const int parts = cm_parts(a, workgroups, t & 63, w0, &note);
  const int rows = note.y;
  if (row0 >= rows) return;
  const int in_band = (t >> 4) % BAND, set = t / (16 * BAND), c0 = (t & 15) * 4;
  const int row = pg_min(row0 + in_band, rows - 1);
  auto at = [&](int i) { return (i == 0 ? w0 * 2 + 1 : (w0 + (int64_t)i * a.hkv) * 2) * ROWS + row; };
  cm_floatx4 acc[C4];
  float sum = 0.f, top = CK_NO_MAX;
#pragma unroll
  for (int c = 0; c < C4; ++c) acc[c] = (cm_floatx4){0, 0, 0, 0};
  for (int i0 = set; i0 < parts; i0 += SETS * CM_AHEAD) {
    float2 ml[CM_AHEAD];
    cm_floatx4 x[CM_AHEAD][C4];
#pragma unroll
    for (int u = 0; u < CM_AHEAD; ++u) {
      const bool there = i0 + u * SETS < parts;
      const int64_t from = at(there ? i0 + u * SETS : i0);
      ml[u] = a.ml_part[from];
      if (!there) ml[u] = make_float2(CK_NO_MAX, 0.f);
#pragma unroll
      for (int c = 0; c < C4; ++c) x[u][c] = *reinterpret_cast<const cm_floatx4*>(a.o_part + from * D + 64 * c + c0);
    }
    float here = top;
#pragma unroll
    for (int u = 0; u < CM_AHEAD; ++u) here = fmaxf(here, ml[u].x);
    const float before = __builtin_amdgcn_exp2f(top - here);
    top = here;
    sum *= before;
#pragma unroll
    for (int c = 0; c < C4; ++c) acc[c] *= before;
#pragma unroll
    for (int u = 0; u < CM_AHEAD; ++u) {
      // (a part that is not there again: weight 0, whatever was read)
      const float w = i0 + u * SETS < parts ? __builtin_amdgcn_exp2f(ml[u].x - top) : 0.f;
      sum += ml[u].y * w;
      if (i0 + u * SETS < parts)
#pragma unroll
        for (int c = 0; c < C4; ++c) acc[c] += x[u][c] * w;
    }
  }
  if ((t & 15) == 0) ml_s[set][in_band] = make_float2(top, sum);
  if (set > 0) {
#pragma unroll
    for (int c = 0; c < C4; ++c) *reinterpret_cast<cm_floatx4*>(&o_s[set - 1][in_band][64 * c + c0]) = acc[c];
  }
  __syncthreads();
  if (set > 0 || row0 + in_band >= rows) return;
  float all = top;
#pragma unroll
  for (int i = 1; i < SETS; ++i) all = fmaxf(all, ml_s[i][in_band].x);
  const float mine = __builtin_amdgcn_exp2f(top - all);
  sum *= mine;
#pragma unroll
  for (int c = 0; c < C4; ++c) acc[c] *= mine;
#pragma unroll
  for (int i = 1; i < SETS; ++i) {
    const float w = __builtin_amdgcn_exp2f(ml_s[i][in_band].x - all);
    sum += ml_s[i][in_band].y * w;
    if (i < parts) {  // (a set without a part: nothing)
#pragma unroll
      for (int c = 0; c < C4; ++c) acc[c] += *reinterpret_cast<const cm_floatx4*>(&o_s[i - 1][in_band][64 * c + c0]) * w;
    }
  }
  const int r = note.z + row, kvh = (int)(w0 % a.hkv), token = (int)pg_div((unsigned)r, a.by_group), head = kvh * a.group + (r - token * a.group);
  if constexpr (RAW) {
    const int64_t to = (int64_t)(note.w + token) * (a.hkv * a.group) + head;
#pragma unroll
    for (int c = 0; c < C4; ++c) *reinterpret_cast<cm_floatx4*>(a.o_row + to * D + 64 * c + c0) = acc[c];
    if ((t & 15) == 0) a.ml_row[to] = make_float2(all, sum);
    return;
  }
  const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
  sp_bf16* dst = a.out + ((int64_t)(note.w + token) * (a.hkv * a.group) + head) * D + c0;
#pragma unroll
  for (int c = 0; c < C4; ++c)
    *reinterpret_cast<uint2*>(dst + 64 * c) = make_uint2(cm_pack2(acc[c][0] * inv, acc[c][1] * inv), cm_pack2(acc[c][2] * inv, acc[c][3] * inv));
}

// single tokens (sp_paged_decode.hip): groups of up to 16 heads
#define PD_MAX_GROUP 16
// groups over their shared keys (sp_chunk.hip): a's sequences are the groups, each row sees all of its group's keys
size_t ck_groups_workspace_bytes(int32_t hkv, int32_t d);
int ck_groups_launch(CkArgs& a, int32_t d, void* workspace, hipStream_t s);
bool pd_takes(const CkArgs& a);
size_t pd_workspace_bytes(int32_t hkv, int32_t d);
int pd_launch(CkArgs& a, int64_t max_keys, int32_t d, void* workspace, hipStream_t s);
