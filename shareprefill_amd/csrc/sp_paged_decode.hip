// Single new tokens of a batch of sequences over what they have cached, in pages or in contiguous tensors, with or without a window and
// sinks: the mathematics of sp_chunk.hip with one position per sequence, for kv groups of up to 16 query heads.
//
// HBM-bound: the visible K and V rows are read once (4 hkv D bytes a key).  The loop is that of the decode ring kernel (sp_decode.hip): the
// waves of a workgroup take steps of 32 keys in turn, each with a running max and a ring of operands in LDS of its own that direct loads
// fill, no barrier between them, and meet in LDS at the end; the probabilities enter the product with V as two bf16 values, so that outputs
// carry their own rounding and little else.  What differs:
//   * a step's 16-key halves lie in a page each (or in the same one): a buffer descriptor of its own, which ends with the sequence.  A step's
//     table entries are scalar loads that are made a step ahead;
//   * a step that reaches past the window's start, the sinks' end or the sequence's reads zeros for the keys that are not seen: whatever
//     stands there takes no part.  Keys are masked by one word of 32 bits a step;
//   * the sequences' steps form a line per kv head that is cut into equal parts, a workgroup each (sp_paged_plan.h): the lengths are known
//     to the device alone and differ widely, and every CU reads as much as the others.  Sequences that a cut goes through leave partials
//     for a second launch; where no cut pays (short caches, many pairs) a workgroup takes a sequence and there is one launch.
#include "sp_chunk.h"
#include "sp_ring.h"

#define PD_ROWS PD_MAX_GROUP

template <int D>
using PdShape = DsShape<D, D / 16, D == 64 ? 8 : 4, 152>;

template <int D, bool PAGED>
__global__ __launch_bounds__((PdShape<D>::WAVES * SP_WAVE)) void sp_paged_decode_kernel(const CkArgs a) {
  using Shape = PdShape<D>;
  constexpr int CT = Shape::CT, KS = D / 32, WAVES = Shape::WAVES, NB = Shape::NB;
  constexpr int CHUNKS = D / 8, ROWS = SP_WAVE / CHUNKS;  // of a row; rows of a load instruction
  constexpr int HALF = 16 / ROWS;                         // instructions of 16 keys
  __shared__ __attribute__((aligned(1024))) char ring_lds[Shape::LDS_BYTES];
  __shared__ float m_s[WAVES][PD_ROWS], l_s[WAVES][PD_ROWS];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lq = lane & 15, gr = lane >> 4;  // head (or key row, channel) in a 16-wide tile, lane group
  const int g = a.group, kvh = blockIdx.x % a.hkv, part = blockIdx.x / a.hkv;

  // ---- which sequences, and which steps of the first and the last ----
  auto span_of = [&](int len) { return ck_span(a, len - 1, len - 1, DS_KEYS); };
  int b, b_end, begin = 0, end = 0;
  if (a.parts == 0) {
    b = part;
    b_end = part + 1;
  } else {
    // every wave for itself, 64 sequences at a time
    auto sums = [&](int b0, int* steps, int64_t* upto) {  // of the lane's sequence; units up to it, it included
      const int i = b0 + lane;
      *steps = i < a.batch ? pg_span_units(span_of(ck_len(a, i))) : -PD_OVERHEAD;  // (none: no room in the line)
      int64_t at = *steps + PD_OVERHEAD;
#pragma unroll
      for (int o = 1; o < SP_WAVE; o <<= 1) {
        const int64_t y = __shfl_up(at, o, SP_WAVE);
        if (lane >= o) at += y;
      }
      *upto = at;
    };
    int steps = 0;
    int64_t upto = 0, total = 0;
    if (a.batch == 1) {  // (no sums to form: half a microsecond of a chat's step)
      steps = pg_span_units(span_of(ck_len(a, 0)));
      upto = total = steps + PD_OVERHEAD;
    } else {
      for (int b0 = 0; b0 < a.batch; b0 += SP_WAVE) {
        sums(b0, &steps, &upto);
        total += __shfl(upto, SP_WAVE - 1, SP_WAVE);
      }
    }
    const int64_t parts = pg_parts(total, a.parts, PD_MIN_SHARE);
    int seq[2], step[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t cut = part < parts ? pg_cut(total, parts, part + e) : total;
      seq[e] = a.batch, step[e] = 0;
      int64_t before = 0;
      if (cut < total)
        for (int b0 = 0; b0 < a.batch; b0 += SP_WAVE) {
          if (a.batch > SP_WAVE) sums(b0, &steps, &upto);
          const uint64_t here = __ballot(cut < before + upto);
          if (here != 0ull) {
            const int i = __builtin_ctzll(here), n = __shfl(steps, i, SP_WAVE);
            const int at = pg_snap(cut - (before + __shfl(upto, i, SP_WAVE) - n - PD_OVERHEAD), n, PD_OVERHEAD, pg_near(total, parts));
            seq[e] = b0 + i + (at < n || at == 0 ? 0 : 1);
            step[e] = at < n ? at : 0;
            break;
          }
          before += __shfl(upto, SP_WAVE - 1, SP_WAVE);
        }
    }
    b = __builtin_amdgcn_readfirstlane(seq[0]), begin = __builtin_amdgcn_readfirstlane(step[0]);
    b_end = __builtin_amdgcn_readfirstlane(seq[1]), end = __builtin_amdgcn_readfirstlane(step[1]);
  }
  int4 note = make_int4(CK_NONE, 0, 0, 0);

  const uint32_t k_row = (uint32_t)a.sk_n * 2u, v_row = (uint32_t)a.sv_n * 2u;  // bytes
  const uint32_t ring = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)ring_lds + wave * NB * Shape::STEP_BYTES;
  const uint32_t k_at = ring + lq * (D * 2);
  const int v_key = 4 * gr + (lq >> 2);  // row of the transposing read; 16 rows further the swizzle is the same
  const uint32_t v_at = ring + Shape::K_BYTES + v_key * (CT * 32) + 8 * (lq & 3);

  for (bool first = true; b < a.batch && (b < b_end || (b == b_end && end > 0)); ++b, begin = 0) {
    const int len = ck_len(a, b), pos = len - 1;
    const PgSpan span = span_of(len);
    const int steps = pg_span_units(span), s_end = b == b_end ? pg_min(end, steps) : steps;
    const bool from_start = begin == 0, to_end = s_end == steps;  // (uniform)
    const int lo = pos - a.window + 1;                            // the window's first key

    dc_bf16x8 qb[KS];
    {
      const sp_bf16* src = a.q + b * (PAGED ? a.sq_n : a.sq_b) + (int64_t)(kvh * g + (lq < g ? lq : 0)) * a.sq_h + 8 * gr;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const dc_u32x4 raw = *reinterpret_cast<const dc_u32x4*>(src + 32 * ks);
        qb[ks] = __builtin_bit_cast(dc_bf16x8, lq < g ? raw : (dc_u32x4){0, 0, 0, 0});
      }
    }
    const char* const kh = (const char*)(a.k + b * a.sk_b + kvh * a.sk_h);
    const char* const vh = (const char*)(a.v + b * a.sv_b + kvh * a.sv_h);
    // (scalar loads: nothing writes the table during the launch)
    const auto table = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(PAGED ? a.table + b * a.table_stride : nullptr);
    struct Ids {
      int id[2];
    };
    auto entries = [&](int s) {  // pages of a step's halves
      Ids x = {{0, 0}};
      if constexpr (PAGED) {
        const int key0 = pg_span_unit(span, s) * DS_KEYS;
#pragma unroll
        for (int h = 0; h < 2; ++h) x.id[h] = table[pg_min((key0 + 16 * h) >> a.shift, a.width - 1)];
      }
      return x;
    };
    auto low = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
    // A step's loads, K's and V's, and which of its keys are seen.
    auto fetch = [&](int buf, int s, Ids ids) {
      const int key0 = pg_span_unit(span, s) * DS_KEYS;
      uint32_t seen = low(pos + 1 - key0) & (~low(lo - key0) | low(a.sinks - key0));
      const uint32_t at = ring + buf * Shape::STEP_BYTES;
      const char *kp[2], *vp[2];
      int there[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = key0 + 16 * h, in = key & ((1 << a.shift) - 1);
        int id = key >> a.shift;
        if constexpr (PAGED) id = id < a.width && (unsigned)ids.id[h] < (unsigned)a.num_pages ? ids.id[h] : -1;
        there[h] = id < 0 ? 0 : pg_max(0, pg_min(len - key, 16));
        if (id < 0) seen &= h == 0 ? 0xffff0000u : 0x0000ffffu;
        kp[h] = kh + (int64_t)pg_max(id, 0) * (a.sk_p * 2) + (uint64_t)(uint32_t)in * k_row;
        vp[h] = vh + (int64_t)pg_max(id, 0) * (a.sv_p * 2) + (uint64_t)(uint32_t)in * v_row;
      }
      auto load = [&](bool edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          auto half = [&](const char* p, uint32_t row_bytes, uint32_t to, auto&& chunk) {
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                (void*)p, 0, there[h] > 0 ? (int)((uint32_t)(there[h] - 1) * row_bytes + 2u * D) : 0, 0x00027000);
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
              const int row = i * ROWS + lane / CHUNKS;
              uint32_t off = (uint32_t)row * row_bytes + 16u * (uint32_t)chunk(16 * h + row);
              if (edge) off = (seen >> (16 * h + row)) & 1u ? off : 0x7ffffff0u;  // (past the buffer's end: zeros)
              __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ds_lds_ptr)(uintptr_t)(to + (h * HALF + i) * 1024), 16, (int)off, 0, 0, 0);
            }
          };
          half(kp[h], k_row, at, [&](int row) { return (lane % CHUNKS) ^ ds_swz_k<D>(row); });
          half(vp[h], v_row, at + Shape::K_BYTES, [&](int row) { return (lane % CHUNKS) ^ (2 * ds_swz_v<CT>(row)); });
        }
      };
      if (seen == ~0u)
        load(false);
      else
        load(true);
      return seen;
    };

    if (!first) __syncthreads();  // the rings are free
    first = false;
    const int s0 = begin + wave;
    uint32_t seen[NB - 1];
#pragma unroll
    for (int i = 0; i < NB - 1; ++i) {
      seen[i] = 0;
      if (s0 + i * WAVES < s_end) seen[i] = fetch(i, s0 + i * WAVES, entries(s0 + i * WAVES));
    }
    Ids next = {{0, 0}};
    if (s0 + (NB - 1) * WAVES < s_end) next = entries(s0 + (NB - 1) * WAVES);

    ds_floatx4 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = (ds_floatx4){0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;  // of head lq; l: this lane group's keys
    int buf = 0;
    for (int s = s0; s < s_end; s += WAVES) {
      // the step's loads have landed, those of the NB - 2 behind it stay in flight (loads return in order)
      if (s + (NB - 2) * WAVES < s_end)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 2) * Shape::LOADS) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const uint32_t mine = seen[0];
#pragma unroll
      for (int i = 0; i + 1 < NB - 1; ++i) seen[i] = seen[i + 1];
      // (the place that is filled here was read in the step before: those reads' results have been used)
      if (s + (NB - 1) * WAVES < s_end) {
        seen[NB - 2] = fetch(buf == 0 ? NB - 1 : buf - 1, s + (NB - 1) * WAVES, next);
        if (s + NB * WAVES < s_end) next = entries(s + NB * WAVES);
      }
      const uint32_t off = buf * Shape::STEP_BYTES;
      dc_u32x4 kr[2][KS];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kr[i][ks] = ds_read_k(k_at + off + i * 16 * (D * 2) + (((4 * ks + gr) ^ ds_swz_k<D>(lq)) << 4));
      if constexpr (KS == 4)
        asm volatile("s_waitcnt lgkmcnt(0)"
                     : "+v"(kr[0][0]), "+v"(kr[0][1]), "+v"(kr[0][2]), "+v"(kr[0][3]), "+v"(kr[1][0]), "+v"(kr[1][1]), "+v"(kr[1][2]), "+v"(kr[1][3]));
      else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(kr[0][0]), "+v"(kr[0][1]), "+v"(kr[1][0]), "+v"(kr[1][1]));
      ds_u32x2 vr[CT][2];  // on their way under the logits
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const uint32_t at = v_at + off + ((ct ^ ds_swz_v<CT>(v_key)) << 5);
        vr[ct][0] = ds_read_v<0>(at);
        vr[ct][1] = ds_read_v<16 * CT * 32>(at);
      }
      ds_floatx4 sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sc[i] = (ds_floatx4){0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, kr[i][ks]), qb[ks], sc[i], 0, 0, 0);
      }
      float mx = -INFINITY;
      const uint32_t bits = mine >> (4 * gr);  // the lane's keys: 16 i + 4 gr + j
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sc[i][j] = bits & (1u << (16 * i + j)) ? sc[i][j] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, sc[i][j]);
        }
      const float m_new = fmaxf(m, ds_quad_max(mx));
      const float base = m_new == -INFINITY ? 0.f : m_new;   // (no key so far has a finite logit: every weight is exp2(-inf) = 0)
      const float alpha = __builtin_amdgcn_exp2f(m - base);  // 0 in the first step
      float add = 0.f;
      uint32_t hi[4], lw[4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const float p0 = __builtin_amdgcn_exp2f(sc[i][j] - base), p1 = __builtin_amdgcn_exp2f(sc[i][j + 1] - base);
          const uint32_t w = dc_pack2(p0, p1);
          hi[2 * i + j / 2] = w;
          lw[2 * i + j / 2] = dc_pack2(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
          add += p0 + p1;
        }
      l = l * alpha + add;
      m = m_new;
      const dc_bf16x8 ph = __builtin_bit_cast(dc_bf16x8, (dc_u32x4){hi[0], hi[1], hi[2], hi[3]});
      const dc_bf16x8 pl = __builtin_bit_cast(dc_bf16x8, (dc_u32x4){lw[0], lw[1], lw[2], lw[3]});
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(vr[ct][0]), "+v"(vr[ct][1]));
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[ct] *= alpha;
        o[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, __builtin_shufflevector(vr[ct][0], vr[ct][1], 0, 1, 2, 3)), ph, o[ct], 0, 0, 0);
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        o[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, ds_finite(__builtin_shufflevector(vr[ct][0], vr[ct][1], 0, 1, 2, 3))), pl, o[ct], 0, 0, 0);
      buf = buf + 1 == NB ? 0 : buf + 1;
    }
    l = ds_quad_sum(l);
    __syncthreads();  // the rings are free
    auto o_s = reinterpret_cast<float(*)[PD_ROWS][D + 4]>(ring_lds);
    if (lq < g) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<ds_floatx4*>(&o_s[wave][lq][16 * ct + 4 * gr]) = o[ct];
      if (gr == 0) {
        m_s[wave][lq] = m;
        l_s[wave][lq] = l;
      }
    }
    __syncthreads();
    const bool whole = from_start && to_end;
    const int64_t slab = (int64_t)blockIdx.x * 2 + (from_start ? 1 : 0);
    if (!whole) {
      if (from_start)
        note.y = g, note.w = b;
      else
        note.x = to_end ? CK_LAST : CK_MIDDLE;
    }
    for (int i = t; i < g * (D / 4); i += WAVES * SP_WAVE) {
      const int h = i / (D / 4), c = i % (D / 4) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, m_s[w][h]);
      ds_floatx4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        // (a wave without keys, or without a finite logit: 0)
        const float f = m_s[w][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_s[w][h] - top);
        sum += l_s[w][h] * f;
        acc += *reinterpret_cast<const ds_floatx4*>(&o_s[w][h][c]) * f;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // (a sequence without keys: zeros)
        *reinterpret_cast<uint2*>(a.out + ((int64_t)b * a.hkv * g + kvh * g + h) * D + c) =
            make_uint2(dc_pack2(acc[0] * inv, acc[1] * inv), dc_pack2(acc[2] * inv, acc[3] * inv));
      } else {
        *reinterpret_cast<ds_floatx4*>(a.o_part + (slab * PD_ROWS + h) * D + c) = acc;
        if (c == 0) a.ml_part[slab * PD_ROWS + h] = make_float2(fmaxf(top, CK_NO_MAX), sum);
      }
    }
  }
  if (a.parts != 0 && t == 0) a.notes[blockIdx.x] = note;
}

// Sequences that cuts went through, one head a workgroup: groups of D / 4 threads take every so many parts, the groups meet in LDS in order.
#define PD_MERGE_THREADS 256
#define PD_MAX_PARTS 256
template <int D>
__global__ __launch_bounds__(PD_MERGE_THREADS) void sp_paged_decode_merge_kernel(const CkArgs a, int workgroups) {
  constexpr int WIDTH = D / 4, GROUPS = PD_MERGE_THREADS / WIDTH;
  __shared__ float2 ml_s[PD_MAX_PARTS];
  __shared__ __attribute__((aligned(16))) float o_s[GROUPS][D];
  const int t = threadIdx.x, h = blockIdx.y;
  int4 note;
  const int parts = cm_parts(a, workgroups, t & 63, blockIdx.x, &note);
  if (parts == 0) return;
  auto row = [&](int i) {
    return (i == 0 ? (int64_t)blockIdx.x * 2 + 1 : ((int64_t)blockIdx.x + (int64_t)i * a.hkv) * 2) * PD_ROWS + h;
  };
  if (t < parts) ml_s[t] = a.ml_part[row(t)];
  __syncthreads();
  float top = CK_NO_MAX;
  for (int i = 0; i < parts; ++i) top = fmaxf(top, ml_s[i].x);
  const int grp = t / WIDTH, c = t % WIDTH * 4;
  ds_floatx4 acc = {0, 0, 0, 0};
  float sum = 0.f;
#pragma unroll 4
  for (int i = grp; i < parts; i += GROUPS)
    acc += *reinterpret_cast<const ds_floatx4*>(a.o_part + row(i) * D + c) * __builtin_amdgcn_exp2f(ml_s[i].x - top);
  for (int i = 0; i < parts; ++i) sum += ml_s[i].y * __builtin_amdgcn_exp2f(ml_s[i].x - top);
  *reinterpret_cast<ds_floatx4*>(&o_s[grp][c]) = acc;
  __syncthreads();
  if (t >= WIDTH) return;
  acc = (ds_floatx4){0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) acc += *reinterpret_cast<const ds_floatx4*>(&o_s[i][c]);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  *reinterpret_cast<uint2*>(a.out + ((int64_t)note.w * a.hkv * a.group + (blockIdx.x % a.hkv) * a.group + h) * D + c) =
      make_uint2(dc_pack2(acc[0] * inv, acc[1] * inv), dc_pack2(acc[2] * inv, acc[3] * inv));
}

// ---- host -------------------------------------------------------------------------------------------------
bool pd_takes(const CkArgs& a) { return a.cu == nullptr && a.n_queries == 1 && a.group <= PD_ROWS; }

static int pd_parts(int32_t hkv) { return hkv >= PD_MAX_PARTS ? 1 : PD_MAX_PARTS / hkv; }

size_t pd_workspace_bytes(int32_t hkv, int32_t d) {
  return (size_t)pd_parts(hkv) * hkv * (2 * PD_ROWS * ((size_t)d * sizeof(float) + sizeof(float2)) + sizeof(int4));
}

int pd_launch(CkArgs& a, int64_t max_keys, int32_t d, void* workspace, hipStream_t s) {
  if (a.window < PG_NO_WINDOW && (int64_t)a.window + a.sinks + 2 * DS_KEYS < max_keys) max_keys = (int64_t)a.window + a.sinks + 2 * DS_KEYS;
  const int64_t pairs = (int64_t)a.batch * a.hkv, units = sp_ceil_div(max_keys, DS_KEYS) + PD_OVERHEAD;
  const int64_t most = pg_parts(units * a.batch, pd_parts(a.hkv), PD_MIN_SHARE);
  // A workgroup a sequence where that takes the longest of them no longer than even parts and their merging launch, in units (of 64 channels
  // one takes half the time).  A table's width only bounds the lengths, which the host does not know: five eighths of it on average is what lengths
  // spread evenly from a quarter of it up come to, an assumption and no measurement of a server's.  Where it is wider than the caches are long, short
  // ones are cut though whole ones would be faster.
  // us, whole / cut, sequences of up to n keys; 32 heads over 8: 1 of 200 7.3 / 9.7, 1 of 1025 18.8 / 10.0, 16 of 1000 19.7 / 19.2, 64 of 500
  // 23.6 / 27.2, 128 of 2000 143 / 127; 14 over 2 of 64 channels: 1 of 1025 10.0 / 9.2, 16 of 1000 10.0 / 13.0, 128 of 2000 19.7 / 27.4.
  const int64_t whole = sp_ceil_div(pairs, 256) * units;
  const int64_t cut = sp_ceil_div(pairs * units, 256) * (a.lens != nullptr ? 5 : 8) / 8 + (d == 64 ? 34 : 16);
  a.parts = whole <= cut || most == 1 ? 0 : (int)most;
  const int64_t grid = a.parts == 0 ? pairs : (int64_t)a.parts * a.hkv;
  a.o_part = (float*)workspace;
  a.ml_part = (float2*)(a.o_part + (size_t)grid * 2 * PD_ROWS * d);
  a.notes = (int4*)(a.ml_part + (size_t)grid * 2 * PD_ROWS);
  auto go = [&](auto kernel, int waves, auto merge) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(waves * SP_WAVE), 0, s, a);
    if (a.parts != 0) hipLaunchKernelGGL(merge, dim3((unsigned)grid, (unsigned)a.group), dim3(PD_MERGE_THREADS), 0, s, a, (int)grid);
  };
  if (d == 64)
    a.table != nullptr ? go(sp_paged_decode_kernel<64, true>, PdShape<64>::WAVES, sp_paged_decode_merge_kernel<64>)
                       : go(sp_paged_decode_kernel<64, false>, PdShape<64>::WAVES, sp_paged_decode_merge_kernel<64>);
  else
    a.table != nullptr ? go(sp_paged_decode_kernel<128, true>, PdShape<128>::WAVES, sp_paged_decode_merge_kernel<128>)
                       : go(sp_paged_decode_kernel<128, false>, PdShape<128>::WAVES, sp_paged_decode_merge_kernel<128>);
  SP_LAUNCH_CHECK();
  return SP_OK;
}
