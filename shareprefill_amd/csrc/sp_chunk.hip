// Attention of new tokens over what a sequence has cached, in pages (sp_paged_attn_bf16) or in contiguous tensors with a sliding window
// (sp_window_attn_bf16).  Query i of a sequence of q_len queries and len keys stands at position p = len - q_len + i and sees the keys
//   j <= p with (j > p - window or j < sinks):   out = sum_j exp(scale q . k_j) v_j / sum_j exp(scale q . k_j)
// in one pass over the keys with a running maximum and sum; a query that sees nothing is zero.
//
// The tile loop is that of the short-prompt kernel (sp_attn_short.hip): 4 waves of 32 rows, K and V tiles of 64 keys double-buffered
// in LDS by direct loads, S^T = K . Q^T, P^T from its accumulators in place, V by the transposing LDS read.  What differs:
//   * a row is a (token, query head of the kv group) pair, the heads of a token side by side, so that a few new tokens fill a tile's 128
//     rows as far as they can and all heads of the group share its keys: a chunk of 32 tokens of 4 heads reads the cache once;
//   * a load's address comes from the sequence's table.  A wave holds 64 entries of it, a lane each; a load instruction covers 4 rows (8 of
//     64 channels), which lie in one page, so a page is a scalar: a buffer descriptor of its own, whose length ends with the sequence: rows
//     behind it, and pages that are none, read as zeros, whatever a page's unused end holds;
//   * tiles in front of the window that hold no sinks are left out, and only tiles that some row of the wave sees in part are masked;
//   * where a launch has few row tiles their tiles form a line that is cut into equal parts, one workgroup each (sp_paged_plan.h): every CU
//     has as much to do as the others, whatever the sequences' lengths, which only the device knows.  A row tile that a cut goes through
//     leaves fp32 partials that a second launch merges; the lengths need no host, so the call can be captured into a graph.
#include "sp_chunk.h"
#include "sp_tiles.h"

#define CK_LDS_BYTES(D) (4 * AS_TILE * (D) * 2)

// the sequence that row tile number x belongs to, by 64 candidates at a time
__device__ __forceinline__ int ck_sequence(const CkArgs& a, int x, int lane) {
  int lo = 0, span = a.batch;  // it is one of lo .. lo + span - 1
  while (span > 1) {
    const int step = (span + SP_WAVE - 1) / SP_WAVE;
    const int b = lo + lane * step;
    const bool at_or_behind = lane * step < span && pg_first_slot(ck_start(a, b), a.group, b) <= x;
    const int n = __builtin_popcountll(__ballot(at_or_behind));
    const int at = pg_max(n - 1, 0) * step;
    span = pg_min(step, span - at);
    lo += at;
  }
  return lo;
}

template <int D, bool PAGED>
__global__ __launch_bounds__(AS_THREADS, 2) void sp_chunk_kernel(const CkArgs a) {
  constexpr int QT = 2;                    // 16-row tiles per wave
  constexpr int KS = D / 32, CT = D / 16;  // channel steps of S, channel tiles of O
  constexpr int TILE_BYTES = AS_TILE * D * 2;
  constexpr int CHUNKS = D / 8, ROWS = SP_WAVE / CHUNKS;          // of a row; rows of a load instruction
  constexpr int ITS = AS_TILE / (ROWS * AS_WAVES);                // instructions of a wave for a tile
  extern __shared__ __attribute__((aligned(1024))) char lds[];  // [buffer][K | V]
  const int t = threadIdx.x, lane = t & 63, lq = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t lds_base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
  const int kvh = blockIdx.x % a.hkv, part = blockIdx.x / a.hkv;  // (workgroups of a kv head share an XCD where that works out)

  // ---- which row tiles, and which tiles of the first and the last ----
  int x, x_end, tile_begin = 0, tile_end = 0;  // row tiles x .. x_end, of the last the tiles in front of tile_end
  if (a.parts == 0) {
    x = a.slots - 1 - part;  // (the last rows of a prompt see the most keys)
    x_end = x + 1;
  } else {
    int* const cu_s = reinterpret_cast<int*>(lds);
    int* const len_s = cu_s + a.batch + 1;
    __shared__ int64_t wave_sums[AS_WAVES];
    __shared__ int found[2][2];
    for (int i = t; i <= a.batch; i += AS_THREADS) {
      cu_s[i] = ck_start(a, i);
      if (i < a.batch) len_s[i] = ck_len(a, i);
    }
    __syncthreads();
    // every thread some row tiles in a row: their units, then the line's prefix sums
    const int per = (a.slots + AS_THREADS - 1) / AS_THREADS, x0 = t * per, x1 = pg_min(x0 + per, a.slots);
    auto walk = [&](auto&& visit) {  // visit(x, units in the line, tiles)
      if (x0 >= x1) return;
      int b = 0, hi = a.batch;
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (pg_first_slot(cu_s[mid], a.group, mid) <= x0)
          b = mid;
        else
          hi = mid;
      }
      for (int i = x0; i < x1; ++i) {
        while (b + 1 < a.batch && pg_first_slot(cu_s[b + 1], a.group, b + 1) <= i) ++b;
        const int q_len = pg_max(0, cu_s[b + 1] - cu_s[b]), rt = (int)(i - pg_first_slot(cu_s[b], a.group, b));
        if (rt < 0 || rt >= pg_row_tiles(q_len, a.group)) continue;
        int p0, p1;
        pg_tile_positions(rt, q_len, len_s[b], a.group, &p0, &p1);
        const int tiles = pg_span_units(ck_span(a, p0, p1, PG_TILE));
        visit(i, tiles + PG_OVERHEAD, tiles);
      }
    };
    int64_t mine = 0;
    walk([&](int, int units, int) { mine += units; });
    int64_t at = mine;
#pragma unroll
    for (int o = 1; o < SP_WAVE; o <<= 1) {
      const int64_t y = __shfl_up(at, o, SP_WAVE);
      if (lane >= o) at += y;
    }
    if (lane == SP_WAVE - 1) wave_sums[wave] = at;
    if (t == 0) found[0][0] = found[1][0] = a.slots, found[0][1] = found[1][1] = 0;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < AS_WAVES; ++w) {
      if (w == wave) at += total;
      total += wave_sums[w];
    }
    at -= mine;
    const int64_t parts = pg_parts(total, a.parts, PG_MIN_SHARE);
    const int64_t cut[2] = {part < parts ? pg_cut(total, parts, part) : total, part < parts ? pg_cut(total, parts, part + 1) : total};
    walk([&](int i, int units, int tiles) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (cut[e] >= at && cut[e] < at + units) {
          const int tile = pg_snap(cut[e] - at, tiles, PG_OVERHEAD);
          found[e][0] = tile < tiles || tile == 0 ? i : i + 1;
          found[e][1] = tile < tiles ? tile : 0;
        }
      at += units;
    });
    __syncthreads();
    x = __builtin_amdgcn_readfirstlane(found[0][0]);
    tile_begin = __builtin_amdgcn_readfirstlane(found[0][1]);
    x_end = __builtin_amdgcn_readfirstlane(found[1][0]);
    tile_end = __builtin_amdgcn_readfirstlane(found[1][1]);
  }
  int4 note = make_int4(CK_NONE, -1, 0, 0);

  const uint32_t k_row = (uint32_t)a.sk_n * 2u, v_row = (uint32_t)a.sv_n * 2u;  // bytes
  const int in_tile = wave * ROWS + lane / CHUNKS;                               // the lane's row of its wave's first instruction
  const uint32_t k_lane = (uint32_t)(lane / CHUNKS) * k_row + 16u * ((lane % CHUNKS) ^ as_swz<D>(in_tile));
  const uint32_t v_lane = (uint32_t)(lane / CHUNKS) * v_row + 16u * ((lane % CHUNKS) ^ as_swz_v<D>(in_tile));
  // LDS byte offsets of the lane's operands: K row lq, logical chunk 4 ks + g; V row 4 g + lq / 4, 8-byte piece lq % 4 of the
  // 32 bytes of channel tile ct.  Rows 16 further have the same swizzle.
  const int koff = lq * (D * 2), kswz = as_swz<D>(lq);
  const int vrow = 4 * g + (lq >> 2);
  const int voff = vrow * (D * 2) + 8 * (lq & 1), vswz = as_swz_v<D>(vrow), vhalf = (lq >> 1) & 1;
  const as_bf16x8 ones = __builtin_bit_cast(as_bf16x8, (as_u32x4){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});

  int b = x < a.slots ? __builtin_amdgcn_readfirstlane(ck_sequence(a, x, lane)) : 0;
  for (; x < a.slots && (x < x_end || (x == x_end && tile_end > 0)); ++x, tile_begin = 0) {
    while (b + 1 < a.batch && pg_first_slot(ck_start(a, b + 1), a.group, b + 1) <= x) ++b;
    const int start = ck_start(a, b), q_len = pg_max(0, ck_start(a, b + 1) - start), len = ck_len(a, b);
    const int rt = (int)(x - pg_first_slot(start, a.group, b));
    const int rows = q_len * a.group - rt * PG_ROWS;  // from here to the sequence's end
    if (rt < 0 || rows <= 0) continue;
    int p0, p1;
    pg_tile_positions(rt, q_len, len, a.group, &p0, &p1);
    const PgSpan span = ck_span(a, p0, p1, PG_TILE);
    const int tiles = pg_span_units(span);
    const int i_end = x == x_end ? pg_min(tile_end, tiles) : tiles;
    const bool from_start = tile_begin == 0, to_end = i_end == tiles;  // (uniform)

    // the lane's rows: token, head and position
    int pos[QT];
    as_bf16x8 qb[QT][KS];
    auto row_of = [&](int qt, int* token, int* head) {
      const int r = rt * PG_ROWS + pg_min(wave * 32 + 16 * qt + lq, rows - 1);
      *token = (int)((unsigned)r / (unsigned)a.group);
      *head = kvh * a.group + (r - *token * a.group);
    };
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      int token, head;
      row_of(qt, &token, &head);
      pos[qt] = len - q_len + token;
      const sp_bf16* src = a.q + b * a.sq_b + (int64_t)((PAGED ? start : 0) + token) * a.sq_n + head * a.sq_h + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qb[qt][ks] = __builtin_bit_cast(as_bf16x8, *reinterpret_cast<const uint4*>(src + 32 * ks));
    }
    const bool has_rows = wave * 32 < rows;  // (uniform in the wave)
    // positions of the wave's first and last row
    const int w0 = len - q_len + (int)((unsigned)(rt * PG_ROWS + pg_min(wave * 32, rows - 1)) / (unsigned)a.group);
    const int w1 = len - q_len + (int)((unsigned)(rt * PG_ROWS + pg_min(wave * 32 + 31, rows - 1)) / (unsigned)a.group);

    // ---- the sequence's pages: 64 entries of its table at hand, a lane each, and the 64 behind them on their way ----
    const int32_t* const table = PAGED ? a.table + b * a.table_stride : nullptr;
    int ids = 0, ids_next = 0, ids_group = -2;
    auto entries = [&](int group) {
      const int i = group * SP_WAVE + lane;
      const int id = table[pg_min(i, a.width - 1)];
      return i < a.width && (unsigned)id < (unsigned)a.num_pages ? id : -1;
    };
    auto turn_to = [&](int tile) {  // (a tile's pages lie in one group of 64)
      if constexpr (PAGED) {
        const int group = (int)(((int64_t)tile * AS_TILE) >> a.shift) >> 6;
        if (group != ids_group) {
          ids = group == ids_group + 1 ? ids_next : entries(group);
          ids_next = entries(group + 1);
          ids_group = group;
        }
      }
    };
    const char* const kh = (const char*)(a.k + b * a.sk_b + kvh * a.sk_h);
    const char* const vh = (const char*)(a.v + b * a.sv_b + kvh * a.sv_h);
    auto issue = [&](int tile, int buf) {
      turn_to(tile);
      const uint32_t at = lds_base + (uint32_t)(buf * 2 * TILE_BYTES + wave * 1024);
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const int key = tile * AS_TILE + (it * AS_WAVES + wave) * ROWS;  // the instruction's first
        const int page = key >> a.shift, in = key & ((1 << a.shift) - 1);
        const int id = PAGED ? __builtin_amdgcn_readlane(ids, page & 63) : page;
        // rows from here that are there, as far as this instruction goes
        const int there = id < 0 ? 0 : pg_max(0, pg_min(len - key, ROWS));
        auto load = [&](const char* x, int64_t stride_page, uint32_t row_bytes, uint32_t lane_off, uint32_t to) {
          const char* p = x + (int64_t)pg_max(id, 0) * (stride_page * 2) + (uint64_t)(uint32_t)in * row_bytes;
          const __amdgpu_buffer_rsrc_t rsrc =
              __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, there > 0 ? (int)((uint32_t)(there - 1) * row_bytes + 2u * D) : 0, 0x00027000);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (as_lds_ptr)(uintptr_t)(to + it * AS_WAVES * 1024), 16, (int)lane_off, 0, 0, 0);
        };
        load(kh, a.sk_p, k_row, k_lane, at);
        load(vh, a.sv_p, v_row, v_lane, at + TILE_BYTES);
      }
    };
    auto missing = [&](int tile) {  // bit kt: keys 16 kt .. 16 kt + 15 of the tile have no page
      uint32_t m = 0;
      if constexpr (PAGED) {
        turn_to(tile);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
          m |= (uint32_t)(__builtin_amdgcn_readlane(ids, ((tile * AS_TILE + 16 * kt) >> a.shift) & 63) < 0) << kt;
      }
      return m;
    };

    as_floatx4 o[CT][QT], l[QT];  // l: row sums (ones . P, every row of the tile holds the sum)
    float m[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct][qt] = (as_floatx4){0, 0, 0, 0};
      l[qt] = (as_floatx4){0, 0, 0, 0};
      m[qt] = AS_NO_MAX;
    }

    __syncthreads();  // the LDS is free: the plan has been read, the row tile in front is done with its last tile
    uint32_t lost_next = 0;
    if (tile_begin < i_end) {
      const int tile = pg_span_unit(span, tile_begin);
      issue(tile, 0);
      lost_next = missing(tile);
    }
    for (int i = tile_begin; i < i_end; ++i) {
      const int buf = (i - tile_begin) & 1, tile = pg_span_unit(span, i);
      const uint32_t lost = lost_next;
      // this wave's loads of the tile have landed, and everybody's; the other buffer's readers are done
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (i + 1 < i_end) {
        const int next = pg_span_unit(span, i + 1);
        issue(next, buf ^ 1);
        lost_next = missing(next);
      }
      const int key0 = tile * AS_TILE, key1 = key0 + AS_TILE - 1;
      // (a tile that no row of the wave sees anything of: behind them all, or between the sinks and all windows)
      if (!has_rows || key0 > w1 || (key1 <= w0 - a.window && key0 >= a.sinks)) continue;
      const bool masked = key1 > w0 || (key0 <= w1 - a.window && key1 >= a.sinks) || lost != 0;
      const uint32_t kt_addr = lds_base + (uint32_t)(buf * 2 * TILE_BYTES);
      const uint32_t vt_addr = lds_base + (uint32_t)(buf * 2 * TILE_BYTES + TILE_BYTES + voff);
      constexpr int GR = CT / 4;  // groups of four channel tiles
      as_u32x2 vr[2][8];
      auto fetch_v = [&](auto hc, auto gc) {  // group gc of half hc, into vr[gc & 1] (the first of the next half: where it is free)
        constexpr int hh = decltype(hc)::value, gi = decltype(gc)::value, to = GR == 1 ? hh & 1 : gi & 1;
        as_static_for<0, 4>([&](auto uc) {
          constexpr int u = decltype(uc)::value;
          const uint32_t ad = vt_addr + (uint32_t)(((2 * (4 * gi + u) + vhalf) ^ vswz) << 4);
          vr[to][2 * u] = as_read_tr<hh * 32 * (D * 2)>(ad);
          vr[to][2 * u + 1] = as_read_tr<hh * 32 * (D * 2) + 16 * (D * 2)>(ad);
        });
      };
      as_floatx4 s[4][QT];
      {
        as_u32x4 kr[2][KS];
        auto fetch_k = [&](auto kc) {
          constexpr int kt = decltype(kc)::value;
          as_static_for<0, KS>([&](auto sc) {
            constexpr int ks = decltype(sc)::value;
            kr[kt & 1][ks] = as_read_k<kt * 16 * (D * 2)>(kt_addr + (uint32_t)(koff + (((4 * ks + g) ^ kswz) << 4)));
          });
        };
        fetch_k(std::integral_constant<int, 0>{});
        fetch_k(std::integral_constant<int, 1>{});
        __builtin_amdgcn_s_setprio(1);
        as_static_for<0, 4>([&](auto kc) {
          constexpr int kt = decltype(kc)::value;
          as_wait_k<(kt < 3 ? KS : 0)>(kr[kt & 1]);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s[kt][qt] = (as_floatx4){0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              s[kt][qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(as_bf16x8, kr[kt & 1][ks]), qb[qt][ks], s[kt][qt], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (kt + 2 < 4) fetch_k(std::integral_constant<int, kt + 2>{});
        });
      }
      if (masked) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (((lost >> kt) & 1u) || !pg_sees(pos[qt], key0 + 16 * kt + 4 * g + j, a.window, a.sinks)) s[kt][qt][j] = -INFINITY;
      }
      __builtin_amdgcn_s_setprio(0);
      fetch_v(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
      uint32_t pk[QT][8];
      auto softmax = [&](int qt, int hh) {  // half hh: 32 keys
#pragma unroll
        for (int kt = 2 * hh; kt < 2 * hh + 2; ++kt) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][qt][j], a.scale_log2, -m[qt]));
          pk[qt][2 * kt] = as_pack2(e[0], e[1]);
          pk[qt][2 * kt + 1] = as_pack2(e[2], e[3]);
        }
      };
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        softmax(qt, 0);
        softmax(qt, 1);
      }
      __builtin_amdgcn_s_setprio(1);
      as_static_for<0, 2>([&](auto hc) {
        constexpr int hh = decltype(hc)::value;
        // The running max is lazy: it moves only when some probability came out at 2 or more (or is inf: a row's first keys), and then
        // the probabilities are formed again before they are used.  P enters the product as bf16, rounded at 2^-9 of its value at most;
        // the sums are those of the rounded values.
        uint32_t det = 0u;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int i = 4 * hh; i < 4 * hh + 4; i += 2) det |= pk[qt][i] | pk[qt][i + 1];
        as_wait_v<0>(vr[GR == 1 ? hh & 1 : 0]);  // the half's first group (no read may be in flight across the branch)
        if (__ballot((det & AS_P_TOO_LARGE) != 0u) != 0ull) {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 2 * hh; kt < 2 * hh + 2; ++kt)
              mx = fmaxf(mx, fmaxf(fmaxf(s[kt][qt][0], s[kt][qt][1]), fmaxf(s[kt][qt][2], s[kt][qt][3])));
            const float m_new = fmaxf(m[qt], as_groupmax(mx * a.scale_log2));
            const float alpha = __builtin_amdgcn_exp2f(m[qt] - m_new);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) o[ct][qt] *= alpha;
            l[qt] *= alpha;
            m[qt] = m_new;
            softmax(qt, hh);
            if constexpr (hh == 0) softmax(qt, 1);
          }
        }
        // O += V^T . P: groups of four channel tiles, the next group's operands on their way
        as_bf16x8 p[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          p[qt] = __builtin_bit_cast(as_bf16x8, (as_u32x4){pk[qt][4 * hh], pk[qt][4 * hh + 1], pk[qt][4 * hh + 2], pk[qt][4 * hh + 3]});
        as_static_for<0, GR>([&](auto gc) {
          constexpr int gi = decltype(gc)::value, from = GR == 1 ? hh & 1 : gi & 1;
          if constexpr (gi > 0) as_wait_v<0>(vr[from]);
          if constexpr (gi + 1 < GR)
            fetch_v(hc, std::integral_constant<int, gi + 1>{});
          else if constexpr (hh == 0)
            fetch_v(std::integral_constant<int, 1>{}, std::integral_constant<int, 0>{});
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const as_u32x4 raw = __builtin_shufflevector(vr[from][2 * u], vr[from][2 * u + 1], 0, 1, 2, 3);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              o[4 * gi + u][qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(as_bf16x8, raw), p[qt], o[4 * gi + u][qt], 0, 0, 0);
          }
          if constexpr (gi == 0) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) l[qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[qt], l[qt], 0, 0, 0);
          }
        });
      });
      __builtin_amdgcn_s_setprio(0);
    }

    // ---- what has come of it: the rows, or a partial ----
    const bool whole = from_start && to_end;  // (uniform)
    const int64_t slab = (int64_t)blockIdx.x * 2 + (from_start ? 1 : 0);
    float* const o_to = a.o_part + slab * (PG_ROWS * D);
    float2* const ml_to = a.ml_part + slab * PG_ROWS;
    if (!whole) {
      if (from_start)
        note.y = b, note.z = rt;
      else
        note.x = to_end ? CK_LAST : CK_MIDDLE;
    }
    bool spoilt[QT];  // a NaN in the lane's part of the row
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int in_rows = wave * 32 + 16 * qt + lq;
      const bool mine = in_rows < rows;
      int token, head;
      row_of(qt, &token, &head);
      spoilt[qt] = false;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 4; ++j) spoilt[qt] |= o[ct][qt][j] != o[ct][qt][j];
      spoilt[qt] &= mine;
      if (whole) {
        const float inv_l = l[qt][0] > 0.f || l[qt][0] != l[qt][0] ? 1.0f / l[qt][0] : 0.f;
        // (lane groups 2i and 2i + 1 trade halves of two neighbouring channel tiles: 16 bytes a store, 64 contiguous ones a row)
        sp_bf16* dst = a.out + ((int64_t)(start + token) * (a.hkv * a.group) + head) * D + 16 * (g & 1) + 8 * (g >> 1);
#pragma unroll
        for (int ct = 0; ct < CT; ct += 2) {
          uint32_t w[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            w[u][0] = as_pack2(o[ct + u][qt][0] * inv_l, o[ct + u][qt][1] * inv_l);
            w[u][1] = as_pack2(o[ct + u][qt][2] * inv_l, o[ct + u][qt][3] * inv_l);
          }
          const auto lo = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
          const auto hi = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
          if (mine) *reinterpret_cast<uint4*>(dst + ct * 16) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
        }
      } else if (mine) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<as_floatx4*>(o_to + in_rows * D + 16 * ct + 4 * g) = o[ct][qt];
        if (g == 0) ml_to[in_rows] = make_float2(m[qt], l[qt][0]);
      }
    }
    // A masked key weighs 0, and 0 times an infinity or a NaN of its value has made a NaN of the sum.  Such rows are formed again key by key,
    // from what they see alone; rows whose NaN is their own come to the same again.
#pragma unroll 1
    for (int qt = 0; qt < QT; ++qt) {
      uint64_t rows_left = __ballot(spoilt[qt]);
      rows_left = (rows_left | rows_left >> 16 | rows_left >> 32 | rows_left >> 48) & 0xffffull;
      if (rows_left == 0ull) continue;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above come first
      while (rows_left != 0ull) {
        const int in_rows = wave * 32 + 16 * qt + __builtin_ctzll(rows_left);
        rows_left &= rows_left - 1ull;
        const int r = rt * PG_ROWS + in_rows, token = (int)((unsigned)r / (unsigned)a.group), head = kvh * a.group + (r - token * a.group);
        const int p = len - q_len + token;
        const sp_bf16* qrow = a.q + b * a.sq_b + (int64_t)((PAGED ? start : 0) + token) * a.sq_n + head * a.sq_h;
        constexpr int CL = D / SP_WAVE;  // channels of a lane
        float acc[CL] = {0.f}, sum = 0.f, top = AS_NO_MAX;
        for (int i = tile_begin; i < i_end; ++i) {
          const int key = pg_span_unit(span, i) * AS_TILE + lane, page = key >> a.shift;
          int id = page;
          if constexpr (PAGED) {
            id = page < a.width ? table[page] : -1;
            if ((unsigned)id >= (unsigned)a.num_pages) id = -1;
          }
          const bool seen = id >= 0 && key < len && pg_sees(p, key, a.window, a.sinks);
          const int64_t in = key & ((1 << a.shift) - 1);
          float logit = -INFINITY;
          if (seen) {
            const sp_bf16* krow = (const sp_bf16*)kh + id * a.sk_p + in * a.sk_n;
            float dot = 0.f;
            for (int c = 0; c < D; ++c) dot = __builtin_fmaf(sp_bf16_to_f32(qrow[c]), sp_bf16_to_f32(krow[c]), dot);
            logit = dot * a.scale_log2;
          }
          const float new_top = fmaxf(top, sp_wave_max(logit)), alpha = __builtin_amdgcn_exp2f(top - new_top);
          const float weight = seen ? __builtin_amdgcn_exp2f(logit - new_top) : 0.f;
          sum = sum * alpha + sp_wave_sum(weight);
          top = new_top;
#pragma unroll
          for (int c = 0; c < CL; ++c) acc[c] *= alpha;
          const int64_t v_at = id < 0 ? 0 : id * a.sv_p + in * a.sv_n;
          for (uint64_t left = __ballot(seen); left != 0ull; left &= left - 1ull) {
            const int j = __builtin_ctzll(left);
            const sp_bf16* vrow_j = (const sp_bf16*)vh + __shfl(v_at, j, SP_WAVE) + lane * CL;
            const float w = __shfl(weight, j, SP_WAVE);
#pragma unroll
            for (int c = 0; c < CL; ++c) acc[c] = __builtin_fmaf(w, sp_bf16_to_f32(vrow_j[c]), acc[c]);
          }
        }
#pragma unroll
        for (int c = 0; c < CL; ++c) {
          if (whole)
            a.out[((int64_t)(start + token) * (a.hkv * a.group) + head) * D + lane * CL + c] = sp_f32_to_bf16(sum == 0.f ? 0.f : acc[c] / sum);
          else
            o_to[in_rows * D + lane * CL + c] = acc[c];
        }
        if (!whole && lane == 0) ml_to[in_rows] = make_float2(top, sum);
      }
    }
  }
  if (a.parts != 0 && t == 0) a.notes[blockIdx.x] = note;
}

// ---- host -------------------------------------------------------------------------------------------------
struct CkPlan {
  int64_t slots, grid;
  int parts;
};
// Workgroups that are resident at once: two a CU with 128 channels.
static int ck_places(int d) { return d == 64 ? 768 : 512; }
static CkPlan ck_plan(int64_t tokens, int32_t batch, int32_t hkv, int32_t group, int32_t d) {
  CkPlan p;
  p.slots = pg_slots(tokens, group, batch);
  const int64_t room = ck_places(d) / hkv;
  p.parts = p.slots * hkv >= 4 * ck_places(d) ? 0 : (int)(room < 1 ? 1 : room);
  p.grid = (p.parts == 0 ? p.slots : p.parts) * hkv;
  return p;
}
static size_t ck_workspace_bytes(int64_t tokens, int32_t batch, int32_t hq, int32_t hkv, int32_t d) {
  if (tokens <= 0 || batch <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || (d != 64 && d != 128)) return 0;
  const CkPlan p = ck_plan(tokens, batch, hkv, hq / hkv, d);
  return p.parts == 0 ? 0 : (size_t)p.grid * (2 * PG_ROWS * ((size_t)d * sizeof(float) + sizeof(float2)) + sizeof(int4));
}

static int ck_launch(const char* who, CkArgs& a, int32_t hq, int32_t d, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const CkPlan plan = ck_plan(a.tokens, a.batch, a.hkv, a.group, d);
  SP_REQUIRE(plan.grid <= 0x7fffffffll && (int64_t)a.tokens * a.group < (1ll << 31), SP_ERR_UNSUPPORTED, "%s: %d tokens of %d heads are too many",
             who, a.tokens, hq);
  const size_t need = ck_workspace_bytes(a.tokens, a.batch, hq, a.hkv, d);
  SP_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), SP_ERR_WORKSPACE,
             "%s: workspace too small or misaligned", who);
  a.slots = (int)plan.slots;
  a.parts = plan.parts;
  a.o_part = (float*)workspace;
  a.ml_part = (float2*)(a.o_part + (size_t)plan.grid * 2 * PG_ROWS * d);
  a.notes = (int4*)(a.ml_part + (size_t)plan.grid * 2 * PG_ROWS);
  const size_t plan_lds = (size_t)(2 * a.batch + 1) * sizeof(int);
  const size_t lds = plan_lds > (size_t)CK_LDS_BYTES(d) ? plan_lds : (size_t)CK_LDS_BYTES(d);
  auto go = [&](auto kernel, auto merge) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)plan.grid), dim3(AS_THREADS), lds, s, a);
    if (plan.parts != 0) hipLaunchKernelGGL(merge, dim3((unsigned)plan.grid, PG_ROWS / CM_ROWS), dim3(CM_THREADS), 0, s, a, (int)plan.grid);
  };
  static bool attr_set[64] = {false};  // per device, once (idempotent)
  int dev = 0;
  SP_HIP(hipGetDevice(&dev));
  SP_REQUIRE(dev >= 0 && dev < 64, SP_ERR_UNSUPPORTED, "%s: device index %d", who, dev);
  if (!attr_set[dev]) {
    const void* kernels[4] = {(const void*)sp_chunk_kernel<64, false>, (const void*)sp_chunk_kernel<64, true>,
                              (const void*)sp_chunk_kernel<128, false>, (const void*)sp_chunk_kernel<128, true>};
    for (const void* f : kernels) SP_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, CK_LDS_BYTES(128)));
    attr_set[dev] = true;
  }
  if (d == 64)
    a.table != nullptr ? go(sp_chunk_kernel<64, true>, sp_chunk_merge_kernel<64, PG_ROWS>) : go(sp_chunk_kernel<64, false>, sp_chunk_merge_kernel<64, PG_ROWS>);
  else
    a.table != nullptr ? go(sp_chunk_kernel<128, true>, sp_chunk_merge_kernel<128, PG_ROWS>) : go(sp_chunk_kernel<128, false>, sp_chunk_merge_kernel<128, PG_ROWS>);
  SP_LAUNCH_CHECK();
  return SP_OK;
}

// checks shared by the two entry points
static int ck_check(const char* who, int64_t hq, int64_t hkv, int64_t d, int64_t window, int64_t sinks, double softmax_scale) {
  SP_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0 && hq <= 0x7fffffffll, SP_ERR_INVALID_ARGUMENT, "%s: bad shape hq=%lld hkv=%lld", who,
             (long long)hq, (long long)hkv);
  SP_REQUIRE(d == 64 || d == 128, SP_ERR_UNSUPPORTED, "%s: head_dim %lld unsupported (64 or 128)", who, (long long)d);
  SP_REQUIRE((float)softmax_scale > 0.f, SP_ERR_INVALID_ARGUMENT, "%s: softmax_scale must be > 0", who);
  SP_REQUIRE(window >= 0 && sinks >= 0, SP_ERR_INVALID_ARGUMENT, "%s: window=%lld sinks=%lld", who, (long long)window, (long long)sinks);
  return SP_OK;
}
static int ck_window(int64_t window) { return window == 0 || window > PG_NO_WINDOW ? PG_NO_WINDOW : (int)window; }
// offsets inside the rows of a load have 32 bits
static bool ck_rows_ok(int64_t stride_n) { return stride_n >= 0 && stride_n < (1ll << 24) && stride_n % 8 == 0; }

extern "C" size_t sp_paged_attn_workspace_bytes(int64_t tokens, int32_t batch, int32_t hq, int32_t hkv, int32_t d, int32_t single_tokens) {
  if (single_tokens && tokens > 0 && hq > 0 && hkv > 0 && hq % hkv == 0 && hq / hkv <= PD_MAX_GROUP && (d == 64 || d == 128))
    return pd_workspace_bytes(hkv, d);
  return ck_workspace_bytes(tokens, batch, hq, hkv, d);
}

extern "C" int sp_paged_attn_bf16(const sp_paged_attn_args* x) {
  const char* who = "sp_paged_attn_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  int rc = ck_check(who, x->hq, x->hkv, x->d, x->window, x->sinks, x->softmax_scale);
  if (rc) return rc;
  SP_REQUIRE(x->batch > 0 && x->tokens >= 0 && x->table_width > 0 && x->num_pages > 0, SP_ERR_INVALID_ARGUMENT,
             "%s: batch=%lld tokens=%lld table_width=%lld num_pages=%lld", who, (long long)x->batch, (long long)x->tokens,
             (long long)x->table_width, (long long)x->num_pages);
  SP_REQUIRE(x->batch <= PG_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, PG_MAX_SEQS);
  int shift = 4;
  while (shift <= 10 && x->page_size != 1ll << shift) ++shift;
  SP_REQUIRE(shift <= 10, SP_ERR_UNSUPPORTED, "%s: page size %lld (a power of two from 16 to 1024)", who, (long long)x->page_size);
  SP_REQUIRE(x->tokens <= PG_MAX_KEYS && x->num_pages <= 0x7fffffffll && x->table_width <= PG_MAX_KEYS && x->table_width << shift <= PG_MAX_KEYS,
             SP_ERR_UNSUPPORTED, "%s: tokens=%lld num_pages=%lld table_width=%lld too large", who, (long long)x->tokens, (long long)x->num_pages,
             (long long)x->table_width);
  SP_REQUIRE(x->cu_q != nullptr || x->tokens == x->batch, SP_ERR_INVALID_ARGUMENT, "%s: without cu_q every sequence has one token (%lld for %lld)",
             who, (long long)x->tokens, (long long)x->batch);
  if (x->tokens == 0) return SP_OK;
  SP_REQUIRE(x->q && x->k_pages && x->v_pages && x->block_table && x->seq_lens && x->out, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->q | (uintptr_t)x->k_pages | (uintptr_t)x->v_pages | (uintptr_t)x->out) % 16 == 0 &&
                 (x->q_stride_n | x->q_stride_h | x->k_stride_page | x->k_stride_h | x->v_stride_page | x->v_stride_h) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  SP_REQUIRE(ck_rows_ok(x->k_stride_slot) && ck_rows_ok(x->v_stride_slot), SP_ERR_UNSUPPORTED, "%s: slot strides %lld / %lld unsupported", who,
             (long long)x->k_stride_slot, (long long)x->v_stride_slot);
  CkArgs a = {};
  a.q = (const sp_bf16*)x->q, a.k = (const sp_bf16*)x->k_pages, a.v = (const sp_bf16*)x->v_pages;
  a.table = x->block_table, a.lens = x->seq_lens, a.cu = x->cu_q, a.out = (sp_bf16*)x->out;
  a.table_stride = x->table_stride;
  a.sq_n = x->q_stride_n, a.sq_h = x->q_stride_h;
  a.sk_p = x->k_stride_page, a.sk_n = x->k_stride_slot, a.sk_h = x->k_stride_h;
  a.sv_p = x->v_stride_page, a.sv_n = x->v_stride_slot, a.sv_h = x->v_stride_h;
  a.batch = (int)x->batch, a.tokens = (int)x->tokens, a.width = (int)x->table_width, a.num_pages = (int)x->num_pages, a.shift = shift;
  a.n_queries = 1;
  a.hkv = (int)x->hkv, a.group = (int)(x->hq / x->hkv), a.window = ck_window(x->window), a.sinks = (int)(x->sinks < PG_MAX_KEYS ? x->sinks : PG_MAX_KEYS);
  a.scale_log2 = (float)x->softmax_scale * 1.4426950408889634f;
  if (pd_takes(a)) return pd_launch(who, a, x->table_width << shift, (int)x->d, x->workspace, (size_t)x->workspace_bytes, (hipStream_t)x->stream);
  return ck_launch(who, a, (int)x->hq, (int)x->d, x->workspace, (size_t)x->workspace_bytes, (hipStream_t)x->stream);
}

extern "C" size_t sp_window_attn_workspace_bytes(int32_t batch, int64_t n, int64_t n_keys, int32_t hq, int32_t hkv, int32_t d) {
  (void)n_keys;
  return batch <= 0 || n <= 0 ? 0 : sp_paged_attn_workspace_bytes(batch * n, batch, hq, hkv, d, n == 1);
}

extern "C" int sp_window_attn_bf16(const sp_window_attn_args* x) {
  const char* who = "sp_window_attn_bf16";
  SP_REQUIRE(x != nullptr, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  int rc = ck_check(who, x->hq, x->hkv, x->d, x->window, x->sinks, x->softmax_scale);
  if (rc) return rc;
  SP_REQUIRE(x->batch > 0 && x->n >= 0 && x->n_keys >= x->n, SP_ERR_INVALID_ARGUMENT, "%s: batch=%lld n=%lld n_keys=%lld", who,
             (long long)x->batch, (long long)x->n, (long long)x->n_keys);
  SP_REQUIRE(x->batch <= PG_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %lld (at most %d)", who, (long long)x->batch, PG_MAX_SEQS);
  SP_REQUIRE(x->n_keys <= PG_MAX_KEYS && x->batch * x->n <= PG_MAX_KEYS, SP_ERR_UNSUPPORTED, "%s: batch=%lld n=%lld n_keys=%lld too large", who,
             (long long)x->batch, (long long)x->n, (long long)x->n_keys);
  if (x->n == 0) return SP_OK;
  SP_REQUIRE(x->q && x->k && x->v && x->out, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->q | (uintptr_t)x->k | (uintptr_t)x->v | (uintptr_t)x->out) % 16 == 0 &&
                 (x->q_stride_b | x->q_stride_n | x->q_stride_h | x->k_stride_b | x->k_stride_h | x->v_stride_b | x->v_stride_h) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  SP_REQUIRE(ck_rows_ok(x->k_stride_n) && ck_rows_ok(x->v_stride_n), SP_ERR_UNSUPPORTED, "%s: token strides %lld / %lld unsupported", who,
             (long long)x->k_stride_n, (long long)x->v_stride_n);
  CkArgs a = {};
  a.q = (const sp_bf16*)x->q, a.k = (const sp_bf16*)x->k, a.v = (const sp_bf16*)x->v, a.out = (sp_bf16*)x->out;
  a.shift = 6;  // a tile is a page
  a.sq_b = x->q_stride_b, a.sq_n = x->q_stride_n, a.sq_h = x->q_stride_h;
  a.sk_b = x->k_stride_b, a.sk_n = x->k_stride_n, a.sk_h = x->k_stride_h, a.sk_p = x->k_stride_n << a.shift;
  a.sv_b = x->v_stride_b, a.sv_n = x->v_stride_n, a.sv_h = x->v_stride_h, a.sv_p = x->v_stride_n << a.shift;
  a.batch = (int)x->batch, a.tokens = (int)(x->batch * x->n), a.n_keys = (int)x->n_keys, a.n_queries = (int)x->n;
  a.hkv = (int)x->hkv, a.group = (int)(x->hq / x->hkv), a.window = ck_window(x->window), a.sinks = (int)(x->sinks < PG_MAX_KEYS ? x->sinks : PG_MAX_KEYS);
  a.scale_log2 = (float)x->softmax_scale * 1.4426950408889634f;
  if (pd_takes(a)) return pd_launch(who, a, x->n_keys, (int)x->d, x->workspace, (size_t)x->workspace_bytes, (hipStream_t)x->stream);
  return ck_launch(who, a, (int)x->hq, (int)x->d, x->workspace, (size_t)x->workspace_bytes, (hipStream_t)x->stream);
}
