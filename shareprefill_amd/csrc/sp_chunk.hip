// Attention of new tokens over what a sequence has cached, in pages (sp_paged_attn_bf16) or in contiguous tensors with a sliding window
// (sp_window_attn_bf16).  Query i of a sequence of q_len queries and len keys stands at position p = len - q_len + i and sees the keys
//   j <= p with (j > p - window or j < sinks):   out = sum_j exp(scale q . k_j) v_j / sum_j exp(scale q . k_j)
// in one pass over the keys with a running maximum and sum; a query that sees nothing is zero.
//
// Rows.  A row is a (token, query head of the kv group) pair, the heads of a token side by side: a few new tokens fill a tile's 256 rows as far
// as they can, and all heads of a group share its keys.  Eight waves of 32 rows work on the same blocks of 128 keys, so K and V are read once
// per 256 rows: with four waves and 128 rows the loads alone held the loop up (2048 tokens over 65001 keys 2630 -> 2330 us).
// Keys.  K and V lie in rings of four sub-tiles of 64 keys each (128 KiB of LDS with 128 channels), filled by direct loads a block ahead; one
// barrier a block.  A wave's own pipeline (sp_pipeline.h: S^T = K . Q^T of a half-tile, the softmax of the one in front and P . V of the one
// in front of that, interleaved instruction by instruction, P^T taken from the accumulators in place, V by the transposing LDS read) keeps the
// matrix cores fed: 2330 -> 2004 us.
// Pages.  A load's address comes from the sequence's table: a lane holds a page's addresses and length, and a load takes them by lane reads
// into a buffer descriptor that ends with the sequence, so rows behind it, and pages that are none, read as zeros, whatever stands there.
// Masks.  Blocks in front of the window that hold no sinks are left out; a wave masks only what its rows see in part.
// Workgroups, one a CU, stay for the launch: the next row tile's first keys and its queries land under the end of the one in front
// (30001 tokens in a window of 4096 2282 -> 1811 us).  The row tiles' blocks form a line that is cut into equal parts, one workgroup each
// (sp_paged_plan.h): every CU has as much to do as the others, whatever the sequences' lengths, which only the device knows; row tiles that a
// cut goes through leave fp32 partials that a second launch merges.  No length comes to the host, so the call can be captured into a graph.
// What it reaches, head_dim 128, 32 heads over 8: 2048 tokens over 65001 keys in pages of 128 1760 to 1830 us by card, 1170 to 1220 TFLOP/s, the
// rate of a large bf16 matrix product; 30001 tokens in a window of 4096 1150 to 1200.  Short calls: some 8 us go by until the line is laid out
// and the first keys have landed, a row tile's turn takes 5 us beside its blocks of 3.5 us each, partials and their merging 15 us.
#include "sp_chunk.h"
#include "sp_pipeline.h"

// Octaves that a moved maximum is set above the largest logit.  A wave that moves its rows' maxima (some probability came out at 2) forms them
// again and rescales its sums while the other seven wait at the block's barrier, and in a row's first thousand keys some wave does in nearly
// every block.  us, 0 / 3 / 5 / 7 octaves: 8192 tokens in a window of 1024 178 / 151.5 / 148.2 / 147.1, 30001 in 4096 1850 / 1663 / 1657 / 1654, 512
// over 8192 94.5 / 84.9 / 84.1 / 84.2, 16384 without a window - / 1796 / 1778 / 1777.  What it costs: the largest probability need not be a power of
// two, which bf16 holds exactly; outputs are 2.14e-3 / 2.22e-3 / 2.23e-3 / 2.23e-3 from 64 bits, 1.6e-3 of it their own rounding.
#define CK_SLACK 7
// Largest magnitude of a row's maximum, in octaves, up to which its probabilities are what the loop forms: exponents of the exact product less a
// maximum that is rounded, off by that rounding for all of a row's keys alike and near nothing.  Beyond it they may all be zero, and the rows are
// formed again from rounded products, whose largest is the maximum itself.
#define CK_FAR 0x1p24f
#define CK_WAVES 8
#define CK_THREADS (CK_WAVES * SP_WAVE)
#define CK_ROWS (32 * CK_WAVES)  // of a row tile
#define CK_SUB 64                // keys of a sub-tile
#define CK_BLOCK (2 * CK_SUB)    // keys of a block, two sub-tiles of a walk: what lies between two barriers
#define CK_RING 4                // sub-tiles of K in LDS, and of V
#define CK_SUB_BYTES(D) (CK_SUB * (D) * 2)
#define CK_LDS_BYTES(D) (2 * CK_RING * CK_SUB_BYTES(D))  // the rings; offsets and lengths of the sequences stand behind them
#define CK_MAX_SEQS 2048  // their offsets and lengths take 16 KiB of LDS

typedef __attribute__((address_space(3))) void* ck_lds_ptr;
typedef uint32_t ck_u32x2 __attribute__((ext_vector_type(2)));

// K and V sub-tiles are [64 keys][D] bf16 in 16-byte chunks, the chunk index XOR-swizzled by the row so that each kind of operand read is
// free of bank conflicts: K's single chunks (16 rows of one chunk), V's pairs (the transposing read takes two neighbouring chunks of
// 8 rows).  Rows of 64 channels are half a bank cycle long: two of them share a swizzle.
template <int D>
__device__ __forceinline__ int ck_swz_k(int row) {
  return D == 128 ? (row & 15) : ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int ck_swz_v(int row) {
  return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
}

// Operands of a block (sp_pipeline.h): sub-tiles 2b and 2b + 1 of K, 2b - 1 (VB 0) and 2b (VB 1) of V.  A V^T operand is two transposing
// reads of 16 keys each; S^T leaves a lane with keys 4g .. 4g + 3 of either 16-key tile, which is what the two deliver.
template <int D>
struct CkAddr {
  static constexpr int V_READS = 2;
  uint32_t ka, va[2];
  template <int KQ, int KS, int T>
  __device__ __forceinline__ bf16x8 k() const {
    return at_lds128_async<(KQ >> 1) * CK_SUB_BYTES(D) + ((KQ & 1) * 32 + T * 16) * (D * 2)>(ka ^ (uint32_t)(KS << 6));
  }
  template <int VB, int KT, int I>
  __device__ __forceinline__ bf16x8 v() const {
    const uint32_t at = va[VB] ^ (uint32_t)(I << 5);
    ck_u32x2 lo, hi;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(lo) : "v"(at), "n"(KT * 32 * (D * 2)));
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(at), "n"((KT * 32 + 16) * (D * 2)));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3));
  }
};

// stages of matrix instructions alone: a walk's first S, its last P . V
template <int KQ, bool HALF, class Addr>
__device__ __forceinline__ void ck_qk_only(const Addr& ad, const bf16x8 (&qb)[2][4], floatx4 (&s_out)[2][2]) {
  constexpr int QS = HALF ? 4 : 8;
  bf16x8 a[QS];  // slot i: channel step i / 2, key tile i % 2
  auto fetch = [&](auto kc) {
    constexpr int i = decltype(kc)::value;
    a[i] = ad.template k<KQ, (i >> 1), (i & 1)>();
  };
  at_static_for<0, 2>(fetch);
  AT_PIN();
  at_static_for<0, QS>([&](auto kc) {
    constexpr int i = decltype(kc)::value;
    AT_WAIT_LGKM(i + 1 < QS ? 1 : 0);
    AT_PIN();
    if constexpr (i + 2 < QS) fetch(std::integral_constant<int, i + 2>{});
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      if ((i >> 1) == 0)
        at_mfma_first(s_out[i & 1][qt], a[i], qb[qt][0]);
      else if (i == QS - 1 && qt == 1)  // the last one: the softmax of the next stage reads S_out right away
        at_mfma_acc_settled(s_out[i & 1][qt], a[i], qb[qt][i >> 1]);
      else
        at_mfma_acc(s_out[i & 1][qt], a[i], qb[qt][i >> 1]);
    }
    AT_PIN();
  });
}
template <int VB, int KT, bool HALF, class Addr>
__device__ __forceinline__ void ck_pv_only(const Addr& ad, const bf16x8 (&p)[2], floatx4 (&o)[9][2], const bf16x8& ones) {
  constexpr int PS = HALF ? 4 : 8;
  bf16x8 a[PS];  // slot i: channel tile i
  auto fetch = [&](auto kc) {
    constexpr int i = decltype(kc)::value;
    a[i] = ad.template v<VB, KT, i>();
  };
  at_static_for<0, 2>(fetch);
  AT_PIN();
  at_static_for<0, PS>([&](auto kc) {
    constexpr int i = decltype(kc)::value;
    AT_WAIT_LGKM(i + 1 < PS ? Addr::V_READS : 0);
    AT_PIN();
    if constexpr (i + 2 < PS) fetch(std::integral_constant<int, i + 2>{});
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) at_mfma_acc(o[i][qt], a[i], p[qt]);
    AT_PIN();
  });
  at_mfma_acc(o[8][0], ones, p[0]);
  at_mfma_acc_settled(o[8][1], ones, p[1]);  // the end of the walk: the epilogue reads O next
}

// blocks of a walk of sub-tiles; the second one of the last block may lie behind them all
__host__ __device__ static inline int ck_blocks(const PgSpan& s) { return (pg_span_units(s) + 1) >> 1; }

// the sequence that row tile number x belongs to, by 64 candidates at a time.  cu: offsets in order
template <int ROWS>
__device__ __forceinline__ int ck_sequence(const CkArgs& a, const int* cu, int x, int lane) {
  int lo = 0, span = a.batch;  // it is one of lo .. lo + span - 1
  while (span > 1) {
    const int step = (span + SP_WAVE - 1) / SP_WAVE;
    const int b = lo + lane * step;
    const bool at_or_behind = lane * step < span && pg_first_slot(cu[b], a.group, b, ROWS) <= x;
    const int n = __builtin_popcountll(__ballot(at_or_behind));
    const int at = pg_max(n - 1, 0) * step;
    span = pg_min(step, span - at);
    lo += at;
  }
  return lo;
}

// WINDOWED: blocks are made of any two sub-tiles of a walk, so that a window's start and the sinks cost a sub-tile, not a block: 8192 tokens in a
// window of 1024 with 4 sinks 155 -> 151 us.  Without a window a block is 128 keys in a row, and nothing asks for windows: a mixed batch of 64
// channels 138 -> 133 us.
template <int D, bool PAGED, bool WINDOWED>
__global__ __launch_bounds__(CK_THREADS, 1) void sp_chunk_kernel(const CkArgs a) {
  constexpr int WAVES = CK_WAVES, THREADS = CK_THREADS, TILE_ROWS = CK_ROWS;
  constexpr bool HALF = D == 64;
  constexpr int QT = 2;                    // 16-row tiles per wave
  constexpr int KS = D / 32, CT = D / 16;  // channel steps of S, channel tiles of O
  constexpr int SUB_BYTES = CK_SUB_BYTES(D);
  constexpr int CHUNKS = D / 8, ROWS = SP_WAVE / CHUNKS;        // of a row; rows of a load instruction
  constexpr int ITS = CK_SUB / (ROWS * WAVES);                  // instructions of a wave for a sub-tile
  extern __shared__ __attribute__((aligned(1024))) char lds[];  // rings of K and of V
  const int t = threadIdx.x, lane = t & 63, lq = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t lds_base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
  const int kvh = blockIdx.x % a.hkv, part = blockIdx.x / a.hkv;  // (workgroups of a kv head share an XCD where that works out)
  // Arguments of what is done once a row tile or a page group are read where they are used: scalar registers do not suffice to keep them, and
  // what the compiler sets aside for them passes through vector lanes in the loop.
  const auto kernel_args = (const __attribute__((address_space(4))) CkArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  auto args = [&] {
    auto p = kernel_args;
    asm volatile("" : "+s"(p));
    return p;
  };

  // ---- which row tiles, and which blocks of the first and the last ----
  // On a line: row tiles x .. x_end, the first from block tile_begin on, of the last the blocks in front of tile_end.
  int x = 0, x_end = 0, tile_begin = 0, tile_end = 0, turn = 0;
  int* const cu_s = reinterpret_cast<int*>(lds + CK_LDS_BYTES(D));
  const uint32_t lds_cu = lds_base + CK_LDS_BYTES(D), lds_len = lds_cu + 4u * (uint32_t)(a.batch + 1);
  if (a.parts != 0) {
    int* const len_s = cu_s + a.batch + 1;
    __shared__ int64_t wave_sums[WAVES];
    __shared__ int found[2][2];
    int back = 0;
    for (int i = t; i <= a.batch; i += THREADS) {
      const int start = ck_start(a, i);
      cu_s[i] = start;
      if (i < a.batch) len_s[i] = ck_len(a, i), back |= ck_start(a, i + 1) < start;
    }
    // Searches need the offsets in order, and must all find the same: notes of row tiles that only some of them find stay unwritten, and the
    // merging launch would read where they happen to point.  An offset that goes back counts as the largest in front of it.
    if (__syncthreads_or(back)) {
      if (t == 0)
        for (int i = 1; i <= a.batch; ++i) cu_s[i] = pg_max(cu_s[i], cu_s[i - 1]);
      __syncthreads();
    }
    // every thread some row tiles in a row: their units, then the line's prefix sums
    const int per = (a.slots + THREADS - 1) / THREADS, x0 = t * per, x1 = pg_min(x0 + per, a.slots);
    auto walk = [&](auto&& visit) {  // visit(x, units in the line, 0: no row tile has the number, blocks)
      if (x0 >= x1) return;
      int b = 0, hi = a.batch;
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (pg_first_slot(cu_s[mid], a.group, mid, TILE_ROWS) <= x0)
          b = mid;
        else
          hi = mid;
      }
      for (int i = x0; i < x1; ++i) {
        while (b + 1 < a.batch && pg_first_slot(cu_s[b + 1], a.group, b + 1, TILE_ROWS) <= i) ++b;
        const int q_len = pg_max(0, cu_s[b + 1] - cu_s[b]), rt = (int)(i - pg_first_slot(cu_s[b], a.group, b, TILE_ROWS));
        if (rt < 0 || rt >= pg_row_tiles(q_len, a.group, TILE_ROWS)) {
          visit(i, 0, 0);
          continue;
        }
        int p0, p1;
        pg_tile_positions(rt, q_len, len_s[b], a.by_group, TILE_ROWS, &p0, &p1);
        const int blocks = ck_blocks(ck_span<WINDOWED>(a, p0, p1, CK_SUB));
        visit(i, blocks + PG_OVERHEAD, blocks);
      }
    };
    int64_t mine = 0;
    int mine_blocks = 0;
    walk([&](int i, int units, int blocks) {
      mine += units;
      mine_blocks = blocks;
      if (units == 0 && part == 0 && a.by_slot != nullptr) a.by_slot[(int64_t)i * a.hkv + kvh].y = 0;  // (no row tile: nothing to merge)
    });
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
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) at += total;
      total += wave_sums[w];
    }
    at -= mine;
    const int64_t parts = pg_parts(total, a.parts, PG_MIN_SHARE);
    const int64_t cut[2] = {part < parts ? pg_cut(total, parts, part) : total, part < parts ? pg_cut(total, parts, part + 1) : total};
    auto cuts = [&](int i, int units, int blocks) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (cut[e] >= at && cut[e] < at + units) {
          const int tile = pg_snap(cut[e] - at, blocks, PG_OVERHEAD, pg_near(total, parts));
          found[e][0] = tile < blocks || tile == 0 ? i : i + 1;
          found[e][1] = tile < blocks ? tile : 0;
        }
      at += units;
    };
    if (per > 1)
      walk(cuts);
    else if (mine > 0)
      cuts(x0, (int)mine, mine_blocks);
    __syncthreads();
    x = __builtin_amdgcn_readfirstlane(found[0][0]);
    tile_begin = __builtin_amdgcn_readfirstlane(found[0][1]);
    x_end = __builtin_amdgcn_readfirstlane(found[1][0]);
    tile_end = __builtin_amdgcn_readfirstlane(found[1][1]);
  }
  int4 note = make_int4(CK_NONE, 0, 0, 0);

  // A row tile, or what of it falls to this workgroup: blocks i0 .. i1 - 1 of its walk.
  struct Piece {
    int slot, b, rt, start, q_len, len, i0, i1, blocks;
    PgSpan span;
  };
  // (LDS reads of its own: the compiler would wait for all that is in flight in front of them)
  auto from_lds = [&](uint32_t at) {
    int v;
    asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(v) : "v"(at));
    return __builtin_amdgcn_readfirstlane(v);
  };
  auto start_of = [&](int b) { return a.cu != nullptr ? from_lds(lds_cu + 4u * b) : b * a.n_queries; };
  int seq = a.parts == 0 || x >= a.slots ? 0 : __builtin_amdgcn_readfirstlane(ck_sequence<TILE_ROWS>(a, cu_s, x, lane));
  auto next_piece = [&](Piece& p) {  // false: there is none
    for (;;) {
      int begin = 0, end = -1;
      if (a.parts == 0) {
        const int wgs = args()->workgroups;
        if (turn * (int64_t)wgs >= (int64_t)a.tiles * a.batch) return false;
        int at_b, at_rt;
        if (!pg_deal(turn++, part, wgs, a.batch, a.tiles, a.together, &at_b, &at_rt)) continue;
        // (quotients come from vector registers)
        p.slot = 0;
        p.b = __builtin_amdgcn_readfirstlane(at_b);
        p.rt = __builtin_amdgcn_readfirstlane(at_rt);
        p.start = p.b * a.n_queries;
        p.q_len = a.n_queries;
        p.len = a.n_keys;
      } else {
        if (x >= a.slots || !(x < x_end || (x == x_end && tile_end > 0))) return false;
        begin = tile_begin;
        if (x == x_end) end = tile_end;
        tile_begin = 0;
        const int here = x++;
        while (seq + 1 < a.batch && pg_first_slot(start_of(seq + 1), a.group, seq + 1, TILE_ROWS) <= here) ++seq;
        p.slot = here;
        p.b = seq;
        p.start = start_of(seq);
        p.q_len = pg_max(0, start_of(seq + 1) - p.start);
        p.len = a.lens != nullptr ? from_lds(lds_len + 4u * seq) : a.n_keys;
        p.rt = (int)(here - pg_first_slot(p.start, a.group, seq, TILE_ROWS));
        if (p.rt < 0 || p.rt >= pg_row_tiles(p.q_len, a.group, TILE_ROWS)) continue;
      }
      int p0, p1;
      pg_tile_positions(p.rt, p.q_len, p.len, a.by_group, TILE_ROWS, &p0, &p1);
      p.span = ck_span<WINDOWED>(a, p0, p1, CK_SUB);
      p.blocks = ck_blocks(p.span);
      p.i0 = begin;
      p.i1 = end >= 0 ? pg_min(end, p.blocks) : p.blocks;
      return true;
    }
  };

  const uint32_t k_row = (uint32_t)a.sk_n * 2u, v_row = (uint32_t)a.sv_n * 2u;  // bytes
  // The lane's place in what its wave's instructions fetch: its row of the page where a page is smaller than a sub-tile (an instruction of all
  // waves is 32 rows, 64 of 64 channels: the place in the page is the same for all), of the sub-tile else.
  const int in_sub = wave * ROWS + lane / CHUNKS, in_page = 1 << a.shift < CK_SUB ? in_sub & ((1 << a.shift) - 1) : in_sub;
  const uint32_t k_lane = (uint32_t)in_page * k_row + 16u * ((lane % CHUNKS) ^ ck_swz_k<D>(in_sub));
  const uint32_t v_lane = (uint32_t)in_page * v_row + 16u * ((lane % CHUNKS) ^ ck_swz_v<D>(in_sub));
  // LDS byte offsets of the lane's operands inside a sub-tile: K row lq, chunk g; V row 4 g + lq / 4, 8-byte piece lq % 4 of the 32 bytes of
  // channel tile 0.  Other steps and tiles are one XOR away, rows 16 further have the same swizzle.
  const uint32_t koff = (uint32_t)(lq * (D * 2) + ((g ^ ck_swz_k<D>(lq)) << 4));
  const int vrow = 4 * g + (lq >> 2);
  const uint32_t voff = (uint32_t)(vrow * (D * 2) + ((((lq >> 1) & 1) ^ ck_swz_v<D>(vrow)) << 4) + 8 * (lq & 1));
  bf16x8 ones = __builtin_bit_cast(bf16x8, (at_u32x4){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  asm volatile("" : "+v"(ones));  // one register set throughout

  // row of the lane's tile qt in a piece: token and head
  auto row_of = [&](const Piece& c, int in_rows, int* token, int* head) {
    const int r = c.rt * TILE_ROWS + pg_min(in_rows, c.q_len * a.group - c.rt * TILE_ROWS - 1);
    *token = (int)pg_div((unsigned)r, a.by_group);
    *head = kvh * a.group + (r - *token * a.group);
  };
  bf16x8 qb[QT][4];
  auto load_q = [&](const Piece& c) {
    const auto r = args();
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      int token, head;
      row_of(c, wave * 32 + 16 * qt + lq, &token, &head);
      const sp_bf16* src = r->q + c.b * r->sq_b + (int64_t)((PAGED ? c.start : 0) + token) * r->sq_n + head * r->sq_h + 8 * g;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qb[qt][ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(src + 32 * ks));
    }
  };

  // ---- a sequence's pages: 64 of them at hand, a lane each ----
  // A lane knows where its page's rows of K and V start and how many bytes of them there are, up to the sequence's end (none: no page): that is
  // what a load's buffer descriptor is made of, three lane reads a load.  Formed from scalars where it is needed it took a fifth of the waves'
  // instructions (65001 keys in pages of 128 2036 -> 1885 us with one descriptor a sub-tile instead of two).
  // Without a table a page is 64 keys of the tensor.
  struct Window {
    int k_lo, k_hi, k_bytes, v_lo, v_hi, v_bytes, group;  // group: pages 64 group .. 64 group + 63
    uint64_t lost;                                        // lanes without a page
  };
  Window win = {0, 0, 0, 0, 0, 0, -2, 0ull};
  auto entries = [&](int b, int group) {
    const int i = group * SP_WAVE + lane;
    if constexpr (!PAGED) return i;
    const auto r = args();
    const int id = r->table[b * r->table_stride + pg_min(i, r->width - 1)];
    return i < r->width && (unsigned)id < (unsigned)r->num_pages ? id : -1;
  };
  auto turn_to = [&](int b, int len, int group, int id) {
    const int rows = id < 0 ? 0 : pg_max(0, pg_min(len - ((group * SP_WAVE + lane) << a.shift), 1 << a.shift));
    auto at = [&](const sp_bf16* x, int64_t stride_b, int64_t stride_page, int64_t stride_h) {
      return (uint64_t)(x + (PAGED ? 0 : b * stride_b) + kvh * stride_h) + (uint64_t)pg_max(id, 0) * (uint64_t)(stride_page * 2);
    };
    const auto r = args();
    const uint64_t k_at = at(r->k, r->sk_b, r->sk_p, r->sk_h), v_at = at(r->v, r->sv_b, r->sv_p, r->sv_h);
    win.k_lo = (int)(uint32_t)k_at, win.k_hi = (int)(uint32_t)(k_at >> 32);
    win.v_lo = (int)(uint32_t)v_at, win.v_hi = (int)(uint32_t)(v_at >> 32);
    win.k_bytes = rows > 0 ? (int)((uint32_t)(rows - 1) * k_row + 2u * D) : 0;
    win.v_bytes = rows > 0 ? (int)((uint32_t)(rows - 1) * v_row + 2u * D) : 0;
    win.group = group;
    if constexpr (PAGED) win.lost = __ballot(id < 0);
  };
  auto group_of = [&](int key) { return (key >> a.shift) >> 6; };  // (a sub-tile's pages lie in one group of 64)
  // the sub-tile at key `first` into slot `sub` % 4 of a ring; want false: zeros, without a read
  auto load = [&](int first, int sub, bool want, int lo, int hi, int bytes, uint32_t row_bytes, uint32_t lane_off, uint32_t to) {
    to += (uint32_t)((sub & 3) * SUB_BYTES + wave * 1024);
    auto rsrc_of = [&](int key) {
      const int i = (key >> a.shift) & 63;
      const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(lo, i) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32;
      return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, want ? __builtin_amdgcn_readlane(bytes, i) : 0, 0x00027000);
    };
    if (!PAGED || 1 << a.shift >= CK_SUB) {  // (uniform)
      const __amdgpu_buffer_rsrc_t rsrc = rsrc_of(first);
      const uint32_t off = lane_off + (PAGED ? (uint32_t)(first & ((1 << a.shift) - 1)) * row_bytes : 0u);
#pragma unroll
      for (int it = 0; it < ITS; ++it)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ck_lds_ptr)(uintptr_t)(to + it * WAVES * 1024), 16,
                                                 (int)(off + (uint32_t)(it * WAVES * ROWS) * row_bytes), 0, 0, 0);
    } else {
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const __amdgpu_buffer_rsrc_t rsrc = rsrc_of(first + (it * WAVES + wave) * ROWS);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ck_lds_ptr)(uintptr_t)(to + it * WAVES * 1024), 16, (int)lane_off, 0, 0, 0);
      }
    }
  };
  auto load_k = [&](int first, int sub, bool want) { load(first, sub, want, win.k_lo, win.k_hi, win.k_bytes, k_row, k_lane, lds_base); };
  auto load_v = [&](int first, int sub, bool want) {
    load(first, sub, want, win.v_lo, win.v_hi, win.v_bytes, v_row, v_lane, lds_base + CK_RING * SUB_BYTES);
  };
  // A block of a walk: its sub-tiles' first keys, and which of its 16-key groups have no page (bits).
  struct Block {
    int key[2];
    uint32_t lost;
  };
  auto lost_of = [&](int first) {  // of a sub-tile of the pages at hand
    uint32_t lost = 0;
    if (PAGED && win.lost != 0ull) {  // (uniform)
#pragma unroll
      for (int i16 = 0; i16 < 4; ++i16) lost |= (uint32_t)((win.lost >> (((first + 16 * i16) >> a.shift) & 63)) & 1ull) << i16;
    }
    return lost;
  };
  auto key_of = [&](const Piece& p, int i, int hf) { return (WINDOWED ? pg_span_unit(p.span, 2 * i + hf) : 2 * i + hf) * CK_SUB; };

  // Block n of the workgroup (over all its pieces) is sub-tiles 2 n and 2 n + 1; sub-tile s lives in slot s % 4 of either ring.  One wait and
  // barrier per block: while it is computed on (K of 2 n, 2 n + 1, V of 2 n - 1, 2 n: P . V trails by a sub-tile) K of 2 n + 2, 2 n + 3 and V of
  // 2 n + 1, 2 n + 2 are on their way, sent out in four parts between the block's steps: V of 2 n + 1, then the next block's sub-tiles one after
  // the other, each of which may lie in other pages than the one in front.  Behind a piece's last block that is the next piece's first one: its
  // tiles land, and its queries, under the end of the piece in front.
  Piece cur_p, next_p;
  bool have = next_piece(cur_p), primed = false;
  Block cur = {{0, 0}, 0u}, nxt = {{0, 0}, 0u};
  int n = 0, ids_first = 0, ids_next = 0;  // table entries of the pages behind those at hand, if there is a block at hand
  if (have) load_q(cur_p);
  if (have) ids_first = entries(cur_p.b, group_of(key_of(cur_p, cur_p.i0, 0)));
  while (have) {
    const Piece pc = cur_p;
    const bool have_next = next_piece(next_p);
    const int b = pc.b, rt = pc.rt, start = pc.start, q_len = pc.q_len, len = pc.len, n_blk = pc.i1 - pc.i0;
    const int rows = q_len * a.group - rt * TILE_ROWS;  // from here to the sequence's end
    const bool from_start = pc.i0 == 0, to_end = pc.i1 == pc.blocks;  // (uniform)
    const bool has_rows = wave * 32 < rows;  // (uniform in the wave)
    // positions of the wave's first and last row
    const int w0 = len - q_len + (int)pg_div((unsigned)(rt * TILE_ROWS + pg_min(wave * 32, rows - 1)), a.by_group);
    const int w1 = len - q_len + (int)pg_div((unsigned)(rt * TILE_ROWS + pg_min(wave * 32 + 31, rows - 1)), a.by_group);
    int pos[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      int token, head;
      row_of(pc, wave * 32 + 16 * qt + lq, &token, &head);
      pos[qt] = len - q_len + token;
    }
    const bool next_blocks = have_next && next_p.i1 > next_p.i0;  // the next piece has a first block to fetch
    const int ids_here = ids_first;
    if (n_blk > 0 && !primed) ids_next = entries(b, group_of(key_of(pc, pc.i0, 0)) + 1);
    if (next_blocks) ids_first = entries(next_p.b, group_of(key_of(next_p, next_p.i0, 0)));

    floatx4 o[9][2];  // [channel tile][row tile]; o[8]: the row sums (ones . P)
#pragma unroll
    for (int ct = 0; ct < 9; ++ct)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) o[ct][qt] = (floatx4){0, 0, 0, 0};
    float m[QT] = {CK_NO_MAX, CK_NO_MAX}, l_mark[QT] = {0.f, 0.f};
    uint32_t det[2] = {0u, 0u};

    // to the pages of a block's second sub-tile
    auto turn_on = [&](int of_b, int of_len, Block& c) {
      const int group = group_of(c.key[1]);
      if (WINDOWED && group != win.group) {  // (uniform)
        turn_to(of_b, of_len, group, group == win.group + 1 ? ids_next : entries(of_b, group));
        ids_next = entries(of_b, group + 1);
      }
      c.lost |= lost_of(c.key[1]) << 4;
    };
    if (n_blk > 0) {
      if (primed) {
        cur = nxt;
      } else {
        __syncthreads();  // the rings are free
        cur = {{key_of(pc, pc.i0, 0), key_of(pc, pc.i0, 1)}, 0u};
        turn_to(b, len, group_of(cur.key[0]), ids_here);
        cur.lost = lost_of(cur.key[0]);
        load_k(cur.key[0], 2 * n, true);
        load_v(cur.key[0], 2 * n, true);
        turn_on(b, len, cur);
        load_k(cur.key[1], 2 * n + 1, true);
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      }
      const int n_last = n + n_blk - 1;
      bool more = false;  // there is a block behind this one
      CkAddr<D> ad;
      auto top = [&](bool wait) {
        // everybody's loads have landed, everybody is past the block in front
        if (wait) asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        load_v(cur.key[1], 2 * n + 1, true);
        more = n < n_last || next_blocks;
        if (n < n_last) {
          const int i = pc.i1 - (n_last - n);
          nxt = {{key_of(pc, i, 0), key_of(pc, i, 1)}, 0u};
          const int group = group_of(nxt.key[0]);
          if (group != win.group) {  // (uniform)
            turn_to(b, len, group, group == win.group + 1 ? ids_next : entries(b, group));
            ids_next = entries(b, group + 1);
          }
          nxt.lost = lost_of(nxt.key[0]);
        } else if (next_blocks) {
          nxt = {{key_of(next_p, next_p.i0, 0), key_of(next_p, next_p.i0, 1)}, 0u};
          const int group = group_of(nxt.key[0]);
          turn_to(next_p.b, next_p.len, group, ids_first);
          ids_next = entries(next_p.b, group + 1);
          nxt.lost = lost_of(nxt.key[0]);
        }
        const uint32_t k_at = lds_base + (uint32_t)(((2 * n) & 3) * SUB_BYTES), v_at = lds_base + CK_RING * SUB_BYTES;
        ad.ka = k_at + koff;
        ad.va[0] = v_at + (uint32_t)(((2 * n + 3) & 3) * SUB_BYTES) + voff;
        ad.va[1] = v_at + (uint32_t)(((2 * n) & 3) * SUB_BYTES) + voff;
      };
      auto feed = [&](int part) {
        if (part == 0) load_k(nxt.key[0], 2 * n + 2, more);
        if (part == 1) load_v(nxt.key[0], 2 * n + 2, more);
        if (part == 2) {
          if (more) turn_on(n < n_last ? b : next_p.b, n < n_last ? len : next_p.len, nxt);
          load_k(nxt.key[1], 2 * n + 3, more);
        }
      };
      // what the wave's rows do not see of a block: nothing to take out in most of them
      auto partly = [&](const Block& c) {
        bool some = c.lost != 0;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int key1 = c.key[hf] + CK_SUB - 1;
          some |= key1 > w0 || (WINDOWED && c.key[hf] <= w1 - a.window && key1 >= a.sinks);
        }
        return some;
      };
      // A half-tile of a block that holds unseen keys: none of its keys may be seen, or all, or some; most need one comparison a key or less.
      struct Mask {
        bool some;                                // the block holds unseen keys
        int key0, w0, w1, p0, p1, window, sinks;  // the half-tile's first key, positions of the wave's first and last row and of the lane's rows
        uint32_t lost;                            // halves of it without a page (bits)
        __device__ __forceinline__ void operator()(floatx4 (&s)[2][2]) const {
          if (!some) return;
          const floatx4 unseen = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          const int key1 = key0 + 31;
          if (key0 > w1 || (WINDOWED && key1 <= w0 - window && key0 >= sinks) || (lost & 3u) == 3u) {
            s[0][0] = s[0][1] = s[1][0] = s[1][1] = unseen;
            return;
          }
          const int key = key0 + 4 * ((threadIdx.x >> 4) & 3);
          const int h[2] = {p0 - key, p1 - key};
          if (key1 > w0) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int qt = 0; qt < 2; ++qt)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[kt][qt][j] = 16 * kt + j <= h[qt] ? s[kt][qt][j] : -INFINITY;
          }
          if (WINDOWED && key0 <= w1 - window && key1 >= sinks) {
            const int front = sinks - key, lo[2] = {h[0] - window, h[1] - window};
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
              for (int qt = 0; qt < 2; ++qt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  s[kt][qt][j] = 16 * kt + j > lo[qt] || 16 * kt + j < front ? s[kt][qt][j] : -INFINITY;
          }
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
            if ((lost >> kt) & 1u) s[kt][0] = s[kt][1] = unseen;
        }
      };
      auto masked = [&](const Block& c, bool some, int quarter) {
        return Mask{some, c.key[quarter >> 1] + 32 * (quarter & 1), w0, w1, pos[0], pos[1], a.window, a.sinks, c.lost >> (2 * quarter)};
      };
      constexpr int MODE = (HALF ? 2 : 0) | (CK_SLACK << 4);
      if (!has_rows) {
        top(false);
        feed(0), feed(1), feed(2);
        for (++n; n <= n_last; ++n) {
          cur = nxt;
          top(true);
          feed(0), feed(1), feed(2);
        }
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (have_next) load_q(next_p);
      } else {
        floatx4 sa[2][2], sb[2][2];  // [key tile][row tile]
        bf16x8 pa[2], pb[2];         // [row tile]
        bf16x8 pre[2];
        Block old = cur;
        bool some = partly(cur), some_old = some;
        // ---- start: S of the first half-tile, nothing to overlap with yet ----
        top(false);
        feed(0);
        ck_qk_only<0, HALF>(ad, qb, sa);
        feed(1);
        at_step<true, false, 1, 0, 0, MODE, false, 2, true>(ad, qb, sb, sa, pb, pa, o, a.scale_log2, m, det, ones, masked(cur, some, 0), l_mark, pre);
        at_step<true, true, 2, 1, 0, MODE, true, 3, true>(ad, qb, sa, sb, pa, pb, o, a.scale_log2, m, det, ones, masked(cur, some, 1), l_mark, pre);
        feed(2);
        at_step<true, true, 3, 1, 1, MODE, true>(ad, qb, sb, sa, pb, pa, o, a.scale_log2, m, det, ones, masked(cur, some, 2), l_mark, pre);
        // ---- steady: four steps per block ----
        for (++n; n <= n_last; ++n) {
          old = cur, some_old = some;
          cur = nxt;
          some = partly(cur);
          top(true);
          if (wave >= WAVES / 2) __builtin_amdgcn_s_setprio(1);
          at_step<true, true, 0, 0, 0, MODE, false, 1, true>(ad, qb, sa, sb, pa, pb, o, a.scale_log2, m, det, ones, masked(old, some_old, 3), l_mark, pre);
          feed(0);
          at_step<true, true, 1, 0, 1, MODE, true, 2, true>(ad, qb, sb, sa, pb, pa, o, a.scale_log2, m, det, ones, masked(cur, some, 0), l_mark, pre);
          if (wave >= WAVES / 2) __builtin_amdgcn_s_setprio(0);
          feed(1);
          at_step<true, true, 2, 1, 0, MODE, true, 3, true>(ad, qb, sa, sb, pa, pb, o, a.scale_log2, m, det, ones, masked(cur, some, 1), l_mark, pre);
          feed(2);
          at_step<true, true, 3, 1, 1, MODE, true>(ad, qb, sb, sa, pb, pa, o, a.scale_log2, m, det, ones, masked(cur, some, 2), l_mark, pre);
        }
        // ---- drain: the last half-tile and its P . V (V of the last block's second sub-tile) ----
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (have_next) load_q(next_p);
        ad.va[0] = lds_base + CK_RING * SUB_BYTES + (uint32_t)(((2 * n + 3) & 3) * SUB_BYTES) + voff;
        at_step<false, true, 0, 0, 0, MODE>(ad, qb, sa, sb, pa, pb, o, a.scale_log2, m, det, ones, masked(cur, some, 3), l_mark, pre);
        at_commit<MODE>(sb, pb, det, o, a.scale_log2, m, l_mark);
        ck_pv_only<0, 1, HALF>(ad, pb, o, ones);
        at_settle_o(o);
      }
    } else if (have_next) {
      load_q(next_p);
    }
    primed = n_blk > 0 && next_blocks;
    const float l[QT] = {o[8][0][0], o[8][1][0]};

    // ---- what has come of it: the rows, or a partial ----
    const bool whole = from_start && to_end;  // (uniform)
    const int64_t slab = (int64_t)blockIdx.x * 2 + (from_start ? 1 : 0);
    const auto dst_args = args();
    float* const o_to = dst_args->o_part + slab * (TILE_ROWS * D);
    float2* const ml_to = dst_args->ml_part + slab * TILE_ROWS;
    sp_bf16* const out = dst_args->out;
    if (from_start && dst_args->by_slot != nullptr && t == 0)
      dst_args->by_slot[(int64_t)pc.slot * a.hkv + kvh] = make_int4(blockIdx.x, whole ? 0 : pg_min(rows, TILE_ROWS), 0, 0);
    if (!whole) {
      if (from_start)
        note.y = pg_min(rows, TILE_ROWS), note.z = rt * TILE_ROWS, note.w = start;
      else
        note.x = to_end ? CK_LAST : CK_MIDDLE;
    }
    bool spoilt[QT], far[QT];  // a NaN in the lane's part of the row; its logits are far from zero
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int in_rows = wave * 32 + 16 * qt + lq;
      const bool mine = in_rows < rows;
      int token, head;
      row_of(pc, in_rows, &token, &head);
      spoilt[qt] = false;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 4; ++j) spoilt[qt] |= o[ct][qt][j] != o[ct][qt][j];
      // (a row whose sum is a NaN saw a logit that is none, or an infinite one: it is a NaN in all its channels as it is)
      spoilt[qt] = spoilt[qt] && mine && l[qt] == l[qt];
      const float size = __builtin_fabsf(m[qt]);
      far[qt] = mine && l[qt] == l[qt] && size >= CK_FAR && size < INFINITY && m[qt] != CK_NO_MAX;
      if (whole) {
        const float inv_l = l[qt] > 0.f || l[qt] != l[qt] ? 1.0f / l[qt] : 0.f;
        // (lane groups 2i and 2i + 1 trade halves of two neighbouring channel tiles: 16 bytes a store, 64 contiguous ones a row)
        sp_bf16* dst = out + ((int64_t)(start + token) * (a.hkv * a.group) + head) * D + 16 * (g & 1) + 8 * (g >> 1);
#pragma unroll
        for (int ct = 0; ct < CT; ct += 2) {
          uint32_t w[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            w[u][0] = at_pack2(o[ct + u][qt][0] * inv_l, o[ct + u][qt][1] * inv_l);
            w[u][1] = at_pack2(o[ct + u][qt][2] * inv_l, o[ct + u][qt][3] * inv_l);
          }
          const auto lo = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
          const auto hi = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
          if (mine) *reinterpret_cast<uint4*>(dst + ct * 16) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
        }
      } else if (mine) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<floatx4*>(o_to + in_rows * D + 16 * ct + 4 * g) = o[ct][qt];
        if (g == 0) ml_to[in_rows] = make_float2(m[qt], l[qt]);
      }
    }
    // A masked key weighs 0, and 0 times an infinity or a NaN of its value has made a NaN of the sum.  Such rows are formed again key by key,
    // from what they see alone, some 7 us a row and sub-tile: 2048 tokens over 32768 keys with one bad new token 1.1 -> 121 ms.  Rows whose NaN came
    // from what they do see keep it: with one bad value in a long cache they are all rows of all later calls (256 tokens over 4096 keys 0.06 -> 2.7
    // ms, with all of them formed again).  Which it was shows in the sub-tiles that not all of the wave's rows see whole, a handful wherever the walk
    // is long.
    uint32_t again[QT];
    {
      uint32_t no_number[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const uint64_t lanes = __ballot(spoilt[qt]);
        no_number[qt] = (uint32_t)(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffffu;
        again[qt] = (uint32_t)__ballot(far[qt]) & 0xffffu;  // (the same in all of a row's lanes)
      }
      const int units = (no_number[0] | no_number[1]) != 0u ? 2 * pc.i1 : 0;
#pragma unroll 1
      for (int i0 = 2 * pc.i0; i0 < units; i0 += SP_WAVE) {
        const int first = key_of(pc, 0, i0 + lane), last = first + CK_SUB - 1;
        const bool whole_seen = last <= w0 && (!WINDOWED || first > w1 - a.window || last < a.sinks);
#pragma unroll 1
        for (uint64_t left = __ballot(i0 + lane < units && !whole_seen); left != 0ull; left &= left - 1ull) {
          const int key = key_of(pc, 0, i0 + __builtin_ctzll(left)) + lane, page = key >> a.shift;
          const auto c = args();
          int id = page;
          if constexpr (PAGED) {
            id = page < c->width ? c->table[b * c->table_stride + page] : -1;
            if ((unsigned)id >= (unsigned)c->num_pages) id = -1;
          }
          uint32_t bad = 0u;  // an exponent of ones: one more carries into the sign
          if (id >= 0 && key < len) {
            const sp_bf16* vrow = c->v + b * c->sv_b + kvh * c->sv_h + id * c->sv_p + (int64_t)(key & ((1 << a.shift) - 1)) * c->sv_n;
            for (int ch = 0; ch < D; ch += 8) {
              const uint4 x = *reinterpret_cast<const uint4*>(vrow + ch);
              for (const uint32_t w : {x.x, x.y, x.z, x.w}) bad |= ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
            }
          }
          if (__ballot(bad != 0u) == 0ull) continue;
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            for (uint32_t rows_left = no_number[qt] & ~again[qt]; rows_left != 0u; rows_left &= rows_left - 1u) {
              const int r = rt * TILE_ROWS + wave * 32 + 16 * qt + __builtin_ctz(rows_left);
              const int p = len - q_len + (int)pg_div((unsigned)r, a.by_group);
              if (__ballot(bad != 0u && !pg_sees(p, key, a.window, a.sinks)) != 0ull) again[qt] |= rows_left & (0u - rows_left);
            }
        }
      }
    }
#pragma unroll 1
    for (int qt = 0; qt < QT; ++qt) {
      uint32_t rows_left = again[qt];
      if (rows_left == 0u) continue;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above come first
      while (rows_left != 0u) {
        const int in_rows = wave * 32 + 16 * qt + __builtin_ctz(rows_left);
        rows_left &= rows_left - 1u;
        const int r = rt * TILE_ROWS + in_rows, token = (int)pg_div((unsigned)r, a.by_group), head = kvh * a.group + (r - token * a.group);
        const int p = len - q_len + token;
        const auto c = args();
        const sp_bf16* qrow = c->q + b * c->sq_b + (int64_t)((PAGED ? start : 0) + token) * c->sq_n + head * c->sq_h;
        constexpr int CL = D / SP_WAVE;  // channels of a lane
        float acc[CL] = {0.f}, sum = 0.f, top = CK_NO_MAX;
        for (int i = 2 * pc.i0; i < 2 * pc.i1; ++i) {
          const int key = key_of(pc, 0, i) + lane, page = key >> a.shift;
          int id = page;
          if constexpr (PAGED) {
            id = page < c->width ? c->table[b * c->table_stride + page] : -1;
            if ((unsigned)id >= (unsigned)c->num_pages) id = -1;
          }
          const bool seen = id >= 0 && key < len && pg_sees(p, key, a.window, a.sinks);
          const int64_t in = key & ((1 << a.shift) - 1);
          float logit = -INFINITY;
          if (seen) {
            const sp_bf16* krow = c->k + b * c->sk_b + kvh * c->sk_h + id * c->sk_p + in * c->sk_n;
            float dot = 0.f;
#pragma unroll 4
            for (int ch = 0; ch < D; ch += 8) {
              const at_u32x4 qx = *reinterpret_cast<const at_u32x4*>(qrow + ch), kx = *reinterpret_cast<const at_u32x4*>(krow + ch);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                dot = __builtin_fmaf(__uint_as_float(qx[i] << 16), __uint_as_float(kx[i] << 16), dot);
                dot = __builtin_fmaf(__uint_as_float(qx[i] & 0xffff0000u), __uint_as_float(kx[i] & 0xffff0000u), dot);
              }
            }
            logit = dot * a.scale_log2;
          }
          const float new_top = fmaxf(top, sp_wave_max(logit)), alpha = __builtin_amdgcn_exp2f(top - new_top);
          const float weight = seen ? __builtin_amdgcn_exp2f(logit - new_top) : 0.f;
          sum = sum * alpha + sp_wave_sum(weight);
          top = new_top;
#pragma unroll
          for (int c = 0; c < CL; ++c) acc[c] *= alpha;
          const uint64_t keys = __ballot(seen);
          const int64_t v_own = seen ? id * c->sv_p + in * c->sv_n : 0;
          const int64_t v_first = __shfl(v_own, keys != 0ull ? __builtin_ctzll(keys) : 0, SP_WAVE), v_at = seen ? v_own : v_first;  // (read, not taken)
          constexpr int AT_ONCE = 8;  // loads in flight
#pragma unroll 1
          for (int j0 = 0; j0 < SP_WAVE; j0 += AT_ONCE) {
            if (((keys >> j0) & ((1ull << AT_ONCE) - 1ull)) == 0ull) continue;
            float x[AT_ONCE][CL];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
              const sp_bf16* vrow_j = c->v + b * c->sv_b + kvh * c->sv_h + __shfl(v_at, j0 + u, SP_WAVE) + lane * CL;
#pragma unroll
              for (int ch = 0; ch < CL; ++ch) x[u][ch] = sp_bf16_to_f32(vrow_j[ch]);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
              const float w = __shfl(weight, j0 + u, SP_WAVE);
#pragma unroll
              for (int ch = 0; ch < CL; ++ch) acc[ch] = __builtin_fmaf(w, (keys >> (j0 + u)) & 1ull ? x[u][ch] : 0.f, acc[ch]);
            }
          }
          bool number = false;  // (a row that is none in any channel stays that)
#pragma unroll
          for (int c = 0; c < CL; ++c) number |= acc[c] == acc[c];
          if (sum > 0.f && __ballot(number) == 0ull) break;
        }
#pragma unroll
        for (int c = 0; c < CL; ++c) {
          if (whole)
            out[((int64_t)(start + token) * (a.hkv * a.group) + head) * D + lane * CL + c] = sp_f32_to_bf16(sum == 0.f ? 0.f : acc[c] / sum);
          else
            o_to[in_rows * D + lane * CL + c] = acc[c];
        }
        if (!whole && lane == 0) ml_to[in_rows] = make_float2(top, sum);
      }
    }
    cur_p = next_p;
    have = have_next;
  }
  if (a.parts != 0 && t == 0) args()->notes[blockIdx.x] = note;
}

// ---- host -------------------------------------------------------------------------------------------------
// Workgroups that are resident at once: one a CU.
#define CK_PLACES 256
static int ck_workgroups(int32_t hkv) { return hkv < CK_PLACES ? CK_PLACES / hkv : 1; }  // of a kv head
static size_t ck_workspace_bytes(int64_t tokens, int32_t batch, int32_t hq, int32_t hkv, int32_t d) {
  if (tokens <= 0 || batch <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || (d != 64 && d != 128)) return 0;
  return (size_t)ck_workgroups(hkv) * hkv * (2 * (size_t)CK_ROWS * ((size_t)d * sizeof(float) + sizeof(float2)) + 2 * sizeof(int4));
}

// Whether row tiles of a call whose sequences have as many rows and keys each stay whole: the longest workgroup against even parts, which take
// a sixteenth longer a block (their row tiles' keys lie further apart) and a merging launch, eight blocks' time.  us, whole / cut, 32 heads
// over 8: 2 tokens 8.3 / 11.9, prompts of 2048 59 / 67, 4096 127 / 155, in a window of 1024 77 / 88, 16384 1803 / 1899, 8 of 1024 88 / 97; cut
// because whole ones leave most of the card idle: 64 tokens over 16384, a row tile a head, 41.
static bool ck_whole(const CkArgs& a, int wgs) {
  if ((int64_t)a.tiles * a.batch >= 4 * wgs) return true;
  int64_t units[CK_PLACES] = {0}, most = 0, total = 0;
  for (int turn = 0; turn * wgs < a.tiles * a.batch; ++turn)
    for (int part = 0; part < wgs; ++part) {
      int b, rt, p0, p1;
      if (!pg_deal(turn, part, wgs, a.batch, a.tiles, a.together, &b, &rt)) continue;
      pg_tile_positions(rt, a.n_queries, a.n_keys, a.by_group, CK_ROWS, &p0, &p1);
      const int n = ck_blocks(pg_span(p0, p1, a.window, a.sinks, CK_SUB)) + PG_OVERHEAD;
      units[part] += n, total += n;
      if (units[part] > most) most = units[part];
    }
  return most <= total / wgs * 17 / 16 + 8;
}

// what a launch needs, checked before anything is launched
static int ck_check_launch(const char* who, const CkArgs& a, size_t need, const void* workspace, size_t workspace_bytes) {
  const int hq = a.hkv * a.group;
  SP_REQUIRE(pg_slots(a.tokens, a.group, a.batch, CK_ROWS) <= 0x7fffffffll && (int64_t)a.tokens * a.group < (1ll << 31) &&
                 (int64_t)a.batch * a.hkv <= 0x7fffffffll,
             SP_ERR_UNSUPPORTED, "%s: %d tokens of %d heads are too many", who, a.tokens, hq);
  SP_REQUIRE(pd_takes(a) || a.batch <= CK_MAX_SEQS, SP_ERR_UNSUPPORTED, "%s: batch %d (at most %d, single tokens %d)", who, a.batch, CK_MAX_SEQS,
             PG_MAX_SEQS);
  SP_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), SP_ERR_WORKSPACE,
             "%s: workspace missing, too small or misaligned", who);
  return SP_OK;
}

// max_keys: no sequence has more that exist.  Behind a table it may be longer, by the lengths that the device holds: its rows' windows lie that much
// further on, and a window as wide as the table leaves keys out.
static int ck_launch(const char* who, CkArgs& a, int64_t max_keys, int32_t d, void* workspace, hipStream_t s) {
  const bool windowed = a.window < (a.table != nullptr ? PG_NO_WINDOW : max_keys) && a.sinks < max_keys;
  if (!windowed) a.window = PG_NO_WINDOW;
  const bool uniform = a.cu == nullptr && a.lens == nullptr;  // as many queries and keys in every sequence
  const int wgs = ck_workgroups(a.hkv), grid = wgs * a.hkv;
  a.workgroups = wgs;
  a.by_group = pg_divisor((unsigned)a.group);
  a.slots = (int)pg_slots(a.tokens, a.group, a.batch, CK_ROWS);
  a.tiles = uniform ? (int)pg_row_tiles(a.n_queries, a.group, CK_ROWS) : 0;
  a.together = uniform ? pg_together(a.tiles, wgs, a.batch) : 0;
  a.parts = uniform && ck_whole(a, wgs) ? 0 : wgs;
  a.o_part = (float*)workspace;
  a.ml_part = (float2*)(a.o_part + (size_t)grid * 2 * (size_t)CK_ROWS * d);
  a.notes = (int4*)(a.ml_part + (size_t)grid * 2 * CK_ROWS);
  const size_t lds = CK_LDS_BYTES(d) + (a.parts != 0 ? (size_t)(2 * a.batch + 1) * sizeof(int) : 0);
  const bool by_slot = (int64_t)a.slots * a.hkv < grid;
  const int merges = by_slot ? a.slots * a.hkv : grid;  // workgroups of the merging launch, a band of rows
  a.by_slot = a.parts != 0 && by_slot ? a.notes + grid : nullptr;
  // Rows a merging workgroup takes: 16 spread few row tiles of many parts over more workgroups, 64 need fewer launches of them.  us, 16 / 64:
  // 64 tokens over 16384 keys (merges 16) 42.3 / 50.4, 2 over 8192 (16) 23.6 / 28.3; 512 over 8192 (72) 86 / 81, 2048 over 2048 (256) 74 / 60.
  const int band = merges <= 32 ? 16 : 64;
  auto go = [&](auto kernel, auto few, auto many) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(CK_THREADS), lds, s, a);
    if (a.parts != 0)
      hipLaunchKernelGGL(band == 16 ? few : many, dim3((unsigned)merges, CK_ROWS / band), dim3(CM_THREADS), 0, s, a, grid);
  };
  static bool attr_set[64] = {false};  // per device, once (idempotent)
  int dev = 0;
  SP_HIP(hipGetDevice(&dev));
  SP_REQUIRE(dev >= 0 && dev < 64, SP_ERR_UNSUPPORTED, "%s: device index %d", who, dev);
  if (!attr_set[dev]) {
    const void* kernels[8] = {(const void*)sp_chunk_kernel<64, false, false>,  (const void*)sp_chunk_kernel<64, true, false>,
                              (const void*)sp_chunk_kernel<128, false, false>, (const void*)sp_chunk_kernel<128, true, false>,
                              (const void*)sp_chunk_kernel<64, false, true>,   (const void*)sp_chunk_kernel<64, true, true>,
                              (const void*)sp_chunk_kernel<128, false, true>,  (const void*)sp_chunk_kernel<128, true, true>};
    for (const void* f : kernels)
      SP_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, CK_LDS_BYTES(128) + (2 * CK_MAX_SEQS + 1) * (int)sizeof(int)));
    attr_set[dev] = true;
  }
  auto pick = [&](auto width, auto in_windows) {
    constexpr int D = decltype(width)::value;
    constexpr bool WINDOWED = decltype(in_windows)::value;
    auto few = sp_chunk_merge_kernel<D, CK_ROWS, 16>, many = sp_chunk_merge_kernel<D, CK_ROWS, 64>;
    a.table != nullptr ? go(sp_chunk_kernel<D, true, WINDOWED>, few, many) : go(sp_chunk_kernel<D, false, WINDOWED>, few, many);
  };
  auto wide = [&](auto width) { windowed ? pick(width, std::true_type{}) : pick(width, std::false_type{}); };
  d == 64 ? wide(std::integral_constant<int, 64>{}) : wide(std::integral_constant<int, 128>{});
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
// offsets inside a page (`rows` of them) have 32 bits
static bool ck_rows_ok(int64_t stride_n, int64_t rows) {
  return stride_n >= 0 && stride_n < (1ll << 24) && stride_n * rows < (1ll << 30) && stride_n % 8 == 0;
}

extern "C" size_t sp_paged_attn_workspace_bytes(int64_t tokens, int32_t batch, int32_t hq, int32_t hkv, int32_t d, int32_t single_tokens) {
  const bool singles = single_tokens && hq > 0 && hkv > 0 && hq % hkv == 0 && hq / hkv <= PD_MAX_GROUP && (d == 64 || d == 128);
  return singles && tokens > 0 ? pd_workspace_bytes(hkv, d) : ck_workspace_bytes(tokens, batch, hq, hkv, d);
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
  const int64_t q_n = pg_used_stride(x->q_stride_n, x->tokens), q_h = pg_used_stride(x->q_stride_h, x->hq);
  const int64_t k_p = pg_used_stride(x->k_stride_page, x->num_pages), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  const int64_t v_p = pg_used_stride(x->v_stride_page, x->num_pages), v_h = pg_used_stride(x->v_stride_h, x->hkv);
  SP_REQUIRE(x->q && x->k_pages && x->v_pages && x->block_table && x->seq_lens && x->out, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->q | (uintptr_t)x->k_pages | (uintptr_t)x->v_pages | (uintptr_t)x->out) % 16 == 0 &&
                 (q_n | q_h | k_p | k_h | v_p | v_h) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  SP_REQUIRE(ck_rows_ok(x->k_stride_slot, x->page_size) && ck_rows_ok(x->v_stride_slot, x->page_size), SP_ERR_UNSUPPORTED,
             "%s: slot strides %lld / %lld unsupported", who, (long long)x->k_stride_slot, (long long)x->v_stride_slot);
  CkArgs a = {};
  a.q = (const sp_bf16*)x->q, a.k = (const sp_bf16*)x->k_pages, a.v = (const sp_bf16*)x->v_pages;
  a.table = x->block_table, a.lens = x->seq_lens, a.cu = x->cu_q, a.out = (sp_bf16*)x->out;
  a.table_stride = x->table_stride;
  a.sq_n = q_n, a.sq_h = q_h;
  a.sk_p = k_p, a.sk_n = x->k_stride_slot, a.sk_h = k_h;
  a.sv_p = v_p, a.sv_n = x->v_stride_slot, a.sv_h = v_h;
  a.batch = (int)x->batch, a.tokens = (int)x->tokens, a.width = (int)x->table_width, a.num_pages = (int)x->num_pages, a.shift = shift;
  a.n_queries = 1;
  a.hkv = (int)x->hkv, a.group = (int)(x->hq / x->hkv), a.window = ck_window(x->window), a.sinks = (int)(x->sinks < PG_MAX_KEYS ? x->sinks : PG_MAX_KEYS);
  a.scale_log2 = (float)x->softmax_scale * 1.4426950408889634f;
  rc = ck_check_launch(who, a, sp_paged_attn_workspace_bytes(x->tokens, (int)x->batch, (int)x->hq, (int)x->hkv, (int)x->d, a.cu == nullptr),
                       x->workspace, (size_t)x->workspace_bytes);
  if (rc) return rc;
  const int64_t room = x->table_width << shift;
  if (pd_takes(a)) return pd_launch(a, room, (int)x->d, x->workspace, (hipStream_t)x->stream);
  return ck_launch(who, a, room, (int)x->d, x->workspace, (hipStream_t)x->stream);
}

extern "C" size_t sp_window_attn_workspace_bytes(int32_t batch, int64_t n, int64_t n_keys, int32_t hq, int32_t hkv, int32_t d) {
  (void)n_keys;
  return batch <= 0 || n <= 0 ? 0 : n == 1 ? sp_paged_attn_workspace_bytes(batch, batch, hq, hkv, d, 1) : ck_workspace_bytes(batch * n, batch, hq, hkv, d);
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
  const int64_t q_b = pg_used_stride(x->q_stride_b, x->batch), q_n = pg_used_stride(x->q_stride_n, x->n), q_h = pg_used_stride(x->q_stride_h, x->hq);
  const int64_t k_b = pg_used_stride(x->k_stride_b, x->batch), k_h = pg_used_stride(x->k_stride_h, x->hkv);
  const int64_t v_b = pg_used_stride(x->v_stride_b, x->batch), v_h = pg_used_stride(x->v_stride_h, x->hkv);
  // (rows behind a sequence's last one are read as what lies behind its end, which a single key has to have too)
  const int64_t k_n = x->n_keys == 1 ? x->d : x->k_stride_n, v_n = x->n_keys == 1 ? x->d : x->v_stride_n;
  SP_REQUIRE(x->q && x->k && x->v && x->out, SP_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  SP_REQUIRE(((uintptr_t)x->q | (uintptr_t)x->k | (uintptr_t)x->v | (uintptr_t)x->out) % 16 == 0 &&
                 (q_b | q_n | q_h | k_b | k_h | v_b | v_h) % 8 == 0,
             SP_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned, strides multiple of 8", who);
  SP_REQUIRE(ck_rows_ok(k_n, CK_SUB) && ck_rows_ok(v_n, CK_SUB), SP_ERR_UNSUPPORTED, "%s: token strides %lld / %lld unsupported", who,
             (long long)x->k_stride_n, (long long)x->v_stride_n);
  CkArgs a = {};
  a.q = (const sp_bf16*)x->q, a.k = (const sp_bf16*)x->k, a.v = (const sp_bf16*)x->v, a.out = (sp_bf16*)x->out;
  a.shift = 6;  // a sub-tile is a page
  a.sq_b = q_b, a.sq_n = q_n, a.sq_h = q_h;
  a.sk_b = k_b, a.sk_n = k_n, a.sk_h = k_h, a.sk_p = k_n << a.shift;
  a.sv_b = v_b, a.sv_n = v_n, a.sv_h = v_h, a.sv_p = v_n << a.shift;
  a.batch = (int)x->batch, a.tokens = (int)(x->batch * x->n), a.n_keys = (int)x->n_keys, a.n_queries = (int)x->n;
  a.hkv = (int)x->hkv, a.group = (int)(x->hq / x->hkv), a.window = ck_window(x->window), a.sinks = (int)(x->sinks < PG_MAX_KEYS ? x->sinks : PG_MAX_KEYS);
  a.scale_log2 = (float)x->softmax_scale * 1.4426950408889634f;
  rc = ck_check_launch(who, a, sp_window_attn_workspace_bytes((int)x->batch, x->n, x->n_keys, (int)x->hq, (int)x->hkv, (int)x->d),
                       x->workspace, (size_t)x->workspace_bytes);
  if (rc) return rc;
  if (pd_takes(a)) return pd_launch(a, x->n_keys, (int)x->d, x->workspace, (hipStream_t)x->stream);
  return ck_launch(who, a, x->n_keys, (int)x->d, x->workspace, (hipStream_t)x->stream);
}
