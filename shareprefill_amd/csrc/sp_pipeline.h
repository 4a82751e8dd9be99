// The software pipeline of one wave: S^T = K . Q^T of one half-tile of 32 keys, O^T += V^T . P^T of another and the softmax of the one in
// between in one instruction stream.  sp_attn.hip runs it on V^T as its repack leaves it, sp_chunk.hip on V as it is; where an operand lies in
// LDS is the caller's (Addr).
#pragma once
#include "sp_common.h"

#include <type_traits>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

#define AT_WAIT_VMCNT0() __builtin_amdgcn_s_waitcnt(0x0F70)  // vmcnt(0) only: the direct-to-LDS loads have landed
#define AT_PIN() __builtin_amdgcn_sched_barrier(0)            // nothing is scheduled across this point

// ---- the software pipeline of one wave ------------------------------------------------------------------------
// A wave owns 32 queries as two 16-query tiles (qt = 0, 1) and works with v_mfma_f32_16x16x32_bf16: A 16x32, B 32x16,
// C/D 16x16 (lane l: column l%16, rows 4*(l/16) .. +3).  Against the 32x32x16 form the same flops read and rewrite
// only half as many accumulator registers (K = 32 per instruction), which is what the power-limited chip rewards.
//   S^T[16 keys x 16 q] = K frag[16 keys x 32 ch] . Q^T frag[32 ch x 16 q]      4 channel steps per tile
//   O^T[16 ch x 16 q]  += V^T frag[16 ch x 32 key slots] . P^T[32 key slots x 16 q]
// Every LDS operand (a K or V^T fragment, 1 KiB) feeds the two query tiles.  A lane holds, per query tile, the
// logits of keys 4g .. 4g+3 of both 16-key tiles of a half-tile (g = l/16): exactly the eight key slots 8g .. 8g+7
// of the P^T operand once the V^T repack orders the keys that way (at_perm32), so P is the S accumulator converted
// to bf16 in place.
// Keys are consumed in half-tiles of 32.  For half-tile j the wave issues, in ONE instruction stream,
//     S(j+1) = K(j+1) . Q^T        16 MFMAs  (matrix core)
//     O     += V^T(j-1) . P(j-1)   16 MFMAs  (matrix core), + 2 for the row sums  ones . P(j-1)
//     P(j)   = exp2(S(j)*scale - m), bf16 packing               ~45 vector instructions
// interleaved one LDS operand read : two MFMAs : two or three vector instructions.  A wave issues in order but
// an MFMA executes for 16 cycles after it is issued, so the vector work of half-tile j runs in the shadow of the
// matrix work of its neighbours; scheduling barriers pin that order.  The running max m is lazy (see at_commit):
// it moves only when some probability came out at 2 or more, and then O and the row sums are rescaled and that
// half-tile's probabilities are formed again before they are used.
typedef uint32_t at_u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t at_pack2(float a, float b) {
  floatx2 f;
  f[0] = a;
  f[1] = b;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

// compile-time loop: f(std::integral_constant<int, K>) for K = 0 .. N-1
template <int K, int N, typename F>
__device__ __forceinline__ void at_static_for(F&& f) {
  if constexpr (K < N) {
    f(std::integral_constant<int, K>{});
    at_static_for<K + 1, N>(f);
  }
}

// LDS operand fetch the compiler does not track: it returns at once and the register is valid only after an
// explicit AT_WAIT_LGKM(n) (n = younger fetches allowed to be still in flight; LDS reads return in order).
// Reason: while direct-to-LDS tile loads are in flight the compiler waits for ALL outstanding LDS reads before
// every use of any of them, which exposes the full LDS latency in front of each MFMA.
template <int IMM>
__device__ __forceinline__ bf16x8 at_lds128_async(uint32_t addr) {
  at_u32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(IMM));
  return __builtin_bit_cast(bf16x8, r);
}
#define AT_WAIT_LGKM(n) __builtin_amdgcn_s_waitcnt(0xC07F | ((n) << 8))

__device__ __forceinline__ uint32_t at_lds_addr(const char* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// The MFMAs of the pipeline are written as inline assembly that accumulates IN PLACE.  Through the builtin the
// register allocator is free to give an MFMA's result other registers than its accumulator operand, and it does so
// for this kernel: the accumulators then change registers from step to step and every step ends in ~80 register
// copies where the rare rescale branch joins the main path.  The compiler does not know the result latency of
// these instructions: a vector instruction that reads an MFMA result sits at least three operand slots behind it
// by construction, and where that is not so (at_settle_*) explicit wait states are inserted.
__device__ __forceinline__ void at_mfma_first(floatx4& d, bf16x8 a, bf16x8 b) {  // d = a . b
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
}
__device__ __forceinline__ void at_mfma_acc(floatx4& d, bf16x8 a, bf16x8 b) {  // d += a . b
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
}
// ... and the same with the wait states that let vector instructions read the results of this and every earlier MFMA
// INSIDE the statement.  A separate settling statement tied to the result registers is not enough where the reader
// follows closely: to satisfy the tie the register allocator may first copy a result into other registers -- with a
// vector move that reads the result while the MFMA is still in flight -- and put the wait states behind that copy
// (seen in the generated code of the pivot instantiation: a copy of the row sums five wait states behind their MFMA).
__device__ __forceinline__ void at_mfma_acc_settled(floatx4& d, bf16x8 a, bf16x8 b) {  // d += a . b, then 16 wait states
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0\n\ts_nop 15" : "+v"(d) : "v"(a), "v"(b));
}
__device__ __forceinline__ void at_settle_o(floatx4 (&o)[9][2]) {
  asm volatile("s_nop 15"
               : "+v"(o[0][0]), "+v"(o[0][1]), "+v"(o[1][0]), "+v"(o[1][1]), "+v"(o[2][0]), "+v"(o[2][1]),
                 "+v"(o[3][0]), "+v"(o[3][1]), "+v"(o[4][0]), "+v"(o[4][1]), "+v"(o[5][0]), "+v"(o[5][1]),
                 "+v"(o[6][0]), "+v"(o[6][1]), "+v"(o[7][0]), "+v"(o[7][1]), "+v"(o[8][0]), "+v"(o[8][1]));
}

// max(a, b, c) / max(a, b) as single instructions: through fmaxf the compiler first quiets every operand it cannot
// prove to be no signalling NaN (v_max x, x), which the MFMA results behind inline assembly all are to it
__device__ __forceinline__ float at_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float at_max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// the lane's 16 logits of a half-tile in softmax order: query tile idx / 8, then key slots 8g .. 8g+7 of the lane
// (key tile (idx / 4) % 2, row idx % 4); s is indexed [key tile][query tile]
#define AT_SVAL(s, idx) (s)[((idx) >> 2) & 1][(idx) >> 3][(idx) & 3]

// KQ: which 32-key quarter (0..3) of the block's two K buffers S_out is computed from; VB / KT: which V^T buffer
// (0: sub-tile 2b-1, 1: sub-tile 2b) and which half of it P_prev belongs to.
// Slot order: the 8 operand slots of S_out first (channel step outermost, so that the four accumulators take turns),
// then the 8 of O (one channel tile each) and the two row-sum MFMAs; det receives the OR of P_out's packed words.
// The first two operands of a stage that starts with the S product of 32-key quarter KQ, fetched ahead of the stage
// (at the end of the one before it, or right behind the block's barrier): the stage then does not open with an LDS
// round trip in which, the other wave of the SIMD being at the same point, nobody issues anything.
template <int KQ, class Addr>
__device__ __forceinline__ void at_prefetch_qk(const Addr& ad, bf16x8 (&pre)[2]) {
  pre[0] = ad.template k<KQ, 0, 0>();
  pre[1] = ad.template k<KQ, 0, 1>();
}

// PRE: operands 0 and 1 of the stage are already in flight in `pre` (at_prefetch_qk<KQ>, and nothing else has been
// read from LDS since).  NEXT >= 0: the stage ends by fetching the first two operands of the next one, quarter NEXT.
// HALF: q, k and v are zero beyond channel 64 (a head_dim of at most 64 padded to the tiles' 128): the S product takes the
// first two of its four channel steps and O the first four of its eight channel tiles -- half the operand slots.
// SETTLE: the stage's last MFMA carries the wait states after which vector instructions may read every MFMA result
// (a run's first stage, whose S the next stage's softmax reads at once; a pivot head's stage in front of the block sums).
// Addr: where the operands of a block lie in LDS.  k<KQ, KS, T>() fetches channel step KS of key tile T of quarter KQ, v<VB, KT, I>() channel
// tile I of half KT of buffer VB, both unseen by the compiler; V_READS: LDS reads of the latter.
// EARLY: they are asked for two slots in front of the stage's end, and have landed there: no branch finds them on their way.
template <bool DO_QK, bool DO_PV, int KQ, int VB, int KT, bool PRE, int NEXT, bool HALF, bool SETTLE, bool EARLY, class Addr>
__device__ __forceinline__ void at_fused(const Addr& ad, const bf16x8 (&qb)[2][4], floatx4 (&s_out)[2][2],
                                         const floatx4 (&s_in)[2][2], const bf16x8 (&p_prev)[2], bf16x8 (&p_out)[2],
                                         floatx4 (&o)[9][2], float sc, const float (&neg_m)[2], uint32_t (&det)[2],
                                         const bf16x8& ones, bf16x8 (&pre)[2]) {
  static_assert(!PRE || DO_QK, "only stages that start with the S product take prefetched operands");
  constexpr int QS = DO_QK ? (HALF ? 4 : 8) : 0;  // operand slots of the S product: (channel step, key tile) pairs
  constexpr int PS = DO_PV ? (HALF ? 4 : 8) : 0;  // operand slots of the P.V product: channel tiles
  constexpr int NP = QS + PS;                     // each slot holds one MFMA per query tile
  static_assert(NP == 4 || NP == 8 || NP == 16, "a fused stage has 4, 8 or 16 operand slots");
  constexpr int EPS = 16 / NP;  // softmax elements handled per operand slot
  constexpr int AHEAD = 2;      // LDS operands are fetched this many slots before their MFMAs
  bf16x8 opnd[NP];
  float x[16], e[16];
  uint32_t pk[8];
  auto fetch = [&](auto kc) {
    constexpr int k = decltype(kc)::value;
    constexpr bool qk = k < QS;
    constexpr int i = qk ? k : k - QS;
    if constexpr (qk)  // slot i: channel step i / 2, key tile i % 2
      opnd[k] = ad.template k<KQ, (i >> 1), (i & 1)>();
    else  // slot i: channel tile i
      opnd[k] = ad.template v<VB, KT, i>();
  };
  static_assert(AHEAD == 2, "the prefetched pair is the stage's look-ahead");
  if constexpr (PRE) {
    opnd[0] = pre[0];
    opnd[1] = pre[1];
  } else {
    at_static_for<0, AHEAD>(fetch);
  }
  AT_PIN();
  at_static_for<0, NP>([&](auto kc) {
    constexpr int k = decltype(kc)::value;
    constexpr bool qk = k < QS;
    constexpr int i = qk ? k : k - QS;
    constexpr bool ahead = EARLY && NEXT >= 0;  // the next stage's operands go out in slot NP - 2
    constexpr int in_flight_after = k + 1 == NP ? (ahead ? 2 : 0) : k + 1 < QS ? 1 : Addr::V_READS;  // reads of operand k + 1, those
    AT_WAIT_LGKM(in_flight_after);  // operand k has landed
    AT_PIN();
    auto mfma = [&](auto qc, auto lastc) {
      constexpr int qt = decltype(qc)::value;
      constexpr bool settle = decltype(lastc)::value;  // the stage's last MFMA, and results are read right behind it
      if constexpr (qk) {
        if constexpr ((i >> 1) == 0)
          at_mfma_first(s_out[i & 1][qt], opnd[k], qb[qt][0]);
        else if constexpr (settle)
          at_mfma_acc_settled(s_out[i & 1][qt], opnd[k], qb[qt][i >> 1]);
        else
          at_mfma_acc(s_out[i & 1][qt], opnd[k], qb[qt][i >> 1]);
      } else {
        at_mfma_acc(o[i][qt], opnd[k], p_prev[qt]);
      }
    };
    // the two query tiles take turns at going first: across a slot boundary the B operand (Q or P of one query tile)
    // stays the same for two MFMAs in a row, as the A operand does inside a slot (+0.5 % under the power cap)
    mfma(std::integral_constant<int, (k & 1)>{}, std::false_type{});
    if constexpr (k + AHEAD < NP) fetch(std::integral_constant<int, k + AHEAD>{});
    if constexpr (ahead && k + AHEAD == NP) at_prefetch_qk<NEXT>(ad, pre);
#pragma unroll
    for (int u = 0; u < EPS; ++u) {
      const int idx = k * EPS + u;
      // The softmax arithmetic depends only on values known before the stage starts, and the optimiser would
      // otherwise move all of it in front of the stage (out of the MFMAs' shadow): the empty asm ties each
      // element to its slot.
      // (the tie goes through a scalar copy of the scale: S(j) itself must stay where it is, the next step may
      // need it again)
      float sc_here = sc;
      asm volatile("" : "+s"(sc_here));
      x[idx] = __builtin_fmaf(AT_SVAL(s_in, idx), sc_here, neg_m[idx >> 3]);
      if (idx >= 1) e[idx - 1] = __builtin_amdgcn_exp2f(x[idx - 1]);
      if (idx >= 3 && ((idx - 3) & 1) == 0) {
        const int m = (idx - 3) >> 1;
        pk[m] = at_pack2(e[idx - 3], e[idx - 2]);
        // OR of the packed probabilities: any exponent >= 128 (P >= 2, inf, NaN) shows in bit 14 or 30
        // (three words at a time: one three-input instruction)
        if ((m & 3) == 2) det[m >> 2] = pk[m - 2] | pk[m - 1] | pk[m];
        if ((m & 3) == 3) det[m >> 2] |= pk[m];
      }
      // ... and the results to the slot they were produced in (instruction selection lets pure arithmetic float)
      asm volatile("" : "+v"(x[idx]));
      if (idx >= 1) asm volatile("" : "+v"(e[idx - 1]));
      if (idx >= 3 && ((idx - 3) & 1) == 0) {
        if ((((idx - 3) >> 1) & 3) >= 2)
          asm volatile("" : "+v"(pk[(idx - 3) >> 1]), "+v"(det[(idx - 3) >> 3]));
        else
          asm volatile("" : "+v"(pk[(idx - 3) >> 1]));
      }
    }
    AT_PIN();
    mfma(std::integral_constant<int, 1 - (k & 1)>{}, std::integral_constant<bool, SETTLE && !DO_PV && k == NP - 1>{});
    if constexpr (DO_PV && k == NP - 1) {  // row sums of P(j-1) as rounded for the P.V product: ones . P
      at_mfma_acc(o[8][0], ones, p_prev[0]);
      if constexpr (SETTLE)
        at_mfma_acc_settled(o[8][1], ones, p_prev[1]);
      else
        at_mfma_acc(o[8][1], ones, p_prev[1]);
    }
    AT_PIN();
  });
  if constexpr (NEXT >= 0 && EARLY) {
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(pre[0]), "+v"(pre[1]));
    AT_PIN();
  } else if constexpr (NEXT >= 0) {
    at_prefetch_qk<NEXT>(ad, pre);
    AT_PIN();
  }
  e[15] = __builtin_amdgcn_exp2f(x[15]);
  pk[7] = at_pack2(e[14], e[15]);
  det[1] |= pk[7];
  static_assert(!(DO_QK && !DO_PV) || SETTLE, "a run's first stage: the next stage's softmax reads S_out at once");
  at_u32x4 w0, w1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w0[j] = pk[j];
    w1[j] = pk[4 + j];
  }
  p_out[0] = __builtin_bit_cast(bf16x8, w0);
  p_out[1] = __builtin_bit_cast(bf16x8, w1);
}

// max over the lane's 8 keys of each query tile
__device__ __forceinline__ void at_lanemax(const floatx4 (&s)[2][2], float (&mx)[2]) {
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    float m = at_max3(s[0][qt][0], s[0][qt][1], s[0][qt][2]);
    m = at_max3(m, s[0][qt][3], s[1][qt][0]);
    m = at_max3(m, s[1][qt][1], s[1][qt][2]);
    mx[qt] = at_max2(m, s[1][qt][3]);
  }
}

// ... and over the three partner lanes (lane ^ 16, ^ 32, ^ 48) that hold the other 24 keys of the query
__device__ __forceinline__ float at_groupmax(float mx) {
  uint32_t u = __builtin_bit_cast(uint32_t, mx);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);  // (own, lane ^ 16) in some order
  const float m1 = at_max2(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  u = __builtin_bit_cast(uint32_t, m1);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // (own, lane ^ 32) in some order
  return at_max2(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// ---- the running max of a query is lazy, its row sum comes off the matrix core ----
// Probabilities are formed against the max as it stood, m_run, which is only ever a lower bound of the true running
// max: they can exceed 1, which costs nothing as long as they stay far from the range limit.  The row sums are taken
// from the probabilities as rounded to bf16 for P.V -- two more MFMAs per step against an all-ones operand,
// accumulated in o[8] -- so numerator and denominator of the softmax see the same values and the result does not
// depend on the largest probability being exactly 1.  No maximum per half-tile: the packed probabilities are OR-ed
// (three instructions per step) and one test of the top exponent bit per step says whether some P(j-1) >= 2, is inf
// or NaN (the first keys of a row, m_run = AT_NO_MAX; a logit more than one octave above the max).  Only then is the max taken from S(j-1)
// -- still intact in the registers the next stage overwrites -- O and the sums are rescaled and P(j-1) is formed again;
// P(j-1) enters O only after this test.
// The max is the largest logit itself, so the probabilities that weigh most are at or near 1, where bf16 loses least of them.
// Set some octaves above it, rescales become rare (32768 tokens 2.93 -> 2.85 ms a layer, 131072 55.84 -> 55.45), but whatever
// logit came first then fixes the fraction all later probabilities are rounded at, and the exponent's argument is coarser: at
// 24 octaves the output was 5 to 7 % further from the attention in 64 bits (16384 tokens 1.96e-3 against 1.84e-3) and the
// pivots' maps nearly twice as far (2.3e-5 against 1.2e-5), so it stays at 0.
#define AT_NO_MAX (-1.0e30f)          // "no key seen yet": finite, so exp2(S * scale - m) is +inf or 0, never NaN
#define AT_P_TOO_LARGE 0x40004000u    // bf16 pair: exponent >= 128 in either half

// s_prev = S(j-1) (causal predicate applied), p = P(j-1), det = OR of its packed words.  On return p is safe to use.
// PIVOT: l_mark (the row sums at the start of the current key block, see the block sums of pivot heads in the
// kernel) follows every rescale.
// MODE: bit 0 = PIVOT, bit 1 = HALF (see at_fused), bit 2 = FINE (sp_attn.hip), bits 4 .. 6 = SLACK: octaves that a moved max is set above the
// largest logit
template <int MODE>
__device__ __forceinline__ void at_commit(const floatx4 (&s_prev)[2][2], bf16x8 (&p)[2], uint32_t (&det)[2],
                                          floatx4 (&o)[9][2], float scale_log2, float (&m_run)[2],
                                          float (&l_mark)[2]) {
  constexpr bool PIVOT = (MODE & 1) != 0, HALF = (MODE & 2) != 0;
  constexpr int SLACK = (MODE >> 4) & 7;
  if (__builtin_amdgcn_ballot_w64(((det[0] | det[1]) & AT_P_TOO_LARGE) != 0u) != 0ull) {
    float mx[2];  // (S(j-1) is a whole stage old: no wait states needed before reading it)
    at_lanemax(s_prev, mx);
    float m_new[2] = {at_groupmax(mx[0] * scale_log2), at_groupmax(mx[1] * scale_log2)};
    // (Past 2^20 a few units in the last place more: the probabilities' exponent has the exact product, and a max rounded down would make them
    // infinite.  They may come out as zero instead, where the caller forms such rows another way.)
    if constexpr (SLACK > 0) {
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        m_new[qt] += (float)SLACK;
        m_new[qt] = __builtin_fmaf(__builtin_amdgcn_fmed3f(__builtin_fabsf(m_new[qt]) - 0x1p20f, 0.f, 0x1.fffffep127f), 0x1p-22f, m_new[qt]);
      }
    }
    m_new[0] = at_max2(m_run[0], m_new[0]), m_new[1] = at_max2(m_run[1], m_new[1]);
    at_settle_o(o);
    // m_run = AT_NO_MAX on a row's first keys: alpha = 0 (O and the sums are still zero then)
    const float alpha[2] = {__builtin_amdgcn_exp2f(m_run[0] - m_new[0]), __builtin_amdgcn_exp2f(m_run[1] - m_new[1])};
    uint32_t pk[8];
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      if constexpr (PIVOT) l_mark[qt] *= alpha[qt];
#pragma unroll
      for (int dt = 0; dt < 9; ++dt) {
        if (HALF && dt >= 4 && dt < 8) continue;  // channel tiles nobody accumulates into
#pragma unroll
        for (int j = 0; j < 4; ++j) o[dt][qt][j] *= alpha[qt];
      }
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(AT_SVAL(s_prev, 8 * qt + j), scale_log2, -m_new[qt]));
#pragma unroll
      for (int j = 0; j < 4; ++j) pk[4 * qt + j] = at_pack2(e[2 * j], e[2 * j + 1]);
      m_run[qt] = m_new[qt];
    }
    at_settle_o(o);
    p[0] = __builtin_bit_cast(bf16x8, (at_u32x4){pk[0], pk[1], pk[2], pk[3]});
    p[1] = __builtin_bit_cast(bf16x8, (at_u32x4){pk[4], pk[5], pk[6], pk[7]});
    asm volatile("s_nop 4" : "+v"(p[0]), "+v"(p[1]));  // vector writes of P are complete before an MFMA reads them
  }
  det[0] = 0u;
  det[1] = 0u;
}

// One pipeline step.  s_in = S(j) (complete), p_prev = P(j-1) not yet applied to O (HAVE_PREV), det the OR of its
// packed words; s_out still holds S(j-1) on entry and S(j+1) on return, p_out = P(j) with its OR in det.
// The fused stage exists once per step: O never lives in two register sets that would have to be merged.
// mask(s): takes out what the half-tile's queries do not see of its keys.
template <bool DO_QK, bool HAVE_PREV, int KQ, int VB, int KT, int MODE, bool PRE = false, int NEXT = -1, bool EARLY = false, class Addr, class Mask>
__device__ __forceinline__ void at_step(const Addr& ad, const bf16x8 (&qb)[2][4], floatx4 (&s_out)[2][2],
                                        floatx4 (&s_in)[2][2], bf16x8 (&p_prev)[2], bf16x8 (&p_out)[2],
                                        floatx4 (&o)[9][2], float scale_log2, float (&m_run)[2], uint32_t (&det)[2],
                                        const bf16x8& ones, Mask&& mask, float (&l_mark)[2], bf16x8 (&pre)[2]) {
  if (HAVE_PREV) at_commit<MODE>(s_out, p_prev, det, o, scale_log2, m_run, l_mark);
  mask(s_in);
  const float neg_m[2] = {-m_run[0], -m_run[1]};
  // wait states inside the stage's last MFMA: a run's first stage (S read at once), and for pivot heads the stage
  // behind which the block sums are taken (emit in the kernel: the second stage of a block in the steady state)
  constexpr bool SETTLE = (DO_QK && !HAVE_PREV) || ((MODE & 1) != 0 && DO_QK && HAVE_PREV && KQ == 1);
  at_fused<DO_QK, HAVE_PREV, KQ, VB, KT, PRE, NEXT, (MODE & 2) != 0, SETTLE, EARLY>(ad, qb, s_out, s_in, p_prev, p_out, o,
                                                                              scale_log2, neg_m, det, ones, pre);
}
