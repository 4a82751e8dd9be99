// What the decode kernels with a ring of operands per wave share (sp_decode.hip, sp_paged_decode.hip): a step's layout in LDS, the operand
// reads and the lane exchanges.
#pragma once
#include "sp_common.h"

typedef uint32_t dc_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 dc_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 dc_bf16x4 __attribute__((ext_vector_type(4)));
typedef float dc_floatx16 __attribute__((ext_vector_type(16)));
typedef float dc_floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 dc_bf16x2 __attribute__((ext_vector_type(2)));
typedef float dc_floatx4 __attribute__((ext_vector_type(4), aligned(8)));  // (partials: 8-byte aligned workspace)

__device__ static __forceinline__ uint32_t dc_pack2(float a, float b) {
  dc_floatx2 f;
  f[0] = a;
  f[1] = b;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, dc_bf16x2));
}

#define DS_GMAX 16
#define DS_KEYS 32  // keys of a wave's step
typedef float ds_floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t ds_u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* ds_lds_ptr;

// CT_: channel tiles of 16 a slice has.  As many waves and steps of the ring as fit the LDS that the workgroup may have.
template <int D_, int CT_, int WAVES_, int KIB>
struct DsShape {
  static constexpr int D = D_, CT = CT_, WAVES = WAVES_;
  static constexpr int K_BYTES = DS_KEYS * D * 2, V_BYTES = DS_KEYS * CT * 32, STEP_BYTES = K_BYTES + V_BYTES;
  static constexpr int NB = KIB * 1024 / (WAVES * STEP_BYTES) < 4 ? KIB * 1024 / (WAVES * STEP_BYTES) : 4;
  static constexpr int LOADS = STEP_BYTES / 1024;  // of a step
  static constexpr int LDS_BYTES = WAVES * NB * STEP_BYTES;
  static_assert(NB >= 2 && LDS_BYTES >= WAVES * DS_GMAX * (16 * CT + 4) * 4, "");
};

__device__ static __forceinline__ float ds_quad_max(float v) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48 that share a head
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  u = __builtin_bit_cast(uint32_t, v);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ static __forceinline__ float ds_quad_sum(float v) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
  u = __builtin_bit_cast(uint32_t, v);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)b[0]) + __builtin_bit_cast(float, (uint32_t)b[1]);
}

// LDS reads the compiler does not track: it would wait for every direct-to-LDS load in flight before each
__device__ static __forceinline__ dc_u32x4 ds_read_k(uint32_t addr) {
  dc_u32x4 r;
  asm volatile("ds_read_b128 %0, %1" : "=v"(r) : "v"(addr));
  return r;
}
template <int IMM>
__device__ static __forceinline__ ds_u32x2 ds_read_v(uint32_t addr) {
  ds_u32x2 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(IMM));
  return r;
}

// V for the product with the probabilities' second part: infinities become the largest value of their sign.  An infinite value has met its
// weight in the first product; the second part is zero or of either sign, and 0 * inf or inf - inf would make a NaN of the sum.  (Finite
// values are what they were, a NaN has made its sum NaN in the first product.)  Two instructions a register, issued under the first
// products: steps take 0.6 % longer in the median, 3 % at most (64 and fewer channels, 300 to 1025 keys); a second walk of the keys only
// where a sum came out NaN made the plain one slower (2 to 16 %).
__device__ static __forceinline__ dc_u32x4 ds_finite(dc_u32x4 v) {
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  const s16x8 pos = __builtin_elementwise_min(__builtin_bit_cast(s16x8, v), (s16x8)(short)0x7f7f);
  return __builtin_bit_cast(dc_u32x4, __builtin_elementwise_min(__builtin_bit_cast(u16x8, pos), (u16x8)(unsigned short)0xff7f));
}

// Steps in LDS: K [32 keys][D], V [32 keys][16 CT channels] in 16-byte chunks, swizzled by the row: K's chunks for reads of one chunk
// of 16 rows, V's pairs of chunks for the transposing reads of a pair of 8 rows (256 bytes, all banks, either way).
template <int D>
__device__ static __forceinline__ int ds_swz_k(int row) {
  return D == 128 ? row & 15 : (row >> 1) & 7;
}
template <int CT>
__device__ static __forceinline__ int ds_swz_v(int row) {
  return CT == 1 ? 0 : (row / (8 / CT)) & (CT - 1);
}
