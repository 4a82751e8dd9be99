// What the attention kernels with tiles of 64 keys share (sp_attn_short.hip, sp_chunk.hip): the tiles' layout in LDS, the operand reads and
// the lane exchanges.
#pragma once
#include "sp_common.h"

#include <type_traits>

typedef __bf16 as_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 as_bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 as_bf16x2 __attribute__((ext_vector_type(2)));
typedef float as_floatx4 __attribute__((ext_vector_type(4)));
typedef float as_floatx2 __attribute__((ext_vector_type(2)));
typedef uint32_t as_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t as_u32x2 __attribute__((ext_vector_type(2)));

#define AS_TILE 64      // keys per step
#define AS_THREADS 256  // 4 waves x 32 queries
#define AS_WAVES 4
#define AS_NO_MAX (-1.0e30f)         // "no key seen yet": finite, so exp2(S * scale - m) is +inf or 0, never NaN
#define AS_P_TOO_LARGE 0x40004000u   // bf16 pair: exponent >= 128 in either half

typedef __attribute__((address_space(3))) void* as_lds_ptr;

// K and V tiles are [64 keys][D] bf16 in 16-byte chunks, the chunk index XOR-swizzled by the row so that each kind of operand read
// is free of bank conflicts.  The LDS serves 256 bytes a cycle: 16 lanes of a K read (one chunk of 16 consecutive rows), so K's
// chunks are permuted by the row; 32 lanes of a transposing V read (two neighbouring chunks of 8 consecutive rows), so V's pairs
// of chunks are: by the single chunks rows 2i and 2i + 1 met in the same banks, a third of the LDS's active cycles.  Rows of 64
// channels are half a bank cycle long: two rows share a swizzle.
template <int D>
__device__ __forceinline__ int as_swz(int row) {
  return D == 128 ? (row & 15) : ((row >> 1) & 7);
}

template <int D>
__device__ __forceinline__ int as_swz_v(int row) {
  return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
}

__device__ __forceinline__ uint32_t as_pack2(float a, float b) {
  as_floatx2 f;
  f[0] = a;
  f[1] = b;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, as_bf16x2));
}

// Transposing LDS read the compiler does not track (valid after as_wait_v on the same registers).  Through the builtin it
// waits for every direct-to-LDS load in flight before each of these reads -- the next tile's whole memory latency in
// every step: 1.6 us per 64 keys where the arithmetic takes half of that.
template <int IMM>
__device__ __forceinline__ as_u32x2 as_read_tr(uint32_t addr) {
  as_u32x2 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(IMM));
  return r;
}
template <int N>
__device__ __forceinline__ void as_wait_v(as_u32x2 (&r)[8]) {  // all but the N youngest LDS reads have landed
  asm volatile("s_waitcnt lgkmcnt(%8)"
               : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]), "+v"(r[4]), "+v"(r[5]), "+v"(r[6]), "+v"(r[7])
               : "n"(N));
}
// The same for a K operand (16 bytes of a lane's row).  Left to itself the compiler waits for each pair of these reads where it
// uses them.
template <int IMM>
__device__ __forceinline__ as_u32x4 as_read_k(uint32_t addr) {
  as_u32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(IMM));
  return r;
}
template <int N>
__device__ __forceinline__ void as_wait_k(as_u32x4 (&r)[4]) {
  asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(r[0]), "+v"(r[1]), "+v"(r[2]), "+v"(r[3]) : "n"(N));
}
template <int N>
__device__ __forceinline__ void as_wait_k(as_u32x4 (&r)[2]) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(r[0]), "+v"(r[1]) : "n"(N));
}
template <int K, int N, typename F>
__device__ __forceinline__ void as_static_for(F&& f) {
  if constexpr (K < N) {
    f(std::integral_constant<int, K>{});
    as_static_for<K + 1, N>(f);
  }
}

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48 that share a query
__device__ __forceinline__ float as_groupmax(float v) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  u = __builtin_bit_cast(uint32_t, v);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
