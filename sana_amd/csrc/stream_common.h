// What the kernels of decay.hip and window.hip share: rows of 16-bit values in LDS, read as MFMA operands as they lie or transposed.
#pragma once
#include "common.h"

namespace sana {

typedef __attribute__((address_space(3))) unsigned char lds_t;  // (pointers, not integers: the compiler sees which array is read)

// 16-byte slots of an LDS row of DK * 64 bytes are exchanged by a key of the row, which spreads 16 consecutive rows of one slot over the banks.
// The key of row 16 i + r is that of r.  LDS cycles of a wave's instruction, by the counters: a plain read of 16 rows 4 without conflicts for DK = 2 and
// 4, 8 of which 4 are conflicts for DK = 1 and 3 (two bits of key); a transposing read 4 of which 2 are conflicts at every DK; a 16-byte write 8, none.
template <int DK>
__device__ __forceinline__ int row_key(int row) {
  return DK == 4 ? (row & 15) : DK == 2 ? ((row >> 1) & 7) : ((row >> 2) & 3);
}
__device__ __forceinline__ u32x2_t lds_read_tr(lds_t* at) {  // 4 rows x 16 channels -> this lane's channel, 4 rows
  typedef short s16x4_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)at));
}
__device__ __forceinline__ u32x4_t lds_read(const lds_t* at) { return *(__attribute__((address_space(3))) const u32x4_t*)at; }
__device__ __forceinline__ u32x2_t lds_read8(const lds_t* at) { return *(__attribute__((address_space(3))) const u32x2_t*)at; }

// What this wave wrote to LDS is there and what it reads from there has come; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// x of the lanes 16, 32 and 48 further (the four lane groups that share a column of an MFMA), combined: two exchanges of register
// halves on the vector unit, where a shuffle through LDS takes some hundred cycles each.
template <typename Op>
__device__ __forceinline__ float over_groups(float x, Op op) {
  const uint32_t a = __float_as_uint(x);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const float y = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const uint32_t b = __float_as_uint(y);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_groups(float x) {
  return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_groups(float x) {
  return over_groups(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float max_wave(float x) {  // over all 64 lanes: rotations within 16, then the groups
#define SANA_ROTATED(by) __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), 0x120 | by, 0xf, 0xf, false))
  x = fmaxf(x, SANA_ROTATED(8));
  x = fmaxf(x, SANA_ROTATED(4));
  x = fmaxf(x, SANA_ROTATED(2));
  x = fmaxf(x, SANA_ROTATED(1));
#undef SANA_ROTATED
  return max_groups(x);
}

// Values that are not finite.  What a query does not see has a probability of 0, but 0 * inf is NaN: through a product of a tile, one
// such value would reach all of the tile's queries.
template <typename T> inline constexpr uint32_t kInf16 = is_f16<T> ? 0x7c00u : 0x7f80u;
template <typename T> inline constexpr uint32_t kOne16 = is_f16<T> ? 0x3c00u : 0x3f80u;
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2_t max_magnitude(u16x2_t most, u32x4_t x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, x[e] & 0x7fff7fffu));
  return most;
}

}  // namespace sana
