// What the kernels of a stream's window and its ring cache share (window.hip: 16-bit rows; window8.hip and heads.hip: a cache of 8 bits): arguments, the
// ring's rows, sizes and alignment.
#pragma once
#include <initializer_list>

#include "stream_common.h"

namespace sana {
namespace {

struct WindowArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out, *cache_k, *cache_v;
  const int *lengths, *positions;
  float *part_o, *part_ml;  // parts: [splits][B * N * H][d] and [splits][B * N * H][2] (maximum, sum)
  int B, N, Nk, H, Hkv, d, window, sinks, splits, qblocks, items;
  int64_t q_b, q_n, k_b, k_n, v_b, v_n, o_b, o_n, ck_b, ck_n, cv_b, cv_n;
  float scale_log2e;
};

// The row of the token at position p (below 2^32) in a cache of sinks + window rows.
__device__ __forceinline__ int wa_slot(uint32_t p, int sinks, int window) {
  return (int)(p < (uint32_t)sinks ? p : (uint32_t)sinks + (p - (uint32_t)sinks) % (uint32_t)window);
}

constexpr int64_t WA_MAX_BLOCKS = 1 << 24;  // of 256 threads: a launch has fewer than 2^32 threads an axis

// One token: the workgroups of a whole cache, one a (stream, key head, 16 query heads).
int64_t step_groups(int B, int H, int Hkv) { return (int64_t)B * Hkv * ((H / Hkv + 15) / 16); }
size_t part_bytes(int splits, int64_t rows, int d) { return splits > 1 ? (size_t)splits * rows * (d + 2) * sizeof(float) : 0; }

bool misaligned(std::initializer_list<const void*> rows, std::initializer_list<int64_t> strides) {
  for (const void* p : rows)
    if (!aligned16(p)) return true;
  for (const int64_t s : strides)
    if (s % 8) return true;
  return false;
}
bool off4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }

// sizes that all calls share
int check_sizes(int B, int N, int H, int Hkv, int d, int window, int sinks, int io_dtype) {
  if (B <= 0 || N <= 0 || H <= 0 || Hkv <= 0 || d <= 0 || window <= 0 || sinks < 0 || H % Hkv) return SANA_ERR_ARG;
  if (io_dtype != SANA_DT_BF16 && io_dtype != SANA_DT_F16) return SANA_ERR_DTYPE;
  if (d % 8 || d > 128 || N > (1 << 30) || window > (1 << 30) || sinks > (1 << 30) || (int64_t)H * d > (1 << 22)) return SANA_ERR_SHAPE;
  return SANA_OK;
}

}  // namespace
}  // namespace sana
