// What the kernels over a window share (window.hip: 16-bit rows; window8.hip: a cache of 8 bits): sizes, the ring's rows, the join of parts of the keys.
#pragma once
#include <initializer_list>

#include "stream_common.h"

namespace sana {
namespace {

constexpr int WA_MAX_SPLITS = 32;  // parts that the keys of a query are split into

struct WindowArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out, *cache_k, *cache_v;
  const int *lengths, *positions;
  float *part_o, *part_ml;  // parts: [splits][B * N * H][d] and [splits][B * N * H][2] (maximum, sum)
  int B, N, Nk, H, Hkv, d, window, sinks, splits, qblocks, items;
  int64_t q_b, q_n, k_b, k_n, v_b, v_n, o_b, o_n, ck_b, ck_n, cv_b, cv_n;
  float scale_log2e;
};

// The parts of a query and head: weights 2^(m_s - m), sums and outputs added up in the order of the parts.  Half a wave a (query, head):
// a lane reads the maximum and the sum of one part, then four channels of all.  A launch and two loads in a row: 3.4 us for 16 heads in 13 parts.
template <typename T>
__global__ __launch_bounds__(256) void window_join_kernel(const WindowArgs a) {
  static_assert(WA_MAX_SPLITS <= 32, "");
  const int64_t rows = (int64_t)a.B * a.N * a.H, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, c = 4 * lane;
  const int64_t bn = row / a.H;
  const int h = (int)(row - bn * a.H), b = (int)(bn / a.N), i = (int)(bn - (int64_t)b * a.N);
  if ((a.lengths && i >= a.lengths[b]) || (a.positions && a.positions[b] < 0)) return;
  f32x2_t ml = {-INFINITY, 0.f};
  if (lane < a.splits) ml = *reinterpret_cast<const f32x2_t*>(a.part_ml + 2 * (lane * rows + row));
  float m = ml[0];
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 32));
  const float mine = lane < a.splits ? __builtin_amdgcn_exp2f(ml[0] - m) : 0.f;
  const float* from = a.part_o + row * a.d + (c < a.d ? c : 0);
  float l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    f32x4_t x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = *reinterpret_cast<const f32x4_t*>(from + min(s0 + s, a.splits - 1) * rows * a.d);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float f = __shfl(mine, s0 + s, 32);  // (0 behind the last part, whose values are repeated there: they may be inf)
      l = fmaf(f, __shfl(ml[1], s0 + s, 32), l);
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // a part whose weight is 0 in fp32 gives what is not finite all the same: its keys are seen
        const float y = s0 + s < a.splits ? x[s][r] : 0.f;
        o[r] = fmaf(f == 0.f && !(fabsf(y) < INFINITY) ? 1.f : f, y, o[r]);
      }
    }
  }
  const float inv = 1.0f / l;
  if (c < a.d)
    *reinterpret_cast<u32x2_t*>(a.out + b * a.o_b + (int64_t)i * a.o_n + h * a.d + c) =
        u32x2_t{pk16<T>(o[0] * inv, o[1] * inv), pk16<T>(o[2] * inv, o[3] * inv)};
}

__device__ __forceinline__ int wa_slot(int64_t p, int sinks, int window) { return (int)(p < sinks ? p : sinks + (p - sinks) % window); }

constexpr int64_t WA_MAX_BLOCKS = 1 << 24;  // of 256 threads: a launch has fewer than 2^32 threads an axis

// One token: the workgroups of a whole cache, one a (stream, key head, 16 query heads).
int64_t step_groups(int B, int H, int Hkv) { return (int64_t)B * Hkv * ((H / Hkv + 15) / 16); }
size_t part_bytes(int splits, int64_t rows, int d) { return splits > 1 ? (size_t)splits * rows * (d + 2) * sizeof(float) : 0; }

template <typename T>
int launch_join(const WindowArgs& a, hipStream_t s) {
  const int64_t groups = ((int64_t)a.B * a.N * a.H + 7) / 8;
  if (groups >= WA_MAX_BLOCKS) return SANA_ERR_SHAPE;
  hipLaunchKernelGGL(window_join_kernel<T>, dim3((unsigned)groups), dim3(256), 0, s, a);
  return SANA_OK;
}

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
