// What happens to a stream's heads between their projection and the attention, in one pass over the rows:
//
//   norm      x' = x * rsqrt(mean(x^2) + eps) * w over the d channels of a head, queries and keys each their weights
//   rotation  of channel pairs (a, b) by t = position * freqs[i], the first 2 * |freqs| channels of the head:
//             (a, b) -> m * (a cos t - b sin t, a sin t + b cos t); pairs (2i, 2i + 1), or (i, i + rotary / 2)
//   8 bits    a head's row of a key or a value as whole numbers c = round(127 x / max|x|), ties to even, and the scale max|x| / 127
//
// all in 32 bits and rounded once, from the unrounded values where a key is rotated and put into 8 bits in the same pass.
#include "window_common.h"

namespace sana {
namespace {

constexpr int MAX_TILES = 1 << 15;

// The scales of a head's rows in a cache begin here: (key, value) pairs, in 64 bits, since two scales each for 2^30 rows are no 32-bit number.
__host__ __device__ constexpr int64_t scales_of_head(int head, int rows) { return 2 * (int64_t)rows * head; }
static_assert(scales_of_head(1, 1 << 30) == int64_t{1} << 31 && scales_of_head(3, 1 << 30) == 3 * (int64_t{1} << 31), "the largest cache's second and last heads");

struct HeadArgs {
  sana_heads_args a;
  int gq, gk, gv, per;  // groups of heads of a token: of queries, of keys, of values; groups that a wave takes
  int whole, skipped;   // tiles behind the first `whole` ones that are left out: nothing of them stays in the cache
  int layers;           // of the grid, of MAX_TILES tiles each, that a stream takes
  float inv_d;
};

// Combined over the LPH (4, 8, 16) lanes that hold a head: exchanges within 16 lanes on the vector unit.
template <int LPH, typename V, typename Op>
__device__ __forceinline__ V over_head(V x, Op op) {
  const auto with = [&](V y, auto ctrl) {
    return op(y, __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, y), decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  x = with(x, std::integral_constant<int, 0xB1>{});   // lane ^ 1
  x = with(x, std::integral_constant<int, 0x4E>{});   // lane ^ 2
  if constexpr (LPH >= 8) x = with(x, std::integral_constant<int, 0x141>{});   // 7 - lane: the other four
  if constexpr (LPH >= 16) x = with(x, std::integral_constant<int, 0x140>{});  // 15 - lane: the other eight
  return x;
}

// x in 8 bits: 127 x / most to the nearest whole number, ties to even; inv is 1 / most up to 2 steps.  The first quotient is mended by what it leaves
// of 127 x (which is exact for 16-bit x): a tie, which fp32 holds, comes out as itself, and a quotient of two 16-bit floats that is none
// is at least 2^-19 of itself away from one.  (5 operations in the place of a division's 10.)
// (Of numbers far from 1 all three may be lifted by a power of two: t = 127 x and most by the same.)
__device__ __forceinline__ uint32_t code_bits(float t, float most, float inv) {
  const float y = t * inv;
  return __float_as_uint(fmaf(fmaf(-y, most, t), inv, y) + 12582912.0f);  // 1.5 * 2^23: the whole number in the low bits
}
__device__ __forceinline__ uint32_t pack_codes(const float* x, float c127, float most, float inv) {
  const auto code = [&](int i) { return code_bits(x[i] * c127, most, inv); };
  const uint32_t lo = __builtin_amdgcn_perm(code(1), code(0), 0x0c0c0400u), hi = __builtin_amdgcn_perm(code(3), code(2), 0x04000c0cu);
  return lo | hi;
}
// m / 127, rounded once: the product with 1 / 127, mended by what it leaves (3 operations; a division takes 10).
__device__ __forceinline__ float scale_of(float m) {
  constexpr float inv = 1.0f / 127.0f;
  const float y = m * inv;
  return m < 0x1p-100f ? m / 127.0f : fmaf(fmaf(-y, 127.0f, m), inv, y);
}

// LPH lanes hold a head, 8 channels each.  FAR: pairs half of the rotated channels apart, a lane holds four channels of either half, so that a pair never
// leaves its lane.  A wave takes one token and `per` groups of 64 / LPH of its heads, or (TOKENS) `per` heads of 64 / LPH consecutive tokens, whose rows
// in the cache lie side by side; U of them are on their way at a time.  Loads are under no condition (a lane without a head, a channel or a token repeats
// another's): the compiler puts what follows a conditional load, and the wait for it, into the same branch (16384 tokens of 20 + 20 heads of 112 78 us that
// way, 60 now).  Memory bounds it, behind some 5 us of ramp and tail a launch: those tokens 294 MB in 51 us = 5.7 TB/s; keys and values of 2 x 4680 tokens
// into the cache 126 MB in 29; queries as well 210 MB in 51 = 4.1 TB/s, of which either the stores of the queries or those of the codes are 4 (the six
// streams of rows in and out are what is slow, not the vector unit: without half of a rotation's or of a code's operations the time is the same).  Many
// short waves beat few long ones: angles in LDS for tiles of 8 to 32 tokens a workgroup 77 us, workgroups in ranges by XCD 69 to 78.
template <typename T, int LPH, bool FAR, bool TOKENS>
__global__ __launch_bounds__(256) void heads_kernel(const HeadArgs h) {
  constexpr int AT_ONCE = 64 / LPH, U = TOKENS ? 2 : 4, TW = TOKENS ? AT_ONCE : 1;  // TW: tokens of a wave
  const sana_heads_args& a = h.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, j = lane % LPH, sub = lane / LPH;
  // workgroup -> (chunk of the heads, tile of tokens, stream); the tiles of a stream in several layers of the grid if they are very many
  int b = blockIdx.z, tile = blockIdx.y;
  if (h.layers > 1) b = blockIdx.z / h.layers, tile += (blockIdx.z - b * h.layers) * MAX_TILES;
  const int chunk = blockIdx.x, first = TW * (4 * (tile + (tile >= h.whole ? h.skipped : 0)) + wave), t = TOKENS ? first + sub : first;
  if (first >= a.N) return;
  const int g0 = chunk * h.per, d = a.d;
  int g1 = min(g0 + h.per, h.gq + h.gk + h.gv);
  // groups: those of the queries, of the keys, of the values; heads one by one: the queries', then key and value in turns
  const auto kind_of = [&](int g) { return g < h.gq ? 0 : !TOKENS ? (g < h.gq + h.gk ? 1 : 2) : h.gv ? 1 + (g - h.gq) % 2 : 1; };
  const auto head_of = [&](int g, int kind) {
    if constexpr (TOKENS) return kind == 0 ? g : h.gv ? (g - h.gq) / 2 : g - h.gq;
    else return (g - (kind == 0 ? 0 : kind == 1 ? h.gq : h.gq + h.gk)) * AT_ONCE + sub;
  };
  // this lane's channels: two runs of four
  const bool in = 8 * j < d, turns = 8 * j < a.rotary, far_pair = FAR && turns;
  const int at8 = in ? 8 * j : 0, e0 = far_pair ? 4 * j : at8, e1 = far_pair ? a.rotary / 2 + 4 * j : at8 + 4;
  const int tc = min(t, a.N - 1);
  const uint16_t* in_rows[3] = {static_cast<const uint16_t*>(a.q) + b * a.q_b + tc * a.q_n, static_cast<const uint16_t*>(a.k) + b * a.k_b + tc * a.k_n,
                                static_cast<const uint16_t*>(a.v) + b * a.v_b + tc * a.v_n};
  u32x2_t x0[U], x1[U];
  const auto request = [&](int g) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int gu = min(g + u, g1 - 1), kind = kind_of(gu), head = TOKENS ? head_of(gu, kind) : min(head_of(gu, kind), (kind == 0 ? a.H : a.Hkv) - 1);
      const uint16_t* row = (kind == 0 ? in_rows[0] : kind == 1 ? in_rows[1] : in_rows[2]) + head * d;
      if constexpr (FAR) {
        x0[u] = *reinterpret_cast<const u32x2_t*>(row + (kind == 2 ? at8 : e0)), x1[u] = *reinterpret_cast<const u32x2_t*>(row + (kind == 2 ? at8 + 4 : e1));
      } else {
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(row + at8);
        x0[u] = u32x2_t{x[0], x[1]}, x1[u] = u32x2_t{x[2], x[3]};
      }
    }
  };
  // (before the position has come, unless there may be rows without a token)
  if (!a.lengths) request(g0);

  const int pos = a.positions ? a.positions[b] : 0;
  const int n = pos < 0 ? 0 : a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;  // tokens that there are
  const bool live = t < n;
  uint16_t* out_rows[2] = {static_cast<uint16_t*>(a.q_out) + b * a.qo_b + tc * a.qo_n, static_cast<uint16_t*>(a.k_out) + b * a.ko_b + tc * a.ko_n};
  if (first + TW > n && a.zero_rest) {  // rows without a token
    for (int g = g0; g < g1; ++g) {
      const int kind = kind_of(g), head = head_of(g, kind);
      if (kind < 2 && (a.zero_rest >> kind & 1) && in && t >= n && t < a.N && head < (kind ? a.Hkv : a.H))
        *reinterpret_cast<u32x4_t*>((kind ? out_rows[1] : out_rows[0]) + head * d + 8 * j) = u32x4_t{0u, 0u, 0u, 0u};
    }
  }
  if (first >= n) return;
  const uint32_t p = (uint32_t)pos + (uint32_t)t;
  const bool kept = live && a.codes_k && (p < (uint32_t)a.sinks || t >= n - a.window);  // (not pushed out by this call's own tokens)
  const bool any_kept = TOKENS ? __any(kept) : kept;
  if (!any_kept && !a.k_out) g1 = min(g1, h.gq);
  if (g0 >= g1) return;
  const int rows = a.window + a.sinks, dp = (d + 15) & ~15;
  if (a.lengths) request(g0);

  float w[2][8];  // the norms' weights
  if (a.q_weight) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint16_t* from = static_cast<const uint16_t*>(k ? a.k_weight : a.q_weight);
      const u32x2_t lo = *reinterpret_cast<const u32x2_t*>(from + e0), hi = *reinterpret_cast<const u32x2_t*>(from + e1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v = i < 2 ? lo[i] : hi[i - 2];
        w[k][2 * i] = lo16<T>(v), w[k][2 * i + 1] = hi16<T>(v);
      }
    }
  }
  float c[4], s[4];
  if (turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // in turns and 64 bits: of far positions only the fraction counts.  (Sine and cosine of -1/2 .. 1/2 turn are off by 2.1 2^-24 at most here.)
      const double at = (double)p * (a.freqs[4 * j + i] * 0.15915494309189533577);
      const float turn = (float)(at - __builtin_rint(at));
      c[i] = __builtin_amdgcn_cosf(turn) * a.magnitude, s[i] = __builtin_amdgcn_sinf(turn) * a.magnitude;
    }
  }
  const int slot = kept ? wa_slot(p, a.sinks, a.window) : 0;
  const int64_t head_codes = (int64_t)rows * dp;
  int8_t *codes_k = a.codes_k + b * a.ck_b + (int64_t)slot * dp, *codes_v = a.codes_v + b * a.cv_b + (int64_t)slot * dp;
  float* scales = a.scales + b * a.sc_b + 2 * (int64_t)slot;

#pragma unroll 1
  for (int g = g0; g < g1; g += U) {
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v = !in ? 0u : i < 2 ? x0[u][i] : x1[u][i - 2];
        x[u][2 * i] = lo16<T>(v), x[u][2 * i + 1] = hi16<T>(v);
      }
    if (g + U < g1) request(g + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int gu = g + u;
      if (gu >= g1) break;
      const int kind = kind_of(gu), head = head_of(gu, kind);
      const bool mine = in && live && (TOKENS || head < (kind == 0 ? a.H : a.Hkv)), near8 = !FAR || kind == 2;
      if (kind < 2 && a.q_weight) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq = fmaf(x[u][i], x[u][i], sq);
        const auto plus = [](float y, float z) { return y + z; };
        sq = over_head<LPH>(sq, plus);
        float eps = a.eps;
        if (!is_f16<T> && __any(sq == INFINITY)) {  // (heads whose squares leave fp32, from some 2^61 on: all of it 2^68 times smaller)
          const float by = sq == INFINITY ? 0x1p-68f : 1.0f;
          eps *= by * by, sq = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[u][i] *= by, sq = fmaf(x[u][i], x[u][i], sq);
          sq = over_head<LPH>(sq, plus);
        }
        const float r = rsqrtf(sq * h.inv_d + eps);  // (of subnormal numbers too, where eps is 0)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][i] = x[u][i] * r * (kind ? w[1][i] : w[0][i]);
      }
      if (kind < 2 && turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int i0 = FAR ? i : 2 * i, i1 = FAR ? 4 + i : 2 * i + 1;
          const float y = x[u][i0], z = x[u][i1];
          x[u][i0] = y * c[i] - z * s[i], x[u][i1] = y * s[i] + z * c[i];
        }
      }
      // The values as they are in 32 bits: f16's conversion would otherwise be one operation with the product in front of it here, where nothing else
      // needs the product, and two there, where it goes into 8 bits as well, and the same call with and without a cache differ in a bit.
#pragma unroll
      for (int i = 0; i < 8; ++i) asm("" : "+v"(x[u][i]));
      if (mine && (kind == 0 || (kind == 1 && a.k_out))) {
        uint16_t* to = (kind == 0 ? out_rows[0] : out_rows[1]) + head * d;
        const u32x4_t o = {pk16<T>(x[u][0], x[u][1]), pk16<T>(x[u][2], x[u][3]), pk16<T>(x[u][4], x[u][5]), pk16<T>(x[u][6], x[u][7])};
        if constexpr (FAR) {
          *reinterpret_cast<u32x2_t*>(to + e0) = u32x2_t{o[0], o[1]};
          *reinterpret_cast<u32x2_t*>(to + e1) = u32x2_t{o[2], o[3]};
        } else {
          *reinterpret_cast<u32x4_t*>(to + at8) = o;
        }
      }
      if (kind > 0 && any_kept) {
        float most = 0.f, odd = 0.f;  // odd: NaN if any of them is not finite
#pragma unroll
        for (int i = 0; i < 8; i += 2) most = fmaxf(fmaxf(fabsf(x[u][i]), fabsf(x[u][i + 1])), most);
#pragma unroll
        for (int i = 0; i < 8; ++i) odd = fmaf(x[u][i], 0.f, odd);
        most = over_head<LPH>(most, [](float y, float z) { return fmaxf(y, z); });
        odd = over_head<LPH>(odd, [](float y, float z) { return y + z; });
        const bool bad = odd != odd;
        // (far from 1 by a power of two towards it: a reciprocal that is a normal number)
        const float lift = most < 0x1p-100f ? 0x1p100f : most > 0x1p100f ? 0x1p-100f : 1.0f, lifted = most * lift;
        const float inv = most > 0.f ? __builtin_amdgcn_rcpf(lifted) : 0.f, c127 = 127.0f * lift;
        const uint32_t lo = bad ? 0u : pack_codes(x[u], c127, lifted, inv), hi = bad ? 0u : pack_codes(x[u] + 4, c127, lifted, inv);
        if (mine && kept) {
          int8_t* codes = (kind == 1 ? codes_k : codes_v) + head * head_codes;
          if (near8) {
            *reinterpret_cast<u32x2_t*>(codes + at8) = u32x2_t{lo, hi};
          } else {
            *reinterpret_cast<uint32_t*>(codes + e0) = lo, *reinterpret_cast<uint32_t*>(codes + e1) = hi;
          }
          if (j == 0) scales[scales_of_head(head, rows) + (kind - 1)] = bad ? __uint_as_float(0x7fc00000u) : scale_of(most);
        }
      }
    }
  }
}

// Heads, or groups of them, that a wave takes: many, and their angles once, where there are waves enough.
int heads_a_wave(int64_t waves, int groups) {
  const int64_t chunks = waves >= 4096 ? 1 : (4096 + waves - 1) / waves;
  return (int)((groups + (chunks < groups ? chunks : groups) - 1) / (chunks < groups ? chunks : groups));
}

template <typename T, int LPH, bool TOKENS>
int launch_heads(const sana_heads_args& a, hipStream_t s) {
  constexpr int AT_ONCE = 64 / LPH, TW = TOKENS ? AT_ONCE : 1, HW = TOKENS ? 1 : AT_ONCE;
  HeadArgs h = {};
  h.a = a, h.inv_d = 1.0f / a.d;
  h.gq = (a.H + HW - 1) / HW, h.gk = (a.Hkv + HW - 1) / HW, h.gv = a.codes_k ? h.gk : 0;
  const int groups = h.gq + h.gk + h.gv;
  // (TOKENS: four heads.  us of 2 / 4 / 6 / 8: 16384 tokens - / 60 / 63 / 64, all in one pass 70 / 54 / 53 / 54, 16 x 4096 tokens into short caches 26 / 23 / 28 / 25; and two
  // of them on their way: 1 / 2 / 4 57 / 55 / 57)
  h.per = TOKENS ? (groups < 4 ? groups : 4) : heads_a_wave((int64_t)a.B * a.N, groups);
  constexpr int TILE = 4 * TW;
  h.whole = (a.sinks + TILE - 1) / TILE;
  h.skipped = a.codes_k && !a.q && !a.k_out && !a.lengths && a.N > a.window ? (a.N - a.window) / TILE - h.whole : 0;
  h.skipped = h.skipped < 0 ? 0 : h.skipped;
  const int chunks = (groups + h.per - 1) / h.per, tiles = (a.N + TILE - 1) / TILE - h.skipped;
  h.layers = (tiles + MAX_TILES - 1) / MAX_TILES;
  if ((int64_t)a.B * h.layers > 65535 || (int64_t)chunks * tiles >= WA_MAX_BLOCKS / a.B) return SANA_ERR_SHAPE;
  const dim3 grid((unsigned)chunks, (unsigned)(h.layers > 1 ? MAX_TILES : tiles), (unsigned)(a.B * h.layers));
  if (a.rotary && !a.interleaved) hipLaunchKernelGGL((heads_kernel<T, LPH, true, TOKENS>), grid, dim3(256), 0, s, h);
  else hipLaunchKernelGGL((heads_kernel<T, LPH, false, TOKENS>), grid, dim3(256), 0, s, h);
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}
// Heads of one token, or runs of tokens where there are many.  us of all in one pass, heads / tokens: 20 + 20 + 20 heads of 112 1 token 4.0 / 5.3, 64 x 1
// 4.9 / 6.2, 1000 x 1 12.6 / 27.6, 64 x 16 10.3 / 10.2, 64 x 64 22.6 / 24.2, 2 x 4680 60 / 56; 32 + 8 + 8 of 128 64 x 64 19.5 / 20.6; 8 x 2047 of 32 + 8 of
// 128 in far pairs without a cache 64 / 60; into a cache alone 2 x 4680 of 5 of 112 16 / 12, 16 x 4096 of 4 of 128 40 / 23, 70 of 32 62 / 38.
// Many tokens stay heads of one where queries are among them and six groups or more of heads fill their lanes: the rows of a token are whole lines that
// one wave reads and writes.  Without a cache, near pairs (far pairs), 250 MB: 70 + 70 of 32 45.0 / 49.7 (48.7 / 63.0), 48 44.6 / 50.7 (51.4 / 62.2), 64
// 43.7 / 42.9 (48.3 / 49.6), 16 + 16 of 72 48.2 / 55.4 (54.0 / 64.1), 96 44.6 / 46.9 (52.1 / 52.8), 112 43.6 / 45.4 (48.5 / 49.3), but of 128 42.6 / 42.2
// (42.5 / 43.3), of 16 69 / 27, and with fewer groups 16 + 4 of 72 46.9 / 46.0 (57.2 / 53.3), 4 + 4 47.5 / 33.6.  With a cache its rows of codes, which lie
// by head, outweigh that up to 64 channels and from 112: 32 85.0 / 75.1, 48 84.1 / 78.0, 64 68.1 / 62.8, 72 80.9 / 91.0, 80 71.8 / 77.4, 96 72.7 / 75.9, 104
// 62.1 / 65.6, 112 65.3 / 67.2 and 52.5 / 51.3 (of two sizes: 3 % either way), 128 47.0 / 48.6 and 60 / 56.
template <typename T, int LPH>
int heads_as(const sana_heads_args& a, hipStream_t s) {
  constexpr int AT_ONCE = 64 / LPH;
  if (a.N < 64 || (int64_t)a.B * a.N < 8192) return launch_heads<T, LPH, false>(a, s);
  const int kv = a.codes_k ? 2 : 1, groups = (a.H + AT_ONCE - 1) / AT_ONCE + kv * ((a.Hkv + AT_ONCE - 1) / AT_ONCE);
  const bool full = groups >= 6 && 10 * ((int64_t)a.H + (int64_t)kv * a.Hkv) >= 7 * (int64_t)AT_ONCE * groups;
  const bool heads = a.q && full && (a.codes_k ? a.d > 64 && a.d < 112 : a.d > 16 && a.d < 128);
  return heads ? launch_heads<T, LPH, false>(a, s) : launch_heads<T, LPH, true>(a, s);
}
template <typename T>
int heads_of(const sana_heads_args& a, hipStream_t s) {
  return a.d <= 32 ? heads_as<T, 4>(a, s) : a.d <= 64 ? heads_as<T, 8>(a, s) : heads_as<T, 16>(a, s);
}

}  // namespace
}  // namespace sana

using namespace sana;

extern "C" __attribute__((visibility("default"))) int sana_hip_heads(const sana_heads_args* args, void* stream) {
  if (!args) return SANA_ERR_ARG;
  const sana_heads_args& a = *args;
  const bool cached = a.codes_k || a.codes_v || a.scales;
  if (!a.k || a.B <= 0 || a.N <= 0 || a.Hkv <= 0 || a.d <= 0 || a.H < 0 || a.rotary < 0 || (a.q == nullptr) != (a.H == 0) ||
      (a.q == nullptr) != (a.q_out == nullptr))
    return SANA_ERR_ARG;
  if (cached ? !a.codes_k || !a.codes_v || !a.scales || !a.v || !a.positions || a.window <= 0 || a.sinks < 0 : !a.k_out) return SANA_ERR_ARG;
  if (a.zero_rest & ~((a.q_out ? 1 : 0) | (a.k_out ? 2 : 0))) return SANA_ERR_ARG;  // (rows of an output that is not there)
  if ((a.q_weight == nullptr) != (a.k_weight == nullptr) || (a.freqs == nullptr) != (a.rotary == 0) || !(a.eps >= 0.f && a.eps < INFINITY) ||
      !(fabsf(a.magnitude) < INFINITY))
    return SANA_ERR_ARG;
  if (a.io_dtype != SANA_DT_BF16 && a.io_dtype != SANA_DT_F16) return SANA_ERR_DTYPE;
  if (a.d % 8 || a.d > 128 || a.rotary % 8 || a.rotary > a.d || a.N > (1 << 30) || (int64_t)a.H * a.d > (1 << 22) || (int64_t)a.Hkv * a.d > (1 << 22))
    return SANA_ERR_SHAPE;
  const int64_t wq = (int64_t)a.H * a.d, wk = (int64_t)a.Hkv * a.d;
  if ((a.q && (a.q_n < wq || a.qo_n < wq || a.q_b < 0 || a.qo_b < 0)) || a.k_n < wk || a.k_b < 0 || (a.k_out && (a.ko_n < wk || a.ko_b < 0)) ||
      (cached && (a.v_n < wk || a.v_b < 0)))
    return SANA_ERR_ARG;
  if (a.B > 1 && ((a.q && a.qo_b < wq) || (a.k_out && a.ko_b < wk))) return SANA_ERR_ARG;  // (entries that would write the same elements)
  // in place: the lane that reads a channel writes it, so its place has to be the same one
  if ((a.q && a.q == a.q_out && (a.q_n != a.qo_n || (a.B > 1 && a.q_b != a.qo_b))) ||
      (a.k == a.k_out && (a.k_n != a.ko_n || (a.B > 1 && a.k_b != a.ko_b))))
    return SANA_ERR_ARG;
  if (cached) {
    if (a.window > (1 << 30) || a.sinks > (1 << 30) || (int64_t)a.window + a.sinks > (1 << 30)) return SANA_ERR_SHAPE;
    const int64_t rows = a.window + a.sinks, codes = a.Hkv * rows * ((a.d + 15) & ~15);
    if (a.ck_b < 0 || a.cv_b < 0 || a.sc_b < 0 || (a.B > 1 && (a.ck_b < codes || a.cv_b < codes || a.sc_b < 2 * a.Hkv * rows))) return SANA_ERR_ARG;
    if (misaligned({a.codes_k, a.codes_v, a.v}, {a.v_b, a.v_n}) || a.ck_b % 16 || a.cv_b % 16 || a.sc_b % 2 ||
        (reinterpret_cast<uintptr_t>(a.scales) & 7u))
      return SANA_ERR_ALIGN;
  }
  if (misaligned({a.q, a.k, a.q_out, a.k_out}, {a.k_b, a.k_n}) || (a.q && misaligned({}, {a.q_b, a.q_n, a.qo_b, a.qo_n})) ||
      (a.k_out && misaligned({}, {a.ko_b, a.ko_n})) || off4(a.positions) || off4(a.lengths) ||
      ((reinterpret_cast<uintptr_t>(a.q_weight) | reinterpret_cast<uintptr_t>(a.k_weight)) & 7u) || (reinterpret_cast<uintptr_t>(a.freqs) & 7u))
    return SANA_ERR_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a.io_dtype == SANA_DT_F16 ? heads_of<F16>(a, s) : heads_of<BF16>(a, s);
}
