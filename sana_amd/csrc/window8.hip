// A stream's ring cache in 8 bits (written by heads.hip): one token's softmax attention over it, and its rows in the order of their tokens.
//
//   out = sum_j softmax_j(scale * sk_j (q . ck_j)) sv_j cv_j,   c whole numbers of -127 .. 127, sk and sv fp32, one of each for a head's row
//
// A head's rows lie one behind the other, [key head][row][d'], d' = d rounded up to 16, their scales as pairs [key head][row][2].
#include "window_common.h"

namespace sana {
namespace {

struct Window8Args {
  WindowArgs w;  // (its caches unused)
  const int8_t *ck, *cv;
  const float* scales;
  int64_t ck_b, cv_b, sc_b;
};

// four codes of a word as floats
__device__ __forceinline__ f32x4_t codes_f32(uint32_t x) {
  return f32x4_t{(float)(int8_t)x, (float)(int8_t)(x >> 8), (float)(int8_t)(x >> 16), (float)((int32_t)x >> 24)};
}
// eight codes as 16-bit floats, which hold them exactly
template <typename T>
__device__ __forceinline__ u32x4_t codes16(uint32_t lo, uint32_t hi) {
  const f32x4_t a = codes_f32(lo), b = codes_f32(hi);
  if constexpr (is_f16<T>) {
    const auto pk = [](float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y)); };
    return u32x4_t{pk(a[0], a[1]), pk(a[2], a[3]), pk(b[0], b[1]), pk(b[2], b[3])};
  } else {
    return u32x4_t{pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(b[0], b[1]), pack_bf16(b[2], b[3])};
  }
}

// One token of each stream.  A workgroup takes a part of the rows of one (stream, key head) and 16 * VP channels of its values, its NW waves in turn a
// tile of 16 * RT rows; the query heads that share the key head are the 16 columns of the products (more than 16 in further workgroups).  K comes from
// memory as the operand it is (16 channels a lane, two products), V through the wave's own LDS as bf16 to be transposed; its scale goes to the probability, and both as
// the sum of two bf16 numbers into the product.  (bf16 for f16 too: a value's scale may be of any size.)
// A probability is 2^(score - reference), and the reference moves only where a score is 8 above it.  It lies 48 above the scores of a tile with a value's scale over
// 2^80, so that sums of up to 2^30 rows, of 2^-40 times 127 times any scale each, stay below 2^127; 48 below those of a tile whose values' scales are all under
// 2^-64, so that neither bf16 number is a subnormal one.  Sums of waves and of parts are relative to their reference, whatever it is.
// Every compute unit busy, memory bounds it: 64 streams x 8196 rows x 8 key heads of 128, 1.05 GB 166 us = 6.3 TB/s, reads alone (179 with loads that stay in
// the caches; 4, 6, 12 waves 169, 175, 173; 64 rows a wave 185).  One stream of 131136 rows, 277 MB in 32 parts: 48 - 49 us a call in a long run over rotating
// caches, 45 - 48 of them this kernel = 6 TB/s (25 parts 55, 48 parts 60: a part a compute unit), but 61 over the first milliseconds of a run, 56 of them this one.
// A short cache is what one compute unit takes in, 37 bytes a ns at most whatever is asked for (two tiles ahead no faster) behind 6 us of launch, first loads and
// the waves' sum, so the values' channels go to several: 16 key heads of 72 x 1028 rows 11.3 us whole, 9.0 by three.  Products of 8-bit numbers in the place of
// the conversions (q in three slices): 4 % less for a cache that one compute unit takes, nothing elsewhere.
template <typename T, int P, int VP, int NW, int RT>
__global__ __launch_bounds__(64 * NW) void window_q8_kernel(const Window8Args x) {
  const WindowArgs& a = x.w;
  constexpr int DP = 16 * P, KS = (P + 3) / 4, DK = (VP + 1) / 2, DT = VP, PITCH = DK * 64, ROWS = 16 * RT, TILE = ROWS * PITCH;
  constexpr int PV = (ROWS * VP + 63) / 64, SUMS = 16 * 16 * DT * 4 + 128;  // PV: 16-byte pieces of V a lane
  constexpr int OWN = (TILE + 2 * 4 * ROWS > SUMS ? TILE + 2 * 4 * ROWS : SUMS);
  __shared__ __attribute__((aligned(16))) unsigned char smem[NW * OWN];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, fr = lane & 15, fg = lane >> 4;
  unsigned char* mine = smem + wave * OWN;
  float* my_scales = reinterpret_cast<float*>(mine + TILE);  // of the keys, then of the values
  const int G = a.H / a.Hkv, blocks = (G + 15) / 16, d = a.d;
  const uint32_t split = blockIdx.y, bk = blockIdx.x / (uint32_t)blocks;
  const int gb = blockIdx.x - bk * blocks, b = bk / (uint32_t)a.Hkv, hk = bk - b * a.Hkv;
  const int pos = a.positions[b], rows = a.window + a.sinks, v0_piece = VP < P ? VP * blockIdx.z : 0;
  const int64_t head_rows = (int64_t)hk * rows;
  const int8_t *ck = x.ck + b * x.ck_b + head_rows * DP, *cv = x.cv + b * x.cv_b + head_rows * DP;
  const float* scales = x.scales + b * x.sc_b + 2 * head_rows;

  const int head = 16 * gb + fr, h = hk * G + min(head, G - 1);
  u32x4_t qf[KS][2];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = 16 * (4 * s + fg) + 8 * half;
      qf[s][half] = *reinterpret_cast<const u32x4_t*>(a.q + b * a.q_b + h * d + (c < d ? c : 0));
      if (c >= d) qf[s][half] = u32x4_t{0u, 0u, 0u, 0u};  // (codes are finite: what lies behind d counts as nothing)
    }

  u32x4_t rk[RT][KS], rv[PV];
  f32x2_t rs[(ROWS + 63) / 64];
  // (scalar bases and 32-bit offsets within a tile; rows that hold no token yet are read, and count as nothing; the hint: what is read once leaves the caches to others)
  auto request = [&](int t) {
    const int left = rows - 1 - ROWS * t;
    const int8_t *k0 = ck + (int64_t)(ROWS * DP) * t, *v0 = cv + (int64_t)(ROWS * DP) * t;
    const float* s0 = scales + (int64_t)(2 * ROWS) * t;
#pragma unroll
    for (int kt = 0; kt < RT; ++kt)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        rk[kt][s] = load_stream<true>(reinterpret_cast<const u32x4_t*>(k0 + (uint32_t)(min(16 * kt + fr, left) * DP + 16 * min(4 * s + fg, P - 1))));
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const int idx = lane + 64 * i, r = idx / VP, c = idx - r * VP;
      rv[i] = load_stream<true>(reinterpret_cast<const u32x4_t*>(v0 + (uint32_t)(min(r, left) * DP + 16 * (VP < P ? min(v0_piece + c, P - 1) : c))));
    }
#pragma unroll
    for (int i = 0; i < (ROWS + 63) / 64; ++i)
      rs[i] = *reinterpret_cast<const f32x2_t*>(s0 + (uint32_t)(2 * min(64 * i + lane, left)));
  };
  // A whole cache's first tiles are on their way before the position has come; of parts it says where they begin.
  const bool whole = a.splits == 1;
  if (whole) request(min(wave, (rows - 1) / ROWS));
  if (pos < 0) {  // an idle stream: zeros
    if (split == 0 && gb == 0 && blockIdx.z == 0)
      for (int c = tid; c < G * d; c += 64 * NW) a.out[b * a.o_b + hk * G * d + c] = 0;
    return;
  }
  const int count = pos < rows ? pos + 1 : rows;
  const int tiles = (count + ROWS - 1) / ROWS;  // (2^25 at most, and 64 parts)
  const int t0 = whole ? 0 : (int)((uint32_t)tiles * split / a.splits), t1 = whole ? tiles : (int)((uint32_t)tiles * (split + 1) / a.splits);
  if (!whole && t0 + wave < t1) request(t0 + wave);
  f32x4_t oc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, sub = 0.f, sum = 0.f;
  const int trow = 4 * fg + (fr >> 2), tkey = row_key<DK>(trow), piece = fr & 3;
#pragma unroll 1
  for (int t = t0 + wave; t < t1; t += NW) {
    f32x4_t sc[RT];
#pragma unroll
    for (int kt = 0; kt < RT; ++kt) sc[kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float sv[(ROWS + 63) / 64];  // the values' scales, 0 of a row that is not there, so that nothing of it counts
#pragma unroll
    for (int i = 0; i < (ROWS + 63) / 64; ++i) {
      sv[i] = 64 * i + lane < min(ROWS, count - ROWS * t) ? rs[i].y : 0.f;
      if (64 * i + lane < ROWS) my_scales[64 * i + lane] = rs[i].x, my_scales[ROWS + 64 * i + lane] = sv[i];
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int kt = 0; kt < RT; ++kt) {
        sc[kt] = mfma_16x16x32<T>(codes16<T>(rk[kt][s][0], rk[kt][s][1]), qf[s][0], sc[kt]);
        sc[kt] = mfma_16x16x32<T>(codes16<T>(rk[kt][s][2], rk[kt][s][3]), qf[s][1], sc[kt]);
      }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const int idx = lane + 64 * i, r = idx / VP, c = idx - r * VP;
      if (ROWS * VP % 64 == 0 || r < ROWS) {
        unsigned char* to = mine + r * PITCH;
        *reinterpret_cast<u32x4_t*>(to + (((2 * c) ^ row_key<DK>(r & 15)) << 4)) = codes16<BF16>(rv[i][0], rv[i][1]);
        *reinterpret_cast<u32x4_t*>(to + (((2 * c + 1) ^ row_key<DK>(r & 15)) << 4)) = codes16<BF16>(rv[i][2], rv[i][3]);
      }
    }
    if (t + NW < t1) request(t + NW);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the wave's own scales and V are there)
    uint64_t over = 0, ordinary = 0;  // rows
#pragma unroll
    for (int i = 0; i < (ROWS + 63) / 64; ++i)
      over |= __builtin_amdgcn_ballot_w64(sv[i] > 0x1p80f), ordinary |= __builtin_amdgcn_ballot_w64(sv[i] >= 0x1p-64f);
    const float lift = over ? 48.f : ordinary ? 0.f : -48.f;
    float most = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < RT; ++kt) {
      const f32x4_t sk = *reinterpret_cast<const f32x4_t*>(my_scales + 16 * kt + 4 * fg);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[kt][r] = ROWS * t + 16 * kt + 4 * fg + r < count ? sc[kt][r] * a.scale_log2e * sk[r] : -INFINITY;
        most = fmaxf(most, sc[kt][r]);
      }
    }
    most += lift;
    if (__any(most > mx + 8.f)) {
      const float now = fmaxf(mx, max_groups(most));
      const float f = __builtin_amdgcn_exp2f(mx - (now == -INFINITY ? 0.f : now));
      mx = now, sub = now == -INFINITY ? 0.f : now;
      sum *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) oc[dt][r] *= f;
    }
#pragma unroll
    for (int k2 = 0; k2 < RT / 2; ++k2) {
      u32x4_t hi, lo;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f32x4_t scale = *reinterpret_cast<const f32x4_t*>(my_scales + ROWS + 16 * (2 * k2 + kt) + 4 * fg);
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = __builtin_amdgcn_exp2f(sc[2 * k2 + kt][r] - sub);
          sum += p[r];
          p[r] *= scale[r];
        }
        hi[2 * kt] = pack_bf16(p[0], p[1]), hi[2 * kt + 1] = pack_bf16(p[2], p[3]);
        lo[2 * kt] = pack_bf16(p[0] - bf16_lo(hi[2 * kt]), p[1] - bf16_hi(hi[2 * kt]));
        lo[2 * kt + 1] = pack_bf16(p[2] - bf16_lo(hi[2 * kt + 1]), p[3] - bf16_hi(hi[2 * kt + 1]));
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        lds_t* from = (lds_t*)mine + (32 * k2 + trow) * PITCH + (((2 * dt + (piece >> 1)) ^ tkey) << 4) + 8 * (piece & 1);
        const u32x2_t v0 = lds_read_tr(from), v1 = lds_read_tr(from + 16 * PITCH);
        const u32x4_t vf = u32x4_t{v0.x, v0.y, v1.x, v1.y};
        oc[dt] = mfma_16x16x32_bf16(vf, lo, oc[dt]);
        oc[dt] = mfma_16x16x32_bf16(vf, hi, oc[dt]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // ---- the waves' parts, through LDS: [channel][head], then the maxima and sums
  sum = sum_groups(sum);
  float* po = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) po[(16 * dt + 4 * fg + r) * 16 + fr] = oc[dt][r];
  if (fg == 0) po[16 * 16 * DT + fr] = mx, po[16 * 16 * DT + 16 + fr] = sum;
  lds_barrier();
  auto part = [&](int w) { return reinterpret_cast<const float*>(smem + w * OWN); };
  const int col = tid & 15, g = 16 * gb + col;
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) m = fmaxf(m, part(w)[16 * 16 * DT + col]);
  const float base = m == -INFINITY ? 0.f : m;
  float f[NW], l = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    f[w] = __builtin_amdgcn_exp2f(part(w)[16 * 16 * DT + col] - base);
    l = fmaf(f[w], part(w)[16 * 16 * DT + 16 + col], l);
  }
  if (g >= G) return;
  const int64_t at = ((int64_t)split * a.B + b) * a.H + hk * G + g;
  const float inv = 1.0f / l;
  for (int c = 16 * v0_piece + (tid >> 4); c < min(d, 16 * (v0_piece + VP)); c += 4 * NW) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) o = fmaf(f[w], part(w)[(c - 16 * v0_piece) * 16 + col], o);
    if (a.splits == 1) a.out[b * a.o_b + (hk * G + g) * d + c] = (uint16_t)pk16<T>(o * inv, 0.f);
    else a.part_o[at * d + c] = o;
  }
  if (a.splits > 1 && tid < 16 && blockIdx.z == 0) a.part_ml[2 * at] = m, a.part_ml[2 * at + 1] = l;
}

// The parts of a query head (32 heads in 32 parts 4.4 us), a workgroup a head: weights 2^(m_s - m) from a lane a part, then eight parts at a time, 32 lanes of four channels each,
// all of a lane's parts on their way at once; sums in a fixed order.
constexpr int Q8_MAX_SPLITS = 64;
constexpr int Q8_NW = 8;
constexpr int64_t Q8_MAX_GROUPS = WA_MAX_BLOCKS * 256 / (64 * Q8_NW);  // (of 512 threads)
template <typename T>
__global__ __launch_bounds__(256) void q8_join_kernel(const WindowArgs a) {
  __shared__ float sums[8][128];
  const int row = blockIdx.x, b = row / a.H, h = row - b * a.H, lane = threadIdx.x & 63, part = threadIdx.x >> 5, c = 4 * (threadIdx.x & 31);
  if (a.positions[b] < 0) return;
  const int64_t rows = (int64_t)a.B * a.H;
  const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(a.part_ml + 2 * (min(lane, a.splits - 1) * rows + row));
  f32x4_t x[Q8_MAX_SPLITS / 8];
#pragma unroll
  for (int i = 0; i < Q8_MAX_SPLITS / 8; ++i)
    x[i] = *reinterpret_cast<const f32x4_t*>(a.part_o + (min(8 * i + part, a.splits - 1) * rows + row) * a.d + min(c, a.d - 4));
  const float m = max_wave(ml[0]), f = lane < a.splits ? __builtin_amdgcn_exp2f(ml[0] - m) : 0.f;
  float l = f == 0.f && ml[1] == ml[1] ? 0.f : f * ml[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < Q8_MAX_SPLITS / 8; ++i) {
    const float fi = __shfl(f, 8 * i + part);
    if (8 * i + part < a.splits)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = fmaf(fi, x[i][r], o[r]);
  }
  *reinterpret_cast<f32x4_t*>(&sums[part][c]) = o;
  __syncthreads();
  if (threadIdx.x >= 32 || c >= a.d) return;
  f32x4_t sum = *reinterpret_cast<const f32x4_t*>(&sums[0][c]);
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += *reinterpret_cast<const f32x4_t*>(&sums[i][c]);
  const float inv = 1.0f / l;
  *reinterpret_cast<u32x2_t*>(a.out + b * a.o_b + h * a.d + c) = u32x2_t{pk16<T>(sum[0] * inv, sum[1] * inv), pk16<T>(sum[2] * inv, sum[3] * inv)};
}

// ---------------------------------------------------------------------------- rows in order

struct ReadArgs {
  const unsigned char *k, *v;  // 16-bit rows or codes
  const float* scales;
  const int* positions;
  uint16_t *out_k, *out_v;
  int B, Hkv, d, dp, window, sinks, last, rows, by_eighths, zero_rest;  // rows: that a wave takes; by_eighths: 2^16 over a row's pieces of 8 channels, rounded up
  int64_t k_b, k_n, v_b, v_n, sc_b, ok_b, ok_n, ov_b, ov_n;  // k_b .. v_n in bytes
  int64_t items;
};

// A stream's rows in order (uniform): how many it has, and by how much its tokens lie further in the ring than their output rows behind the sinks.
struct InOrder {
  int count, turned;
};
__device__ __forceinline__ InOrder in_order(const ReadArgs& a, int pos) {
  const int held = a.sinks + a.last;
  if (pos <= held) return {max(pos, 0), 0};  // tokens 0 .. pos - 1, none pushed out: row i is row i
  return {held, (int)((uint32_t)(pos - held) % (uint32_t)a.window)};
}
__device__ __forceinline__ int read_slot(const ReadArgs& a, InOrder o, int i) {
  const int row = i + o.turned;
  return i < a.sinks ? i : row < a.sinks + a.window ? row : row - a.window;  // (last <= window: once round at most)
}

// 16-bit rows: a wave copies a row of keys or of values.
__global__ __launch_bounds__(256) void read16_kernel(const ReadArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t item = 4 * blockIdx.x + wave, held = a.sinks + a.last, rest = item >> 1;
  if (item >= (uint32_t)a.items) return;
  const int of_v = item & 1, b = rest / held, i = rest - b * held, width = a.Hkv * a.d;
  const InOrder o = in_order(a, a.positions[b]);
  uint16_t* to = of_v ? a.out_v + b * a.ov_b + i * a.ov_n : a.out_k + b * a.ok_b + i * a.ok_n;
  if (i >= o.count) {
    if (a.zero_rest)
      for (int c = 8 * lane; c < width; c += 512) *reinterpret_cast<u32x4_t*>(to + c) = u32x4_t{0u, 0u, 0u, 0u};
    return;
  }
  const int64_t slot = read_slot(a, o, i);
  const unsigned char* from = of_v ? a.v + b * a.v_b + slot * a.v_n : a.k + b * a.k_b + slot * a.k_n;
  for (int c0 = 8 * lane; c0 < width; c0 += 2048) {
    u32x4_t x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const u32x4_t*>(from + 2 * min(c0 + 512 * u, width - 8));
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + 512 * u < width) *reinterpret_cast<u32x4_t*>(to + c0 + 512 * u) = x[u];
  }
}

constexpr int READ_STEPS = 4;

// Narrow 16-bit rows (up to 256 channels): a wave copies READ_STEPS times as many rows of keys or of values as it has lanes for.  292968 rows of 64 channels of two
// streams 266 us by a wave a row, 56 so; 146484 of 128 144 and 56.
__global__ __launch_bounds__(256) void read16_narrow_kernel(const ReadArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t item = 4 * blockIdx.x + wave;
  if (item >= (uint32_t)a.items) return;
  const int of_v = item & 1, b = blockIdx.y, i0 = a.rows * (item >> 1);
  const int eighths = a.Hkv * a.d / 8, step = 64 / eighths, r = lane * a.by_eighths >> 16, c = lane - r * eighths, end = min(i0 + a.rows, a.sinks + a.last);
  const InOrder o = in_order(a, a.positions[b]);
  const unsigned char* from = (of_v ? a.v + b * a.v_b : a.k + b * a.k_b) + 16 * c;
  uint16_t* to = (of_v ? a.out_v + b * a.ov_b : a.out_k + b * a.ok_b) + 8 * c;
  const int64_t from_n = of_v ? a.v_n : a.k_n, to_n = of_v ? a.ov_n : a.ok_n;
  u32x4_t x[READ_STEPS];
#pragma unroll
  for (int u = 0; u < READ_STEPS; ++u) x[u] = *reinterpret_cast<const u32x4_t*>(from + read_slot(a, o, min(i0 + u * step + r, end - 1)) * from_n);
#pragma unroll
  for (int u = 0; u < READ_STEPS; ++u) {
    const int i = i0 + u * step + r;
    if (r < step && i < end && (i < o.count || a.zero_rest)) *reinterpret_cast<u32x4_t*>(to + i * to_n) = i < o.count ? x[u] : u32x4_t{0u, 0u, 0u, 0u};
  }
}

// Codes: a wave takes READ_STEPS * R rows of a head's keys or values, R = 64 / (d / 8) in a step, 8 channels a lane.  Memory bounds it: 2 x 10920 rows of 20
// heads of 112, 297 MB 55 - 61 us = 5.2 TB/s (2, 3, 4, 6, 8 steps 64, 62, 62, 63, 64 us a call; with loads under a condition 86).
// Stores that stay in the caches: a chunk's attention reads the rows next, and takes 12 us longer where they were streamed past (2 x 10920 rows of 20 heads
// of 112, in front of 1 to 4680 queries), though the call alone, behind the one that wrote the codes, is up to 15 % shorter.
template <typename T, bool NT>
__global__ __launch_bounds__(256) void read8_kernel(const ReadArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // wave -> (head of keys or of values, block of rows); grid -> (four waves, stream)
  const uint32_t item = 4 * blockIdx.x + wave, pairs = 2 * a.Hkv, block = item / pairs, pair = item - block * pairs;
  if (item >= (uint32_t)a.items) return;
  const int of_v = pair >= (uint32_t)a.Hkv, hk = of_v ? pair - a.Hkv : pair, b = blockIdx.y, i0 = a.rows * block;
  const int eighths = a.d / 8, step = 64 / eighths, r = lane * a.by_eighths >> 16, c = lane - r * eighths;
  const int end = min(i0 + a.rows, a.sinks + a.last), cached = a.sinks + a.window;
  const InOrder o = in_order(a, a.positions[b]);
  const unsigned char* from = (of_v ? a.v + b * a.v_b : a.k + b * a.k_b) + (int64_t)hk * cached * a.dp + 8 * c;
  const float* scales = a.scales + b * a.sc_b + 2 * (int64_t)hk * cached + of_v;
  uint16_t* to = (of_v ? a.out_v + b * a.ov_b : a.out_k + b * a.ok_b) + hk * a.d + 8 * c;
  const int64_t to_n = of_v ? a.ov_n : a.ok_n;
  u32x2_t x[READ_STEPS];
  float s[READ_STEPS];
#pragma unroll
  for (int u = 0; u < READ_STEPS; ++u) {  // (under no condition, so that none waits for another: lanes without a row repeat one)
    const int64_t slot = read_slot(a, o, min(i0 + u * step + r, end - 1));
    x[u] = load_stream<NT>(reinterpret_cast<const u32x2_t*>(from + slot * a.dp));
    s[u] = scales[2 * slot];
  }
#pragma unroll
  for (int u = 0; u < READ_STEPS; ++u) {
    const int i = i0 + u * step + r;
    const f32x4_t y = codes_f32(x[u].x), z = codes_f32(x[u].y);
    u32x4_t v = {pk16<T>(y[0] * s[u], y[1] * s[u]), pk16<T>(y[2] * s[u], y[3] * s[u]), pk16<T>(z[0] * s[u], z[1] * s[u]), pk16<T>(z[2] * s[u], z[3] * s[u])};
    if (i >= o.count) v = u32x4_t{0u, 0u, 0u, 0u};
    if (r < step && i < end && (i < o.count || a.zero_rest)) *reinterpret_cast<u32x4_t*>(to + i * to_n) = v;
  }
}

template <typename T, bool NT>
void read8(const ReadArgs& a, dim3 grid, hipStream_t s) { hipLaunchKernelGGL((read8_kernel<T, NT>), grid, dim3(256), 0, s, a); }

// Parts of a cache's rows.  Short caches are taken whole: parts cost a second launch, 2 us on the device and 3.5 of the host's where calls are issued one by
// one.  Longer ones of few streams in as many parts as the 256 compute units take at once, one each, but of 64 rows and more; where a few workgroups
// more than that leave most of a second round idle, in three.  us a call, whole / in these parts: 8 key heads of 128 x 1600 rows 12.1 / 13.5, x 2052 15.7 /
// 13.7, x 4100 34.7 / 15.0, x 16388 122 / 14.7; 20 of 112 x 1500 13.0 / 13.7, x 2052 16.2 / 13.5; 80 x 1300 13.2 / 14.0, x 1700 16.1 / 14.9, x 4100 35.3 / 21.1; 120 x
// 1300 13.6 / 16.2, x 2052 19.9 / 19.2; 70 of 64 x 2052 12.8 / 14.1, x 3000 16.6 / 14.2; 70 of 32 x 1028 10 / 14.7, x 4100 19.2 / 13.7; 160 of 112 x 4100 38 / whole; 260 x
// 2052 40 / 42, x 4100 73 / 65, 300 x 8200 135 / 113, 400 x 4100 79 / whole (in three 83).
int q8_splits(int B, int H, int Hkv, int rows, int d) {
  const int64_t groups = step_groups(B, H, Hkv);
  if (groups <= 256 ? rows <= (d <= 64 ? 2048 : 1600) : (int64_t)rows * d * 2 <= (768 << 10)) return 1;
  const int most = rows / 64 < Q8_MAX_SPLITS ? rows / 64 : Q8_MAX_SPLITS;
  const int64_t want = groups <= 256 ? 256 / groups : groups * 100 < (groups + 255) / 256 * 256 * 65 ? 3 : 1;
  return (int)(want > most ? most : want < 1 ? 1 : want);
}

template <typename T, int P>
int launch_q8(const Window8Args& x, hipStream_t s) {
  const WindowArgs& a = x.w;
  const int64_t groups = step_groups(a.B, a.H, a.Hkv);
  const int64_t workgroups = groups * a.splits;
  const auto launch = [&](auto tiles) {
    constexpr int VP = decltype(tiles)::value;
    hipLaunchKernelGGL((window_q8_kernel<T, P, VP, Q8_NW, 2>), dim3((unsigned)groups, (unsigned)a.splits, (P + VP - 1) / VP), dim3(64 * Q8_NW), 0, s, x);
  };
  // The values' channels over several workgroups where compute units are left: each takes all keys and 32 channels, or half, of the values, which is 5/8
  // or 3/4 of what one would have to take in.  us on the device of one / two / four a key head, caches taken whole: 16 heads of 72 x 1028 rows 11.3 / 10.1 /
  // 9.0 (three), 20 of 112 x 1028 13.5 / 11.6 / 10.4, x 516 9.6 / 8.5 / 7.6, 8 of 128 x 260 7.6 / 6.7 / 6.5, 80 of 112 x 1028 14.2 / 11.8 / 17.4, 35 of 64 x
  // 1028 9.4 / 8.4 / 9.1 (16 channels each), 36 of 32 x 1028 8.1 / 8.0 (16 each).
  if constexpr (P >= 3) {
    if (workgroups * ((P + 1) / 2) <= 256) {
      launch(std::integral_constant<int, 2>{});
    } else if (P >= 5 && workgroups * 2 <= 256) {
      launch(std::integral_constant<int, (P + 1) / 2>{});
    } else {
      launch(std::integral_constant<int, P>{});
    }
  } else {
    launch(std::integral_constant<int, P>{});
  }
  if (a.splits > 1) hipLaunchKernelGGL(q8_join_kernel<T>, dim3((unsigned)(a.B * a.H)), dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}
template <typename T>
int q8_of(const Window8Args& x, hipStream_t s) {
  switch ((x.w.d + 15) / 16) {
    case 1: return launch_q8<T, 1>(x, s);
    case 2: return launch_q8<T, 2>(x, s);
    case 3: return launch_q8<T, 3>(x, s);
    case 4: return launch_q8<T, 4>(x, s);
    case 5: return launch_q8<T, 5>(x, s);
    case 6: return launch_q8<T, 6>(x, s);
    case 7: return launch_q8<T, 7>(x, s);
    default: return launch_q8<T, 8>(x, s);
  }
}

}  // namespace
}  // namespace sana

using namespace sana;

#define SANA_API extern "C" __attribute__((visibility("default")))

SANA_API size_t sana_hip_window_q8_workspace_bytes(int B, int H, int Hkv, int d, int window, int sinks) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || d <= 0 || d > 128 || window <= 0 || sinks < 0 || (int64_t)window + sinks > (1 << 30)) return 0;
  if (step_groups(B, H, Hkv) >= Q8_MAX_GROUPS) return 0;
  return part_bytes(q8_splits(B, H, Hkv, window + sinks, d), (int64_t)B * H, d);
}

SANA_API int sana_hip_window_q8(const sana_window_q8_args* args, void* stream) {
  if (!args) return SANA_ERR_ARG;
  const void *q = args->q, *codes_k = args->codes_k, *codes_v = args->codes_v;
  const float* scales = args->scales;
  const int32_t* positions = args->positions;
  void *out = args->out, *workspace = args->workspace;
  const int B = args->B, H = args->H, Hkv = args->Hkv, d = args->d, window = args->window, sinks = args->sinks, io_dtype = args->io_dtype;
  const int64_t q_stride_b = args->q_b, o_stride_b = args->o_b, ck_stride_b = args->ck_b, cv_stride_b = args->cv_b, scales_stride_b = args->sc_b;
  const float scale = args->scale;
  if (!q || !codes_k || !codes_v || !scales || !positions || !out || !(scale > 0.f && scale * 1.44269504088896341f < INFINITY)) return SANA_ERR_ARG;
  const int rc = check_sizes(B, 1, H, Hkv, d, window, sinks, io_dtype);
  if (rc != SANA_OK) return rc;
  for (const int64_t sb : {q_stride_b, o_stride_b, ck_stride_b, cv_stride_b, scales_stride_b})
    if (sb < 0) return SANA_ERR_ARG;
  if (B > 1 && o_stride_b < (int64_t)H * d) return SANA_ERR_ARG;  // (entries that would write the same elements)
  if ((int64_t)window + sinks > (1 << 30) || step_groups(B, H, Hkv) >= Q8_MAX_GROUPS) return SANA_ERR_SHAPE;
  if (misaligned({q, codes_k, codes_v}, {q_stride_b}) || ck_stride_b % 16 || cv_stride_b % 16 || scales_stride_b % 2 ||
      (reinterpret_cast<uintptr_t>(scales) & 7u) || (reinterpret_cast<uintptr_t>(out) & 7u) || o_stride_b % 4 || off4(positions))
    return SANA_ERR_ALIGN;
  Window8Args x = {};
  WindowArgs& a = x.w;
  a.q = static_cast<const uint16_t*>(q), a.out = static_cast<uint16_t*>(out), a.positions = positions;
  a.B = B, a.N = 1, a.Nk = 1, a.H = H, a.Hkv = Hkv, a.d = d, a.window = window, a.sinks = sinks, a.q_b = q_stride_b, a.o_b = o_stride_b;
  a.scale_log2e = scale * 1.44269504088896341f;
  x.ck = args->codes_k, x.cv = args->codes_v, x.scales = scales, x.ck_b = ck_stride_b, x.cv_b = cv_stride_b, x.sc_b = scales_stride_b;
  a.splits = q8_splits(B, H, Hkv, window + sinks, d);
  const int64_t rows = (int64_t)B * H;
  if (a.splits > 1) {
    if (!workspace || args->workspace_bytes < part_bytes(a.splits, rows, d)) return SANA_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SANA_ERR_ALIGN;
    a.part_o = static_cast<float*>(workspace), a.part_ml = a.part_o + a.splits * rows * d;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return io_dtype == SANA_DT_F16 ? q8_of<F16>(x, s) : q8_of<BF16>(x, s);
}

SANA_API int sana_hip_window_cache_read(const sana_cache_read_args* args, void* stream) {
  if (!args) return SANA_ERR_ARG;
  const void *cache_k = args->cache_k, *cache_v = args->cache_v;
  const float* scales = args->scales;
  const int32_t* positions = args->positions;
  void *out_k = args->out_k, *out_v = args->out_v;
  const int B = args->B, Hkv = args->Hkv, d = args->d, window = args->window, sinks = args->sinks, last = args->last, io_dtype = args->io_dtype;
  const int64_t ck_stride_b = args->ck_b, ck_stride_n = args->ck_n, cv_stride_b = args->cv_b, cv_stride_n = args->cv_n, scales_stride_b = args->sc_b;
  const int64_t ok_stride_b = args->ok_b, ok_stride_n = args->ok_n, ov_stride_b = args->ov_b, ov_stride_n = args->ov_n;
  if (!cache_k || !cache_v || !positions || !out_k || !out_v || last < 0 || last > window) return SANA_ERR_ARG;
  // (16-bit rows are copied whole: no head's width)
  const int rc = check_sizes(B, 1, Hkv, Hkv, scales ? d : 8, window, sinks, io_dtype);
  if (rc != SANA_OK) return rc;
  if ((int64_t)sinks + last < 1 || d <= 0) return SANA_ERR_ARG;
  if (d % 8 || (int64_t)Hkv * d > (1 << 22) || (int64_t)window + sinks > (1 << 30)) return SANA_ERR_SHAPE;
  const int64_t width = (int64_t)Hkv * d, held = (int64_t)sinks + last;
  for (const int64_t sb : {ck_stride_b, cv_stride_b, scales_stride_b, ok_stride_b, ov_stride_b})
    if (sb < 0) return SANA_ERR_ARG;
  if (ok_stride_n < width || ov_stride_n < width || (!scales && (ck_stride_n < width || cv_stride_n < width))) return SANA_ERR_ARG;
  if (B > 1 && (ok_stride_b < width || ov_stride_b < width)) return SANA_ERR_ARG;  // (entries that would write the same elements)
  if (misaligned({cache_k, cache_v, out_k, out_v}, {ok_stride_b, ok_stride_n, ov_stride_b, ov_stride_n}) || off4(positions)) return SANA_ERR_ALIGN;
  ReadArgs a = {};
  a.k = static_cast<const unsigned char*>(cache_k), a.v = static_cast<const unsigned char*>(cache_v), a.scales = scales, a.positions = positions;
  a.out_k = static_cast<uint16_t*>(out_k), a.out_v = static_cast<uint16_t*>(out_v);
  a.B = B, a.Hkv = Hkv, a.d = d, a.dp = (d + 15) & ~15, a.window = window, a.sinks = sinks, a.last = last, a.zero_rest = args->zero_rest;
  a.ok_b = ok_stride_b, a.ok_n = ok_stride_n, a.ov_b = ov_stride_b, a.ov_n = ov_stride_n;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!scales) {
    if (misaligned({}, {ck_stride_b, ck_stride_n, cv_stride_b, cv_stride_n})) return SANA_ERR_ALIGN;
    a.k_b = 2 * ck_stride_b, a.k_n = 2 * ck_stride_n, a.v_b = 2 * cv_stride_b, a.v_n = 2 * cv_stride_n;
    if (B * held >= WA_MAX_BLOCKS << 1) return SANA_ERR_SHAPE;
    if (width <= 256 && B <= 65535) {
      a.rows = READ_STEPS * (64 / (int)(width / 8)), a.by_eighths = (65536 + (int)width / 8 - 1) / (int)(width / 8);
      a.items = (held + a.rows - 1) / a.rows * 2;
      hipLaunchKernelGGL(read16_narrow_kernel, dim3((unsigned)((a.items + 3) / 4), (unsigned)B), dim3(256), 0, s, a);
      return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
    }
    a.items = 2 * B * held;
    if ((a.items + 3) / 4 >= WA_MAX_BLOCKS) return SANA_ERR_SHAPE;
    hipLaunchKernelGGL(read16_kernel, dim3((unsigned)((a.items + 3) / 4)), dim3(256), 0, s, a);
  } else {
    if (ck_stride_b % 16 || cv_stride_b % 16 || scales_stride_b % 2 || (reinterpret_cast<uintptr_t>(scales) & 7u)) return SANA_ERR_ALIGN;
    a.k_b = ck_stride_b, a.v_b = cv_stride_b, a.sc_b = scales_stride_b;
    a.rows = READ_STEPS * (64 / (d / 8));
    a.by_eighths = (65536 + d / 8 - 1) / (d / 8);
    a.items = (held + a.rows - 1) / a.rows * 2 * Hkv;
    if (B > 65535 || B * a.items >= WA_MAX_BLOCKS << 2 || (a.items + 3) / 4 >= WA_MAX_BLOCKS) return SANA_ERR_SHAPE;
    const dim3 grid((unsigned)((a.items + 3) / 4), (unsigned)B);
    // Codes beyond the 32 MB of the L2s are read once and past them.  us, written and read back, kept / streamed: 24 MB 26 / 30; 34 MB 47 / 41, 56 MB 40 / 36, 98 MB
    // 116 / 118 (and in front of a chunk's attention 143 / 138).
    const bool nt = 2 * B * held * Hkv * a.dp > (32 << 20);
    if (io_dtype == SANA_DT_F16) nt ? read8<F16, true>(a, grid, s) : read8<F16, false>(a, grid, s);
    else nt ? read8<BF16, true>(a, grid, s) : read8<BF16, false>(a, grid, s);
  }
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}
