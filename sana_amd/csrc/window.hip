// Softmax attention over a sliding window and a few first tokens (sinks), causal, bf16 or f16; key heads may be shared by
// several query heads.  Query at position p sees key j where j <= p and (p - j < window or j < sinks):
//
//   out_p = sum_j softmax_j(scale * q_p . k_j) v_j
//
// in one pass over the keys with a running maximum m and sum l: of a block of scores s (in powers of two, scale * log2(e) inside),
// m' = max(m, max s), p = 2^(s - m'), l' = 2^(m - m') l + sum p, o' = 2^(m - m') o + p v; out = o / l.
// What a stream keeps of its past is a cache of sinks + window rows: row p for a position p below the sinks, then a ring.
// The order of the keys does not matter to the sum, so a token's attention reads the rows as they lie.
#include <initializer_list>

#include "stream_common.h"

namespace sana {
namespace {

constexpr int WK = 64;            // keys of a tile
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

template <typename T> inline constexpr float kShift = is_f16<T> ? 6.f : 0.f;

// A prompt or a chunk: the queries are the last N of Nk keys.  A workgroup takes NW * 16 * QT queries of one head through its
// tiles of 64 keys, the tiles of the sinks first; K and V go to LDS by direct loads, V a tile behind K, one barrier a tile.  scores^T = K Q^T: a
// lane owns a query (its column) and four keys of every 16; the probabilities are fed back from the accumulators, V by transposing reads in
// the order of keys that this gives.  The running maximum moves only when some score is 2^8 above it: until then p <= 2^8 and nothing is
// rescaled (the 16-bit p keeps its relative step, l and o are fp32).  f16: p times 2^6, the small ones away from its subnormal numbers.
// Of a tile of 64 keys x 32 queries x 112 channels the matrix pipe takes 960 cycles, the vector unit some 1000 (half of them powers) and
// the LDS 350 for each of four waves.  The time is the sum of the first two: the matrix pipes work 48 % of it (counters), the two waves of a SIMD, which come
// from workgroups of no relation in phase, do not overlap.  16384 tokens x 20 heads over a window of 4096 run at 0.84 - 0.88 PFLOP/s (633 - 606 us), f16 with
// shared key heads at 0.86 - 0.90.  Through registers instead of direct loads 705 us; each tile's scores in front of its own powers instead of those of the tile
// before: 630 - 690, by how the compiler mixes them; each operand read from LDS where it is used instead of an MFMA group ahead, and the
// maxima in front of the powers instead of beside the values' MFMAs: 653; where in a tile the rest of the vector work stands, wave priorities
// and reads further ahead change it by less than 0.5 %; three or four query tiles a wave: the registers do not hold them.
template <typename T, int DK, int DT, int QT, int NW>
__global__ __launch_bounds__(64 * NW, QT == 1 && DK < 4 ? 3 : 2) void window_attn_kernel(const WindowArgs a) {
  constexpr int PITCH = DK * 64, TILE = WK * PITCH, LOADS = TILE / 1024 / NW, QB = NW * 16 * QT;
  static_assert(TILE % (1024 * NW) == 0 && DT <= 2 * DK, "");
  __shared__ __attribute__((aligned(1024))) unsigned char k_even[TILE], k_odd[TILE], v_even[TILE], v_odd[TILE];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, fr = lane & 15, fg = lane >> 4;

  // The blocks of a head and of those that share its keys on one XCD; the streams, which may be of unlike length, one after the other.
  const int per = (a.items + 7) >> 3, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= a.items) return;
  const int share = a.H / a.Hkv, split = item % a.splits, r1 = item / a.splits, qb = a.qblocks - 1 - r1 % a.qblocks, r2 = r1 / a.qblocks;
  const int r3 = r2 / share, hk = r3 / a.B, b = r3 - hk * a.B, h = hk * share + (r2 - r3 * share), d = a.d;
  const int queries = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;  // that there are
  const int q0 = qb * QB;
  if (q0 >= queries) return;
  const int past = a.Nk - a.N, keys = past + queries;
  const int p0 = past + q0, p1 = past + min(q0 + QB, queries) - 1;  // positions of the block
  const int band = max(p0 - a.window + 1, 0);                       // first key of any window
  // tiles: those of the sinks, then from the band's first on
  const int last_tile = p1 / WK, sink_tiles = min((a.sinks + WK - 1) / WK, last_tile + 1);
  const int band_tile = max(band / WK, sink_tiles), tiles = sink_tiles + max(last_tile + 1 - band_tile, 0);
  const int t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);

  // ---- queries: column operand, lane -> query fr, k = 32 s + 8 fg .. + 7
  const int w0 = q0 + 16 * QT * wave;  // this wave's first query
  u32x4_t qf[QT][DK];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint16_t* row = a.q + b * a.q_b + (int64_t)min(w0 + 16 * t + fr, queries - 1) * a.q_n + h * d;
#pragma unroll
    for (int s = 0; s < DK; ++s) {
      qf[t][s] = *reinterpret_cast<const u32x4_t*>(row + (32 * s + 8 * fg < d ? 32 * s + 8 * fg : 0));
      if (32 * s + 8 * fg >= d) qf[t][s] = u32x4_t{0u, 0u, 0u, 0u};
    }
  }
  const int wp0 = past + w0, wp1 = min(wp0 + 16 * QT - 1, p1);

  // K and V of a tile by direct loads to LDS, 1 KB each, arrays of their own, by which the compiler sees that no read waits for another tile:
  // a lane's 16 bytes are at the place that its number gives, so it fetches the piece that the row's exchange puts there.  Outside of the rows: zeros.  (63 rows are less than 2^31 bytes: nothing comes back in.)
  const uint16_t *kp = a.k + b * a.k_b + hk * d, *vp = a.v + b * a.v_b + hk * d;
  const uint32_t k2 = 2 * (uint32_t)a.k_n, v2 = 2 * (uint32_t)a.v_n;
  auto tile_of = [&](int t) { return t < sink_tiles ? t : band_tile + (t - sink_tiles); };
  auto request = [&](const uint16_t* rows, int64_t stride, uint32_t ld2, int t, unsigned char* to) {
    const int j0 = tile_of(t) * WK, count = min(keys - j0, WK);
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(rows + (int64_t)j0 * stride), 0, (int)((uint32_t)(count - 1) * ld2 + 2 * d), 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = 64 * (NW * i + wave) + lane, row = at / (4 * DK), c = (at - row * (4 * DK)) ^ row_key<DK>(row);
      const uint32_t off = 8 * c < d ? (uint32_t)row * ld2 + 16 * c : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_t*)(to + 1024 * (NW * i + wave)), 16, (int)off, 0, 0, 0);
    }
  };
  auto landed = [&]() {  // this wave's loads have, and everyone's behind the barrier
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), as a builtin: the compiler counts on it and waits for no tile a second time
    lds_barrier();
  };

  const int key = row_key<DK>(fr), trow = 4 * fg + (fr >> 2), tkey = row_key<DK>(trow), piece = fr & 3;
  uint32_t k_at[DK];
#pragma unroll
  for (int s = 0; s < DK; ++s) k_at[s] = fr * PITCH + (((4 * s + fg) ^ key) << 4);
  uint32_t v_slot = ((piece >> 1) ^ tkey) << 4;
  const uint32_t v_row = trow * PITCH + 8 * (piece & 1);
  auto v_at = [&](int dt) { return v_row + (v_slot ^ (dt << 5)); };  // slot (2 dt + (piece >> 1)) ^ tkey

  f32x4_t oc[QT][DT];  // out^T: channel 16 dt + 4 fg + r, query fr
  float mx[QT], sub[QT], sum[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    mx[t] = -INFINITY, sub[t] = 0.f, sum[t] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oc[t][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto whole = [&](int t) {  // whether this wave's queries see all keys of a tile (uniform)
    const int j0 = tile_of(t) * WK, j1 = j0 + WK - 1;
    return j1 <= wp0 && (j1 < a.sinks || wp1 - j0 < a.window);
  };
  // Scores of KP tiles of 16 keys at a time: one where two query tiles take turns, two otherwise (an MFMA that adds to what the one before
  // it has just summed waits for twice its own time).  Values are read AHEAD products in front of their own.
  constexpr int KP = QT == 1 ? 2 : 1, AHEAD = 2;
  auto keys_of = [&](const unsigned char* from, int k0, u32x4_t (&kf)[KP][DK]) {
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int s = 0; s < DK; ++s) kf[j][s] = lds_read((const lds_t*)from + 16 * (k0 + j) * PITCH + k_at[s]);
  };
  auto score = [&](const u32x4_t (&kf)[KP][DK], int k0, f32x4_t (&sc)[QT][4]) {
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int q = 0; q < QT; ++q) sc[q][k0 + j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DK; ++s)
#pragma unroll
      for (int j = 0; j < KP; ++j)
#pragma unroll
        for (int q = 0; q < QT; ++q) sc[q][k0 + j] = mfma_16x16x32<T>(kf[j][s], qf[q][s], sc[q][k0 + j]);
  };
  auto mask = [&](int t, f32x4_t (&sc)[QT][4]) {
    const int lane_key = tile_of(t) * WK + 4 * fg, to_sinks = a.sinks - lane_key;  // c = 16 kt + r is key lane_key + c
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      const int to_query = past + w0 + 16 * q + fr - lane_key, to_window = to_query - a.window;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int c = 16 * kt + r;
          if ((c > to_query) | ((c <= to_window) & (c >= to_sinks))) sc[q][kt][r] = -INFINITY;
        }
    }
  };
  float top[QT];  // of the tile whose scores are there, this lane's keys
  auto highest = [&](int q, int kt, const f32x4_t (&sc)[QT][4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) top[q] = fmaxf(kt + r == 0 ? -INFINITY : top[q], sc[q][kt][r]);
  };
  auto maxima = [&]() {
    // (the scale is positive: the maximum of the scaled scores is the scaled maximum)
    float most[QT];
    bool above = false;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      most[q] = top[q] * a.scale_log2e;
      above |= most[q] > mx[q] + 8.f;
    }
    if (__any(above)) {
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const float now = fmaxf(mx[q], max_groups(most[q]));
        const float f = __builtin_amdgcn_exp2f(mx[q] - (now == -INFINITY ? 0.f : now));  // (nothing yet: 0)
        mx[q] = now, sub[q] = now == -INFINITY ? 0.f : now - kShift<T>;
        sum[q] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) oc[q][dt][r] *= f;
      }
    }
  };
  auto powers = [&](int q, int kt, const f32x4_t (&sc)[QT][4], u32x2_t (&pk)[QT][4]) {
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(sc[q][kt][r], a.scale_log2e, -sub[q]));
      sum[q] += p[r];
    }
    pk[q][kt] = u32x2_t{pk16<T>(p[0], p[1]), pk16<T>(p[2], p[3])};
  };
  auto values_of = [&](unsigned char* from, int i) {  // 32 keys i / DT of 16 channels i % DT
    lds_t* at = (lds_t*)from + v_at(i % DT) + 32 * (i / DT) * PITCH;
    const u32x2_t x = lds_read_tr(at), y = lds_read_tr(at + 16 * PITCH);
    return u32x4_t{x.x, x.y, y.x, y.y};
  };
  // Tile t: its softmax and its product with V, and the scores of the tile behind it, whose MFMAs the vector work need not wait for.
  // A buffer is written again two barriers after its last read.  No branch decides whether a tile is worked on: what a wave does not see is
  // masked (one tile or two a block), and behind the last tile the scores of whatever lies there are not used.
  auto step = [&](int t, f32x4_t (&sc)[QT][4], f32x4_t (&next)[QT][4], unsigned char* k_here, unsigned char* k_next, unsigned char* v_here,
                  unsigned char* v_next) {
    landed();  // K of t + 1, V of t
    if (t + 2 < t1) request(kp, a.k_n, k2, t + 2, k_here);
    if (t + 1 < t1) request(vp, a.v_n, v2, t + 1, v_next);
    u32x4_t kf[2][KP][DK], vf[AHEAD + 1];
    keys_of(k_next, 0, kf[0]);
    __builtin_amdgcn_sched_barrier(0);
    if (!whole(t)) {
      mask(t, sc);
#pragma unroll
      for (int u = 0; u < 4 * QT; ++u) highest(u % QT, u / QT, sc);
    }
    maxima();
    asm volatile("" : "+v"(v_slot));  // (addresses are worked out here again: kept, they would take the registers of the tiles)
    // 16 or 32 keys of the next tile at a time, and the powers of half of the keys between their MFMAs
    u32x2_t pk[QT][4];
#pragma unroll
    for (int kt = 0; kt < 4; kt += KP) {
      __builtin_amdgcn_sched_barrier(0);
      if (kt + KP < 4) keys_of(k_next, kt + KP, kf[(kt / KP + 1) & 1]);
      else
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) vf[i] = values_of(v_here, i);
      __builtin_amdgcn_sched_barrier(0);
      score(kf[(kt / KP) & 1], kt, next);
#pragma unroll
      for (int u = kt * QT / 2; u < (kt + KP) * QT / 2; ++u) powers(u % QT, u / QT, sc, pk);
    }
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + AHEAD < 2 * DT) vf[(i + AHEAD) % (AHEAD + 1)] = values_of(v_here, i + AHEAD);
      const int s = i / DT, dt = i % DT;
#pragma unroll
      for (int q = 0; q < QT; ++q)
        oc[q][dt] = mfma_16x16x32<T>(vf[i % (AHEAD + 1)], u32x4_t{pk[q][2 * s].x, pk[q][2 * s].y, pk[q][2 * s + 1].x, pk[q][2 * s + 1].y}, oc[q][dt]);
#pragma unroll
      for (int u = 0; u < 2 * QT; ++u)
        if (i == u * DT / (2 * QT)) powers(u % QT, 2 + u / QT, sc, pk);
#pragma unroll
      for (int u = 0; u < 4 * QT; ++u)
        if (i == DT + u * DT / (4 * QT)) highest(u % QT, u / QT, next);
    }
  };
  if (t0 < t1) {
    f32x4_t even[QT][4], odd[QT][4];
    request(kp, a.k_n, k2, t0, k_even);
    request(vp, a.v_n, v2, t0, v_even);
    if (t0 + 1 < t1) request(kp, a.k_n, k2, t0 + 1, k_odd);
    landed();
#pragma unroll
    for (int kt = 0; kt < 4; kt += KP) {
      u32x4_t kf[KP][DK];
      keys_of(k_even, kt, kf);
      score(kf, kt, even);
#pragma unroll
      for (int u = kt * QT; u < (kt + KP) * QT; ++u) highest(u % QT, u / QT, even);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll 1
    for (int t = t0; t < t1; t += 2) {
      step(t, even, odd, k_even, k_odd, v_even, v_odd);
      if (t + 1 < t1) step(t + 1, odd, even, k_odd, k_even, v_odd, v_even);
    }
  }
  // ---- Values that are not finite: the products with V once more, so that they reach the queries that see them and no others.  32 keys at a
  // time straight from memory, the finite values; the others counted, and their signs summed, over the keys that are seen.  (All blocks of 16384
  // tokens with a window of 4096: 5.9 ms where finite values take 0.65 - 0.78.)
  bool odd = false;
#pragma unroll
  for (int q = 0; q < QT; ++q)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= !(fabsf(oc[q][dt][r]) < INFINITY);
  if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) oc[q][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int half = 2 * t0; half < 2 * t1; ++half) {
      const int j0 = tile_of(half >> 1) * WK + 32 * (half & 1);
      u32x4_t p[QT], seen[QT];
#pragma unroll
      for (int q = 0; q < QT; ++q) p[q] = seen[q] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        f32x4_t sc[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) sc[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < DK; ++s) {
          const int c = 32 * s + 8 * fg;
          u32x4_t kf = *reinterpret_cast<const u32x4_t*>(kp + (int64_t)min(j0 + 16 * kt + fr, keys - 1) * a.k_n + (c < d ? c : 0));
          if (c >= d) kf = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
          for (int q = 0; q < QT; ++q) sc[q] = mfma_16x16x32<T>(kf, qf[q][s], sc[q]);
        }
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = j0 + 16 * kt + 4 * fg + r, i = past + w0 + 16 * q + fr;
            if (j > i || (i - j >= a.window && j >= a.sinks)) continue;
            const float x = __builtin_amdgcn_exp2f(fmaf(sc[q][r], a.scale_log2e, -sub[q]));
            p[q][2 * kt + (r >> 1)] |= (pk16<T>(x, 0.f) & 0xffffu) << (16 * (r & 1)), seen[q][2 * kt + (r >> 1)] |= kOne16<T> << (16 * (r & 1));
          }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        u32x4_t finite = {0u, 0u, 0u, 0u}, other = finite, sign = finite;
        const int c = 16 * dt + fr;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = j0 + 16 * (e >> 2) + 4 * fg + (e & 3), at = 16 * (e & 1);
          const uint32_t x = c < d && j < keys ? vp[(int64_t)j * a.v_n + c] : 0u, m = x & 0x7fffu;
          finite[e >> 1] |= (m < kInf16<T> ? x : 0u) << at, other[e >> 1] |= (m < kInf16<T> ? 0u : kOne16<T>) << at;
          sign[e >> 1] |= (m == kInf16<T> ? kOne16<T> | (x & 0x8000u) : 0u) << at;
        }
#pragma unroll
        for (int q = 0; q < QT; ++q) {
          oc[q][dt] = mfma_16x16x32<T>(finite, p[q], oc[q][dt]);
          const f32x4_t zero = {0.f, 0.f, 0.f, 0.f}, n = mfma_16x16x32<T>(other, seen[q], zero), to = mfma_16x16x32<T>(sign, seen[q], zero);
#pragma unroll
          for (int r = 0; r < 4; ++r) oc[q][dt][r] += n[r] == 0.f ? 0.f : to[r] == n[r] ? INFINITY : to[r] == -n[r] ? -INFINITY : NAN;
        }
      }
    }
  }
  // ---- out, or this part's
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int qi = w0 + 16 * t + fr;
    const float l = sum_groups(sum[t]);
    if (qi >= queries) continue;
    if (a.splits == 1) {
      const float inv = 1.0f / l;
      uint16_t* row = a.out + b * a.o_b + (int64_t)qi * a.o_n + h * d;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int c = 16 * dt + 4 * fg;
        if (c < d) *reinterpret_cast<u32x2_t*>(row + c) = u32x2_t{pk16<T>(oc[t][dt][0] * inv, oc[t][dt][1] * inv), pk16<T>(oc[t][dt][2] * inv, oc[t][dt][3] * inv)};
      }
    } else {
      const int64_t at = ((int64_t)split * a.B * a.N + (int64_t)b * a.N + qi) * a.H + h;
      if (fg == 0) a.part_ml[2 * at] = mx[t], a.part_ml[2 * at + 1] = l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int c = 16 * dt + 4 * fg;
        if (c < d) *reinterpret_cast<f32x4_t*>(a.part_o + at * d + c) = oc[t][dt];
      }
    }
  }
}

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

// One token of each stream over its cache.  A workgroup takes a part of the rows of one (stream, key head), its NW waves in turn a
// tile of 32 rows; the query heads that share the key head are the 16 columns of the products (more than 16 in further workgroups).  K comes
// from memory as the operand it is, V through the wave's own LDS to be transposed.  The new token's row is taken from k and v, wherever its
// slot is met, and written to the cache by the workgroup whose part holds the slot: nobody reads that row of the cache.
// Every compute unit busy, memory bounds it: 64 streams x 8192 rows x 8 key heads of 128, 2.0 GB 358 us = 5.7 TB/s, more than a copy reaches (it only
// reads).  With fewer workgroups than that, what one compute unit takes in: 16 key heads of 72 x 1028 rows 296 KB each, 12.4 us, some 30 bytes
// a ns; twelve or sixteen waves in the place of eight (13.9, 17.4 us) and more tiles requested ahead do not change that, more parts do.
template <typename T, int DK, int DT, int NW>
__global__ __launch_bounds__(64 * NW) void window_step_kernel(const WindowArgs a) {
  constexpr int PITCH = DK * 64, TILE = 32 * PITCH, PV = DK * 2;  // PV: 16-byte pieces of V a lane
  __shared__ __attribute__((aligned(16))) unsigned char smem[NW * (TILE > 16 * 16 * DT * 4 + 128 ? TILE : 16 * 16 * DT * 4 + 128)];
  constexpr int OWN = sizeof(smem) / NW;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, fr = lane & 15, fg = lane >> 4;
  unsigned char* mine = smem + wave * OWN;
  const int G = a.H / a.Hkv, blocks = (G + 15) / 16, d = a.d;
  const int split = blockIdx.y, gb = blockIdx.x % blocks, bk = blockIdx.x / blocks, b = bk / a.Hkv, hk = bk - b * a.Hkv;
  const int pos = a.positions[b];
  if (pos < 0) {  // an idle stream: zeros
    if (split == 0 && gb == 0)
      for (int c = tid; c < G * d; c += 64 * NW) a.out[b * a.o_b + hk * G * d + c] = 0;
    return;
  }
  const int rows = a.window + a.sinks, count = pos < rows ? pos + 1 : rows, slot = wa_slot(pos, a.sinks, a.window);
  const int tiles = (count + 31) / 32, t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);

  const int head = 16 * gb + fr, h = hk * G + min(head, G - 1);
  u32x4_t qf[DK];
#pragma unroll
  for (int s = 0; s < DK; ++s) {
    qf[s] = *reinterpret_cast<const u32x4_t*>(a.q + b * a.q_b + h * d + (32 * s + 8 * fg < d ? 32 * s + 8 * fg : 0));
    if (32 * s + 8 * fg >= d) qf[s] = u32x4_t{0u, 0u, 0u, 0u};
  }
  const uint16_t *new_k = a.k + b * a.k_b + hk * d, *new_v = a.v + b * a.v_b + hk * d;
  uint16_t *ck = a.cache_k + b * a.ck_b + hk * d, *cv = a.cache_v + b * a.cv_b + hk * d;
  if (gb == 0 && slot / 32 >= t0 && slot / 32 < t1 && tid < 32 * DK / 4) {  // (t0 <= slot's tile < t1 holds for one part)
    const int c = 8 * (tid % (4 * DK));
    if (c < d) {
      const bool of_v = tid >= 4 * DK;
      *reinterpret_cast<u32x4_t*>((of_v ? cv + (int64_t)slot * a.cv_n : ck + (int64_t)slot * a.ck_n) + c) =
          *reinterpret_cast<const u32x4_t*>((of_v ? new_v : new_k) + c);
    }
  }

  u32x4_t rk[2][DK], rv[PV];
  auto request = [&](int t) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int row = min(32 * t + 16 * kt + fr, count - 1);
      const uint16_t* from = row == slot ? new_k : ck + (int64_t)row * a.ck_n;
#pragma unroll
      for (int s = 0; s < DK; ++s) rk[kt][s] = *reinterpret_cast<const u32x4_t*>(from + (32 * s + 8 * fg < d ? 32 * s + 8 * fg : 0));
    }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const int idx = lane + 64 * i, r = idx / (DK * 4), c = idx - r * (DK * 4), row = min(32 * t + r, count - 1);
      const uint16_t* from = row == slot ? new_v : cv + (int64_t)row * a.cv_n;
      rv[i] = *reinterpret_cast<const u32x4_t*>(from + (8 * c < d ? 8 * c : 0));
    }
  };
  f32x4_t oc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float mx = -INFINITY, sub = 0.f, sum = 0.f;
  const int trow = 4 * fg + (fr >> 2), tkey = row_key<DK>(trow), piece = fr & 3;
  if (t0 + wave < t1) request(t0 + wave);
#pragma unroll 1
  for (int t = t0 + wave; t < t1; t += NW) {
    f32x4_t sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < DK; ++s)  // (channels past d: K repeats others there, q is zero; an inf there must not count)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        u32x4_t kf = rk[kt][s];
        if (32 * s + 8 * fg >= d) kf = u32x4_t{0u, 0u, 0u, 0u};
        sc[kt] = mfma_16x16x32<T>(kf, qf[s], sc[kt]);
      }
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const int idx = lane + 64 * i, r = idx / (DK * 4), c = idx - r * (DK * 4);
      *reinterpret_cast<u32x4_t*>(mine + r * PITCH + ((c ^ row_key<DK>(r)) << 4)) = 32 * t + r < count ? rv[i] : u32x4_t{0u, 0u, 0u, 0u};
    }
    if (t + NW < t1) request(t + NW);
    float most = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[kt][r] = 32 * t + 16 * kt + 4 * fg + r < count ? sc[kt][r] * a.scale_log2e : -INFINITY;
        most = fmaxf(most, sc[kt][r]);
      }
    if (__any(most > mx + 8.f)) {
      const float now = fmaxf(mx, max_groups(most));
      const float f = __builtin_amdgcn_exp2f(mx - (now == -INFINITY ? 0.f : now));
      mx = now, sub = now == -INFINITY ? 0.f : now - kShift<T>;
      sum *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) oc[dt][r] *= f;
    }
    u32x4_t pf;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = __builtin_amdgcn_exp2f(sc[kt][r] - sub);
        sum += p[r];
      }
      pf[2 * kt] = pk16<T>(p[0], p[1]), pf[2 * kt + 1] = pk16<T>(p[2], p[3]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the wave's own V is there)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      lds_t* from = (lds_t*)mine + trow * PITCH + (((2 * dt + (piece >> 1)) ^ tkey) << 4) + 8 * (piece & 1);
      const u32x2_t x = lds_read_tr(from), y = lds_read_tr(from + 16 * PITCH);
      oc[dt] = mfma_16x16x32<T>(u32x4_t{x.x, x.y, y.x, y.y}, pf, oc[dt]);
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
  for (int c = tid >> 4; c < d; c += 4 * NW) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) o = fmaf(f[w], part(w)[c * 16 + col], o);
    if (a.splits == 1) a.out[b * a.o_b + (hk * G + g) * d + c] = (uint16_t)pk16<T>(o * inv, 0.f);
    else a.part_o[at * d + c] = o;
  }
  if (a.splits > 1 && tid < 16) a.part_ml[2 * at] = m, a.part_ml[2 * at + 1] = l;
}

// New tokens into the caches, 16 bytes a thread; a token that later ones of the same call push out is not written, so no row is
// written twice.  Memory bounds it: 168 MB 33 us = 5.1 TB/s, a copy's rate.
__global__ __launch_bounds__(256) void window_append_kernel(const WindowArgs a) {
  const int width = a.d / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.N * width) return;
  const int t = (int)(i / width), c = 8 * (int)(i - (int64_t)t * width), b = blockIdx.y;
  const int n = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
  const int64_t pos = a.positions[b], p = pos + t;
  if (pos < 0 || t >= n || (p >= a.sinks && t < n - a.window)) return;
  const int slot = wa_slot(p, a.sinks, a.window);
  *reinterpret_cast<u32x4_t*>(a.cache_k + b * a.ck_b + (int64_t)slot * a.ck_n + c) =
      *reinterpret_cast<const u32x4_t*>(a.k + b * a.k_b + (int64_t)t * a.k_n + c);
  *reinterpret_cast<u32x4_t*>(a.cache_v + b * a.cv_b + (int64_t)slot * a.cv_n + c) =
      *reinterpret_cast<const u32x4_t*>(a.v + b * a.v_b + (int64_t)t * a.v_n + c);
}

constexpr int WA_NW = 4;
constexpr int64_t WA_MAX_BLOCKS = 1 << 24;  // of 256 threads: a launch has fewer than 2^32 threads an axis
// What the rules below take without leaving 64 bits, and what a launch could take at most: a block for each (batch entry, head).
bool prompt_fits(int B, int N, int Nk, int H, int d) {
  return Nk <= (1 << 30) && N <= Nk && d <= 128 && (int64_t)B * H <= WA_MAX_BLOCKS - 8;
}
// 16-query tiles of a wave, 64 or 128 queries a workgroup.  Two feed twice the MFMAs with a read of K or V and pay where heads are wide
// and the blocks many; one gives more and shorter workgroups, and up to 96 channels three and more waves a SIMD.  us, two / one, window 4096:
// 20 heads of 112 1500 tokens 38 / 30, 2000 59 / 48, 2560 66 / 66, 3000 70 / 88, 8000 294 / 351; 16 of 128 3000 70 / 60, 4680 123 / 122, 8000 231 / 261;
// window 256: 20 of 112 16384 136 / 143.  Narrower heads have one: 70 of 32 3000 108 / 94, 8000 388 / 400; 35 of 64 3000 89 / 74, 8000 312 / 305,
// 16384 657 / 676; 16 of 72 3000 55 / 51, 8000 175 / 185; 12 of 96 4680 99 / 86, 8000 182 / 184; window 256: 70 of 32 8000 91 / 81, 35 of 64 8000
// 74 / 60, 16 of 72 8000 42 / 38, 12 of 96 8000 39 / 31.  (From 72 channels on, long prompts over a long window would be faster by two, which are not
// built for them: 2 x 16384 of 16 of 72 732 / 872, 16384 of 12 of 96 316 / 373, 8000 of 20 of 80 232 / 261.)
int query_tiles(int B, int N, int H, int d) { return d <= 96 || (int64_t)B * H * ((N + 127) / 128) <= 400 ? 1 : 2; }
// Parts of a prompt's keys: where the blocks of queries leave compute units idle and have tiles of keys enough to pay for a second launch
// (600 tokens, 20 heads of 112, ten tiles: whole 13.9 us, in two parts over 20; 128 of 1128 keys 22.7 / 17.0 (four parts), 300 of 4300 67 / 32 (five), 1 of
// 4096 62 / 16 (sixteen), 64 of 764, four streams of 16 heads of 128 17 / 17; two tiles a part are no faster than four).
int prompt_splits(int B, int N, int Nk, int H, int d, int window, int sinks) {
  const int qb = WA_NW * 16 * query_tiles(B, N, H, d);
  const int64_t blocks = (int64_t)B * H * ((N + qb - 1) / qb);
  const int64_t seen = (int64_t)window + qb + sinks;
  const int tiles = (int)((seen < Nk ? seen : Nk) / WK);
  if (blocks >= 256 || tiles < 16) return 1;
  int64_t want = 512 / blocks;
  want = want > tiles / 4 ? tiles / 4 : want;
  return (int)(want < 1 ? 1 : want > WA_MAX_SPLITS ? WA_MAX_SPLITS : want);
}
// One token: the workgroups of a whole cache, one a (stream, key head, 16 query heads).
int64_t step_groups(int B, int H, int Hkv) { return (int64_t)B * Hkv * ((H / Hkv + 15) / 16); }
// Parts of a cache's rows.  A short cache is taken whole: a second launch that joins parts takes 3.4 us, and 3.6 of the host's where calls are issued
// one by one.  us on the device, whole / best of 2 to 32 parts: 20 key heads of 112 x 260 rows 8.4 / 8.8, 516 11.6 / 10.1, 1028 16.3 / 12.3; 8 of 128
// x 260 7.7 / 8.8, 1028 14 / 9.3; 80 of 112 x 516 12 / 14; 70 of 32 x 1028 8.0 / 10.8; where there are more, longer ones too: 160 of 112 x 1028
// 27 / 29, 140 of 32 x 4100 27 / 29.  Otherwise the least number with which the last round of compute units is not mostly idle: 20 of 112 x
// 4100 47 / 18 (10 parts), 120 of 112 x 4100 79 / 57 (2), 200 90 / 88, 260 167 / 112 (12; 4: 122), 512 of 128 x 8192 366 / 380 (2).
// (Two tiles of a wave requested ahead in the place of one make a whole cache slower: 20 of 112 x 1028 16.3 / 19.9.)
int step_splits(int B, int H, int Hkv, int rows, int d) {
  const int64_t groups = step_groups(B, H, Hkv), bytes = (int64_t)rows * d * 4;
  if (bytes <= (groups <= 128 ? 384 << 10 : 1 << 20)) return 1;
  const int most = rows / 64 < WA_MAX_SPLITS ? rows / 64 : WA_MAX_SPLITS;
  for (int s = 1; s < most; ++s)
    if (groups * s * 32 >= (groups * s + 255) / 256 * 256 * 25) return s;
  return most > 1 ? most : 1;
}
size_t part_bytes(int splits, int64_t rows, int d) { return splits > 1 ? (size_t)splits * rows * (d + 2) * sizeof(float) : 0; }

template <typename T>
int launch_join(const WindowArgs& a, hipStream_t s) {
  const int64_t groups = ((int64_t)a.B * a.N * a.H + 7) / 8;
  if (groups >= WA_MAX_BLOCKS) return SANA_ERR_SHAPE;
  hipLaunchKernelGGL(window_join_kernel<T>, dim3((unsigned)groups), dim3(256), 0, s, a);
  return SANA_OK;
}

template <typename T, int DK, int DT>
int launch_prompt(WindowArgs a, hipStream_t s) {
  const bool one = DK < 4 || query_tiles(a.B, a.N, a.H, a.d) == 1;
  const int qb = WA_NW * 16 * (one ? 1 : 2);
  a.qblocks = (a.N + qb - 1) / qb;
  const int64_t items = (int64_t)a.B * a.H * a.qblocks * a.splits;
  if (items > WA_MAX_BLOCKS - 8) return SANA_ERR_SHAPE;
  a.items = (int)items;
  const dim3 grid((unsigned)((items + 7) / 8 * 8)), block(64 * WA_NW);
  if (one) hipLaunchKernelGGL((window_attn_kernel<T, DK, DT, 1, WA_NW>), grid, block, 0, s, a);
  else if constexpr (DK == 4) hipLaunchKernelGGL((window_attn_kernel<T, DK, DT, 2, WA_NW>), grid, block, 0, s, a);
  if (a.splits > 1) {
    const int rc = launch_join<T>(a, s);
    if (rc != SANA_OK) return rc;
  }
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}

template <typename T, int DK, int DT>
int launch_step(const WindowArgs& a, hipStream_t s) {
  const int64_t groups = step_groups(a.B, a.H, a.Hkv);
  // (eight waves where a cache is not split and the chip has room for them: 20 key heads of 112 x 772 rows 13.7 us, four 15.3; 320 x 516 29.8 / 28.3)
  if (a.splits == 1 && groups <= 256)
    hipLaunchKernelGGL((window_step_kernel<T, DK, DT, 8>), dim3((unsigned)groups), dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((window_step_kernel<T, DK, DT, 4>), dim3((unsigned)groups, (unsigned)a.splits), dim3(256), 0, s, a);
  if (a.splits > 1) {
    const int rc = launch_join<T>(a, s);
    if (rc != SANA_OK) return rc;
  }
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}

// head dims in classes: 32-channel steps of the scores, 16-channel tiles of the values
#define SANA_WA_DIMS(F, ...)                     \
  (a.d <= 32   ? F<T, 1, 2>(__VA_ARGS__)         \
   : a.d <= 64 ? F<T, 2, 4>(__VA_ARGS__)         \
   : a.d <= 80 ? F<T, 3, 5>(__VA_ARGS__)         \
   : a.d <= 96 ? F<T, 3, 6>(__VA_ARGS__)         \
   : a.d <= 112 ? F<T, 4, 7>(__VA_ARGS__)        \
                : F<T, 4, 8>(__VA_ARGS__))
template <typename T>
int prompt_of(const WindowArgs& a, hipStream_t s) { return SANA_WA_DIMS(launch_prompt, a, s); }
template <typename T>
int step_of(const WindowArgs& a, hipStream_t s) { return SANA_WA_DIMS(launch_step, a, s); }

bool misaligned(std::initializer_list<const void*> rows, std::initializer_list<int64_t> strides) {
  for (const void* p : rows)
    if (!aligned16(p)) return true;
  for (const int64_t s : strides)
    if (s % 8) return true;
  return false;
}
bool off4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }

// sizes that all three calls share
int check_sizes(int B, int N, int H, int Hkv, int d, int window, int sinks, int io_dtype) {
  if (B <= 0 || N <= 0 || H <= 0 || Hkv <= 0 || d <= 0 || window <= 0 || sinks < 0 || H % Hkv) return SANA_ERR_ARG;
  if (io_dtype != SANA_DT_BF16 && io_dtype != SANA_DT_F16) return SANA_ERR_DTYPE;
  if (d % 8 || d > 128 || N > (1 << 30) || window > (1 << 30) || sinks > (1 << 30) || (int64_t)H * d > (1 << 22)) return SANA_ERR_SHAPE;
  return SANA_OK;
}

}  // namespace
}  // namespace sana

using namespace sana;

#define SANA_API extern "C" __attribute__((visibility("default")))

SANA_API size_t sana_hip_window_attention_workspace_bytes(int B, int N, int Nk, int H, int d, int window, int sinks) {
  if (B <= 0 || N <= 0 || H <= 0 || d <= 0 || window <= 0 || sinks < 0 || !prompt_fits(B, N, Nk, H, d)) return 0;
  return part_bytes(prompt_splits(B, N, Nk, H, d, window, sinks), (int64_t)B * N * H, d);
}

SANA_API int sana_hip_window_attention_query_tiles(int B, int N, int H, int d) {
  return B <= 0 || N <= 0 || H <= 0 || d <= 0 || !prompt_fits(B, N, N, H, d) ? 0 : query_tiles(B, N, H, d);
}

SANA_API int sana_hip_window_attention(const void* q, const void* k, const void* v, void* out, const int32_t* lengths, void* workspace,
                                       size_t workspace_bytes, int B, int N, int Nk, int H, int Hkv, int d, int window, int sinks,
                                       int64_t q_stride_b, int64_t q_stride_n, int64_t k_stride_b, int64_t k_stride_n,
                                       int64_t v_stride_b, int64_t v_stride_n, int64_t o_stride_b, int64_t o_stride_n, float scale,
                                       int io_dtype, void* stream) {
  if (!q || !k || !v || !out || Nk < N || !(scale > 0.f && scale * 1.44269504088896341f < INFINITY)) return SANA_ERR_ARG;
  const int rc = check_sizes(B, N, H, Hkv, d, window, sinks, io_dtype);
  if (rc != SANA_OK) return rc;
  if (!prompt_fits(B, N, Nk, H, d)) return SANA_ERR_SHAPE;
  if (q_stride_n < (int64_t)H * d || o_stride_n < (int64_t)H * d || k_stride_n < (int64_t)Hkv * d || v_stride_n < (int64_t)Hkv * d)
    return SANA_ERR_ARG;
  for (const int64_t sb : {q_stride_b, k_stride_b, v_stride_b, o_stride_b})
    if (sb < 0) return SANA_ERR_ARG;
  if (B > 1 && o_stride_b < (int64_t)H * d) return SANA_ERR_ARG;  // (entries that would write the same elements)
  if (k_stride_n >= (1 << 23) || v_stride_n >= (1 << 23)) return SANA_ERR_SHAPE;  // 32-bit byte offsets within a tile
  if (misaligned({q, k, v}, {q_stride_b, q_stride_n, k_stride_b, k_stride_n, v_stride_b, v_stride_n}) ||
      (reinterpret_cast<uintptr_t>(out) & 7u) || o_stride_b % 4 || o_stride_n % 4 || off4(lengths))
    return SANA_ERR_ALIGN;
  WindowArgs a = {};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out), a.lengths = lengths;
  a.B = B, a.N = N, a.Nk = Nk, a.H = H, a.Hkv = Hkv, a.d = d, a.window = window, a.sinks = sinks;
  a.q_b = q_stride_b, a.q_n = q_stride_n, a.k_b = k_stride_b, a.k_n = k_stride_n, a.v_b = v_stride_b, a.v_n = v_stride_n;
  a.o_b = o_stride_b, a.o_n = o_stride_n, a.scale_log2e = scale * 1.44269504088896341f;
  a.splits = prompt_splits(B, N, Nk, H, d, window, sinks);
  const int64_t rows = (int64_t)B * N * H;
  if (a.splits > 1) {
    if (!workspace || workspace_bytes < part_bytes(a.splits, rows, d)) return SANA_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SANA_ERR_ALIGN;
    a.part_o = static_cast<float*>(workspace), a.part_ml = a.part_o + a.splits * rows * d;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return io_dtype == SANA_DT_F16 ? prompt_of<F16>(a, s) : prompt_of<BF16>(a, s);
}

SANA_API int sana_hip_window_cache_append(void* cache_k, void* cache_v, const void* k, const void* v, const int32_t* positions,
                                          const int32_t* lengths, int B, int N, int C, int window, int sinks,
                                          int64_t ck_stride_b, int64_t ck_stride_n, int64_t cv_stride_b, int64_t cv_stride_n,
                                          int64_t k_stride_b, int64_t k_stride_n, int64_t v_stride_b, int64_t v_stride_n,
                                          int io_dtype, void* stream) {
  if (!cache_k || !cache_v || !k || !v || !positions) return SANA_ERR_ARG;
  const int rc = check_sizes(B, N, 1, 1, 8, window, sinks, io_dtype);
  if (rc != SANA_OK) return rc;
  if (C <= 0) return SANA_ERR_ARG;
  const int64_t groups = ((int64_t)N * (C / 8) + 255) / 256;
  if (ck_stride_n < C || cv_stride_n < C || k_stride_n < C || v_stride_n < C) return SANA_ERR_ARG;
  for (const int64_t sb : {ck_stride_b, cv_stride_b, k_stride_b, v_stride_b})
    if (sb < 0) return SANA_ERR_ARG;
  if (B > 1 && (ck_stride_b < C || cv_stride_b < C)) return SANA_ERR_ARG;  // (streams that would write the same elements)
  if ((int64_t)window + sinks > (1 << 30)) return SANA_ERR_SHAPE;
  if (C % 8 || groups >= WA_MAX_BLOCKS || B > 65535) return SANA_ERR_SHAPE;
  if (misaligned({cache_k, cache_v, k, v}, {ck_stride_b, ck_stride_n, cv_stride_b, cv_stride_n, k_stride_b, k_stride_n, v_stride_b, v_stride_n}) ||
      off4(positions) || off4(lengths))
    return SANA_ERR_ALIGN;
  WindowArgs a = {};
  a.cache_k = static_cast<uint16_t*>(cache_k), a.cache_v = static_cast<uint16_t*>(cache_v);
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v), a.positions = positions, a.lengths = lengths;
  a.B = B, a.N = N, a.d = C, a.window = window, a.sinks = sinks;
  a.ck_b = ck_stride_b, a.ck_n = ck_stride_n, a.cv_b = cv_stride_b, a.cv_n = cv_stride_n;
  a.k_b = k_stride_b, a.k_n = k_stride_n, a.v_b = v_stride_b, a.v_n = v_stride_n;
  hipLaunchKernelGGL(window_append_kernel, dim3((unsigned)groups, (unsigned)B), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}

SANA_API size_t sana_hip_window_step_workspace_bytes(int B, int H, int Hkv, int d, int window, int sinks) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || d <= 0 || d > 128 || window <= 0 || sinks < 0 || (int64_t)window + sinks > (1 << 30)) return 0;
  if (step_groups(B, H, Hkv) >= WA_MAX_BLOCKS) return 0;
  return part_bytes(step_splits(B, H, Hkv, window + sinks, d), (int64_t)B * H, d);
}

SANA_API int sana_hip_window_step(const void* q, const void* k, const void* v, void* cache_k, void* cache_v, const int32_t* positions,
                                  void* out, void* workspace, size_t workspace_bytes, int B, int H, int Hkv, int d, int window,
                                  int sinks, int64_t q_stride_b, int64_t k_stride_b, int64_t v_stride_b, int64_t ck_stride_b,
                                  int64_t ck_stride_n, int64_t cv_stride_b, int64_t cv_stride_n, int64_t o_stride_b, float scale,
                                  int io_dtype, void* stream) {
  if (!q || !k || !v || !cache_k || !cache_v || !positions || !out || !(scale > 0.f && scale * 1.44269504088896341f < INFINITY)) return SANA_ERR_ARG;
  const int rc = check_sizes(B, 1, H, Hkv, d, window, sinks, io_dtype);
  if (rc != SANA_OK) return rc;
  const int64_t C = (int64_t)Hkv * d;
  if (ck_stride_n < C || cv_stride_n < C) return SANA_ERR_ARG;
  for (const int64_t sb : {q_stride_b, k_stride_b, v_stride_b, ck_stride_b, cv_stride_b, o_stride_b})
    if (sb < 0) return SANA_ERR_ARG;
  if (B > 1 && (o_stride_b < (int64_t)H * d || ck_stride_b < C || cv_stride_b < C)) return SANA_ERR_ARG;  // (streams that would write the same elements)
  if ((int64_t)window + sinks > (1 << 30) || step_groups(B, H, Hkv) >= WA_MAX_BLOCKS) return SANA_ERR_SHAPE;
  if (misaligned({q, k, v, cache_k, cache_v}, {q_stride_b, k_stride_b, v_stride_b, ck_stride_b, ck_stride_n, cv_stride_b, cv_stride_n}) ||
      (reinterpret_cast<uintptr_t>(out) & 7u) || o_stride_b % 4 || off4(positions))
    return SANA_ERR_ALIGN;
  WindowArgs a = {};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out), a.cache_k = static_cast<uint16_t*>(cache_k), a.cache_v = static_cast<uint16_t*>(cache_v);
  a.positions = positions, a.B = B, a.N = 1, a.Nk = 1, a.H = H, a.Hkv = Hkv, a.d = d, a.window = window, a.sinks = sinks;
  a.q_b = q_stride_b, a.k_b = k_stride_b, a.v_b = v_stride_b, a.o_b = o_stride_b;
  a.ck_b = ck_stride_b, a.ck_n = ck_stride_n, a.cv_b = cv_stride_b, a.cv_n = cv_stride_n;
  a.scale_log2e = scale * 1.44269504088896341f;
  a.splits = step_splits(B, H, Hkv, window + sinks, d);
  const int64_t rows = (int64_t)B * H;
  if (a.splits > 1) {
    if (!workspace || workspace_bytes < part_bytes(a.splits, rows, d)) return SANA_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SANA_ERR_ALIGN;
    a.part_o = static_cast<float*>(workspace), a.part_ml = a.part_o + a.splits * rows * d;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return io_dtype == SANA_DT_F16 ? step_of<F16>(a, s) : step_of<BF16>(a, s);
}
