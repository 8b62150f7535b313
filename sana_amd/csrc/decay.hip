// Linear attention with a decay for each head, causal, bf16 or f16 in and out, the state in fp32:
//
//   S_t = exp(g_h) S_{t-1} + v_t k_t^T,   o_t = scale * S_t q_t,   S [d of v][d of k] per (batch, head).
//
// One token (the serving loop) is the recurrence itself: the state is read and written once, nothing else is of any size.
// A prompt goes in chunks of C = 64 tokens.  With a = exp(g_h), token t of a chunk and S0 the state in front of it,
//
//   o_t = scale * (a^(t+1) S0 q_t + sum_{j <= t} a^(t-j) (q_t . k_j) v_j),     S = a^C S0 + sum_j a^(C-1-j) v_j k_j^T:
//
// four products of 64 rows on the matrix pipes, 4 C d + 4 d^2 operations a token and head against 8 d bytes of memory.
#include "stream_common.h"

namespace sana {
namespace {

constexpr int DC = 64;  // tokens of a chunk

struct DecayArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  const float *log_decay, *state_in;
  float *state_out, *segments;  // segments: [B * H][nseg][d * d], the states in front of each segment
  const int* lengths;
  int N, H, d, nseg, seg_tokens, units;
  int64_t q_b, q_n, k_b, k_n, v_b, v_n, o_b, o_n;
  float scale;
};

// (addresses as integers: through pointers the compiler reads further ahead than the registers hold)
__device__ __forceinline__ u32x2_t dc_read_tr(uint32_t at) { return lds_read_tr((lds_t*)(size_t)at); }
__device__ __forceinline__ u32x4_t dc_read(uint32_t at) { return lds_read((const lds_t*)(size_t)at); }
__device__ __forceinline__ u32x2_t dc_read8(uint32_t at) { return lds_read8((const lds_t*)(size_t)at); }
// exp(g) as a power of two; below 2^-256 a decay is 0 in every power but the 0th, and -inf * 0 must not be NaN
__device__ __forceinline__ float dc_log2(float g) {
  const float g2 = g * 1.44269504088896341f;
  return g2 < -256.0f ? -256.0f : g2;
}
__device__ __forceinline__ float dc_pow(float g2, int n) { return __builtin_amdgcn_exp2f(g2 * (float)n); }
// the power of two that takes a maximum to 2^14 .. 2^15 (f16 ends at 2^16), within 2^-90 .. 2^40
__device__ __forceinline__ float dc_fit(float most) {
  const int e = (int)((__float_as_uint(most) >> 23) & 255u);  // 255: inf or NaN stay what they are
  const int f = e == 255 ? 127 : min(max(127 + 14 + 127 - e, 37), 167);
  return __uint_as_float((uint32_t)f << 23);
}

// What a launch of the chunks gives: the sums of a segment alone, the outputs of segments whose states are known, or both for whole streams.
enum { DC_SUMS, DC_OUT, DC_WHOLE };

// One workgroup of four waves takes a (batch, head, segment) through its chunks.  NV of its waves share the channels of v, 16 VT
// each, whose columns of the state stay in their registers (fp32) from chunk to chunk; where the head has fewer channels, 4 / NV waves
// with the same ones share the queries.  Each wave scores 16 queries for all, through LDS.
// The operands of the MFMAs (16 x 16 x 32):
//   scores^T = K Q^T   both from LDS as they lie;
//   out^T    = S Q^T   S as its own accumulators hold it (row v of the product: lane; a lane's 8 values of k: the accumulators of two
//                      tiles, channels 32 s + 4 g + {0..3} and + 16), Q in that order of k: two 8-byte reads;
//   out^T   += V^T P^T V by transposing reads, P^T from LDS in the key order that these give;
//   S       += K^T V   both by transposing reads.
// Roundings.  Each product of the output has one operand of 16 bits that is rounded, P or S, as attention kernels round P: with the rounding of
// the result the error is 1.4 times that of the result's rounding alone.  The weighted values a^(C-1-j) v_j enter the state as a sum of
// 16-bit values: three of bf16 where the state is given back (fp32's accuracy; with two it is 1.3e-6 off after 32760
// tokens), two of bf16 where it only goes on to outputs, two of f16, the second times 2^11 (22 bits from 2^-14 on; smaller values end at 2^-36, as f16
// values themselves end at 2^-25).
// f16 ends at 65504: S goes in scaled by a power of two for each wave, P for each query.
// A value that is not finite must not reach the queries in front of it (0 * inf): it is staged as 0, and its channel is set to NaN from its
// token on.
// What bounds it: where all compute units work, memory (32760 tokens x 20 heads of 112, 25 segments, rows of 224 bytes: sums 80 us = 318 MB at 4.0 TB/s;
// outputs 159 us = 612 MB at 3.8 TB/s, of which their loads and stores alone take 132, 4.6 TB/s) and, for the rest, the chain of a chunk's steps;
// few chunks, that chain alone, some 2 us
// (32 channels) to 4 us (112) each: three barriers, each with the LDS and MFMA latencies in front of it (300 tokens x 70 heads of 32: five
// chunks, 12 us; 2 x 4680 tokens, one stream half as long: outputs 48 us, their loads and stores alone 36).  Two chunks requested ahead, three workgroups a compute unit and eight waves a workgroup were no faster.
template <typename T, int DK, int KT, int VT, int NV, int MODE>
__global__ __launch_bounds__(256, 2) void decay_chunk_kernel(const DecayArgs a) {
  constexpr bool OUT = MODE != DC_SUMS, F = is_f16<T>;
  constexpr int PITCH = DK * 64, TILE = DC * PITCH;  // LDS row / tensor in bytes
  constexpr int NT = 256, PIECES = DC * DK * 4 / NT, TERMS = F || MODE == DC_OUT ? 2 : 3;
  constexpr int NQ = 4 / NV, QN = 4 / NQ;  // shares of the queries, query tiles of a share
  static_assert(KT <= 2 * DK && DC * DK * 4 % NT == 0 && 4 % NV == 0, "");
  __shared__ __attribute__((aligned(16))) unsigned char smem[(OUT ? 3 : 2) * TILE + (OUT ? DC * 128 + DC * 4 + DK * 128 + 16 : 0)];
  const uint32_t sk = (uint32_t)(size_t)(lds_t*)smem;
  const uint32_t sv = sk + TILE, sq = sk + 2 * TILE, sp = sk + 3 * TILE;
  float* fit = reinterpret_cast<float*>(smem + 3 * TILE + DC * 128);  // f16: the scale of a query's P
  int* odd = reinterpret_cast<int*>(fit + DC);  // each channel's first row that is not finite; behind them: the last chunk that holds one
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = tid & 15, fg = (tid >> 4) & 3;
  const int v0 = 16 * VT * (wave % NV), qt0 = QN * (wave / NV);

  // Four neighbouring heads, whose rows share cache lines, go to one XCD, the next four to the next: streams of unlike length, whose last
  // segments are not there, leave no XCD idle.
  const int slot = blockIdx.x >> 3, unit = (slot >> 2) * 8 + (blockIdx.x & 7), parts = (a.H + 3) >> 2;
  if (unit >= a.units) return;
  const int h = 4 * (unit % parts) + (slot & 3), rest = unit / parts, seg = rest % a.nseg, b = rest / a.nseg, d = a.d, bh = b * a.H + h;
  if (h >= a.H) return;
  const int n = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
  const int first = seg * a.seg_tokens, last = min(n, first + a.seg_tokens);  // (host: seg * seg_tokens < N)
  if (MODE != DC_WHOLE && first >= n) return;
  const float g2 = dc_log2(a.log_decay[h]);

  // ---- the state: st[vt][kt][r] = row v = v0 + 16 vt + fr, column k = 16 kt + 4 fg + r
  f32x4_t st[VT][KT];
  const float* s0 = MODE == DC_SUMS ? nullptr : MODE == DC_OUT ? a.segments + ((int64_t)bh * a.nseg + seg) * d * d : a.state_in ? a.state_in + (int64_t)bh * d * d : nullptr;
#pragma unroll
  for (int vt = 0; vt < VT; ++vt)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int v = v0 + 16 * vt + fr, k = 16 * kt + 4 * fg;
      st[vt][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (s0 && v < d && k < d) st[vt][kt] = *reinterpret_cast<const f32x4_t*>(s0 + v * d + k);
    }

  // ---- powers of the decay.  A chunk of fewer than 64 tokens fills the last rows of its tile, zeros in front of it, so only `since`
  // and `over` depend on how many there are.  Exponents are split into a part of the lane and one of the tile, none below 0.
  auto uniform = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); };
  const float lane12 = dc_pow(g2, 12 - 4 * fg);
  float to_end[2][8];  // a^(C - 1 - t) of the tokens of this lane's transposed values, less 12 - 4 fg
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) to_end[s][e] = uniform(dc_pow(g2, 63 - 12 - 32 * s - 16 * (e >> 2) - (e & 3)));
  // scale * a^(t - j): of the tile on the diagonal (0 where j > t); in front of it the lane's part, that of the tile's row
  float diagonal[4], before = 0.f, row4[4], step16 = 0.f;
  if constexpr (OUT) {
    before = a.scale * lane12 * dc_pow(g2, fr);
    step16 = uniform(dc_pow(g2, 16));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      diagonal[r] = fr >= 4 * fg + r ? a.scale * dc_pow(g2, fr - 4 * fg - r) : 0.f;
      row4[r] = uniform(dc_pow(g2, 4 - r));
    }
  }
  float since[QN], over;  // scale * a^(t + 1); a^count
  auto counted = [&](int count) {
    over = dc_pow(g2, count);
#pragma unroll
    for (int q = 0; q < QN; ++q) since[q] = a.scale * dc_pow(g2, max(16 * (qt0 + q) + fr + 1 - (DC - count), 0));
  };
  counted(DC);

  // ---- a chunk's rows: requested into registers a chunk ahead, then to LDS.  K, Q and V each at a time of its own: a wave that issues
  // more loads than the memory pipeline holds waits there, and the LDS tile of V is not needed before the scores are done.
  u32x4_t rk[PIECES], rv[PIECES], rq[OUT ? PIECES : 1];
  const uint32_t k2 = 2 * (uint32_t)a.k_n, v2 = 2 * (uint32_t)a.v_n, q2 = 2 * (uint32_t)a.q_n;
  auto request = [&](const uint16_t* tokens, int64_t stride, uint32_t ld2, int at, u32x4_t* r) {
    const int count = min(last - at, DC), empty = DC - count;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(tokens + (int64_t)at * stride), 0, (int)((uint32_t)(count - 1) * ld2 + 2 * d), 0x00020000);
    // (outside, as rows below 0 are: zeros.  63 rows are less than 2^31 bytes, so nothing comes back in)
    if constexpr (NT % (DK * 4) == 0) {
      const int row = tid / (DK * 4), c = tid - row * (DK * 4);
      const uint32_t off = (8 * c < d ? (uint32_t)row * ld2 + 16 * c : 0x80000000u) - empty * ld2;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        r[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(off + i * (NT / (DK * 4)) * ld2), 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int idx = tid + NT * i, row = idx / (DK * 4), c = idx - row * (DK * 4);
        const uint32_t off = 8 * c < d ? (uint32_t)(row - empty) * ld2 + 16 * c : 0x80000000u;
        r[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)off, 0, 0));
      }
    }
  };
  auto stage = [&](const u32x4_t* r, int tile) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int idx = tid + NT * i, row = idx / (DK * 4), c = idx - row * (DK * 4);
      *reinterpret_cast<u32x4_t*>(smem + tile * TILE + row * PITCH + ((c ^ row_key<DK>(row)) << 4)) = r[i];
    }
  };
  auto clean = [&](const u32x4_t* r, int chunk) {  // V as it is staged
    u16x2_t most = {0, 0};
#pragma unroll
    for (int i = 0; i < PIECES; ++i) most = max_magnitude(most, r[i]);
    if (__builtin_expect(most.x >= kInf16<T> || most.y >= kInf16<T>, 0)) {
      int me = tid;
      asm volatile("" : "+v"(me));  // (here and where `odd` is read: no address of this is worked out ahead and kept)
#pragma unroll 1
      for (int at = 0; at < 8 * PIECES; ++at) {  // this thread's own pieces, in LDS
        const int idx = me + NT * (at >> 3), row = idx / (DK * 4), c = idx - row * (DK * 4);
        uint16_t* x = reinterpret_cast<uint16_t*>(smem + TILE + row * PITCH + ((c ^ row_key<DK>(row)) << 4)) + (at & 7);
        if ((*x & 0x7fffu) < kInf16<T>) continue;
        *x = 0;
        __hip_atomic_fetch_min(odd + 8 * c + (at & 7), row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      odd[32 * DK] = chunk;
    }
  };
  if (OUT && tid <= 32 * DK) odd[tid] = tid < 32 * DK ? DC : -1;
  const uint16_t *kp = a.k + b * a.k_b + h * d, *vp = a.v + b * a.v_b + h * d, *qp = a.q + b * a.q_b + h * d;
  // bf16 sums are weighted up to the segment's end at once: they need no decay from chunk to chunk (f16 would run out of range) and no
  // order, and go backwards, so that the rows with which the outputs begin are the ones that the memory-side cache has seen last.
  constexpr bool FAR = MODE == DC_SUMS && !F;
  const int chunks = (last - first + DC - 1) / DC;
  auto token_of = [&](int i) { return first + DC * (FAR ? chunks - 1 - i : i); };
  if (first < last) {
    request(kp, a.k_n, k2, token_of(0), rk);
    if constexpr (OUT) request(qp, a.q_n, q2, token_of(0), rq);
    request(vp, a.v_n, v2, token_of(0), rv);
  }

  // ---- this lane's places in LDS
  const int key = row_key<DK>(fr);
  uint32_t row16[DK];  // row fr, k = 32 s + 8 fg
#pragma unroll
  for (int s = 0; s < DK; ++s) row16[s] = fr * PITCH + (((4 * s + fg) ^ key) << 4);
  const int trow = 4 * fg + (fr >> 2), tkey = row_key<DK>(trow), piece = fr & 3;  // of a transposing read
  uint32_t vt_at[VT];
#pragma unroll
  for (int vt = 0; vt < VT; ++vt) vt_at[vt] = sv + trow * PITCH + (((v0 / 8 + 2 * vt + (piece >> 1)) ^ tkey) << 4) + 8 * (piece & 1);
  auto kt_at = [&](int kt) { return sk + trow * PITCH + (((2 * kt + (piece >> 1)) ^ tkey) << 4) + 8 * (piece & 1); };
  auto row8 = [&](int kt) { return (uint32_t)(fr * PITCH + (((2 * kt + (fg >> 1)) ^ key) << 4) + 8 * (fg & 1)); };  // row fr, k = 16 kt + 4 fg
  const bool own = v0 < 32 * DK;  // (DK = 3: the fourth wave has no channels of v, and its reads would leave the rows)

#pragma unroll 1
  for (int i = 0; i < chunks; ++i) {
    const int at = token_of(i), count = min(last - at, DC), next = token_of(i + 1);
    const bool more = i + 1 < chunks;
    stage(rk, 0);
    if constexpr (OUT) stage(rq, 2);
    else stage(rv, 1);
    lds_barrier();
    if (more) request(kp, a.k_n, k2, next, rk);
    __builtin_amdgcn_sched_barrier(0);
    if (count < DC) counted(count);
    f32x4_t oc[VT][QN];  // out^T: channel v0 + 16 vt + 4 fg + r, query 16 (qt0 + q) + fr
    u32x4_t vf[2][VT];   // values of two ranges of 32 tokens
    bool some_odd = false;
    if constexpr (OUT) {
      // ---- scores, decayed, to LDS: row = query, 16-byte slot 4 s + g = keys 32 s + 4 g + {0..3}, + 16
      f32x4_t sc[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) sc[kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DK; ++s) {
        const u32x4_t qf = dc_read(sq + 16 * wave * PITCH + row16[s]);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
          if (kt <= wave) sc[kt] = mfma_16x16x32<T>(dc_read(sk + 16 * kt * PITCH + row16[s]), qf, sc[kt]);
      }
      float most = 0.f, f = 1.f;
      float ahead = before;  // of tile kt: a^(16 (tiles between it and the diagonal)), from the last in front of the diagonal on
      // (selects, no branches: a tile's place is uniform, and each of these as a branch of its own takes longer than the arithmetic)
#pragma unroll
      for (int kt = 3; kt >= 0; --kt) {
        const bool in_front = kt < wave, at_diagonal = kt == wave;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = sc[kt][r] * (in_front ? ahead * row4[r] : diagonal[r]);
          sc[kt][r] = in_front | (at_diagonal & (fr >= 4 * fg + r)) ? x : 0.f;
          if constexpr (F) most = fmaxf(most, fabsf(sc[kt][r]));
        }
        ahead *= in_front ? step16 : 1.f;
      }
      if constexpr (F) {
        f = dc_fit(max_groups(most));
        if (fg == 0) fit[16 * wave + fr] = f;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int q = 16 * wave + fr;
        u32x4_t p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4_t x = sc[2 * s + (e >> 1)];
          p[e] = F ? pk16<T>(x[2 * (e & 1)] * f, x[2 * (e & 1) + 1] * f) : pk16<T>(x[2 * (e & 1)], x[2 * (e & 1) + 1]);
        }
        *reinterpret_cast<u32x4_t*>(smem + 3 * TILE + q * 128 + (((4 * s + fg) ^ ((q >> 1) & 7)) << 4)) = p;
      }
      __builtin_amdgcn_sched_barrier(0);
      // ---- the state in front of the chunk
      float sfit = 1.f;
      if constexpr (F) {
        float most = 0.f;
#pragma unroll
        for (int vt = 0; vt < VT; ++vt)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(st[vt][kt][r]));
        most = max_wave(most);
        if (__builtin_expect(most == INFINITY, 0)) {  // (a carried inf: the other channels go in by their own maximum.  1 - 1.5 % of an f16 call)
          most = 0.f;
#pragma unroll
          for (int vt = 0; vt < VT; ++vt)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
              for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(st[vt][kt][r]) < INFINITY ? fabsf(st[vt][kt][r]) : 0.f);
          most = max_wave(most);
        }
        sfit = dc_fit(most);
      }
#pragma unroll
      for (int vt = 0; vt < VT; ++vt)
#pragma unroll
        for (int q = 0; q < QN; ++q) oc[vt][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DK; ++s) {
        u32x4_t sf[VT];
#pragma unroll
        for (int vt = 0; vt < VT; ++vt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (2 * s + (e >> 1) >= KT) {
              sf[vt][e] = 0u;
              continue;
            }
            const f32x4_t x = st[vt][2 * s + (e >> 1)];
            sf[vt][e] = F ? pk16<T>(x[2 * (e & 1)] * sfit, x[2 * (e & 1) + 1] * sfit) : pk16<T>(x[2 * (e & 1)], x[2 * (e & 1) + 1]);
          }
#pragma unroll
        for (int q = 0; q < QN; ++q) {
          const uint32_t from = sq + 16 * (qt0 + q) * PITCH;
          const u32x2_t lo = dc_read8(from + row8(2 * s)), hi = dc_read8(from + row8(2 * s + 1));
          const u32x4_t qf = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int vt = 0; vt < VT; ++vt) oc[vt][q] = mfma_16x16x32<T>(sf[vt], qf, oc[vt][q]);
        }
      }
      stage(rv, 1);
      clean(rv, i);
      if (more) request(qp, a.q_n, q2, next, rq);
      lds_barrier();
      some_odd = __builtin_amdgcn_readfirstlane(odd[32 * DK]) == i;
      if (more) request(vp, a.v_n, v2, next, rv);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < QN; ++q) {
        const float m = F ? since[q] * fit[16 * (qt0 + q) + fr] / sfit : since[q];
#pragma unroll
        for (int vt = 0; vt < VT; ++vt)
#pragma unroll
          for (int r = 0; r < 4; ++r) oc[vt][q][r] *= m;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int vt = 0; vt < VT; ++vt) {
        vf[s][vt] = u32x4_t{0u, 0u, 0u, 0u};
        if (own) {
          const u32x2_t x = dc_read_tr(vt_at[vt] + 32 * s * PITCH), y = dc_read_tr(vt_at[vt] + (32 * s + 16) * PITCH);
          vf[s][vt] = u32x4_t{x.x, x.y, y.x, y.y};
        }
      }
    if constexpr (OUT) {
      // ---- the scores' part
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int q = 0; q < QN; ++q) {
          if (NQ == 1 && 2 * s > q) continue;  // (queries of the first 32 see none of the second 32 tokens)
          const int row = 16 * (qt0 + q) + fr;
          const u32x4_t pf = dc_read(sp + row * 128 + (((4 * s + fg) ^ ((row >> 1) & 7)) << 4));
#pragma unroll
          for (int vt = 0; vt < VT; ++vt) oc[vt][q] = mfma_16x16x32<T>(vf[s][vt], pf, oc[vt][q]);
        }
      if (__builtin_expect(some_odd && own, 0)) {
        int at = tid;
        asm volatile("" : "+v"(at));
        const int first_row = 16 * qt0 + (at & 15), c = v0 + 4 * ((at >> 4) & 3);
#pragma unroll
        for (int vt = 0; vt < VT; ++vt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int from = odd[c + 16 * vt + r] - first_row;
#pragma unroll
            for (int q = 0; q < QN; ++q) oc[vt][q][r] = 16 * q >= from ? NAN : oc[vt][q][r];
          }
      }
      // (rows below 0 and channels past d lie outside the resource: not stored)
      const uint32_t o2 = 2 * (uint32_t)a.o_n;
      const __amdgpu_buffer_rsrc_t ro =
          __builtin_amdgcn_make_buffer_rsrc(a.out + b * a.o_b + (int64_t)at * a.o_n + h * d, 0, (int)((uint32_t)(count - 1) * o2 + 2 * d), 0x00020000);
#pragma unroll
      for (int q = 0; q < QN; ++q) {
        const int row = 16 * (qt0 + q) + fr;
        const float m = F ? 1.0f / fit[row] : 1.f;
#pragma unroll
        for (int vt = 0; vt < VT; ++vt) {
          const int c = v0 + 16 * vt + 4 * fg;
          const uint32_t off = (c < d ? (uint32_t)(16 * qt0 + fr) * o2 + 2 * c : 0x80000000u) - (DC - count) * o2 + 16 * q * o2;
          const f32x4_t x = oc[vt][q];
          const u32x2_t y = F ? u32x2_t{pk16<T>(x[0] * m, x[1] * m), pk16<T>(x[2] * m, x[3] * m)} : u32x2_t{pk16<T>(x[0], x[1]), pk16<T>(x[2], x[3])};
          __builtin_amdgcn_raw_buffer_store_b64(y, ro, (int)off, 0, 0);
        }
      }
    }
    // ---- the state behind the chunk
    if (!OUT && more) request(vp, a.v_n, v2, next, rv);
    const float lane = FAR ? lane12 * dc_pow(g2, last - at - count) : lane12;
    __builtin_amdgcn_sched_barrier(0);
    if (own) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        __builtin_amdgcn_sched_barrier(0);
        u32x4_t w[TERMS][VT];
#pragma unroll
        for (int vt = 0; vt < VT; ++vt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x0 = lo16<T>(vf[s][vt][e]) * (lane * to_end[s][2 * e]), x1 = hi16<T>(vf[s][vt][e]) * (lane * to_end[s][2 * e + 1]);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) {
              w[i][vt][e] = pk16<T>(x0, x1);
              x0 -= lo16<T>(w[i][vt][e]), x1 -= hi16<T>(w[i][vt][e]);
              if constexpr (F) x0 *= 2048.f, x1 *= 2048.f;
            }
          }
        // (two tiles of k at a time, term by term: an MFMA that adds to what the one before it has just summed waits for twice its own time)
#pragma unroll
        for (int k0 = 0; k0 < KT; k0 += 2) {
          u32x4_t kf[2];
          f32x4_t y[2][VT];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (k0 + j >= KT) continue;
            const uint32_t from = kt_at(k0 + j) + 32 * s * PITCH;
            const u32x2_t lo = dc_read_tr(from), hi = dc_read_tr(from + 16 * PITCH);
            kf[j] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
            for (int vt = 0; vt < VT; ++vt) {
              if (s == 0 && !FAR)
#pragma unroll
                for (int r = 0; r < 4; ++r) st[vt][k0 + j][r] *= over;
              y[j][vt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            }
          }
#pragma unroll
          for (int i = 0; i < TERMS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int vt = 0; vt < VT; ++vt) {
                if (k0 + j >= KT) continue;
                f32x4_t& x = F && i == 1 ? y[j][vt] : st[vt][k0 + j];
                x = mfma_16x16x32<T>(kf[j], w[i][vt], x);
              }
          if constexpr (F) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int vt = 0; vt < VT; ++vt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (k0 + j < KT) st[vt][k0 + j][r] = fmaf(y[j][vt][r], 1.0f / 2048.f, st[vt][k0 + j][r]);
          }
        }
      }
    }
    if constexpr (OUT) {
      if (__builtin_expect(some_odd && own, 0)) {
        int at = tid;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int vt = 0; vt < VT; ++vt) {
          const float x = odd[v0 + 16 * vt + (at & 15)] < DC ? NAN : 0.f;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) st[vt][kt][r] += x;
        }
      }
    }
    lds_barrier();
  }
  // ---- the state behind the last token, or the segment's sum
  if (MODE != DC_OUT && qt0 == 0) {
    float* to = MODE == DC_SUMS ? a.segments + ((int64_t)bh * a.nseg + seg) * d * d : a.state_out + (int64_t)bh * d * d;
#pragma unroll
    for (int vt = 0; vt < VT; ++vt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const int v = v0 + 16 * vt + fr, k = 16 * kt + 4 * fg;
        if (v < d && k < d) *reinterpret_cast<f32x4_t*>(to + v * d + k) = st[vt][kt];
      }
  }
}

// The segments' own sums -> the states in front of them, and the one behind the last: run = S0; run = a^(tokens) run + sum.  Four
// values a thread, eight segments requested at a time, so that a chain of 25 waits for memory four times: 10 us for 25 MB read and written (with 20
// heads of 112, one pass over the workspace; its threads are too few to do better).
__global__ __launch_bounds__(64) void decay_scan_kernel(const DecayArgs a) {
  constexpr int AHEAD = 8;
  const int bh = blockIdx.y, b = bh / a.H, i = blockIdx.x * 64 + threadIdx.x, dd4 = a.d * a.d / 4;
  if (i >= dd4) return;
  const int n = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
  const float g2 = dc_log2(a.log_decay[bh % a.H]);
  f32x4_t* s = reinterpret_cast<f32x4_t*>(a.segments) + (int64_t)bh * a.nseg * dd4 + i;
  f32x4_t run = {0.f, 0.f, 0.f, 0.f};
  if (a.state_in) run = reinterpret_cast<const f32x4_t*>(a.state_in)[(int64_t)bh * dd4 + i];
  const int used = (n + a.seg_tokens - 1) / a.seg_tokens;
  for (int seg = 0; seg < used; seg += AHEAD) {
    f32x4_t own[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) own[j] = s[(int64_t)min(seg + j, used - 1) * dd4];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (seg + j >= used) break;
      s[(int64_t)(seg + j) * dd4] = run;
      const float over = dc_pow(g2, min(n - (seg + j) * a.seg_tokens, a.seg_tokens));
#pragma unroll
      for (int r = 0; r < 4; ++r) run[r] = fmaf(run[r], over, own[j][r]);
    }
  }
  reinterpret_cast<f32x4_t*>(a.state_out)[(int64_t)bh * dd4 + i] = run;
}

// One token of each stream.  A row of the state is d floats in LPR lanes of four; a wave holds 64 / LPR rows at a time.  Memory alone bounds it: 128
// streams x 35 heads of 64, 147 MB of state in and out, 30.6 us = 4.8 TB/s, as a large copy; one stream is a launch and two loads (20 heads
// of 112 4.5 us).
template <typename T, int LPR>
__global__ __launch_bounds__(256) void decay_step_kernel(const DecayArgs a) {
  constexpr int RW = 64 / LPR;  // rows of a wave
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H, d = a.d;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = 4 * (lane % LPR);
  const bool idle = a.lengths && a.lengths[b] <= 0;
  const float decay = idle ? 1.f : dc_pow(dc_log2(a.log_decay[h]), 1);
  const uint16_t *qp = a.q + b * a.q_b + h * d, *kp = a.k + b * a.k_b + h * d, *vp = a.v + b * a.v_b + h * d;
  uint16_t* op = a.out + b * a.o_b + h * d;
  float q[4], k[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = k[e] = 0.f;
  if (c < d && !idle) {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(qp + c), y = *reinterpret_cast<const u32x2_t*>(kp + c);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      q[2 * e] = a.scale * lo16<T>(x[e]), q[2 * e + 1] = a.scale * hi16<T>(x[e]);
      k[2 * e] = lo16<T>(y[e]), k[2 * e + 1] = hi16<T>(y[e]);
    }
  }
  const int64_t base = (int64_t)bh * d * d;
  for (int row = (blockIdx.y * 4 + wave) * RW + lane / LPR; row - lane / LPR < d; row += 4 * RW * gridDim.y) {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
    const bool in = row < d && c < d;
    if (in && a.state_in) s = *reinterpret_cast<const f32x4_t*>(a.state_in + base + row * d + c);
    float v = 0.f;
    if (row < d && !idle) v = lo16<T>(vp[row]);
    float o = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = fmaf(decay, s[e], v * k[e]);
      o = fmaf(q[e], s[e], o);
    }
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) o += __shfl_xor(o, m);
    if (in) *reinterpret_cast<f32x4_t*>(a.state_out + base + row * d + c) = s;
    if (row < d && c == 0 && !idle) op[row] = (uint16_t)pk16<T>(o, 0.f);
  }
}

// Segments of a stream, whole chunks each.  A head alone is a chain of chunks, some 2 us each (112 channels 4), on one compute unit;
// segments run side by side, but read K and V twice, and each reads and writes a state three times.  us, whole / in segments:
//   enough of them to fill the chip: 20 heads of 112 x 4096 tokens 274 / 51 (12 segments), 32768 tokens 2143 / 234 (25), 140 of 112 x 4680
//   330 / 251 (3), 200 of 112 x 4096 296 / 313 (2): at least three, or none;
//   one workgroup a compute unit where the segments are short (20 of 112 x 4096, 11 and 22 segments: 51 / 57; 48 of 128 x 2048, 5 and 11: 62 / 66),
//   as many as it holds where they are long (20 of 112 x 16384, 12 and 24: 142 / 132) or the head narrow (70 of 32 x 2048, 4 and 11: 29 / 22);
//   two chunks at least (20 of 112 x 1024, 8 and 16: 26 / 28) and 64 segments at most (the scan is a chain too: 8 of 64 x 32768, 64 and 128: 57 / 71);
//   few chunks pay for two more launches where the heads are few: 8 of 64 x 384 15 / 13, 20 of 112 x 384 31 / 23, 80 of 112 x 640 48 / 40, but 64 of 64
//   x 320 14 / 18, 128 of 64 x 640 24 / 27, 70 of 32 x 512 14 / 15.
int segment_count(int B, int N, int H, int d, int* tokens) {
  const int chunks = (N + DC - 1) / DC;
  const int64_t heads = (int64_t)B * H;
  const int room = 256 * (d <= 32 ? 4 : d <= 64 ? 3 : 2);  // workgroups that the chip holds at a time
  int64_t want = room / heads;
  if (d > 64 && heads <= 256 && chunks < 12 * (256 / heads)) want = 256 / heads;
  want = want > 64 ? 64 : want;
  want = want > chunks / 2 ? chunks / 2 : want;
  if (want < 3 || chunks < 4 + heads / (d > 64 ? 16 : 8)) want = 1;
  const int per = (int)((chunks + want - 1) / want);
  *tokens = per * DC;
  return (chunks + per - 1) / per;
}

template <typename T, int DK, int KT, int VT, int NV>
int launch_chunks(const DecayArgs& a, int B, hipStream_t s) {
  const int64_t units = (int64_t)B * a.nseg * ((a.H + 3) / 4);
  if (units > (1 << 22) - 8) return SANA_ERR_SHAPE;  // 4 blocks of 256 threads a unit: fewer than 2^32 threads
  DecayArgs args = a;
  args.units = (int)units;
  const dim3 grid((unsigned)((units + 7) / 8 * 32)), block(256);
  if (a.nseg > 1) {
    hipLaunchKernelGGL((decay_chunk_kernel<T, DK, KT, VT, NV, DC_SUMS>), grid, block, 0, s, args);
    hipLaunchKernelGGL(decay_scan_kernel, dim3((unsigned)((a.d * a.d / 4 + 63) / 64), (unsigned)(B * a.H)), dim3(64), 0, s, args);
    hipLaunchKernelGGL((decay_chunk_kernel<T, DK, KT, VT, NV, DC_OUT>), grid, block, 0, s, args);
  } else {
    hipLaunchKernelGGL((decay_chunk_kernel<T, DK, KT, VT, NV, DC_WHOLE>), grid, block, 0, s, args);
  }
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}

template <typename T>
int launch_step(const DecayArgs& a, int B, hipStream_t s) {
  // (workgroups of a head: 1 stream of 20 heads of 112 with 1, 2, 4 8.5, 5.6, 4.5 us, 64 streams 29, 27, 26; 35 of 64
  // with 1, 2, 4 4.2, 3.5, 3.2, 16 streams 6.7, 6.0, 6.7; 16 streams of 70 of 32 with 1, 4 4.5, 5.4)
  const dim3 grid((unsigned)(B * a.H), a.d > 64 ? 4 : a.d > 32 ? 2 : 1), block(256);
  if (a.d > 64) hipLaunchKernelGGL((decay_step_kernel<T, 32>), grid, block, 0, s, a);
  else if (a.d > 32) hipLaunchKernelGGL((decay_step_kernel<T, 16>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((decay_step_kernel<T, 8>), grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? SANA_OK : SANA_ERR_LAUNCH;
}

template <typename T>
int decay_attention(const DecayArgs& a, int B, hipStream_t s) {
  if (a.N == 1) return launch_step<T>(a, B, s);
  if (a.d <= 32) return launch_chunks<T, 1, 2, 1, 2>(a, B, s);
  if (a.d <= 64) return launch_chunks<T, 2, 4, 1, 4>(a, B, s);
  if (a.d <= 96) return launch_chunks<T, 3, 6, 2, 4>(a, B, s);
  if (a.d <= 112) return launch_chunks<T, 4, 7, 2, 4>(a, B, s);
  return launch_chunks<T, 4, 8, 2, 4>(a, B, s);
}

}  // namespace
}  // namespace sana

using namespace sana;

#define SANA_API extern "C" __attribute__((visibility("default")))

SANA_API size_t sana_hip_decay_attention_workspace_bytes(int B, int N, int H, int d) {
  if (B <= 0 || N <= 1 || N > (1 << 30) || H <= 0 || d <= 0 || d > 128 || (int64_t)B * H >= (1 << 24)) return 0;
  int tokens;
  const int nseg = segment_count(B, N, H, d, &tokens);
  return nseg > 1 ? (size_t)B * H * nseg * d * d * sizeof(float) : 0;
}

SANA_API int sana_hip_decay_attention(const void* q, const void* k, const void* v, const float* log_decay, const float* state_in,
                                      float* state_out, void* out, const int32_t* lengths, void* workspace, size_t workspace_bytes,
                                      int B, int N, int H, int d, int64_t q_stride_b, int64_t q_stride_n, int64_t k_stride_b,
                                      int64_t k_stride_n, int64_t v_stride_b, int64_t v_stride_n, int64_t o_stride_b,
                                      int64_t o_stride_n, float scale, int io_dtype, void* stream) {
  if (!q || !k || !v || !log_decay || !state_out || !out || B <= 0 || N <= 0 || H <= 0 || d <= 0) return SANA_ERR_ARG;
  if (io_dtype != SANA_DT_BF16 && io_dtype != SANA_DT_F16) return SANA_ERR_DTYPE;
  if (d % 8 || d > 128 || (int64_t)B * H >= (1 << 24) || N > (1 << 30)) return SANA_ERR_SHAPE;
  for (const int64_t ld : {q_stride_n, k_stride_n, v_stride_n, o_stride_n}) {
    if (ld < (int64_t)H * d) return SANA_ERR_ARG;
    if (ld >= (1 << 23)) return SANA_ERR_SHAPE;  // 32-bit byte offsets within a chunk
  }
  for (const int64_t sb : {q_stride_b, k_stride_b, v_stride_b, o_stride_b})
    if (sb < 0) return SANA_ERR_ARG;
  if (B > 1 && o_stride_b < (int64_t)H * d) return SANA_ERR_ARG;  // (entries that would write the same elements)
  for (const void* p : {q, k, v, (const void*)state_in, (const void*)state_out})
    if (!aligned16(p)) return SANA_ERR_ALIGN;
  for (const int64_t st : {q_stride_b, q_stride_n, k_stride_b, k_stride_n, v_stride_b, v_stride_n})
    if (st % 8) return SANA_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(out) & 7u) || o_stride_b % 4 || o_stride_n % 4 || (reinterpret_cast<uintptr_t>(log_decay) & 3u) ||
      (reinterpret_cast<uintptr_t>(lengths) & 3u))
    return SANA_ERR_ALIGN;
  DecayArgs a;
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.log_decay = log_decay, a.state_in = state_in, a.state_out = state_out, a.segments = nullptr, a.lengths = lengths;
  a.N = N, a.H = H, a.d = d, a.nseg = 1, a.seg_tokens = N, a.units = 0;
  a.q_b = q_stride_b, a.q_n = q_stride_n, a.k_b = k_stride_b, a.k_n = k_stride_n, a.v_b = v_stride_b, a.v_n = v_stride_n;
  a.o_b = o_stride_b, a.o_n = o_stride_n, a.scale = scale;
  if (N > 1) a.nseg = segment_count(B, N, H, d, &a.seg_tokens);
  if (a.nseg > 1) {
    if (!workspace || workspace_bytes < sana_hip_decay_attention_workspace_bytes(B, N, H, d)) return SANA_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SANA_ERR_ALIGN;
    a.segments = static_cast<float*>(workspace);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return io_dtype == SANA_DT_F16 ? decay_attention<F16>(a, B, s) : decay_attention<BF16>(a, B, s);
}
