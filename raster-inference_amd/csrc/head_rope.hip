// Norms of query, key and value heads and the rotary positions in one pass.
//
// Per head row x of hd values: y = x * scale * gain (scale = 1 / sqrt(mean of
// the squares + eps), each product rounded to Q16.16), then for every pair
// (a, b) of the rotated part a' = a c - b s, b' = b c + a s with c, s the
// cosine and sine of position * frequency (times the amplitude).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "det_arith.h"
#include "verify.h"
#include "wave.h"

namespace det {

namespace {

template <int V>
struct Vec;
template <>
struct Vec<1> {
  static __device__ void load(const int32_t* p, int32_t* x) { x[0] = p[0]; }
  static __device__ void store(int32_t* p, const int32_t* x) { p[0] = x[0]; }
};
template <>
struct Vec<4> {
  static __device__ void load(const int32_t* p, int32_t* x) {
    const int4 v = *reinterpret_cast<const int4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
  static __device__ void store(int32_t* p, const int32_t* x) {
    *reinterpret_cast<int4*>(p) = make_int4(x[0], x[1], x[2], x[3]);
  }
};

// Q16.16 values as the doubles that they are: mul_sat(a, b) for b given as b
// 2^-16 (products below 2^62, so the rounded quotient is below 2^46).
__device__ __forceinline__ double clamp32(double v) {
  return __builtin_fmin(__builtin_fmax(v, -2147483648.0), 2147483647.0);
}
__device__ __forceinline__ double mul_q16(double a, double b16) { return clamp32(mul_rint(a, b16)); }

// One workgroup per token: its threads compute the token's cosines and sines
// once into LDS, then each group of `lanes` lanes takes up to U head rows at a
// time, V consecutive values per lane and step, E steps; the first rows' loads
// are on their way while the cosines are computed. A pair of the half layout
// meets through the rows' LDS copies, an interleaved pair in one lane (V = 4) or
// through them as well. WAVE: a wave per row (the rows' pointers are scalar). The
// products are double multiply-adds (2 instructions and the clamp, against 11 for
// one of 64-bit integers). Bound by these instructions at many tokens, then by the
// bytes: 4096 tokens of 8 / 2 heads of 256 in 28 us, 20 at a copy's rate.
template <int V, int E, int U, bool WAVE>
__global__ __launch_bounds__(256) void k_head_rope(HeadRopeArgs a, uint32_t lane_group) {
  extern __shared__ __attribute__((aligned(16))) double table[];  // cosines, sines (times 2^-16), U rows per lane group
  const uint32_t tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), lanes = WAVE ? 64 : lane_group;
  const uint32_t per_wave = 64 / lanes, li = lane % lanes, hd = a.hd, pairs = a.pairs;
  const uint32_t entries = (pairs + 3) & ~3u, row_ld = (hd + 3) & ~3u;
  const uint64_t t = blockIdx.x;
  double* cs = table;
  double* sn = table + entries;
  int32_t* row = reinterpret_cast<int32_t*>(table + 2 * entries) + (wave * per_wave + lane / lanes) * U * row_ld;
  const bool meet = !(V == 4 && a.interleaved);  // pairs meet in LDS
  const uint32_t step = waves * per_wave;
  for (uint32_t r0 = wave * per_wave;; r0 += step * U) {
    const bool turn = r0 == wave * per_wave;  // (every wave's first round)
    if (!turn && r0 >= a.total) break;
    // the rows' sets and heads, their values
    HeadSet s[U];
    const int32_t* src[U];
    int32_t* dst[U];
    bool on[U];
    int32_t x[U][E][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * step + (WAVE ? 0 : lane / lanes);
      on[u] = r < a.total;
      uint32_t h = on[u] ? r : 0;
      s[u] = a.set[0];
#pragma unroll
      for (uint32_t q = 1; q < kHeadSets; ++q)
        if (q < a.n_sets && h >= s[u].heads) {
          h -= s[u].heads;
          s[u] = a.set[q];
        }
      src[u] = s[u].x + t * s[u].ld + uint64_t(h) * hd;
      dst[u] = s[u].out + t * s[u].out_ld + uint64_t(h) * hd;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
#pragma unroll
        for (int v = 0; v < V; ++v) x[u][e][v] = 0;
        if (on[u] && c < hd) Vec<V>::load(src[u] + c, x[u][e]);
      }
    }
    if (turn && pairs) {
      const uint64_t pos = a.positions[t];
      for (uint32_t i = tid; i < pairs; i += blockDim.x) {
        int32_t c, sv;
        sin_cos_rint(rope_angle(pos, a.freq[i]), &c, &sv);
        cs[i] = (a.amplitude == kOneAct ? c : mul_sat(c, a.amplitude)) * 0x1p-16;
        sn[i] = (a.amplitude == kOneAct ? sv : mul_sat(sv, a.amplitude)) * 0x1p-16;
      }
      lds_barrier();
    }
    // sums of squares, saturating: the terms are non-negative, so that is the
    // least of the sum and i64::MAX in any order, and below 2^26 nothing saturates
    uint32_t large = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int v = 0; v < V; ++v) large |= uint32_t(x[u][e][v] ^ (x[u][e][v] >> 31));
    int64_t ss[U] = {};
    if (!__any(large >> 26)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) ss[u] += sq_term(x[u][e][v]);
        if (WAVE) ss[u] = wave_sum_wrap64(ss[u]);
        else
          for (uint32_t off = 1; off < lanes; off <<= 1) ss[u] += __shfl_xor(ss[u], int(off), 64);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) ss[u] = add_sat64_nn(ss[u], sq_term(x[u][e][v]));
        if (WAVE) ss[u] = wave_sum_sat64(ss[u]);
        else
          for (uint32_t off = 1; off < lanes; off <<= 1) ss[u] = add_sat64_nn(ss[u], __shfl_xor(ss[u], int(off), 64));
      }
    }
    // (a wave's U rows: lane u finds the scale of row u)
    int64_t mine = ss[0];
    if (WAVE)
#pragma unroll
      for (int u = 1; u < U; ++u) mine = lane == uint32_t(u) ? ss[u] : mine;
    const int32_t found = WAVE ? rms_scale_from_sumsq(mine, hd, a.eps) : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!(s[u].flags & 1)) continue;
      const int32_t scale = WAVE ? __builtin_amdgcn_readlane(found, u) : rms_scale_from_sumsq(ss[u], hd, a.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
        if (c >= hd) continue;
        int32_t g[V];
        if (s[u].gain) Vec<V>::load(s[u].gain + c, g);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          double y = mul_q16(double(x[u][e][v]), double(scale) * 0x1p-16);
          if (s[u].gain) y = mul_q16(y, double(g[v]) * 0x1p-16);
          x[u][e][v] = int32_t(y);
        }
      }
    }
    if (pairs) {
      if (meet) {
        wave_lds_sync();  // the previous round's rows have been read
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const uint32_t c = V * (li + 64 * e);
            if (c < hd && (s[u].flags & 2)) Vec<V>::store(row + u * row_ld + c, x[u][e]);
          }
        wave_lds_sync();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!(s[u].flags & 2)) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          int32_t y[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const uint32_t c = V * (li + 64 * e) + v;
            y[v] = x[u][e][v];
            if (c >= 2 * pairs) continue;
            const bool second = a.interleaved ? (c & 1) : c >= pairs;
            const uint32_t i = a.interleaved ? c >> 1 : (second ? c - pairs : c);
            const int32_t other =
                meet ? row[u * row_ld + (a.interleaved ? (c ^ 1) : (second ? c - pairs : c + pairs))] : x[u][e][v ^ (V > 1)];
            const double p = mul_q16(double(x[u][e][v]), cs[i]), q = mul_q16(double(other), sn[i]);
            y[v] = int32_t(clamp32(second ? p + q : p - q));
          }
#pragma unroll
          for (int v = 0; v < V; ++v) x[u][e][v] = y[v];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
        if (on[u] && c < hd) Vec<V>::store(dst[u] + c, x[u][e]);
      }
  }
}

template <int V, int E, int U>
void launch(const HeadRopeArgs& a, hipStream_t s) {
  uint32_t lanes = 64;
  if (E == 1)
    while (lanes > 1 && lanes / 2 * V >= a.hd) lanes /= 2;
  const uint32_t per_wave = 64 / lanes;
  uint32_t waves = (a.total + per_wave * U - 1) / (per_wave * U);
  waves = std::min(std::max(waves, a.pairs > 64 ? 2u : 1u), 4u);
  const size_t bytes = (4 * ((a.pairs + 3) & ~3u) + waves * per_wave * U * ((a.hd + 3) & ~3u)) * 4;
  const dim3 grid(unsigned(a.rows)), block(64 * waves);
  if (lanes == 64) hipLaunchKernelGGL((k_head_rope<V, E, U, true>), grid, block, bytes, s, a, lanes);
  else if constexpr (E == 1) hipLaunchKernelGGL((k_head_rope<V, E, U, false>), grid, block, bytes, s, a, lanes);
}

}  // namespace

void launch_head_rope(const HeadRopeArgs& a, hipStream_t s) {
  if (a.rows == 0 || a.total == 0) return;
  bool wide = a.hd % 4 == 0;
  for (uint32_t i = 0; i < a.n_sets; ++i) {
    const HeadSet& h = a.set[i];
    wide = wide && h.ld % 4 == 0 && h.out_ld % 4 == 0 &&
           ((reinterpret_cast<uintptr_t>(h.x) | reinterpret_cast<uintptr_t>(h.out) |
             reinterpret_cast<uintptr_t>(h.gain)) & 15) == 0;
  }
  if (wide) {
    if (a.hd <= 256) launch<4, 1, 3>(a, s);
    else if (a.hd <= 512) launch<4, 2, 3>(a, s);
    else launch<4, 4, 1>(a, s);
  } else {
    if (a.hd <= 64) launch<1, 1, 3>(a, s);
    else if (a.hd <= 256) launch<1, 4, 2>(a, s);
    else launch<1, 16, 1>(a, s);
  }
}

}  // namespace det
