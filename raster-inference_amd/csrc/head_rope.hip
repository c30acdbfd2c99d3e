// Norms of query, key and value heads and the rotary positions in one pass.
//
// Per head row x of hd values: y = x * scale * gain (scale = 1 / sqrt(mean of
// the squares + eps), each product rounded to Q16.16), then for every pair
// (a, b) of the rotated part a' = a c - b s, b' = b c + a s with c, s the
// cosine and sine of position * frequency (times the amplitude).
#include <hip/hip_runtime.h>

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

// One workgroup per token: its threads compute the token's cosines and sines
// once into LDS, then each group of `lanes` lanes takes one head row at a
// time, V consecutive values per lane and step, E steps. A pair of the half
// layout meets through the wave's LDS row; an interleaved pair sits in one
// lane (V = 4) or in neighbouring ones.
template <int V, int E>
__global__ __launch_bounds__(512) void k_head_rope(HeadRopeArgs a, uint32_t lanes) {
  extern __shared__ __attribute__((aligned(16))) int32_t lds[];  // cosines, sines, a row per lane group
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const uint32_t per_wave = 64 / lanes, li = lane % lanes, hd = a.hd, pairs = a.pairs;
  const uint64_t t = blockIdx.x;
  int32_t* cs = lds;
  int32_t* sn = lds + ((pairs + 3) & ~3u);
  int32_t* row = lds + 2 * ((pairs + 3) & ~3u) + (wave * per_wave + lane / lanes) * ((hd + 3) & ~3u);
  if (pairs) {
    const uint64_t pos = a.positions[t];
    for (uint32_t i = tid; i < pairs; i += blockDim.x) {
      int32_t c, s;
      sin_cos(rope_angle(pos, a.freq[i]), &c, &s);
      cs[i] = a.amplitude == kOneAct ? c : mul_sat(c, a.amplitude);
      sn[i] = a.amplitude == kOneAct ? s : mul_sat(s, a.amplitude);
    }
    __syncthreads();
  }
  for (uint32_t r0 = wave * per_wave; r0 < a.total; r0 += waves * per_wave) {
    const uint32_t r = r0 + lane / lanes;
    const bool on = r < a.total;
    // the row's set and head
    uint32_t h = on ? r : 0;
    HeadSet s = a.set[0];
#pragma unroll
    for (uint32_t q = 1; q < kHeadSets; ++q)
      if (q < a.n_sets && h >= s.heads) {
        h -= s.heads;
        s = a.set[q];
      }
    const int32_t* src = s.x + t * s.ld + uint64_t(h) * hd;
    int32_t* dst = s.out + t * s.out_ld + uint64_t(h) * hd;
    int32_t x[E][V];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t c = V * (li + 64 * e);
#pragma unroll
      for (int v = 0; v < V; ++v) x[e][v] = 0;
      if (on && c < hd) Vec<V>::load(src + c, x[e]);
    }
    if (s.flags & 1) {
      // (non-negative terms: the saturating sum is the least of the sum and i64::MAX in any order)
      int64_t ss = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int v = 0; v < V; ++v) ss = add_sat64_nn(ss, sq_term(x[e][v]));
      for (uint32_t off = 1; off < lanes; off <<= 1) ss = add_sat64_nn(ss, __shfl_xor(ss, int(off), 64));
      const int32_t scale = rms_scale_from_sumsq(ss, hd, a.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
        if (c >= hd) continue;
        int32_t g[V];
        if (s.gain) Vec<V>::load(s.gain + c, g);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          x[e][v] = mul_sat(x[e][v], scale);
          if (s.gain) x[e][v] = mul_sat(x[e][v], g[v]);
        }
      }
    }
    if (pairs && __any(s.flags & 2)) {
      wave_lds_sync();  // the previous rows have been read
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
        if (c < hd) Vec<V>::store(row + c, x[e]);
      }
      wave_lds_sync();
      if (s.flags & 2) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const uint32_t c = V * (li + 64 * e) + v;
            if (c >= 2 * pairs) continue;
            const bool second = a.interleaved ? (c & 1) : c >= pairs;
            const uint32_t i = a.interleaved ? c >> 1 : (second ? c - pairs : c);
            const int32_t other = row[a.interleaved ? (c ^ 1) : (second ? c - pairs : c + pairs)];
            const int32_t p = mul_sat(x[e][v], cs[i]), q = mul_sat(other, sn[i]);
            x[e][v] = second ? add_sat(p, q) : sub_sat(p, q);
          }
      }
    }
    if (on)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
        if (c < hd) Vec<V>::store(dst + c, x[e]);
      }
  }
}

template <int V, int E>
void launch(const HeadRopeArgs& a, hipStream_t s) {
  uint32_t lanes = 64;
  if (E == 1)
    while (lanes > 1 && lanes / 2 * V >= a.hd) lanes /= 2;
  const uint32_t per_wave = 64 / lanes;
  uint32_t waves = (a.total + per_wave - 1) / per_wave;
  if (waves > 4) waves = 4;
  if (waves < 2 && a.pairs > 64) waves = 2;
  const size_t bytes = (2 * ((a.pairs + 3) & ~3u) + waves * per_wave * ((a.hd + 3) & ~3u)) * 4;
  hipLaunchKernelGGL((k_head_rope<V, E>), dim3(unsigned(a.rows)), dim3(64 * waves), bytes, s, a, lanes);
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
    if (a.hd <= 256) launch<4, 1>(a, s);
    else if (a.hd <= 512) launch<4, 2>(a, s);
    else launch<4, 4>(a, s);
  } else {
    if (a.hd <= 64) launch<1, 1>(a, s);
    else if (a.hd <= 256) launch<1, 4>(a, s);
    else launch<1, 16>(a, s);
  }
}

}  // namespace det
