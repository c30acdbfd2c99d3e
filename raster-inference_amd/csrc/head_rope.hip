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

// round(a b 2^16) 2^-16 for |a b| below 2^35 (mul_rint at a unit of 2^-16).
__device__ __forceinline__ double mul_rint16(double a, double b) {
  constexpr double kWhole = 103079215104.0;  // 1.5 2^36
  return __builtin_fma(a, b, kWhole) - kWhole;
}
// round(a b) where it is an i32: the low word of the sum with 1.5 2^52 (one
// multiply-add, no conversion).
__device__ __forceinline__ int32_t mul_word(double a, double b) {
  return int32_t(uint32_t(__builtin_bit_cast(uint64_t, __builtin_fma(a, b, 6755399441055744.0))));
}
// a c - b s or b c + a s of one rotated value (s with its sign): each product
// rounded and saturated, then the sum.
__device__ __forceinline__ int32_t turned(int32_t x, int32_t other, double c, double s, bool second) {
  const int32_t p = to_i32(mul_rint(double(x), c)), q = to_i32(mul_rint(double(other), second ? s : -s));
  return second ? __builtin_elementwise_add_sat(p, q) : __builtin_elementwise_sub_sat(p, q);
}
// The same for |x|, |other| <= 2^30 and |c|, |s| < 2: both products are i32.
__device__ __forceinline__ int32_t turned_small(int32_t x, int32_t other, double c, double s) {
  return __builtin_elementwise_add_sat(mul_word(double(x), c), mul_word(double(other), s));
}

// Wave totals of four values at once: lane l ends with the total of value l % 4
// (two halvings that keep one of two values per lane, then four whole steps: 40
// instructions against 24 per value alone).
__device__ __forceinline__ uint64_t add_rows16(uint64_t v) {
  const auto lo = __builtin_amdgcn_permlane16_swap(uint32_t(v), uint32_t(v), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(uint32_t(v >> 32), uint32_t(v >> 32), false, false);
  return ((uint64_t(hi[0]) << 32) | lo[0]) + ((uint64_t(hi[1]) << 32) | lo[1]);
}
__device__ __forceinline__ uint64_t add_rows32(uint64_t v) {
  const auto lo = __builtin_amdgcn_permlane32_swap(uint32_t(v), uint32_t(v), false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap(uint32_t(v >> 32), uint32_t(v >> 32), false, false);
  return ((uint64_t(hi[0]) << 32) | lo[0]) + ((uint64_t(hi[1]) << 32) | lo[1]);
}
__device__ __forceinline__ uint64_t wave_sum4(uint64_t a, uint64_t b, uint64_t c, uint64_t d, uint32_t lane) {
  const bool o1 = lane & 1, o2 = lane & 2;
  const uint64_t ab = (o1 ? b : a) + dpp_move64<0xb1>(o1 ? a : b), cd = (o1 ? d : c) + dpp_move64<0xb1>(o1 ? c : d);
  uint64_t v = (o2 ? cd : ab) + dpp_move64<0x4e>(o2 ? ab : cd);
  v += dpp_move64<0x124>(v);
  v += dpp_move64<0x128>(v);
  return add_rows32(add_rows16(v));
}

// rms_scale_from_sumsq; a power of two divides by a shift (about 100
// instructions fewer).
__device__ __forceinline__ int32_t norm_scale(int64_t sum, uint32_t hd, int64_t eps) {
  if (hd & (hd - 1)) return rms_scale_from_sumsq(sum, hd, eps);
  const uint64_t s = uint64_t(sum), q = s >> __builtin_ctz(hd), twice = (s & (hd - 1)) << 1;
  return inv_sqrt_acc(add_sat64(int64_t(q + (twice > hd || (twice == hd && (q & 1)))), eps));
}

// One workgroup per token: its threads compute the token's cosines and sines
// once into LDS, then each group of `lanes` lanes takes up to U head rows at a
// time, V consecutive values per lane and step, E steps; the first rows' loads
// are on their way while the cosines are computed. A pair of the half layout
// meets through the rows' LDS copies, an interleaved pair in one lane (V = 4) or
// through them as well. WAVE: a wave per row (the rows' pointers are scalar).
// Bound by its instructions at many tokens, then by the bytes, so the products are
// double multiply-adds whose low words are the rounded results (one instruction
// against 11 for one of 64-bit integers) wherever nothing can saturate, which the
// wave sees from the values; otherwise its rows are read again and clamped. 4096
// tokens of 12 heads of 256: 31 us (35 from cold memory), a copy of the same 50 MB
// takes 21; 39 with saturating products throughout. Four waves per SIMD at five
// spilled registers are worth more than three without (31 against 35), and U = 6 in
// two waves or 12 in one (fewer scales, more registers) took 32 and 35.
template <int V, int E, int U, bool WAVE>
__global__ __launch_bounds__(256, WAVE && U * E * V <= 12 ? 4 : 1) void k_head_rope(HeadRopeArgs a, uint32_t lane_group) {
  extern __shared__ __attribute__((aligned(16))) double table[];  // cosines, sines (times 2^-16), G rows per lane group
  constexpr int G = U < 4 ? U : 4;
  const uint32_t tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), lanes = WAVE ? 64 : lane_group;
  const uint32_t per_wave = 64 / lanes, li = lane % lanes, hd = a.hd, pairs = a.pairs;
  const uint32_t entries = (pairs + 3) & ~3u, row_ld = (hd + 3) & ~3u;
  const uint64_t t = blockIdx.x;
  double* cs = table;
  double* sn = table + entries;
  int32_t* row = reinterpret_cast<int32_t*>(table + 2 * entries) + (wave * per_wave + lane / lanes) * G * row_ld;
  const bool grouped = V == 4 && pairs % (a.interleaved ? 2 : 4) == 0;
  const bool meet = !(grouped && a.interleaved);  // pairs meet in LDS
  const uint32_t step = waves * per_wave, first = wave * per_wave;
  for (uint32_t r0 = first;; r0 += step * U) {
    if (r0 != first && r0 >= a.total) break;
    // the rows' sets and heads, their values
    const auto find = [&](int u, uint32_t* head) {
      const uint32_t r = r0 + u * step + (WAVE ? 0 : lane / lanes);
      uint32_t h = r < a.total ? r : 0, k = 0;
#pragma unroll
      for (uint32_t q = 0; q + 1 < kHeadSets; ++q)
        if (k == q && h >= a.set[q].heads) {
          h -= a.set[q].heads;
          ++k;
        }
      *head = h;
      return k;
    };
    const auto on = [&](int u) { return r0 + u * step + (WAVE ? 0 : lane / lanes) < a.total; };
    int32_t x[U][E][V];
    uint32_t flags[U];
    const auto load = [&]() {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t h;
        const HeadSet& s = a.set[find(u, &h)];
        flags[u] = s.flags;
        const int32_t* src = s.x + t * s.ld + uint64_t(h) * hd;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t c = V * (li + 64 * e);
#pragma unroll
          for (int v = 0; v < V; ++v) x[u][e][v] = 0;
          if (on(u) && c < hd) Vec<V>::load(src + c, x[u][e]);
        }
      }
    };
    const auto load_gain = [&](int u, int32_t(*g)[V]) {
      uint32_t h;
      const int32_t* gain = a.set[find(u, &h)].gain;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
#pragma unroll
        for (int v = 0; v < V; ++v) g[e][v] = kOneAct;
        if (gain && c < hd) Vec<V>::load(gain + c, g[e]);
      }
    };
    load();
    int32_t g[2][E][V];
    load_gain(0, g[0]);
    if (r0 == first && pairs) {
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
    bool small = !__any(large >> 26);
    int64_t ss[U] = {};
    int64_t mine = 0;  // (a wave's U rows: lane u finds the scale of row u)
    if (small) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) ss[u] += sq_term(x[u][e][v]);
      if (WAVE) {
#pragma unroll
        for (int u = 0; u < U; u += 4) {
          const int64_t sum = int64_t(wave_sum4(ss[u], u + 1 < U ? ss[u + 1] : 0, u + 2 < U ? ss[u + 2] : 0, u + 3 < U ? ss[u + 3] : 0, lane));
          mine = int(lane / 4) == u / 4 ? sum : mine;
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
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
        mine = int(lane) == u ? ss[u] : mine;
      }
    }
    int32_t scale[U];
    if (WAVE) {
      const int32_t found = norm_scale(mine, hd, a.eps);
      small = small && !__any(int(lane) < U && found >> 21);
#pragma unroll
      for (int u = 0; u < U; ++u) scale[u] = __builtin_amdgcn_readlane(found, u);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        scale[u] = norm_scale(ss[u], hd, a.eps);
        small = small && !__any(scale[u] >> 21);
      }
    }
    // Values below 2^26 times scales below 2^21 stay below 2^31. Their products
    // with the gain are taken 2^30 up: the high word then is 1.5 2^52's and the low
    // word below 2^31 exactly for a result in [-2^30, 2^30), which one
    // conjunction over all of them shows.
    if (small) {
      constexpr double kUp = 6755399441055744.0 + 1073741824.0;
      constexpr uint32_t kHigh = 0x43380000;
      uint32_t high = kHigh, low = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u + 1 < U) load_gain(u + 1, g[(u + 1) & 1]);
        if (flags[u] & 1) {
          const double by = double(scale[u]) * 0x1p-32;
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const uint64_t y = __builtin_bit_cast(
                  uint64_t, __builtin_fma(mul_rint16(double(x[u][e][v]), by), double(g[u & 1][e][v]), kUp));
              high |= uint32_t(y >> 32);
              low |= uint32_t(y);
              x[u][e][v] = int32_t(uint32_t(y) - (1u << 30));
            }
        }
      }
      small = !__any(high != kHigh || low >> 31);
      if (!small) load();
    }
    if (!small) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!(flags[u] & 1)) continue;
        load_gain(u, g[0]);
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const double y = mul_rint16(double(x[u][e][v]), double(scale[u]) * 0x1p-32);
            const double z = __builtin_fmin(__builtin_fmax(y, -32768.0), 2147483647.0 / 65536.0);
            x[u][e][v] = to_i32(mul_rint(z, double(g[0][e][v])));
          }
      }
    }
    // (rows without a norm: values below 2^26 are below 2^30)
    small = small && uint32_t(a.amplitude) < 2u << 16;
    if (pairs) {
#pragma unroll
      for (int u0 = 0; u0 < U; u0 += G) {
        if (meet) {
          wave_lds_sync();  // the previous rows have been read
#pragma unroll
          for (int u = u0; u < u0 + G && u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const uint32_t c = V * (li + 64 * e);
              if (c < hd) Vec<V>::store(row + (u - u0) * row_ld + c, x[u][e]);
            }
          wave_lds_sync();
        }
        if (grouped && small) {
          // a lane's four values belong to one half, or are two pairs
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const uint32_t c = V * (li + 64 * e);
            double cv[4] = {1, 1, 1, 1}, sv[4] = {};  // behind the rotated part
            const bool second = c >= pairs;
            if (c < 2 * pairs) {
              if (a.interleaved) {
                const double2 c2 = *reinterpret_cast<const double2*>(cs + c / 2), s2 = *reinterpret_cast<const double2*>(sn + c / 2);
                cv[0] = cv[1] = c2.x, cv[2] = cv[3] = c2.y;
                sv[0] = -s2.x, sv[1] = s2.x, sv[2] = -s2.y, sv[3] = s2.y;
              } else {
                const uint32_t i = second ? c - pairs : c;
#pragma unroll
                for (int v = 0; v < 4; ++v) cv[v] = cs[i + v], sv[v] = second ? sn[i + v] : -sn[i + v];
              }
            }
            const uint32_t meets = c >= 2 * pairs ? 0 : (second ? c - pairs : c + pairs);
#pragma unroll
            for (int u = u0; u < u0 + G && u < U; ++u) {
              if (!(flags[u] & 2)) continue;
              int32_t other[V];
              if (a.interleaved) {
#pragma unroll
                for (int v = 0; v < V; ++v) other[v] = x[u][e][v ^ (V > 1)];
              } else {
                Vec<V>::load(row + (u - u0) * row_ld + meets, other);
              }
#pragma unroll
              for (int v = 0; v < V; ++v) x[u][e][v] = turned_small(x[u][e][v], other[v], cv[v & 3], sv[v & 3]);
            }
          }
        } else {
#pragma unroll
          for (int u = u0; u < u0 + G && u < U; ++u) {
            if (!(flags[u] & 2)) continue;
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
                const int32_t other = meet ? row[(u - u0) * row_ld + (a.interleaved ? (c ^ 1) : (second ? c - pairs : c + pairs))]
                                           : x[u][e][v ^ (V > 1)];
                y[v] = turned(x[u][e][v], other, cs[i], second ? sn[i] : -sn[i], second);
              }
#pragma unroll
              for (int v = 0; v < V; ++v) x[u][e][v] = y[v];
            }
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t h;
      const HeadSet& s = a.set[find(u, &h)];
      int32_t* dst = s.out + t * s.out_ld + uint64_t(h) * hd;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = V * (li + 64 * e);
        if (on(u) && c < hd) Vec<V>::store(dst + c, x[u][e]);
      }
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
  const size_t bytes = (4 * ((a.pairs + 3) & ~3u) + waves * per_wave * std::min(U, 4) * ((a.hd + 3) & ~3u)) * 4;
  const dim3 grid(unsigned(a.rows)), block(64 * waves);
  if (lanes == 64) hipLaunchKernelGGL((k_head_rope<V, E, U, true>), grid, block, bytes, s, a, lanes);
  else if constexpr (E == 1) hipLaunchKernelGGL((k_head_rope<V, E, U, false>), grid, block, bytes, s, a, lanes);
}

}  // namespace

// (tokens in ranges: a grid has less than 2^32 threads)
constexpr uint64_t kRange = uint64_t(1) << 22;
static void launch_range(const HeadRopeArgs& a, hipStream_t s) {
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
void launch_head_rope(const HeadRopeArgs& a, hipStream_t s) {
  if (a.total == 0) return;
  HeadRopeArgs r = a;
  for (uint64_t t = 0; t < a.rows; t += kRange) {
    r.rows = std::min(a.rows - t, kRange);
    if (a.positions) r.positions = a.positions + t;
    for (uint32_t i = 0; i < a.n_sets; ++i) {
      r.set[i].x = a.set[i].x + t * a.set[i].ld;
      r.set[i].out = a.set[i].out + t * a.set[i].out_ld;
    }
    launch_range(r, s);
  }
}

}  // namespace det
