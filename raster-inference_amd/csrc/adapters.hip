// Low-rank adapters of many requests beside a shared projection:
// out[t] = add_sat(out[t], scale_act(B (A x_t), scale)) with the adapter of
// row t, both products requantized (out holds W x on entry).
//
// The rows are grouped by adapter into tiles of 16 rows that share one, so that
// each adapter's matrices are read once per tile:
//   k_adapter_sort  the tiles of more than 64 rows (fewer rows: every workgroup
//                   finds its tile itself, which costs less than a launch)
//   k_adapter_down  A x of a tile on int8 MFMA, K in chunks over the grid ->
//                   wrapping int64 partial sums
//   k_adapter_up    the partial sums joined and requantized to h, B h on int8
//                   MFMA, the scaled result added to the rows
// Activations and h are taken apart into balanced base-256 digits, x = sum
// 256^j c_j with c_0 .. c_3 the signed bytes of (x + 0x80808080) ^ 0x80808080
// and c_4 = 1 for x > 0x7f7f7f7f; digits 3 and 4 are zero for |x| < 128.0, and
// the products with them are left out where a whole step has none. Weights of P
// digit planes take P products per digit; digit j and plane p add to the int32
// sum j + p (at most four pairs of 128 x 128 over 8192 columns).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "det_arith.h"
#include "verify.h"
#include "wave.h"

namespace det {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
constexpr uint32_t kOp = 1024;       // one MFMA operand: 64 lanes x 16 bytes
constexpr uint32_t kNoRow = ~0u;
constexpr uint32_t kSmallRows = 64;  // rows whose tiles every workgroup finds itself
constexpr uint32_t kStepCols = 256;  // columns per step of A x

struct Plan {
  AdapterArgs a;
  uint32_t tiles;      // most tiles
  uint32_t chunk, chunks;  // steps of kStepCols per chunk of K
  uint32_t ranks;      // values per row of the partial sums (max_rank)
  uint32_t up_tiles;   // 16-row tiles of B per workgroup of B h
  int vec;             // 16-byte aligned activation rows
  int out4;            // 16-byte aligned output rows
  int64_t* planes;     // [chunk][16 tile + row][ranks]
  uint32_t* tile_of;   // [tile]: adapter (more than kSmallRows rows)
  uint32_t* perm;      // [16 tile + row]: row of the call, kNoRow where none
  uint32_t* n_tiles;
};

// Parts into which a group of up to 64 rank rows splits the steps: its four
// waves take one 16-row tile each, or share one or two.
__device__ inline uint32_t tile_waves(uint32_t rank_tiles) { return rank_tiles == 1 ? 1 : rank_tiles == 2 ? 2 : 4; }

// Tile `k` of the call: its adapter (kNoRow past the last tile) and rows.
struct Tile {
  uint32_t adapter;
  uint32_t row[16];
};
__device__ inline void find_tile(const Plan& p, uint32_t k, Tile& t) {
  const uint32_t tid = threadIdx.x;
  if (p.a.m > kSmallRows) {
    if (tid == 0) t.adapter = k < *p.n_tiles ? p.tile_of[k] : kNoRow;
    if (tid < 16) t.row[tid] = p.perm[uint64_t(k) * 16 + tid];
  } else if (tid < 64) {
    if (tid < 16) t.row[tid] = kNoRow;
    if (tid == 0) t.adapter = kNoRow;
    const uint32_t v = tid < p.a.m ? p.a.index[tid] : kNoRow;
    uint64_t left = __ballot(v < p.a.n);
    wave_lds_sync();
    while (left) {
      const uint32_t a = __builtin_amdgcn_readlane(v, int(__builtin_ctzll(left)));
      const uint64_t same = __ballot(v == a);
      const uint32_t n = (__popcll(same) + 15) / 16;
      if (k < n) {
        const uint32_t at = __popcll(same & ((1ull << tid) - 1));
        if (v == a && at / 16 == k) t.row[at % 16] = tid;
        if (tid == 0) t.adapter = a;
        break;
      }
      k -= n;
      left &= ~same;
    }
  }
  __syncthreads();
}

// One workgroup: rows by adapter, each adapter's run filled up to whole tiles.
constexpr uint32_t kSortThreads = 1024;
__global__ __launch_bounds__(kSortThreads) void k_adapter_sort(Plan p) {
  __shared__ uint32_t count[kAdapterMost];  // then each adapter's next slot
  __shared__ uint32_t part[kSortThreads];
  const uint32_t tid = threadIdx.x, n = p.a.n;
  for (uint32_t i = tid; i < n; i += kSortThreads) count[i] = 0;
  __syncthreads();
  for (uint64_t t = tid; t < p.a.m; t += kSortThreads) {
    const uint32_t v = p.a.index[t];
    if (v < n) atomicAdd(&count[v], 1u);
  }
  __syncthreads();
  // tiles before each adapter: a run of adapters per thread, then the threads
  const uint32_t per = (n + kSortThreads - 1) / kSortThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
  uint32_t mine = 0;
  for (uint32_t i = i0; i < i1; ++i) mine += (count[i] + 15) / 16;
  part[tid] = mine;
  __syncthreads();
  for (uint32_t o = 1; o < kSortThreads; o <<= 1) {
    const uint32_t v = tid >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] += v;
    __syncthreads();
  }
  uint32_t tile = part[tid] - mine;
  for (uint32_t i = i0; i < i1; ++i) {
    const uint32_t c = count[i], e = tile + (c + 15) / 16;
    for (uint32_t k = 16 * tile + c; k < 16 * e; ++k) p.perm[k] = kNoRow;
    count[i] = 16 * tile;
    for (; tile < e; ++tile) p.tile_of[tile] = i;
  }
  if (tid == kSortThreads - 1) *p.n_tiles = part[tid];
  __syncthreads();
  for (uint64_t t = tid; t < p.a.m; t += kSortThreads) {
    const uint32_t v = p.a.index[t];
    if (v < n) p.perm[atomicAdd(&count[v], 1u)] = uint32_t(t);
  }
}

// Digits of 16 values in operand order: word q of digit j holds values 4 q ..
// 4 q + 3; returns whether a digit 3 or 4 is set.
__device__ __forceinline__ bool digits16(const int32_t (&x)[16], v4i (&d)[5]) {
  uint32_t any = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t u[4], t = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = (uint32_t(x[4 * q + e]) + 0x80808080u) ^ 0x80808080u;
      t |= uint32_t(x[4 * q + e] > 0x7f7f7f7f) << (8 * e);
    }
    const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u), e = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
    d[0][q] = int(__builtin_amdgcn_perm(b, a, 0x05040100u));
    d[1][q] = int(__builtin_amdgcn_perm(b, a, 0x07060302u));
    d[2][q] = int(__builtin_amdgcn_perm(e, c, 0x05040100u));
    d[3][q] = int(__builtin_amdgcn_perm(e, c, 0x07060302u));
    d[4][q] = int(t);
    any |= uint32_t(d[3][q]) | t;
  }
  return any != 0;
}

// acc[j + q] += (plane q of the weights) x (digit j of the rows)
template <int P>
__device__ __forceinline__ void multiply(const v4i (&w)[P], const v4i* digits, uint32_t l, bool wide, v4i (&acc)[8]) {
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    const v4i x = digits[j * 64 + l];
#pragma unroll
    for (int q = 0; q < P; ++q) acc[j + q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[q], x, acc[j + q], 0, 0, 0);
  }
  if (wide)
#pragma unroll
    for (int j = 3; j < 5; ++j) {
      const v4i x = digits[j * 64 + l];
#pragma unroll
      for (int q = 0; q < P; ++q) acc[j + q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[q], x, acc[j + q], 0, 0, 0);
    }
}
// The sum of component r.
__device__ __forceinline__ int64_t total(const v4i (&acc)[8], int r) {
  uint64_t y = 0;
#pragma unroll
  for (int s = 0; s < 8; ++s) y += uint64_t(int64_t(acc[s][r])) << (8 * s);
  return int64_t(y);
}

// requant(sum times by) of one component where the digits j have 0 .. 2 only, as
// the whole double that it is: sums below 2^52 times scales are one rounded
// multiply-add (the products of the integer form stay below 2^62, so that nothing
// has wrapped there either). About 12 instructions against 40.
template <int P>
__device__ __forceinline__ double scaled(const v4i (&acc)[8], int r, int32_t by, bool& far) {
  // (from the top: a partial sum past 2^53 leaves the whole one past 2^52)
  double y = 0;
#pragma unroll
  for (int s = P + 1; s >= 0; --s) y = __builtin_fma(y, 256.0, double(acc[s][r]));
  const double b = double(by);
  far = far || !(__builtin_fabs(y) < 4503599627370496.0) || !(__builtin_fabs(y * b) < 4611686018427387904.0);
  return mul_rint(y, b * 0x1p-16);
}

// A x of one tile, one chunk of K and up to 64 rank rows. Per step of 256
// columns each wave takes its 64 columns of the rows apart into LDS (the
// weights' tile-steps: half h of step s, lane 16 g + i, holds columns 128 s +
// 32 g + 16 h .. of row i); then wave w multiplies its rank tile with all of
// them or its share. The next step's activations are on their way meanwhile. One
// row of 2560 columns 4.2 us (latency), 1024 rows of 10240 columns and rank 64 in 16
// bits 22.5 us, where the rows' 42 MB take 8.5 at a copy's rate: bound by the digits'
// conversion and the LDS reads, four products per operand.
template <int P>
__device__ __forceinline__ void down_steps(const Plan& p, const DevAdapter& ad, const Tile& t, int8_t* lds,
                                           uint32_t* wide, uint32_t rank_tile, uint32_t part, uint32_t parts, bool on,
                                           v4i (&acc)[8]) {
  const uint32_t tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = l & 15, g = l >> 4;
  const uint64_t steps = p.a.kpad / 128, c_end = p.a.cols;
  const uint32_t s0 = blockIdx.y * p.chunk, s1 = min(s0 + p.chunk, uint32_t((p.a.kpad + kStepCols - 1) / kStepCols));
  const uint32_t row = t.row[i] == kNoRow ? t.row[0] : t.row[i];
  const int32_t* src = p.a.act + uint64_t(row) * p.a.cols;
  const uint32_t col = 128 * (wave >> 1) + 32 * g + 16 * (wave & 1);
  auto load = [&](uint32_t s, int32_t (&x)[16]) {
    // (columns past the end have zero weights)
    const uint64_t c = uint64_t(s) * kStepCols + col;
    if (p.vec) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int4 v = load_int4(to_global(src) + min(c + 4 * q, c_end - 4));
        x[4 * q] = v.x, x[4 * q + 1] = v.y, x[4 * q + 2] = v.z, x[4 * q + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = to_global(src)[min(c + e, c_end - 1)];
    }
  };
  int32_t x[16];
  load(s0, x);
  for (uint32_t s = s0, buf = 0; s < s1; ++s, buf ^= 1) {
    v4i* dst = reinterpret_cast<v4i*>(lds) + (buf * 4 + wave) * 5 * 64 + l;
    v4i d[5];
    const bool any = __any(digits16(x, d));
#pragma unroll
    for (int j = 0; j < 5; ++j) dst[j * 64] = d[j];
    if (l == 0) wide[buf * 4 + wave] = any;
    if (s + 1 < s1) load(s + 1, x);
    lds_barrier();
    if (on)
      for (uint32_t u = part; u < 4; u += parts) {
        const uint64_t step = uint64_t(s) * 2 + (u >> 1);
        if (step >= steps) break;
        v4i w[P];
#pragma unroll
        for (int q = 0; q < P; ++q)
          w[q] = *reinterpret_cast<const v4i*>(ad.a + ((uint64_t(rank_tile) * P + q) * steps + step) * 2048 +
                                               (u & 1) * kTileHalfBytes + l * 16);
        multiply<P>(w, reinterpret_cast<const v4i*>(lds) + (buf * 4 + u) * 5 * 64, l, wide[buf * 4 + u] != 0, acc);
      }
  }
}
__global__ __launch_bounds__(256) void k_adapter_down(Plan p) {
  __shared__ __attribute__((aligned(16))) int8_t lds[2 * 4 * 5 * kOp];
  __shared__ uint32_t wide[8];
  __shared__ Tile t;
  find_tile(p, blockIdx.x, t);
  if (t.adapter == kNoRow) return;
  const DevAdapter ad = p.a.set[t.adapter];
  const uint32_t first = blockIdx.z * 4, all = (ad.rank + 15) / 16;  // rank tiles
  if (first >= all) return;
  const uint32_t tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tiles = min(all - first, 4u), waves = tile_waves(tiles), parts = 4 / waves;
  const uint32_t rank_tile = first + wave % waves, part = wave / waves;
  const bool on = wave % waves < tiles;
  v4i acc[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) acc[s] = v4i{0, 0, 0, 0};
  const uint32_t at = on ? rank_tile : first;
  if (ad.a_planes == 1) down_steps<1>(p, ad, t, lds, wide, at, part, parts, on, acc);
  else if (ad.a_planes == 2) down_steps<2>(p, ad, t, lds, wide, at, part, parts, on, acc);
  else down_steps<4>(p, ad, t, lds, wide, at, part, parts, on, acc);
  // lane l, component r: rank row 16 rank_tile + 4 (l >> 4) + r of row l & 15;
  // the first part's wave adds the others' shares
  int64_t y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = total(acc, r);
  if (parts > 1) {
    int64_t* share = reinterpret_cast<int64_t*>(lds);  // [wave][component][lane]
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) share[(wave * 4 + r) * 64 + l] = y[r];
    __syncthreads();
    if (part) return;
    for (uint32_t w = wave + waves; w < 4; w += waves)
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = int64_t(uint64_t(y[r]) + uint64_t(share[(w * 4 + r) * 64 + l]));
  }
  if (!on || t.row[l & 15] == kNoRow) return;
  int64_t* o = p.planes + ((uint64_t(blockIdx.y) * p.tiles + blockIdx.x) * 16 + (l & 15)) * p.ranks + 16 * rank_tile +
               4 * (l >> 4);
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = y[r];
}

// h of one tile: its chunks' sums, a value per thread, then their digits, 16
// values per thread (one operand lane).
__device__ __forceinline__ void rank_rows(const Plan& p, const DevAdapter& ad, const Tile& t, int8_t* lds, uint32_t* wide) {
  const uint32_t tid = threadIdx.x, subs = (ad.kg + 3) / 4, ranks = 64 * subs;
  int32_t* hs = reinterpret_cast<int32_t*>(lds + subs * 5 * kOp);  // [row][ranks]
  for (uint32_t u = tid; u < 16 * 16 * ad.kg; u += 256) {
    const uint32_t i = u / (16 * ad.kg), k = u % (16 * ad.kg);
    int32_t h = 0;
    if (k < ad.rank && t.row[i] != kNoRow) {
      const int64_t* src = p.planes + (uint64_t(blockIdx.x) * 16 + i) * p.ranks + k;
      const uint64_t ld = uint64_t(p.tiles) * 16 * p.ranks;
      uint64_t y = 0;
      uint32_t c = 0;
      for (; c + 8 <= p.chunks; c += 8) {
        uint64_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = uint64_t(src[(c + e) * ld]);
#pragma unroll
        for (int e = 0; e < 8; ++e) y += v[e];
      }
      for (; c < p.chunks; ++c) y += uint64_t(src[c * ld]);
      h = requant(int64_t(y * uint64_t(int64_t(ad.a_scale[k]))));
    }
    hs[i * ranks + k] = h;
  }
  lds_barrier();
  for (uint32_t u = tid; u < subs * 64; u += 256) {
    const int4* src = reinterpret_cast<const int4*>(hs + (u & 15) * ranks + 16 * (u >> 4));
    int32_t h[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int4 v = (u >> 4) < ad.kg ? src[q] : make_int4(0, 0, 0, 0);
      h[4 * q] = v.x, h[4 * q + 1] = v.y, h[4 * q + 2] = v.z, h[4 * q + 3] = v.w;
    }
    v4i d[5];
    if (digits16(h, d)) *wide = 1;
    v4i* dst = reinterpret_cast<v4i*>(lds) + (u >> 6) * 5 * 64 + (u & 63);
#pragma unroll
    for (int j = 0; j < 5; ++j) dst[j * 64] = d[j];
  }
  lds_barrier();
}
// B h of one tile and p.up_tiles 16-row tiles of B, round the four waves. What
// the first 64 rank rows take from memory is loaded a tile ahead, for the first
// tile while h is made.
template <int P>
__device__ __forceinline__ void up_tiles(const Plan& p, const DevAdapter& ad, const Tile& t, int8_t* lds, uint32_t* wide_h) {
  const uint32_t l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = l & 15, g = l >> 4;
  const uint32_t subs = (ad.kg + 3) / 4, row = t.row[i];
  const uint64_t tiles = (p.a.rows + 15) / 16, end = min(uint64_t(blockIdx.y + 1) * p.up_tiles, tiles);
  int32_t* out = p.a.out + uint64_t(row == kNoRow ? 0 : row) * p.a.rows;
  auto weights = [&](uint64_t T, uint32_t s, v4i (&w)[P]) {
#pragma unroll
    for (int q = 0; q < P; ++q)
      w[q] = 4 * s + g < ad.kg ? *reinterpret_cast<const v4i*>(ad.b + ((T * P + q) * ad.kg + 4 * s + g) * 256 + i * 16)
                               : v4i{0, 0, 0, 0};
  };
  v4i w[P];
  int4 scale, old;
  auto load = [&](uint64_t T) {  // lane l, component r: output 16 T + 4 g + r of row i
    const uint64_t n = 16 * T + 4 * g;
    weights(T, 0, w);
    scale = *reinterpret_cast<const int4*>(ad.b_scale + n);  // (b_scale holds whole tiles)
    if (p.out4 && row != kNoRow && n < p.a.rows) old = *reinterpret_cast<const int4*>(out + n);
  };
  uint64_t T = uint64_t(blockIdx.y) * p.up_tiles + wave;
  if (T < end) load(T);
  rank_rows(p, ad, t, lds, wide_h);
  const v4i* digits = reinterpret_cast<const v4i*>(lds);
  const bool wide = *wide_h != 0;
  const double by_all = double(ad.scale) * 0x1p-16;
#pragma unroll 1
  for (; T < end; T += 4) {
    v4i acc[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) acc[s] = v4i{0, 0, 0, 0};
    uint32_t s = 0;
    do {
      if (s) weights(T, s, w);
      multiply<P>(w, digits + s * 5 * 64, l, wide, acc);
    } while (++s < subs);
    const int32_t by[4] = {scale.x, scale.y, scale.z, scale.w}, was[4] = {old.x, old.y, old.z, old.w};
    if (T + 4 < end) load(T + 4);
    const uint64_t n = 16 * T + 4 * g;
    if (row == kNoRow || n >= p.a.rows) continue;
    int32_t y[4];
    bool far = wide;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = to_i32(mul_rint(double(to_i32(scaled<P>(acc, r, by[r], far))), by_all));
    if (__any(far)) {
#pragma unroll
      for (int s = 0; s < 8; ++s) asm volatile("" : "+v"(acc[s]));  // (a branch in earnest)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        y[r] = mul_sat(requant(int64_t(uint64_t(total(acc, r)) * uint64_t(int64_t(by[r])))), ad.scale);
    }
    if (p.out4) {
      *reinterpret_cast<int4*>(out + n) =
          make_int4(add_sat(was[0], y[0]), add_sat(was[1], y[1]), add_sat(was[2], y[2]), add_sat(was[3], y[3]));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.a.rows) out[n + r] = add_sat(out[n + r], y[r]);
    }
  }
}
__global__ __launch_bounds__(256) void k_adapter_up(Plan p) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];  // digits of h: [64 rank rows][digit][lane], then h
  __shared__ uint32_t wide;
  __shared__ Tile t;
  if (threadIdx.x == 0) wide = 0;
  find_tile(p, blockIdx.x, t);
  if (t.adapter == kNoRow) return;
  const DevAdapter ad = p.a.set[t.adapter];
  if (ad.b_planes == 1) up_tiles<1>(p, ad, t, lds, &wide);
  else if (ad.b_planes == 2) up_tiles<2>(p, ad, t, lds, &wide);
  else up_tiles<4>(p, ad, t, lds, &wide);
}

uint64_t up(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

uint64_t plan(const AdapterArgs& a, Plan& p) {
  p = Plan{};
  p.a = a;
  p.ranks = a.max_rank;
  // an adapter's last tile may be partly filled
  p.tiles = uint32_t(std::min<uint64_t>(a.m, a.m / 16 + std::min<uint64_t>(a.n, a.m)));
  // chunks of K until the full tiles fill the device
  const uint32_t steps = uint32_t((a.kpad + kStepCols - 1) / kStepCols);
  const uint64_t full = (a.m + 15) / 16 * ((a.max_rank + 63) / 64);
  p.chunk = uint32_t(std::min<uint64_t>(std::max<uint64_t>(full * steps / 512, 1), 8192 / kStepCols));
  p.chunks = (steps + p.chunk - 1) / p.chunk;
  // of B's tiles one per wave, up to 16 of them as soon as three workgroups per
  // CU are left (h is made by every one)
  p.up_tiles = 4;
  while (p.up_tiles < 16 && uint64_t(p.tiles) * ((a.rows + 15) / 16) / p.up_tiles > 768) p.up_tiles *= 2;
  p.vec = a.cols % 4 == 0 && reinterpret_cast<uintptr_t>(a.act) % 16 == 0;
  p.out4 = a.rows % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  p.planes = reinterpret_cast<int64_t*>(take(uint64_t(p.chunks) * p.tiles * 16 * p.ranks * 8));
  p.tile_of = reinterpret_cast<uint32_t*>(take(uint64_t(p.tiles) * 4));
  p.perm = reinterpret_cast<uint32_t*>(take(uint64_t(p.tiles) * 64));
  p.n_tiles = reinterpret_cast<uint32_t*>(take(4));
  return at;
}

}  // namespace

// (rows in ranges, which bounds the partial sums)
constexpr uint64_t kRange = 8192;
static AdapterArgs range_of(const AdapterArgs& a, uint64_t t0) {
  AdapterArgs r = a;
  r.m = std::min(a.m - t0, kRange);
  r.index += t0;
  r.act += t0 * a.cols;
  r.out += t0 * a.rows;
  return r;
}
uint64_t adapter_work_bytes(const AdapterArgs& a) {
  Plan p;
  uint64_t most = 0;
  for (uint64_t t0 = 0; t0 < a.m; t0 += kRange) most = std::max(most, plan(range_of(a, t0), p));
  return most;
}
void launch_adapters(const AdapterArgs& a, void* work, hipStream_t s) {
  if (a.n == 0 || a.rows == 0) return;
  for (uint64_t t0 = 0; t0 < a.m; t0 += kRange) {
    Plan p;
    plan(range_of(a, t0), p);
    auto place = [&](auto*& q) {
      q = reinterpret_cast<std::remove_reference_t<decltype(q)>>(static_cast<uint8_t*>(work) +
                                                                  reinterpret_cast<uintptr_t>(q));
    };
    place(p.planes), place(p.tile_of), place(p.perm), place(p.n_tiles);
    const unsigned rank_groups = (a.max_rank + 63) / 64;
    if (p.a.m > kSmallRows) hipLaunchKernelGGL(k_adapter_sort, dim3(1), dim3(kSortThreads), 0, s, p);
    hipLaunchKernelGGL(k_adapter_down, dim3(p.tiles, p.chunks, rank_groups), dim3(256), 0, s, p);
    hipLaunchKernelGGL(k_adapter_up, dim3(p.tiles, unsigned((a.rows + 16 * p.up_tiles - 1) / (16 * p.up_tiles))), dim3(256),
                       rank_groups * (5 + 4) * kOp, s, p);
  }
}

}  // namespace det
