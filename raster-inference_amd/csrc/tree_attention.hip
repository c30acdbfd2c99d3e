// Attention of drafted rows over caches.
//
// Row i of a sequence sees its cached rows from start_i on and the drafted
// rows of its mask, in this order: s_r = requant(q . k_r), the integer softmax
// of the scores (terms exp(s_r - max) in Q32.32, weights requant(term / sum),
// the residual to 65536 added to the first maximum), out = requant(sum w_r v_r),
// all sums exact in wrapping 64-bit integers.
//
// The terms are defined relative to the row's maximum with a rounding at every
// step, so partial sums of another maximum cannot be rescaled: the scores of
// all keys come first, then the terms and their sum, then the weights. Keys are
// cut into chunks over the grid at each step and the chunks' maxima, sums and
// outputs (whole numbers: any order) joined by the next one:
//   k_tree_scores   q.k on int8 MFMA -> scores, a maximum per (row, chunk)
//   k_tree_terms    scores -> exp terms in place, a sum and a first maximum
//   k_tree_wsum     terms -> weights, w.v on int8 MFMA -> partial sums
//   k_tree_join     partial sums + residual * v[first maximum] -> out
//
// int32 values are taken apart into balanced base-256 digits, x = sum 256^j c_j
// with c_0 .. c_3 in [-128, 127] the bytes of (x + 0x80808080) ^ 0x80808080 and
// c_4 = 1 for x > 0x7f7f7f7f. Digits 3 and 4 are zero for |x| < 128.0 (narrow):
// normalised rows cost 9 (q.k) and 6 (w.v) byte products per value; rows that
// are not narrow take 24 and 11. Products of digits i, j share the int32
// accumulator i + j.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "det_arith.h"
#include "verify.h"
#include "wave.h"

namespace det {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr uint32_t kSeqs = 32;  // sequences per launch (by value in the arguments)
constexpr uint32_t kWaves = 8;
constexpr uint32_t kThreads = 64 * kWaves;
constexpr uint32_t kOp = 1024;  // one MFMA operand: 64 lanes x 16 bytes

// Sequence of a launch. Query rows of (sequence, kv head) are its drafted rows
// times the head's query heads, row l = draft * groups + head in group; row
// ids count them over the launch, kv head by kv head.
struct Seq {
  const int32_t* k;
  const int32_t* v;
  uint64_t ld, first, wrap;
  uint64_t row0;     // first drafted row
  uint64_t score0;   // first value of its score rows
  uint32_t rows, drafts;
  uint32_t id0;      // row id of its first row
  uint32_t score_ld;
};
struct Launch {
  TreeArgs a;
  int32_t* scores;     // then the terms
  int32_t* pmax;       // [row id][chunks]
  int64_t* psum;
  uint32_t* pfirst;
  int64_t* planes;     // [plane][row id][hd]
  int32_t* pweight;    // [row id][chunks of the weighted sums]
  uint32_t kv0, nkv;   // kv heads of the launch
  uint32_t n_seq, rows;  // row ids
  uint32_t chunk, chunks;    // keys per chunk of the scores and terms
  uint32_t wchunk, wchunks;  // of the weighted sums
  uint32_t splits, groups;   // waves of a weighted-sum block: key splits x groups of 32 dims
  uint32_t row_blocks;
  uint32_t block_rows;
  int wide_k, wide_v;  // 16-byte aligned q and k rows, 8-byte aligned v rows
  Seq s[kSeqs];
};
static_assert(sizeof(Launch) <= 4096, "kernel arguments");

// The work item of this workgroup: items (sequence, kv head, chunk) go round
// the eight XCDs, an item's row blocks one after the other on one XCD, so that
// they find its keys in that XCD's L2.
struct Item {
  uint32_t seq, kvh, chunk, rb;
  bool on;
};
__device__ inline Item item_of(const Launch& p, uint32_t chunks) {
  const uint32_t id = blockIdx.x, w = (id / 8 / p.row_blocks) * 8 + id % 8;
  Item it;
  it.rb = id / 8 % p.row_blocks;
  it.chunk = w % chunks;
  const uint32_t u = w / chunks;
  it.kvh = u % p.nkv;
  it.seq = u / p.nkv;
  it.on = it.seq < p.n_seq;
  return it;
}

// What a query row sees.
struct Sight {
  uint32_t start;
  uint64_t mask;
};
__device__ inline Sight sight_of(const TreeArgs& a, const Seq& s, uint32_t draft) {
  const uint64_t row = s.row0 + draft;
  Sight v;
  v.start = a.starts ? a.starts[row] : 0;
  v.mask = a.masks[row] & (s.drafts == 64 ? ~0ull : (1ull << s.drafts) - 1);
  return v;
}
__device__ inline bool sees(const Sight& v, uint32_t rows, uint32_t key) {
  return key < rows ? key >= v.start : (key - rows < 64 && ((v.mask >> (key - rows)) & 1));
}
// Row `key` of the cached rows followed by the drafted ones (this kv head's
// values); keys past them give the last drafted row.
__device__ inline const int32_t* row_ptr(const Seq& s, const int32_t* cache, const int32_t* drafted, uint64_t kv_ld,
                                         uint32_t key, uint64_t off) {
  uint64_t p = s.first + key;
  if (s.wrap && p >= s.wrap) p -= s.wrap;
  const bool cached = key < s.rows;
  const uint64_t d = s.row0 + min(key - s.rows, s.drafts - 1);
  return (cached ? cache : drafted) + (cached ? p * s.ld : d * kv_ld) + off;
}

// Digits of four values: word j holds digit j of each; `all` collects the words.
__device__ __forceinline__ void digits4(const int32_t (&x)[4], uint32_t (&w)[4], uint32_t& all) {
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = (uint32_t(x[e]) + 0x80808080u) ^ 0x80808080u;
  const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(u[1], u[0], 0x07030602u), d = __builtin_amdgcn_perm(u[3], u[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
  all |= w[3];
}
// Digit 4 of four values; a value above 0x7f7f7f7f has digit 3 at -128 or
// -127, so `all` is non-zero whenever one is set.
__device__ __forceinline__ uint32_t top4(const int32_t (&x)[4]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) w |= uint32_t(x[e] > 0x7f7f7f7f) << (8 * e);
  return w;
}
// How head rows are read: 16 bytes at a time from whole substeps of 64 dims
// (immediate offsets from the row), 16 bytes at a time, or value by value.
enum { kWhole = 2, kVec4 = 1, kScalar = 0 };
// Values [d, d + 4) of a row of hd; past its end any of its values.
template <int MODE>
__device__ __forceinline__ void load4(const int32_t* row, uint32_t d, uint32_t hd, int32_t (&x)[4]) {
  if constexpr (MODE == kScalar) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = to_global(row)[min(d + e, hd - 1)];
  } else {
    const int4 v = load_int4(to_global(row) + (MODE == kWhole ? d : min(d, hd - 4)));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
}

// Operand layout of q and k: lane 16 g + i holds row i, byte 4 j + e of its 16
// is dim 64 s + 16 j + 4 g + e of substep s (any order of the dims serves, and
// with this one four lanes load 64 consecutive bytes). Dims past the head's are
// zero in q, so that k may hold anything there, as it may in keys that no query
// sees.

// The products of one narrow key tile (digits in registers) with one narrow
// query tile (in LDS): lane l gets keys 4 (l >> 4) + r, query l & 15.
template <int NSUB>
__device__ __forceinline__ void score_tile(const v4i (&k)[NSUB][3], const v4i* q, uint32_t l, int32_t (&out)[4]) {
  v4i acc[5];
#pragma unroll
  for (int s = 0; s < 5; ++s) acc[s] = v4i{0, 0, 0, 0};
  v4i b[2][3];  // (a substep's operands are read during the one before; more of them at a time would spill)
#pragma unroll
  for (int i = 0; i < 3; ++i) b[0][i] = q[i * 64 + l];
#pragma unroll
  for (int s = 0; s < NSUB; ++s) {
    if (s + 1 < NSUB)
#pragma unroll
      for (int i = 0; i < 3; ++i) b[(s + 1) & 1][i] = q[((s + 1) * 3 + i) * 64 + l];
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int j = 0; j < 3; ++j)
        acc[i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[s][j], b[s & 1][i], acc[i + j], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
  // dot = a0 + 2^8 a1 + .. + 2^32 a4, each sum below 2^25: carries of the low
  // bytes leave floor(dot / 2^16) = v + 2^8 a3 + 2^16 a4 and a 16-bit remainder.
  // Below 2^30 (any score under 4096.0) that is 32-bit arithmetic.
  uint32_t far = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int32_t u = (acc[0][r] >> 8) + acc[1][r], v = (u >> 8) + acc[2][r];
    const uint32_t rem = ((uint32_t(u) & 0xffu) << 8) | (uint32_t(acc[0][r]) & 0xffu);
    far |= ((uint32_t(acc[4][r]) + 0x1000u) >> 13) | ((uint32_t(acc[3][r]) + 0x100000u) >> 21);
    const uint32_t q = uint32_t(v) + (uint32_t(acc[3][r]) << 8) + (uint32_t(acc[4][r]) << 16);
    out[r] = int32_t(q + uint32_t(rem + (q & 1u) > 0x8000u));
  }
  if (__any(far != 0))
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      uint64_t dot = 0;
#pragma unroll
      for (int s = 0; s < 5; ++s) dot += uint64_t(int64_t(acc[s][r])) << (8 * s);
      out[r] = requant(int64_t(dot));
    }
}

// Scores: a block takes up to 64 query rows (digits in LDS, converted once) and
// the keys of one chunk, 16 per wave and step, which each wave loads and takes
// apart in registers: no wave waits for another between its tiles.
template <int NSUB, int MODE>
__global__ __launch_bounds__(kThreads, NSUB <= 4 ? 4 : 2) void k_tree_scores(Launch p) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];  // [query tile][substep][digit][lane]
  __shared__ int32_t rmax[64];  // each row's largest score so far
  __shared__ Sight sight[64];
  __shared__ uint32_t qwide, last_start;
  const Item it = item_of(p, p.chunks);
  if (!it.on) return;
  const Seq& s = p.s[it.seq];
  const TreeArgs& a = p.a;
  const uint32_t R = s.drafts * a.groups, r0 = it.rb * p.block_rows, n = s.rows + s.drafts;
  const uint32_t k0 = it.chunk * p.chunk, k1 = min(k0 + p.chunk, n);
  if (r0 >= R || k0 >= k1) return;
  const uint32_t rows = min(R - r0, p.block_rows), tiles = (rows + 15) / 16;
  const uint32_t tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = l & 15, g = l >> 4;
  const uint32_t kvh = p.kv0 + it.kvh, hd = a.hd;
  if (tid < 64) {
    const Sight v = sight_of(a, s, min(r0 + tid, R - 1) / a.groups);
    const uint32_t m = uint32_t(wave_max64(int64_t(v.start)));
    sight[tid] = v;
    rmax[tid] = INT32_MIN;
    if (tid == 0) qwide = 0, last_start = m;
  }
  __syncthreads();
  // this lane's row of query tile T, and its values [dim, dim + 4)
  auto q_row = [&](uint32_t T) {
    const uint32_t row = min(r0 + 16 * T + i, R - 1);
    return a.q + (s.row0 + row / a.groups) * a.q_ld + uint64_t(kvh * a.groups + row % a.groups) * hd;
  };
  auto load_q = [&](const int32_t* src, uint32_t dim, int32_t (&x)[4]) {
    load4<MODE>(src, dim, hd, x);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (dim + e >= hd) x[e] = 0;
  };
  for (uint32_t u = wave; u < tiles * NSUB; u += kWaves) {
    const uint32_t sub = u % NSUB;
    const int32_t* src = q_row(u / NSUB);
    uint32_t d[3][4], all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int32_t x[4];
      load_q(src, 64 * sub + 16 * j + 4 * g, x);
      uint32_t w[4];
      digits4(x, w, all);
#pragma unroll
      for (int q = 0; q < 3; ++q) d[q][j] = w[q];
    }
    v4i* dst = reinterpret_cast<v4i*>(lds) + uint64_t(u) * 3 * 64 + l;
#pragma unroll
    for (int q = 0; q < 3; ++q) dst[q * 64] = v4i{int(d[q][0]), int(d[q][1]), int(d[q][2]), int(d[q][3])};
    if (__any(all != 0) && l == 0) qwide = 1;
  }
  __syncthreads();
  const bool qw = qwide != 0;
  const uint32_t id0 = s.id0 + it.kvh * R + r0;
  int32_t* sc = p.scores + s.score0 + uint64_t(it.kvh * R + r0) * s.score_ld;
  const uint64_t off = uint64_t(kvh) * hd;
  const uint32_t seen_from = __builtin_amdgcn_readfirstlane(last_start);
  // scores of tile T and the keys from key0 on: stored, and the largest seen one kept
  auto finish = [&](uint32_t T, uint32_t key0, const int32_t (&out)[4]) {
    if (16 * T + i < rows)
      *reinterpret_cast<int4*>(sc + uint64_t(16 * T + i) * s.score_ld + key0 + 4 * g) =
          make_int4(out[0], out[1], out[2], out[3]);
    int32_t m = INT32_MIN;
    if (key0 >= seen_from && key0 + 16 <= s.rows) {  // (every row sees every key: wave-uniform)
      m = max(max(out[0], out[1]), max(out[2], out[3]));
    } else {
      const Sight v = sight[16 * T + i];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (sees(v, s.rows, key0 + 4 * g + r)) m = max(m, out[r]);
    }
    atomicMax(&rmax[16 * T + i], m);
  };
  uint64_t later0 = 0, later1 = 0;  // key tiles that are not narrow (at most 128 per wave and chunk; wave-uniform)
  for (uint32_t key0 = k0 + 16 * wave, t = 0; key0 < k1; key0 += 16 * kWaves, ++t) {
    const int32_t* src = row_ptr(s, s.k, a.k, a.kv_ld, key0 + i, off);
    v4i k3[NSUB][3];
    int32_t x[NSUB][4][4];
    uint32_t hdl = hd;
    if (MODE != kWhole) asm volatile("" : "+s"(hdl));  // (offsets kept over the loop would spill)
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (the rows' last substep only can pass their end, but for the eight of 257 to 512 dims)
        if (MODE == kVec4 && sub + 1 < NSUB && NSUB < 8) load4<kWhole>(src, 64 * sub + 16 * j + 4 * g, hd, x[sub][j]);
        else load4<MODE>(src, 64 * sub + 16 * j + 4 * g, hdl, x[sub][j]);
        if (MODE == kScalar) __builtin_amdgcn_sched_barrier(0);  // (addresses of four values at a time)
      }
    uint32_t all = 0;
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
        digits4(x[sub][j], w, all);
#pragma unroll
        for (int q = 0; q < 3; ++q) k3[sub][q][j] = int(w[q]);
      }
    // (in registers here: moved past the branch they would keep the values as well)
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int q = 0; q < 3; ++q) asm volatile("" : "+v"(k3[sub][q]));
    if (qw || __any(all != 0)) {
      if (t < 64) later0 |= 1ull << t;
      else later1 |= 1ull << (t - 64);
      continue;
    }
#pragma unroll 1
    for (uint32_t T = 0; T < tiles; ++T) {
      int32_t out[4];
      score_tile<NSUB>(k3, reinterpret_cast<const v4i*>(lds) + uint64_t(T) * NSUB * 3 * 64, l, out);
      finish(T, key0, out);
    }
  }
  // the others with all five digits, a substep at a time
  uint32_t nsub = NSUB;
  asm volatile("" : "+s"(nsub));  // (a loop in earnest: unrolled it would spill)
#pragma unroll 1
  for (uint32_t h = 0; h < 2; ++h)
    for (uint64_t bits = h ? later1 : later0; bits; bits &= bits - 1) {
      const uint32_t key0 = k0 + 16 * wave + 16 * kWaves * (64 * h + uint32_t(__builtin_ctzll(bits)));
      const int32_t* src = row_ptr(s, s.k, a.k, a.kv_ld, key0 + i, off);
#pragma unroll 1
      for (uint32_t T = 0; T < tiles; ++T) {
        const int32_t* qsrc = q_row(T);
        uint64_t dot[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (uint32_t sub = 0; sub < nsub; ++sub) {
          v4i k5[5], q5[5];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            int32_t y[4];
            uint32_t w[4], unused = 0;
            load4<MODE>(src, 64 * sub + 16 * j + 4 * g, hd, y);
            digits4(y, w, unused);
#pragma unroll
            for (int c = 0; c < 4; ++c) k5[c][j] = int(w[c]);
            k5[4][j] = int(top4(y));
            load_q(qsrc, 64 * sub + 16 * j + 4 * g, y);
            digits4(y, w, unused);
#pragma unroll
            for (int c = 0; c < 4; ++c) q5[c][j] = int(w[c]);
            q5[4][j] = int(top4(y));
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {  // (digits 4 times 4 are past 2^64)
            v4i acc{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 5; ++j)
              if (c - j >= 0 && c - j < 5)
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(k5[j], q5[c - j], acc, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) dot[r] += uint64_t(int64_t(acc[r])) << (8 * c);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        int32_t out[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = requant(int64_t(dot[r]));
        finish(T, key0, out);
      }
    }
  // the chunk's maximum of every row (a row that sees none of the chunk's keys
  // leaves the lowest value, which changes no maximum; the terms look at what is
  // seen again)
  __syncthreads();
  if (tid < rows) p.pmax[uint64_t(id0 + tid) * p.chunks + it.chunk] = rmax[tid];
}

// An exp term (at most 2^32, and otherwise below 2^32 - 65000) from its 32 bits.
__device__ inline int64_t unpack_term(uint32_t e) { return int64_t(uint64_t(e) + (e == 0xffffffffu)); }

// Terms: one wave per (row, chunk).
__global__ __launch_bounds__(256) void k_tree_terms(Launch p) {
  const uint32_t l = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6), chunk = blockIdx.y;
  if (id >= p.rows) return;
  uint32_t b = 0;
  while (b + 1 < p.n_seq && p.s[b + 1].id0 <= id) ++b;
  const Seq& s = p.s[b];
  const uint32_t R = s.drafts * p.a.groups, local = id - s.id0, n = s.rows + s.drafts;
  const uint32_t k0 = chunk * p.chunk, k1 = min(k0 + p.chunk, n);
  if (k0 >= k1) return;
  const uint32_t used = (n + p.chunk - 1) / p.chunk;
  int32_t m = INT32_MIN;
  for (uint32_t c = l; c < used; c += 64) m = max(m, p.pmax[uint64_t(id) * p.chunks + c]);
  m = int32_t(wave_max64(m));
  const Sight v = sight_of(p.a, s, local % R / p.a.groups);
  int32_t* sc = p.scores + s.score0 + uint64_t(local) * s.score_ld;
  double sum = 0;  // (whole numbers below 2^53: exact in any order)
  uint32_t first = 0xffffffffu;
  const uint32_t k2 = min((k1 + 63) & ~63u, s.score_ld);  // (whole substeps of the weighted sums)
  const bool plain = v.start <= k0 && k1 <= s.rows;       // the row sees the whole chunk
  for (uint32_t kb = k0; kb < k2; kb += 256) {
    int32_t x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = sc[min(kb + 64 * u + l, k2 - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t k = kb + 64 * u + l, gap = uint32_t(m) - uint32_t(x[u]);
      bool in = k < k1 && gap < (1u << 20);
      if (!plain) in = in && sees(v, s.rows, k);
      double e = 0;
      if (__any(in)) {
        e = in ? softmax_term(gap) : 0.0;
        if (in && gap == 0) first = min(first, k);
        sum += e;
      }
      // (2^32 in 32 bits: all ones, which no other term is)
      if (k < k2) sc[k] = int32_t(uint32_t(__builtin_fmin(e, 4294967295.0)));
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  first = ~uint32_t(wave_max64(int64_t(~first)));
  if (l == 0) {
    p.psum[uint64_t(id) * p.chunks + chunk] = int64_t(sum);
    p.pfirst[uint64_t(id) * p.chunks + chunk] = first;
  }
}

// A weight from its term: round(round(e 2^32 / S) / 2^16). With m = 2^(48 + sh)
// / S, at most 2^31, hi = floor(e m / 2^32) is less than 3 below e 2^(16 + sh) /
// S, so hi + half rounds to the weight unless it lies within 2^(sh - 13) (at
// least 4) of a border (the inner rounding moves it by at most 2^(sh - 17));
// then the exact quotient decides. 15 <= sh <= 31.
struct Recip {
  uint32_t m, sh;
  int64_t sum;
};
__device__ inline Recip recip_of(int64_t sum) {
  Recip r{0, 15, sum};
  if (sum <= 0) return r;
  // sum in [2^32, 2^53): 2^lz sum in [2^63, 2^64), q = 2^94 / (2^lz sum) in (2^30, 2^31]
  const uint32_t lz = __clzll(sum);
  const double q = 2147483648.0 * (9223372036854775808.0 / double(uint64_t(sum) << lz));
  r.sh = 46 - lz;
  r.m = uint32_t(q);
  if (r.sh > 31) {
    r.m >>= r.sh - 31;
    r.sh = 31;
  }
  return r;
}
__device__ __forceinline__ uint32_t weight_of(uint32_t e, uint32_t m, uint32_t sh, bool& unsure) {
  const uint32_t half = 1u << (sh - 1), near = 1u << (sh - 13);
  const uint32_t y = __umulhi(e, m) + half, f = y & (2 * half - 1);
  unsure = f - near >= 2 * half - 2 * near;
  return y >> sh;
}

// Weighted sums: a block takes up to 16 RT query rows, one chunk of keys and
// 256 head dims; wave (dim group of 32, key split). Per step of 64 keys per
// split the block turns the terms into weight digits in LDS, while each wave
// loads the next values and multiplies the present ones. Lane 16 g + i of a
// wave loads dims 2 i, 2 i + 1 of the keys 16 g + e: 128 consecutive bytes per
// key.
// Weights above 32639 (at most two of a row) need a third digit; they go on
// without 65536, which is added from the list of their keys.
constexpr uint32_t wsum_rounds(int RT) { return RT == 4 ? 1 : 2; }
constexpr uint32_t most_splits(int RT) { return wsum_rounds(RT) * kThreads / (RT * 128); }
template <int RT>
__global__ __launch_bounds__(kThreads, 2) void k_tree_wsum(Launch p) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];  // [2][split][query tile][digit][lane]
  __shared__ Recip recip[16 * RT];
  __shared__ uint32_t big_key[16 * RT][2], big_n[16 * RT];
  __shared__ int32_t total[16 * RT];
  __shared__ uint32_t vwide;
  const Item it = item_of(p, p.wchunks);
  if (!it.on) return;
  const Seq& s = p.s[it.seq];
  const TreeArgs& a = p.a;
  const uint32_t R = s.drafts * a.groups, r0 = it.rb * p.block_rows, n = s.rows + s.drafts;
  const uint32_t k0 = it.chunk * p.wchunk, k1 = min(k0 + p.wchunk, n);
  if (r0 >= R || k0 >= k1) return;
  const uint32_t rows = min(R - r0, p.block_rows), id0 = s.id0 + it.kvh * R + r0;
  const uint32_t tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = l & 15, g = l >> 4;
  const uint32_t kvh = p.kv0 + it.kvh, hd = a.hd, splits = p.splits, groups = p.groups;
  const uint32_t split = wave / groups, dim0 = blockIdx.y * 256 + 32 * (wave % groups);
  const int32_t* terms = p.scores + s.score0 + uint64_t(it.kvh * R + r0) * s.score_ld;
  const uint32_t used = (n + p.chunk - 1) / p.chunk;
  if (tid == 0) vwide = 0;
  for (uint32_t r = wave; r < 16 * RT; r += kWaves) {
    int64_t sum = 0;
    if (r < rows)
      for (uint32_t c = l; c < used; c += 64) sum += p.psum[uint64_t(id0 + r) * p.chunks + c];
    sum = wave_sum_wrap64(sum);
    if (l == 0) {
      recip[r] = recip_of(sum);
      big_n[r] = 0;
      total[r] = 0;
    }
  }
  __syncthreads();
  const uint32_t per = 64 * splits;  // keys per step
  // Weights of a step: eight keys of a row per thread and round, whose terms
  // are loaded a step ahead.
  constexpr uint32_t kRounds = wsum_rounds(RT);
  const uint32_t items = splits * RT * 128;
  auto load_terms = [&](uint32_t k, uint32_t u, uint32_t (&e)[8]) {
    const uint32_t r = u / 8 % (16 * RT), key = k + 64 * (u / (128 * RT)) + 8 * (u % 8);
    // (rows and keys past the end: any in range, not used)
    const int4* src = reinterpret_cast<const int4*>(terms + uint64_t(min(r, rows - 1)) * s.score_ld + min(key, s.score_ld - 8));
    const int4 t0 = src[0], t1 = src[1];
    e[0] = uint32_t(t0.x), e[1] = uint32_t(t0.y), e[2] = uint32_t(t0.z), e[3] = uint32_t(t0.w);
    e[4] = uint32_t(t1.x), e[5] = uint32_t(t1.y), e[6] = uint32_t(t1.z), e[7] = uint32_t(t1.w);
  };
  auto put_weights = [&](uint32_t k, uint32_t buf, uint32_t u, const uint32_t (&e)[8]) {
    const uint32_t r = u / 8 % (16 * RT), sp = u / (128 * RT), o = u % 8, key = k + 64 * sp + 8 * o;
    uint32_t w[8], d[2][2] = {{0, 0}, {0, 0}};
    if (r < rows && key < k1) {
      const uint32_t m = recip[r].m, sh = recip[r].sh;
      uint32_t unsure = 0, most = 0;
      int32_t tot = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        bool no;
        w[q] = weight_of(e[q], m, sh, no);
        unsure |= uint32_t(no) << q;
      }
#pragma unroll 1
      for (; unsure; unsure &= unsure - 1) {
        const int at = __builtin_ctz(unsure);
        uint32_t x = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) x = q == at ? e[q] : x;
        x = x ? uint32_t(softmax_weight(unpack_term(x), recip[r].sum)) : 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = q == at ? x : w[q];
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        tot += int32_t(w[q]);
        most = max(most, w[q]);
      }
      if (most > 32639)
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
          uint32_t x = 0;
#pragma unroll
          for (int c = 0; c < 8; ++c) x = q == c ? w[c] : x;
          if (x > 32639) {
            const uint32_t at = atomicAdd(&big_n[r], 1u);
            if (at < 2) big_key[r][at] = key + q;
          }
        }
      if (tot) {
        if (blockIdx.y == 0) atomicAdd(&total[r], tot);
        // digits of four weights at a time: bytes 0 and 1 of (w + 0x8080) ^ 0x8080
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t z[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) z[q] = w[4 * h + q] + 0x8080u;
          const uint32_t a = __builtin_amdgcn_perm(z[1], z[0], 0x05010400u), b = __builtin_amdgcn_perm(z[3], z[2], 0x05010400u);
          d[0][h] = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u;
          d[1][h] = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u;
        }
      }
    }
    // lane 16 (o / 2) + r % 16, bytes 8 (o % 2) ..
    int8_t* at = lds + (buf * splits * RT + sp * RT + r / 16) * 2 * kOp + (16 * (o / 2) + r % 16) * 16 + 8 * (o % 2);
    *reinterpret_cast<uint2*>(at) = make_uint2(d[0][0], d[0][1]);
    *reinterpret_cast<uint2*>(at + kOp) = make_uint2(d[1][0], d[1][1]);
  };
  const uint64_t off = uint64_t(kvh) * hd;
  const uint32_t dim = dim0 + 2 * i;
  const bool dims_on = split < splits && dim0 < hd;  // (wave-uniform)
  const uint32_t dim_in = dim + 1 < hd ? dim : (hd > 1 ? hd - 2 : 0);  // (sums of dims past hd are dropped)
  auto load_v = [&](uint32_t k, int32_t (&x)[16][2]) {
    if (!dims_on) return;
    const uint32_t kk = k + 64 * split;
    uint64_t at = s.first + kk;
    if (s.wrap && at >= s.wrap) at -= s.wrap;
    if (p.wide_v && kk + 64 <= min(s.rows, k1) && (!s.wrap || at + 64 <= s.wrap) && s.ld < (1u << 22)) {
      // whole substeps of one run of cached rows: scalar row addresses
      const uint32_t o = 16 * g * uint32_t(s.ld) + dim_in;
      const int32_t* base = s.v + at * s.ld + off;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        typedef int v2 __attribute__((ext_vector_type(2)));
        const v2 t = *(global_ptr<const v2>)(to_global(base + e * s.ld) + o);
        x[e][0] = t.x, x[e][1] = t.y;
      }
      return;
    }
    // (weights are zero from k1 on)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int32_t* row = row_ptr(s, s.v, a.v, a.kv_ld, min(kk + 16 * g + e, k1 - 1), off);
      x[e][0] = to_global(row)[min(dim, hd - 1)];
      x[e][1] = to_global(row)[min(dim + 1, hd - 1)];
      __builtin_amdgcn_sched_barrier(0);  // (one row's address at a time)
    }
  };
  auto digit_words = [&](const int32_t (&x)[16][2], int c, v4i (&d)[4], uint32_t& all) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int32_t y[4] = {x[4 * j][c], x[4 * j + 1][c], x[4 * j + 2][c], x[4 * j + 3][c]};
      uint32_t w[4];
      digits4(y, w, all);
#pragma unroll
      for (int q = 0; q < 4; ++q) d[q][j] = int(w[q]);
    }
  };
  v4i acc[RT][2][4];
#pragma unroll
  for (int T = 0; T < RT; ++T)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[T][c][q] = v4i{0, 0, 0, 0};
  int32_t x[16][2] = {};
  uint32_t e[kRounds][8];
  auto all_terms = [&](uint32_t k) {
#pragma unroll
    for (uint32_t c = 0; c < kRounds; ++c)
      if (tid + kThreads * c < items) load_terms(k, tid + kThreads * c, e[c]);
  };
  auto all_weights = [&](uint32_t k, uint32_t buf) {
#pragma unroll
    for (uint32_t c = 0; c < kRounds; ++c)
      if (tid + kThreads * c < items) put_weights(k, buf, tid + kThreads * c, e[c]);
  };
  all_terms(k0);
  load_v(k0, x);
  all_weights(k0, 0);
  if (k0 + per < k1) all_terms(k0 + per);
  __syncthreads();
  uint32_t all = 0, buf = 0;
  for (uint32_t k = k0; k < k1; k += per, buf ^= 1) {
    v4i d[2][4];
    digit_words(x, 0, d[0], all);
    digit_words(x, 1, d[1], all);
    if (k + per < k1) {
      load_v(k + per, x);
      all_weights(k + per, buf ^ 1);
      if (k + 2 * per < k1) all_terms(k + 2 * per);
    }
    if (dims_on) {
      const v4i* w = reinterpret_cast<const v4i*>(lds + (buf * splits + split) * RT * 2 * kOp);
#pragma unroll
      for (int T = 0; T < RT; ++T)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const v4i wq = w[(T * 2 + q) * 64 + l];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 3; ++j)
              acc[T][c][q + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wq, d[c][j], acc[T][c][q + j], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
    }
    lds_barrier();  // (the next step's loads stay in flight)
  }
  if (all) vwide = 1;
  __syncthreads();
  // lane l, component r: row 16 T + 4 g + r, dims dim and dim + 1
  const uint32_t plane = it.chunk * splits + split;
  int64_t* out = p.planes + (uint64_t(plane) * p.rows + id0) * hd;
  // the first `count` sums, sum q at digit q + shift
  auto put = [&](auto count, auto shift, bool add) {
    if (!dims_on) return;
#pragma unroll
    for (int T = 0; T < RT; ++T)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint64_t y[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int q = 0; q < decltype(count)::value; ++q)
            y[c] += uint64_t(int64_t(acc[T][c][q][r])) << (8 * (q + decltype(shift)::value));
        const uint32_t row = 16 * T + 4 * g + r;
        int64_t* o = out + uint64_t(row) * hd + dim;
        if (row < rows && dim < hd) *o = int64_t((add ? uint64_t(*o) : 0) + y[0]);
        if (row < rows && dim + 1 < hd) o[1] = int64_t((add ? uint64_t(o[1]) : 0) + y[1]);
      }
  };
  put(std::integral_constant<int, 4>(), std::integral_constant<int, 0>(), false);
  if (blockIdx.y == 0 && tid < rows) p.pweight[uint64_t(id0 + tid) * p.wchunks + it.chunk] = total[tid];
  __syncthreads();
  // the 65536 that weights above 32639 went without (in the first split's plane)
  const uint32_t d_end = min(hd, blockIdx.y * 256 + 256);
  for (uint32_t r = wave; r < rows; r += kWaves)
    for (uint32_t b = 0; b < min(big_n[r], 2u); ++b) {
      const int32_t* v = row_ptr(s, s.v, a.v, a.kv_ld, big_key[r][b], off);
      int64_t* o = p.planes + (uint64_t(it.chunk * splits) * p.rows + id0 + r) * hd;
      for (uint32_t d = blockIdx.y * 256 + l; d < d_end; d += 64)
        o[d] = int64_t(uint64_t(o[d]) + (uint64_t(int64_t(to_global(v)[d])) << 16));
    }
  __syncthreads();
  if (!vwide) return;  // (workgroup-uniform)
  // a value of the chunk is not narrow: its digits 3 and 4, in a pass of their own
#pragma unroll
  for (int T = 0; T < RT; ++T)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int q = 0; q < 3; ++q) acc[T][c][q] = v4i{0, 0, 0, 0};
  if (tid < 16 * RT) big_n[tid] = 2;  // (no more entries)
#pragma unroll 1
  for (uint32_t k = k0; k < k1; k += per) {
    __syncthreads();
    all_terms(k);
    all_weights(k, 0);
    load_v(k, x);
    __syncthreads();
    if (!dims_on) continue;
    const v4i* w = reinterpret_cast<const v4i*>(lds + split * RT * 2 * kOp);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      v4i d[4], t;
      uint32_t unused = 0;
      digit_words(x, c, d, unused);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t y[4] = {x[4 * j][c], x[4 * j + 1][c], x[4 * j + 2][c], x[4 * j + 3][c]};
        t[j] = int(top4(y));
      }
#pragma unroll
      for (int T = 0; T < RT; ++T)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const v4i wq = w[(T * 2 + q) * 64 + l];
          acc[T][c][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wq, d[3], acc[T][c][q], 0, 0, 0);
          acc[T][c][q + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wq, t, acc[T][c][q + 1], 0, 0, 0);
        }
    }
  }
  put(std::integral_constant<int, 3>(), std::integral_constant<int, 3>(), true);
}

// Join: a wave per (row, 64 dims), or four with a share of the planes each where
// there are many.
template <int SHARES>
__global__ __launch_bounds__(256) void k_tree_join(Launch p) {
  const uint32_t l = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t id = blockIdx.x;
  uint32_t b = 0;
  while (b + 1 < p.n_seq && p.s[b + 1].id0 <= id) ++b;
  const Seq& s = p.s[b];
  const TreeArgs& a = p.a;
  const uint32_t R = s.drafts * a.groups, local = id - s.id0, n = s.rows + s.drafts;
  const uint32_t kvh = p.kv0 + local / R, row = local % R, used = (n + p.chunk - 1) / p.chunk;
  const uint32_t wused = (n + p.wchunk - 1) / p.wchunk;
  int64_t tot = 0, sum = 0;
  uint32_t first = 0xffffffffu;
  for (uint32_t c = l; c < used; c += 64) {
    sum += p.psum[uint64_t(id) * p.chunks + c];
    first = min(first, p.pfirst[uint64_t(id) * p.chunks + c]);
  }
  for (uint32_t c = l; c < wused; c += 64) tot += p.pweight[uint64_t(id) * p.wchunks + c];
  sum = wave_sum_wrap64(sum);
  tot = wave_sum_wrap64(tot);
  first = ~uint32_t(wave_max64(int64_t(~first)));
  int32_t* out = a.out + (s.row0 + row / a.groups) * a.out_ld + uint64_t(kvh * a.groups + row % a.groups) * a.hd;
  int64_t extra = 0;
  const int32_t* v = nullptr;
  if (first != 0xffffffffu) {
    // the residual goes to the first maximum, with saturation
    const int32_t w = softmax_weight(int64_t(1) << 32, sum);
    extra = int64_t(add_sat(w, sub_sat(kOneAct, sat32(tot)))) - w;
    v = row_ptr(s, s.v, a.v, a.kv_ld, first, uint64_t(kvh) * a.hd);
  }
  const uint32_t d = 64 * (blockIdx.y * (4 / SHARES) + wave / SHARES) + l, in = min(d, a.hd - 1);
  const uint32_t planes = wused * p.splits;
  const int64_t* src = p.planes + uint64_t(id) * a.hd + in;
  const uint64_t ld = uint64_t(p.rows) * a.hd;
  uint64_t y = 0;
  uint32_t q = wave % SHARES;
  for (; q + 3 * SHARES < planes; q += 4 * SHARES) {
    uint64_t t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) t[u] = uint64_t(src[(q + u * SHARES) * ld]);
#pragma unroll
    for (int u = 0; u < 4; ++u) y += t[u];
  }
  for (; q < planes; q += SHARES) y += uint64_t(src[q * ld]);
  if constexpr (SHARES > 1) {
    __shared__ uint64_t share[4][64];
    share[wave][l] = y;
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < 4; ++w) y += share[w][l];
  }
  if (d < a.hd) out[d] = v ? requant(int64_t(y + uint64_t(extra * to_global(v)[d]))) : 0;
}

uint64_t up(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

// One launch group: sequences [b0, b1), kv heads [kv0, kv0 + nkv).
struct Group {
  uint32_t b0, b1, kv0, nkv;
};
constexpr uint64_t kScoreBytes = uint64_t(256) << 20;  // score rows of a group (the Infinity Cache)
constexpr uint32_t kMaxDimsBlock = 256;

uint32_t score_ld(const TreeSeq& s) { return uint32_t(up(uint64_t(s.rows) + s.drafts, 64)); }
uint64_t seq_score_bytes(const TreeArgs& a, const TreeSeq& s) { return uint64_t(s.drafts) * a.groups * score_ld(s) * 4; }

template <class F>
void for_groups(const TreeArgs& a, const TreeSeq* seqs, uint32_t n, F&& f) {
  for (uint32_t b = 0; b < n;) {
    uint64_t bytes = seq_score_bytes(a, seqs[b]) * a.nkv;
    if (bytes > kScoreBytes) {
      // one sequence in ranges of kv heads
      const uint32_t per = uint32_t(std::max<uint64_t>(kScoreBytes / seq_score_bytes(a, seqs[b]), 1));
      for (uint32_t h = 0; h < a.nkv; h += per) f(Group{b, b + 1, h, std::min(per, a.nkv - h)});
      ++b;
      continue;
    }
    uint32_t e = b + 1;
    while (e < n && e - b < kSeqs && bytes + seq_score_bytes(a, seqs[e]) * a.nkv <= kScoreBytes)
      bytes += seq_score_bytes(a, seqs[e++]) * a.nkv;
    f(Group{b, e, 0, a.nkv});
    b = e;
  }
}

// Keys per chunk: equal shares of the longest sequence, so that `units` blocks
// per chunk make `want` blocks, what the device runs at once (in whole granules;
// at most 16384 keys, which bounds the int32 sums and a wave's key tiles).
uint32_t chunk_of(uint64_t keys, uint64_t units, uint64_t want, uint32_t granule) {
  const uint64_t n = std::max<uint64_t>(want / units, 1);
  return uint32_t(std::min<uint64_t>(up((keys + n - 1) / n, granule), 16384 / granule * granule));
}

// The launch of a group without its scratch pointers; returns the scratch's bytes.
uint64_t plan(const TreeArgs& a, const TreeSeq* seqs, const Group& g, Launch& p) {
  p = Launch{};
  p.a = a;
  p.kv0 = g.kv0;
  p.nkv = g.nkv;
  p.n_seq = g.b1 - g.b0;
  uint64_t scores = 0, keys = 0, units = 0;
  uint32_t most = 0;
  auto aligned = [](const void* q, uint64_t to) { return reinterpret_cast<uintptr_t>(q) % to == 0; };
  bool w4 = a.hd % 4 == 0 && a.q_ld % 4 == 0 && a.kv_ld % 4 == 0 && aligned(a.q, 16) && aligned(a.k, 16);
  bool w2 = a.hd % 2 == 0 && a.kv_ld % 2 == 0 && aligned(a.v, 8);
  for (uint32_t b = g.b0; b < g.b1; ++b) {
    const TreeSeq& t = seqs[b];
    Seq& s = p.s[b - g.b0];
    s = {t.k, t.v, t.ld, t.first, t.wrap, t.row0, scores, t.rows, t.drafts, p.rows, score_ld(t)};
    if (t.rows) {
      w4 = w4 && t.ld % 4 == 0 && aligned(t.k, 16);
      w2 = w2 && t.ld % 2 == 0 && aligned(t.v, 8);
    }
    const uint32_t R = t.drafts * a.groups;
    p.rows += R * g.nkv;
    scores += uint64_t(R) * g.nkv * s.score_ld;
    keys = std::max<uint64_t>(keys, s.score_ld);
    most = std::max(most, R);
  }
  p.wide_k = w4;
  p.wide_v = w2;
  // 64 query rows per block; 32 where their digits would take more than half the
  // LDS, or where the waves of a weighted-sum block share the keys instead of the dims
  p.block_rows = std::min<uint32_t>(uint32_t(up(most, 16)), a.hd > 128 && a.hd <= 256 ? 64 : 32);
  p.row_blocks = (most + p.block_rows - 1) / p.block_rows;
  units = uint64_t(p.n_seq) * g.nkv * p.row_blocks;
  p.chunk = chunk_of(keys, units, 512, 16 * kWaves);
  p.chunks = uint32_t((keys + p.chunk - 1) / p.chunk);
  p.groups = a.hd <= 32 ? 1 : a.hd <= 64 ? 2 : a.hd <= 128 ? 4 : 8;
  p.splits = std::min(kWaves / p.groups, most_splits(p.block_rows <= 16 ? 1 : p.block_rows <= 32 ? 2 : 4));
  p.wchunk = chunk_of(keys, units * ((a.hd + kMaxDimsBlock - 1) / kMaxDimsBlock), p.block_rows <= 16 ? 512 : 256, 64 * p.splits);
  p.wchunks = uint32_t((keys + p.wchunk - 1) / p.wchunk);
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  p.scores = reinterpret_cast<int32_t*>(take(scores * 4));
  p.pmax = reinterpret_cast<int32_t*>(take(uint64_t(p.rows) * p.chunks * 4));
  p.psum = reinterpret_cast<int64_t*>(take(uint64_t(p.rows) * p.chunks * 8));
  p.pfirst = reinterpret_cast<uint32_t*>(take(uint64_t(p.rows) * p.chunks * 4));
  p.planes = reinterpret_cast<int64_t*>(take(uint64_t(p.wchunks) * p.splits * p.rows * a.hd * 8));
  p.pweight = reinterpret_cast<int32_t*>(take(uint64_t(p.rows) * p.wchunks * 4));
  return at;
}

template <int NSUB>
void launch_scores(const Launch& p, uint32_t blocks, hipStream_t s) {
  const uint32_t lds = p.block_rows / 16 * NSUB * 3 * kOp;
  auto go = [&](auto kernel) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), lds, s, p);
  };
  if (!p.wide_k) go(&k_tree_scores<NSUB, kScalar>);
  else if (p.a.hd == 64 * NSUB) go(&k_tree_scores<NSUB, kWhole>);
  else go(&k_tree_scores<NSUB, kVec4>);
}
template <int RT>
void launch_wsum(const Launch& p, uint32_t blocks, hipStream_t s) {
  const uint32_t lds = 2 * p.splits * RT * 2 * kOp;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_tree_wsum<RT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
  (void)attr;
  hipLaunchKernelGGL(k_tree_wsum<RT>, dim3(blocks, (p.a.hd + kMaxDimsBlock - 1) / kMaxDimsBlock), dim3(kThreads), lds, s, p);
}

}  // namespace

uint64_t tree_work_bytes(const TreeArgs& a, const TreeSeq* seqs, uint32_t n) {
  uint64_t most = 0;
  for_groups(a, seqs, n, [&](const Group& g) {
    Launch p;
    most = std::max(most, plan(a, seqs, g, p));
  });
  return most;
}

void launch_tree_attention(const TreeArgs& a, const TreeSeq* seqs, uint32_t n, void* work, hipStream_t s) {
  for_groups(a, seqs, n, [&](const Group& g) {
    Launch p;
    plan(a, seqs, g, p);
    auto place = [&](auto*& q) {
      q = reinterpret_cast<std::remove_reference_t<decltype(q)>>(static_cast<uint8_t*>(work) + reinterpret_cast<uintptr_t>(q));
    };
    place(p.scores), place(p.pmax), place(p.psum), place(p.pfirst), place(p.planes), place(p.pweight);
    const uint32_t units = p.n_seq * p.nkv;
    auto blocks = [&](uint32_t chunks) { return uint32_t(up(uint64_t(units) * chunks, 8)) * p.row_blocks; };
    const uint32_t nsub = (a.hd + 63) / 64;
    if (nsub == 1) launch_scores<1>(p, blocks(p.chunks), s);
    else if (nsub == 2) launch_scores<2>(p, blocks(p.chunks), s);
    else if (nsub == 3) launch_scores<3>(p, blocks(p.chunks), s);
    else if (nsub == 4) launch_scores<4>(p, blocks(p.chunks), s);
    else launch_scores<8>(p, blocks(p.chunks), s);
    hipLaunchKernelGGL(k_tree_terms, dim3((p.rows + 3) / 4, p.chunks), dim3(256), 0, s, p);
    if (p.block_rows <= 16) launch_wsum<1>(p, blocks(p.wchunks), s);
    else if (p.block_rows <= 32) launch_wsum<2>(p, blocks(p.wchunks), s);
    else launch_wsum<4>(p, blocks(p.wchunks), s);
    if (p.wchunks * p.splits > 16)
      hipLaunchKernelGGL(k_tree_join<4>, dim3(p.rows, (a.hd + 63) / 64), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL(k_tree_join<1>, dim3(p.rows, (a.hd + 255) / 256), dim3(256), 0, s, p);
  });
}

}  // namespace det
