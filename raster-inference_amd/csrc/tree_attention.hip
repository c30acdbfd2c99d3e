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
//   k_tree_rows     scores of whole rows -> exp terms, their sum, weights; or, for
//                   few long rows, over the chunks of each:
//     k_tree_terms    scores -> terms in place, a sum and a first maximum
//     k_tree_weights  terms -> weights
//   k_tree_wsum     w.v on int8 MFMA -> partial sums
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
constexpr uint32_t kSumDims = 32 * kWaves;  // of a weighted-sum block
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
  uint32_t score_ld;
};
// What a row's output has besides its two-digit weights.
struct RowEnd {
  int64_t extra;     // times v of the first maximum: the residual
  uint32_t first;    // the first maximum, kNone in a row that sees nothing
  uint32_t n_big;    // keys of weights above 32639, at most two of a row: 65536
  uint32_t big0, big1;  // times their v
};
constexpr uint32_t kNone = 0xffffffffu;
struct Launch {
  TreeArgs a;
  int32_t* scores;     // of short rows then the weights, of long ones the terms
  int8_t* weights;     // [score row][64 keys]: their weights' digits 0, then 1 (2 bytes a key)
  int32_t* pmax;       // [row id][chunks]
  int64_t* psum;
  uint32_t* pfirst;
  int64_t* planes;     // [plane][row id][hd]
  int32_t* pweight;    // [row id][chunks]
  RowEnd* ends;        // [row id]
  uint32_t kv0, nkv;   // kv heads of the launch
  uint32_t n_seq, rows;  // row ids
  uint32_t chunk, chunks, items;     // keys per chunk of the scores and terms
  uint32_t wchunk, wchunks, witems;  // of the weighted sums
  uint32_t splits, groups;   // waves of a weighted-sum block: key splits x groups of 32 dims
  uint32_t row_blocks, block_rows;  // of the scores
  uint32_t sum_blocks, sum_rows;    // of the weighted sums
  int whole;                 // rows are turned into weights whole
  int wide_k, wide_v;  // 16-byte aligned q and k rows, 8-byte aligned v rows
  int deep_v;          // 16-byte aligned v rows, more than 128 dims
  // per sequence: the row id of its first row, the first of its items (chunks x kv
  // heads) in the scores and in the weighted sums
  uint32_t id0[kSeqs], item0[kSeqs], witem0[kSeqs];
  Seq s[kSeqs];
};
static_assert(sizeof(Launch) <= 4096, "kernel arguments");

// The sequence that number `at` belongs to, of the sequences' first ones (a vector
// load and a ballot: reading them one after the other takes a latency each).
__device__ inline uint32_t find_seq(const uint32_t (&first)[kSeqs], uint32_t n_seq, uint32_t at) {
  const uint32_t l = threadIdx.x & 63, v = first[min(l, kSeqs - 1)];
  return uint32_t(__popcll(__ballot(l < n_seq && v <= at))) - 1;
}
// The work item of this workgroup: items (sequence, chunk, kv head) go round
// the eight XCDs, an item's row blocks one after the other on one XCD, so that
// they find its keys in that XCD's L2.
struct Item {
  uint32_t seq, kvh, chunk, rb;
  bool on;
};
__device__ inline Item item_of(const Launch& p, const uint32_t (&item0)[kSeqs], uint32_t items, uint32_t row_blocks) {
  const uint32_t id = blockIdx.x, w = (id / 8 / row_blocks) * 8 + id % 8;
  Item it{};
  it.on = w < items;
  if (!it.on) return it;
  it.rb = id / 8 % row_blocks;
  it.seq = p.n_seq > 1 ? find_seq(item0, p.n_seq, w) : 0;
  const uint32_t u = w - (p.n_seq > 1 ? item0[it.seq] : 0);
  it.kvh = u % p.nkv;
  it.chunk = u / p.nkv;
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
// The cached rows of a sequence followed by its drafted ones, one kv head's
// values. Held in registers: read from the arguments in each lane's branch they
// would cost a round trip to memory per row.
struct Rows {
  const int32_t* cache;
  const int32_t* drafted;  // its first drafted row
  uint64_t ld, kv_ld, first, wrap;
  uint32_t rows, drafts;
  __device__ __forceinline__ Rows(const Seq& s, const int32_t* c, const int32_t* d, uint64_t kv, uint64_t off) {
    const int32_t *c0 = c + off, *d0 = d + s.row0 * kv + off;
    uint64_t l0 = s.ld, f0 = s.first, w0 = s.wrap;
    uint32_t r0 = s.rows, n0 = s.drafts;
    asm volatile("" : "+s"(c0), "+s"(d0), "+s"(l0), "+s"(kv));
    asm volatile("" : "+s"(f0), "+s"(w0), "+s"(r0), "+s"(n0));
    cache = c0, drafted = d0, ld = l0, kv_ld = kv, first = f0, wrap = w0, rows = r0, drafts = n0;
  }
  // Row `key`; keys past them give the last drafted row.
  __device__ __forceinline__ const int32_t* at(uint32_t key) const {
    uint64_t p = first + key;
    p -= wrap && p >= wrap ? wrap : 0;
    // (values here: a choice between the members would become one of their addresses)
    const int32_t *c = cache, *d = drafted;
    uint64_t cl = ld, dl = kv_ld;
    asm("" : "+s"(c), "+s"(d), "+s"(cl), "+s"(dl));
    const bool cached = key < rows;
    const uint64_t row = cached ? p : uint64_t(min(key - rows, drafts - 1));
    return (cached ? c : d) + row * (cached ? cl : dl);
  }
};

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
  if (__any(far != 0)) {
    // (a branch in earnest: the 64-bit sums would be computed in any case)
#pragma unroll
    for (int s = 0; s < 5; ++s) asm volatile("" : "+v"(acc[s]));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      uint64_t dot = 0;
#pragma unroll
      for (int s = 0; s < 5; ++s) dot += uint64_t(int64_t(acc[s][r])) << (8 * s);
      out[r] = requant(int64_t(dot));
    }
  }
}

// Scores: a block takes up to 64 query rows (digits in LDS, converted once) and
// the keys of one chunk, 16 per wave and step, which each wave loads and takes
// apart in registers: no wave waits for another between its tiles. AHEAD: up to
// 128 rows, half the waves, each step's keys loaded during the step before. At
// 4096 rows of 8256 keys of 256 dims (16 sets of 256 rows) that takes 102 us
// against 122 (the device copies its 330 MB, of which the scores are 135, in 67).
// Up to 64 rows both are as fast (28 rows of 2000 keys 8.6 and 8.7 us, 64 rows 14.2
// and 13.3, 4 rows of 60 K keys for each of two heads 28 and 27, whose
// 123 MB are 25 at a copy's rate).
template <int NSUB, int MODE, bool AHEAD>
__global__ __launch_bounds__(kThreads, NSUB <= 4 && !AHEAD ? 4 : 2) void k_tree_scores(Launch p) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];  // [query tile][substep][digit][lane]
  constexpr uint32_t kRows = AHEAD ? 128 : 64;
  __shared__ int32_t rmax[kRows];  // each row's largest score so far
  __shared__ Sight sight[kRows];
  __shared__ uint32_t qwide[kWaves], last_start;
  const Item it = item_of(p, p.item0, p.items, p.row_blocks);
  if (!it.on) return;
  const Seq& s = p.s[it.seq];
  const TreeArgs& a = p.a;
  const uint32_t R = s.drafts * a.groups, r0 = it.rb * p.block_rows, n = s.rows + s.drafts;
  const uint32_t k0 = it.chunk * p.chunk, k1 = min(k0 + p.chunk, n);
  if (r0 >= R || k0 >= k1) return;
  const uint32_t rows = min(R - r0, p.block_rows), tiles = (rows + 15) / 16;
  const uint32_t tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = l & 15, g = l >> 4;
  const uint32_t kvh = p.kv0 + it.kvh, hd = a.hd;
  const uint64_t off = uint64_t(kvh) * hd;
  const Rows keys(s, s.k, a.k, a.kv_ld, off);
  int32_t x[NSUB][4][4];
  auto load_k = [&](uint32_t key0) {
    const int32_t* src = keys.at(key0 + i);
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
  };
  if (tid < 64) {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t r = tid; r < kRows; r += 64) {
      const Sight v = sight_of(a, s, min(r0 + r, R - 1) / a.groups);
      m = max(m, v.start);
      sight[r] = v;
      rmax[r] = INT32_MIN;
    }
    m = uint32_t(wave_max64(int64_t(m)));
    if (tid == 0) last_start = m;
  }
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
  uint32_t q_all = 0;
  for (uint32_t u = wave; u < tiles * NSUB; u += kWaves) {
    const uint32_t sub = u % NSUB;
    const int32_t* src = q_row(u / NSUB);
    uint32_t d[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int32_t y[4];
      load_q(src, 64 * sub + 16 * j + 4 * g, y);
      uint32_t w[4];
      digits4(y, w, q_all);
#pragma unroll
      for (int q = 0; q < 3; ++q) d[q][j] = w[q];
    }
    v4i* dst = reinterpret_cast<v4i*>(lds) + uint64_t(u) * 3 * 64 + l;
#pragma unroll
    for (int q = 0; q < 3; ++q) dst[q * 64] = v4i{int(d[q][0]), int(d[q][1]), int(d[q][2]), int(d[q][3])};
  }
  const bool q_any = __any(q_all != 0);
  if (l == 0) qwide[wave] = q_any;
  lds_barrier();
  const bool qw = __any(qwide[l % kWaves] != 0);
  const uint32_t id0 = p.id0[it.seq] + it.kvh * R + r0;
  int32_t* sc = p.scores + s.score0 + uint64_t(it.kvh * R + r0) * s.score_ld;
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
  if (AHEAD && k0 + 16 * wave < k1) load_k(k0 + 16 * wave);
  for (uint32_t key0 = k0 + 16 * wave, t = 0; key0 < k1; key0 += 16 * kWaves, ++t) {
    v4i k3[NSUB][3];
    if (!AHEAD) load_k(key0);
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
    if (AHEAD && key0 + 16 * kWaves < k1) load_k(key0 + 16 * kWaves);
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
      const int32_t* src = keys.at(key0 + i);
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

// Terms of long rows: one wave per (row, chunk). 8 rows of 60 K keys: 5.8 us.
__global__ __launch_bounds__(256) void k_tree_terms(Launch p) {
  const uint32_t l = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6), chunk = blockIdx.y;
  if (id >= p.rows) return;
  const uint32_t seq = find_seq(p.id0, p.n_seq, id);
  const Seq& s = p.s[seq];
  const uint32_t R = s.drafts * p.a.groups, local = id - p.id0[seq], n = s.rows + s.drafts;
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
        e = softmax_term(gap, in);
        if (in && gap == 0) first = min(first, k);
        sum += e;
      }
      // (2^32 in 32 bits: all ones, which no other term is)
      if (k < k2) sc[k] = int32_t(to_u32(e));
    }
  }
  sum = double(wave_sum_wrap64(int64_t(sum)));
  first = ~uint32_t(wave_max64(int64_t(~first)));
  if (l == 0) {
    p.psum[uint64_t(id) * p.chunks + chunk] = int64_t(sum);
    p.pfirst[uint64_t(id) * p.chunks + chunk] = first;
    if (chunk == 0) p.ends[id].n_big = 0;
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
__device__ __forceinline__ uint32_t weight_of(uint32_t e, uint32_t m, uint32_t sh, uint32_t& margin) {
  const uint32_t half = 1u << (sh - 1), near = 1u << (sh - 13);
  const uint32_t y = __umulhi(e, m) + half;
  margin = (y & (2 * half - 1)) - near;  // from 2 half - 2 near on: next to a border
  return y >> sh;
}

// Weights of four terms: their digits 0 and 1 (the bytes of (w + 0x8080) ^
// 0x8080), a word each, their sum; keys of weights above 32639 go to `end` (their
// digits are those of w - 65536).
__device__ __forceinline__ uint2 weights4(const uint32_t (&e)[4], const Recip& rc, uint32_t key, int32_t& total, RowEnd* end) {
  uint32_t w[4], margin[4], unsure = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = weight_of(e[q], rc.m, rc.sh, margin[q]);
  const uint32_t border = (1u << rc.sh) - (2u << (rc.sh - 13));
  if (max(max(margin[0], margin[1]), max(margin[2], margin[3])) >= border)
#pragma unroll
    for (int q = 0; q < 4; ++q) unsure |= uint32_t(margin[q] >= border) << q;
#pragma unroll 1
  for (; unsure; unsure &= unsure - 1) {
    const int at = __builtin_ctz(unsure);
    uint32_t x = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) x = q == at ? e[q] : x;
    x = x ? uint32_t(softmax_weight(unpack_term(x), rc.sum)) : 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = q == at ? x : w[q];
  }
  total += int32_t((w[0] + w[1]) + (w[2] + w[3]));
  if (max(max(w[0], w[1]), max(w[2], w[3])) > 32639)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (w[q] > 32639) {
        const uint32_t at = atomicAdd(&end->n_big, 1u);
        if (at == 0) end->big0 = key + q;
        if (at == 1) end->big1 = key + q;
      }
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] += 0x8080u;
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  return make_uint2(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u,
                    __builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
}
// Where they go in a row of digits.
__device__ __forceinline__ void put4(int8_t* row, uint32_t key, uint2 w) {
  uint32_t* o = reinterpret_cast<uint32_t*>(row + (key >> 6) * 128 + (key & 63));
  o[0] = w.x;
  o[16] = w.y;
}
// The residual of a row: what its first maximum gets past its weight, with saturation.
__device__ inline int64_t residual(int64_t total, int64_t sum) {
  const int32_t w = softmax_weight(int64_t(1) << 32, sum);
  return int64_t(add_sat(w, sub_sat(kOneAct, sat32(total)))) - w;
}
// Whole rows: W waves turn a row's scores into weights through LDS, four
// consecutive keys per lane; the weights' digits replace the scores in place (from
// the row's start on). With rows enough to fill the device this reads the scores
// once and writes half their bytes, where terms and weights by chunks read and write
// 2.5 times as much. 4096 rows of 8256 keys: 73 us, bound by about 60 instructions
// per score (its 200 MB are 41 us at a copy's rate).
constexpr uint32_t kRowKeys = 16384;  // most keys of a row (64 KB of terms)
template <int W>
__global__ __launch_bounds__(256) void k_tree_rows(Launch p, uint32_t lds_row) {
  extern __shared__ __attribute__((aligned(16))) uint32_t row_terms[];
  __shared__ double red_sum[4];
  __shared__ uint32_t red_first[4];
  __shared__ int32_t red_total[4];
  __shared__ RowEnd ends[4 / W];
  const uint32_t l = threadIdx.x & 63, wave = threadIdx.x >> 6, in = wave / W, lane = threadIdx.x % (64 * W);
  const uint32_t id = __builtin_amdgcn_readfirstlane(min(blockIdx.x * (4 / W) + in, p.rows - 1));
  const bool on = blockIdx.x * (4 / W) + in < p.rows;
  const uint32_t seq = find_seq(p.id0, p.n_seq, id);
  const Seq& s = p.s[seq];
  const uint32_t R = s.drafts * p.a.groups, local = id - p.id0[seq], n = s.rows + s.drafts, n64 = (n + 63) & ~63u;
  const uint32_t used = (n + p.chunk - 1) / p.chunk;
  int32_t* sc = p.scores + s.score0 + uint64_t(local) * s.score_ld;
  // (each step's scores are loaded before the step that uses the ones before)
  int4 t = 4 * lane < n64 ? *reinterpret_cast<const int4*>(sc + 4 * lane) : make_int4(0, 0, 0, 0);
  int32_t m = INT32_MIN;
  for (uint32_t c = l; c < used; c += 64) m = max(m, p.pmax[uint64_t(id) * p.chunks + c]);
  const Sight v = sight_of(p.a, s, local % R / p.a.groups);
  m = int32_t(wave_max64(m));
  uint32_t* terms = row_terms + in * lds_row;
  if (lane == 0) ends[in].n_big = 0;
  double sum = 0;  // (whole numbers below 2^53: exact in any order)
  uint32_t first = kNone;
  for (uint32_t k = 4 * lane; k < n64; k += 256 * W) {
    const int32_t x[4] = {t.x, t.y, t.z, t.w};
    if (k + 256 * W < n64) t = *reinterpret_cast<const int4*>(sc + k + 256 * W);
    uint32_t e[4];
    // what of the four keys is seen
    uint32_t vis = k >= v.start && k + 4 <= s.rows ? 15u : 0u;
    if (__any(vis == 0)) {
      asm volatile("");
      vis = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) vis |= uint32_t(k + q < n && sees(v, s.rows, k + q)) << q;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t gap = uint32_t(m) - uint32_t(x[q]);
      const bool seen = gap < (1u << 20) && ((vis >> q) & 1u);
      double y = 0;
      if (__any(seen)) {
        y = softmax_term(gap, seen);
        if (__any(gap == 0)) {
          asm volatile("");
          if (seen && gap == 0) first = min(first, k + q);
        }
        sum += y;
      }
      e[q] = to_u32(y);  // (2^32: all ones, which no other term is)
    }
    *reinterpret_cast<uint4*>(terms + k) = make_uint4(e[0], e[1], e[2], e[3]);
  }
  sum = double(wave_sum_wrap64(int64_t(sum)));
  first = ~uint32_t(wave_max64(int64_t(~first)));
  if (l == 0) red_sum[wave] = sum, red_first[wave] = first;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == 0) sum = 0, first = kNone;
    sum += red_sum[in * W + w];
    first = min(first, red_first[in * W + w]);
  }
  const Recip rc = recip_of(int64_t(sum));
  int32_t total = 0;
  for (uint32_t k = 4 * lane; k < n64; k += 256 * W) {
    const uint4 t = *reinterpret_cast<const uint4*>(terms + k);
    const uint32_t e[4] = {t.x, t.y, t.z, t.w};
    const uint2 w = weights4(e, rc, k, total, &ends[in]);
    if (on) put4(reinterpret_cast<int8_t*>(sc), k, w);
  }
  total = int32_t(wave_sum_wrap64(total));
  if (l == 0) red_total[wave] = total;
  __syncthreads();
  if (lane == 0 && on) {
    int64_t all = 0;
    for (int w = 0; w < W; ++w) all += red_total[in * W + w];
    RowEnd end = ends[in];
    end.first = first;
    end.extra = first == kNone ? 0 : residual(all, rc.sum);
    p.ends[id] = end;
  }
}

// Weights of long rows: one wave per (row, chunk). 8 rows of 60 K keys: 4.8 us.
__global__ __launch_bounds__(256) void k_tree_weights(Launch p) {
  const uint32_t l = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6), chunk = blockIdx.y;
  if (id >= p.rows) return;
  const uint32_t seq = find_seq(p.id0, p.n_seq, id);
  const Seq& s = p.s[seq];
  const uint32_t local = id - p.id0[seq], n = s.rows + s.drafts, used = (n + p.chunk - 1) / p.chunk;
  const uint32_t k0 = chunk * p.chunk, k2 = min((min(k0 + p.chunk, n) + 63) & ~63u, s.score_ld);
  if (k0 >= n) return;
  int64_t sum = 0;
  for (uint32_t c = l; c < used; c += 64) sum += p.psum[uint64_t(id) * p.chunks + c];
  const Recip rc = recip_of(wave_sum_wrap64(sum));
  const uint64_t row = s.score0 + uint64_t(local) * s.score_ld;
  int32_t total = 0;
  for (uint32_t k = k0 + 4 * l; k < k2; k += 256) {
    const uint4 t = *reinterpret_cast<const uint4*>(p.scores + row + k);
    const uint32_t e[4] = {t.x, t.y, t.z, t.w};
    put4(p.weights + 2 * row, k, weights4(e, rc, k, total, &p.ends[id]));
  }
  total = int32_t(wave_sum_wrap64(total));
  if (l == 0) p.pweight[uint64_t(id) * p.chunks + chunk] = total;
}

// Weighted sums: a block takes up to 16 RT query rows, one chunk of keys and
// 256 head dims; each wave a group of 32 dims and a split of the keys, 64 of
// them per step. Lane 16 g + i has dims 2 i, 2 i + 1 of the keys 16 g + e (128
// consecutive bytes per key), loaded a step ahead. The weights' digits (128 bytes
// per row and step) come through a ring of three LDS stages, copied two steps
// ahead: 1 KB slots of eight rows, of whose 16-byte pieces piece q of row r lies at
// place q ^ (r >> 1 & 7), so that the 16 rows of an operand read hit different banks.
// DEEP: 64 rows of more than 128 dims, where the 128 sums of a lane leave two waves
// per SIMD: the values come through LDS as well, two steps ahead, and the second half
// of the waves pass each step's barrier after their conversions instead of before, so
// that of a SIMD's two waves one converts while the other multiplies. At 4096 rows of
// 8256 keys of 256 dims that takes 78 us, 89 with all waves in phase, 93 with values
// loaded a step ahead and 122 with the digits loaded by every wave; the bytes alone (67
// MB of digits, 135 of values) take 41. One row of each of 8 heads over 60 K keys (123
// MB): 30 us, 25 at a copy's rate.
constexpr int kStages = 3;
template <int RT, bool DEEP>
__global__ __launch_bounds__(kThreads, 2) void k_tree_wsum(Launch p) {
  extern __shared__ __attribute__((aligned(16))) int8_t ring[];  // [stage][split][row][128]
  const Item it = item_of(p, p.witem0, p.witems, p.sum_blocks);
  if (!it.on) return;
  const Seq& s = p.s[it.seq];
  const TreeArgs& a = p.a;
  const uint32_t R = s.drafts * a.groups, r0 = it.rb * p.sum_rows, n = s.rows + s.drafts;
  const uint32_t c0 = it.chunk * p.wchunk, c1 = min(c0 + p.wchunk, n);
  if (r0 >= R || c0 >= c1) return;  // (workgroup-uniform)
  const uint32_t tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = l & 15, g = l >> 4;
  const uint32_t kvh = p.kv0 + it.kvh, hd = a.hd, splits = p.splits;
  const uint32_t split = wave / p.groups, dim0 = blockIdx.y * kSumDims + 32 * (wave % p.groups);
  // the splits' equal shares of the chunk, in whole steps
  const uint32_t steps = ((c1 - c0 + 63) / 64 + splits - 1) / splits;
  const uint32_t k0 = c0 + split * steps * 64, k1 = min(k0 + steps * 64, c1);
  const bool on = split < splits && dim0 < hd && k0 < k1;
  const uint32_t rows = min(R - r0, p.sum_rows), id0 = p.id0[it.seq] + it.kvh * R + r0;
  const uint64_t off = uint64_t(kvh) * hd;
  const Rows values(s, s.v, a.v, a.kv_ld, off);
  const uint32_t dim = dim0 + 2 * i, dim_in = dim + 1 < hd ? dim : (hd > 1 ? hd - 2 : 0);  // (sums of dims past hd are dropped)
  const uint32_t run_off = 16 * g * uint32_t(s.ld) + dim_in;
  auto load_v = [&](uint32_t k, int32_t (&x)[16][2]) {
    uint64_t at = s.first + k;
    if (s.wrap && at >= s.wrap) at -= s.wrap;
    if (p.wide_v && k + 64 <= s.rows && (!s.wrap || at + 64 <= s.wrap) && s.ld < (1u << 22)) {
      // one run of cached rows: scalar row addresses
      const int32_t* base = s.v + at * s.ld + off;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        typedef int v2 __attribute__((ext_vector_type(2)));
        const v2 t = *(global_ptr<const v2>)(to_global(base + e * s.ld) + run_off);
        x[e][0] = t.x, x[e][1] = t.y;
      }
      return;
    }
    // (weights are zero from the row's end on)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int32_t* row = values.at(min(k + 16 * g + e, n - 1));
      if (p.wide_v) {
        typedef int v2 __attribute__((ext_vector_type(2)));
        const v2 t = *(global_ptr<const v2>)(to_global(row) + dim_in);
        x[e][0] = t.x, x[e][1] = t.y;
      } else {
        x[e][0] = to_global(row)[min(dim, hd - 1)];
        x[e][1] = to_global(row)[min(dim + 1, hd - 1)];
      }
      if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (four rows' addresses at a time)
    }
  };
  // this lane's pieces of the digits of step `st`: slot c of a split's 2 RT has rows 8 c ..
  const uint64_t wrow = s.score0 + uint64_t(it.kvh * R + r0) * s.score_ld;
  const int8_t* wbase = p.whole ? reinterpret_cast<const int8_t*>(p.scores + wrow) : p.weights + 2 * wrow;
  const uint32_t wld = (p.whole ? 4 : 2) * s.score_ld;
  const uint32_t slots = splits * RT * 2;
  auto copy_w = [&](uint32_t st) {
    for (uint32_t c = wave; c < slots; c += kWaves) {
      const uint32_t r = 8 * (c % (2 * RT)) + l / 8, q = (l % 8) ^ (r >> 1 & 7);
      // (rows past the last and steps past a share: in range, not used)
      const uint32_t key = min(c0 + (c / (2 * RT) * steps + st) * 64, (n - 1) & ~63u);
      __builtin_amdgcn_global_load_lds(
          (const void __attribute__((address_space(1)))*)(wbase + uint64_t(min(r, rows - 1)) * wld + 2 * key + 16 * q),
          (void __attribute__((address_space(3)))*)(ring + ((st % kStages) * slots + c) * kOp), 16, 0, 0);
    }
  };
  // DEEP: the wave's values of step `st`, into one of two LDS stages: 128 bytes per
  // key (16 per lane, eight keys per copy), keys 16 g + e with odd g at place 16 g +
  // (e ^ 1), so that two groups of lanes read from different banks
  constexpr uint32_t kValueBytes = 64 * 128;
  int8_t* vring = ring + kStages * slots * kOp;
  const uint32_t piece = min(dim0 + 4 * (l % 8), hd >= 4 ? hd - 4 : 0);
  auto copy_v = [&](uint32_t st) {
    const uint32_t k = k0 + 64 * st;
    int8_t* dst = vring + ((st & 1) * kWaves + wave) * kValueBytes;
    uint64_t at = s.first + k;
    if (s.wrap && at >= s.wrap) at -= s.wrap;
    const bool run = k + 64 <= s.rows && (!s.wrap || at + 64 <= s.wrap) && s.ld < (1u << 22);
    const int32_t* base = s.v + at * s.ld + off;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
      const uint32_t key = (l / 8) ^ (e / 2 & 1);
      const int32_t* src = run ? base + 8 * e * s.ld + (key * uint32_t(s.ld) + piece)
                               : values.at(min(k + 8 * e + key, n - 1)) + piece;
      __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)src,
                                       (void __attribute__((address_space(3)))*)(dst + e * kOp), 16, 0, 0);
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
  // digit q of the 16 weights of row 16 T + i from key 16 g on, of stage `st`
  const uint32_t place = split * RT * 2 * kOp + i * 128;
  auto weights = [&](uint32_t st, int T, int q) {
    return *reinterpret_cast<const v4i*>(ring + (st % kStages) * slots * kOp + place + T * 2048 +
                                         16 * ((4 * q + g) ^ (i >> 1)));
  };
  v4i acc[RT][2][4];
#pragma unroll
  for (int T = 0; T < RT; ++T)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[T][c][q] = v4i{0, 0, 0, 0};
  int32_t x[16][2] = {};
  uint32_t all = 0;
  // every copy and load that a wave has in flight, then the workgroup
  auto step_barrier = [&] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0 | (7 << 4));  // vmcnt 0, lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // (DEEP: one share, so that a wave is on in every step or in none; nine copies a step, or one)
  if (DEEP && on) copy_v(0);
  copy_w(0);
  if (DEEP && on && steps > 1) copy_v(1);
  if (steps > 1) copy_w(1);
  if (!DEEP && on) load_v(k0, x);
#pragma unroll 1
  for (uint32_t st = 0; st < steps; ++st) {
    const uint32_t k = k0 + 64 * st;
    v4i d[2][4];
    if (DEEP) {
      // this step's copies; the next one's may be on their way
      asm volatile("" ::: "memory");
      if (st + 1 == steps) __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (15 << 8));
      else if (on) __builtin_amdgcn_s_waitcnt(9 | (7 << 4) | (15 << 8));
      else __builtin_amdgcn_s_waitcnt(1 | (7 << 4) | (15 << 8));
      if (wave < kWaves / 2) __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int8_t* src = vring + ((st & 1) * kWaves + wave) * kValueBytes + 8 * i;
#pragma unroll
      for (uint32_t e = 0; e < 16; ++e) {
        const int2 t = *reinterpret_cast<const int2*>(src + ((16 * g + e) ^ (g & 1)) * 128);
        x[e][0] = t.x, x[e][1] = t.y;
      }
    }
    digit_words(x, 0, d[0], all);
    digit_words(x, 1, d[1], all);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int q = 0; q < 3; ++q) asm volatile("" : "+v"(d[c][q]));
    if (DEEP) {
      asm volatile("" ::: "memory");
      if (on && st + 2 < steps) copy_v(st + 2);
      if (wave >= kWaves / 2) __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (st + 2 < steps) copy_w(st + 2);
    } else {
      step_barrier();
      if (st + 2 < steps) copy_w(st + 2);
      if (on && k + 64 < k1) load_v(k + 64, x);
    }
    if (on && k < k1)
#pragma unroll
      for (int T = 0; T < RT; ++T) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const v4i w = weights(st, T, q);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 3; ++j)
              acc[T][c][q + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, d[c][j], acc[T][c][q + j], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  // lane l, component r: row 16 T + 4 g + r, dims dim and dim + 1
  const bool planes_on = split < splits && dim0 < hd;
  int64_t* out = p.planes + (uint64_t(it.chunk * splits + split) * p.rows + id0) * hd;
  // the first `count` sums, sum q at digit q + shift
  auto put = [&](auto count, auto shift, bool add) {
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
        if (planes_on && row < rows && dim < hd) *o = int64_t((add ? uint64_t(*o) : 0) + y[0]);
        if (planes_on && row < rows && dim + 1 < hd) o[1] = int64_t((add ? uint64_t(o[1]) : 0) + y[1]);
      }
  };
  put(std::integral_constant<int, 4>(), std::integral_constant<int, 0>(), false);
  if (!__syncthreads_or(all != 0)) return;
  // a value of the block's is not narrow: digits 3 and 4, in a pass of their own
#pragma unroll
  for (int T = 0; T < RT; ++T)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int q = 0; q < 3; ++q) acc[T][c][q] = v4i{0, 0, 0, 0};
#pragma unroll 1
  for (uint32_t st = 0; st < steps; ++st) {
    const uint32_t k = k0 + 64 * st;
    __syncthreads();
    copy_w(st);
    if (on && k < k1) load_v(k, x);
    step_barrier();
    if (!on || k >= k1) continue;
    v4i d[2][4], t[2];
    uint32_t unused = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      digit_words(x, c, d[c], unused);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t y[4] = {x[4 * j][c], x[4 * j + 1][c], x[4 * j + 2][c], x[4 * j + 3][c]};
        t[c][j] = int(top4(y));
      }
    }
#pragma unroll
    for (int T = 0; T < RT; ++T)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const v4i w = weights(st, T, q);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          acc[T][c][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, d[c][3], acc[T][c][q], 0, 0, 0);
          acc[T][c][q + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, t[c], acc[T][c][q + 1], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  put(std::integral_constant<int, 3>(), std::integral_constant<int, 3>(), true);
}

// Join: a wave per (row, 64 dims), or four with a share of the planes each where
// there are many. 4096 rows of 256 dims of four planes: 11.5 us for 38 MB, a wave's
// few reads one after the other.
template <int SHARES>
__global__ __launch_bounds__(256) void k_tree_join(Launch p) {
  const uint32_t l = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t id = blockIdx.x;
  const uint32_t seq = find_seq(p.id0, p.n_seq, id);
  const Seq& s = p.s[seq];
  const TreeArgs& a = p.a;
  const uint32_t R = s.drafts * a.groups, local = id - p.id0[seq], n = s.rows + s.drafts;
  const uint32_t kvh = p.kv0 + local / R, row = local % R, used = (n + p.chunk - 1) / p.chunk;
  const uint32_t wused = (n + p.wchunk - 1) / p.wchunk;
  RowEnd end = p.ends[id];
  if (!p.whole) {
    int64_t total = 0, sum = 0;
    uint32_t first = kNone;
    for (uint32_t c = l; c < used; c += 64) {
      sum += p.psum[uint64_t(id) * p.chunks + c];
      first = min(first, p.pfirst[uint64_t(id) * p.chunks + c]);
      total += p.pweight[uint64_t(id) * p.chunks + c];
    }
    sum = wave_sum_wrap64(sum);
    total = wave_sum_wrap64(total);
    end.first = ~uint32_t(wave_max64(int64_t(~first)));
    end.extra = end.first == kNone ? 0 : residual(total, sum);
  }
  int32_t* out = a.out + (s.row0 + row / a.groups) * a.out_ld + uint64_t(kvh * a.groups + row % a.groups) * a.hd;
  const uint64_t off = uint64_t(kvh) * a.hd;
  const Rows values(s, s.v, a.v, a.kv_ld, off);
  const int32_t* v = values.at(min(end.first, n - 1));
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
  if (d >= a.hd) return;
  y += uint64_t(end.extra * to_global(v)[d]);
  if (end.n_big > 0) y += uint64_t(int64_t(to_global(values.at(end.big0))[d])) << 16;
  if (end.n_big > 1) y += uint64_t(int64_t(to_global(values.at(end.big1))[d])) << 16;
  out[d] = end.first == kNone ? 0 : requant(int64_t(y));
}

uint64_t up(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

// One launch group: sequences [b0, b1), kv heads [kv0, kv0 + nkv).
struct Group {
  uint32_t b0, b1, kv0, nkv;
};
constexpr uint64_t kScoreBytes = uint64_t(256) << 20;  // score rows of a group (the Infinity Cache)

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

// Keys per chunk, in whole granules (at most 16384 keys, which bounds the int32
// sums and a wave's key tiles): the share of the longest sequence, among some, that
// ends first when the device runs `want` blocks at a time, each for its chunk and
// `extra` keys' time besides. An item has `per_item` blocks, those past a sequence's
// own rows too (they wait for a place as the others do).
uint32_t chunk_of(const Launch& p, uint64_t keys, uint64_t per_item, uint64_t want, uint32_t granule, uint32_t extra) {
  const uint64_t even = std::max<uint64_t>(want / (p.n_seq * p.nkv * per_item), 1);
  uint64_t best = 0, least = UINT64_MAX, last = 0;
  for (uint64_t n = even; n <= 4 * even; n += (even + 3) / 4) {
    const uint64_t c = std::min<uint64_t>(up((keys + n - 1) / n, granule), 16384 / granule * granule);
    if (c == last) continue;
    last = c;
    uint64_t blocks = 0;
    for (uint32_t b = 0; b < p.n_seq; ++b) blocks += (uint64_t(p.s[b].rows) + p.s[b].drafts + c - 1) / c;
    blocks *= p.nkv * per_item;
    const uint64_t cost = (blocks + want - 1) / want * (std::min(c, keys) + extra);
    if (cost < least) least = cost, best = c;
  }
  return uint32_t(best);
}

// The launch of a group without its scratch pointers; returns the scratch's bytes.
uint64_t plan(const TreeArgs& a, const TreeSeq* seqs, const Group& g, Launch& p) {
  p = Launch{};
  p.a = a;
  p.kv0 = g.kv0;
  p.nkv = g.nkv;
  p.n_seq = g.b1 - g.b0;
  uint64_t scores = 0, keys = 0;
  uint32_t most = 0;
  auto aligned = [](const void* q, uint64_t to) { return reinterpret_cast<uintptr_t>(q) % to == 0; };
  bool w4 = a.hd % 4 == 0 && a.q_ld % 4 == 0 && a.kv_ld % 4 == 0 && aligned(a.q, 16) && aligned(a.k, 16);
  bool w2 = a.hd % 2 == 0 && a.kv_ld % 2 == 0 && aligned(a.v, 8);
  bool v4 = a.hd % 4 == 0 && a.kv_ld % 4 == 0 && aligned(a.v, 16);
  for (uint32_t b = g.b0; b < g.b1; ++b) {
    const TreeSeq& t = seqs[b];
    Seq& s = p.s[b - g.b0];
    s = {t.k, t.v, t.ld, t.first, t.wrap, t.row0, scores, t.rows, t.drafts, score_ld(t)};
    p.id0[b - g.b0] = p.rows;
    if (t.rows) {
      w4 = w4 && t.ld % 4 == 0 && aligned(t.k, 16);
      w2 = w2 && t.ld % 2 == 0 && aligned(t.v, 8);
      v4 = v4 && t.ld % 4 == 0 && aligned(t.v, 16);
    }
    const uint32_t R = t.drafts * a.groups;
    p.rows += R * g.nkv;
    scores += uint64_t(R) * g.nkv * s.score_ld;
    keys = std::max<uint64_t>(keys, s.score_ld);
    most = std::max(most, R);
  }
  p.wide_k = w4;
  p.wide_v = w2;
  p.deep_v = v4 && a.hd > 128;
  // 64 query rows per block, 128 with loads a step ahead; 32 where their digits or
  // their sums' registers would leave the device half empty
  p.block_rows = std::min<uint32_t>(uint32_t(up(most, 16)), a.hd <= 256 ? (most > 64 && w4 ? 128 : 64) : 32);
  p.row_blocks = (most + p.block_rows - 1) / p.block_rows;
  p.chunk = chunk_of(p, keys, p.row_blocks, p.block_rows > 64 ? 256 : 512, 16 * kWaves, 256);
  p.chunks = uint32_t((keys + p.chunk - 1) / p.chunk);
  // (28 rows of 3000 keys 32 us whole and 34 by chunks, of 6000 39 and 39, of 15000
  // 51 and 46; 160 rows of 15000 84 and 86)
  p.whole = keys <= kRowKeys && (p.rows >= 256 || keys <= 4096);
  p.groups = a.hd <= 32 ? 1 : a.hd <= 64 ? 2 : a.hd <= 128 ? 4 : 8;
  p.splits = kWaves / p.groups;
  p.sum_rows = std::min<uint32_t>(uint32_t(up(most, 16)), a.hd <= 64 ? 32 : 64);
  p.sum_blocks = (most + p.sum_rows - 1) / p.sum_rows;
  p.wchunk = chunk_of(p, keys, uint64_t(p.sum_blocks) * ((a.hd + kSumDims - 1) / kSumDims), 256, 64, 128);
  p.splits = std::min(p.splits, p.wchunk / 64);
  p.wchunks = uint32_t((keys + p.wchunk - 1) / p.wchunk);
  for (uint32_t b = 0; b < p.n_seq; ++b) {
    const uint64_t n = uint64_t(p.s[b].rows) + p.s[b].drafts;
    p.item0[b] = p.items, p.witem0[b] = p.witems;
    p.items += g.nkv * uint32_t((n + p.chunk - 1) / p.chunk);
    p.witems += g.nkv * uint32_t((n + p.wchunk - 1) / p.wchunk);
  }
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
  p.pweight = reinterpret_cast<int32_t*>(take(uint64_t(p.rows) * p.chunks * 4));
  p.ends = reinterpret_cast<RowEnd*>(take(uint64_t(p.rows) * sizeof(RowEnd)));
  p.weights = reinterpret_cast<int8_t*>(take(p.whole ? 0 : scores * 2));
  return at;
}

template <int NSUB>
void launch_scores(const Launch& p, uint32_t blocks, hipStream_t s) {
  const uint32_t lds = p.block_rows / 16 * NSUB * 3 * kOp;
  auto go = [&](auto kernel) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), lds, s, p);
  };
  if constexpr (NSUB <= 4)
    if (p.block_rows > 64) {
      if (p.a.hd == 64 * NSUB) go(&k_tree_scores<NSUB, kWhole, true>);
      else go(&k_tree_scores<NSUB, kVec4, true>);
      return;
    }
  if (!p.wide_k) go(&k_tree_scores<NSUB, kScalar, false>);
  else if (p.a.hd == 64 * NSUB) go(&k_tree_scores<NSUB, kWhole, false>);
  else go(&k_tree_scores<NSUB, kVec4, false>);
}
template <int RT>
void launch_wsum(const Launch& p, uint32_t blocks, hipStream_t s) {
  const uint32_t lds = kStages * p.splits * RT * 2 * kOp;
  auto go = [&](auto kernel, uint32_t bytes) {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 156 << 10);
    hipLaunchKernelGGL(kernel, dim3(blocks, (p.a.hd + kSumDims - 1) / kSumDims), dim3(kThreads), bytes, s, p);
  };
  if constexpr (RT == 4)
    if (p.deep_v) return go(&k_tree_wsum<RT, true>, lds + 2 * kWaves * 8192);
  go(&k_tree_wsum<RT, false>, lds);
}
void launch_rows(const Launch& p, hipStream_t s) {
  uint32_t ld = 0;
  for (uint32_t b = 0; b < p.n_seq; ++b) ld = std::max(ld, p.s[b].score_ld);
  if (ld <= 1024) {
    hipLaunchKernelGGL(k_tree_rows<1>, dim3((p.rows + 3) / 4), dim3(256), 4 * ld * 4, s, p, ld);
  } else {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&k_tree_rows<4>), hipFuncAttributeMaxDynamicSharedMemorySize,
                              kRowKeys * 4);
    hipLaunchKernelGGL(k_tree_rows<4>, dim3(p.rows), dim3(256), ld * 4, s, p, ld);
  }
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
    place(p.ends), place(p.weights);
    const uint32_t score_blocks = uint32_t(up(p.items, 8)) * p.row_blocks, sum_blocks = uint32_t(up(p.witems, 8)) * p.sum_blocks;
    const uint32_t nsub = (a.hd + 63) / 64;
    if (nsub == 1) launch_scores<1>(p, score_blocks, s);
    else if (nsub == 2) launch_scores<2>(p, score_blocks, s);
    else if (nsub == 3) launch_scores<3>(p, score_blocks, s);
    else if (nsub == 4) launch_scores<4>(p, score_blocks, s);
    else launch_scores<8>(p, score_blocks, s);
    if (p.whole) {
      launch_rows(p, s);
    } else {
      hipLaunchKernelGGL(k_tree_terms, dim3((p.rows + 3) / 4, p.chunks), dim3(256), 0, s, p);
      hipLaunchKernelGGL(k_tree_weights, dim3((p.rows + 3) / 4, p.chunks), dim3(256), 0, s, p);
    }
    if (p.sum_rows <= 16) launch_wsum<1>(p, sum_blocks, s);
    else if (p.sum_rows <= 32) launch_wsum<2>(p, sum_blocks, s);
    else launch_wsum<4>(p, sum_blocks, s);
    if (p.wchunks * p.splits > 16)
      hipLaunchKernelGGL(k_tree_join<4>, dim3(p.rows, (a.hd + 63) / 64), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL(k_tree_join<1>, dim3(p.rows, (a.hd + 255) / 256), dim3(256), 0, s, p);
  });
}

}  // namespace det
