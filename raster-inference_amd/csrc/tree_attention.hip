// Attention of drafted rows over caches.
//
// Row i of a sequence sees its cached rows from start_i on and the drafted
// rows of its mask, in this order: s_r = requant(q . k_r), the integer softmax
// of the scores (terms exp(s_r - max) in Q32.32, weights requant(term / sum),
// the residual to 65536 added to the first maximum), out = requant(sum w_r v_r),
// all sums exact in wrapping 64-bit integers.
#include <hip/hip_runtime.h>

#include "det_arith.h"
#include "verify.h"
#include "wave.h"

namespace det {

namespace {

constexpr uint32_t kSeqs = 40;  // sequences per launch (by value in the arguments)
struct SeqBlock {
  TreeSeq s[kSeqs];
};
constexpr int kThreads = 256;

__device__ inline uint64_t cache_row(const TreeSeq& s, uint32_t r) {
  const uint64_t p = s.first + r;
  return s.wrap && p >= s.wrap ? p - s.wrap : p;
}

__device__ inline int64_t block_reduce_add(int64_t v, int64_t* red) {
  v = wave_sum_wrap64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int64_t r = 0;
  for (int w = 0; w < kThreads / 64; ++w) r += red[w];
  return r;
}
__device__ inline int64_t block_reduce_max(int64_t v, int64_t* red) {
  v = wave_max64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int64_t r = red[0];
  for (int w = 1; w < kThreads / 64; ++w) r = r > red[w] ? r : red[w];
  return r;
}

// One workgroup per (drafted row, head): scores into the work area, the three
// softmax passes over them, then a thread per output dim.
__global__ __launch_bounds__(kThreads) void k_tree_simple(TreeArgs a, SeqBlock b, int32_t* work, uint64_t work_ld) {
  __shared__ int64_t red[kThreads / 64];
  const TreeSeq& s = b.s[blockIdx.z];
  const uint32_t h = blockIdx.x, i = blockIdx.y, kvh = h / a.groups, hd = a.hd, tid = threadIdx.x;
  if (i >= s.drafts) return;
  const uint64_t row = s.row0 + i;
  const uint64_t mask = a.masks[row] & (s.drafts == 64 ? ~0ull : (1ull << s.drafts) - 1);
  uint32_t start = a.starts ? a.starts[row] : 0;
  if (start > s.rows) start = s.rows;
  const uint32_t cached = s.rows - start, n = cached + __popcll(mask);
  int32_t* out = a.out + row * a.out_ld + uint64_t(h) * hd;
  if (n == 0) {
    for (uint32_t d = tid; d < hd; d += kThreads) out[d] = 0;
    return;
  }
  auto drafted = [&](uint32_t j) {  // the j-th set bit
    uint64_t m = mask;
    for (uint32_t q = 0; q < j; ++q) m &= m - 1;
    return s.row0 + uint32_t(__builtin_ctzll(m));
  };
  auto key = [&](uint32_t r, const int32_t* c, const int32_t* d) {
    return (r < cached ? c + cache_row(s, start + r) * s.ld : d + drafted(r - cached) * a.kv_ld) + uint64_t(kvh) * hd;
  };
  const int32_t* q = a.q + row * a.q_ld + uint64_t(h) * hd;
  int32_t* w = work + (row * a.nh + h) * work_ld;
  int64_t best = INT64_MIN;
  for (uint32_t r = tid; r < n; r += kThreads) {
    const int32_t* k = key(r, s.k, a.k);
    int64_t acc = 0;
    for (uint32_t d = 0; d < hd; ++d) acc = mac(acc, q[d], k[d]);
    const int32_t x = requant(acc);
    w[r] = x;
    const int64_t cand = (int64_t(x) << 32) | int64_t(0xffffffffu - r);
    best = cand > best ? cand : best;
  }
  best = block_reduce_max(best, red);
  const int32_t mx = int32_t(best >> 32);
  const uint32_t first = 0xffffffffu - uint32_t(best);
  int64_t sum = 0;
  for (uint32_t r = tid; r < n; r += kThreads) sum += softmax_exp(w[r], mx);
  sum = block_reduce_add(sum, red);
  int64_t tot = 0;
  for (uint32_t r = tid; r < n; r += kThreads) {
    const int32_t x = softmax_weight(softmax_exp(w[r], mx), sum);
    w[r] = x;
    tot += x;
  }
  tot = block_reduce_add(tot, red);
  __syncthreads();
  if (tid == 0) w[first] = add_sat(w[first], sub_sat(kOneAct, sat32(tot)));
  __syncthreads();
  for (uint32_t d = tid; d < hd; d += kThreads) {
    int64_t acc = 0;
    for (uint32_t r = 0; r < n; ++r) acc = mac(acc, key(r, s.v, a.v)[d], w[r]);
    out[d] = requant(acc);
  }
}

}  // namespace

static uint64_t tree_ld(const TreeSeq* seqs, uint32_t n) {
  uint64_t most = 0;
  for (uint32_t i = 0; i < n; ++i) most = seqs[i].rows > most ? seqs[i].rows : most;
  return (most + kTreeMaxDrafts + 63) / 64 * 64;
}
uint64_t tree_work_bytes(const TreeArgs& a, const TreeSeq* seqs, uint32_t n) {
  uint64_t rows = 0;
  for (uint32_t i = 0; i < n; ++i) rows += seqs[i].drafts;
  return rows * a.nh * tree_ld(seqs, n) * 4;
}
void launch_tree_attention(const TreeArgs& a, const TreeSeq* seqs, uint32_t n, void* work, hipStream_t s) {
  const uint64_t ld = tree_ld(seqs, n);
  for (uint32_t i = 0; i < n; i += kSeqs) {
    SeqBlock b{};
    uint32_t c = 0, most = 0;
    for (; c < kSeqs && i + c < n; ++c) {
      b.s[c] = seqs[i + c];
      most = seqs[i + c].drafts > most ? seqs[i + c].drafts : most;
    }
    if (most) hipLaunchKernelGGL(k_tree_simple, dim3(a.nh, most, c), dim3(kThreads), 0, s, a, b, static_cast<int32_t*>(work), ld);
  }
}

}  // namespace det
