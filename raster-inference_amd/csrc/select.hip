// Decoding rules on logits and the choice of the next tokens.
//
// x' = sat(rep(x) - c frequency - [c > 0] presence + sum of biases) with c the
// token's count in the row's history, i32::MIN where the mask forbids it, then
// the first maximum among the allowed tokens.
#include <hip/hip_runtime.h>

#include "det_arith.h"
#include "verify.h"
#include "wave.h"

namespace det {

namespace {

constexpr uint32_t kThreads = 512;
constexpr uint32_t kQuads = 2;                     // groups of four tokens per thread
constexpr uint32_t kSpan = kThreads * 4 * kQuads;  // tokens per workgroup
constexpr uint32_t kBatch = 4;                // history ids of a thread in flight

// A row's choice so far: value (offset to unsigned) over the inverted index,
// so that the larger key is the larger value, then the lower index; 0: none.
__device__ inline uint64_t choice_key(int32_t x, uint32_t token) {
  return (uint64_t(uint32_t(x) ^ 0x80000000u) << 32) | uint64_t(0xffffffffu - token);
}
struct OpMaxU64 {
  __device__ __forceinline__ uint64_t operator()(uint64_t p, uint64_t q) const { return p > q ? p : q; }
};

// One workgroup per row and 4096 tokens, eight tokens per thread, whose
// logits and mask bits are loaded before the rules are looked at. A token that
// a rule names has its bit in `named` (history: `seen`) and its sum in `sum`:
// minus its penalties, plus its biases; only those entries are ever written or
// read. Bound by the logits' bytes: 208 rows of 262144 tokens with histories,
// biases and masks, adjusted logits written, 117 us, where copying them takes 81;
// one row 6 us, a latency or two above an empty launch.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void k_select(SelectArgs a, uint64_t* keys, uint32_t parts) {
  __shared__ unsigned long long sum[kSpan];
  __shared__ uint32_t seen[kSpan / 32], named[kSpan / 32];
  __shared__ uint64_t red[kThreads / 64];
  const uint32_t tid = threadIdx.x, part = blockIdx.x;
  const uint64_t r = blockIdx.y, base = uint64_t(part) * kSpan;
  const uint32_t span = uint32_t(a.vocab - base < kSpan ? a.vocab - base : kSpan);
  // the rules' extents, then everything the workgroup reads in one go: its
  // share of the history and the biases, its logits and mask bits
  const bool penal = a.penalties && a.spans && a.ids, biased = a.bias_begin && a.bias_ids && a.bias_values;
  const uint32_t* spans = a.spans + r * a.spans_per_row * 2;
  const uint32_t n_ids = uint32_t(a.n_ids), n_bias = uint32_t(a.n_bias);  // (at most 2^28)
  uint32_t total = 0, b0 = 0, b1 = 0;
  SelectPenalty p{kOneAct, 0, 0};
  if (penal) {
    p = a.penalties[r];
    for (uint32_t s = 0; s < a.spans_per_row; ++s) {
      const uint32_t lo = spans[2 * s], hi = min(spans[2 * s + 1], n_ids);
      total += hi > lo ? hi - lo : 0;
    }
  }
  if (biased) {
    b1 = min(a.bias_begin[r + 1], n_bias);
    b0 = min(a.bias_begin[r], b1);
  }
  // the batch of the row's history from entry `from` on (its spans one after the
  // other): offsets into this part, kSpan for other parts' tokens
  auto load_ids = [&](uint32_t from, uint32_t (&id)[kBatch]) {
    uint32_t u[kBatch], at[kBatch];
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) u[b] = from + tid + kThreads * b, at[b] = 0xffffffffu;
    for (uint32_t s = 0; s < a.spans_per_row; ++s) {
      const uint32_t lo = spans[2 * s], hi = min(spans[2 * s + 1], n_ids), len = hi > lo ? hi - lo : 0;
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        const bool in = u[b] < len;
        if (in) at[b] = lo + u[b];
        u[b] = in ? 0xffffffffu : u[b] - len;  // (stays above every length)
      }
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) id[b] = a.ids[min(at[b], n_ids - 1)];  // (n_ids > 0 here)
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) id[b] = at[b] < n_ids ? id[b] : 0xffffffffu;
  };
  auto offsets = [&](uint32_t (&id)[kBatch]) {
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      const uint32_t o = id[b] - uint32_t(base);  // (ids below the part wrap past it)
      id[b] = o < span ? o : kSpan;
    }
  };
  uint32_t id[kBatch], bias_id = 0xffffffffu;
  int32_t bias_value = 0;
  if (total) load_ids(0, id);
  if (b0 + tid < b1) bias_id = a.bias_ids[b0 + tid], bias_value = a.bias_values[b0 + tid];
  const int32_t* src = a.logits + r * a.ld + base;
  int32_t x[kQuads][4];
  uint32_t bits[kQuads];
  // (a wave's 256 tokens of one quad group are eight words of the mask: lane 8 q +
  // w loads word w of group q, and each lane takes its four bits from there below)
  uint32_t word = 0;
  if (a.mask) {
    const uint32_t l = tid & 63, t = 4 * (tid - l + kThreads * (l / 8 % kQuads)) + 32 * (l % 8);
    word = a.mask[r * a.mask_ld + (base + min(t, span - 1)) / 32];
  }
  if (VEC && span == kSpan) {  // (workgroup-uniform)
#pragma unroll
    for (uint32_t q = 0; q < kQuads; ++q) {
      const int4 v = *reinterpret_cast<const int4*>(src + 4 * (tid + kThreads * q));
      x[q][0] = v.x, x[q][1] = v.y, x[q][2] = v.z, x[q][3] = v.w;
    }
  } else {
#pragma unroll
    for (uint32_t q = 0; q < kQuads; ++q)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) x[q][e] = src[min(4 * (tid + kThreads * q) + e, span - 1)];
  }
  if (total || b0 < b1) {
    for (uint32_t i = tid; i < kSpan / 32; i += kThreads) seen[i] = named[i] = 0;
    constexpr uint32_t kStep = kThreads * kBatch;
    if (total) offsets(id);
    lds_barrier();
    // the named tokens' sums start at zero
    auto name = [&](uint32_t o, uint32_t* set) {
      sum[o] = 0;
      atomicOr(&set[o / 32], 1u << (o % 32));
    };
    for (uint32_t from = 0; from < total; from += kStep) {
      if (from) load_ids(from, id), offsets(id);
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b)
        if (id[b] < kSpan) name(id[b], seen);
    }
    if (bias_id - uint32_t(base) < span) name(bias_id - uint32_t(base), named);
    for (uint32_t i = b0 + kThreads + tid; i < b1; i += kThreads)
      if (a.bias_ids[i] - uint32_t(base) < span) name(a.bias_ids[i] - uint32_t(base), named);
    lds_barrier();
    const auto minus = static_cast<unsigned long long>(-int64_t(p.frequency));
    for (uint32_t from = 0; from < total; from += kStep) {
      if (total > kStep) load_ids(from, id), offsets(id);
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b)
        if (id[b] < kSpan) atomicAdd(&sum[id[b]], minus);
    }
    auto raise = [&](uint32_t o, int32_t v) { atomicAdd(&sum[o], static_cast<unsigned long long>(int64_t(v))); };
    if (bias_id - uint32_t(base) < span) raise(bias_id - uint32_t(base), bias_value);
    for (uint32_t i = b0 + kThreads + tid; i < b1; i += kThreads)
      if (a.bias_ids[i] - uint32_t(base) < span) raise(a.bias_ids[i] - uint32_t(base), a.bias_values[i]);
    lds_barrier();
#pragma unroll
    for (uint32_t q = 0; q < kQuads; ++q) {
      const uint32_t t = 4 * (tid + kThreads * q), old = seen[t / 32] >> (t % 32), any = old | (named[t / 32] >> (t % 32));
      if (!(any & 15u)) continue;
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        if (!((any >> e) & 1u)) continue;
        int32_t v = x[q][e];
        int64_t add = int64_t(sum[t + e]);
        if ((old >> e) & 1u) {
          if (p.repetition > 0 && p.repetition != kOneAct) v = v > 0 ? div_act(v, p.repetition) : mul_sat(v, p.repetition);
          add -= p.presence;
        }
        x[q][e] = sat32(int64_t(v) + add);
      }
    }
  }
#pragma unroll
  for (uint32_t q = 0; q < kQuads; ++q) {
    const uint32_t t = 4 * (tid + kThreads * q);
    bits[q] = a.mask ? uint32_t(__shfl(int(word), int(8 * q + (tid & 63) / 8), 64)) >> (t % 32) : 15u;
    if (t + 4 > span) bits[q] &= t < span ? (1u << (span - t)) - 1 : 0u;
  }
  uint64_t best = 0;
  int32_t* dst = a.out ? a.out + r * a.out_ld + base : nullptr;
#pragma unroll
  for (uint32_t q = 0; q < kQuads; ++q) {
    const uint32_t t = 4 * (tid + kThreads * q);
    uint32_t at = 4;
    int32_t top = INT32_MIN;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      const bool ok = (bits[q] >> e) & 1u;
      if (!ok) x[q][e] = INT32_MIN;
      if (ok && (at == 4 || x[q][e] > top)) top = x[q][e], at = e;
    }
    if (at < 4) {
      const uint64_t k = choice_key(top, uint32_t(base) + t + at);
      best = k > best ? k : best;
    }
    if (!dst) continue;
    if (VEC && t + 4 <= span) {
      *reinterpret_cast<int4*>(dst + t) = make_int4(x[q][0], x[q][1], x[q][2], x[q][3]);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (t + e < span) dst[t + e] = x[q][e];
    }
  }
  if (!keys) return;
  best = wave_reduce(best, OpMaxU64());
  if ((tid & 63) == 0) red[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < int(kThreads / 64); ++w) best = red[w] > best ? red[w] : best;
    keys[r * parts + part] = best;
  }
}

__global__ __launch_bounds__(64) void k_select_final(const uint64_t* keys, uint32_t parts, uint32_t* tokens) {
  uint64_t best = 0;
  for (uint32_t i = threadIdx.x; i < parts; i += 64) {
    const uint64_t k = keys[uint64_t(blockIdx.x) * parts + i];
    best = k > best ? k : best;
  }
  best = wave_reduce(best, OpMaxU64());
  if (threadIdx.x == 0) tokens[blockIdx.x] = best ? 0xffffffffu - uint32_t(best) : 0xffffffffu;
}

uint32_t parts_of(const SelectArgs& a) { return uint32_t((a.vocab + kSpan - 1) / kSpan); }

}  // namespace

uint64_t select_work_bytes(const SelectArgs& a) { return a.tokens ? a.n * parts_of(a) * 8 : 0; }
void launch_select(const SelectArgs& a, void* work, hipStream_t s) {
  if (a.n == 0 || (!a.tokens && !a.out)) return;
  const uint32_t parts = parts_of(a);
  uint64_t* keys = a.tokens ? static_cast<uint64_t*>(work) : nullptr;
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  const bool vec = a.ld % 4 == 0 && aligned(a.logits) && (!a.out || (a.out_ld % 4 == 0 && aligned(a.out)));
  if (vec) hipLaunchKernelGGL(k_select<true>, dim3(parts, unsigned(a.n)), dim3(kThreads), 0, s, a, keys, parts);
  else hipLaunchKernelGGL(k_select<false>, dim3(parts, unsigned(a.n)), dim3(kThreads), 0, s, a, keys, parts);
  if (a.tokens) hipLaunchKernelGGL(k_select_final, dim3(unsigned(a.n)), dim3(64), 0, s, keys, parts, a.tokens);
}

}  // namespace det
