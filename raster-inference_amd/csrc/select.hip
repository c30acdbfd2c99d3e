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

constexpr uint32_t kSpan = 4096;  // tokens per workgroup

// A row's choice so far: value (offset to unsigned) over the inverted index,
// so that the larger key is the larger value, then the lower index; 0: none.
__device__ inline uint64_t choice_key(int32_t x, uint32_t token) {
  return (uint64_t(uint32_t(x) ^ 0x80000000u) << 32) | uint64_t(0xffffffffu - token);
}
struct OpMaxU64 {
  __device__ __forceinline__ uint64_t operator()(uint64_t p, uint64_t q) const { return p > q ? p : q; }
};

__global__ __launch_bounds__(256) void k_select(SelectArgs a, uint64_t* keys, uint32_t parts) {
  __shared__ uint32_t count[kSpan];
  __shared__ unsigned long long bias[kSpan];
  __shared__ uint64_t red[4];
  const uint32_t tid = threadIdx.x, part = blockIdx.x;
  const uint64_t r = blockIdx.y, base = uint64_t(part) * kSpan;
  const uint32_t span = uint32_t(a.vocab - base < kSpan ? a.vocab - base : kSpan);
  for (uint32_t i = tid; i < kSpan; i += 256) count[i] = 0, bias[i] = 0;
  __syncthreads();
  if (a.penalties && a.spans && a.ids)
    for (uint32_t s = 0; s < a.spans_per_row; ++s) {
      const uint64_t lo = a.spans[(r * a.spans_per_row + s) * 2], e = a.spans[(r * a.spans_per_row + s) * 2 + 1];
      const uint64_t hi = e < a.n_ids ? e : a.n_ids;
      for (uint64_t i = lo + tid; i < hi; i += 256) {
        const uint64_t id = a.ids[i];
        if (id >= base && id - base < span) atomicAdd(&count[id - base], 1u);
      }
    }
  if (a.bias_begin && a.bias_ids && a.bias_values) {
    const uint64_t lo = a.bias_begin[r], e = a.bias_begin[r + 1], hi = e < a.n_bias ? e : a.n_bias;
    for (uint64_t i = lo + tid; i < hi; i += 256) {
      const uint64_t id = a.bias_ids[i];
      if (id >= base && id - base < span)
        atomicAdd(&bias[id - base], static_cast<unsigned long long>(int64_t(a.bias_values[i])));
    }
  }
  __syncthreads();
  SelectPenalty p{kOneAct, 0, 0};
  if (a.penalties) p = a.penalties[r];
  uint64_t best = 0;
  for (uint32_t i = tid; i < span; i += 256) {
    const uint64_t token = base + i;
    int32_t x = a.logits[r * a.ld + token];
    const uint32_t c = count[i];
    const int64_t b = int64_t(bias[i]);
    if (c | (b != 0)) {
      if (c && p.repetition > 0 && p.repetition != kOneAct) x = x > 0 ? div_act(x, p.repetition) : mul_sat(x, p.repetition);
      x = sat32(int64_t(x) - int64_t(c) * p.frequency - (c ? p.presence : 0) + b);
    }
    const bool ok = !a.mask || ((a.mask[r * a.mask_ld + token / 32] >> (token % 32)) & 1u);
    if (!ok) x = INT32_MIN;
    if (a.out) a.out[r * a.out_ld + token] = x;
    const uint64_t k = ok ? choice_key(x, uint32_t(token)) : 0;
    best = k > best ? k : best;
  }
  best = wave_reduce(best, OpMaxU64());
  if ((tid & 63) == 0) red[tid >> 6] = best;
  __syncthreads();
  if (tid == 0 && keys) {
    for (int w = 1; w < 4; ++w) best = red[w] > best ? red[w] : best;
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
  hipLaunchKernelGGL(k_select, dim3(parts, unsigned(a.n)), dim3(256), 0, s, a, keys, parts);
  if (a.tokens) hipLaunchKernelGGL(k_select_final, dim3(unsigned(a.n)), dim3(64), 0, s, keys, parts, a.tokens);
}

}  // namespace det
