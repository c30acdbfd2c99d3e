// Low-rank adapters of many requests beside a shared projection:
// out[t] = add_sat(out[t], scale_act(B (A x_t), scale)) with the adapter of
// row t, both products requantized (out holds W x on entry).
#include <hip/hip_runtime.h>

#include "det_arith.h"
#include "verify.h"
#include "wave.h"

namespace det {

namespace {

// h[t][j] = requant(A_j . x_t): a wave per rank row.
__global__ __launch_bounds__(256) void k_down_simple(AdapterArgs a, int32_t* h) {
  const uint64_t t = blockIdx.x;
  const uint32_t idx = a.index[t];
  if (idx >= a.n) return;
  const DevAdapter ad = a.set[idx];
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t j = threadIdx.x >> 6; j < ad.rank; j += 4) {
    int64_t acc = 0;
    for (uint64_t c = lane; c < a.cols; c += 64) {
      int64_t w = 0;
      for (uint32_t p = 0; p < ad.a_planes; ++p)
        w += int64_t(ad.a[tiled_offset(a.kpad, digit_row(j, int(ad.a_planes), int(p)), c)]) << (8 * p);
      acc += w * a.act[t * a.cols + c];
    }
    acc = wave_sum_wrap64(acc);
    if (lane == 0) h[t * a.max_rank + j] = requant(acc * ad.a_scale[j]);
  }
}

__global__ __launch_bounds__(256) void k_up_simple(AdapterArgs a, const int32_t* h) {
  const uint64_t t = blockIdx.y, n = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t idx = a.index[t];
  if (idx >= a.n || n >= a.rows) return;
  const DevAdapter ad = a.set[idx];
  int64_t acc = 0;
  for (uint32_t j = 0; j < ad.rank; ++j) {
    int64_t w = 0;
    for (uint32_t p = 0; p < ad.b_planes; ++p)
      w += int64_t(ad.b[(((n >> 4) * ad.b_planes + p) * ad.kg + j / 16) * 256 + (n & 15) * 16 + j % 16]) << (8 * p);
    acc += w * h[t * a.max_rank + j];
  }
  int32_t* o = a.out + t * a.rows + n;
  *o = add_sat(*o, mul_sat(requant(acc * ad.b_scale[n]), ad.scale));
}

}  // namespace

uint64_t adapter_work_bytes(const AdapterArgs& a) { return a.m * a.max_rank * 4; }
void launch_adapters(const AdapterArgs& a, void* work, hipStream_t s) {
  if (a.m == 0 || a.n == 0 || a.rows == 0) return;
  int32_t* h = static_cast<int32_t*>(work);
  hipLaunchKernelGGL(k_down_simple, dim3(unsigned(a.m)), dim3(256), 0, s, a, h);
  hipLaunchKernelGGL(k_up_simple, dim3(unsigned((a.rows + 255) / 256), unsigned(a.m)), dim3(256), 0, s, a, h);
}

}  // namespace det
