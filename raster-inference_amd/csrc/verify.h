// Launch-side declarations of the operators that verify drafted tokens for
// many requests (gfx950).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace det {

// Head norms and rotation (head_rope.hip).
constexpr uint32_t kHeadMaxDim = 1024;
constexpr uint32_t kHeadSets = 4;
struct HeadSet {
  const int32_t* x;
  int32_t* out;
  const int32_t* gain;
  uint64_t ld, out_ld;
  uint32_t heads;
  uint32_t flags;  // 1 norm, 2 rotate
};
struct HeadRopeArgs {
  HeadSet set[kHeadSets];
  uint32_t n_sets, hd, pairs, interleaved;
  uint32_t total;  // head rows of one token: the sets' heads
  int32_t amplitude;
  int64_t eps;
  const int64_t* freq;  // [pairs]
  const uint32_t* positions;
  uint64_t rows;
};
void launch_head_rope(const HeadRopeArgs& a, hipStream_t s);

// Attention of drafted rows over caches (tree_attention.hip).
constexpr uint32_t kTreeMaxDrafts = 64;
constexpr uint64_t kTreeMaxRows = uint64_t(1) << 20;
struct TreeSeq {
  const int32_t* k;
  const int32_t* v;
  uint64_t ld, first, wrap;
  uint32_t rows, drafts;
  uint64_t row0;  // its first drafted row
};
struct TreeArgs {
  const int32_t* q;
  const int32_t* k;
  const int32_t* v;
  const uint64_t* masks;
  const uint32_t* starts;
  int32_t* out;
  uint64_t q_ld, kv_ld, out_ld;
  uint32_t nh, nkv, groups, hd;
};
// Scratch bytes of a call, and the call (seqs: host array, copied into the
// launches' arguments).
uint64_t tree_work_bytes(const TreeArgs& a, const TreeSeq* seqs, uint32_t n);
void launch_tree_attention(const TreeArgs& a, const TreeSeq* seqs, uint32_t n, void* work, hipStream_t s);

// Low-rank adapters (adapters.hip). A is an int8 / digit-plane matrix of
// rank rows (DevMatrix); B's rows are packed in 16-column groups: plane p of
// the 16-row tile T at ((T * planes + p) * kg) * 256 bytes, group g's 256
// bytes hold columns [16 g, +16) of the tile's rows (16 bytes each).
struct DevAdapter {
  const int8_t* a;
  const int32_t* a_scale;
  const int8_t* b;
  const int32_t* b_scale;
  uint32_t rank, kg;
  uint32_t a_planes, b_planes;
  int32_t scale;
};
constexpr uint32_t kAdapterMaxRank = 256;
constexpr uint32_t kAdapterMost = 4096;  // adapters of one set
struct AdapterArgs {
  const DevAdapter* set;
  uint32_t n;
  uint32_t max_rank;  // of the set, in whole tiles of 16
  const uint32_t* index;
  const int32_t* act;
  uint64_t m, cols, kpad, rows;
  int32_t* out;  // holds W x on entry
};
uint64_t adapter_work_bytes(const AdapterArgs& a);
void launch_adapters(const AdapterArgs& a, void* work, hipStream_t s);

// Decoding rules and token choice (select.hip).
struct SelectPenalty {
  int32_t repetition, frequency, presence;
};
struct SelectArgs {
  const int32_t* logits;
  uint64_t ld, n, vocab;
  const SelectPenalty* penalties;
  const uint32_t* ids;
  uint64_t n_ids;
  const uint32_t* spans;
  uint32_t spans_per_row;
  const uint32_t* bias_begin;
  const uint32_t* bias_ids;
  const int32_t* bias_values;
  uint64_t n_bias;
  const uint32_t* mask;
  uint64_t mask_ld;
  int32_t* out;
  uint64_t out_ld;
  uint32_t* tokens;
};
uint64_t select_work_bytes(const SelectArgs& a);
void launch_select(const SelectArgs& a, void* work, hipStream_t s);

}  // namespace det
