// What the kernels of the shared-prefix attention (shared_prefix.cu, shared_prefix_sm100.cu) are told.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace b200 {

struct SharedPrefixParams {
  const void* q;            // [B * T, Hq, D], ldq elements between tokens
  const void* k_cache;      // [num_blocks, page, Hkv, D]
  const void* v_cache;
  const int* kv_lens;       // [B], the T new tokens counted
  const int* block_table;   // [B, width], bt_stride between rows
  const int* prefix_table;  // [>= ceil(shared / page)]
  float* o_part;            // [B * T * Hq, S, D]
  float* lse_part;          // [B * T * Hq, S], natural logarithm; -inf: an empty range, whose o_part is not read
  uint32_t* status;         // nullable: set non-zero when a pipeline wait expired
  long long ldq;
  int bt_stride, width, B, T, Hq, Hkv, num_blocks, page;
  int shared;               // keys that all sequences begin with
  int prefix_splits, own_splits, S;   // ranges of keys per row: S = prefix_splits + own_splits
  int prefix_chunk;         // keys per CTA of the shared ones, a multiple of 64 (span kernel) or 128
  int prefix_ctas;          // CTAs of the shared keys in the span kernel's grid
  int late_wait;            // the kernel in front is this call's own: only the end of the span kernel waits for it
  float scale_log2e;        // softmax scale * log2(e)
};

constexpr int kPrefixMostKeys = 1 << 30;   // per sequence: sums of a length and a range of keys stay in 32 bits
__device__ __forceinline__ int prefix_len(const SharedPrefixParams& p, int b) { return min(max(p.kv_lens[b], 0), kPrefixMostKeys); }

bool shared_prefix_tc_takes(const SharedPrefixParams& p, int D);
int shared_prefix_tc_launch(const SharedPrefixParams& p, int D, int dtype, cudaStream_t s);

}  // namespace b200
