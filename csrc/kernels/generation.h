// Launchers of the operators that draw several continuations of one history:
// attention over a shared prefix plus own tails, and token sampling.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace b200 {

// ------------------------------------------------------- shared-prefix MLA
struct PrefixMLAArgs {
  const __nv_bfloat16* q;       // [G = B * T, H, 576] contiguous
  const __nv_bfloat16* prefix;  // [P, 576], rows ld_prefix elements apart
  const __nv_bfloat16* tail;    // [B, S, 576], strides ld_batch / ld_tail elements
  const int* tail_lens;         // [B] visible tail rows of the last query token; null: S
  __nv_bfloat16* out;           // [G, H, 512]
  float* lse;                   // optional [G, H], natural logarithm
  int64_t ld_prefix, ld_tail, ld_batch;
  int B, T, H, P, S;
  float scale;
  int* err;
};
// FP32 workspace of a call (0: none); the same arguments give the same plan.
size_t shared_prefix_mla_scratch_floats(const PrefixMLAArgs& a);
void launch_shared_prefix_mla(const PrefixMLAArgs& a, float* scratch, cudaStream_t stream);

// ---------------------------------------------------------------- sampling
struct SampleArgs {
  const void* logits;  // [R, V] FP32 or BF16, rows ld elements apart
  bool bf16;
  int64_t ld;
  int R, V;
  const float* u;            // [R]
  const float* temperature;  // per-row values; null: the scalars below
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature0, top_p0, min_p0;
  int top_k0;
  int64_t* tokens;  // [R]
  float* logprobs;  // [R]
};
int sample_max_vocabulary();
void launch_sample_tokens(const SampleArgs& a, cudaStream_t stream);

}  // namespace b200
