// MLA of a batch of continuations over one shared history plus own tails.
//
//   s(j) = scale * q . k_j over the P prefix rows and the first
//          len[b] - (T - 1 - t) tail rows of the continuation,
//   out  = sum_j exp(s(j) - m) v_j / sum_j exp(s(j) - m),  m = max_j s(j),
//   lse  = m + log sum_j exp(s(j) - m),  v_j = the first 512 dims of k_j.
//
// One warp per (query, head) walks the keys once with a running maximum and
// sum (FP32); each lane holds 18 query dims and 16 output dims.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "generation.h"

namespace b200 {
namespace {

constexpr int D = 576;
constexpr int DV = 512;
constexpr int kWarps = 8;

__global__ void __launch_bounds__(kWarps * 32) prefix_mla_kernel(PrefixMLAArgs a) {
  const int lane = threadIdx.x % 32;
  const int64_t row = int64_t(blockIdx.x) * kWarps + threadIdx.x / 32;
  const int64_t rows = int64_t(a.B) * a.T * a.H;
  if (row >= rows) return;
  const int g = int(row / a.H), b = g / a.T, t = g % a.T;
  int len = a.S;
  if (a.tail_lens) {
    len = a.tail_lens[b];
    if (len < 0 || len > a.S) {
      if (lane == 0) record_error(a.err, kErrBadIndex);
      len = min(max(len, 0), a.S);
    }
  }
  const int seen = max(0, len - (a.T - 1 - t));
  // Lane l holds dims 2l + 64i, 2l + 64i + 1 (i < 9); i < 8 are the value dims.
  float qf[18], acc[16];
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(a.q + row * D + 64 * i + 2 * lane);
    qf[2 * i] = bf16_lo(v) * a.scale;
    qf[2 * i + 1] = bf16_hi(v) * a.scale;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  // The sum runs over blocks of 32 keys first: 1/32 of the roundings of one long chain.
  float m = -INFINITY, l = 0.f, block = 0.f;
  for (int j = 0; j < a.P + seen; ++j) {
    const __nv_bfloat16* k =
        j < a.P ? a.prefix + int64_t(j) * a.ld_prefix : a.tail + int64_t(b) * a.ld_batch + int64_t(j - a.P) * a.ld_tail;
    float kf[18];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(k + 64 * i + 2 * lane));
      kf[2 * i] = bf16_lo(v);
      kf[2 * i + 1] = bf16_hi(v);
      s = fmaf(qf[2 * i], kf[2 * i], s);
      s = fmaf(qf[2 * i + 1], kf[2 * i + 1], s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (s > m) {
      const float f = m == -INFINITY ? 0.f : expf(m - s);
      l *= f;
      block *= f;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] *= f;
      m = s;
    }
    const float p = m == -INFINITY ? 0.f : expf(s - m);
    block += p;
    if (j % 32 == 31) {
      l += block;
      block = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = fmaf(p, kf[i], acc[i]);
  }
  l += block;
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<uint32_t*>(a.out + row * DV + 64 * i + 2 * lane) = pack_bf16(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  if (a.lse && lane == 0) a.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace

void launch_shared_prefix_mla(const PrefixMLAArgs& a, cudaStream_t stream) {
  const int64_t rows = int64_t(a.B) * a.T * a.H;
  if (rows == 0) return;
  prefix_mla_kernel<<<dim3(unsigned((rows + kWarps - 1) / kWarps)), kWarps * 32, 0, stream>>>(a);
  cuda_check(cudaGetLastError(), "shared_prefix_mla launch");
}

}  // namespace b200
