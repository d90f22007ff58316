// Token sampling: temperature, top-k, top-p and min-p from given uniform numbers.
//
//   d_i = (x_i - max x) / T,  w_i = exp(d_i),  W_i = floor(2^36 w_i)
//   kept: a prefix of the order (x descending, index ascending): its first k
//   entries, while the mass before them is below p times the mass of those k,
//   and w_i >= min_p; the first entry always.
//   token = first index whose cumulative kept W exceeds floor(u * sum W).
//
// The masses are whole numbers, so sums do not depend on their order: a draw
// is the same whatever the batch, the split over threads or the kernel.
//
// One CTA per row; the thresholds are built bit by bit over the order-
// preserving integer keys of the logits, one pass over the row per bit.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "generation.h"

namespace b200 {
namespace {

constexpr int kThreads = 1024;
constexpr float kFixed = 68719476736.f;  // 2^36

__device__ __forceinline__ float load_logit(const SampleArgs& a, int64_t row, int i) {
  float x = a.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.logits)[row * a.ld + i])
                   : static_cast<const float*>(a.logits)[row * a.ld + i];
  return x == x ? x + 0.f : -INFINITY;  // NaN counts as masked; -0 as +0
}

__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T, typename Op>
__device__ T block_reduce(T v, Op op, T* red) {
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = red[threadIdx.x % 32];
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sum over the threads before this one.
__device__ uint64_t block_exclusive(uint64_t v, uint64_t* red) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint64_t inc = v;
  for (int o = 1; o < 32; o *= 2) {
    const uint64_t n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  uint64_t before = 0;
  for (int w = 0; w < warp; ++w) before += red[w];
  return before + inc - v;
}

__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ uint64_t red[32];
  __shared__ int s_token;
  const int64_t row = blockIdx.x;
  const int V = a.V;
  const float T = a.temperature ? a.temperature[row] : a.temperature0;
  const int k = a.top_k ? a.top_k[row] : a.top_k0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0;
  const float mp = a.min_p ? a.min_p[row] : a.min_p0;
  const int per = (V + kThreads - 1) / kThreads;
  const int i0 = min(V, int(threadIdx.x) * per), i1 = min(V, i0 + per);  // this thread's entries, in index order
  auto add = [](uint64_t x, uint64_t y) { return x + y; };

  float mx = -INFINITY;
  for (int i = i0; i < i1; ++i) mx = fmaxf(mx, load_logit(a, row, i));
  mx = block_reduce(mx, [](float x, float y) { return fmaxf(x, y); }, reinterpret_cast<float*>(red));
  int first = V;
  for (int i = i0; i < i1; ++i)
    if (load_logit(a, row, i) == mx) {
      first = i;
      break;
    }
  first = block_reduce(first, [](int x, int y) { return min(x, y); }, reinterpret_cast<int*>(red));
  if (mx == -INFINITY || !(T > 0.f)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = mx == -INFINITY ? -1 : first;
      a.logprobs[row] = mx == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  auto dist = [&](float x) { return x == mx ? 0.f : (x - mx) / T; };
  auto weight = [&](float x) { return x == -INFINITY ? 0.f : expf(dist(x)); };
  auto mass = [&](float x) { return uint64_t(weight(x) * kFixed); };
  auto sum_over = [&](auto&& f) {
    uint64_t s = 0;
    for (int i = i0; i < i1; ++i) s += f(load_logit(a, row, i));
    return block_reduce(s, add, red);
  };

  // Kept: key > cut, or key == cut and fewer than `ties` equal keys before it.
  uint32_t cut = 0;
  int64_t ties = V;
  if (k > 0 && k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = cut | (1u << bit);
      if (sum_over([&](float x) { return uint64_t(order_key(x) >= t); }) >= uint64_t(k)) cut = t;
    }
    ties = k - int64_t(sum_over([&](float x) { return uint64_t(order_key(x) > cut); }));
  }
  if (p < 1.f) {
    const uint64_t above = sum_over([&](float x) { return order_key(x) > cut ? mass(x) : 0; });
    const uint64_t equal = sum_over([&](float x) { return uint64_t(order_key(x) == cut); });
    const uint32_t cb = cut & 0x80000000u ? cut & 0x7fffffffu : ~cut;
    const uint64_t cut_mass = equal ? mass(__uint_as_float(cb)) : 0;
    const double want = double(p) * double(above + cut_mass * min(uint64_t(ties), equal));
    if (!(want > 0.)) {
      cut = order_key(mx);
      ties = 1;
    } else {
      // Largest key whose mass at or above it reaches `want` (the top-k cut itself when none above does).
      uint32_t c = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t t = c | (1u << bit);
        if (t <= cut || !(double(sum_over([&](float x) { return order_key(x) >= t ? mass(x) : 0; })) < want)) c = t;
      }
      const uint64_t before = sum_over([&](float x) { return order_key(x) > c ? mass(x) : 0; });
      const uint64_t eq = sum_over([&](float x) { return uint64_t(order_key(x) == c); });
      const uint32_t b = c & 0x80000000u ? c & 0x7fffffffu : ~c;
      const uint64_t one = eq ? mass(__uint_as_float(b)) : 0;
      // Equal entries kept: those with before + j * one < want.
      uint64_t j = 0;
      if (one) {
        j = uint64_t(fmax(0., (want - double(before)) / double(one)));
        while (j > 0 && !(double(before + (j - 1) * one) < want)) --j;
        while (double(before + j * one) < want) ++j;
      }
      if (c == cut) ties = min(ties, int64_t(j));
      else ties = int64_t(j);
      cut = c;
    }
  }
  auto kept = [&](int i, float x, int64_t rank) {
    const uint32_t key = order_key(x);
    return (i == first) || ((key > cut || (key == cut && rank < ties)) && !(weight(x) < mp));
  };
  uint64_t my_ties = 0;
  for (int i = i0; i < i1; ++i) my_ties += order_key(load_logit(a, row, i)) == cut;
  const int64_t rank0 = int64_t(block_exclusive(my_ties, red));
  uint64_t mine = 0;
  int64_t rank = rank0;
  for (int i = i0; i < i1; ++i) {
    const float x = load_logit(a, row, i);
    if (kept(i, x, rank)) mine += mass(x);
    rank += order_key(x) == cut;
  }
  const uint64_t before = block_exclusive(mine, red);
  const uint64_t total = block_reduce(mine, add, red);
  uint64_t r = uint64_t(fmax(0., floor(double(a.u[row]) * double(total))));
  r = min(r, total - 1);
  if (threadIdx.x == 0) s_token = first;
  __syncthreads();
  if (r >= before && r < before + mine) {
    uint64_t c = before;
    rank = rank0;
    for (int i = i0; i < i1; ++i) {
      const float x = load_logit(a, row, i);
      if (kept(i, x, rank)) c += mass(x);
      rank += order_key(x) == cut;
      if (c > r) {
        s_token = i;
        break;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.tokens[row] = s_token;
    a.logprobs[row] = float(double(dist(load_logit(a, row, s_token))) - log(double(total) / double(kFixed)));
  }
}

}  // namespace

void launch_sample_tokens(const SampleArgs& a, cudaStream_t stream) {
  if (a.R == 0) return;
  sample_kernel<<<a.R, kThreads, 0, stream>>>(a);
  cuda_check(cudaGetLastError(), "sample_tokens launch");
}

}  // namespace b200
