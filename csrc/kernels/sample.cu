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
// One cluster of 1 to 16 CTAs per row: a row of 129,280 FP32 logits (517 KB)
// is read from HBM once, in slices that stay in the CTAs' shared memory for all
// later passes.  The order is never sorted: a histogram of d (2,048 bins over
// the range where W > 0, counts and masses) finds the bin in which a filter
// cuts, and the few entries of that bin are ranked against each other.  A bin
// with more entries than fit the list (equal logits) is split again by the bits
// of the logits until it fits or holds one value, which is cut by index.
//
// Sums over the cluster go through distributed shared memory; every CTA merges
// and scans 1 / C of the histogram's bins.  Nothing spins: the CTAs meet at
// hardware cluster barriers only.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "generation.h"

namespace b200 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
// A warp's share of a slice is at most 32 blocks of 32 entries; a bin's 18-bit halves of up to
// 16,383 masses fit 32 bits.
constexpr int kMaxSlice = 16352;
constexpr int kBins = 2048;
constexpr int kList = 512;
constexpr float kFixed = 68719476736.f;  // 2^36
constexpr float kHalf = 262144.f;        // 2^18
constexpr float kSpan = 25.f;            // exp(-25) * 2^36 < 1: entries further down have no mass
constexpr uint64_t kNothing = ~0ull;     // composite above every entry

struct alignas(16) Shared {
  uint64_t xch[2][4][kMaxCluster];  // exchanged values (double buffered)
  uint64_t red[kWarps];
  uint64_t wsum[kWarps];
  uint64_t decision[2][4];          // written by the CTA that owns the cut (double buffered)
  uint64_t list[kList];             // CTA 0: entries of the cut bin
  uint64_t list_mass[kList];
  uint32_t list_count;
  uint32_t cnt[kBins], lo[kBins], hi[kBins];
};

__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void remote_st64(const void* local, uint32_t rank, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(local), rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t remote_ld32(const void* local, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(local), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t remote_add32(const void* local, uint32_t rank, uint32_t v) {
  uint32_t old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;"
               : "=r"(old)
               : "r"(mapa_shared(smem_u32(local), rank)), "r"(v)
               : "memory");
  return old;
}

__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Larger = earlier in the order.
__device__ __forceinline__ uint64_t composite(float x, int index) {
  return (uint64_t(order_key(x)) << 32) | uint32_t(~index);
}

// floor(2^36 w), w in [0, 1], as 2^18 hi + lo: the truncations are additions of 2^23 rounded to zero.
__device__ __forceinline__ void mass_halves(float w, uint32_t& hi, uint32_t& lo) {
  const float s = w * kHalf;
  const float t = __fadd_rz(s, 8388608.f);
  hi = __float_as_uint(t) & 0x7fffffu;
  const float rest = s - (t - 8388608.f);  // exact, in [0, 1)
  lo = __float_as_uint(__fadd_rz(rest * kHalf, 8388608.f)) & 0x7fffffu;
}
__device__ __forceinline__ uint64_t mass_of(float w) {
  uint32_t hi, lo;
  mass_halves(w, hi, lo);
  return (uint64_t(hi) << 18) + lo;
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_inclusive64(uint64_t v) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint64_t n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

template <bool BF16>
struct Row {
  Shared& s;
  float* v;  // the slice: logits, then d, then the kept weights
  const void* src;
  int V, C, rank, begin, n;
  int chunk, w0, w1;  // this warp's entries of the slice
  float mx, T;
  int first;          // index of the best token
  int phase = 0, event = 0;  // exchange and decision buffers

  __device__ Row(Shared& s_) : s(s_) {}

  __device__ float logit(int i) const {
    float x;
    if constexpr (BF16) x = __bfloat162float(static_cast<const __nv_bfloat16*>(src)[i]);
    else x = static_cast<const float*>(src)[i];
    return x == x ? x + 0.f : -INFINITY;  // NaN counts as masked; -0 as +0
  }
  // d of a logit; -inf stays -inf whatever T is.
  __device__ float dist(float x) const { return x == mx ? 0.f : x == -INFINITY ? -INFINITY : (x - mx) / T; }
  __device__ static float weight(float d) { return expf(d); }
  __device__ static int bin(float d) { return min(kBins - 1, int(-d * (kBins / kSpan))); }

  // Sum over the CTA (every thread gets it).
  __device__ uint64_t block_sum(uint64_t x) {
    x = warp_sum64(x);
    __syncthreads();
    if (threadIdx.x % 32 == 0) s.red[threadIdx.x / 32] = x;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) t += s.red[i];
    return t;
  }
  template <typename Op>
  __device__ uint64_t block_pick(uint64_t x, Op op) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) s.red[threadIdx.x / 32] = x;
    __syncthreads();
    uint64_t t = s.red[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) t = op(t, s.red[i]);
    return t;
  }
  // Hand `a` (and `b`) of every CTA to every CTA; the values are uniform in the CTA.
  __device__ const uint64_t (*exchange(uint64_t a, uint64_t b = 0))[kMaxCluster] {
    uint64_t(*x)[kMaxCluster] = s.xch[phase];
    phase ^= 1;
    if (int(threadIdx.x) < C) {
      remote_st64(&x[0][rank], threadIdx.x, a);
      remote_st64(&x[1][rank], threadIdx.x, b);
    }
    cluster_sync_all();
    return x;
  }
  // One thread of the cluster tells every CTA; all read after `decided()`.
  __device__ void decide(uint64_t a, uint64_t b = 0, uint64_t c = 0, uint64_t d = 0) {
    for (int q = 0; q < C; ++q) {
      remote_st64(&s.decision[event][0], q, a);
      remote_st64(&s.decision[event][1], q, b);
      remote_st64(&s.decision[event][2], q, c);
      remote_st64(&s.decision[event][3], q, d);
    }
  }
  __device__ const uint64_t* decided() {
    cluster_sync_all();
    const uint64_t* d = s.decision[event];
    event ^= 1;
    return d;
  }

  // First local index whose cumulative weight in index order exceeds r, in the
  // warp that holds it (the weights before the warp's chunk sum to warp_before).
  template <typename W>
  __device__ int select_in_warp(W&& weight_at, uint64_t r, uint64_t warp_before) {
    const int lane = threadIdx.x % 32;
    uint64_t mine = 0;
    for (int t = 0; t < 32; ++t) {
      const int j = w0 + lane * 32 + ((lane + t) & 31);
      if (j < w1) mine += weight_at(j);
    }
    const uint64_t inc = warp_inclusive64(mine);
    const uint32_t over = __ballot_sync(0xffffffffu, warp_before + inc > r);
    const int block = __ffs(over) - 1;
    const uint64_t before = warp_before + __shfl_sync(0xffffffffu, inc - mine, block);
    const int j = w0 + block * 32 + lane;
    const uint64_t e = warp_inclusive64(j < w1 ? weight_at(j) : 0);
    const uint32_t hit = __ballot_sync(0xffffffffu, before + e > r);
    return w0 + block * 32 + __ffs(hit) - 1;
  }

  // ---------------------------------------------------------------- cuts
  // Histogram over the entries whose (bin, mass) `entry(j, b, w)` gives; merged over the cluster, CTA c
  // ends up with the bins [c, c + 1) * kBins / C (masses as 64 bits in hi:lo).
  template <typename F>
  __device__ void histogram(F&& entry, bool masses) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.cnt[b] = s.lo[b] = s.hi[b] = 0;
    __syncthreads();
    const int lane = threadIdx.x % 32;
    for (int j = w0 + lane; j < w1; j += 32) {
      int b;
      float w;
      if (entry(j, b, w)) {
        atomicAdd(&s.cnt[b], 1u);
        if (masses) {
          uint32_t h, l;
          mass_halves(w, h, l);
          atomicAdd(&s.hi[b], h);
          atomicAdd(&s.lo[b], l);
        }
      }
    }
    cluster_sync_all();
    const int per = kBins / C;
    for (int b = rank * per + threadIdx.x; b < (rank + 1) * per; b += kThreads) {
      uint32_t c = 0;
      uint64_t m = 0;
      for (int q = 0; q < C; ++q) {
        c += remote_ld32(&s.cnt[b], q);
        if (masses) m += (uint64_t(remote_ld32(&s.hi[b], q)) << 18) + remote_ld32(&s.lo[b], q);
      }
      s.cnt[b] = c;
      s.lo[b] = uint32_t(m);
      s.hi[b] = uint32_t(m >> 32);
    }
    // The segment is only read by this CTA from here on.
    __syncthreads();
    uint64_t c = 0, m = 0;
    for (int b = rank * per + threadIdx.x; b < (rank + 1) * per; b += kThreads) {
      c += s.cnt[b];
      m += (uint64_t(s.hi[b]) << 32) | s.lo[b];
    }
    seg_count = block_sum(c);
    seg_mass = block_sum(m);
    const uint64_t(*x)[kMaxCluster] = exchange(seg_count, seg_mass);
    count_before = mass_before = total_count = total_mass = 0;
    for (int q = 0; q < C; ++q) {
      if (q < rank) {
        count_before += x[0][q];
        mass_before += x[1][q];
      }
      total_count += x[0][q];
      total_mass += x[1][q];
    }
  }
  uint64_t seg_count, seg_mass, count_before, mass_before, total_count, total_mass;

  // What a cut looks for: the first bin where the count (top-k) or the mass
  // (top-p), added to what lies before the histogram, reaches its goal.
  struct Goal {
    bool by_mass;
    uint64_t k;
    double want;
    __device__ bool reached(uint64_t count, uint64_t mass) const {
      return by_mass ? !(double(mass) < want) : count >= k;
    }
  };
  struct Cut {
    int bin;
    uint64_t count, mass, entries;  // before the bin; entries in it
  };
  // The goal is reached within this histogram (count0 / mass0 lie before it).
  __device__ Cut find_bin(const Goal& g, uint64_t count0, uint64_t mass0) {
    const uint64_t cb = count0 + count_before, mb = mass0 + mass_before;
    if (!g.reached(cb, mb) && g.reached(cb + seg_count, mb + seg_mass)) {  // in this CTA's segment
      const int per = kBins / C, q = (per + kThreads - 1) / kThreads;
      const int b0 = rank * per + threadIdx.x * q, b1 = min(b0 + q, (rank + 1) * per);
      uint64_t c = 0, m = 0;
      for (int b = b0; b < b1; ++b) {
        c += s.cnt[b];
        m += (uint64_t(s.hi[b]) << 32) | s.lo[b];
      }
      const uint64_t ci = warp_inclusive64(c), mi = warp_inclusive64(m);
      __syncthreads();
      if (threadIdx.x % 32 == 31) {
        s.red[threadIdx.x / 32] = ci;
        s.wsum[threadIdx.x / 32] = mi;
      }
      __syncthreads();
      uint64_t cs = cb + ci - c, ms = mb + mi - m;
      for (int i = 0; i < int(threadIdx.x / 32); ++i) {
        cs += s.red[i];
        ms += s.wsum[i];
      }
      for (int b = b0; b < b1; ++b) {
        const uint64_t ce = cs + s.cnt[b], me = ms + ((uint64_t(s.hi[b]) << 32) | s.lo[b]);
        if (!g.reached(cs, ms) && g.reached(ce, me)) decide(uint64_t(b), cs, ms, s.cnt[b]);
        cs = ce;
        ms = me;
      }
    }
    const uint64_t* d = decided();
    return Cut{int(d[0]), d[1], d[2], d[3]};
  }

  // Gather the entries that pass `in(j)` (at most kList) into CTA 0's list, rank them and return the
  // composite of the last kept one (kNothing: none) and the mass through it.
  template <typename F>
  __device__ uint64_t rank_list(F&& in, const Goal& g, const Cut& c, uint64_t floor_, uint64_t& mass_through) {
    if (threadIdx.x == 0) s.list_count = 0;
    cluster_sync_all();
    const int lane = threadIdx.x % 32;
    for (int jb = w0; jb < w1; jb += 32) {
      const int j = jb + lane;
      const bool take = j < w1 && in(j);
      const uint32_t m = __ballot_sync(0xffffffffu, take);
      if (!m) continue;
      uint32_t at = 0;
      if (lane == 0) at = remote_add32(&s.list_count, 0, __popc(m));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(m & ((1u << lane) - 1));
      if (take && at < kList) {
        const float x = logit(begin + j);
        remote_st64(&s.list[at], 0, composite(x, begin + j));
        remote_st64(&s.list_mass[at], 0, mass_of(weight(dist(x))));
      }
    }
    cluster_sync_all();
    if (rank == 0) {
      // Warp w ranks entries w, w + 16, ...: what lies before each in the order.
      const int m = min(int(s.list_count), kList);
      uint64_t last = kNothing, through = c.mass;
      for (int e = threadIdx.x / 32; e < m; e += kWarps) {
        const uint64_t mine = s.list[e];
        uint64_t cnt = 0, mass = 0;
        for (int f = lane; f < m; f += 32)
          if (s.list[f] > mine) {
            ++cnt;
            mass += s.list_mass[f];
          }
        cnt = c.count + warp_sum64(cnt);
        mass = c.mass + warp_sum64(mass);
        if (!g.reached(cnt, mass) && mine >= floor_) {
          last = min(last, mine);
          through = max(through, mass + s.list_mass[e]);
        }
      }
      last = block_pick(last, [](uint64_t a, uint64_t b) { return a < b ? a : b; });
      through = block_pick(through, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
      if (threadIdx.x == 0) decide(last, through);
    }
    const uint64_t* d = decided();
    mass_through = d[1];
    return d[0];
  }

  // The last kept entry of a goal (composite; entries of composite >= it are kept) and the mass through
  // it.  `floor_`: an earlier cut that also holds.  The histogram of d must be built.
  __device__ uint64_t find_cut(const Goal& g, uint64_t floor_, uint64_t& mass_through, bool& rebuilt) {
    Cut c = find_bin(g, 0, 0);
    if (c.entries <= kList)
      return rank_list([&](int j) { return v[j] > -kSpan && bin(v[j]) == c.bin; }, g, c, floor_, mass_through);
    // Too many: split by the keys' bits inside the bin.  Any entry between the
    // bin's lowest and highest key belongs to it (d is monotone in x).
    rebuilt = true;
    uint64_t top = 0, low = kNothing;
    for (int j = w0 + int(threadIdx.x % 32); j < w1; j += 32)
      if (v[j] > -kSpan && bin(v[j]) == c.bin) {
        const uint64_t k = order_key(logit(begin + j));
        top = max(top, k);
        low = min(low, k);
      }
    while (true) {
      top = block_pick(top, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
      low = block_pick(low, [](uint64_t a, uint64_t b) { return a < b ? a : b; });
      const uint64_t(*x)[kMaxCluster] = exchange(top, low);
      for (int q = 0; q < C; ++q) {
        top = max(top, x[0][q]);
        low = min(low, x[1][q]);
      }
      const uint32_t khi = uint32_t(top), klo = uint32_t(low);
      auto inside = [&](int j) {
        const uint32_t k = order_key(logit(begin + j));
        return k >= klo && k <= khi;
      };
      if (c.entries <= kList) return rank_list(inside, g, c, floor_, mass_through);
      if (khi == klo) return cut_equal(khi, g, c, floor_, mass_through);
      int shift = 0;
      while (((khi - klo) >> shift) >= uint32_t(kBins)) ++shift;
      const uint64_t count0 = c.count, mass0 = c.mass;
      histogram(
          [&](int j, int& b, float& w) {
            const float xv = logit(begin + j);
            const uint32_t k = order_key(xv);
            if (k < klo || k > khi) return false;
            b = int((khi - k) >> shift);
            w = weight(dist(xv));
            return true;
          },
          true);
      c = find_bin(g, count0, mass0);
      // The bin's own lowest and highest keys.
      const uint32_t h = khi - (uint32_t(c.bin) << shift);
      const uint32_t span = (1u << shift) - 1;
      const uint32_t l = h - klo > span ? h - span : klo;
      top = 0;
      low = kNothing;
      for (int j = w0 + int(threadIdx.x % 32); j < w1; j += 32) {
        const uint64_t k = order_key(logit(begin + j));
        if (k >= l && k <= h) {
          top = max(top, k);
          low = min(low, k);
        }
      }
    }
  }

  // Many entries of one value: the goal keeps the first m of them in index order.
  __device__ uint64_t cut_equal(uint32_t key, const Goal& g, const Cut& c, uint64_t floor_, uint64_t& mass_through) {
    const uint64_t one = mass_of(weight(dist(key_value(key))));
    uint64_t m;
    if (g.by_mass) {
      m = uint64_t(fmax(0., (g.want - double(c.mass)) / double(one)));
      while (m > 0 && g.reached(0, c.mass + (m - 1) * one)) --m;
      while (!g.reached(0, c.mass + m * one)) ++m;
    } else {
      m = g.k - c.count;
    }
    auto equal = [&](int j) { return uint64_t(order_key(logit(begin + j)) == key); };
    uint64_t mine = 0;
    for (int j = w0 + int(threadIdx.x % 32); j < w1; j += 32) mine += equal(j);
    mine = warp_sum64(mine);
    const uint64_t total = block_sum(threadIdx.x % 32 == 0 ? mine : 0);
    if (threadIdx.x % 32 == 0) s.wsum[threadIdx.x / 32] = mine;
    const uint64_t(*x)[kMaxCluster] = exchange(total);
    uint64_t before = 0;
    for (int q = 0; q < rank; ++q) before += x[0][q];
    for (int i = 0; i < int(threadIdx.x / 32); ++i) before += s.wsum[i];
    if (m - 1 >= before && m - 1 < before + mine) {  // this warp holds the m-th one
      const int j = select_in_warp(equal, m - 1, before);
      if (threadIdx.x % 32 == 0) decide(composite(key_value(key), begin + j));
    }
    mass_through = c.mass + m * one;
    return max(decided()[0], floor_);
  }
};

template <bool BF16>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a, int C) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  pdl_trigger();
  pdl_wait();
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  constexpr int VEC = BF16 ? 8 : 4;
  constexpr int kSize = BF16 ? 2 : 4;
  const int64_t row = blockIdx.x / C;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Row<BF16> r(s);
  r.C = C;
  r.V = a.V;
  r.rank = int(cluster_ctarank());
  r.src = static_cast<const uint8_t*>(a.logits) + row * a.ld * kSize;
  const float T = a.temperature ? a.temperature[row] : a.temperature0;
  const int k = a.top_k ? a.top_k[row] : a.top_k0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0;
  const float mp = a.min_p ? a.min_p[row] : a.min_p0;
  r.T = T;

  // Slices of whole 16-byte vectors; CTA 0 also takes the entries before the first aligned one.
  const int head = min(a.V, int((16 - reinterpret_cast<uintptr_t>(r.src) % 16) % 16 / kSize));
  const int per = ((a.V - head + VEC - 1) / VEC + C - 1) / C * VEC;
  const int vec0 = min(a.V, head + r.rank * per);  // first vector entry of this CTA
  const int end = min(a.V, vec0 + per);
  r.begin = r.rank == 0 ? 0 : vec0;
  r.n = end - r.begin;
  const int pad = r.rank == 0 ? (8 - head) % 8 : 0;  // vectors land on aligned addresses
  r.v = reinterpret_cast<float*>(smem_raw + sizeof(Shared)) + pad;
  r.chunk = (r.n + kWarps * 32 - 1) / (kWarps * 32) * 32;
  r.w0 = min(r.n, warp * r.chunk);
  r.w1 = min(r.n, r.w0 + r.chunk);

  uint64_t best = 0;
  {
    float bx = -INFINITY;
    int bi = 0x7fffffff;
    auto take = [&](float x, int i) {
      if (x > bx || (x == bx && i < bi)) {
        bx = x;
        bi = i;
      }
    };
    auto clean = [](float x) { return x == x ? x + 0.f : -INFINITY; };
    if (r.rank == 0 && int(threadIdx.x) < head) {
      const float x = r.logit(threadIdx.x);
      r.v[threadIdx.x] = x;
      take(x, threadIdx.x);
    }
    const int vecs = (end - vec0) / VEC;
#pragma unroll 4
    for (int g = threadIdx.x; g < vecs; g += kThreads) {
      const int i = vec0 + g * VEC, j = i - r.begin;
      const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(r.src) + int64_t(i) * kSize));
      float x[VEC];
      if constexpr (BF16) {
        const uint32_t q[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = clean(bf16_lo(q[e]));
          x[2 * e + 1] = clean(bf16_hi(q[e]));
        }
      } else {
        x[0] = clean(__uint_as_float(raw.x));
        x[1] = clean(__uint_as_float(raw.y));
        x[2] = clean(__uint_as_float(raw.z));
        x[3] = clean(__uint_as_float(raw.w));
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) take(x[e], i + e);
#pragma unroll
      for (int e = 0; e < VEC; e += 4)
        *reinterpret_cast<float4*>(&r.v[j + e]) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    }
    const int rest0 = vec0 + vecs * VEC;
    if (rest0 + int(threadIdx.x) < end) {
      const int i = rest0 + threadIdx.x;
      const float x = r.logit(i);
      r.v[i - r.begin] = x;
      take(x, i);
    }
    best = composite(bx, bi);
  }
  best = r.block_pick(best, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
  {
    const uint64_t(*x)[kMaxCluster] = r.exchange(best);
    for (int q = 0; q < C; ++q) best = max(best, x[0][q]);
  }
  r.mx = key_value(uint32_t(best >> 32));
  r.first = int(~uint32_t(best));
  if (r.mx == -INFINITY || !(T > 0.f)) {  // the same in all CTAs of the row; no remote access follows
    if (r.rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = r.mx == -INFINITY ? -1 : r.first;
      a.logprobs[row] = r.mx == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const int w0 = r.w0, w1 = r.w1;
  const bool cut_k = k > 0 && k < a.V, cut_p = p < 1.f;
  uint64_t cut = 0;  // entries of composite >= cut are kept
  if (cut_k || cut_p) {
    for (int j = w0 + lane; j < w1; j += 32) r.v[j] = r.dist(r.v[j]);
    auto by_distance = [&](int j, int& b, float& w) {
      const float d = r.v[j];
      if (!(d > -kSpan)) return false;
      b = Row<BF16>::bin(d);
      w = Row<BF16>::weight(d);
      return true;
    };
    r.histogram(by_distance, cut_p);
    bool rebuilt = false;
    uint64_t through = r.total_mass;
    typename Row<BF16>::Goal g;
    if (cut_k && uint64_t(k) < r.total_count) {
      g.by_mass = false;
      g.k = k;
      g.want = 0.;
      cut = r.find_cut(g, 0, through, rebuilt);
    }
    if (cut_p) {
      g.by_mass = true;
      g.k = 0;
      g.want = double(p) * double(through);
      if (!(g.want > 0.)) {
        cut = best;
      } else {
        if (rebuilt) r.histogram(by_distance, true);
        uint64_t unused;
        cut = max(cut, r.find_cut(g, cut, unused, rebuilt));
      }
    }
  }
  // Weights of the kept entries, their mass, then the draw.
  cut = min(cut, best);
  const float cut_x = key_value(uint32_t(cut >> 32));
  const float cut_d = cut == 0 ? -INFINITY : r.dist(cut_x);
  uint32_t sh = 0, sl = 0;
  const bool filtered = cut_k || cut_p;
  for (int j = w0 + lane; j < w1; j += 32) {
    float d = r.v[j];
    if (!filtered) d = r.dist(d);
    float w = 0.f;
    if (d > -kSpan && d >= cut_d) {
      w = Row<BF16>::weight(d);
      const int i = r.begin + j;
      if (w < mp) w = 0.f;
      else if (d == cut_d && cut != 0 && composite(r.logit(i), i) < cut) w = 0.f;
      if (i == r.first) w = 1.f;
      uint32_t h, l;
      mass_halves(w, h, l);
      sh += h;
      sl += l;
    }
    r.v[j] = w;
  }
  uint64_t mass = warp_sum64((uint64_t(sh) << 18) + sl);  // at most 32 halves of 18 bits each
  if (lane == 0) s.wsum[warp] = mass;
  __syncthreads();
  uint64_t mine = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) mine += s.wsum[i];
  const uint64_t(*x)[kMaxCluster] = r.exchange(mine);
  uint64_t total = 0, before = 0;
  for (int q = 0; q < C; ++q) {
    if (q < r.rank) before += x[0][q];
    total += x[0][q];
  }
  uint64_t target = uint64_t(fmax(0., floor(double(a.u[row]) * double(total))));
  target = min(target, total - 1);
  if (target < before || target >= before + mine) return;
  for (int i = 0; i < warp; ++i) before += s.wsum[i];
  if (target < before || target >= before + mass) return;
  const int j = r.select_in_warp([&](int e) { return mass_of(r.v[e]); }, target, before);
  if (lane == 0) {
    const int i = r.begin + j;
    a.tokens[row] = i;
    a.logprobs[row] = float(double(r.dist(r.logit(i))) - log(double(total) / double(kFixed)));
  }
}

}  // namespace

int sample_max_vocabulary() { return kMaxCluster * (kMaxSlice - 16); }

void launch_sample_tokens(const SampleArgs& a, cudaStream_t stream) {
  if (a.R == 0) return;
  if (a.V < 1 || a.V > sample_max_vocabulary()) throw std::invalid_argument("sample_tokens: vocabulary size");
  auto slice = [&](int c) { return ((a.V + 7) / 8 + c - 1) / c * 8 + 8; };
  int C = 1;
  while (C < kMaxCluster && slice(C) > 8192 + 8) C *= 2;
  const int cap = slice(C) + 8;
  const size_t smem = sizeof(Shared) + size_t(cap) * 4;
  auto kernel = a.bf16 ? sample_kernel<true> : sample_kernel<false>;
  cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)), "sample_tokens smem");
  cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "sample_tokens cluster");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.R) * C, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel starts with pdl_wait()
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_flag() ? 2 : 1;
  cuda_check(cudaLaunchKernelEx(&cfg, kernel, a, C), "sample_tokens launch");
}

}  // namespace b200
