// Log probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits (include/q4gpu.h: q4gpu_token_logprobs).
#include <cstdint>
#include <type_traits>

#include "q4_paged.cuh"
#include "q4gpu_internal.h"

using namespace q4::paged;

namespace {

constexpr int kMostThreads = 512;
constexpr int kMostParts = 16;    // CTAs of a row, a cluster
constexpr int kCandidates = 1024;
constexpr float kLog2e = 1.4426950408889634f;

// Numbers that order like the logits: NaN above all, zeros of both signs alike.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return ~0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
  return order == ~0u ? __uint_as_float(0x7fffffffu)
                      : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// ... and like (logit, lower index first); above 0.
__device__ __forceinline__ uint64_t key_of(float v, int index) {
  return (uint64_t)order_of(v) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ bool is_number(float v) { return v < INFINITY; }  // neither NaN nor +infinity

template <int N>
__device__ __forceinline__ float largest(const float* x) {  // NaN if one is
  float m = x[0];
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) m = max3(m, x[i], x[i + 1]);
  if constexpr (N % 2 == 0) m = max3(m, x[N - 1], x[N - 1]);
  return m;
}

// 16 bytes of logits, which is how a row is read.
template <typename T>
struct Unit {
  static constexpr int V = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void load(const uint4* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "l"(p));
  }
  __device__ __forceinline__ void lowest() {  // all -infinity
    const uint32_t inf = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
    w = make_uint4(inf, inf, inf, inf);
  }
  __device__ __forceinline__ void get(float* x) const {
    if constexpr (sizeof(T) == 4)
      x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    else
      unpack8<T>(w, x);
  }
};

// How many logits are at least a bound; NaNs count as less.
template <typename T>
struct Counter {  // two at a time: the halves of a mask of ones are -1 each, and so is what they leave in a sum
  uint32_t sum = 0;
  int total = 0;
  static __device__ __forceinline__ uint32_t bound(T v) {
    const uint16_t b = *reinterpret_cast<const uint16_t*>(&v);
    return (uint32_t)b * 0x10001u;
  }
  __device__ __forceinline__ void add(const Unit<T>& u, uint32_t c) {
    const uint32_t w[4] = {u.w.x, u.w.y, u.w.z, u.w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, __half))
        sum += __hge2_mask(*reinterpret_cast<const __half2*>(&w[i]), *reinterpret_cast<const __half2*>(&c));
      else
        sum += __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), *reinterpret_cast<const __nv_bfloat162*>(&c));
    }
  }
  // sum = low (2^16 - 1) - high 2^16; at most 4 of each a unit
  __device__ __forceinline__ void flush() {
    const uint32_t low = (0u - sum) & 0xffffu, high = (low - (uint32_t)((sum + low) >> 16)) & 0xffffu;
    total += low + high, sum = 0;
  }
};
template <>
struct Counter<float> {
  int total = 0;
  static __device__ __forceinline__ float bound(float v) { return v; }
  __device__ __forceinline__ void add(const Unit<float>& u, float c) {
    total += (__uint_as_float(u.w.x) >= c) + (__uint_as_float(u.w.y) >= c) + (__uint_as_float(u.w.z) >= c) +
             (__uint_as_float(u.w.w) >= c);
  }
  __device__ __forceinline__ void flush() {}
};
// The next value of the type above v (NaN above infinity).
template <typename T>
__device__ __forceinline__ T above(T v) {
  using B = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
  constexpr B kSign = (B)1 << (sizeof(T) * 8 - 1);
  B b = *reinterpret_cast<const B*>(&v);
  if (b == kSign) b = 0;  // the zeros are one
  b = b & kSign ? b - 1 : b + 1;
  return *reinterpret_cast<const T*>(&b);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// What is known of some of a row's logits: the largest number m (-infinity: none), and over all but one place of it
// S = sum e^(x - m) and T = sum e^(x - m) (x - m).
struct Sums {
  float m, s, t;
  // The same against a larger m, with the place of the old one.
  __device__ __forceinline__ void raise(float to) {
    const float f = m == -INFINITY ? 0.f : ex2((m - to) * kLog2e);
    t = f == 0.f ? 0.f : f * fmaf(m - to, s + 1.f, t);
    s = f == 0.f ? 0.f : (s + 1.f) * f;
    m = to;
  }
};
// The sums of each lane's logits joined; every lane gets them.
__device__ __forceinline__ Sums join(Sums x) {
  const float m = warp_max(x.m);
  const unsigned first = __ballot_sync(~0u, x.m == m);
  if ((threadIdx.x & 31) != (unsigned)(__ffs(first) - 1)) x.raise(m);
  return Sums{m, warp_sum(x.s), warp_sum(x.t)};
}

// What a CTA knows of its part of a row.
struct Part {
  Sums sums;
  int ahead, odd;
  uint64_t top[Q4GPU_TOP_MAX];  // its first ones, falling; 0: no more
};

// `parts` CTAs a row (a cluster), each a stretch of its 16-byte units; what stands before the first and behind the last
// boundary of 16 bytes is the first CTA's.  With m the row's largest logit,
//   log p_t = (x_t - m) - log1p(S),   H = log1p(S) - T / (1 + S),
// (see Sums) sums without cancellation however certain the row is.  The logits are read once: a warp
// holds its sums against its own largest so far, which few steps change.
// Of the likeliest only the largest of each thread is followed on the way.  The top-th of the largest of 32 groups of threads
// bounds the top-th of all from below, and about as many logits as are wanted lie above
// it: the few threads whose largest does are read again, from L2, and what lies above
// the bound is ranked by counting.
template <typename T>
__global__ void __launch_bounds__(kMostThreads) token_logprobs_kernel(q4gpu_logprob_args a, int parts) {
  constexpr int V = Unit<T>::V, U = 2;
  __shared__ Part s_part;
  __shared__ Sums s_sums[kMostThreads / 32];
  __shared__ int s_ahead[kMostThreads / 32], s_odd, s_threads, s_found;
  __shared__ uint64_t s_group[32], s_key[kCandidates];
  __shared__ uint16_t s_thread[kMostThreads];
  const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
  const int part = blockIdx.x % (unsigned)parts;
  const int64_t row = blockIdx.x / (unsigned)parts;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const int head = min(a.vocab, (int)((0 - reinterpret_cast<uintptr_t>(x)) & 15) / (int)sizeof(T));
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int units = (a.vocab - head) / V, tail = head + units * V;  // where the last few begin
  const int share = (units + parts - 1) / parts, u0 = min(units, part * share), u1 = min(units, u0 + share);

  Unit<T> next[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    next[j].lowest();
    if (u0 + tid + j * threads < u1) next[j].load(body + u0 + tid + j * threads);
  }
  const int64_t given = a.targets ? a.targets[row] : -1;
  const bool known = given >= 0 && given < a.vocab;
  const T mine = known ? x[given] : from_f32<T>(__uint_as_float(0x7fffffffu));
  // logits before the target's unit count from its value on, later ones above it
  const int mine_unit = !known ? 0 : given < head ? -1 : given >= tail ? units : (int)(given - head) / V;
  const auto from = Counter<T>::bound(mine), past = Counter<T>::bound(above(mine));
  // the ends of the row, one logit a lane of one warp, and the logits before the target in its unit
  const bool ends = part == 0 && warp == 0;
  const int end_at = lane < 16 ? lane : tail + lane - 16;
  const bool end_there = ends && (lane < 16 ? lane < head : end_at < a.vocab);
  const float end = end_there ? to_f32(x[end_at]) : -INFINITY;
  const int near_at = head + mine_unit * V + lane;
  const bool tie = known && warp == 0 && mine_unit >= u0 && mine_unit < u1 && near_at < given &&
                   to_f32(x[near_at]) == to_f32(mine);
  if (tid == 0) s_odd = s_threads = s_found = 0;
  if (tid < Q4GPU_TOP_MAX) s_part.top[tid] = 0;

  Sums sums{-INFINITY, 0.f, 0.f};  // m: the warp's; s, t: this lane's share
  bool odd = false;                // a NaN or +infinity
  // N more logits of each lane (-infinity for none), where one reaches the warp's largest
  auto careful = [&](float* v, auto count) {
    constexpr int N = decltype(count)::value;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!is_number(v[i])) odd = true, v[i] = -INFINITY;
      most = fmaxf(most, v[i]);
    }
    most = warp_max(most);
    int same = 0;  // one place of the largest is left out of the sums
    if (most > sums.m) {
      const float f = sums.m == -INFINITY ? 0.f : ex2((sums.m - most) * kLog2e);
      const float place = lane == 0 ? 1.f : 0.f;  // that of the old largest comes in
      sums.t = f == 0.f ? 0.f : f * fmaf(sums.m - most, sums.s + place, sums.t);
      sums.s = f == 0.f ? 0.f : (sums.s + place) * f;
      sums.m = most;
      same = -1;
    }
    if (most == -INFINITY && sums.m == -INFINITY) return;
    int mine_same = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = v[i] - sums.m, e = ex2(d * kLog2e);
      if (v[i] == sums.m) {
        ++mine_same;
      } else if (e > 0.f) {
        sums.s += e, sums.t = fmaf(e, d, sums.t);
      }
    }
    same += __reduce_add_sync(~0u, mine_same);
    if (lane == 0) sums.s += (float)same;
  };

  float most = -INFINITY;  // this thread's largest and the first unit that holds it
  int most_unit = u0 + tid;
  Counter<T> counter;
  const int steps = (u1 - u0 + threads * U - 1) / (threads * U);
  for (int step = 0; step < steps; ++step) {
    Unit<T> now[U];
    const int u = u0 + tid + step * U * threads;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      now[j] = next[j];
      const int later = u + (U + j) * threads;
      if (later < u1) next[j].load(body + later);
      else next[j].lowest();
    }
    float v[U * V], tops[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      now[j].get(v + j * V);
      tops[j] = largest<V>(v + j * V);
      if (!(tops[j] <= most) && most == most) most = tops[j], most_unit = u + j * threads;
      const int uj = u + j * threads;
      if (uj < u1) counter.add(now[j], uj < mine_unit ? from : past);
    }
    if ((step & 4095) == 4095) counter.flush();
    if (__any_sync(~0u, !(largest<U>(tops) < sums.m))) {
      careful(v, std::integral_constant<int, U * V>());
    } else {
      const float before = sums.t;
      const uint64_t m2 = pair_of(-sums.m, -sums.m), c2 = pair_of(kLog2e, kLog2e);
      uint64_t s2 = 0, t2 = 0;
#pragma unroll
      for (int i = 0; i < U * V; i += 2) {
        const uint64_t d = add_pair(pair_of(v[i], v[i + 1]), m2);
        float ex, ey;
        split_pair(mul_pair(d, c2), ex, ey);
        const uint64_t e = pair_of(ex2(ex), ex2(ey));
        s2 = add_pair(s2, e);
        t2 = fma_pair(e, d, t2);
      }
      float p, q;
      split_pair(s2, p, q);
      sums.s += p + q;
      split_pair(t2, p, q);
      p += q;
      if (!(p == p)) {  // 0 times -infinity
        p = 0.f;
#pragma unroll
        for (int i = 0; i < U * V; ++i) {
          const float d = v[i] - sums.m, e = ex2(d * kLog2e);
          if (e > 0.f) p = fmaf(e, d, p);
        }
      }
      sums.t = before + p;
    }
  }
  counter.flush();
  int ahead = counter.total;
  const uint64_t end_key = end_there ? key_of(end, end_at) : 0, mine_key = known ? key_of(to_f32(mine), (int)given) : ~0ull;
  if (ends) {
    float v = end;
    careful(&v, std::integral_constant<int, 1>());
    ahead += end_key > mine_key;
  }
  if (odd) s_odd = 1;
  {
    Sums w = sums;
    w.s = warp_sum(w.s), w.t = warp_sum(w.t);
    ahead = __reduce_add_sync(~0u, ahead);
    if (lane == 0) s_sums[warp] = w, s_ahead[warp] = ahead;
  }
  // the groups' largest: `warps` neighbouring lanes each
  uint64_t key = u0 + tid < u1 ? (uint64_t)order_of(most) << 32 | (uint32_t)~most_unit : 0;
  if (a.top) {
    uint64_t g = key;
    for (int o = 1; o < warps; o <<= 1) g = max(g, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)g, o));
    if (tid % warps == 0) s_group[tid / warps] = g;
  }
  __syncthreads();
  if (a.top) {
    const uint64_t g = s_group[lane];
    int before = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) before += s_group[i] > g || (s_group[i] == g && i < lane);
    const unsigned at = __ballot_sync(~0u, before == a.top - 1);
    const uint64_t bound = __shfl_sync(~0u, (unsigned long long)g, __ffs(at) - 1);
    if (key && key >= bound) s_thread[atomicAdd(&s_threads, 1)] = (uint16_t)tid;
    auto found = [&](uint64_t k) {
      const int n = atomicAdd(&s_found, 1);
      if (n < kCandidates) s_key[n] = k;
    };
    if (end_there && end_key >= (bound & ~0xffffffffull)) found(end_key);
    __syncthreads();
    for (int i = warp; i < s_threads; i += warps)
      for (int u = u0 + s_thread[i] + lane * threads; u < u1; u += 32 * threads) {
        Unit<T> w;
        float v[V];
        w.load(body + u);
        w.get(v);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (((uint64_t)order_of(v[e]) << 32 | (uint32_t)~u) >= bound) found(key_of(v[e], head + u * V + e));
      }
    __syncthreads();
    const int n = s_found;
    if (n <= kCandidates) {
      for (int i = tid; i < n; i += threads) {
        const uint64_t k = s_key[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_key[j] > k;
        if (rank < a.top) s_part.top[rank] = k;
      }
    } else {  // many logits in few threads: one after another over the whole part
      uint64_t last = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        uint64_t best = end_key < last ? end_key : 0;
        for (int u = u0 + tid; u < u1; u += threads)
          for (int e = 0; e < V; ++e) {
            const uint64_t c = key_of(to_f32(x[head + u * V + e]), head + u * V + e);
            if (c < last) best = max(best, c);
          }
        for (int o = 16; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)best, o));
        __syncthreads();
        if (lane == 0) s_key[warp] = best;
        __syncthreads();
        for (int w = 0; w < warps; ++w) best = max(best, s_key[w]);
        if (tid == 0) s_part.top[k] = best;
        last = best;
      }
    }
  }
  if (s_odd && known) {  // the order has NaNs, which comparisons leave out
    __syncthreads();
    ahead = end_key > mine_key;
    for (int u = u0 + tid; u < u1; u += threads)
      for (int e = 0; e < V; ++e) ahead += key_of(to_f32(x[head + u * V + e]), head + u * V + e) > mine_key;
    ahead = __reduce_add_sync(~0u, ahead);
    if (lane == 0) s_ahead[warp] = ahead;
    __syncthreads();
  }
  if (warp == 0) {
    Sums w{-INFINITY, 0.f, 0.f};
    if (lane < warps) w = s_sums[lane];
    w = join(w);
    int n = (lane < warps ? s_ahead[lane] : 0) + (tie && !s_odd);
    n = __reduce_add_sync(~0u, n);
    if (lane == 0) s_part.sums = w, s_part.ahead = n, s_part.odd = s_odd;
  }

  // the parts joined by the first CTA
  const Part* all = &s_part;
  auto part_at = [&](int p) {
    const Part* q = all;
    if (parts > 1)
      asm("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(all), "r"(p));
    return q;
  };
  if (parts > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  if (part == 0) {
    const float nan = __uint_as_float(0x7fffffffu);
    if (warp == 0 || a.top) {  // (every warp that writes likeliest tokens needs the sums)
      Sums w{-INFINITY, 0.f, 0.f};
      int n = 0, no = 0;
      if (lane < parts) {
        const Part* q = part_at(lane);
        w = q->sums, n = q->ahead, no = q->odd;
      }
      w = join(w);
      n = __reduce_add_sync(~0u, n);
      const bool bad = __any_sync(~0u, no), none = w.m == -INFINITY;
      const float norm = log1pf(w.s);
      auto logprob = [&](float v) { return bad ? nan : none ? -INFINITY : (v - w.m) - norm; };
      if (tid == 0) {
        if (a.targets) {
          a.logprob[row] = known ? logprob(to_f32(mine)) : 0.f;
          a.rank[row] = known ? n + 1 : 0;
          if (given >= a.vocab && a.err_flag) *a.err_flag = 1;
        }
        a.entropy[row] = bad ? nan : none ? 0.f : norm - w.t / (1.f + w.s);
      }
      for (int i = tid; i < parts * a.top; i += threads) {
        const int p = i / a.top, k = i - p * a.top;
        const uint64_t c = part_at(p)->top[k];
        int rank = k;
        for (int q = 0; q < parts; ++q) {
          if (q == p) continue;
          const uint64_t* t = part_at(q)->top;
          int lo = 0;  // how many of the part's are before this one
#pragma unroll
          for (int s = Q4GPU_TOP_MAX / 2; s; s >>= 1)
            if (t[lo + s - 1] > c) lo += s;
          rank += lo + (t[lo] > c);
        }
        if (c && rank < a.top) {
          a.top_logprob[row * a.top + rank] = logprob(logit_of((uint32_t)(c >> 32)));
          a.top_index[row * a.top + rank] = ~(int)(uint32_t)c;
        }
      }
    }
  }
  if (parts > 1)  // the first CTA has read the others' memory
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CTAs of a row and threads of a CTA.
struct Shape {
  int parts, threads;
};
Shape shape_of(const q4gpu_logprob_args& a) {
  const int64_t units = (int64_t)a.vocab * (a.dtype == Q4GPU_F32 ? 4 : 2) / 16;
  Shape s{1, kMostThreads};
  while (s.threads > 32 && units <= s.threads * 2) s.threads /= 4;
  if (s.threads < 32) s.threads = 32;
  while (s.parts < kMostParts && a.rows * s.parts * s.threads < 148 * 1024 && units / s.parts >= 4 * s.threads)
    s.parts *= 2;
  return s;
}

template <typename T>
int launch(const q4gpu_logprob_args& a, cudaStream_t stream) {
  const Shape s = shape_of(a);
  if (a.rows * s.parts > INT32_MAX) return q4gpu_fail(Q4GPU_ERR_SHAPE, "logprobs: too many rows");
  static unsigned char ready[Q4GPU_MAX_DEVICES];
  if (s.parts > 8) {  // more CTAs than any cluster may have: once per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(dev < Q4GPU_MAX_DEVICES && ready[dev]))
      e = cudaFuncSetAttribute(token_logprobs_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "logprobs: cluster size: %s", cudaGetErrorString(e));
    if (dev < Q4GPU_MAX_DEVICES) ready[dev] = 1;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = s.parts, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * s.parts)), cfg.blockDim = dim3(s.threads);
  cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = s.parts > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a, s.parts);
  if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "logprobs: launch: %s", cudaGetErrorString(e));
  return q4gpu_check_launch();
}

int check(const q4gpu_logprob_args* a) {
  if (!a) return q4gpu_fail(Q4GPU_ERR_ARG, "logprobs: null arguments");
  if (a->dtype != Q4GPU_F32 && a->dtype != Q4GPU_F16 && a->dtype != Q4GPU_BF16)
    return q4gpu_fail(Q4GPU_ERR_ARG, "logprobs: dtype is F32, F16 or BF16");
  if (a->rows < 0 || a->rows > INT32_MAX)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "logprobs: %lld rows", (long long)a->rows);
  if (a->vocab < 1) return q4gpu_fail(Q4GPU_ERR_SHAPE, "logprobs: a vocabulary of %d", a->vocab);
  if (a->top < 0 || a->top > Q4GPU_TOP_MAX || a->top > a->vocab)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "logprobs: top = %d of a vocabulary of %d, at most %d", a->top, a->vocab,
                      Q4GPU_TOP_MAX);
  if (a->rows == 0) return Q4GPU_OK;
  if (!a->logits || !a->entropy || (a->targets && (!a->logprob || !a->rank)) ||
      (a->top && (!a->top_logprob || !a->top_index)))
    return q4gpu_fail(Q4GPU_ERR_ARG, "logprobs: null pointer");
  const uintptr_t size = a->dtype == Q4GPU_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->logits) % size)
    return q4gpu_fail(Q4GPU_ERR_ALIGN, "logprobs: logits start on a boundary of their type");
  return Q4GPU_OK;
}

}  // namespace

extern "C" int q4gpu_token_logprobs(const q4gpu_logprob_args* a, void* stream) {
  const int rc = check(a);
  if (rc != Q4GPU_OK || a->rows == 0) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == Q4GPU_F32) return launch<float>(*a, s);
  return a->dtype == Q4GPU_F16 ? launch<__half>(*a, s) : launch<__nv_bfloat16>(*a, s);
}
