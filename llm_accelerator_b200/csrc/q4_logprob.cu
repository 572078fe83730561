// Log probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits (include/q4gpu.h: q4gpu_token_logprobs).
#include <cstdint>
#include <type_traits>

#include "q4_paged.cuh"
#include "q4gpu_internal.h"

using namespace q4::paged;

namespace {

constexpr int kMostThreads = 512;
constexpr int kMostParts = 8;  // CTAs of a row, a cluster
constexpr int kUnit = 16;       // logits of a lane and step
constexpr int kGroups = 64;     // of a row's threads, at most
constexpr int kCandidates = 1024;  // of a CTA, for the likeliest
constexpr int kReach = 48;         // threads whose largest reach the bound that are looked at without a better one
constexpr int kFew = 64;           // ... that go to the first CTA as they are
static_assert(Q4GPU_TOP_MAX <= kFew && kCandidates * 8 <= 64 * kUnit * 2 * 4, "the candidates fit in the smallest ring");
static_assert(Q4GPU_TOP_MAX <= kGroups, "a group for each of the likeliest");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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

// 16 neighbouring logits in pieces of 16 bytes, what a lane takes of a row at a time.
template <typename T>
struct Unit {
  static constexpr int kPieces = kUnit * sizeof(T) / 16;
  static constexpr int kStages = sizeof(T) == 4 ? 3 : 4;  // steps of the ring: all but one of them in flight
  uint4 w[kPieces];
  __device__ __forceinline__ void load(const uint4* p) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                   : "l"(p + i));
  }
  __device__ __forceinline__ void take(int i, uint32_t at) {  // piece i from shared memory
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                 : "r"(at)
                 : "memory");
  }
  // Place of piece c of lane r's unit among a warp's: neighbouring lanes' pieces lie in different banks.
  static __device__ __forceinline__ int place(int r, int c) {
    return r * kPieces + (c ^ (sizeof(T) == 4 ? (r >> 1) & 3 : (r >> 2) & 1));
  }
  static __device__ __forceinline__ void put_lowest(uint32_t at) {  // a piece of -infinities to shared memory
    const uint32_t inf = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(inf) : "memory");
  }
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if constexpr (sizeof(T) == 4)
        x[4 * i] = __uint_as_float(w[i].x), x[4 * i + 1] = __uint_as_float(w[i].y),
              x[4 * i + 2] = __uint_as_float(w[i].z), x[4 * i + 3] = __uint_as_float(w[i].w);
      else
        unpack8<T>(w[i], x + 8 * i);
    }
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4& p = u.w[i / 4];
      const uint32_t w = i % 4 == 0 ? p.x : i % 4 == 1 ? p.y : i % 4 == 2 ? p.z : p.w;
      if constexpr (__is_same(T, __half))
        sum += __hge2_mask(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&c));
      else
        sum += __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&c));
    }
  }
  // sum = low (2^16 - 1) - high 2^16; at most 8 of each a unit
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
    float x[kUnit];
    u.get(x);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) total += x[i] >= c;
  }
  __device__ __forceinline__ void flush() {}
};
// The next value of the type above v (NaN above infinity, and above NaN, whose next bits may be those of a zero).
template <typename T>
__device__ __forceinline__ T above(T v) {
  using B = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
  constexpr B kSign = (B)1 << (sizeof(T) * 8 - 1);
  B b = *reinterpret_cast<const B*>(&v);
  if (to_f32(v) != to_f32(v)) return v;
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

// What a warp knows of its logits: m, the largest number of its own and of its CTA's first step (-infinity: none), and
// sums of e^(x - m) and e^(x - m) (x - m).  One place of m is left out of the row's sums; `own`: it is one of this warp's.
struct Sums {
  float m, s, t;
  int own;
  // The same against a larger m; `place`: with that of the old one.
  __device__ __forceinline__ void raise(float to, bool place) {
    const float f = m == -INFINITY ? 0.f : ex2((m - to) * kLog2e), all = place ? s + 1.f : s;
    t = f == 0.f ? 0.f : f * fmaf(m - to, all, t);
    s = f == 0.f ? 0.f : all * f;
    m = to;
  }
};

// What a lane holds of its warp's steps; s and t are the lane's share, the rest is the same in all.
struct Held {
  Sums sums{-INFINITY, 0.f, 0.f, 0};
  bool left = false;  // the place to leave out is among the logits to come
  bool odd = false;   // a NaN or +infinity (this lane's)
  // The steps' reference, m log2e rounded, and what the rounding left out: e^(x - m) = 2^(x log2e - ref) 2^-rest.  Not
  // for numbers so large that the rest is.
  float ref = 0.f, rest = 0.f, back = 1.f;
  bool tame = false;

  __device__ __forceinline__ void raise(float to, bool own) {
    sums.raise(to, sums.own && (threadIdx.x & 31) == 0);
    sums.own = own;
    ref = to * kLog2e, rest = fmaf(to, kLog2e, -ref), back = ex2(-rest);
    tame = fabsf(to) < 65536.f;
  }
  // N more logits of each lane (-infinity for none), where one may reach m.
  template <int N>
  __device__ __forceinline__ void careful(float* v) {
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!is_number(v[i])) odd = true, v[i] = -INFINITY;
      most = fmaxf(most, v[i]);
    }
    most = warp_max(most);
    int same = 0;
    if (most > sums.m) {  // one place of the largest is left out of the sums
      raise(most, true);
      same = -1;
    }
    if (sums.m == -INFINITY) return;
    if (left) same = -1, left = false;
    int mine = 0;
    float s = 0.f, t[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = v[i] - sums.m;
      float e = ex2(d * kLog2e);
      if (v[i] == sums.m) ++mine, e = 0.f;
      s += e;
      if (e > 0.f) t[i & 1] = fmaf(e, d, t[i & 1]);
    }
    same += __reduce_add_sync(~0u, mine);
    sums.s += (threadIdx.x & 31) == 0 ? s + (float)same : s, sums.t += t[0] + t[1];
  }
};
// Out of line: few steps come here, and the registers it takes cost the steps that do not.
template <typename T>
__device__ __noinline__ Held careful_step(Held h, uint32_t warp_at) {
  Unit<T> now;
#pragma unroll
  for (int i = 0; i < Unit<T>::kPieces; ++i) now.take(i, warp_at + Unit<T>::place(threadIdx.x & 31, i) * 16);
  float v[kUnit];
  now.get(v);
  h.careful<kUnit>(v);
  return h;
}

// What a warp knows in the end: its sums, its logits before the target, whether there is a NaN or +infinity among them.
struct Record {
  Sums sums;
  int ahead, odd;
};
// What the CTAs of a row tell each other.
struct Board {
  uint64_t group[kGroups];  // the largest of each group of threads
  uint64_t key[kMostParts * kFew];
  Record record[kMostParts * kMostThreads / 32];
  int found;
};

// `parts` CTAs a row (a cluster), each a stretch of its units of 16 logits; what stands before the first boundary
// of 16 bytes and behind the last whole unit is the first CTA's.  With m the row's largest logit, S the sum of
// e^(x - m) over all but one place of it and T = sum e^(x - m) (x - m),
//   log p_t = (x_t - m) - log1p(S),   H = log1p(S) - T / (1 + S),
// sums without cancellation however certain the row is.  The logits are read once; a warp holds its sums against the
// largest logit of its own and of the CTA's first step, which few steps change.
// Of the likeliest only each thread's largest is followed on the way.  The top-th of the largest of 32 or 64 groups of
// threads bounds the top-th of all from below, and about as many logits as are wanted lie above it: the units with the
// few threads' largest that do are read again, from L2 (all of a thread's units where a second one's does), and what
// lies above the bound is ranked by counting.  A CTA whose many threads reach the bound goes by the top-th of those.
// Only where a few threads hold more than 1024 of the logits above it (large ones at a distance that is a multiple of
// 16 times the threads) the first CTA takes one after another over the whole row.
// 2048 rows of 151936 in bf16 take 165 us (3.8 TB/s), bound by instructions (63700 of a warp's a row with a target and 5
// alternatives, which fill 65 % of the issue slots) and by a row's beginning and end, 11 of its 24 us beside one other
// CTA; 1024 rows in float32 112 us (5.6 TB/s), bound by memory.
template <typename T>
__global__ void __launch_bounds__(kMostThreads, 2) token_logprobs_kernel(q4gpu_logprob_args a, int parts) {
  constexpr int P = Unit<T>::kPieces, S = Unit<T>::kStages;
  extern __shared__ uint4 ring[];  // [warp][stage][Unit::place]
  __shared__ Board s_board;
  __shared__ uint64_t s_bound, s_top[Q4GPU_TOP_MAX];
  __shared__ uint16_t s_thread[kMostThreads];
  __shared__ int s_unit[kMostThreads], s_threads, s_units, s_found;
  __shared__ float s_first[kMostThreads / 32];
  __shared__ Record s_all;
  const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
  const int part = blockIdx.x % (unsigned)parts;
  const int64_t row = blockIdx.x / (unsigned)parts;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const int head = min(a.vocab, (int)((0 - reinterpret_cast<uintptr_t>(x)) & 15) / (int)sizeof(T));
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int units = (a.vocab - head) / kUnit, tail = head + units * kUnit;  // where the last few begin
  const int share = (units + parts - 1) / parts, u0 = min(units, part * share), u1 = min(units, u0 + share);
  const int whole = (u1 - u0) / threads, steps = (u1 - u0 + threads - 1) / threads;

  // A warp fetches its lanes' units together, neighbouring pieces by neighbouring lanes.
  constexpr uint32_t kStage = 32 * P * 16;
  const uint32_t warp_at = (uint32_t)__cvta_generic_to_shared(ring) + warp * S * kStage;
  const uint32_t put_at = warp_at + Unit<T>::place(lane / P, lane % P) * 16;  // the next 32 pieces' are 512 bytes on
  const uint4* source = body + (int64_t)(u0 + warp * 32) * P + lane;          // of the step that is fetched next
  auto fetch = [&](int stage) {
#pragma unroll
    for (int i = 0; i < P; ++i) cp16(put_at + stage * kStage + i * 512, source + 32 * i, true);
    cp_commit();
    source += threads * P;
  };
  auto fetch_some = [&](int step) {  // that may not be whole, or not there
    if (step < whole) return fetch(step % S);
    if (step < steps) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint32_t to = put_at + step % S * kStage + i * 512;
        if (u0 + step * threads + warp * 32 + (32 * i + lane) / P < u1)
          cp16(to, source + 32 * i, true);
        else
          Unit<T>::put_lowest(to);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch_some(i);

  const int64_t given = a.targets ? a.targets[row] : -1;
  const bool known = given >= 0 && given < a.vocab;
  const T mine = known ? x[given] : from_f32<T>(__uint_as_float(0x7fffffffu));
  // logits before the target's unit count from its value on, later ones above it
  const int mine_unit = !known ? 0 : given < head ? -1 : given >= tail ? units : (int)(given - head) / kUnit;
  const auto from = Counter<T>::bound(mine), past = Counter<T>::bound(above(mine));
  // the ends of the row, one logit a lane of one warp, and the logits before the target in its unit
  const bool ends = part == 0 && warp == 0 && (head > 0 || tail < a.vocab);
  // (places are compared by their distance: next to 2^31 a sum with the lane would wrap)
  const bool end_there = ends && (lane < 8 ? lane < head : lane - 8 < a.vocab - tail);
  const int end_at = !end_there ? 0 : lane < 8 ? lane : tail + lane - 8;
  const float end = end_there ? to_f32(x[end_at]) : -INFINITY;
  const int near = head + mine_unit * kUnit;
  const bool tie = known && mine_unit >= u0 && mine_unit < u1 && warp == ((mine_unit - u0) & (threads - 1)) >> 5 &&
                   lane < (int)given - near && to_f32(x[near + lane]) == to_f32(mine);
  if (tid < kGroups) s_board.group[tid] = 0;
  if (tid == 0) s_board.found = s_threads = s_units = s_found = 0;
  __syncwarp();  // (the cluster's barriers are for whole warps, and lanes have taken ways of their own)
  if (parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  auto board = [&](int p) {  // part p's
    Board* q = &s_board;
    if (parts > 1) asm("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(&s_board), "r"(p));
    return q;
  };

  Held h;
  float most = -INFINITY;  // this thread's largest and the first unit that holds it
  int most_unit = u0 + tid;
  float second = -INFINITY;  // no other unit of the thread has a larger one
  Counter<T> counter;
  int counted = 0;
  const float target = known ? to_f32(mine) : INFINITY;
  float limit = -INFINITY;  // m where the fast way may go up to it
  uint32_t get_at[P];
#pragma unroll
  for (int i = 0; i < P; ++i) get_at[i] = warp_at + Unit<T>::place(lane, i) * 16;
  if (steps > 0) {  // the largest of the CTA's first step (of no later one, or it would depend on how far each warp is)
    cp_wait<S - 2>();
    __syncwarp();
    Unit<T> now;
    float v[kUnit];
#pragma unroll
    for (int i = 0; i < P; ++i) now.take(i, get_at[i]);
    now.get(v);
    const float top = largest<kUnit>(v), w = warp_max(is_number(top) ? top : -INFINITY);
    if (lane == 0) s_first[warp] = w;
    __syncthreads();
    const float m = lane < warps ? s_first[lane] : -INFINITY, all = warp_max(m);
    h.left = __ffs(__ballot_sync(~0u, m == all)) - 1 == warp;
    if (all > -INFINITY) h.raise(all, h.left);
    limit = h.tame ? h.sums.m : -INFINITY;
  }
  int u = u0 + tid;
  auto add = [&](int stage, auto whole_step, auto fetch_next) {
    constexpr bool kWhole = decltype(whole_step)::value;
    cp_wait<S - 2>();
    __syncwarp();
    Unit<T> now;
#pragma unroll
    for (int i = 0; i < P; ++i) now.take(i, get_at[i] + stage * kStage);
    fetch_next();  // into the stage that was read a step before: the warp was whole since
    float v[kUnit];
    now.get(v);
    const float top = largest<kUnit>(v);
    second = fmaxf(second, fminf(top, most));
    if (!(top <= most) && most == most) most = top, most_unit = u;
    if (__any_sync(~0u, !(top < target))) {  // a warp's logits mostly lie below the target's
      if (kWhole || u < u1) counter.add(now, u < mine_unit ? from : past);
      if ((++counted & 4095) == 0) counter.flush();
    }
    if (__any_sync(~0u, !(top < limit))) {
      h = careful_step<T>(h, warp_at + stage * kStage);
      limit = h.tame ? h.sums.m : -INFINITY;
    } else {
      // e = 2^(x log2e - ref), a product and a sum with one rounding
      const uint64_t r2 = pair_of(-h.ref, -h.ref), c2 = pair_of(kLog2e, kLog2e);
      uint64_t s2 = 0, p2 = 0;
#pragma unroll
      for (int i = 0; i < kUnit; i += 2) {
        const uint64_t d = fma_pair(pair_of(v[i], v[i + 1]), c2, r2);
        float x, y;
        split_pair(d, x, y);
        const uint64_t e = pair_of(ex2(x), ex2(y));
        s2 = i ? add_pair(s2, e) : e;
        p2 = fma_pair(e, d, p2);
      }
      float s, p, x;
      split_pair(s2, s, x);
      s += x;
      split_pair(p2, p, x);
      p += x;
      if (kWhole || u < u1) {
        h.sums.s = fmaf(s, h.back, h.sums.s);
        h.sums.t = fmaf(fmaf(-h.rest, s, p), h.back * kLn2, h.sums.t);
      }
    }
    u += threads;
  };
  int step = 0;
  for (; step + 2 * S - 1 <= whole; step += S) {
#pragma unroll
    for (int i = 0; i < S; ++i) add(i, std::true_type(), [&] { fetch((i + S - 1) % S); });
  }
  for (; step < steps; ++step) add(step % S, std::false_type(), [&] { fetch_some(step + S - 1); });
  Sums sums = h.sums;
  if (__any_sync(~0u, sums.t != sums.t)) {  // 0 times -infinity: rows with masks, whose sums are taken again
    sums.t = 0.f;
    for (int i = u0 + tid; i < u1; i += threads) {
      Unit<T> now;
      float v[kUnit];
      now.load(body + (int64_t)i * P);
      now.get(v);
#pragma unroll
      for (int k = 0; k < kUnit; ++k) {
        const float d = v[k] - sums.m, e = ex2(d * kLog2e);
        if (e > 0.f) sums.t = fmaf(e, d, sums.t);
      }
    }
  }
  h.sums = sums;
  counter.flush();
  int ahead = counter.total + tie;
  const uint64_t end_key = end_there ? key_of(end, end_at) : 0;
  const uint64_t mine_key = known ? key_of(to_f32(mine), (int)given) : ~0ull;
  if (ends) {
    float v = end;
    h.careful<1>(&v);
    ahead += end_key > mine_key;
  }
  const bool odd = __any_sync(~0u, h.odd);
  if (odd && known) {  // the order has NaNs, which comparisons leave out
    ahead = end_key > mine_key;
    for (int u = u0 + tid; u < u1; u += threads)
      for (int i = head + u * kUnit; i < head + (u + 1) * kUnit; ++i) ahead += key_of(to_f32(x[i]), i) > mine_key;
  }
  ahead = __reduce_add_sync(~0u, ahead);
  sums = h.sums;
  sums.s = warp_sum(sums.s), sums.t = warp_sum(sums.t);
  uint64_t key = u0 + tid < u1 ? (uint64_t)order_of(most) << 32 | (uint32_t)~most_unit : 0;
  const int groups = a.top <= kGroups / 4 ? kGroups / 2 : kGroups;  // (fewer for a few, whose bound is as good)
  const int span = threads * parts / groups, lanes = min(span, 32);  // threads of a group, and those of them in a warp
  uint64_t group = key;
  if (a.top)
    for (int o = 1; o < lanes; o <<= 1)
      group = max(group, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)group, o));

  __syncwarp();
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all boards are clean
  Board* const first = board(0);
  if (lane == 0) first->record[part * warps + warp] = Record{sums, ahead, odd};
  if (a.top) {
    const int g = (part * threads + tid) / span;
    if (span > 32) {
      if (lane < parts) atomicMax(reinterpret_cast<unsigned long long*>(&board(lane)->group[g]), (unsigned long long)group);
    } else if (lane % lanes == 0) {
      for (int p = 0; p < parts; ++p) board(p)->group[g] = group;
    }
  }
  uint64_t* const list = reinterpret_cast<uint64_t*>(ring);  // (its logits are read) this CTA's candidates
  auto meet = [&] {  // of the row's CTAs
    __syncwarp();
    if (parts > 1)
      asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else
      __syncthreads();
  };
  meet();
  if (a.top) {
    // the group whose largest is the top-th: `peers` neighbouring lanes compare one with all
    const int peers = threads / groups, g = tid / peers;
    const uint64_t k = s_board.group[g];
    int before = 0;
    for (int i = tid % peers; i < groups; i += peers) before += s_board.group[i] > k || (s_board.group[i] == k && i < g);
    for (int o = 1; o < peers; o <<= 1) before += __shfl_xor_sync(~0u, before, o);
    if (before == a.top - 1) s_bound = k;
    __syncthreads();
    uint64_t bound = s_bound;
    auto look = [&] {  // threads that reach the bound; mostly one unit is all there is to look at
      if (!key || key < bound) return;
      if (most == most && order_of(second) < (uint32_t)(bound >> 32))
        s_unit[atomicAdd(&s_units, 1)] = most_unit;
      else
        s_thread[atomicAdd(&s_threads, 1)] = (uint16_t)tid;
    };
    look();
    __syncthreads();
    // Mostly they are few.  Where they are many (equal logits, as masks leave them, or logits that fall or rise along the
    // row) the top-th of theirs is the better bound: this CTA has no more to offer.
    const int reach = s_units + s_threads;
    if (reach > kReach) {
      __syncthreads();
      if (tid == 0) s_units = s_threads = 0;
      __syncthreads();
      if (key && key >= bound) list[atomicAdd(&s_threads, 1)] = key;
      __syncthreads();
      if (key && key >= bound) {
        int rank = 0;
        for (int i = 0; i < reach; ++i) rank += list[i] > key;
        if (rank == a.top - 1) s_bound = key;
      }
      if (tid == 0) s_threads = 0;
      __syncthreads();
      bound = s_bound;
      look();
      __syncthreads();
    }
    const uint32_t bound_value = (uint32_t)(bound >> 32);
    auto found = [&](uint64_t k) {
      const int n = atomicAdd(&s_found, 1);
      if (n < kCandidates) list[n] = k;
    };
    if (end_there && end_key >= (bound & ~0xffffffffull)) found(end_key);
    const int single = s_units, looks = single + s_threads * steps;
    for (int i = tid; i < looks; i += threads) {
      const int j = i - single, k = j / max(steps, 1);
      const int u = j < 0 ? s_unit[i] : u0 + s_thread[k] + (j - k * steps) * threads;
      if (u >= u1) continue;
      Unit<T> w;
      float v[kUnit];
      w.load(body + (int64_t)u * P);
      w.get(v);
      if (order_of(largest<kUnit>(v)) < bound_value) continue;
#pragma unroll
      for (int e = 0; e < kUnit; ++e)
        if (((uint64_t)order_of(v[e]) << 32 | (uint32_t)~u) >= bound) found(key_of(v[e], head + u * kUnit + e));
    }
    if (part != 0) {  // to the first CTA together: one trip for the place, one for the keys
      __syncthreads();
      const int n = s_found;
      const uint64_t* from = list;
      int give = n;
      if (n > kFew && n <= kCandidates) {  // the first `top` of them
        for (int i = tid; i < n; i += threads) {
          const uint64_t k = list[i];
          int rank = 0;
          for (int j = 0; j < n; ++j) rank += list[j] > k;
          if (rank < a.top) s_top[rank] = k;
        }
        from = s_top, give = a.top;
      }
      if (tid == 0) s_units = atomicAdd(&first->found, n > kCandidates ? kMostParts * kFew + 1 : give);
      __syncthreads();
      if (n <= kCandidates)
        for (int i = tid; i < give; i += threads) first->key[min(s_units + i, kMostParts * kFew - 1)] = from[i];
    }
  }
  meet();
  if (part != 0) return;

  // the first CTA has everything
  const int own = a.top ? s_found : 0, n = own + (a.top ? s_board.found : 0);
  if (own <= kCandidates && n - own <= kMostParts * kFew) {
    for (int i = tid; i < n; i += threads) {
      const uint64_t k = i < own ? list[i] : s_board.key[i - own];
      int rank = 0;
      for (int j = 0; j < own; ++j) rank += list[j] > k;
      for (int j = own; j < n; ++j) rank += s_board.key[j - own] > k;
      if (rank < a.top) s_top[rank] = k;
    }
  } else {  // many of a few threads' logits: one after another over the whole row
    uint64_t last = 0;
    for (int k = 0; k < a.top; ++k) {
      uint64_t best = 0;
      for (int64_t i = tid; i < a.vocab; i += threads) {
        const uint64_t c = key_of(to_f32(x[i]), (int)i);
        if (k == 0 || c < last) best = max(best, c);  // (no key is above a NaN's at index 0)
      }
      for (int o = 16; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(~0u, (unsigned long long)best, o));
      __syncthreads();
      if (lane == 0) s_board.key[warp] = best;
      __syncthreads();
      for (int w = 0; w < warps; ++w) best = max(best, s_board.key[w]);
      if (tid == 0) s_top[k] = best;
      last = best;
    }
  }
  if (warp == 0) {
    const int all = parts * warps;
    float m = -INFINITY;
    for (int i = lane; i < all; i += 32) m = fmaxf(m, s_board.record[i].sums.m);
    m = warp_max(m);
    Sums w{m, 0.f, 0.f, 0};
    int owners = 0, ahead = 0, odd = 0;  // owners: of places of m, one of which is left out
    for (int i = lane; i < all; i += 32) {
      Sums v = s_board.record[i].sums;
      ahead += s_board.record[i].ahead, odd |= s_board.record[i].odd;
      if (v.m == m)
        owners += v.own;
      else
        v.raise(m, v.own);
      w.s += v.s, w.t += v.t;
    }
    owners = __reduce_add_sync(~0u, owners), ahead = __reduce_add_sync(~0u, ahead);
    odd = __any_sync(~0u, odd);
    w.s = warp_sum(w.s) + (float)max(owners - 1, 0), w.t = warp_sum(w.t);
    if (lane == 0) s_all = Record{w, ahead, odd};
  }
  __syncthreads();
  const Sums w = s_all.sums;
  const bool bad = s_all.odd, none = w.m == -INFINITY;
  const float norm = log1pf(w.s), nan = __uint_as_float(0x7fffffffu);
  auto logprob = [&](float v) { return bad ? nan : none ? -INFINITY : (v - w.m) - norm; };
  if (tid == 0) {
    if (a.targets) {
      a.logprob[row] = known ? logprob(to_f32(mine)) : 0.f;
      a.rank[row] = known ? s_all.ahead + 1 : 0;
      if (given >= a.vocab && a.err_flag) *a.err_flag = 1;
    }
    a.entropy[row] = bad ? nan : none ? 0.f : norm - w.t / (1.f + w.s);
  }
  if (tid < a.top) {
    a.top_logprob[row * a.top + tid] = logprob(logit_of((uint32_t)(s_top[tid] >> 32)));
    a.top_index[row * a.top + tid] = ~(int)(uint32_t)s_top[tid];
  }
}

// CTAs of a row and threads of a CTA.  More than 128 threads have at least four units each (alone, one in a cluster),
// since a warp's start and end take as long as six steps (us; 700 rows of 4099: 8.7 with 128 threads, 11.4 with 256; 4000 of 32000: 128 with
// 256, 137 with 128, 157 with 512; 2048 of 151936: 164 with 512, 171 with 256).  Few rows take a cluster each, as long
// as that gives no SM a second CTA: clusters wait for one another's SMs (one row of 151936 floats: 17.1 alone, 14.3,
// 12.1 and 11.1 with 2, 4 and 8 CTAs; 64 rows: 21.2, 17.6, 18.7, 30.2).
struct Shape {
  int parts, threads;
};
Shape shape_of(const q4gpu_logprob_args& a) {
  const int64_t units = a.vocab / kUnit;
  Shape s{1, 64};
  while (s.threads < kMostThreads && units >= (s.threads < 128 ? 2 : 8) * s.threads) s.threads *= 2;
  while (s.parts < kMostParts && a.rows * s.parts * s.threads * 2 <= 148 * kMostThreads &&
         units / s.parts >= 2 * s.threads)
    s.parts *= 2;
  return s;
}

template <typename T>
int launch(const q4gpu_logprob_args& a, cudaStream_t stream) {
  const Shape s = shape_of(a);
  if (a.rows * s.parts > INT32_MAX) return q4gpu_fail(Q4GPU_ERR_SHAPE, "logprobs: too many rows");
  constexpr int kPerThread = kUnit * (int)sizeof(T) * Unit<T>::kStages;  // of the ring
  static unsigned char ready[Q4GPU_MAX_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < Q4GPU_MAX_DEVICES && ready[dev])) {  // once per device
    e = cudaFuncSetAttribute(token_logprobs_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kPerThread * kMostThreads);
    if (e == cudaSuccess && dev < Q4GPU_MAX_DEVICES) ready[dev] = 1;
  }
  if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "logprobs: attributes: %s", cudaGetErrorString(e));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = s.parts, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * s.parts)), cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = (size_t)kPerThread * s.threads;
  cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = s.parts > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a, s.parts);
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
