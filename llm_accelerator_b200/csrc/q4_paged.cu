// 16-bit paged serving operators: residual add + RMS norm (16- or 8-bit
// output), rotary positions with storage in a paged cache, and forking and
// compacting of the cache's pages.  Declared in include/q4gpu.h; attention is
// in q4_paged_attn.cu.
#include <cuda_fp8.h>

#include <cstdint>

#include "q4_paged.cuh"
#include "q4gpu_internal.h"

using namespace q4::paged;

namespace {

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// ---------------------------------------------------------------------------
// residual add + RMS norm
// ---------------------------------------------------------------------------
enum { kSame = 0, kE4m3 = 1, kS8 = 2 };

// V consecutive values as they are stored, fetched in as few accesses as V's
// bytes allow.
template <typename T, int V>
struct Raw {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void get(float* f) const { f[0] = to_f32(v); }
};
template <typename T>
struct Raw<T, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* f) const { unpack8<T>(v, f); }
};
template <>
struct Raw<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float* f) {
  if constexpr (sizeof(T) == 4 && V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    *reinterpret_cast<uint4*>(p) = pack8<T>(f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = from_f32<T>(f[i]);
  }
}
template <int OUT, int V>
__device__ __forceinline__ void store_8bit(uint8_t* p, const float* f, float inv) {
  auto s8 = [&](float v) {
    const int q = __float2int_rn(v * inv);
    return (uint32_t)(q < -127 ? -127 : (q > 127 ? 127 : q)) & 0xffu;
  };
  auto e4m3 = [&](float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
  };
  if constexpr (V == 8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      if constexpr (OUT == kE4m3)
        w[i / 4] = e4m3(f[i], f[i + 1]) | e4m3(f[i + 2], f[i + 3]) << 16;
      else
        w[i / 4] = s8(f[i]) | s8(f[i + 1]) << 8 | s8(f[i + 2]) << 16 | s8(f[i + 3]) << 24;
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    static_assert(V == 1, "single values or eight");
    if constexpr (OUT == kE4m3)
      *p = __nv_cvt_float_to_fp8(f[0] * inv, __NV_SATFINITE, __NV_E4M3);
    else
      *p = (uint8_t)s8(f[0]);
  }
}

struct NormParams {
  const void *x, *residual, *weight;
  void *out, *residual_out;
  float* scale;
  int64_t rows, xs, rs, os, ros;
  int n, group;
  float eps;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
// NaN if a lane has one; over spans of `n` lanes (a power of two).
__device__ __forceinline__ float span_max(float v, int n) {
  for (int o = n >> 1; o; o >>= 1) {
    const float u = __shfl_xor_sync(~0u, v, o);
    v = max3(v, u, u);
  }
  return v;
}

// Whether a thread's registers hold the next row's values and the weights too.
template <typename T, int V, int E>
__host__ __device__ constexpr bool norm_ahead() { return sizeof(T) == 2 && V == 8 && E <= 16; }

// One row per blockDim.x threads (a power of two from 32), blockDim.y rows at a
// time per CTA (1 unless a row is one warp).  A thread holds E values of its
// row, V consecutive ones at a time, so x and the residual are read once.  Where
// registers allow it (norm_ahead) CTAs stay and go from row to row: the next
// row's values are on their way while this one is summed, scaled and stored.
// Maxima pass NaNs on, so one reaches the scale.  8192 x 4096 bf16 with a
// residual into e4m3 moves 237 MB in 49.5 us, 4.8 TB/s; the SMs' busiest pipe is
// at 65 % and 27 of 64 warps are resident, so a row's chain of steps shows beside
// the memory.
template <typename T, int OUT, int V, int E>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(NormParams p) {
  constexpr int N = E / V;
  constexpr bool kAhead = norm_ahead<T, V, E>();
  const int tx = threadIdx.x, lanes = blockDim.x;
  __shared__ float part[2][32];  // by turns, so that one barrier a row is enough
  __shared__ float partm[32];
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const T* w = static_cast<const T*>(p.weight);
  Raw<T, V> xr[N], rr[N], wr[N];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int at = (c * lanes + tx) * V;
      if (at < p.n) {
        xr[c].load(x + row * p.xs + at);
        if (res) rr[c].load(res + row * p.rs + at);
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (kAhead && row < p.rows) fetch(row);
  if constexpr (kAhead) {
#pragma unroll
    for (int c = 0; c < N; ++c)
      if ((c * lanes + tx) * V < p.n) wr[c].load(w + (c * lanes + tx) * V);
  }
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    float h[E], ss = 0.f;
    if constexpr (!kAhead) fetch(row);
#pragma unroll
    for (int c = 0; c < N; ++c) {
#pragma unroll
      for (int i = 0; i < V; ++i) h[c * V + i] = 0.f;
      if ((c * lanes + tx) * V < p.n) {
        xr[c].get(h + c * V);
        if (res) {
          float r[V];
          rr[c].get(r);
#pragma unroll
          for (int i = 0; i < V; ++i) h[c * V + i] += r[i];
        }
      }
    }
    if (kAhead && row + step < p.rows) fetch(row + step);
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fmaf(h[i], h[i], ss);
    ss = warp_sum(ss);
    if (lanes > 32) {
      if ((tx & 31) == 0) part[turn][tx >> 5] = ss;
      __syncthreads();
      ss = warp_sum((tx & 31) < (lanes >> 5) ? part[turn][tx & 31] : 0.f);
    }
    const float inv = rsqrtf(ss / (float)p.n + p.eps);
    if (p.residual_out) {
      T* ro = static_cast<T*>(p.residual_out) + row * p.ros;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const int at = (c * lanes + tx) * V;
        if (at < p.n) store_v<T, V>(ro + at, h + c * V);
      }
    }
    float most[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      most[c] = 0.f;
      if ((c * lanes + tx) * V < p.n) {
        float g[V];
        if constexpr (!kAhead) wr[c].load(w + (c * lanes + tx) * V);
        wr[c].get(g);
#pragma unroll
        for (int i = 0; i < V; ++i) h[c * V + i] = h[c * V + i] * inv * g[i];
        if constexpr (OUT != kSame && V > 1) {
#pragma unroll
          for (int i = 0; i < V; i += 2) most[c] = max3(most[c], fabsf(h[c * V + i]), fabsf(h[c * V + i + 1]));
        } else if constexpr (OUT != kSame) {
          most[c] = fabsf(h[c]);
        }
      }
    }
    if constexpr (OUT == kSame) {
      T* o = static_cast<T*>(p.out) + row * p.os;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const int at = (c * lanes + tx) * V;
        if (at < p.n) store_v<T, V>(o + at, h + c * V);
      }
    } else {
      constexpr float kMost = OUT == kE4m3 ? 448.f : 127.f;
      uint8_t* o = static_cast<uint8_t*>(p.out) + row * p.os;
      // The factor of values v[0 .. n) whose largest is `top`.  A quarter of each side of the quotient: __fdividef gives
      // 0 for divisors above 2^126.  Tiny values are made larger first, or the factor would be infinite.
      auto factor = [&](float top, float* v, int n) {
        if (top < 0x1p-96f) {
          top *= 0x1p64f;
          for (int i = 0; i < n; ++i) v[i] *= 0x1p64f;
        }
        return top == 0.f ? 0.f : __fdividef(kMost * 0.25f, top * 0.25f);
      };
      if (p.group == 0) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < N; ++c) top = max3(top, most[c], most[c]);
        top = span_max(top, 32);
        if (lanes > 32) {
          if ((tx & 31) == 0) partm[tx >> 5] = top;
          __syncthreads();
          top = span_max((tx & 31) < (lanes >> 5) ? partm[tx & 31] : 0.f, 32);
        }
        if (tx == 0) p.scale[row] = top * (1.f / kMost);
        const float f = factor(top, h, E);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const int at = (c * lanes + tx) * V;
          if (at < p.n) store_8bit<OUT, V>(o + at, h + c * V, f);
        }
      } else if constexpr (V == 8) {
        // a group is group / 8 neighbouring lanes of one access
        const int span = p.group / 8, groups = p.n / p.group;
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const int at = (c * lanes + tx) * V;
          const float top = span_max(most[c], span);
          if (at < p.n) {
            if ((tx & (span - 1)) == 0) p.scale[row * groups + at / p.group] = top * (1.f / kMost);
            const float f = factor(top, h + c * V, V);
            store_8bit<OUT, V>(o + at, h + c * V, f);
          }
        }
      }
    }
    if constexpr (!kAhead) break;  // one row a CTA
  }
}

template <typename T, int OUT, int V>
void launch_norm_v(const NormParams& p, cudaStream_t s) {
  // A thread takes 8 values of its row where there are too few rows to fill the
  // GPU, else 16: two accesses of x and two of the residual in flight in each of
  // 1024 threads an SM (8192 x 4096 into e4m3: 70.8 us with 32 values a thread,
  // whose loads went one after the other to stay within 64 registers; 63.1 with
  // 16; 48.6 with 16 and the next row on its way).  32 only where a row is longer
  // than 1024 threads x 16.
  const int per = p.n > 16384 ? 32 : p.rows < 148 * 4 && p.n <= 8192 ? 8 : 16;
  int lanes = 32;
  while (lanes * per < p.n) lanes *= 2;
  const int ny = lanes == 32 ? 4 : 1;
  const dim3 block(lanes, ny);
  // rows at a time; with 64 registers a thread 1024 threads stay on each SM
  const int64_t all = (p.rows + ny - 1) / ny, some = 148 * (1024 / (lanes * ny));
  const bool stay = per <= 16 && norm_ahead<T, V, 16>();
  const unsigned grid = (unsigned)(stay ? std::min(all, some) : all);
  if (per == 8)
    add_rmsnorm_kernel<T, OUT, V, 8><<<grid, block, 0, s>>>(p);
  else if (per == 16)
    add_rmsnorm_kernel<T, OUT, V, 16><<<grid, block, 0, s>>>(p);
  else
    add_rmsnorm_kernel<T, OUT, V, 32><<<grid, block, 0, s>>>(p);
}
template <typename T, int OUT>
void launch_norm(const NormParams& p, bool vec, cudaStream_t s) {
  if (vec)
    launch_norm_v<T, OUT, 8>(p, s);
  else
    launch_norm_v<T, OUT, 1>(p, s);
}

template <typename T>
void launch_norm_out(const NormParams& p, int out_dtype, bool vec, cudaStream_t s) {
  if (out_dtype == Q4GPU_E4M3)
    launch_norm<T, kE4m3>(p, vec, s);
  else if (out_dtype == Q4GPU_S8)
    launch_norm<T, kS8>(p, vec, s);
  else
    launch_norm<T, kSame>(p, vec, s);
}

// ---------------------------------------------------------------------------
// rotary positions + storage in the paged cache
// ---------------------------------------------------------------------------
// A head vector is cut into units of 16 values: a rotated unit is 8 pairs (8
// values and their 8 partners, or 16 neighbours where pairs are interleaved),
// the rest are plain.  `lanes` threads (a power of two) share a head vector,
// one unit each, and a thread takes its unit of VECS head vectors of one token
// (heads s, s + slots, ..), so the token's cosines and sines are fetched once
// for all of them and 32 VECS bytes of data are in flight per thread.  Bound by
// memory, and by the way from a token's position to its table row: 8192 tokens of
// 16 + 8 + 8 heads of 128, normed, take 34.4 us (4.0 TB/s; a plain copy of the same
// bytes 24.8).
template <typename T, bool INTERLEAVED, int VECS>
__global__ void __launch_bounds__(256, VECS == 1 ? 5 : 4)
    rope_append_kernel(q4gpu_rope_args a, int lanes, int heads, int slots) {
  const uint32_t flat = blockIdx.x * blockDim.x + threadIdx.x;
  const int u = flat & (lanes - 1);
  const uint32_t group = flat / lanes, token = group / (uint32_t)slots, slot = group - token * slots;
  const bool there = token < (uint32_t)a.tokens;
  const int nq = a.q ? a.q_heads : 0, nk = a.k ? a.kv_heads : 0;
  const int turned = a.rot_dim / 16;
  int at0, at1;
  if (u < turned) {
    at0 = INTERLEAVED ? 16 * u : 8 * u;
    at1 = INTERLEAVED ? at0 + 8 : a.rot_dim / 2 + 8 * u;
  } else {
    at0 = 16 * u;
    at1 = at0 + 8;
  }
  const bool has0 = there && at0 < a.dim, has1 = there && at1 < a.dim;

  const int64_t row = there && a.rows ? a.rows[token] : -1;
  const int pos = there && a.positions ? a.positions[token] : 0;
  uint4 raw[VECS][2];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    int head = slot + i * slots;
    raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (head >= heads) continue;
    const T* src;
    if (head < nq)
      src = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
    else if ((head -= nq) < nk)
      src = static_cast<const T*>(a.k) + token * a.k_token_stride + head * a.k_head_stride;
    else
      src = static_cast<const T*>(a.v) + token * a.v_token_stride + (head - nk) * a.v_head_stride;
    if (has0) raw[i][0] = *reinterpret_cast<const uint4*>(src + at0);
    if (has1) raw[i][1] = *reinterpret_cast<const uint4*>(src + at1);
  }

  bool known = true;  // the position has a table row
  float cs[8], sn[8];
  if (there && turned && nq + nk > 0) {
    known = pos >= 0 && pos < a.table_positions;
    if (known && u < turned) {
      Raw<float, 8> w;
      w.load(a.cos + (int64_t)pos * (a.rot_dim / 2) + 8 * u);
      w.get(cs);
      w.load(a.sin + (int64_t)pos * (a.rot_dim / 2) + 8 * u);
      w.get(sn);
    }
  }
  // (tested at each store instead, an unknown position costs 8192 tokens 38.8 us, not 34.4)
  bool stored = row >= 0 && row < a.n_rows;
  if (there && (!known || row >= a.n_rows)) {
    stored = false;
    if (a.err_flag) *a.err_flag = 1;
  }
  // (a 32-bit division where the row allows it)
  const int64_t page = !stored     ? 0
                       : row >> 32 ? row / a.page_tokens
                                   : (int64_t)((uint32_t)row / (uint32_t)a.page_tokens);
  const int64_t cache = page * a.page_stride + (row - page * a.page_tokens) * a.row_stride;

#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    int head = slot + i * slots;
    const bool is_q = head < nq, is_k = !is_q && head < nq + nk;
    const T* gamma = static_cast<const T*>(is_q ? a.q_gamma : is_k ? a.k_gamma : nullptr);
    float f[16];
    unpack8<T>(raw[i][0], f);
    unpack8<T>(raw[i][1], f + 8);
    if (a.q_gamma || a.k_gamma) {
      float ss = 0.f;
#pragma unroll
      for (int x = 0; x < 16; ++x) ss = fmaf(f[x], f[x], ss);
      for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
      if (gamma) {
        const float inv = rsqrtf(ss / (float)a.dim + a.eps);
        float g[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) g[x] = 0.f;
        if (has0) unpack8<T>(*reinterpret_cast<const uint4*>(gamma + at0), g);
        if (has1) unpack8<T>(*reinterpret_cast<const uint4*>(gamma + at1), g + 8);
#pragma unroll
        for (int x = 0; x < 16; ++x) f[x] = f[x] * inv * g[x];
      }
    }
    T* dst;
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + token * a.q_out_token_stride + head * a.q_out_head_stride;
    } else {
      head -= nq + (is_k ? 0 : nk);
      dst = static_cast<T*>(is_k ? a.k_cache : a.v_cache) + cache + head * a.head_stride;
    }
    if (slot + i * slots >= heads || (!is_q && !stored) || ((is_q || is_k) && !known)) continue;
    if ((is_q || is_k) && u < turned) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const int x = INTERLEAVED ? 2 * p : p, y = INTERLEAVED ? 2 * p + 1 : p + 8;
        const float v = f[x], w = f[y];
        f[x] = v * cs[p] - w * sn[p];
        f[y] = w * cs[p] + v * sn[p];
      }
    }
    if (has0) *reinterpret_cast<uint4*>(dst + at0) = pack8<T>(f);
    if (has1) *reinterpret_cast<uint4*>(dst + at1) = pack8<T>(f + 8);
  }
}

template <typename T, bool INTERLEAVED>
void launch_rope(const q4gpu_rope_args& a, int lanes, int heads, cudaStream_t s) {
  // Two head vectors a thread once that still gives every SM 1024 threads; one
  // where latency counts (8192 tokens: 36.3 us with one, 34.4 with two at 64
  // registers, 38.0 with four at 99).
  const bool many = (int64_t)a.tokens * heads * lanes >= (int64_t)2 * 148 * 1024;
  const int slots = many ? (heads + 1) / 2 : heads;
  const int64_t threads = (int64_t)a.tokens * slots * lanes;
  const int block = (int)std::min<int64_t>(256, (threads + 31) / 32 * 32);
  const unsigned grid = (unsigned)((threads + block - 1) / block);
  if (many)
    rope_append_kernel<T, INTERLEAVED, 2><<<grid, block, 0, s>>>(a, lanes, heads, slots);
  else
    rope_append_kernel<T, INTERLEAVED, 1><<<grid, block, 0, s>>>(a, lanes, heads, slots);
}

// ---------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------
// A CTA's copy of n 16-byte words, eight loads of a thread in flight.
__device__ __forceinline__ void copy16(uint4* d, const uint4* s, int n) {
  constexpr int kFlight = 8;
  for (int i = threadIdx.x; i < n; i += kFlight * blockDim.x) {
    uint4 v[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i + k * (int)blockDim.x < n) v[k] = s[i + k * blockDim.x];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i + k * (int)blockDim.x < n) d[i + k * blockDim.x] = v[k];
  }
}

// Tokens that slot s holds, inside what its table row can name.
__device__ __forceinline__ int64_t held(const q4gpu_pages_args& a, int64_t s) {
  const int64_t most = a.table_stride * a.page_tokens, n = a.lens[s];
  return n < 0 ? 0 : (n < most ? n : most);
}
__device__ __forceinline__ bool fits(const q4gpu_pages_args& a, int64_t s) { return a.lens[s] == held(a, s); }

// blockIdx.y = fork, blockIdx.x strides over the page's blocks.  Only filled rows
// are copied; forks of one parent read it from L2.  48 forks of 12 prompts
// write 111 MB in 30 us; half of a warp's time between instructions is the wait for
// its loads.
__global__ void __launch_bounds__(128) pages_fork_kernel(q4gpu_pages_args a, const int32_t* parents,
                                                         const int32_t* children, const int32_t* fresh) {
  const int i = blockIdx.y;
  const int par = parents[i], chi = children[i];
  const bool first = blockIdx.x == 0;
  bool ok = par >= 0 && par < a.n_slots && chi >= 0 && chi < a.n_slots && par != chi;
  int64_t n = 0;
  int part = 0, source = 0, to = 0;
  int64_t last = -1;
  ok = ok && fits(a, par);
  if (ok) {
    n = held(a, par);
    part = (int)(n % a.page_tokens);
    last = (n + a.page_tokens - 1) / a.page_tokens - 1;
    if (part) {
      source = a.table[par * a.table_stride + last];
      to = fresh[i];
      ok = source >= 0 && source < a.n_pages && to >= 0 && to < a.n_pages && source != to;
    }
  }
  if (!ok) {
    if (first && threadIdx.x == 0 && a.err_flag) *a.err_flag = 1;
    return;
  }
  if (first) {
    const int32_t* from = a.table + par * a.table_stride;
    int32_t* row = a.table + chi * a.table_stride;
    for (int64_t c = threadIdx.x; c < a.table_stride; c += blockDim.x)
      row[c] = c > last ? -1 : (c == last && part ? to : from[c]);
    if (threadIdx.x == 0) a.lens[chi] = (int32_t)n;
  }
  if (!part) return;
  const int vecs = (int)(a.block_bytes / a.page_tokens * part / 16);
  const char* s = static_cast<const char*>(a.pool) + source * a.page_bytes;
  char* d = static_cast<char*>(a.pool) + to * a.page_bytes;
  const int64_t blocks = a.page_bytes / a.block_bytes;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x)
    copy16(reinterpret_cast<uint4*>(d + b * a.block_bytes), reinterpret_cast<const uint4*>(s + b * a.block_bytes),
           vecs);
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWords = 4096;  // bit words in shared memory: pools up to 131,072 pages

// One CTA: marks the pages in use, counts them, and pairs each used page past
// the packed end with an unused one below it (in order, so the result does not
// depend on timing).  moves = {source, destination} pairs, *n_moves of them.
__global__ void __launch_bounds__(kPlanThreads) pages_plan_kernel(q4gpu_pages_args a, int32_t* remap, int32_t* n_live,
                                                                  uint32_t* ws_bits, int32_t* ws_below,
                                                                  int32_t* n_moves, int2* moves) {
  __shared__ uint32_t s_bits[kPlanWords];
  __shared__ int32_t s_below[kPlanWords];  // used pages below a word
  __shared__ int s_warp[kPlanThreads / 32];
  __shared__ int s_before;
  const int t = threadIdx.x;
  const int words = (a.n_pages + 31) / 32;
  const bool small = words <= kPlanWords;
  uint32_t* bits = small ? s_bits : ws_bits;
  // global words were changed by atomics, which pass L1 by
  auto word = [&](int w) { return small ? s_bits[w] : __ldcg(ws_bits + w); };
  for (int w = t; w < words; w += kPlanThreads) bits[w] = 0u;
  __syncthreads();
  for (int s = t >> 5; s < a.n_slots; s += kPlanThreads / 32) {
    const int64_t used = (held(a, s) + a.page_tokens - 1) / a.page_tokens;
    if (a.err_flag && !fits(a, s)) *a.err_flag = 1;
    for (int64_t c = t & 31; c < used; c += 32) {
      const int id = a.table[s * a.table_stride + c];
      if (id >= 0 && id < a.n_pages)
        atomicOr(&bits[id >> 5], 1u << (id & 31));
      else if (a.err_flag)
        *a.err_flag = 1;
    }
  }
  __syncthreads();
  // each thread owns a run of words; `before` = used pages below its run
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int lo = min(words, t * per), hi = min(words, lo + per);
  int mine = 0;
  for (int w = lo; w < hi; ++w) mine += __popc(word(w));
  int run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, run, o);
    if ((t & 31) >= o) run += v;
  }
  if ((t & 31) == 31) s_warp[t >> 5] = run;
  __syncthreads();
  const int wv = s_warp[t & 31];
  int wrun = wv;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, wrun, o);
    if ((t & 31) >= o) wrun += v;
  }
  const int total = __shfl_sync(~0u, wrun, 31);
  const int warps_before = __shfl_sync(~0u, wrun - wv, t >> 5);
  const int before = warps_before + run - mine;
  // used pages below page number `total` (the packed end)
  if (t == 0) s_before = total;
  __syncthreads();
  {
    const int w = total >> 5;
    if (w >= lo && w < hi) {
      int c = before;
      for (int k = lo; k < w; ++k) c += __popc(word(k));
      s_before = c + __popc(word(w) & ((1u << (total & 31)) - 1u));
    }
  }
  __syncthreads();
  const int low = s_before;
  if (t == 0) {
    *n_live = total;
    *n_moves = total - low;
  }
  int below = before;
  for (int w = lo; w < hi; ++w) {
    (small ? s_below : ws_below)[w] = below;
    below += __popc(word(w));
  }
  __syncthreads();
  for (int page = t; page < a.n_pages; page += kPlanThreads) {
    const int w = page >> 5, k = page & 31;
    const uint32_t b = word(w);
    const bool live = (b >> k) & 1u;
    const int used = (small ? s_below[w] : __ldcg(ws_below + w)) + __popc(b & ((1u << k) - 1u));
    remap[page] = live ? page : -1;
    if (live && page >= total) moves[used - low].x = page;
    if (!live && page < total) moves[page - used].y = page;
  }
  __syncthreads();
  for (int i = t; i < total - low; i += kPlanThreads) remap[moves[i].x] = moves[i].y;
}

constexpr int64_t kMoveBytes = 1 << 16;  // a work item of the page copy

// Copies `count` moved pages, kMoveBytes at a time, all CTAs together.
template <typename Move>
__device__ __forceinline__ void move_pages(const q4gpu_pages_args& a, int count, Move move) {
  const int64_t per = (a.page_bytes + kMoveBytes - 1) / kMoveBytes, items = (int64_t)count * per;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int64_t m = i / per, off = (i - m * per) * kMoveBytes;
    const int2 mv = move((int)m);
    const int64_t bytes = min(kMoveBytes, a.page_bytes - off);
    copy16(reinterpret_cast<uint4*>(static_cast<char*>(a.pool) + mv.y * a.page_bytes + off),
           reinterpret_cast<const uint4*>(static_cast<const char*>(a.pool) + mv.x * a.page_bytes + off),
           (int)(bytes / 16));
  }
}

// Renumbers the tables and copies the moved pages, kMoveBytes at a time.
// Sources lie at or past the packed end and destinations below it, so no copy
// reads what another writes.  Bound by memory: 0.55 GB of pages move in 176 to
// 192 us, 6.2 to 5.7 TB/s read and written.
__global__ void __launch_bounds__(512) pages_move_kernel(q4gpu_pages_args a, int32_t* new_table, const int32_t* remap,
                                                         const int32_t* n_moves, const int2* moves) {
  const int64_t entries = (int64_t)a.n_slots * a.table_stride;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t s = e / a.table_stride, c = e - s * a.table_stride;
    const int id = a.table[e];
    new_table[e] = c * a.page_tokens < held(a, s) && id >= 0 && id < a.n_pages ? remap[id] : -1;
  }
  move_pages(a, *n_moves, [&](int m) { return moves[m]; });
}

constexpr int kOnePages = 2048;     // pools of one launch
constexpr int kOneEntries = 32768;  // and their tables

// The same plan and moves in one launch for a small pool whose tables go to new
// memory: every CTA makes the plan for itself, so none waits for another.
__global__ void __launch_bounds__(512) pages_compact_kernel(q4gpu_pages_args a, int32_t* new_table, int32_t* remap,
                                                            int32_t* n_live) {
  __shared__ uint32_t s_bits[kOnePages / 32];
  __shared__ int s_below[kOnePages / 32], s_total, s_src[kOnePages / 2], s_dst[kOnePages / 2];
  const int t = threadIdx.x, lane = t & 31;
  if (t < kOnePages / 32) s_bits[t] = 0u;
  __syncthreads();
  for (int s = t >> 5; s < a.n_slots; s += blockDim.x / 32) {
    const int64_t used = (held(a, s) + a.page_tokens - 1) / a.page_tokens;
    if (a.err_flag && !fits(a, s)) *a.err_flag = 1;
    for (int64_t c = lane; c < used; c += 32) {
      const int id = a.table[s * a.table_stride + c];
      if (id >= 0 && id < a.n_pages)
        atomicOr(&s_bits[id >> 5], 1u << (id & 31));
      else if (a.err_flag)
        *a.err_flag = 1;
    }
  }
  __syncthreads();
  if (t < 32) {
    int before = 0;
    for (int w = lane; w < kOnePages / 32; w += 32) {
      const int n = __popc(s_bits[w]);
      int run = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, run, o);
        if (lane >= o) run += v;
      }
      s_below[w] = before + run - n;
      before += __shfl_sync(~0u, run, 31);
    }
    if (lane == 0) s_total = before;
  }
  __syncthreads();
  const int total = s_total;
  auto live = [&](int page) { return (s_bits[page >> 5] >> (page & 31)) & 1u; };
  auto used_below = [&](int page) {
    return s_below[page >> 5] + __popc(s_bits[page >> 5] & ((1u << (page & 31)) - 1u));
  };
  const int low = total < a.n_pages ? used_below(total) : total, moves = total - low;
  for (int page = t; page < a.n_pages; page += blockDim.x) {
    if (live(page) && page >= total) s_src[used_below(page) - low] = page;
    if (!live(page) && page < total) s_dst[page - used_below(page)] = page;
  }
  __syncthreads();
  auto renumbered = [&](int page) { return page < total ? page : s_dst[used_below(page) - low]; };
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + t, step = (int64_t)gridDim.x * blockDim.x;
  if (first == 0) *n_live = total;
  for (int64_t page = first; page < a.n_pages; page += step)
    remap[page] = live((int)page) ? renumbered((int)page) : -1;
  for (int64_t e = first; e < (int64_t)a.n_slots * a.table_stride; e += step) {
    const int64_t s = e / a.table_stride, c = e - s * a.table_stride;
    const int id = a.table[e];
    new_table[e] = c * a.page_tokens < held(a, s) && id >= 0 && id < a.n_pages ? renumbered(id) : -1;
  }
  move_pages(a, moves, [&](int m) { return make_int2(s_src[m], s_dst[m]); });
}

int check_pages(const q4gpu_pages_args* a) {
  if (!a || !a->pool || !a->table || !a->lens) return q4gpu_fail(Q4GPU_ERR_ARG, "pages: null pointer");
  if (a->n_pages < 1 || a->page_tokens < 1 || a->n_slots < 1 || a->table_stride < 1 || a->block_bytes < 1 ||
      a->page_bytes < 1)
    return q4gpu_fail(Q4GPU_ERR_ARG, "pages: n_pages, page_tokens, n_slots, table_stride and sizes must be positive");
  if (a->page_bytes % a->block_bytes || a->block_bytes % a->page_tokens)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "pages: a page is whole blocks and a block page_tokens equal rows");
  if (a->block_bytes > INT32_MAX) return q4gpu_fail(Q4GPU_ERR_SHAPE, "pages: a block is at most 2 GiB");
  if (!aligned(a->pool, 16) || (a->block_bytes / a->page_tokens) % 16)
    return q4gpu_fail(Q4GPU_ERR_ALIGN, "pages: the pool and its rows are multiples of 16 bytes");
  return Q4GPU_OK;
}

}  // namespace

extern "C" {

int q4gpu_add_rmsnorm(const q4gpu_norm_args* a, void* stream) {
  if (!a || !a->weight || (a->rows != 0 && (!a->x || !a->out)))
    return q4gpu_fail(Q4GPU_ERR_ARG, "norm: null pointer");
  if (a->rows < 0 || a->n < 1 || a->n > Q4GPU_NORM_MAX_N)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "norm: n = %d outside 1..%d", a->n, Q4GPU_NORM_MAX_N);
  if (a->rows > INT32_MAX) return q4gpu_fail(Q4GPU_ERR_SHAPE, "norm: too many rows");
  if (a->dtype < Q4GPU_F32 || a->dtype > Q4GPU_BF16)
    return q4gpu_fail(Q4GPU_ERR_ARG, "norm: dtype is F32, F16 or BF16");
  const bool narrow = a->out_dtype == Q4GPU_E4M3 || a->out_dtype == Q4GPU_S8;
  if (!narrow && a->out_dtype != a->dtype) return q4gpu_fail(Q4GPU_ERR_ARG, "norm: out_dtype is dtype, E4M3 or S8");
  if (narrow && !a->scale && a->rows != 0) return q4gpu_fail(Q4GPU_ERR_ARG, "norm: an 8-bit output needs its scales");
  if (a->group && (!narrow || a->group < 8 || a->group > 256 || (a->group & (a->group - 1)) || a->n % a->group))
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "norm: group = %d is not 0 or a power of two 8..256 dividing n, 8-bit only",
                      a->group);
  if (a->rows == 0) return Q4GPU_OK;
  const int64_t es = a->dtype == Q4GPU_F32 ? 4 : 2, oes = narrow ? 1 : es;
  const bool vec = a->n % 8 == 0 && aligned(a->x, 16) && aligned(a->weight, 16) && a->x_stride * es % 16 == 0 &&
                   (!a->residual || (aligned(a->residual, 16) && a->residual_stride * es % 16 == 0)) &&
                   (!a->residual_out || (aligned(a->residual_out, 16) && a->residual_out_stride * es % 16 == 0)) &&
                   aligned(a->out, narrow ? 8 : 16) && a->out_stride * oes % (narrow ? 8 : 16) == 0;
  if (a->group && !vec) return q4gpu_fail(Q4GPU_ERR_ALIGN, "norm: grouped 8-bit output needs 16-byte aligned rows");
  NormParams p{a->x,        a->residual,        a->weight,     a->out,
               a->residual_out, a->scale,       a->rows,       a->x_stride,
               a->residual_stride, a->out_stride, a->residual_out_stride, a->n,
               a->group,    a->eps};
  cudaStream_t s = as_stream(stream);
  if (a->dtype == Q4GPU_F32)
    launch_norm_out<float>(p, a->out_dtype, vec, s);
  else if (a->dtype == Q4GPU_F16)
    launch_norm_out<__half>(p, a->out_dtype, vec, s);
  else
    launch_norm_out<__nv_bfloat16>(p, a->out_dtype, vec, s);
  return q4gpu_check_launch();
}

int q4gpu_rope_append(const q4gpu_rope_args* a, void* stream) {
  if (!a) return q4gpu_fail(Q4GPU_ERR_ARG, "rope: null arguments");
  if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 0) return q4gpu_fail(Q4GPU_ERR_ARG, "rope: negative size");
  if (a->q_heads > 65535 || a->kv_heads > 65535) return q4gpu_fail(Q4GPU_ERR_SHAPE, "rope: too many heads");
  if (a->tokens == 0) return Q4GPU_OK;
  const bool turns = (a->q || a->k) && a->rot_dim > 0, stores = a->k || a->v;
  if ((!a->q && !stores) || (a->q && !a->q_out) || (a->k && !a->k_cache) || (a->v && !a->v_cache) ||
      (turns && (!a->cos || !a->sin || !a->positions)) || (stores && !a->rows))
    return q4gpu_fail(Q4GPU_ERR_ARG, "rope: null pointer");
  if (a->dtype != Q4GPU_F16 && a->dtype != Q4GPU_BF16) return q4gpu_fail(Q4GPU_ERR_ARG, "rope: dtype is F16 or BF16");
  if (a->dim < 8 || a->dim > 512 || a->dim % 8) return q4gpu_fail(Q4GPU_ERR_SHAPE, "rope: dim = %d", a->dim);
  if (a->rot_dim < 0 || a->rot_dim > a->dim || a->rot_dim % 16)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "rope: rot_dim = %d is not a multiple of 16 up to dim", a->rot_dim);
  if (turns && a->table_positions < 1) return q4gpu_fail(Q4GPU_ERR_ARG, "rope: empty cos / sin tables");
  if (stores && (a->page_tokens < 1 || a->n_rows < 0)) return q4gpu_fail(Q4GPU_ERR_ARG, "rope: bad cache size");
  auto ok = [](const void* p, int64_t ts, int64_t hs) { return !p || (aligned(p, 16) && ts % 8 == 0 && hs % 8 == 0); };
  if (!ok(a->q, a->q_token_stride, a->q_head_stride) || !ok(a->k, a->k_token_stride, a->k_head_stride) ||
      !ok(a->v, a->v_token_stride, a->v_head_stride) ||
      !ok(a->q ? a->q_out : nullptr, a->q_out_token_stride, a->q_out_head_stride) ||
      !ok(a->k ? a->k_cache : nullptr, a->page_stride, a->head_stride) ||
      !ok(a->v ? a->v_cache : nullptr, a->page_stride, a->head_stride) || (stores && a->row_stride % 8) ||
      !ok(a->q_gamma, 0, 0) || !ok(a->k_gamma, 0, 0) || (turns && (!aligned(a->cos, 16) || !aligned(a->sin, 16))))
    return q4gpu_fail(Q4GPU_ERR_ALIGN, "rope: head vectors and tables start on 16-byte boundaries");
  const int heads = (a->q ? a->q_heads : 0) + (a->k ? a->kv_heads : 0) + (a->v ? a->kv_heads : 0);
  if (heads == 0) return Q4GPU_OK;
  const int units = a->rot_dim / 16 + (a->dim - a->rot_dim + 15) / 16;
  int lanes = 1;
  while (lanes < units) lanes *= 2;
  if ((int64_t)a->tokens * heads * lanes > INT32_MAX) return q4gpu_fail(Q4GPU_ERR_SHAPE, "rope: too many tokens");
  cudaStream_t s = as_stream(stream);
  if (a->dtype == Q4GPU_F16) {
    if (a->interleaved)
      launch_rope<__half, true>(*a, lanes, heads, s);
    else
      launch_rope<__half, false>(*a, lanes, heads, s);
  } else {
    if (a->interleaved)
      launch_rope<__nv_bfloat16, true>(*a, lanes, heads, s);
    else
      launch_rope<__nv_bfloat16, false>(*a, lanes, heads, s);
  }
  return q4gpu_check_launch();
}

int q4gpu_pages_fork(const q4gpu_pages_args* a, const int32_t* parents, const int32_t* children, const int32_t* fresh,
                     int32_t n, void* stream) {
  const int rc = check_pages(a);
  if (rc != Q4GPU_OK) return rc;
  if (n < 0 || n > 65535) return q4gpu_fail(Q4GPU_ERR_ARG, "pages: n = %d forks outside 0..65535", n);
  if (n == 0) return Q4GPU_OK;
  if (!parents || !children || !fresh) return q4gpu_fail(Q4GPU_ERR_ARG, "pages: null pointer");
  const int64_t blocks = a->page_bytes / a->block_bytes;
  const unsigned x = (unsigned)std::min<int64_t>(blocks, std::max(1, 148 * 64 / n));
  pages_fork_kernel<<<dim3(x, n), 128, 0, as_stream(stream)>>>(*a, parents, children, fresh);
  return q4gpu_check_launch();
}

// workspace: {count, padding}, moves, bit words, used pages below each word
size_t q4gpu_pages_compact_workspace_bytes(int32_t n_pages) {
  if (n_pages < 1) return 0;
  const size_t moves = ((size_t)n_pages * sizeof(int2) + 15) / 16 * 16;
  return 16 + moves + ((size_t)n_pages + 31) / 32 * 8;
}

int q4gpu_pages_compact(const q4gpu_pages_args* a, int32_t* new_table, int32_t* remap, int32_t* n_live,
                        void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_pages(a);
  if (rc != Q4GPU_OK) return rc;
  if (!new_table || !remap || !n_live || !workspace) return q4gpu_fail(Q4GPU_ERR_ARG, "pages: null pointer");
  if (workspace_bytes < q4gpu_pages_compact_workspace_bytes(a->n_pages))
    return q4gpu_fail(Q4GPU_ERR_WORKSPACE, "pages: workspace of %zu bytes is too small", workspace_bytes);
  if (!aligned(workspace, 16)) return q4gpu_fail(Q4GPU_ERR_ALIGN, "pages: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  const size_t moves_bytes = ((size_t)a->n_pages * sizeof(int2) + 15) / 16 * 16;
  int32_t* count = reinterpret_cast<int32_t*>(ws);
  int2* moves = reinterpret_cast<int2*>(ws + 16);
  uint32_t* bits = reinterpret_cast<uint32_t*>(ws + 16 + moves_bytes);
  int32_t* below = reinterpret_cast<int32_t*>(bits + ((size_t)a->n_pages + 31) / 32);
  cudaStream_t s = as_stream(stream);
  // One launch where each CTA's own plan is short and nothing is read that another CTA changes: 96 small pages
  // take 5.5 us on the device and 8.8 us a call in two launches, 5.7 us a call in one.
  if (new_table != a->table && a->n_pages <= kOnePages && (int64_t)a->n_slots * a->table_stride <= kOneEntries) {
    const int64_t items = (a->page_bytes + kMoveBytes - 1) / kMoveBytes * ((a->n_pages + 1) / 2);
    pages_compact_kernel<<<(unsigned)std::min<int64_t>(148 * 4, items), 512, 0, s>>>(*a, new_table, remap, n_live);
    return q4gpu_check_launch();
  }
  pages_plan_kernel<<<1, kPlanThreads, 0, s>>>(*a, remap, n_live, bits, below, count, moves);
  pages_move_kernel<<<148 * 4, 512, 0, s>>>(*a, new_table, remap, count, moves);
  return q4gpu_check_launch();
}

}  // extern "C"
