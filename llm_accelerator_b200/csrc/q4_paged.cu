// 16-bit paged serving operators: residual add + RMS norm (16- or 8-bit
// output), rotary positions with storage in a paged cache, and forking and
// compacting of the cache's pages.  Declared in include/q4gpu.h; attention is
// in q4_paged_attn.cu.
#include <cuda_fp8.h>

#include <cfloat>
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

// V consecutive values at p as floats, in as few accesses as V's bytes allow.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float* f) {
  if constexpr (sizeof(T) == 4 && V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 w = *reinterpret_cast<const float4*>(p + i);
      f[i] = w.x, f[i + 1] = w.y, f[i + 2] = w.z, f[i + 3] = w.w;
    }
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(p[i]);
  }
}
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
  uint32_t w[(V + 3) / 4];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    uint32_t b;
    if constexpr (OUT == kE4m3) {
      b = __nv_cvt_float_to_fp8(f[i] * inv, __NV_SATFINITE, __NV_E4M3);
    } else {
      const int q = __float2int_rn(f[i] * inv);
      b = (uint32_t)(q < -127 ? -127 : (q > 127 ? 127 : q)) & 0xffu;
    }
    w[i / 4] = (i % 4 ? w[i / 4] : 0u) | (b << (8 * (i % 4)));
  }
  if constexpr (V == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
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
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(~0u, v); }

// One row per blockDim.x threads (a power of two from 32), blockDim.y rows per
// CTA (1 unless a row is one warp).  A thread holds E values of its row, V
// consecutive ones at a time, so x and the residual are read once.  Magnitudes
// are compared as the bits of |y|: a NaN is above everything and reaches the
// scale.
template <typename T, int OUT, int V, int E>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(NormParams p) {
  constexpr int N = E / V;
  const int tx = threadIdx.x, lanes = blockDim.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  __shared__ float part[32];
  __shared__ uint32_t partm[32];
  if (row >= p.rows) return;  // only where a row is one warp
  const T* x = static_cast<const T*>(p.x) + row * p.xs;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.rs : nullptr;
  const T* w = static_cast<const T*>(p.weight);
  float h[E];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const int at = (c * lanes + tx) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) h[c * V + i] = 0.f;
    if (at < p.n) {
      load_v<T, V>(x + at, h + c * V);
      if (res) {
        float r[V];
        load_v<T, V>(res + at, r);
#pragma unroll
        for (int i = 0; i < V; ++i) h[c * V + i] += r[i];
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) ss = fmaf(h[i], h[i], ss);
  ss = warp_sum(ss);
  if (lanes > 32) {
    if ((tx & 31) == 0) part[tx >> 5] = ss;
    __syncthreads();
    ss = warp_sum((tx & 31) < (lanes >> 5) ? part[tx & 31] : 0.f);
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
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const int at = (c * lanes + tx) * V;
    if (at < p.n) {
      float g[V];
      load_v<T, V>(w + at, g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[c * V + i] = h[c * V + i] * inv * g[i];
        if constexpr (OUT != kSame) most = max(most, __float_as_uint(h[c * V + i]) & 0x7fffffffu);
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
    if (p.group == 0) {
      most = warp_max(most);
      if (lanes > 32) {
        if ((tx & 31) == 0) partm[tx >> 5] = most;
        __syncthreads();
        most = warp_max((tx & 31) < (lanes >> 5) ? partm[tx & 31] : 0u);
      }
      const float top = __uint_as_float(most);
      // a subnormal maximum would give an infinite factor
      const float f = most ? fminf(__fdiv_rn(kMost, top), FLT_MAX) : 0.f;
      if (tx == 0) p.scale[row] = __fdiv_rn(top, kMost);
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
        uint32_t m = 0;
        const int at = (c * lanes + tx) * V;
        if (at < p.n) {
#pragma unroll
          for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(h[c * V + i]) & 0x7fffffffu);
        }
        for (int o2 = span >> 1; o2; o2 >>= 1) m = max(m, __shfl_xor_sync(~0u, m, o2));
        if (at < p.n) {
          const float top = __uint_as_float(m);
          const float f = m ? fminf(__fdiv_rn(kMost, top), FLT_MAX) : 0.f;
          if ((tx & (span - 1)) == 0) p.scale[row * groups + at / p.group] = __fdiv_rn(top, kMost);
          store_8bit<OUT, V>(o + at, h + c * V, f);
        }
      }
    }
  }
}

template <typename T, int OUT>
void launch_norm(const NormParams& p, bool vec, cudaStream_t s) {
  // A thread takes 8 values where that already gives a row enough threads
  // and there are too few rows to fill the GPU, else 32.
  const bool few = p.rows < 148 * 4 && p.n <= 8192;
  const int per = few ? 8 : 32;
  int lanes = 32;
  while (lanes * per < p.n) lanes *= 2;
  const int ny = lanes == 32 ? 4 : 1;
  const dim3 block(lanes, ny);
  const unsigned grid = (unsigned)((p.rows + ny - 1) / ny);
  if (vec) {
    if (few)
      add_rmsnorm_kernel<T, OUT, 8, 8><<<grid, block, 0, s>>>(p);
    else
      add_rmsnorm_kernel<T, OUT, 8, 32><<<grid, block, 0, s>>>(p);
  } else {
    if (few)
      add_rmsnorm_kernel<T, OUT, 1, 8><<<grid, block, 0, s>>>(p);
    else
      add_rmsnorm_kernel<T, OUT, 1, 32><<<grid, block, 0, s>>>(p);
  }
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
// one unit each.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_append_kernel(q4gpu_rope_args a, int lanes, int heads) {
  const int64_t flat = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int u = (int)(flat & (lanes - 1));
  const int64_t vec = flat / lanes;
  const int64_t token = vec / heads;
  int head = (int)(vec - token * heads);
  const bool there = token < a.tokens;
  const int nq = a.q ? a.q_heads : 0, nk = a.k ? a.kv_heads : 0;
  const T* src = nullptr;
  T* dst = nullptr;
  const T* gamma = nullptr;
  bool rotate = true;
  if (there) {
    if (head < nq) {
      src = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
      dst = static_cast<T*>(a.q_out) + token * a.q_out_token_stride + head * a.q_out_head_stride;
      gamma = static_cast<const T*>(a.q_gamma);
    } else {
      head -= nq;
      const bool is_k = head < nk;
      if (!is_k) head -= nk;
      rotate = is_k;
      src = is_k ? static_cast<const T*>(a.k) + token * a.k_token_stride + head * a.k_head_stride
                 : static_cast<const T*>(a.v) + token * a.v_token_stride + head * a.v_head_stride;
      gamma = is_k ? static_cast<const T*>(a.k_gamma) : nullptr;
      const int64_t row = a.rows[token];
      if (row >= a.n_rows) {
        if (a.err_flag) *a.err_flag = 1;
      } else if (row >= 0) {
        const int64_t page = row / a.page_tokens;
        dst = static_cast<T*>(is_k ? a.k_cache : a.v_cache) + page * a.page_stride + head * a.head_stride +
              (row - page * a.page_tokens) * a.row_stride;
      }
    }
  }
  const int turned = a.rot_dim / 16;
  int at0, at1;
  if (u < turned) {
    at0 = INTERLEAVED ? 16 * u : 8 * u;
    at1 = INTERLEAVED ? at0 + 8 : a.rot_dim / 2 + 8 * u;
  } else {
    at0 = 16 * u;
    at1 = at0 + 8;
  }
  const bool has0 = src && at0 < a.dim, has1 = src && at1 < a.dim;
  float f[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = 0.f;
  if (has0) unpack8<T>(*reinterpret_cast<const uint4*>(src + at0), f);
  if (has1) unpack8<T>(*reinterpret_cast<const uint4*>(src + at1), f + 8);
  if (a.q_gamma || a.k_gamma) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(f[i], f[i], ss);
    for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    if (gamma) {
      const float inv = rsqrtf(ss / (float)a.dim + a.eps);
      float g[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) g[i] = 0.f;
      if (has0) unpack8<T>(*reinterpret_cast<const uint4*>(gamma + at0), g);
      if (has1) unpack8<T>(*reinterpret_cast<const uint4*>(gamma + at1), g + 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = f[i] * inv * g[i];
    }
  }
  if (rotate && src && turned) {
    const int pos = a.positions[token];
    if (pos < 0 || pos >= a.table_positions) {
      if (a.err_flag) *a.err_flag = 1;
      dst = nullptr;
    } else if (u < turned) {
      const float* cs = a.cos + (int64_t)pos * (a.rot_dim / 2) + 8 * u;
      const float* sn = a.sin + (int64_t)pos * (a.rot_dim / 2) + 8 * u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = INTERLEAVED ? 2 * i : i, y = INTERLEAVED ? 2 * i + 1 : i + 8;
        const float c = cs[i], t = sn[i], p = f[x], q = f[y];
        f[x] = p * c - q * t;
        f[y] = q * c + p * t;
      }
    }
  }
  if (dst && has0) *reinterpret_cast<uint4*>(dst + at0) = pack8<T>(f);
  if (dst && has1) *reinterpret_cast<uint4*>(dst + at1) = pack8<T>(f + 8);
}

// ---------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint4* d, const uint4* s, int64_t n, int64_t first, int64_t step) {
  for (int64_t i = first; i < n; i += step) d[i] = s[i];
}

// Tokens that slot s holds, inside what its table row can name.
__device__ __forceinline__ int64_t held(const q4gpu_pages_args& a, int64_t s) {
  const int64_t most = a.table_stride * a.page_tokens, n = a.lens[s];
  return n < 0 ? 0 : (n < most ? n : most);
}

// blockIdx.y = fork, blockIdx.x strides over the page's blocks.
__global__ void __launch_bounds__(256) pages_fork_kernel(q4gpu_pages_args a, const int32_t* parents,
                                                         const int32_t* children, const int32_t* fresh) {
  const int i = blockIdx.y;
  const int par = parents[i], chi = children[i];
  const bool first = blockIdx.x == 0;
  bool ok = par >= 0 && par < a.n_slots && chi >= 0 && chi < a.n_slots && par != chi;
  int64_t n = 0;
  int part = 0, source = 0, to = 0;
  int64_t last = -1;
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
  const int64_t vecs = a.block_bytes / a.page_tokens * part / 16;
  const char* s = static_cast<const char*>(a.pool) + source * a.page_bytes;
  char* d = static_cast<char*>(a.pool) + to * a.page_bytes;
  const int64_t blocks = a.page_bytes / a.block_bytes;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x)
    copy16(reinterpret_cast<uint4*>(d + b * a.block_bytes), reinterpret_cast<const uint4*>(s + b * a.block_bytes),
           vecs, threadIdx.x, blockDim.x);
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWords = 8192;  // bit words in shared memory: pools up to 262,144 pages

// One CTA: marks the pages in use, counts them, and pairs each used page past
// the packed end with an unused one below it (in order, so the result does not
// depend on timing).  moves = {source, destination} pairs, *n_moves of them.
__global__ void __launch_bounds__(kPlanThreads) pages_plan_kernel(q4gpu_pages_args a, int32_t* remap, int32_t* n_live,
                                                                  uint32_t* ws_bits, int32_t* n_moves, int2* moves) {
  __shared__ uint32_t s_bits[kPlanWords];
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
  int used = before;
  for (int w = lo; w < hi; ++w) {
    const uint32_t b = word(w);
    for (int k = 0; k < 32 && w * 32 + k < a.n_pages; ++k) {
      const int page = w * 32 + k;
      const bool live = (b >> k) & 1u;
      remap[page] = live ? page : -1;
      if (live && page >= total) moves[used - low].x = page;
      if (!live && page < total) moves[page - used].y = page;
      used += live;
    }
  }
  __syncthreads();
  for (int i = t; i < total - low; i += kPlanThreads) remap[moves[i].x] = moves[i].y;
}

constexpr int64_t kMoveBytes = 1 << 16;  // a work item of the page copy

// Renumbers the tables and copies the moved pages, kMoveBytes at a time.
// Sources lie at or past the packed end and destinations below it, so no copy
// reads what another writes.
__global__ void __launch_bounds__(512) pages_move_kernel(q4gpu_pages_args a, int32_t* new_table, const int32_t* remap,
                                                         const int32_t* n_moves, const int2* moves) {
  const int64_t entries = (int64_t)a.n_slots * a.table_stride;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t s = e / a.table_stride, c = e - s * a.table_stride;
    const int id = a.table[e];
    new_table[e] = c * a.page_tokens < held(a, s) && id >= 0 && id < a.n_pages ? remap[id] : -1;
  }
  const int64_t per = (a.page_bytes + kMoveBytes - 1) / kMoveBytes, items = (int64_t)*n_moves * per;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int64_t m = i / per, off = (i - m * per) * kMoveBytes;
    const int2 mv = moves[m];
    const int64_t bytes = min(kMoveBytes, a.page_bytes - off);
    copy16(reinterpret_cast<uint4*>(static_cast<char*>(a.pool) + mv.y * a.page_bytes + off),
           reinterpret_cast<const uint4*>(static_cast<const char*>(a.pool) + mv.x * a.page_bytes + off), bytes / 16,
           threadIdx.x, blockDim.x);
  }
}

int check_pages(const q4gpu_pages_args* a) {
  if (!a || !a->pool || !a->table || !a->lens) return q4gpu_fail(Q4GPU_ERR_ARG, "pages: null pointer");
  if (a->n_pages < 1 || a->page_tokens < 1 || a->n_slots < 1 || a->table_stride < 1 || a->block_bytes < 1 ||
      a->page_bytes < 1)
    return q4gpu_fail(Q4GPU_ERR_ARG, "pages: n_pages, page_tokens, n_slots, table_stride and sizes must be positive");
  if (a->page_bytes % a->block_bytes || a->block_bytes % a->page_tokens)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "pages: a page is whole blocks and a block page_tokens equal rows");
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
      !ok(a->q_gamma, 0, 0) || !ok(a->k_gamma, 0, 0))
    return q4gpu_fail(Q4GPU_ERR_ALIGN, "rope: head vectors start on 16-byte boundaries");
  const int heads = (a->q ? a->q_heads : 0) + (a->k ? a->kv_heads : 0) + (a->v ? a->kv_heads : 0);
  if (heads == 0) return Q4GPU_OK;
  const int units = a->rot_dim / 16 + (a->dim - a->rot_dim + 15) / 16;
  int lanes = 1;
  while (lanes < units) lanes *= 2;
  const int64_t threads = (int64_t)a->tokens * heads * lanes;
  const int64_t blocks = (threads + 255) / 256;
  if (blocks > INT32_MAX) return q4gpu_fail(Q4GPU_ERR_SHAPE, "rope: too many tokens");
  const unsigned grid = (unsigned)blocks;
  cudaStream_t s = as_stream(stream);
  if (a->dtype == Q4GPU_F16) {
    if (a->interleaved)
      rope_append_kernel<__half, true><<<grid, 256, 0, s>>>(*a, lanes, heads);
    else
      rope_append_kernel<__half, false><<<grid, 256, 0, s>>>(*a, lanes, heads);
  } else {
    if (a->interleaved)
      rope_append_kernel<__nv_bfloat16, true><<<grid, 256, 0, s>>>(*a, lanes, heads);
    else
      rope_append_kernel<__nv_bfloat16, false><<<grid, 256, 0, s>>>(*a, lanes, heads);
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
  const unsigned x = (unsigned)std::min<int64_t>(blocks, std::max(1, 148 * 16 / n));
  pages_fork_kernel<<<dim3(x, n), 256, 0, as_stream(stream)>>>(*a, parents, children, fresh);
  return q4gpu_check_launch();
}

// workspace: {count, padding}, moves, bit words
size_t q4gpu_pages_compact_workspace_bytes(int32_t n_pages) {
  if (n_pages < 1) return 0;
  const size_t moves = ((size_t)n_pages * sizeof(int2) + 15) / 16 * 16;
  return 16 + moves + ((size_t)n_pages + 31) / 32 * 4;
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
  cudaStream_t s = as_stream(stream);
  pages_plan_kernel<<<1, kPlanThreads, 0, s>>>(*a, remap, n_live, bits, count, moves);
  pages_move_kernel<<<148 * 4, 512, 0, s>>>(*a, new_table, remap, count, moves);
  return q4gpu_check_launch();
}

}  // extern "C"
