// Attention of each sequence's newest tokens to its pages (16-bit paged
// serving operators, include/q4gpu.h: q4gpu_paged_attention).
#include <cstdint>

#include "q4_paged.cuh"
#include "q4gpu_internal.h"

using namespace q4::paged;

namespace {

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Sequence that owns a query token: the last i with cu_q[i] <= token.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int n, int token) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= token)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// One warp per (token, query head): 32 keys at a time, lane k scoring key k,
// with the running maximum and sum of the softmax in 32 bits.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(q4gpu_attn_args a) {
  const int lane = threadIdx.x & 31;
  const int token = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  __shared__ float s_q[4][D];
  if (head >= a.q_heads) return;
  float* q = s_q[threadIdx.x >> 5];
  const T* qp = static_cast<const T*>(a.q) + token * a.q_token_stride + head * a.q_head_stride;
  for (int d = lane; d < D; d += 32) q[d] = to_f32(qp[d]);
  __syncwarp();
  const int i = sequence_of(a.cu_q, a.n_seqs, token);
  const int slot = a.seq_ids ? a.seq_ids[i] : i;
  int len = slot >= 0 && slot < a.n_slots ? a.lens[slot] : 0;
  len = (int)min((int64_t)len, a.table_stride * a.page_tokens);
  const int pos = len - (a.cu_q[i + 1] - a.cu_q[i]) + (token - a.cu_q[i]);
  const int kvh = head / (a.q_heads / a.kv_heads);
  const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  float top = -INFINITY, sum = 0.f, acc[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) acc[c] = 0.f;
  for (int k0 = first; k0 <= pos; k0 += 32) {
    const int key = k0 + lane;
    int64_t off = -1;
    if (key <= pos) {
      const int page = a.table[slot * a.table_stride + key / a.page_tokens];
      if (page >= 0 && page < a.n_pages)
        off = page * a.page_stride + kvh * a.head_stride + (key % a.page_tokens) * a.row_stride;
    }
    float s = -INFINITY;
    if (off >= 0) {
      const T* kp = static_cast<const T*>(a.k_cache) + off;
      s = 0.f;
      for (int d = 0; d < D; d += 8) {
        float f[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(kp + d), f);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(f[j], q[d + j], s);
      }
      s *= a.scale;
    }
    float m = s;
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    m = fmaxf(m, top);
    if (__all_sync(~0u, off < 0)) continue;
    const float base = m == -INFINITY ? 0.f : m;  // a row of NaN scores has no maximum
    const float p = off < 0 ? 0.f : expf(s - base), shrink = expf(top - base);
    top = m;
    float ps = p;
    for (int o = 16; o; o >>= 1) ps += __shfl_xor_sync(~0u, ps, o);
    sum = sum * shrink + ps;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) acc[c] *= shrink;
    for (int k = 0; k < 32; ++k) {
      const int64_t o = __shfl_sync(~0u, off, k);
      const float w = __shfl_sync(~0u, p, k);
      if (o < 0) continue;
      const T* vp = static_cast<const T*>(a.v_cache) + o;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(w, to_f32(vp[c * 32 + lane]), acc[c]);
    }
  }
  T* o = static_cast<T*>(a.out) + token * a.out_token_stride + head * a.out_head_stride;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) o[c * 32 + lane] = from_f32<T>(sum == 0.f ? 0.f : acc[c] / sum);
  if (a.lse && lane == 0) a.lse[(int64_t)token * a.q_heads + head] = sum == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : top) + logf(sum);
}

int check_attn(const q4gpu_attn_args* a) {
  if (!a || !a->k_cache || !a->v_cache || !a->table || !a->lens || !a->cu_q)
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null pointer");
  if (a->dtype != Q4GPU_F16 && a->dtype != Q4GPU_BF16)
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: dtype is F16 or BF16");
  if (a->dim != 64 && a->dim != 128) return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: dim = %d is not 64 or 128", a->dim);
  if (a->page_tokens != 16 && a->page_tokens != 32 && a->page_tokens != 64 && a->page_tokens != 128)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: page_tokens = %d is not 16, 32, 64 or 128", a->page_tokens);
  if (a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: %d query heads over %d key heads", a->q_heads, a->kv_heads);
  if (a->q_heads > 256 || a->kv_heads > 256)
    return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: at most 256 heads");
  if (a->n_seqs < 0 || a->n_seqs > 65535 || a->tokens < 0 || a->max_q < 0 || a->max_ctx < 0 || a->window < 0 ||
      a->n_slots < 1 || a->n_pages < 1 || a->table_stride < 1)
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: negative or empty size");
  if (a->tokens != 0 && (!a->q || !a->out)) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null pointer");
  if (!(a->scale == a->scale)) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: scale is not a number");
  if (!aligned(a->q, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16) || !aligned(a->out, 16) ||
      a->q_token_stride % 8 || a->q_head_stride % 8 || a->out_token_stride % 8 || a->out_head_stride % 8 ||
      a->page_stride % 8 || a->head_stride % 8 || a->row_stride % 8)
    return q4gpu_fail(Q4GPU_ERR_ALIGN, "attention: head vectors start on 16-byte boundaries");
  return Q4GPU_OK;
}

}  // namespace

extern "C" {

size_t q4gpu_paged_attention_workspace_bytes(const q4gpu_attn_args*) { return 0; }

int q4gpu_paged_attention(const q4gpu_attn_args* a, void* stream) {
  const int rc = check_attn(a);
  if (rc != Q4GPU_OK) return rc;
  if (a->n_seqs == 0 || a->tokens == 0) return Q4GPU_OK;
  const dim3 grid(a->tokens, (a->q_heads + 3) / 4);
  cudaStream_t s = as_stream(stream);
  if (a->dtype == Q4GPU_F16) {
    if (a->dim == 64)
      paged_attn_kernel<__half, 64><<<grid, 128, 0, s>>>(*a);
    else
      paged_attn_kernel<__half, 128><<<grid, 128, 0, s>>>(*a);
  } else {
    if (a->dim == 64)
      paged_attn_kernel<__nv_bfloat16, 64><<<grid, 128, 0, s>>>(*a);
    else
      paged_attn_kernel<__nv_bfloat16, 128><<<grid, 128, 0, s>>>(*a);
  }
  return q4gpu_check_launch();
}

}  // extern "C"
