// Log probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits (include/q4gpu.h: q4gpu_token_logprobs).
#include <cstdint>

#include "q4_paged.cuh"
#include "q4gpu_internal.h"

using namespace q4::paged;

namespace {

constexpr int kThreads = 512;

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

// One CTA a row.  With m the row's largest logit, S the sum of e^(x - m) over all
// but one place of the largest and T = sum e^(x - m) (x - m):
//   log p_t = (x_t - m) - log1p(S),   H = log1p(S) - T / (1 + S),
// sums without cancellation however certain the row is.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(q4gpu_logprob_args a) {
  __shared__ uint64_t s_key[kThreads / 32];
  __shared__ float s_sum[2][kThreads / 32];
  __shared__ int s_ahead[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  auto block_max = [&](uint64_t k) {
    for (int o = 16; o; o >>= 1) k = max(k, __shfl_xor_sync(~0u, k, o));
    __syncthreads();
    if (lane == 0) s_key[warp] = k;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) k = max(k, s_key[w]);
    return k;
  };
  const int64_t given = a.targets ? a.targets[row] : -1;
  const bool known = given >= 0 && given < a.vocab;
  const uint64_t mine = known ? key_of(to_f32(x[given]), (int)given) : ~0ull;
  uint64_t top = 0;
  int ahead = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const uint64_t k = key_of(to_f32(x[i]), i);
    top = max(top, k);
    ahead += k > mine;
  }
  top = block_max(top);
  const float m = logit_of((uint32_t)(top >> 32));
  const int best = ~(int)(uint32_t)top;
  const bool none = m == -INFINITY, odd = !(m < INFINITY);
  float sum = 0.f, held = 0.f;
  if (!none && !odd)
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const float d = to_f32(x[i]) - m, e = ex2(d * 1.4426950408889634f);
      if (i != best) sum += e;
      if (e > 0.f) held = fmaf(e, d, held);
    }
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, o);
    held += __shfl_xor_sync(~0u, held, o);
    ahead += __shfl_xor_sync(~0u, ahead, o);
  }
  if (lane == 0) s_sum[0][warp] = sum, s_sum[1][warp] = held, s_ahead[warp] = ahead;
  __syncthreads();
  sum = held = 0.f, ahead = 0;
  for (int w = 0; w < kThreads / 32; ++w) sum += s_sum[0][w], held += s_sum[1][w], ahead += s_ahead[w];
  const float norm = log1pf(sum), nan = __uint_as_float(0x7fffffffu);
  auto logprob = [&](float v) { return odd ? nan : none ? -INFINITY : (v - m) - norm; };
  if (threadIdx.x == 0) {
    if (a.targets) {
      a.logprob[row] = known ? logprob(to_f32(x[given])) : 0.f;
      a.rank[row] = known ? ahead + 1 : 0;
      if (given >= a.vocab && a.err_flag) *a.err_flag = 1;
    }
    a.entropy[row] = odd ? nan : none ? 0.f : norm - held / (1.f + sum);
  }
  for (int k = 0; k < a.top; ++k) {
    if (threadIdx.x == 0) {
      a.top_logprob[row * a.top + k] = logprob(logit_of((uint32_t)(top >> 32)));
      a.top_index[row * a.top + k] = ~(int)(uint32_t)top;
    }
    uint64_t next = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const uint64_t key = key_of(to_f32(x[i]), i);
      if (key < top) next = max(next, key);
    }
    top = block_max(next);
  }
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
  const unsigned grid = (unsigned)a->rows;
  if (a->dtype == Q4GPU_F32)
    token_logprobs_kernel<float><<<grid, kThreads, 0, s>>>(*a);
  else if (a->dtype == Q4GPU_F16)
    token_logprobs_kernel<__half><<<grid, kThreads, 0, s>>>(*a);
  else
    token_logprobs_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(*a);
  return q4gpu_check_launch();
}
