// Attention of each sequence's newest tokens to its pages (16-bit paged
// serving operators, include/q4gpu.h: q4gpu_paged_attention).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cstdint>

#include "q4_paged.cuh"
#include "q4_paged_chunk.cuh"
#include "q4gpu_internal.h"

using namespace q4::paged;

namespace {

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// What a CTA needs to know of sequence i.
struct Seq {
  int slot, len, first, n;  // cache slot, stored keys, first query token, query tokens
};
__device__ __forceinline__ Seq sequence(const q4gpu_attn_args& a, int i) {
  Seq s;
  s.first = max(0, min(a.cu_q[i], a.tokens));
  s.n = max(0, min(a.cu_q[i + 1], a.tokens) - s.first);
  s.slot = a.seq_ids ? a.seq_ids[i] : i;
  const bool known = s.slot >= 0 && s.slot < a.n_slots;
  s.len = known ? (int)max((int64_t)0, min((int64_t)a.lens[s.slot], most_keys(a))) : 0;
  return s;
}

// ---------------------------------------------------------------------------
// few query rows (decode): at most 16 (token, head) pairs share a key head
// ---------------------------------------------------------------------------
constexpr int kRows = 16;        // rows of one mma.sync tile
constexpr int kTileKeys = 16;    // keys of a warp's step; a page holds whole steps
constexpr int kRowWarps = 8;
constexpr int kRowStages = 3;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int D>
constexpr int row_smem() { return kRowWarps * kRowStages * 2 * kTileKeys * D * 2; }

// 16-byte piece c of row r in a tile of D-value rows: pieces are exchanged
// inside each 128-byte line by the row number, so the eight rows that an
// ldmatrix phase reads lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t piece(int r, int c) { return (uint32_t)(r * D * 2 + ((c ^ (r & 7)) * 16)); }

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Work is laid out on one axis: sequence by sequence, key head by key head, in
// units of 128 keys, each (sequence, head) behind kPieceCost units that stand for
// what starting it costs (64 decodes at 1 to 8704 keys: 59.3 us with 2, 56.7 with
// 3, 60.2 with 4).  Every CTA takes an equal stretch of that axis, so the
// longest sequence does not decide; a stretch's ends cut at most two (sequence,
// head) items, whose pieces are joined by the CTA that finishes last, in the
// order of the pieces.
constexpr int kUnitKeys = kRowWarps * kTileKeys;
constexpr int kPieceCost = 3;
constexpr int kMostCtas = 1024;   // counters, always at the workspace's start: no other call's data gets there
constexpr int kLeastStretch = 6;  // units: shorter pieces cost more to join than they save

struct RowPlan {
  int ctas;
  float* o;       // [cta][2][kRows][D] unnormalised sums: of a piece begun earlier, of one that goes on
  float2* ml;     // [cta][2][kRows] their running maximum (log2 units) and sum
  int32_t* done;  // [cta] finished pieces of the item whose first piece goes on from this CTA
};

// Keys that the kernel below walks for sequence i, from `lo` on; -1: not its
// sequence (no queries, or more rows than a tile).
__device__ __forceinline__ int row_keys(const q4gpu_attn_args& a, const Seq& s, int group, int& lo) {
  lo = 0;
  if (s.n == 0 || s.n > kRows / group) return -1;
  if (a.window > 0) lo = first_seen(s.len - s.n, a.window) & ~(kTileKeys - 1);
  return max(0, s.len - lo);
}
__device__ __forceinline__ int row_cost(const q4gpu_attn_args& a, int i, int group) {  // of one head
  int lo;
  const int keys = row_keys(a, sequence(a, i), group, lo);
  return keys < 0 ? 0 : kPieceCost + (keys + kUnitKeys - 1) / kUnitKeys;
}

// Each warp runs over its own 16-key steps of a piece with its own running
// maximum and sum, so no barrier stands in the loop; the eight are joined at its
// end.  (Eight warps and one CTA per SM for heads of 128, two for 64; four warps
// and twice the CTAs start short pieces a little faster, 64 decodes at 1 to 8704
// keys 55.6 us against 57.0, but take 33.0 against 24.0 for one at 16384 and 122
// against 94 for 16 of 64-value heads.)  Bound by memory: every key and value is
// read once, for all heads of its group; 16 decodes at 16384 keys stream 6.1 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) attn_rows_kernel(q4gpu_attn_args a, RowPlan plan) {
  constexpr int kThreads = kRowWarps * 32;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float s_m[kRowWarps][kRows], s_l[kRowWarps][kRows];
  __shared__ int64_t s_sum[kRowWarps], s_start;
  __shared__ int s_most[kRowWarps], s_seq, s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.q_heads / a.kv_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the chunk kernel reads nothing of this one
  // the axis: each thread adds up a run of sequences
  const int per = (a.n_seqs + kThreads - 1) / kThreads;
  const int run0 = min(a.n_seqs, (int)threadIdx.x * per), run1 = min(a.n_seqs, run0 + per);
  int64_t mine_cost = 0;
  int most = 0;
  // without a chunk kernel beside this one nobody computes a sequence longer than max_q and a tile: its rows become zeros
  const bool alone = (int64_t)a.max_q * group <= kRows;
  bool over = false;
  for (int i = run0; i < run1; ++i) {
    over |= alone && sequence(a, i).n > kRows / group;
    if (blockIdx.x == 0 && a.err_flag && !sequence_ok(a, i)) *a.err_flag = 1;
    const int c = row_cost(a, i, group);
    mine_cost += (int64_t)c * a.kv_heads;
    most = max(most, c);
  }
  int64_t upto = mine_cost;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(~0u, upto, o);
    if (lane >= o) upto += v;
  }
  most = __reduce_max_sync(~0u, most);
  if (lane == 31) s_sum[warp] = upto;
  if (lane == 0) s_most[warp] = most;
  over = __syncthreads_or(over);
  int64_t total = 0, before = upto - mine_cost;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
    most = max(most, s_most[w]);
  }
  // (32-bit divisions where the numbers allow them)
  auto quotient = [](int64_t x, int64_t y) {
    return (x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
  };
  const int64_t stretch = max(quotient(total + plan.ctas - 1, plan.ctas), (int64_t)min(most, kLeastStretch));
  const int64_t first_unit = blockIdx.x * stretch, last_unit = min(total, first_unit + stretch);
  if (first_unit < last_unit) {
    if (before <= first_unit && first_unit < before + mine_cost) {  // one thread's run holds it
      int i = run0;
      for (int64_t c; before + (c = (int64_t)row_cost(a, i, group) * a.kv_heads) <= first_unit; ++i) before += c;
      s_seq = i, s_start = before;
    }
    __syncthreads();
    int seq = s_seq, lo;
    int64_t start = s_start;  // where the sequence's first head begins
    Seq s = sequence(a, seq);
    int keys = row_keys(a, s, group, lo), cost = row_cost(a, seq, group), kvh = (int)quotient(first_unit - start, cost);
    for (;;) {
      const int64_t head_start = start + (int64_t)kvh * cost + kPieceCost;  // of its first real unit
      if (head_start - kPieceCost >= last_unit) break;
      const int units = cost - kPieceCost;
      const int u0 = (int)max((int64_t)0, first_unit - head_start);
      const int u1 = (int)min((int64_t)units, last_unit - head_start);
      // (a sequence without keys: its zeros are written by the CTA where its cost begins)
      if (u1 > u0 || (units == 0 && head_start - kPieceCost >= first_unit)) {
        const int rows = s.n * group;
        const int64_t cta0 = quotient(head_start, stretch),
                      cta1 = units == 0 ? cta0 : quotient(head_start + units - 1, stretch);
        const int parts = (int)(cta1 - cta0) + 1, part = (int)(blockIdx.x - cta0);
        const int pos0 = s.len - s.n, pos1 = s.len - 1;  // of the first and the last query
        const int begin = lo + u0 * kUnitKeys, end = min(s.len, lo + u1 * kUnitKeys);

        // the queries as A fragments: row g and g + 8, 16 values of a head per step
        const int g = lane >> 2, tq = lane & 3;
        uint32_t qf[D / 16][4];
        int row_pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = g + 8 * h, t = r / group;
          row_pos[h] = r < rows ? pos0 + t : -1;
          const T* qp = static_cast<const T*>(a.q) + (int64_t)(s.first + t) * a.q_token_stride +
                        (int64_t)(kvh * group + r - t * group) * a.q_head_stride + 2 * tq;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            qf[k][h] = r < rows ? *reinterpret_cast<const uint32_t*>(qp + 16 * k) : 0u;
            qf[k][h + 2] = r < rows ? *reinterpret_cast<const uint32_t*>(qp + 16 * k + 8) : 0u;
          }
        }

        const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kRowStages * 2 * kTileKeys * D * 2);
        constexpr int kTileBytes = kTileKeys * D * 2;
        const int32_t* table = a.table + (int64_t)max(0, min(s.slot, a.n_slots - 1)) * a.table_stride;
        const int steps = units > 0 ? (end - begin + kTileKeys - 1) / kTileKeys : 0;
        const int mine = steps > warp ? (steps - warp + kRowWarps - 1) / kRowWarps : 0;
        const int shift = 31 - __clz(a.page_tokens);
        auto page_of = [&](int i) {
          if (i >= mine) return -1;
          const int p = table[(begin + kTileKeys * (warp + kRowWarps * i)) >> shift];
          if (p >= 0 && p < a.n_pages) return p;
          if (a.err_flag) *a.err_flag = 1;
          return -1;
        };
        int next_page = page_of(0);
        uint32_t valid = 0;  // bit i % 32: step i's page exists
        auto load = [&](int i) {
          const int page = next_page;
          next_page = page_of(i + 1);
          if (i < mine) valid = (valid & ~(1u << (i & 31))) | ((page >= 0 ? 1u : 0u) << (i & 31));
          if (i < mine && page >= 0) {
            const int key = begin + kTileKeys * (warp + kRowWarps * i);
            const int64_t off = page * a.page_stride + kvh * a.head_stride + (key & (a.page_tokens - 1)) * a.row_stride;
            const uint32_t at = ring + (i % kRowStages) * 2 * kTileBytes;
            constexpr int kPieces = D / 8, kPer = 32 / kPieces;  // lanes per row, rows per pass
            const int c = lane % kPieces;
#pragma unroll
            for (int r0 = 0; r0 < kTileKeys; r0 += kPer) {
              const int r = r0 + lane / kPieces;
              // rows past the last key are zeros: whatever the page holds there meets a zero weight
              const bool there = key + r < end;
              const int64_t o = off + (there ? r : 0) * a.row_stride + c * 8;
              cp16(at + piece<D>(r, c), static_cast<const T*>(a.k_cache) + o, there);
              cp16(at + kTileBytes + piece<D>(r, c), static_cast<const T*>(a.v_cache) + o, there);
            }
          }
          cp_commit();
        };
#pragma unroll
        for (int i = 0; i < kRowStages - 1; ++i) load(i);

        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        const float c2 = a.scale * kLog2e;
        for (int i = 0; i < mine; ++i) {
          cp_wait<kRowStages - 2>();
          __syncwarp();
          load(i + kRowStages - 1);
          if (!((valid >> (i & 31)) & 1u)) continue;
          const uint32_t kt = ring + (i % kRowStages) * 2 * kTileBytes, vt = kt + kTileBytes;
          const int key = begin + kTileKeys * (warp + kRowWarps * i);
          float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];  // keys 0-7: b[0], b[1]; keys 8-15: b[2], b[3]
            ldsm4(b, kt + piece<D>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
            mma16816<T>(sc[0], qf[k], b[0], b[1]);
            mma16816<T>(sc[1], qf[k], b[2], b[3]);
          }
          // element e of sc[n]: row g + 8 (e / 2), key 8 n + 2 tq + e % 2
          const bool whole = key + kTileKeys <= pos0 + 1 && (a.window == 0 || key > pos1 - a.window);
          float top[2] = {m[0], m[1]};
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = sc[n][e] * c2;
              if (!whole) {
                const int j = key + 8 * n + 2 * tq + (e & 1), p = row_pos[e >> 1];
                if (j > p || (a.window > 0 && j <= p - a.window)) v = -INFINITY;
              }
              sc[n][e] = v;
              top[e >> 1] = fmaxf(top[e >> 1], v);
            }
          float shrink[2], base[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 2));
            base[h] = top[h] == -INFINITY ? 0.f : top[h];  // nothing seen yet
            shrink[h] = ex2(m[h] - base[h]);
            m[h] = top[h];
            l[h] *= shrink[h];
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sc[n][e] = ex2(sc[n][e] - base[e >> 1]);
              l[e >> 1] += sc[n][e];  // this lane's keys; the four lanes of a row are added at the end
            }
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= shrink[e >> 1];
          // Some rows see a key of this step and some do not: an infinity or NaN in its value row may reach only the
          // former, and a product would carry it to both (0 times infinity).  Such values are added by hand and zeroed.
          if (key + kTileKeys > pos0 + 1 || (a.window > 0 && key <= pos1 - a.window)) {
            unsigned char* v = smem + (vt - (uint32_t)__cvta_generic_to_shared(smem));
            bool odd = false;
            for (int x = lane; x < kTileKeys * D; x += 32)
              odd |= !isfinite(to_f32(*reinterpret_cast<const T*>(v + x * 2)));
            if (__any_sync(~0u, odd)) {
              for (int j = 0; j < kTileKeys; ++j)
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int col = 8 * n + 2 * tq + (e & 1), p = row_pos[e >> 1];
                    const float x = to_f32(*reinterpret_cast<const T*>(v + piece<D>(j, col / 8) + (col % 8) * 2));
                    if (!isfinite(x) && key + j <= p && (a.window == 0 || key + j > p - a.window)) o[n][e] += x;
                  }
              __syncwarp();
              for (int x = lane; x < kTileKeys * D; x += 32) {
                T* at = reinterpret_cast<T*>(v + x * 2);
                if (!isfinite(to_f32(*at))) *at = from_f32<T>(0.f);
              }
              __syncwarp();
            }
          }
          // weights rounded to the cache's type for the tensor cores (their sum is not)
          const uint32_t pf[4] = {pack2<T>(sc[0][0], sc[0][1]), pack2<T>(sc[0][2], sc[0][3]),
                                  pack2<T>(sc[1][0], sc[1][1]),
                                  pack2<T>(sc[1][2], sc[1][3])};
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            uint32_t b[4];  // 16 keys x 16 values
            ldsm4_t(b, vt + piece<D>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * n + (lane >> 4)));
            mma16816<T>(o[2 * n], pf, b[0], b[1]);
            mma16816<T>(o[2 * n + 1], pf, b[2], b[3]);
          }
        }
        cp_wait<0>();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          l[h] += __shfl_xor_sync(~0u, l[h], 1);
          l[h] += __shfl_xor_sync(~0u, l[h], 2);
          if (tq == 0) s_m[warp][g + 8 * h] = m[h], s_l[warp][g + 8 * h] = l[h];
        }
        __syncthreads();  // every warp is done with its ring
        // the warps' sums, side by side in the ring's memory
        float* so = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (g + 8 * h < rows)
              *reinterpret_cast<float2*>(so + (warp * kRows + g + 8 * h) * D + 8 * n + 2 * tq) =
                  make_float2(o[n][2 * h], o[n][2 * h + 1]);
        __syncthreads();
        auto put = [&](int r, int d, float m_all, float l_all, float v) {
          const int t = r / group, head = kvh * group + r - t * group;
          static_cast<T*>(a.out)[(int64_t)(s.first + t) * a.out_token_stride + (int64_t)head * a.out_head_stride + d] =
              from_f32<T>(l_all == 0.f ? 0.f : v / l_all);
          if (a.lse && d == 0)
            a.lse[(int64_t)(s.first + t) * a.q_heads + head] = l_all == 0.f ? -INFINITY : (m_all + log2f(l_all)) * kLn2;
        };
        for (int x = threadIdx.x; x < rows * D; x += kRowWarps * 32) {
          const int r = x / D, d = x - r * D;
          float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
          for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, s_m[w][r]);
          const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int w = 0; w < kRowWarps; ++w) {
            const float f = ex2(s_m[w][r] - base);
            sum = fmaf(s_l[w][r], f, sum);
            v = fmaf(so[(w * kRows + r) * D + d], f, v);
          }
          if (parts == 1) {
            put(r, d, base, sum, v);
          } else {
            const int64_t at = (2 * (int64_t)blockIdx.x + (part == 0)) * kRows + r;
            plan.o[at * D + d] = v;
            if (d == 0) plan.ml[at] = make_float2(top, sum);
          }
        }
        if (parts > 1) {
          __threadfence();
          __syncthreads();
          if (threadIdx.x == 0) {
            s_last = atomicAdd(plan.done + cta0, 1) == parts - 1;
            if (s_last) plan.done[cta0] = 0;
          }
          __syncthreads();
          if (s_last) __threadfence();
        }
        if (parts > 1 && s_last)
          for (int x = threadIdx.x; x < rows * D; x += kRowWarps * 32) {
            const int r = x / D, d = x - r * D;
            auto slot = [&](int k) { return (2 * (cta0 + k) + (k == 0)) * kRows + r; };
            float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll 8
            for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(&plan.ml[slot(k)]).x);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 8
            for (int k = 0; k < parts; ++k) {
              const float2 w = __ldcg(&plan.ml[slot(k)]);
              const float f = ex2(w.x - base);
              sum = fmaf(w.y, f, sum);
              v = fmaf(__ldcg(&plan.o[slot(k) * D + d]), f, v);
            }
            put(r, d, base, sum, v);
          }
        __syncthreads();  // the ring and the shared words are free for the next piece
      }
      if (++kvh == a.kv_heads) {
        kvh = 0;
        start += (int64_t)cost * a.kv_heads;
        do {
          if (++seq >= a.n_seqs) break;
          s = sequence(a, seq);
          keys = row_keys(a, s, group, lo);
          cost = row_cost(a, seq, group);
        } while (cost == 0);
        if (seq >= a.n_seqs) break;
      }
    }
  }
  if (over)
    for (int i = blockIdx.x; i < a.n_seqs; i += gridDim.x) {
      const Seq s = sequence(a, i);
      if (s.n <= kRows / group) continue;
      for (int64_t x = threadIdx.x; x < (int64_t)s.n * a.q_heads * D; x += kThreads) {
        const int64_t row = x / D, t = s.first + row / a.q_heads, head = row % a.q_heads;
        static_cast<T*>(a.out)[t * a.out_token_stride + head * a.out_head_stride + x % D] = from_f32<T>(0.f);
        if (a.lse && x % D == 0) a.lse[t * a.q_heads + head] = -INFINITY;
      }
    }
}

int check_sizes(const q4gpu_attn_args* a) {
  if (!a) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null arguments");
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
      a->n_slots < 1 || a->n_pages < 1 || a->table_stride < 1 || a->table_pages < 0)
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: negative or empty size");
  return Q4GPU_OK;
}

int check_attn(const q4gpu_attn_args* a) {
  const int rc = check_sizes(a);
  if (rc != Q4GPU_OK) return rc;
  if (!a->k_cache || !a->v_cache || !a->table || !a->lens || !a->cu_q)
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null pointer");
  if (a->tokens != 0 && (!a->q || !a->out)) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null pointer");
  if (!(a->scale == a->scale)) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: scale is not a number");
  if (!aligned(a->q, 16) || !aligned(a->k_cache, 16) || !aligned(a->v_cache, 16) || !aligned(a->out, 16) ||
      a->q_token_stride % 8 || a->q_head_stride % 8 || a->out_token_stride % 8 || a->out_head_stride % 8 ||
      a->page_stride % 8 || a->head_stride % 8 || a->row_stride % 8)
    return q4gpu_fail(Q4GPU_ERR_ALIGN, "attention: head vectors start on 16-byte boundaries");
  return Q4GPU_OK;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int kSms = 148;

// The arguments as the kernels take them.
q4gpu_attn_args settled(const q4gpu_attn_args& a) {
  q4gpu_attn_args b = a;
  if (b.table_pages == 0) b.table_pages = (int32_t)std::min<int64_t>(b.table_stride, INT32_MAX);
  // a window that no slot's keys fill is none (position - window would pass 31 bits for queries before the first key)
  if (b.window >= std::min<int64_t>((int64_t)b.table_pages * b.page_tokens, INT32_MAX)) b.window = 0;
  return b;
}

RowPlan row_plan(const q4gpu_attn_args& a, char* ws, size_t* bytes) {
  RowPlan p{};
  const size_t items = (size_t)a.n_seqs * a.kv_heads;
  // no CTA without at least one (sequence, head) or kLeastStretch units of one
  const int64_t units = ((int64_t)a.max_ctx + kUnitKeys - 1) / kUnitKeys + kPieceCost;
  const int64_t most = (int64_t)items * std::max<int64_t>(1, (units + kLeastStretch - 1) / kLeastStretch + 1);
  p.ctas = (int)std::min<int64_t>(most, kSms * (a.dim == 64 ? 2 : 1));
  static_assert(kSms * 4 <= kMostCtas, "a counter a CTA");
  const size_t done = kMostCtas * sizeof(int32_t), rows = (size_t)p.ctas * 2 * kRows;
  if (bytes) *bytes = done + rows * (8 + (size_t)a.dim * 4);
  p.done = reinterpret_cast<int32_t*>(ws);
  p.ml = reinterpret_cast<float2*>(ws + done);
  p.o = reinterpret_cast<float*>(p.ml + rows);
  return p;
}

// Parts of a chunk's keys: one where the (row pair, key head) items fill the
// GPU, else as many as fill it once, each of at least kMinPart keys.  (Cutting
// the last wave of many items in two evens the SMs out, 348 steps on the longest
// instead of 370 for 8192 tokens over 16384 keys, but the parts' traffic and the
// join took more: 814 us against 771.)
ChunkPlan chunk_plan(const q4gpu_attn_args& a, size_t* bytes) {
  ChunkPlan p{};
  const int64_t group = a.q_heads / a.kv_heads;
  if (a.max_q * group <= kRows || a.n_seqs == 0 || a.tokens == 0) {  // nothing for the chunk kernel
    if (bytes) *bytes = 0;
    return p;
  }
  // (a lone sequence of any length is the chunk kernel's: one launch)
  p.least = a.n_seqs == 1 ? 1 : (int)(kRows / group) + 1;
  const int64_t rows = a.tokens * group;
  p.tiles = (int)std::min<int64_t>(a.n_seqs == 1 ? (rows + kPair - 1) / kPair : rows / kPair + a.n_seqs, INT32_MAX);
  const int64_t items = (int64_t)p.tiles * a.kv_heads;
  const int64_t span = a.window > 0 ? std::min<int64_t>(a.max_ctx, (int64_t)a.window + kPair + kNTile) : a.max_ctx;
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(kSms / items, span / kMinPart));
  if (bytes) *bytes = p.parts > 1 ? (size_t)p.tiles * a.kv_heads * p.parts * kPair * (8 + (size_t)a.dim * 4) : 0;
  return p;
}

int encode_map(CUtensorMap* map, const q4gpu_attn_args& a, const void* base) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (!encode) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", reinterpret_cast<void**>(&encode), cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess || !encode)
      return q4gpu_fail(Q4GPU_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  }
  // one 128-byte line of every row of a page per box; a stride that nothing takes (one head, heads that share their
  // keys, one page) is given as the least that the map allows
  const cuuint64_t unused = (cuuint64_t)a.dim * 2;
  const bool heads = a.kv_heads > 1 && a.head_stride != 0;
  const cuuint64_t dims[4] = {(cuuint64_t)a.dim, (cuuint64_t)a.page_tokens, heads ? (cuuint64_t)a.kv_heads : 1,
                              (cuuint64_t)a.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)a.row_stride * 2, heads ? (cuuint64_t)a.head_stride * 2 : unused,
                                 a.n_pages > 1 ? (cuuint64_t)a.page_stride * 2 : unused};
  const cuuint32_t box[4] = {64, (cuuint32_t)a.page_tokens, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type =
      a.dtype == Q4GPU_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = encode(map, type, 4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return q4gpu_fail(Q4GPU_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return Q4GPU_OK;
}

// Raises a kernel's shared-memory limit once per device.
int allow_smem(const void* kernel, int bytes, unsigned char* ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < Q4GPU_MAX_DEVICES && ready[dev]) return Q4GPU_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "attention: shared memory: %s", cudaGetErrorString(e));
  if (dev < Q4GPU_MAX_DEVICES) ready[dev] = 1;
  return Q4GPU_OK;
}

template <typename T, int D>
int launch(const q4gpu_attn_args& a, cudaStream_t s) {
  static unsigned char ready[2][Q4GPU_MAX_DEVICES];
  size_t rows_bytes;
  const RowPlan few = row_plan(a, static_cast<char*>(a.workspace), &rows_bytes);
  const bool chunks = (int64_t)a.max_q * (a.q_heads / a.kv_heads) > kRows;
  ChunkPlan plan = chunk_plan(a, nullptr);
  if (plan.tiles > 65535) return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: too many query rows");
  const bool short_ones = !chunks || plan.least > 1;  // sequences for attn_rows_kernel
  int rc = Q4GPU_OK;
  if (short_ones) {
    rc = allow_smem(reinterpret_cast<const void*>(attn_rows_kernel<T, D>), row_smem<D>(), ready[0]);
    if (rc != Q4GPU_OK) return rc;
  }
  CUtensorMap kmap, vmap;
  if (chunks) {
    char* ws = static_cast<char*>(a.workspace) + (rows_bytes + 15) / 16 * 16;
    plan.ml = reinterpret_cast<float2*>(ws);
    plan.o = reinterpret_cast<float*>(plan.ml + (size_t)plan.tiles * a.kv_heads * plan.parts * kPair);
    rc = encode_map(&kmap, a, a.k_cache);
    if (rc == Q4GPU_OK) rc = encode_map(&vmap, a, a.v_cache);
    if (rc == Q4GPU_OK)
      rc = allow_smem(reinterpret_cast<const void*>(attn_chunk_kernel<T, D>), chunk_smem<D>(), ready[1]);
    if (rc != Q4GPU_OK) return rc;
  }
  if (short_ones) attn_rows_kernel<T, D><<<few.ctas, kRowWarps * 32, row_smem<D>(), s>>>(a, few);
  if (chunks) {
    // starts beside the short sequences' kernel, on the SMs that it leaves free
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.kv_heads, plan.tiles, plan.parts);
    cfg.blockDim = dim3(kChunkThreads);
    cfg.dynamicSmemBytes = chunk_smem<D>();
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = short_ones ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_chunk_kernel<T, D>, kmap, vmap, a, plan);
    if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "attention: launch: %s", cudaGetErrorString(e));
    if (plan.parts > 1) attn_join_kernel<T, D><<<dim3(a.kv_heads, plan.tiles, kPair / 8), 256, 0, s>>>(a, plan);
  }
  return q4gpu_check_launch();
}

}  // namespace

extern "C" {

size_t q4gpu_paged_attention_workspace_bytes(const q4gpu_attn_args* a) {
  if (check_sizes(a) != Q4GPU_OK) return 0;
  const q4gpu_attn_args b = settled(*a);
  size_t rows, chunks;
  row_plan(b, nullptr, &rows);
  chunk_plan(b, &chunks);
  return (rows + 15) / 16 * 16 + chunks;
}

int q4gpu_paged_attention(const q4gpu_attn_args* a, void* stream) {
  const int rc = check_attn(a);
  if (rc != Q4GPU_OK) return rc;
  if (a->n_seqs == 0 || a->tokens == 0) return Q4GPU_OK;
  const size_t need = q4gpu_paged_attention_workspace_bytes(a);
  if (a->workspace_bytes < need || (need && !a->workspace))
    return q4gpu_fail(Q4GPU_ERR_WORKSPACE, "attention: needs a workspace of %zu bytes", need);
  if (!aligned(a->workspace, 16)) return q4gpu_fail(Q4GPU_ERR_ALIGN, "attention: workspace must be 16-byte aligned");
  const q4gpu_attn_args b = settled(*a);
  cudaStream_t s = as_stream(stream);
  if (b.dtype == Q4GPU_F16) return b.dim == 64 ? launch<__half, 64>(b, s) : launch<__half, 128>(b, s);
  return b.dim == 64 ? launch<__nv_bfloat16, 64>(b, s) : launch<__nv_bfloat16, 128>(b, s);
}

}  // extern "C"
