// Attention of each sequence's newest tokens to its pages (16-bit paged
// serving operators, include/q4gpu.h: q4gpu_paged_attention, q4gpu_sink_attention,
// q4gpu_shared_attention).
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

// ---------------------------------------------------------------------------
// few query rows (decode): at most 16 (token, head) pairs share a key head
// ---------------------------------------------------------------------------
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

// Work is laid out on one axis: item by item (a sequence, or with kShared the own
// keys of one or the shared keys of a group), block of key heads by block, tile
// of 16 rows by tile, in units of keys (128 keys of one head, or as many of all of
// a block's together), each such subitem behind kPieceCost units that stand for
// what starting it costs (64 decodes at 1 to 8704 keys: 59.3 us with 2, 56.7 with
// 3, 60.2 with 4).  Every CTA takes an equal stretch of that axis, so the
// longest sequence does not decide; a stretch's ends cut at most two subitems,
// whose pieces are joined in the order of the pieces, by the CTA that finishes
// last, or with kShared by the kernel that joins own and shared keys.
constexpr int kCounters = 4096;  // always at the workspace's start: no other call's data gets there

// Each warp runs over its own 16-key steps of a piece with its own running
// maximum and sum, so no barrier stands in the loop; those of a head are joined at
// its end (with a head a warp there is nothing to join, and no barrier at all).
// (Eight warps and one CTA per SM for heads of 128, two for 64; four warps
// and twice the CTAs start short pieces a little faster, 64 decodes at 1 to 8704
// keys 55.6 us against 57.0, but take 33.0 against 24.0 for one at 16384 and 122
// against 94 for 16 of 64-value heads.)  Bound by memory: every key and value is
// read once, for all heads of its group; 16 decodes at 16384 keys stream 6.1 TB/s.
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kRowWarps * 32, D == 64 ? 2 : 1)
    attn_rows_kernel(q4gpu_attn_args a, More x, RowPlan plan) {
  constexpr int W = kRowWarps, kThreads = W * 32;
  const int heads = MODE == kPlain ? 1 : 1 << plan.heads_log;  // of a piece; each has `slices` of the warps
  const int slices = MODE == kPlain ? W : W >> plan.heads_log, unit_keys = slices * kTileKeys;
  const int blocks = MODE == kPlain ? a.kv_heads : a.kv_heads >> plan.heads_log;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float s_m[W][kRows], s_l[W][kRows];
  __shared__ int64_t s_sum[W], s_start;
  __shared__ int s_most[W], s_seq, s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.q_heads / a.kv_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the chunk kernel reads nothing of this one
  __shared__ __align__(16) unsigned char s_staged[MODE != kPlain ? sizeof(Staged) : 16];
  __shared__ Item s_item[MODE != kPlain ? 2 * kStaged : 1];
  const bool known = few<MODE>(a, x);
  const Where where = where_of<MODE>(a, x, reinterpret_cast<Staged*>(s_staged));
  if constexpr (MODE != kPlain) __syncthreads();
  // the axis: each thread adds up a run of sequences
  const int items = item_count<MODE>(a, x), per = (items + kThreads - 1) / kThreads;
  const int run0 = min(items, (int)threadIdx.x * per), run1 = min(items, run0 + per);
  int64_t mine_cost = 0;
  int most = 0;
  bool malformed = false;
  // without a chunk kernel beside this one nobody computes a sequence longer than max_q and a tile: its rows become zeros
  // (with kShared, attn_shared_join_kernel writes the zeros)
  const bool alone = MODE != kShared && (int64_t)a.max_q * group <= kRows;
  bool over = false;
  for (int i = run0; i < run1; ++i) {
    const Item s = item_of<MODE>(a, x, where, i);
    if (MODE != kPlain && known) s_item[i] = s;
    over |= alone && s.n > kRows / group;
    if constexpr (MODE == kShared) {  // (which the joining kernel reports)
      if (blockIdx.x == 0 && !few<MODE>(a, x)) malformed |= !ascends(a, where, i);
    } else if constexpr (MODE == kPlain) {
      if (blockIdx.x == 0 && a.err_flag && !sequence_ok(a, i)) *a.err_flag = 1;
    }
    const int c = row_cost<MODE>(a, x, plan, s, group);
    mine_cost += (int64_t)c * blocks * row_tiles<MODE>(s, group);
    most = max(most, c);
  }
  auto item = [&](int i) { return MODE != kPlain && known ? s_item[i] : item_of<MODE>(a, x, where, i); };
  int64_t upto = mine_cost;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(~0u, upto, o);
    if (lane >= o) upto += v;
  }
  most = __reduce_max_sync(~0u, most);
  if (lane == 31) s_sum[warp] = upto;
  if (lane == 0) s_most[warp] = most;
  if constexpr (MODE == kShared) {
    malformed = __syncthreads_or(malformed);
    if (blockIdx.x == 0 && threadIdx.x == 0 && !few<MODE>(a, x)) *x.malformed = malformed;
  } else {
    over = __syncthreads_or(over);
  }
  int64_t total = 0, before = upto - mine_cost;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
    most = max(most, s_most[w]);
  }
  const int64_t stretch = stretch_of(plan, total, most);
  const int64_t first_unit = blockIdx.x * stretch, last_unit = min(total, first_unit + stretch);
  if (first_unit < last_unit) {
    if (before <= first_unit && first_unit < before + mine_cost) {  // one thread's run holds it
      int i = run0;
      for (;; ++i) {
        const Item s = item(i);
        const int64_t c = (int64_t)row_cost<MODE>(a, x, plan, s, group) * blocks * row_tiles<MODE>(s, group);
        if (before + c > first_unit) break;
        before += c;
      }
      s_seq = i, s_start = before;
    }
    __syncthreads();
    int seq = s_seq, lo;
    Gap gap;
    int64_t start = s_start;  // where the sequence's first head begins
    Item s = item(seq);
    const int piece_cost = MODE == kPlain ? kPieceCost : plan.piece_cost;
    row_keys<MODE>(a, x, s, group, lo, gap);
    int cost = row_cost<MODE>(a, x, plan, s, group), tiles = row_tiles<MODE>(s, group);
    int sub = (int)quotient(first_unit - start, cost);  // block of heads, tile of rows
    for (;;) {
      const int64_t head_start = start + (int64_t)sub * cost + piece_cost;  // of its first real unit
      if (head_start - piece_cost >= last_unit) break;
      const int units = MODE != kPlain && s.len - gap.skip - lo <= 0 ? 0 : cost - piece_cost;
      const int u0 = (int)max((int64_t)0, first_unit - head_start);
      const int u1 = (int)min((int64_t)units, last_unit - head_start);
      // (a sequence without keys: its zeros are written by the CTA where its cost begins)
      if (u1 > u0 || (units == 0 && head_start - piece_cost >= first_unit)) {
        const int tile = MODE == kShared ? sub % tiles : 0;
        const int kvh = (MODE == kShared ? sub / tiles : sub) * heads;  // the first of the piece's heads
        const int row0 = tile * kRows, rows = MODE == kShared ? min(kRows, s.n * group - row0) : s.n * group;
        const int my_kvh = kvh + (MODE == kPlain ? 0 : warp % heads), slice = MODE == kPlain ? warp : warp / heads;
        const int64_t cta0 = quotient(head_start, stretch),
                      cta1 = units == 0 ? cta0 : quotient(head_start + units - 1, stretch);
        const int parts = (int)(cta1 - cta0) + 1, part = (int)(blockIdx.x - cta0);
        // of the first and the last query
        const int pos0 = MODE != kShared ? s.len - s.n : s.flat ? s.len - 1 : s.len - s.n + row0 / group, pos1 = s.len - 1;
        // along the walk; key_at gives the key
        const int begin = lo + u0 * unit_keys, end = min(s.len - gap.skip, lo + u1 * unit_keys);
        auto key_at = [&](int walk) { return MODE == kSinks && walk >= gap.from ? walk + gap.skip : walk; };
        auto unseen = [&](int j, int p) {
          if (MODE == kShared && j < s.lo) return true;
          return j > p || (a.window > 0 && j <= p - a.window && (MODE != kSinks || j >= x.sinks));
        };

        const int g = lane >> 2, tq = lane & 3;
        uint32_t qf[D / 16][4];
        int row_pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = g + 8 * h, t = (row0 + r) / group;
          row_pos[h] = r >= rows ? -1 : MODE == kShared && s.flat ? pos0 : s.len - s.n + t;
        }

        const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kRowStages * 2 * kTileKeys * D * 2);
        constexpr int kTileBytes = kTileKeys * D * 2;
        const int32_t* table = a.table + (int64_t)max(0, min(s.slot, a.n_slots - 1)) * a.table_stride;
        const int steps = units > 0 ? (end - begin + kTileKeys - 1) / kTileKeys : 0;
        const int mine = steps > slice ? (steps - slice + slices - 1) / slices : 0;
        const int shift = 31 - __clz(a.page_tokens);
        auto page_of = [&](int i) {
          if (i >= mine) return -1;
          const int p = table[key_at(begin + kTileKeys * (slice + slices * i)) >> shift];
          if (p >= 0 && p < a.n_pages) return p;
          if (a.err_flag) *a.err_flag = 1;
          return -1;
        };
        int next_page = page_of(0);
        // the queries of the warp's head come through the last stage, which the keys need last
        const uint32_t q_at = ring + (kRowStages - 1) * 2 * kTileBytes;
        {
          constexpr int kPieces = D / 8, kPer = 32 / kPieces;
          const int c = lane % kPieces;
#pragma unroll
          for (int r0 = 0; r0 < kRows; r0 += kPer) {
            const int r = r0 + lane / kPieces, t = (row0 + r) / group;
            const bool there = r < rows;
            const int64_t at = there ? (int64_t)(s.first + t) * a.q_token_stride +
                                           (int64_t)(my_kvh * group + row0 + r - t * group) * a.q_head_stride + c * 8
                                     : 0;
            cp16(q_at + piece<D>(r, c), static_cast<const T*>(a.q) + at, there);
          }
          cp_commit();
        }
        uint32_t valid = 0;  // bit i % 32: step i's page exists
        auto load = [&](int i) {
          const int page = next_page;
          next_page = page_of(i + 1);
          if (i < mine) valid = (valid & ~(1u << (i & 31))) | ((page >= 0 ? 1u : 0u) << (i & 31));
          if (i < mine && page >= 0) {
            const int walk = begin + kTileKeys * (slice + slices * i), key = key_at(walk);
            const int64_t off = page * a.page_stride + my_kvh * a.head_stride + (key & (a.page_tokens - 1)) * a.row_stride;
            const uint32_t at = ring + (i % kRowStages) * 2 * kTileBytes;
            constexpr int kPieces = D / 8, kPer = 32 / kPieces;  // lanes per row, rows per pass
            const int c = lane % kPieces;
#pragma unroll
            for (int r0 = 0; r0 < kTileKeys; r0 += kPer) {
              const int r = r0 + lane / kPieces;
              // rows past the last key are zeros: whatever the page holds there meets a zero weight
              const bool there = walk + r < end;
              const int64_t o = off + (there ? r : 0) * a.row_stride + c * 8;
              cp16(at + piece<D>(r, c), static_cast<const T*>(a.k_cache) + o, there);
              cp16(at + kTileBytes + piece<D>(r, c), static_cast<const T*>(a.v_cache) + o, there);
            }
          }
          cp_commit();
        };
#pragma unroll
        for (int i = 0; i < kRowStages - 1; ++i) load(i);

        cp_wait<kRowStages - 1>();
        __syncwarp();
        // as A fragments: rows g and g + 8, 16 values of a head per step
#pragma unroll
        for (int k = 0; k < D / 16; ++k) ldsm4(qf[k], q_at + piece<D>(lane & 15, 2 * k + (lane >> 4)));
        __syncwarp();

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
          const int key = key_at(begin + kTileKeys * (slice + slices * i));
          float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];  // keys 0-7: b[0], b[1]; keys 8-15: b[2], b[3]
            ldsm4(b, kt + piece<D>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
            mma16816<T>(sc[0], qf[k], b[0], b[1]);
            mma16816<T>(sc[1], qf[k], b[2], b[3]);
          }
          // element e of sc[n]: row g + 8 (e / 2), key 8 n + 2 tq + e % 2
          const bool whole = key + kTileKeys <= pos0 + 1 &&
                             (a.window == 0 || key > pos1 - a.window || (MODE == kSinks && key + kTileKeys <= x.sinks)) &&
                             (MODE != kShared || key >= s.lo);
          float top[2] = {m[0], m[1]};
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = sc[n][e] * c2;
              if (!whole) {
                const int j = key + 8 * n + 2 * tq + (e & 1), p = row_pos[e >> 1];
                if (unseen(j, p)) v = -INFINITY;
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
          if (!whole) {
            unsigned char* v = smem + (vt - (uint32_t)__cvta_generic_to_shared(smem));
            bool odd = false;
            for (int i = lane; i < kTileKeys * D; i += 32)
              odd |= !isfinite(to_f32(*reinterpret_cast<const T*>(v + i * 2)));
            if (__any_sync(~0u, odd)) {
              for (int j = 0; j < kTileKeys; ++j)
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int col = 8 * n + 2 * tq + (e & 1), p = row_pos[e >> 1];
                    const float f = to_f32(*reinterpret_cast<const T*>(v + piece<D>(j, col / 8) + (col % 8) * 2));
                    if (!isfinite(f) && !unseen(key + j, p)) o[n][e] += f;
                  }
              __syncwarp();
              for (int i = lane; i < kTileKeys * D; i += 32) {
                T* at = reinterpret_cast<T*>(v + i * 2);
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
        }
        const bool joined_here = !(MODE == kShared && known);  // else the joining kernel finds the pieces itself
        if (MODE != kPlain && slices == 1) {
          // The warp has its head to itself: no barrier stands in the walk from piece to piece, and while one waits for
          // its first keys the others compute.
          const int hw = warp;
          __syncwarp();  // every lane is done with the ring
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h, t = (row0 + r) / group, head = my_kvh * group + row0 + r - t * group;
            if (r >= rows) continue;
            const int64_t row = (int64_t)(s.first + t) * a.q_heads + head;
            if (parts > 1 || MODE == kShared) {
              const int64_t at = parts > 1 ? ((2 * (int64_t)blockIdx.x + (part == 0)) * heads + hw) * kRows + r
                                           : (int64_t)(s.flat ? x.own_parts : 0) * a.tokens * a.q_heads + row;
              float* to = (parts > 1 ? plan.o : x.o) + at * D + 2 * tq;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(to + 8 * n) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
              if (tq == 0) (parts > 1 ? plan.ml : x.ml)[at] = make_float2(l[h] == 0.f ? -INFINITY : m[h], l[h]);
            } else {
              T* to = static_cast<T*>(a.out) + (int64_t)(s.first + t) * a.out_token_stride +
                      (int64_t)head * a.out_head_stride + 2 * tq;
              const bool none = l[h] == 0.f;
#pragma unroll
              for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<uint32_t*>(to + 8 * n) =
                    pack2<T>(none ? 0.f : o[n][2 * h] / l[h], none ? 0.f : o[n][2 * h + 1] / l[h]);
              if (a.lse && tq == 0) a.lse[row] = none ? -INFINITY : (m[h] + log2f(l[h])) * kLn2;
            }
          }
          if (parts > 1 && joined_here) {
            __threadfence();
            __syncwarp();
            int last = 0;
            if (lane == 0) {
              int32_t* const done = plan.done + cta0 * heads + hw;
              last = atomicAdd(done, 1) == parts - 1;
              if (last) *done = 0;
            }
            if (__shfl_sync(~0u, last, 0)) {
              __threadfence();
              for (int i = lane; i < rows * (D / 4); i += 32) {
                const int r = i / (D / 4), d = (i - r * (D / 4)) * 4, t = (row0 + r) / group;
                const int head = my_kvh * group + row0 + r - t * group;
                auto slot = [&](int k) { return ((2 * (cta0 + k) + (k == 0)) * heads + hw) * kRows + r; };
                float top = -INFINITY, sum = 0.f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(&plan.ml[slot(k)]).x);
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 8
                for (int k = 0; k < parts; ++k) {
                  const float2 w = __ldcg(&plan.ml[slot(k)]);
                  const float f = ex2(w.x - base);
                  const float4 p = __ldcg(reinterpret_cast<const float4*>(plan.o + slot(k) * D + d));
                  sum = fmaf(w.y, f, sum);
                  v.x = fmaf(p.x, f, v.x), v.y = fmaf(p.y, f, v.y), v.z = fmaf(p.z, f, v.z), v.w = fmaf(p.w, f, v.w);
                }
                if constexpr (MODE == kShared) {
                  const int64_t at = ((int64_t)(s.flat ? x.own_parts : 0) * a.tokens + s.first + t) * a.q_heads + head;
                  *reinterpret_cast<float4*>(x.o + at * D + d) = v;
                  if (d == 0) x.ml[at] = make_float2(sum == 0.f ? -INFINITY : base, sum);
                  continue;
                }
                const bool none = sum == 0.f;
                *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(s.first + t) * a.out_token_stride +
                                          (int64_t)head * a.out_head_stride + d) =
                    make_uint2(pack2<T>(none ? 0.f : v.x / sum, none ? 0.f : v.y / sum),
                               pack2<T>(none ? 0.f : v.z / sum, none ? 0.f : v.w / sum));
                if (a.lse && d == 0)
                  a.lse[(int64_t)(s.first + t) * a.q_heads + head] = none ? -INFINITY : (base + log2f(sum)) * kLn2;
              }
            }
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
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
          // four neighbouring values a thread
          auto put = [&](int hw, int r, int d, float m_all, float l_all, const float4& v) {
            const int t = (row0 + r) / group, head = (kvh + hw) * group + row0 + r - t * group;
            if constexpr (MODE == kShared) {
              const int64_t at = ((int64_t)(s.flat ? x.own_parts : 0) * a.tokens + s.first + t) * a.q_heads + head;
              *reinterpret_cast<float4*>(x.o + at * D + d) = v;
              if (d == 0) x.ml[at] = make_float2(l_all == 0.f ? -INFINITY : m_all, l_all);
              return;
            }
            const bool none = l_all == 0.f;
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(s.first + t) * a.out_token_stride +
                                      (int64_t)head * a.out_head_stride + d) =
                make_uint2(pack2<T>(none ? 0.f : v.x / l_all, none ? 0.f : v.y / l_all),
                           pack2<T>(none ? 0.f : v.z / l_all, none ? 0.f : v.w / l_all));
            if (a.lse && d == 0)
              a.lse[(int64_t)(s.first + t) * a.q_heads + head] = none ? -INFINITY : (m_all + log2f(l_all)) * kLn2;
          };
          auto add = [](float4& v, const float4& w, float f) {
            v.x = fmaf(w.x, f, v.x), v.y = fmaf(w.y, f, v.y), v.z = fmaf(w.z, f, v.z), v.w = fmaf(w.w, f, v.w);
          };
          for (int i = threadIdx.x; i < heads * rows * (D / 4); i += W * 32) {
            const int hr = i / (D / 4), d = (i - hr * (D / 4)) * 4, hw = MODE == kPlain ? 0 : hr / rows, r = hr - hw * rows;
            float top = -INFINITY, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < W; ++w)
              if (MODE == kPlain || w % heads == hw) top = fmaxf(top, s_m[w][r]);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < W; ++w) {
              if (MODE != kPlain && w % heads != hw) continue;
              const float f = ex2(s_m[w][r] - base);
              sum = fmaf(s_l[w][r], f, sum);
              add(v, *reinterpret_cast<const float4*>(so + (w * kRows + r) * D + d), f);
            }
            if (parts == 1) {
              put(hw, r, d, base, sum, v);
            } else {
              const int64_t at = ((2 * (int64_t)blockIdx.x + (part == 0)) * heads + hw) * kRows + r;
              *reinterpret_cast<float4*>(plan.o + at * D + d) = v;
              if (d == 0) plan.ml[at] = make_float2(top, sum);
            }
          }
          if (parts > 1 && joined_here) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
              s_last = atomicAdd(plan.done + cta0, 1) == parts - 1;
              if (s_last) plan.done[cta0] = 0;
            }
            __syncthreads();
            if (s_last) __threadfence();
          }
          if (parts > 1 && joined_here && s_last)
            for (int i = threadIdx.x; i < heads * rows * (D / 4); i += W * 32) {
              const int hr = i / (D / 4), d = (i - hr * (D / 4)) * 4, hw = MODE == kPlain ? 0 : hr / rows, r = hr - hw * rows;
              auto slot = [&](int k) { return ((2 * (cta0 + k) + (k == 0)) * heads + hw) * kRows + r; };
              float top = -INFINITY, sum = 0.f;
              float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
              for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(&plan.ml[slot(k)]).x);
              const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 8
              for (int k = 0; k < parts; ++k) {
                const float2 w = __ldcg(&plan.ml[slot(k)]);
                const float f = ex2(w.x - base);
                sum = fmaf(w.y, f, sum);
                add(v, __ldcg(reinterpret_cast<const float4*>(plan.o + slot(k) * D + d)), f);
              }
              put(hw, r, d, base, sum, v);
            }
          __syncthreads();  // the ring and the shared words are free for the next piece
        }
      }
      if (++sub == blocks * tiles) {
        sub = 0;
        start += (int64_t)cost * blocks * tiles;
        do {
          if (++seq >= items) break;
          s = item(seq);
          row_keys<MODE>(a, x, s, group, lo, gap);
          cost = row_cost<MODE>(a, x, plan, s, group), tiles = row_tiles<MODE>(s, group);
        } while (cost == 0);
        if (seq >= items) break;
      }
    }
  }
  if (MODE == kSinks && blockIdx.x == 0 && a.err_flag)
    for (int i = threadIdx.x; i < a.n_seqs; i += kThreads)
      if (!sequence_ok(a, i)) *a.err_flag = 1;
  if (over)
    for (int i = blockIdx.x; i < a.n_seqs; i += gridDim.x) {
      const Item s = item_of<MODE>(a, x, where, i);
      if (s.n <= kRows / group) continue;
      for (int64_t e = threadIdx.x; e < (int64_t)s.n * a.q_heads * D; e += kThreads) {
        const int64_t row = e / D, t = s.first + row / a.q_heads, head = row % a.q_heads;
        static_cast<T*>(a.out)[t * a.out_token_stride + head * a.out_head_stride + e % D] = from_f32<T>(0.f);
        if (a.lse && e % D == 0) a.lse[t * a.q_heads + head] = -INFINITY;
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
  if (b.window >= most_keys(b)) b.window = 0;
  return b;
}

// Parts of a chunk's keys: one where the (row pair, key head) items fill the
// GPU, else as many as fill it once, each of at least kMinPart keys.  (Cutting
// the last wave of many items in two evens the SMs out, 348 steps on the longest
// instead of 370 for 8192 tokens over 16384 keys, but the parts' traffic and the
// join took more: 814 us against 771.)
template <int MODE>
ChunkPlan chunk_plan(const q4gpu_attn_args& a, const More& x, size_t* bytes) {
  ChunkPlan p{};
  const int64_t group = a.q_heads / a.kv_heads, rows = a.tokens * group;
  if constexpr (MODE == kShared) {
    // a group's queries count together: tiles for its shared keys, and for own keys of long chunks
    p.least = (int)(kMostTiles * kRows / group) + 1, p.parts = 1;
    const int64_t most = a.tokens / p.least;  // items of so many queries
    int64_t tiles = 0;
    if (rows > kMostTiles * kRows) tiles = rows / kPair + std::min<int64_t>(x.n_groups, most);
    if (a.max_q * group > kMostTiles * kRows) tiles += rows / kPair + std::min<int64_t>(a.n_seqs, most);
    p.tiles = (int)std::min<int64_t>(tiles, INT32_MAX);
    // The shared keys get SMs of their own, beside attn_rows_kernel's: half of them, or more where they are most of the
    // keys.  (64 sequences, 8192 shared keys and up to 512 own ones: 29.6 us with half, 33.1 with 65 %, 36 with 35 %, 49.8
    // after one another; 2 groups of 32 x 4 tokens, 4096 and 100 keys: 66.6 with 72 %, 95 with half.)
    const double shared = (double)tiles * std::min(x.max_prefix, a.max_ctx);
    const double own = (double)a.n_seqs * std::max(1, a.max_ctx - x.max_prefix);
    const int sms = (int)(kSms * std::min(0.8, std::max(0.5, shared / (shared + own))));
    if (tiles)
      p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(sms / (tiles * a.kv_heads), a.max_ctx / kMinPart));
    return p;
  }
  if (a.max_q * group <= kRows || a.n_seqs == 0 || a.tokens == 0) {  // nothing for the chunk kernel
    if (bytes) *bytes = 0;
    return p;
  }
  // (a lone sequence of any length is the chunk kernel's: one launch)
  p.least = a.n_seqs == 1 ? 1 : (int)(kRows / group) + 1;
  p.tiles = (int)std::min<int64_t>(a.n_seqs == 1 ? (rows + kPair - 1) / kPair : rows / kPair + a.n_seqs, INT32_MAX);
  const int64_t items = (int64_t)p.tiles * a.kv_heads;
  const int64_t span =
      a.window > 0 ? std::min<int64_t>(a.max_ctx, (int64_t)a.window + kPair + kNTile + x.sinks) : a.max_ctx;
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(kSms / items, span / kMinPart));
  if (bytes) *bytes = p.parts > 1 ? (size_t)p.tiles * a.kv_heads * p.parts * kPair * (8 + (size_t)a.dim * 4) : 0;
  return p;
}

template <int MODE>
RowPlan row_plan(const q4gpu_attn_args& a, const More& x, char* ws, size_t* bytes) {
  RowPlan p{};
  const int64_t seqs = a.n_seqs + x.n_groups;
  p.least_stretch = 6, p.piece_cost = kPieceCost;
  if constexpr (MODE != kPlain) {
    // Several key heads a piece, a warp or a few each, where there are sequences enough: pieces are fewer (64 decodes
    // through a window of 2048 over 1 to 8704 keys: 46 us with one, 38.5 with two, 41 with eight, whose pieces are
    // cut and joined more often; 64 sequences of 1 to 512 own keys beside 8192 shared ones, which another kernel
    // joins: 40.8 with two, 32.2 with eight).
    const int most = MODE == kSinks ? 160 : 32;
    while (2 << p.heads_log <= kRowWarps && a.kv_heads % (2 << p.heads_log) == 0 &&
           seqs * (a.kv_heads >> (p.heads_log + 1)) >= most)
      ++p.heads_log;
    // Where a unit a CTA is all there is, that is how it is cut (one token of 1028 seen keys: 12.0 us, 16.4 in
    // stretches of 6).
    const int64_t unit = (kRowWarps * kTileKeys) >> p.heads_log, blocks = a.kv_heads >> p.heads_log;
    const int64_t shared = MODE == kShared ? std::min(x.max_prefix, a.max_ctx) : 0;
    const int64_t seen = MODE == kSinks ? std::min<int64_t>(a.max_ctx, (int64_t)a.window + a.max_q + x.sinks + 2 * unit)
                                        : a.max_ctx - shared;
    const int64_t all = blocks * (a.n_seqs * ((seen + unit - 1) / unit) + x.n_groups * ((shared + unit - 1) / unit));
    if (all <= kSms) p.piece_cost = 0, p.least_stretch = 1;
  }
  p.unit_log = 31 - __builtin_clz((kRowWarps * kTileKeys) >> p.heads_log);
  const size_t items = (size_t)seqs * (a.kv_heads >> p.heads_log) * (MODE == kShared ? kMostTiles : 1);
  // no CTA without at least one item or least_stretch units of one
  const int unit = (kRowWarps * kTileKeys) >> p.heads_log;
  const int64_t units = ((int64_t)a.max_ctx + unit - 1) / unit + p.piece_cost;
  const int64_t most = (int64_t)items * std::max<int64_t>(1, (units + p.least_stretch - 1) / p.least_stretch + 1);  // (of a stretch's two ends)
  int sms = kSms;
  if (MODE == kShared && (int64_t)a.tokens * (a.q_heads / a.kv_heads) > (int64_t)kMostTiles * kRows * x.n_groups) {
    // groups for the chunk kernel, which runs beside this one
    const ChunkPlan c = chunk_plan<MODE>(a, x, nullptr);
    sms = (int)std::max<int64_t>(kSms / 4, kSms - (int64_t)c.tiles * a.kv_heads * c.parts);
  }
  p.ctas = (int)std::min<int64_t>(most, sms * (a.dim == 64 ? 2 : 1));
  static_assert(kSms * 2 * kRowWarps <= kCounters, "a counter a CTA and head");
  const size_t done = kCounters * sizeof(int32_t), rows = ((size_t)p.ctas * 2 * kRows) << p.heads_log;  // (even)
  if (bytes) *bytes = done + rows * (8 + (size_t)a.dim * 4);
  p.done = reinterpret_cast<int32_t*>(ws);
  p.ml = reinterpret_cast<float2*>(ws + done);
  p.o = reinterpret_cast<float*>(p.ml + rows);
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

template <typename T, int D, int MODE>
int launch(const q4gpu_attn_args& a, const More& x, cudaStream_t s) {
  static unsigned char ready[Q4GPU_MAX_DEVICES];
  size_t rows_bytes;
  const RowPlan few = row_plan<MODE>(a, x, static_cast<char*>(a.workspace), &rows_bytes);
  ChunkPlan plan = chunk_plan<MODE>(a, x, nullptr);
  const bool chunks = plan.tiles > 0;
  if (plan.tiles > 65535) return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: too many query rows");
  // sequences for attn_rows_kernel (with kShared it also looks at what only the device sees)
  const bool short_ones = MODE == kShared || !chunks || plan.least > 1;
  int rc = Q4GPU_OK;
  CUtensorMap kmap, vmap;
  if (chunks) {
    char* ws = static_cast<char*>(a.workspace) + (rows_bytes + 15) / 16 * 16;
    plan.ml = reinterpret_cast<float2*>(ws);
    plan.o = reinterpret_cast<float*>(plan.ml + (size_t)plan.tiles * a.kv_heads * plan.parts * kPair);
    if constexpr (MODE == kShared) plan.o = nullptr, plan.ml = nullptr;
    rc = encode_map(&kmap, a, a.k_cache);
    if (rc == Q4GPU_OK) rc = encode_map(&vmap, a, a.v_cache);
    if (rc == Q4GPU_OK)
      rc = allow_smem(reinterpret_cast<const void*>(attn_chunk_kernel<T, D, MODE>), chunk_smem<D>(), ready);
    if (rc != Q4GPU_OK) return rc;
  }
  if (short_ones) {
    static unsigned char ready[Q4GPU_MAX_DEVICES];
    const auto kernel = attn_rows_kernel<T, D, MODE>;
    rc = allow_smem(reinterpret_cast<const void*>(kernel), row_smem<D>(), ready);
    if (rc == Q4GPU_OK) kernel<<<few.ctas, kRowWarps * 32, row_smem<D>(), s>>>(a, x, few);
    if (rc != Q4GPU_OK) return rc;
  }
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_chunk_kernel<T, D, MODE>, kmap, vmap, a, x, plan);
    if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "attention: launch: %s", cudaGetErrorString(e));
    if (MODE != kShared && plan.parts > 1) attn_join_kernel<T, D, MODE><<<dim3(a.kv_heads, plan.tiles, kPair / 8), 256, 0, s>>>(a, x, plan);
  }
  if constexpr (MODE == kShared) {
    const int64_t rows = (int64_t)a.max_q * a.q_heads;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // it waits for the others itself
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.n_seqs, (unsigned)std::max<int64_t>(1, std::min<int64_t>((rows + 7) / 8, 64)));
    cfg.blockDim = dim3(256);
    cfg.stream = s, cfg.attrs = attr, cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_shared_join_kernel<T, D>, a, x, plan, few);
    if (e != cudaSuccess) return q4gpu_fail(Q4GPU_ERR_CUDA, "attention: launch: %s", cudaGetErrorString(e));
  }
  return q4gpu_check_launch();
}

template <int MODE>
int launch(const q4gpu_attn_args& a, const More& x, cudaStream_t s) {
  if (a.dtype == Q4GPU_F16) return a.dim == 64 ? launch<__half, 64, MODE>(a, x, s) : launch<__half, 128, MODE>(a, x, s);
  return a.dim == 64 ? launch<__nv_bfloat16, 64, MODE>(a, x, s) : launch<__nv_bfloat16, 128, MODE>(a, x, s);
}

// Sinks as the kernels take them: without a window every key is seen anyway.
More settled_sinks(const q4gpu_attn_args& settled, int32_t sinks) {
  More x{};
  x.sinks = settled.window > 0 ? sinks : 0;
  return x;
}

// The workspace behind the few-row kernel's: the two sets of parts and a word.  False: too large to count.
struct SharedRoom {
  size_t ml, o, word, bytes;
};
bool shared_room(const q4gpu_attn_args& a, const More& x, SharedRoom& r, int& own_parts) {
  const ChunkPlan p = chunk_plan<kShared>(a, x, nullptr);
  own_parts = (int64_t)a.max_q * (a.q_heads / a.kv_heads) > kMostTiles * kRows ? p.parts : 1;
  size_t rows_bytes;
  row_plan<kShared>(a, x, nullptr, &rows_bytes);
  const size_t rows = (size_t)(own_parts + p.parts) * a.tokens * a.q_heads;
  r.ml = (rows_bytes + 15) / 16 * 16;
  r.o = r.ml + (rows * sizeof(float2) + 15) / 16 * 16;
  r.word = r.o + rows * a.dim * sizeof(float);
  r.bytes = r.word + 16;
  return p.tiles <= 65535;
}

// The workspace of a call without shared keys: the few-row kernel's, and the chunk kernel's parts behind it.  By the
// plans of the mode that is launched, which lay it out.
template <int MODE>
size_t room_of(const q4gpu_attn_args& a, const More& x) {
  size_t rows, chunks;
  row_plan<MODE>(a, x, nullptr, &rows);
  chunk_plan<MODE>(a, x, &chunks);
  return (rows + 15) / 16 * 16 + chunks;
}

int check_shared(const q4gpu_attn_args* a, const q4gpu_shared_args* sh) {
  if (!sh) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null arguments");
  if (a->window) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: shared keys and a window do not go together");
  if (sh->n_groups < 0 || sh->n_groups > 65535 || sh->max_prefix < 0)
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: %d groups, shared keys up to %d", sh->n_groups, sh->max_prefix);
  return Q4GPU_OK;
}
More settled_groups(const q4gpu_shared_args& sh) {
  More x{};
  x.cu_group = sh.cu_group, x.prefix_lens = sh.prefix_lens, x.n_groups = sh.n_groups, x.max_prefix = sh.max_prefix;
  return x;
}

}  // namespace

extern "C" {

size_t q4gpu_shared_attention_workspace_bytes(const q4gpu_attn_args* a, const q4gpu_shared_args* sh) {
  if (check_sizes(a) != Q4GPU_OK || check_shared(a, sh) != Q4GPU_OK) return 0;
  SharedRoom room;
  int own_parts;
  shared_room(settled(*a), settled_groups(*sh), room, own_parts);
  return room.bytes;
}

int q4gpu_shared_attention(const q4gpu_attn_args* a, const q4gpu_shared_args* sh, void* stream) {
  int rc = check_attn(a);
  if (rc == Q4GPU_OK) rc = check_shared(a, sh);
  if (rc != Q4GPU_OK) return rc;
  if (sh->n_groups > 0 && (!sh->cu_group || !sh->prefix_lens))
    return q4gpu_fail(Q4GPU_ERR_ARG, "attention: null pointer");
  if (a->n_seqs == 0 || a->tokens == 0) return Q4GPU_OK;
  const q4gpu_attn_args b = settled(*a);
  More x = settled_groups(*sh);
  SharedRoom room;
  if (!shared_room(b, x, room, x.own_parts)) return q4gpu_fail(Q4GPU_ERR_SHAPE, "attention: too many query rows");
  if (a->workspace_bytes < room.bytes || !a->workspace)
    return q4gpu_fail(Q4GPU_ERR_WORKSPACE, "attention: needs a workspace of %zu bytes", room.bytes);
  if (!aligned(a->workspace, 16)) return q4gpu_fail(Q4GPU_ERR_ALIGN, "attention: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(a->workspace);
  x.ml = reinterpret_cast<float2*>(ws + room.ml), x.o = reinterpret_cast<float*>(ws + room.o);
  x.malformed = reinterpret_cast<int*>(ws + room.word);
  return launch<kShared>(b, x, as_stream(stream));
}

size_t q4gpu_sink_attention_workspace_bytes(const q4gpu_attn_args* a, int32_t sinks) {
  if (check_sizes(a) != Q4GPU_OK || sinks < 0) return 0;
  const q4gpu_attn_args b = settled(*a);
  const More x = settled_sinks(b, sinks);
  return x.sinks ? room_of<kSinks>(b, x) : room_of<kPlain>(b, x);
}

int q4gpu_sink_attention(const q4gpu_attn_args* a, int32_t sinks, void* stream) {
  const int rc = check_attn(a);
  if (rc != Q4GPU_OK) return rc;
  if (sinks < 0) return q4gpu_fail(Q4GPU_ERR_ARG, "attention: %d sinks", sinks);
  if (a->n_seqs == 0 || a->tokens == 0) return Q4GPU_OK;
  const size_t need = q4gpu_sink_attention_workspace_bytes(a, sinks);
  if (a->workspace_bytes < need || (need && !a->workspace))
    return q4gpu_fail(Q4GPU_ERR_WORKSPACE, "attention: needs a workspace of %zu bytes", need);
  if (!aligned(a->workspace, 16)) return q4gpu_fail(Q4GPU_ERR_ALIGN, "attention: workspace must be 16-byte aligned");
  const q4gpu_attn_args b = settled(*a);
  const More x = settled_sinks(b, sinks);
  return x.sinks ? launch<kSinks>(b, x, as_stream(stream)) : launch<kPlain>(b, x, as_stream(stream));
}

size_t q4gpu_paged_attention_workspace_bytes(const q4gpu_attn_args* a) {
  return q4gpu_sink_attention_workspace_bytes(a, 0);
}
int q4gpu_paged_attention(const q4gpu_attn_args* a, void* stream) { return q4gpu_sink_attention(a, 0, stream); }

}  // extern "C"
