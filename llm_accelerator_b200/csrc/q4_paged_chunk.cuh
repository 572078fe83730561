// Attention of a chunk of query tokens over a paged cache on the 5th-generation
// tensor cores: the kernel of q4gpu_paged_attention for sequences with more
// than 16 (token, head) rows per key head.
#pragma once
#include "q4_paged.cuh"
#include "q4_umma.cuh"
#include "q4gpu_internal.h"

namespace q4 {
namespace paged {

constexpr int kMTile = 128;             // query rows of one accumulator
constexpr int kPair = 2 * kMTile;       // query rows of a CTA
constexpr int kNTile = 128;             // keys of one load
constexpr int kStep = 64;               // keys of one step
constexpr int kChunkThreads = 12 * 32;  // two softmax warpgroups; a TMA warp, two MMA warps, an idle one

template <int D>
__host__ __device__ constexpr int chunk_stages() { return D == 128 ? 5 : 10; }
template <int D>
__host__ __device__ constexpr int chunk_smem() { return 1024 + (2 * kMTile + chunk_stages<D>() * kNTile) * D * 2; }

struct ChunkPlan {
  int tiles;  // grid of query row pairs over all sequences, an upper bound
  int least;  // sequences with fewer queries are attn_rows_kernel's
  int parts;  // of a pair's keys, each of at least kMinPart
  float* o;    // [pair * kv_heads + head][part][kPair][D] unnormalised sums (parts > 1)
  float2* ml;  // the same rows: running maximum (log2 units) and sum
};
constexpr int kMinPart = 512;
// Keys of one part of `keys`, a multiple of kNTile.
__device__ __forceinline__ int part_keys(const ChunkPlan& plan, int keys) {
  return max(kMinPart, ((keys + plan.parts - 1) / plan.parts + kNTile - 1) & ~(kNTile - 1));
}

// Keys that a slot's row of the table can name.
__device__ __forceinline__ int64_t most_keys(const q4gpu_attn_args& a) { return (int64_t)a.table_pages * a.page_tokens; }

// First key that a query at position pos (negative: before all keys) sees through a window.
__device__ __forceinline__ int first_seen(int pos, int window) { return (int)max((int64_t)0, (int64_t)pos - window + 1); }

// Whether what only the device sees of sequence i is in range: its query tokens, and if it has any its slot and that
// slot's length.  (What is not is cut off or taken as empty; one kernel of a call reports it.)
__device__ __forceinline__ bool sequence_ok(const q4gpu_attn_args& a, int i) {
  const int c0 = a.cu_q[i], c1 = a.cu_q[i + 1];
  if (c0 < 0 || c1 < c0 || c1 > a.tokens || c1 - c0 > a.max_q) return false;
  if (c0 == c1) return true;
  const int s = a.seq_ids ? a.seq_ids[i] : i;
  return s >= 0 && s < a.n_slots && a.lens[s] >= 0 && a.lens[s] <= most_keys(a);
}

// Sequence and row pair of one grid index, and what its CTA needs to know of the
// sequence: first query token, query tokens, cache slot, stored keys.
struct ChunkTile {
  int seq, row0, index, first, n, slot, len;
};
// Row pairs of sequence i (none where it has few rows); keys: about how many one walks.
__device__ __forceinline__ int pairs_of(const q4gpu_attn_args& a, int i, int group, int least, ChunkTile& t, int& keys) {
  keys = 0;
  if (i >= a.n_seqs) return 0;
  t.first = max(0, min(a.cu_q[i], a.tokens));
  t.n = max(0, min(a.cu_q[i + 1], a.tokens) - t.first);
  t.slot = a.seq_ids ? a.seq_ids[i] : i;
  const bool known = t.slot >= 0 && t.slot < a.n_slots;
  t.len = known ? (int)max((int64_t)0, min((int64_t)a.lens[t.slot], most_keys(a))) : 0;
  if (t.n < least) return 0;
  keys = a.window > 0 ? min(t.len, a.window) : t.len;
  return (int)(((int64_t)t.n * group + kPair - 1) / kPair);
}
// The pair of grid row y; seq = -1 where there are fewer.  By one full warp.
// Pairs with many keys come first, so that they do not start when the others
// end: sequences in four classes (at least half, a quarter, an eighth of the most
// keys, the rest), and within a class from its last row pair to its first, as
// later rows see more keys.
__device__ __forceinline__ ChunkTile find_tile(const q4gpu_attn_args& a, int least, int y) {
  const int lane = threadIdx.x & 31, group = a.q_heads / a.kv_heads;
  ChunkTile t{-1, 0, y, 0, 0, 0, 0}, own;
  int most = 0, keys;
  for (int i = lane; i < a.n_seqs; i += 32) {
    pairs_of(a, i, group, least, own, keys);
    most = max(most, keys);
  }
  most = __reduce_max_sync(~0u, most);
  auto rank = [&](int k) { return k >= most / 2 ? 0 : k >= most / 4 ? 1 : k >= most / 8 ? 2 : 3; };
  int count[4] = {0, 0, 0, 0};
  for (int i = lane; i < a.n_seqs; i += 32) {
    const int n = pairs_of(a, i, group, least, own, keys);
#pragma unroll
    for (int c = 0; c < 4; ++c) count[c] += rank(keys) == c ? n : 0;
  }
  int wanted = -1;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int n = __reduce_add_sync(~0u, count[c]);
    if (wanted >= 0) continue;
    if (y < n)
      wanted = c, y = n - 1 - y;
    else
      y -= n;
  }
  if (wanted < 0) return t;
  int before = 0;
  for (int i0 = 0; i0 < a.n_seqs; i0 += 32) {
    int mine = pairs_of(a, i0 + lane, group, least, own, keys);
    if (rank(keys) != wanted) mine = 0;
    int run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(~0u, run, o);
      if (lane >= o) run += v;
    }
    const unsigned hit = __ballot_sync(~0u, before + run > y);
    if (hit) {
      const int k = __ffs(hit) - 1;
      t.seq = i0 + k;
      t.row0 = (y - before - __shfl_sync(~0u, run - mine, k)) * kPair;
      t.first = __shfl_sync(~0u, own.first, k), t.n = __shfl_sync(~0u, own.n, k);
      t.slot = __shfl_sync(~0u, own.slot, k), t.len = __shfl_sync(~0u, own.len, k);
      return t;
    }
    before += __shfl_sync(~0u, run, 31);
  }
  return t;
}

// ---- tensor memory, 32 columns at a time ---------------------------------------
__device__ __forceinline__ void tm_ld32(uint32_t at, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(at));
}
// Waits for the loads above; the values pass through, so no use moves before it.
__device__ __forceinline__ void tm_ld_wait32(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                 "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
                 "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]),
      "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]),
      "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- products --------------------------------------------------------------------
// kind::f16 instruction descriptor: float32 accumulator, both operands f16 or
// bf16, M x N; the B operand K-major, or MN-major (values: keys are its rows).
__host__ __device__ constexpr uint32_t f16_idesc(bool bf16, int M, int N, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// An MN-major tile in 128-byte swizzled lines of 64 values: 8-row groups 1024
// bytes apart (stride), the next 64 columns `chunk` bytes on (leading).
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t chunk) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0)
      : "memory");
}
// Waits for a phase; false after about 0.3 s.  (umma::bar_wait reads the global
// timer after its first miss, which took longer than most waits here.)  A wait
// that lasts sleeps between its tests.
__device__ __forceinline__ bool wait_phase(uint64_t* b, unsigned parity) {
  if (umma::bar_try_wait(b, parity)) return true;
  long long since = 0;
  for (uint32_t it = 1;; ++it) {
    if (umma::bar_try_wait(b, parity)) return true;
    if (it > 16) __nanosleep(40);
    if ((it & 255u) == 0) {
      const long long now = clock64();
      if (!since)
        since = now;
      else if (now - since > 500000000ll)
        return false;
    }
  }
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(umma::smem_addr(b))
      : "memory");
}

// ---- pairs of float32 --------------------------------------------------------
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split_pair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two values on the FMA pipe, for x <= 127.  Range reduction after Cody
// and Waite: x = n + f with n = floor(x) from the low bits of x + 1.5 2^23
// rounded down; 2^f on [0, 1] by the degree-4 polynomial with value 1 at 0 whose
// largest relative error is least (3.0e-6, mean below 1e-8, against 2^-9 of a
// bf16 weight; found by linear programming over 4001 points); n is added to the
// exponent.  x below -127 (a masked score) gives exactly 0.
__device__ __forceinline__ void ex2_pair(uint64_t x2, float& x, float& y) {
  constexpr float kMagic = 12582912.f;
  split_pair(x2, x, y);
  const uint64_t v = pair_of(fmaxf(x, -127.f), fmaxf(y, -127.f));
  uint64_t r, f;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r) : "l"(v), "l"(pair_of(kMagic, kMagic)));
  f = add_pair(r, pair_of(-kMagic, -kMagic));
  f = fma_pair(f, pair_of(-1.f, -1.f), v);
  uint64_t p = fma_pair(f, pair_of(0.013425154611468315f, 0.013425154611468315f),
                        pair_of(0.0522453747689724f, 0.0522453747689724f));
  p = fma_pair(p, f, pair_of(0.24127855896949768f, 0.24127855896949768f));
  p = fma_pair(p, f, pair_of(0.6930451393127441f, 0.6930451393127441f));
  p = fma_pair(p, f, pair_of(1.f, 1.f));
  float a, b, n, m;
  split_pair(p, a, b);
  split_pair(r, n, m);
  x = __uint_as_float(__float_as_uint(a) + (__float_as_uint(n) << 23));
  y = __uint_as_float(__float_as_uint(b) + (__float_as_uint(m) << 23));
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A share of a value tile's cleaning by one thread of `threads`: 16-byte pieces of
// the rows that not every query sees (keys outside all_lo .. all_hi - 1; all rows
// where pages may be missing, then `table` is given).  Rows outside lo .. end and
// of missing pages become zeros, and so do infinities and NaNs in the others;
// true if there were any.  Out of line: few steps come here, and the registers it
// takes cost the steps that do not.
template <typename T, int D>
__device__ __noinline__ bool clean_values(unsigned char* v, int key, int lo, int all_lo, int all_hi, int end,
                                          const int32_t* table, int shift, int n_pages, int threads) {
  constexpr int kPieces = D / 8;
  // an all-ones exponent carries into the bit above it when one is added at its lowest bit
  constexpr bool kBf16 = !__is_same(T, __half);
  constexpr uint32_t kExp = kBf16 ? 0x7f807f80u : 0x7c007c00u, kOne = kBf16 ? 0x00800080u : 0x04000400u;
  const int r0 = table ? kNTile : max(0, min(kNTile, all_lo - key));
  const int r1 = table ? kNTile : max(r0, min(kNTile, all_hi - key));
  bool any = false;
#pragma unroll 4
  for (int x = threadIdx.x; x < (r0 + kNTile - r1) * kPieces; x += threads) {
    const int c = x % kPieces, y = x / kPieces, r = y < r0 ? y : y - r0 + r1, k = key + r;
    uint4* w = reinterpret_cast<uint4*>(v + (c / 8) * (kNTile * 128) + r * 128 + (c & 7) * 16);
    bool zero = k < lo || k >= end;
    if (table && !zero) zero = table[k >> shift] < 0 || table[k >> shift] >= n_pages;
    const uint4 b = *w;
    const uint32_t u[4] = {b.x, b.y, b.z, b.w};
    uint32_t o[4], found = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t high = ((u[i] & kExp) + kOne) & 0x80008000u;  // each half that is not finite
      found |= high;
      o[i] = zero ? 0u : u[i] & ~((high >> 15) * 0xffffu);
    }
    if (zero || (found && (k < all_lo || k >= all_hi))) *w = make_uint4(o[0], o[1], o[2], o[3]);
    any |= found && !zero;
  }
  return any;
}

// One CTA: 256 query rows (row = token * group + head of the group) of one
// sequence and key head against one part of its keys.  Two accumulators of 128
// rows share the keys.  Per step of 64 keys and tile
//   S = Q K^T (shared x shared -> TMEM);  P = exp2(S c - m) -> TMEM, over S;
//   O += P V (TMEM x shared -> TMEM),
// a thread holding one row of S.  A tile has two score buffers, so the scores
// of step i + 1 are there when the softmax of step i ends: from a product's
// issue to its barrier's wake-up take about 400 clocks besides its own 64.  A
// step of both tiles takes about 1930 clocks, 1510 of them products (64-key
// score products 62 clocks per 16 values of a head, as long as 128-key ones).
// One buffer of 128 keys has fewer products (2048 clocks per 128 keys, not
// 3020) but waits for each: 8192 tokens over 16384 keys, heads of 128, 770 us
// against 759 in a burst of ten and 830 against 821 repeated; heads of 64, 720
// against 726.  O is rescaled only when a row's maximum grows by more than 8 (in
// log2): until then P <= 2^8, which 16-bit weights and 32-bit sums hold without
// loss.
template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ q4gpu_attn_args a, const __grid_constant__ ChunkPlan plan) {
  using namespace umma;
  constexpr int kStages = chunk_stages<D>();
  constexpr int kLines = D / 64;                  // 128-byte lines of a head vector
  constexpr uint32_t kLineTile = kNTile * 128;    // bytes of one line of a 128-row tile
  constexpr uint32_t kTile = kLineTile * kLines;  // bytes of a 128-row tile
  constexpr bool kBf16 = !__is_same(T, __half);
  constexpr uint32_t kSCol = 0, kOCol = 2 * kNTile;  // TMEM columns: S0, S1, O0, O1
  extern __shared__ unsigned char raw[];
  unsigned char* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
  __shared__ uint64_t full[kStages], empty[kStages], s_full[2][2], p_full[2][2], o_full[2], clean[2];
  __shared__ uint32_t tmem_slot;
  __shared__ ChunkTile s_tile;
  __shared__ int s_bad, s_odd, s_dead;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x, part = blockIdx.z;
  // One CTA waits for the kernel before (the short sequences') at its end, so that this one is not complete earlier.
  const bool waits = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
  auto wait_before = [&] {
    if (waits) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (warp == 0) {
    const ChunkTile t = find_tile(a, plan.least, blockIdx.y);
    if (lane == 0) s_tile = t, s_bad = s_odd = s_dead = 0;
  }
  if (waits && warp == 11 && plan.least == 1 && a.err_flag)  // no other kernel in this call looks at the sequences
    for (int i = lane; i < a.n_seqs; i += 32)
      if (!sequence_ok(a, i)) *a.err_flag = 1;
  __syncthreads();
  const ChunkTile tile = s_tile;
  if (tile.seq < 0) return wait_before();
  const int group = a.q_heads / a.kv_heads;
  const int first = tile.first, n = tile.n, slot = tile.slot, len = tile.len;
  const int64_t all_rows = (int64_t)n * group;
  const int rows = (int)min((int64_t)kPair, all_rows - tile.row0);
  const int t0 = tile.row0 / group, t1 = (tile.row0 + rows - 1) / group;  // first and last query of the pair
  const int pos0 = len - n + t0, pos1 = len - n + t1;
  // keys that some row sees, and those that every row sees
  const int lo = a.window > 0 ? first_seen(pos0, a.window) : 0, hi = max(0, pos1 + 1);
  const int all_lo = a.window > 0 ? first_seen(pos1, a.window) : 0, all_hi = pos0 + 1;
  const int base = lo & ~(kNTile - 1);
  const int chunk = part_keys(plan, hi - base);
  const int parts = hi > base ? (hi - base + chunk - 1) / chunk : 1;
  if (part >= parts) return wait_before();
  const int begin = base + part * chunk, end = min(hi, begin + chunk);
  const int steps = begin < end ? (end - begin + kNTile - 1) / kNTile : 0;
  const int subs = begin < end ? (end - begin + kStep - 1) / kStep : 0;
  const int tiles = rows > kMTile ? 2 : 1;
  const int32_t* table = a.table + (int64_t)max(0, min(slot, a.n_slots - 1)) * a.table_stride;
  const int shift = 31 - __clz(a.page_tokens);
  const uint32_t sq = smem_addr(smem), ring = sq + 2 * kTile;

  if (warp == 9) tmem_alloc(&tmem_slot, 512);
  if (threadIdx.x == 8 * 32) {
    for (int i = 0; i < kStages; ++i) bar_init(&full[i], 1), bar_init(&empty[i], tiles);
    for (int i = 0; i < 2; ++i) {
      for (int k = 0; k < 2; ++k) bar_init(&s_full[i][k], 1), bar_init(&p_full[i][k], 4);
      bar_init(&o_full[i], 1), bar_init(&clean[i], 4 * tiles);
    }
    bar_init_fence();
  }
  // the first keys are on their way before the queries are
  auto pages_of = [&](int key, int& id) {  // which pages of the load at `key` exist; lane p gets page p's number
    const int pages = min(kNTile >> shift, (int)((end - key + a.page_tokens - 1) >> shift));
    id = lane < pages ? table[(key >> shift) + lane] : -1;
    return __ballot_sync(~0u, id >= 0 && id < a.n_pages);
  };
  auto load = [&](const CUtensorMap* map, uint32_t at, int id, unsigned ok, uint64_t* bar) {
    const uint32_t bytes = (uint32_t)__popc(ok) * a.page_tokens * D * 2;
    if (lane == 0) {
      if (bytes)
        bar_expect_tx(bar, bytes);
      else
        bar_arrive(bar);
    }
    __syncwarp();
    if ((ok >> lane) & 1u) {
#pragma unroll
      for (int c = 0; c < kLines; ++c)
        tma_load4(at + c * kLineTile + lane * a.page_tokens * 128, map, c * 64, 0, a.head_stride ? kvh : 0, id, bar);
    }
  };
  if (warp == 8 && steps > 0) {
    int id;
    const unsigned ok = pages_of(begin, id);
    load(&kmap, ring, id, ok, &full[0]);
  }

  // is any page of the seen keys missing? (looked up here, needed after the queries are on their way; `begin` may lie
  // before the first seen key, whose pages a window has left behind may be gone)
  const int64_t page0 = ((int64_t)max(begin, lo) >> shift) + threadIdx.x;
  const int id0 = page0 << shift < end ? table[page0] : 0;
  const bool missing = id0 < 0 || id0 >= a.n_pages;
  // Row r of the pair is query t0 + (rem0 + r) / group: a product with 2^20 / group, rounded
  // up, is exact for these small numbers.
  const int rem0 = tile.row0 - t0 * group;
  const uint32_t per_group = ((1u << 20) + group - 1) / group;
  // queries into shared memory, 128-byte swizzled lines (rows past the last: zeros)
  for (int x = threadIdx.x; x < tiles * kMTile * (D / 8); x += kChunkThreads) {
    const int r = x / (D / 8), c = x % (D / 8), row = r & (kMTile - 1);
    const bool there = r < rows;
    const int q = there ? rem0 + r : 0, dt = (int)((q * per_group) >> 20), t = t0 + dt, h = q - dt * group;
    cp16(sq + (r / kMTile) * kTile + (c / 8) * kLineTile + row * 128 + (((c & 7) ^ (row & 7)) * 16),
         static_cast<const T*>(a.q) + (int64_t)(first + t) * a.q_token_stride +
             (int64_t)(kvh * group + h) * a.q_head_stride + c * 8,
         there);
  }
  auto gone = [&] {
    s_bad = 1;
    if (a.err_flag) *a.err_flag = 1;
  };
  if (missing) gone();
  for (int64_t p = page0 + kChunkThreads; p << shift < end; p += kChunkThreads)
    if (table[p] < 0 || table[p] >= a.n_pages) gone();
  cp_commit();
  cp_wait<0>();
  if (a.scale < 0.f) {  // a negative scale turns the queries' sign (each thread its own words)
    for (int x = threadIdx.x; x < tiles * kMTile * (D / 8); x += kChunkThreads) {
      const int r = x / (D / 8), c = x % (D / 8), row = r & (kMTile - 1);
      uint4* w = reinterpret_cast<uint4*>(smem + (r / kMTile) * kTile + (c / 8) * kLineTile + row * 128 +
                                          (((c & 7) ^ (row & 7)) * 16));
      w->x ^= 0x80008000u, w->y ^= 0x80008000u, w->z ^= 0x80008000u, w->w ^= 0x80008000u;
    }
  }
  fence_async();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const bool bad = s_bad != 0;
  volatile int* dead = &s_dead;

  // Values of keys that a row does not see meet a zero weight in its product, so
  // they have to be finite.  A tile with rows that not every query of the pair
  // sees, or that are not there, is cleaned by the softmax warps before its
  // product: rows outside lo .. end and of missing pages become zeros; infinities
  // and NaNs in rows that only some queries see become zeros too and are added at
  // the end for the queries that do see them.
  auto careful = [&](int key) { return key < all_lo || key + kNTile > all_hi || bad; };
  // 384 threads x 168 registers at launch = 64,512; a row of scores can use more: 256 x 208 + 128 x 80 = 63,488
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
      // ---- loads: K and V of a step take one ring stage each ----------------------
      int id, next_id, issued = 0;
      unsigned ok = pages_of(begin, id), next_ok = ok;
      bool stop = false;  // the same in every lane: the loads below are by full warps
      for (int j = 0; j < steps && !stop; ++j) {
        const int key = begin + j * kNTile;
        if (j + 1 < steps) next_ok = pages_of(key + kNTile, next_id);
        for (int kind = 0; kind < 2; ++kind) {
          const int use = 2 * j + kind, st = use % kStages;
          if (use >= kStages && !wait_phase(&empty[st], ((use / kStages) - 1) & 1)) *dead = 1;
          stop = __any_sync(~0u, *dead);
          if (stop) break;
          if (use > 0) load(kind ? &vmap : &kmap, ring + st * kTile, id, ok, &full[st]);
          issued = use + 1;
        }
        id = next_id, ok = next_ok;
      }
      // copies in flight end first (they have, unless a wait ran out)
      for (int use = max(0, issued - kStages); use < issued; ++use)
        wait_phase(&full[use % kStages], (use / kStages) & 1);
    } else if (warp >= 9 && warp < 9 + tiles) {
      // ---- products: one warp a tile, together; an elected thread issues ---------------
      // Descriptors and addresses are the same in every lane and stay in uniform
      // registers (issued from a divergent branch each product took twice as long).
      // A warp's barrier tests queue up behind the products it has issued, so each
      // tile has a warp of its own.
      if (subs > 0) {
        constexpr uint32_t qk = f16_idesc(kBf16, kMTile, kStep, false), pv = f16_idesc(kBf16, kMTile, D, true);
        const int t = warp - 9;
        const bool leader = elect_one();
        const uint32_t sc = kSCol + t * 2 * kStep, oc = kOCol + t * D;
        const uint64_t q = sw128_desc(sq) + t * (kTile / 16), k_desc = sw128_desc(ring),
                       v_desc = sw128_mn_desc(ring, kLineTile);
        auto stage_full = [&](int use) { return wait_phase(&full[use % kStages], (use / kStages) & 1); };
        auto scores = [&](int i) {
          const int use = i & ~1, st = use % kStages;
          if (!stage_full(use)) return false;
          fence_after_sync();
          const uint64_t k = k_desc + st * (kTile / 16) + (i & 1) * (kStep * 128 / 16);
          if (leader) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
              const int at = ((x / 4) * kLineTile + (x & 3) * 32) / 16;
              mma_ss(sc + (i & 1) * kStep, q + at, k + at, qk, x > 0);
            }
            mma_commit(&s_full[t][i & 1]);
            if ((i & 1) || i + 1 == subs) mma_commit(&empty[st]);
          }
          return true;
        };
        // all 512 columns are this CTA's, so they start at 0
        bool live = tmem == 0 && scores(0) && (subs == 1 || scores(1));
        int cleaned = 0;
        for (int i = 0; i < subs; ++i) {
          const int use = i | 1, st = use % kStages;
          live = live && stage_full(use);
          if (!(i & 1) && careful(begin + i * kStep)) {
            live = live && wait_phase(&clean[cleaned & 1], (cleaned >> 1) & 1);
            ++cleaned;
          }
          // no lane is a step ahead of another: one that fell behind would wait for a barrier's next phase
          live = __all_sync(~0u, live && wait_phase(&p_full[t][i & 1], (i >> 1) & 1));
          if (!live) break;
          fence_after_sync();
          const uint64_t v = v_desc + st * (kTile / 16) + (i & 1) * (kStep * 128 / 16);
          if (leader) {
#pragma unroll
            for (int x = 0; x < kStep / 16; ++x)
              mma_ts(oc, sc + (i & 1) * kStep + x * 8, v + x * 128, pv, i > 0 || x > 0);
            if ((i & 1) || i + 1 == subs) mma_commit(&empty[st]);
          }
          if (i + 2 < subs)
            live = scores(i + 2);
          else if (leader)
            mma_commit(&s_full[t][i & 1]);  // no scores: it tells that O is complete up to step i
        }
        if (!live) *dead = 1;
        if (leader) mma_commit(&o_full[t]);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax: one row a thread ------------------------------------------------
    const int t = warp >> 2, r = t * kMTile + (threadIdx.x & (kMTile - 1));
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
    const uint32_t ts = tmem + lanes + kSCol + t * 2 * kStep, to = tmem + lanes + kOCol + t * D;
    const bool mine = r < rows;
    const int pos = mine ? len - n + (tile.row0 + r) / group : -1;
    // (not 0: masked scores are -infinity before the factor; with the least number above 0 the exponents of finite
    // scores still vanish, and the weights are equal as a scale of 0 asks)
    const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const uint64_t c22 = pair_of(c2, c2);
    float m = -INFINITY, sum = 0.f;
    bool live = true;
    if (t < tiles) {
      int cleaned = 0;
      for (int i = 0; i < subs; ++i) {
        if (!(i & 1) && careful(begin + i * kStep)) {
          live = __all_sync(~0u, wait_phase(&full[(i | 1) % kStages], ((i | 1) / kStages) & 1));
          if (!live) break;
          if (clean_values<T, D>(smem + (ring - sq) + (i | 1) % kStages * kTile, begin + i * kStep, lo, all_lo, all_hi,
                                 end, bad ? table : nullptr, shift, a.n_pages, tiles * kMTile))
            s_odd = 1;
          fence_async();
          __syncwarp();
          if (lane == 0) bar_arrive(&clean[cleaned & 1]);
          ++cleaned;
        }
        live = __all_sync(~0u, wait_phase(&s_full[t][i & 1], (i >> 1) & 1));
        if (!live) break;
        fence_after_sync();
        const int key = begin + i * kStep;
        const uint32_t at = ts + (i & 1) * kStep;
        float s[kStep], tops[4] = {m, m, m, m};
        tm_ld32(at, s);
        tm_ld32(at + 32, s + 32);
        tm_ld_wait32(s);
        tm_ld_wait32(s + 32);
        if (key < all_lo || key + kStep > all_hi || bad) {
          const int last = pos - key, low = a.window > 0 ? pos - a.window + 1 - key : 0;
          unsigned ok = ~0u;  // pages that exist
          const int in_page = key & (a.page_tokens - 1);  // 64 in the second half of a 128-token page
          if (bad) {
            ok = 0;
            for (int p = key >> shift; p << shift < min(key + kStep, end); ++p)
              ok |= (table[p] >= 0 && table[p] < a.n_pages ? 1u : 0u) << (p - (key >> shift));
          }
#pragma unroll
          for (int c = 0; c < kStep; ++c)
            if (c > last || c < low || !((ok >> ((in_page + c) >> shift)) & 1u)) s[c] = -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < kStep; c += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) tops[k] = max3(tops[k], s[c + 2 * k], s[c + 2 * k + 1]);
        const float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]);
        // The first step sets the reference; later ones move it when a maximum
        // leaves it behind by more than 8 (or is NaN).
        const bool move = i > 0 && !(top <= m) && !((top - m) * c2 <= 8.f);
        if (i == 0) m = top;
        if (__any_sync(~0u, move)) {
          // O has to hold still: its products up to step i - 1 are done when the
          // barrier of step i + 1's scores is through
          live = __all_sync(~0u, wait_phase(&s_full[t][(i + 1) & 1], ((i + 1) >> 1) & 1));
          if (!live) break;
          fence_after_sync();
          const float f = !move ? 1.f : m == -INFINITY ? 0.f : ex2((m - top) * c2);
          if (move) m = top;
          sum *= f;
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tm_ld32(to + c, o);
            tm_ld_wait32(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= f;
            tm_st32(to + c, reinterpret_cast<const uint32_t*>(o));
          }
        }
        // (m - m is 0, or NaN where a score was infinite or NaN: the whole row becomes NaN, as it should)
        const float off = m == -INFINITY ? 0.f : fmaf(-m, c2, m - m);
        const uint64_t off2 = pair_of(off, off);
        uint64_t add[2] = {0, 0};
        uint32_t p[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          float x, y;
          const uint64_t e = fma_pair(pair_of(s[2 * k], s[2 * k + 1]), c22, off2);
          if (k % 4 == 1) {  // a quarter on the FMA pipe: the exponential unit takes 8 clocks a warp
            ex2_pair(e, x, y);
          } else {
            split_pair(e, x, y);
            x = ex2(x), y = ex2(y);
          }
          add[k & 1] = add_pair(add[k & 1], pair_of(x, y));
          p[k] = pack2<T>(x, y);  // weights in the cache's type for the tensor cores; their sum is not rounded
        }
        tm_st32(at, p);
        tm_st_wait();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) bar_arrive(&p_full[t][i & 1]);
        float x, y;
        split_pair(add_pair(add[0], add[1]), x, y);
        sum += x + y;
      }
      if (subs > 0) live = live && wait_phase(&o_full[t], 0);
      live = __all_sync(~0u, live) && !*dead;
      if (!live && lane == 0) {
        *dead = 1;
        if (a.err_flag) *a.err_flag = 2;
      }
      if (live) {
        fence_after_sync();
        const int dt = (int)(((rem0 + r) * per_group) >> 20), q = t0 + dt, head = kvh * group + rem0 + r - dt * group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum, mm = m == -INFINITY ? 0.f : m * c2;
        const int64_t item = (int64_t)tile.index * a.kv_heads + kvh;
        const int64_t at = (item * plan.parts + part) * kPair + r;
        const bool odd = s_odd != 0;
        if (mine && parts == 1 && a.lse)
          a.lse[(int64_t)(first + q) * a.q_heads + head] =
              sum == 0.f ? -INFINITY : (mm + log2f(sum)) * 0.6931471805599453f;
        if (mine && parts > 1) plan.ml[at] = make_float2(m == -INFINITY ? m : mm, sum);
        // The row goes through shared memory, where its queries were, so that whole rows are stored together.
        unsigned char* stage = smem + t * kTile;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          if (subs > 0) {
            __syncwarp();  // rows took their own ways below
            tm_ld32(to + c, o);
            tm_ld_wait32(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (odd && mine) {  // the infinities and NaNs that were kept out of the products
            for (int k = begin; k < end; ++k) {
              if (k >= all_lo && k < all_hi) continue;  // went through the products
              if (k > pos || (a.window > 0 && k <= pos - a.window)) continue;
              const int id = table[k >> shift];
              if (id < 0 || id >= a.n_pages) continue;
              const T* v = static_cast<const T*>(a.v_cache) + id * a.page_stride + kvh * a.head_stride +
                           (k & (a.page_tokens - 1)) * a.row_stride + c;
              for (int i = 0; i < 32; ++i) {
                const float x = to_f32(v[i]);
                if (!isfinite(x)) {
#pragma unroll
                  for (int e = 0; e < 32; ++e)
                    if (e == i) o[e] += x;
                }
              }
            }
          }
          if (parts > 1) {
            if (mine) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(plan.o + at * D + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          } else {
            const int row = r & (kMTile - 1);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= inv;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(stage + (c / 64) * kLineTile + row * 128 +
                                        ((((c + i) / 8 & 7) ^ (row & 7)) * 16)) = pack8<T>(o + i);
          }
        }
        if (parts == 1) {
          __syncwarp();
          constexpr int kPieces = D / 8, kTogether = 32 / kPieces;  // 16-byte pieces of a row, rows at a time
          const int c = lane % kPieces, row0 = (warp & 3) * 32;
#pragma unroll 4
          for (int i = 0; i < 32; i += kTogether) {
            const int row = row0 + i + lane / kPieces, x = t * kMTile + row;
            if (x >= rows) continue;
            const int d = (int)(((rem0 + x) * per_group) >> 20), h = kvh * group + rem0 + x - d * group;
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t)(first + t0 + d) * a.out_token_stride +
                                      (int64_t)h * a.out_head_stride + c * 8) =
                *reinterpret_cast<const uint4*>(stage + (c / 8) * kLineTile + row * 128 + (((c & 7) ^ (row & 7)) * 16));
          }
        }
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (*dead && warp == 9 && subs > 0)  // after a wait that ran out: products in flight end first
    for (int i = 0; i < tiles; ++i) wait_phase(&o_full[i], 0);
  if (warp == 9) {
    __syncwarp();
    fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
  wait_before();
}

// Joins the parts of each row, in order: one warp a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(q4gpu_attn_args a, ChunkPlan plan) {
  __shared__ ChunkTile s_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.x;
  if (warp == 0) {
    const ChunkTile t = find_tile(a, plan.least, blockIdx.y);
    if (lane == 0) s_tile = t;
  }
  __syncthreads();
  const ChunkTile tile = s_tile;
  if (tile.seq < 0) return;
  const int group = a.q_heads / a.kv_heads;
  const int first = tile.first, n = tile.n, len = tile.len;
  const int rows = (int)min((int64_t)kPair, (int64_t)n * group - tile.row0);
  const int pos0 = len - n + tile.row0 / group, pos1 = len - n + (tile.row0 + rows - 1) / group;
  const int lo = a.window > 0 ? first_seen(pos0, a.window) : 0, hi = max(0, pos1 + 1), base = lo & ~(kNTile - 1);
  const int chunk = part_keys(plan, hi - base);
  const int parts = hi > base ? (hi - base + chunk - 1) / chunk : 1;
  if (parts == 1) return;
  const int r = blockIdx.z * 8 + warp;
  if (r >= rows) return;
  const int64_t at = ((int64_t)tile.index * a.kv_heads + kvh) * plan.parts * kPair + r;
  float top = -INFINITY, sum = 0.f, o[D / 32];
  for (int k = 0; k < parts; ++k) top = fmaxf(top, plan.ml[at + (int64_t)k * kPair].x);
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) o[c] = 0.f;
  for (int k = 0; k < parts; ++k) {
    const float2 w = plan.ml[at + (int64_t)k * kPair];
    const float f = ex2(w.x - ref);
    sum = fmaf(w.y, f, sum);
    const float* p = plan.o + (at + (int64_t)k * kPair) * D + lane;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = fmaf(p[c * 32], f, o[c]);
  }
  const int t = (tile.row0 + r) / group, head = kvh * group + tile.row0 + r - t * group;
  T* out = static_cast<T*>(a.out) + (int64_t)(first + t) * a.out_token_stride + (int64_t)head * a.out_head_stride;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) out[c * 32 + lane] = from_f32<T>(sum == 0.f ? 0.f : o[c] / sum);
  if (a.lse && lane == 0)
    a.lse[(int64_t)(first + t) * a.q_heads + head] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace paged
}  // namespace q4
