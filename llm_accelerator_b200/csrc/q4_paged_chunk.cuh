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

// Keys that a slot's row of the table can name, and that sums of two places of a walk in 31 bits allow (as many
// different keys of the smallest kind, 256 bytes with their values, are more than the memory holds).
constexpr int kMostKeys = 1 << 30;
__host__ __device__ __forceinline__ int64_t most_keys(const q4gpu_attn_args& a) {
  const int64_t named = (int64_t)a.table_pages * a.page_tokens;
  return named < kMostKeys ? named : kMostKeys;
}

// Which keys a query sees: those up to its own (through a window the last of them), or those and the first few keys of
// the sequence as well, or, in two items of work that are joined afterwards, those that its group of sequences shares
// and its sequence's own.
enum Mode { kPlain, kSinks, kShared };
struct More {  // what the modes need besides the arguments they share
  int sinks;   // kSinks: the first keys that every query sees
  // kShared: group g is sequences cu_group[g] .. cu_group[g + 1] - 1, its first prefix_lens[g] keys are shared
  const int32_t *cu_group, *prefix_lens;
  int n_groups, max_prefix;
  // what a row got from its own keys and from the shared ones: unnormalised sums [set][part][token][q_head][D], with
  // the running maximum (log2 units) and sum; the own set has own_parts parts
  float* o;
  float2* ml;
  int own_parts, *malformed;  // *malformed: cu_q or cu_group does not ascend
};
// A walk over a sequence's keys that leaves out `skip` keys from key `from` on.
struct Gap {
  int from, skip;
};
// Between the sinks, rounded up to whole steps of the walk, and the first key `lo` (a multiple of the step) of a window.
__device__ __forceinline__ Gap gap_before(int lo, int sinks, int step) {
  Gap g;
  g.from = (int)min((int64_t)lo, ((int64_t)sinks + step - 1) & ~(int64_t)(step - 1));
  g.skip = lo - g.from;
  return g;
}

// The lowest n bits of 64 (none where n is negative, all from 64 on).
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }

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

// What a CTA needs to know of an item of work, which is a sequence, or with kShared (in this order) the own keys of a
// sequence or the shared keys of a group.
struct Item {
  int slot, len, first, n;  // cache slot, end of the keys, first query token, query tokens
  int lo;                   // kShared: the first key
  bool flat;                // ... whether every query sees all of them (query t of n stands at len - n + t otherwise)
};
template <int MODE>
__device__ __forceinline__ int item_count(const q4gpu_attn_args& a, const More& x) {
  return a.n_seqs + (MODE == kShared ? x.n_groups : 0);
}
__device__ __forceinline__ int keys_of(const q4gpu_attn_args& a, int slot) {
  return slot >= 0 && slot < a.n_slots ? (int)max((int64_t)0, min((int64_t)a.lens[slot], most_keys(a))) : 0;
}
// The index arrays of a call, in global memory or staged.
struct Where {
  const int32_t *cu_q, *slots, *keys;  // keys (staged): of each sequence's slot
  const int32_t *cu_group, *prefix_lens;
};
// A CTA looks at several of them for each item, one after another: with few sequences it first brings them into shared
// memory, which takes two trips.
constexpr int kStaged = 128;
struct Staged {
  int32_t cu_q[kStaged + 1], slots[kStaged], keys[kStaged], cu_group[kStaged + 1], prefix_lens[kStaged];
};
template <int MODE>
__device__ __forceinline__ bool few(const q4gpu_attn_args& a, const More& x) {
  return MODE != kPlain && a.n_seqs <= kStaged && x.n_groups <= kStaged;
}
// By all threads of a CTA; a barrier has to follow.
template <int MODE>
__device__ __forceinline__ Where where_of(const q4gpu_attn_args& a, const More& x, Staged* s) {
  if (!few<MODE>(a, x)) return Where{a.cu_q, a.seq_ids, nullptr, x.cu_group, x.prefix_lens};
  for (int i = threadIdx.x; i <= a.n_seqs; i += blockDim.x) {
    s->cu_q[i] = a.cu_q[i];
    if (i == a.n_seqs) break;
    const int slot = a.seq_ids ? a.seq_ids[i] : i;
    s->slots[i] = slot, s->keys[i] = keys_of(a, slot);
  }
  if (x.n_groups > 0)
    for (int i = threadIdx.x; i <= x.n_groups; i += blockDim.x) {
      s->cu_group[i] = x.cu_group[i];
      if (i < x.n_groups) s->prefix_lens[i] = x.prefix_lens[i];
    }
  return Where{s->cu_q, s->slots, s->keys, s->cu_group, s->prefix_lens};
}
__device__ __forceinline__ int shared_keys(const q4gpu_attn_args& a, const Where& w, int g) {
  return (int)max((int64_t)0, min((int64_t)w.prefix_lens[g], most_keys(a)));
}
// The group of sequence i, or -1: the last that begins at or before it, if it reaches it.
__device__ __forceinline__ int group_of(const More& x, const Where& w, int i) {
  int g = 0, end = x.n_groups;
  while (g < end) {
    const int mid = (g + end) / 2;
    if (w.cu_group[mid] <= i)
      g = mid + 1;
    else
      end = mid;
  }
  return g > 0 && i < w.cu_group[g] ? g - 1 : -1;
}
template <int MODE>
__device__ __forceinline__ Item item_of(const q4gpu_attn_args& a, const More& x, const Where& w, int i) {
  Item s;
  s.lo = 0, s.flat = false;
  int last = i + 1;
  if (MODE == kShared && i >= a.n_seqs) {
    const int g = i - a.n_seqs;
    s.flat = true;
    i = max(0, min(w.cu_group[g], a.n_seqs)), last = max(i, min(w.cu_group[g + 1], a.n_seqs));
    s.lo = shared_keys(a, w, g);  // (their end, for now)
  }
  s.first = max(0, min(w.cu_q[i], a.tokens));
  s.n = max(0, min(w.cu_q[last], a.tokens) - s.first);
  if (MODE == kShared && i == last) {  // a group without sequences: its first may not be there
    s.slot = -1, s.len = s.lo = s.n = 0;
    return s;
  }
  s.slot = w.slots ? w.slots[i] : i;
  s.len = MODE != kPlain && w.keys ? w.keys[i] : keys_of(a, s.slot);
  if constexpr (MODE == kShared) {
    if (s.flat) {
      s.len = min(s.len, s.lo);
      s.lo = 0;
      if (s.len == 0) s.n = 0;
    } else {
      const int g = group_of(x, w, i);
      s.lo = g < 0 ? 0 : shared_keys(a, w, g);
      // its queries have to stand behind the shared keys (else its rows become zeros)
      if (s.lo > 0 && s.lo > s.len - s.n) s.lo = s.len = 0;
      if (s.n > a.max_q) s.n = 0;  // likewise
    }
  }
  return s;
}

// Row pair of one grid index and its item.
struct ChunkTile : Item {
  int seq, row0, index;
};
// Row pairs of item i (none where it has few rows); keys: about how many one walks.
template <int MODE>
__device__ __forceinline__ int pairs_of(const q4gpu_attn_args& a, const More& x, const Where& w, int i, int group,
                                        int least, ChunkTile& t, int& keys) {
  keys = 0;
  if (i >= item_count<MODE>(a, x)) return 0;
  static_cast<Item&>(t) = item_of<MODE>(a, x, w, i);
  if (t.n < least) return 0;
  keys = a.window > 0 ? min(t.len, a.window) : t.len - t.lo;  // (of sinks there are few)
  return (int)(((int64_t)t.n * group + kPair - 1) / kPair);
}
// The pair of grid row y; seq = -1 where there are fewer.  By one full warp.
// Pairs with many keys come first, so that they do not start when the others
// end: sequences in four classes (at least half, a quarter, an eighth of the most
// keys, the rest), and within a class from its last row pair to its first, as
// later rows see more keys.
template <int MODE>
__device__ __forceinline__ ChunkTile find_tile(const q4gpu_attn_args& a, const More& x, const Where& w, int least,
                                               int y) {
  const int lane = threadIdx.x & 31, group = a.q_heads / a.kv_heads, items = item_count<MODE>(a, x);
  // where no sequence has so many queries only groups have
  const int first = MODE == kShared && a.max_q < least ? a.n_seqs : 0;
  ChunkTile t{}, own{};
  t.seq = -1, t.index = y;
  int most = 0, keys;
  for (int i = first + lane; i < items; i += 32) {
    pairs_of<MODE>(a, x, w, i, group, least, own, keys);
    most = max(most, keys);
  }
  most = __reduce_max_sync(~0u, most);
  auto rank = [&](int k) { return k >= most / 2 ? 0 : k >= most / 4 ? 1 : k >= most / 8 ? 2 : 3; };
  int count[4] = {0, 0, 0, 0};
  for (int i = first + lane; i < items; i += 32) {
    const int n = pairs_of<MODE>(a, x, w, i, group, least, own, keys);
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
  for (int i0 = first; i0 < items; i0 += 32) {
    int mine = pairs_of<MODE>(a, x, w, i0 + lane, group, least, own, keys);
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
      if constexpr (MODE == kShared) t.lo = __shfl_sync(~0u, own.lo, k), t.flat = t.seq >= a.n_seqs;
      return t;
    }
    before += __shfl_sync(~0u, run, 31);
  }
  return t;
}

// The walk of a row pair whose rows see keys lo .. hi - 1, and the sinks before those.
struct Span {
  int begin, end;
  Gap gap;
};
template <int MODE>
__device__ __forceinline__ Span span_of(int lo, int hi, const More& more) {
  const int base = lo & ~(kNTile - 1);
  if constexpr (MODE == kSinks) {
    const Gap gap = gap_before(base, more.sinks, kNTile);
    return Span{0, hi - gap.skip, gap};
  }
  return Span{base, hi, Gap{0, 0}};
}

// attn_rows_kernel's work lies on one axis: item by item, subitem by subitem, in units of keys (q4_paged_attn.cu).
constexpr int kRows = 16;      // rows of one mma.sync tile
constexpr int kTileKeys = 16;  // keys of a warp's step; a page holds whole steps
constexpr int kRowWarps = 8;   // of a CTA, at most
constexpr int kPieceCost = 3;
constexpr int kMostTiles = 4;  // kShared: tiles of 16 rows that an item may have there; more are attn_chunk_kernel's
struct RowPlan {
  int ctas, unit_log;  // log2 of the keys of a unit
  int heads_log;      // log2 of the key heads of a piece, which share the CTA's warps
  int least_stretch;  // units: shorter pieces cost more to join than they save
  int piece_cost;     // units
  float* o;       // [cta][2][head][kRows][D] unnormalised sums: of a piece begun earlier, of one that goes on
  float2* ml;     // [cta][2][head][kRows] their running maximum (log2 units) and sum
  int32_t* done;  // [cta] finished pieces of the item whose first piece goes on from this CTA
};

// Keys that the kernel below walks for item s, from `lo` on; -1: not its
// item (no queries, or more rows than a tile).  With sinks the walk starts
// at key 0 and leaves out `gap.skip` keys from key gap.from on.
template <int MODE>
__device__ __forceinline__ int row_keys(const q4gpu_attn_args& a, const More& x, const Item& s, int group, int& lo,
                                        Gap& gap) {
  lo = 0;
  gap = Gap{0, 0};
  if (s.n == 0 || s.n > (MODE == kShared ? kMostTiles : 1) * kRows / group) return -1;
  if (a.window > 0) lo = first_seen(s.len - s.n, a.window) & ~(kTileKeys - 1);
  if constexpr (MODE == kSinks) {
    gap = gap_before(lo, x.sinks, kTileKeys);
    lo = 0;
  } else if constexpr (MODE == kShared) {
    lo = s.lo & ~(kTileKeys - 1);
  }
  return max(0, s.len - gap.skip - lo);
}
// Cost of one of an item's subitems, which are its tiles of rows for each block of key heads (0: not this kernel's).
template <int MODE>
__device__ __forceinline__ int row_cost(const q4gpu_attn_args& a, const More& x, const RowPlan& plan, const Item& s,
                                        int group) {
  int lo;
  Gap gap;
  const int keys = row_keys<MODE>(a, x, s, group, lo, gap);
  constexpr int kUnit = kRowWarps * kTileKeys;
  if constexpr (MODE == kPlain) return keys < 0 ? 0 : kPieceCost + (keys + kUnit - 1) / kUnit;
  return keys < 0 ? 0 : plan.piece_cost + max(1, (keys + (1 << plan.unit_log) - 1) >> plan.unit_log);
}
template <int MODE>
__device__ __forceinline__ int row_tiles(const Item& s, int group) {
  return MODE == kShared ? (s.n * group + kRows - 1) / kRows : 1;
}

// (32-bit divisions where the numbers allow them)
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  return (x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}
// Units of each CTA of an axis of `total`, whose longest subitem has `most`.
__device__ __forceinline__ int64_t stretch_of(const RowPlan& plan, int64_t total, int most) {
  return max(quotient(total + plan.ctas - 1, plan.ctas), (int64_t)min(most, plan.least_stretch));
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

// ---- exponentials -------------------------------------------------------------
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
// where pages may be missing, then `table` is given).  Rows outside lo .. end
// (but for the first `sinks`) and of missing pages become zeros, and so do infinities and NaNs in the others;
// true if there were any.  Out of line: few steps come here, and the registers it
// takes cost the steps that do not.
template <typename T, int D>
__device__ __noinline__ bool clean_values(unsigned char* v, int key, int lo, int all_lo, int all_hi, int end,
                                          int sinks, const int32_t* table, int shift, int n_pages, int threads) {
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
    bool zero = (k < lo && k >= sinks) || k >= end;
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

// Scores of keys that a row does not see (a 0 among its 64 bits of `seen`) become -infinity where they are, in tensor
// memory.  Few steps come here, and masked in registers, between a step's loads and its maxima, the others were slower as
// well: 8192 tokens over 16384 keys 779 us against 752, through a window of 4096 322 against 312, with 64 sinks besides
// 359 against 345.
__device__ __noinline__ void mask_scores(uint32_t at, uint64_t seen) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float s[32];
    tm_ld32(at + 32 * half, s);
    tm_ld_wait32(s);
    const uint32_t word = (uint32_t)(seen >> (32 * half));
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (!(word & (1u << c))) s[c] = -INFINITY;
    tm_st32(at + 32 * half, reinterpret_cast<const uint32_t*>(s));
  }
  tm_st_wait();
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
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kChunkThreads, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ q4gpu_attn_args a, const __grid_constant__ More more,
                      const __grid_constant__ ChunkPlan plan) {
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
  if constexpr (MODE == kShared) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Where where = where_of<MODE>(a, more, reinterpret_cast<Staged*>(smem));  // (where the queries go later)
  if constexpr (MODE != kPlain) __syncthreads();
  if (warp == 0) {
    const ChunkTile t = find_tile<MODE>(a, more, where, plan.least, blockIdx.y);
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
  const bool flat = MODE == kShared && tile.flat;
  const int pos0 = flat ? len - 1 : len - n + t0, pos1 = flat ? len - 1 : len - n + t1;
  // keys that some row sees, and those that every row sees
  const int item_lo = MODE == kShared ? tile.lo : 0;
  const int lo = a.window > 0 ? first_seen(pos0, a.window) : item_lo, hi = max(0, pos1 + 1);
  const int all_lo = a.window > 0 ? first_seen(pos1, a.window) : item_lo, all_hi = pos0 + 1;
  const Span span = span_of<MODE>(lo, hi, more);
  const int chunk = part_keys(plan, span.end - span.begin);
  const int parts = span.end > span.begin ? (span.end - span.begin + chunk - 1) / chunk : 1;
  if (part >= parts) return wait_before();
  const int begin = span.begin + part * chunk, end = min(span.end, begin + chunk);
  // `begin`, `end` and what lies between are places of the walk; the key that stands there:
  auto key_at = [&](int walk) { return MODE == kSinks && walk >= span.gap.from ? walk + span.gap.skip : walk; };
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
  auto pages_of = [&](int walk, int& id) {  // which pages of the load at `walk` exist; lane p gets page p's number
    const int pages = min(kNTile >> shift, (int)((end - walk + a.page_tokens - 1) >> shift));
    id = lane < pages ? table[(key_at(walk) >> shift) + lane] : -1;
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
  const int64_t walk0 = (int64_t)(MODE == kSinks ? begin : max(begin, lo) & ~(a.page_tokens - 1)) +
                        ((int64_t)threadIdx.x << shift);
  auto page_missing = [&](int64_t walk) {
    if (walk >= end) return false;
    const int key = key_at((int)walk);
    if (MODE == kSinks && key >= more.sinks && key + a.page_tokens <= lo) return false;  // between the sinks and a window
    const int id = table[key >> shift];
    return id < 0 || id >= a.n_pages;
  };
  const bool missing = page_missing(walk0);
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
  for (int64_t w = walk0 + ((int64_t)kChunkThreads << shift); w < end; w += (int64_t)kChunkThreads << shift)
    if (page_missing(w)) gone();
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
        if (j + 1 < steps) next_ok = pages_of(begin + (j + 1) * kNTile, next_id);
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
          if (!(i & 1) && careful(key_at(begin + i * kStep))) {
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
    const int pos = mine ? flat ? len - 1 : len - n + (tile.row0 + r) / group : -1;
    // (not 0: masked scores are -infinity before the factor; with the least number above 0 the exponents of finite
    // scores still vanish, and the weights are equal as a scale of 0 asks)
    const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const uint64_t c22 = pair_of(c2, c2);
    float m = -INFINITY, sum = 0.f;
    bool live = true;
    if (t < tiles) {
      int cleaned = 0;
      for (int i = 0; i < subs; ++i) {
        const int key = key_at(begin + i * kStep), key_end = key + end - (begin + i * kStep);
        if (!(i & 1) && careful(key)) {
          live = __all_sync(~0u, wait_phase(&full[(i | 1) % kStages], ((i | 1) / kStages) & 1));
          if (!live) break;
          if (clean_values<T, D>(smem + (ring - sq) + (i | 1) % kStages * kTile, key, lo, all_lo, all_hi, key_end,
                                 MODE == kSinks ? more.sinks : 0, bad ? table : nullptr, shift, a.n_pages, tiles * kMTile))
            s_odd = 1;
          fence_async();
          __syncwarp();
          if (lane == 0) bar_arrive(&clean[cleaned & 1]);
          ++cleaned;
        }
        live = __all_sync(~0u, wait_phase(&s_full[t][i & 1], (i >> 1) & 1));
        if (!live) break;
        fence_after_sync();
        const uint32_t at = ts + (i & 1) * kStep;
        if (key < all_lo || key + kStep > all_hi || bad) {
          // a bit for each key of the step that the row sees
          const int low = a.window > 0 ? pos - a.window + 1 - key : MODE == kShared ? lo - key : 0;
          uint64_t seen = bits_below(pos - key + 1) & ~bits_below(low);
          if constexpr (MODE == kSinks) seen |= bits_below(min(pos + 1, more.sinks) - key);
          if (bad) {  // pages that exist
            uint64_t there = 0;
            for (int p = key >> shift; p << shift < min(key + kStep, key_end); ++p)
              if (table[p] >= 0 && table[p] < a.n_pages)
                there |= bits_below(((p + 1) << shift) - key) & ~bits_below((p << shift) - key);
            seen &= there;
          }
          mask_scores(at, seen);
        }
        float s[kStep], tops[4] = {m, m, m, m};
        tm_ld32(at, s);
        tm_ld32(at + 32, s + 32);
        tm_ld_wait32(s);
        tm_ld_wait32(s + 32);
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
        int64_t at = (item * plan.parts + part) * kPair + r;
        if constexpr (MODE == kShared)
          at = ((int64_t)((flat ? more.own_parts : 0) + part) * a.tokens + first + q) * a.q_heads + head;
        float* const part_o = MODE == kShared ? more.o : plan.o;
        const bool joined = MODE == kShared || parts > 1;  // by another kernel
        const bool odd = s_odd != 0;
        if (mine && !joined && a.lse)
          a.lse[(int64_t)(first + q) * a.q_heads + head] =
              sum == 0.f ? -INFINITY : (mm + log2f(sum)) * 0.6931471805599453f;
        if (mine && joined) (MODE == kShared ? more.ml : plan.ml)[at] = make_float2(m == -INFINITY ? m : mm, sum);
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
            for (int w = begin; w < end; ++w) {
              const int k = key_at(w);
              if (k >= all_lo && k < all_hi) continue;  // went through the products
              if (MODE == kShared && k < lo) continue;
              if (k > pos || (a.window > 0 && k <= pos - a.window && (MODE != kSinks || k >= more.sinks))) continue;
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
          if (joined) {
            if (mine) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(part_o + at * D + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
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
        if (!joined) {
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
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(256) attn_join_kernel(q4gpu_attn_args a, More more, ChunkPlan plan) {
  __shared__ ChunkTile s_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.x;
  if (warp == 0) {
    const ChunkTile t =
        find_tile<MODE>(a, more, where_of<kPlain>(a, more, nullptr), plan.least, blockIdx.y);
    if (lane == 0) s_tile = t;
  }
  __syncthreads();
  const ChunkTile tile = s_tile;
  if (tile.seq < 0) return;
  const int group = a.q_heads / a.kv_heads;
  const int first = tile.first, n = tile.n, len = tile.len;
  const int rows = (int)min((int64_t)kPair, (int64_t)n * group - tile.row0);
  const int pos0 = len - n + tile.row0 / group, pos1 = len - n + (tile.row0 + rows - 1) / group;
  const Span span = span_of<MODE>(a.window > 0 ? first_seen(pos0, a.window) : 0, max(0, pos1 + 1), more);
  const int chunk = part_keys(plan, span.end - span.begin);
  const int parts = span.end > span.begin ? (span.end - span.begin + chunk - 1) / chunk : 1;
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

// Whether cu_q (i < n_seqs) or cu_group ascends at item i, within what it indexes.
__device__ __forceinline__ bool ascends(const q4gpu_attn_args& a, const Where& w, int i) {
  const bool group = i >= a.n_seqs;
  const int32_t* cu = group ? w.cu_group + (i - a.n_seqs) : w.cu_q + i;
  return cu[0] >= 0 && cu[1] >= cu[0] && cu[1] <= (group ? a.n_seqs : a.tokens);
}
// Whether what only the device sees of a call with shared keys is in range, for a sequence or a group.
__device__ __forceinline__ bool shared_ok(const q4gpu_attn_args& a, const More& x, const Where& w, int i) {
  if (i < a.n_seqs) {
    if (!sequence_ok(a, i)) return false;
    const int n = a.cu_q[i + 1] - a.cu_q[i], g = group_of(x, w, i);
    return n == 0 || g < 0 || w.prefix_lens[g] <= 0 ||
           w.prefix_lens[g] <= a.lens[a.seq_ids ? a.seq_ids[i] : i] - n;
  }
  const int g = i - a.n_seqs, c = w.cu_group[g];
  if (!ascends(a, w, i) || w.prefix_lens[g] < 0) return false;
  if (c == w.cu_group[g + 1] || w.prefix_lens[g] == 0) return true;
  const int s = a.seq_ids ? a.seq_ids[c] : c;  // whose pages hold the shared keys
  return s >= 0 && s < a.n_slots && w.prefix_lens[g] <= keys_of(a, s);
}

// Joins what each row got from its own keys and from the shared ones, part by part in order: one warp a row.  It is
// launched early and works out for itself where the pieces of attn_rows_kernel lie (with many sequences that kernel
// joins them, which takes it a fence, a counter and a trip of its own: 48 sequences of 12 prompts 39.5 us, 32.8 without).
// Bound by the latency of trips to L2, so eight parts are on their way at a time and the places are known before the
// wait (64 sequences over one prompt 32.2 us without either, 30 with both).  Rows of a sequence that the others left out (an unknown slot, queries among the shared
// keys, more than max_q of them) become zeros, and those of all where cu_q or cu_group does not ascend.  It also
// reports what only the device sees.
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_shared_join_kernel(q4gpu_attn_args a, More more, ChunkPlan plan,
                                                                RowPlan rows) {
  constexpr int V = D / 32;  // neighbouring values of a lane
  __shared__ Staged s_staged;
  __shared__ int64_t s_before[2 * kStaged], s_sum[8];
  __shared__ int s_most[8];
  const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Where where = where_of<kShared>(a, more, &s_staged);
  const bool known = few<kShared>(a, more);
  __syncthreads();
  const int group = a.q_heads / a.kv_heads, g = group_of(more, where, i), blocks = a.kv_heads >> rows.heads_log;
  bool malformed = false;
  int64_t stretch = 1;
  if (known) {  // the axis: an item a thread
    static_assert(2 * kStaged <= 256, "an item a thread");
    const int k = threadIdx.x;
    int64_t cost = 0;
    int most = 0;
    if (k < a.n_seqs + more.n_groups) {
      malformed = !ascends(a, where, k);
      const Item s = item_of<kShared>(a, more, where, k);
      most = row_cost<kShared>(a, more, rows, s, group);
      cost = (int64_t)most * blocks * row_tiles<kShared>(s, group);
    }
    int64_t upto = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += v;
    }
    most = __reduce_max_sync(~0u, most);
    if (lane == 31) s_sum[warp] = upto;
    if (lane == 0) s_most[warp] = most;
    malformed = __syncthreads_or(malformed);
    int64_t total = 0, before = upto - cost;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w], most = max(most, s_most[w]);
    }
    s_before[k] = before;
    stretch = max((int64_t)1, stretch_of(rows, total, most));
    __syncthreads();
  }
  if (blockIdx.y == 0 && a.err_flag) {
    if (threadIdx.x == 0 && !shared_ok(a, more, where, i)) *a.err_flag = 1;
    for (int64_t k = i + (int64_t)threadIdx.x * gridDim.x; k < more.n_groups; k += (int64_t)256 * gridDim.x)
      if (!shared_ok(a, more, where, a.n_seqs + (int)k)) *a.err_flag = 1;
  }
  const Item own = item_of<kShared>(a, more, where, i);
  const int all = max(0, min(where.cu_q[i + 1], a.tokens) - own.first);
  Item pre{};
  if (g >= 0) pre = item_of<kShared>(a, more, where, a.n_seqs + g);

  // What a row has of item s: `n` parts, `step` rows of the sums apart from `first` on (of the sets', or of the pieces').
  struct Parts {
    int n;
    bool pieces;
    int64_t first, step;
  };
  auto parts_of = [&](const Item& s, int id, int64_t token, int head, int set0) {
    Parts p{0, false, 0, 0};
    if (s.n == 0) return p;
    const int64_t set = (int64_t)a.tokens * a.q_heads;
    p.first = set0 * set + token * a.q_heads + head, p.step = set;
    const int64_t r = (token - s.first) * group + head % group;  // the row's number in its key head
    if (s.n >= plan.least) {                                     // attn_chunk_kernel's
      const int64_t row0 = r / kPair * kPair;
      const int n = (int)min((int64_t)kPair, (int64_t)s.n * group - row0);
      const int hi = s.flat ? s.len : max(0, s.len - s.n + (int)((row0 + n - 1) / group) + 1);
      const Span span = span_of<kShared>(s.lo, hi, more);
      const int chunk = part_keys(plan, span.end - span.begin);
      p.n = span.end > span.begin ? (span.end - span.begin + chunk - 1) / chunk : 1;
      return p;
    }
    p.n = 1;
    if (!known) return p;
    const int kvh = head / group, heads = 1 << rows.heads_log, tiles = row_tiles<kShared>(s, group);
    const int cost = row_cost<kShared>(a, more, rows, s, group);
    int lo;
    Gap gap;
    if (row_keys<kShared>(a, more, s, group, lo, gap) <= 0) return p;
    const int64_t start = s_before[id] + (int64_t)((kvh >> rows.heads_log) * tiles + (int)(r / kRows)) * cost +
                          rows.piece_cost;  // of its first real unit
    const int64_t cta0 = quotient(start, stretch), cta1 = quotient(start + cost - rows.piece_cost - 1, stretch);
    if (cta0 == cta1) return p;
    p.n = (int)(cta1 - cta0) + 1, p.pieces = true, p.step = 2 * heads * kRows;
    p.first = (2 * cta0 * heads + (kvh & (heads - 1))) * kRows + r % kRows;  // (the first piece lies `heads` rows on)
    return p;
  };
  bool waited = false;
  for (int64_t y = (int64_t)blockIdx.y * 8 + warp; y < (int64_t)all * a.q_heads; y += (int64_t)gridDim.y * 8) {
    const int t = (int)quotient(y, a.q_heads), head = (int)(y - (int64_t)t * a.q_heads);
    const int64_t token = own.first + t, row = token * a.q_heads + head;
    Parts mine = parts_of(own, i, token, head, 0), shared{0, false, 0, 0};
    if (g >= 0) shared = parts_of(pre, a.n_seqs + g, token, head, more.own_parts);
    if (!waited) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // now the parts are there
      if (!known) malformed = *more.malformed != 0;
      waited = true;
    }
    if (malformed || own.n == 0 || own.len == 0) mine.n = shared.n = 0;
    const int parts = mine.n + shared.n;
    auto place = [&](int k, bool& pieces) {
      const bool first = k < mine.n;
      const Parts& p = first ? mine : shared;
      const int j = first ? k : k - mine.n;
      pieces = p.pieces;
      return p.first + j * p.step + (p.pieces && j == 0 ? (int64_t)kRows << rows.heads_log : 0);
    };
    float top = -INFINITY, sum = 0.f, o[V];
#pragma unroll
    for (int c = 0; c < V; ++c) o[c] = 0.f;
    for (int k0 = 0; k0 < parts; k0 += 32) {  // a lane a part
      bool pieces = false;
      const int64_t at = k0 + lane < parts ? place(k0 + lane, pieces) : 0;
      const float2 w = k0 + lane < parts ? (pieces ? rows.ml : more.ml)[at] : make_float2(-INFINITY, 0.f);
      const float* const from = (pieces ? rows.o : more.o) + at * D;
      float most = w.x;
      bool nan = w.x != w.x || w.y != w.y;
#pragma unroll
      for (int s = 16; s; s >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, s));
      nan = __any_sync(~0u, nan);
      const float next = fmaxf(top, most), ref = next == -INFINITY ? 0.f : next;
      const float shrink = top == -INFINITY ? 0.f : ex2(top - ref), f = ex2(w.x - ref);
      sum *= shrink;
#pragma unroll
      for (int c = 0; c < V; ++c) o[c] *= shrink;
      top = next;
      const float part = nan ? w.x * 0.f + w.y : f * w.y;
      float total = part;
#pragma unroll
      for (int s = 16; s; s >>= 1) total += __shfl_xor_sync(~0u, total, s);
      sum += total;
      const int n = min(32, parts - k0);
      for (int k1 = 0; k1 < n; k1 += 8) {  // eight loads on their way at a time
        float v[8][V];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float* p = reinterpret_cast<const float*>(
                               __shfl_sync(~0u, reinterpret_cast<unsigned long long>(from), (k1 + k) & 31)) + lane * V;
          if (k1 + k >= n) {
#pragma unroll
            for (int c = 0; c < V; ++c) v[k][c] = 0.f;
          } else if constexpr (V == 4) {
            const float4 q = *reinterpret_cast<const float4*>(p);
            v[k][0] = q.x, v[k][1] = q.y, v[k][2] = q.z, v[k][3] = q.w;
          } else {
            const float2 q = *reinterpret_cast<const float2*>(p);
            v[k][0] = q.x, v[k][1] = q.y;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float weight = __shfl_sync(~0u, f, (k1 + k) & 31);
          if (k1 + k < n)
#pragma unroll
            for (int c = 0; c < V; ++c) o[c] = fmaf(v[k][c], weight, o[c]);
        }
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(a.out) + token * a.out_token_stride + (int64_t)head * a.out_head_stride + lane * V;
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(out) = pack2<T>(o[0] * inv, o[1] * inv);
    if (a.lse && lane == 0)
      a.lse[row] = sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(sum)) * 0.6931471805599453f;
  }
  // Where no sequence has a row nobody has waited: one CTA does, so that this kernel is not complete before the others
  // and what comes next in the stream may change their inputs.
  if (!waited && blockIdx.x == 0 && blockIdx.y == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace paged
}  // namespace q4
