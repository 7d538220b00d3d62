// Attention over the paged cache with a mask per row (b200_paged_attn_tree): trees of drafted tokens, beams that share a prompt.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),  over the tokens j that the row sees: those in front of ctx_lens[t], and ctx_lens[t] + i for each
//   bit i of its mask.
//
// Two launches.  The main kernel, one CTA an SM: every CTA makes the step's plan for itself: rows -> runs of one sequence -> items of up to two tiles of 128 (row, head) pairs of a kv
// head; the list of (item, kv head, tile of 64 tokens) is cut into equal shares, one a CTA, which walks its own on tcgen05,
//   S = Q K^T (M = 128 pairs, N = 64 tokens), O += P V (N = 128),
// scores, weights and O in tensor memory, keys and values by TMA through a ring of eight tiles.  An item of two tiles of pairs has a group of four softmax warps for each, and a warp
// that issues its MMAs; one of a single tile lets the two groups take its key tiles in turn, each with a maximum, a sum and an O of its own, which are put together at its end.  Items
// that a cut goes through leave fp32 sums, which the second launch joins in the order of the cut: the result has the same bits every time.
// A tile that lies in front of every row's context is seen whole; in the others a thread (a pair) makes 64 bits of what it sees from its context and mask, and the values that
// are no numbers are taken out of the tile, since 0 x NaN would reach every row; rows that see them get them back at the end.
//
// Roundings: weights go to the tensor cores as a bf16 high and a bf16 low term, 16 bits together, so that a result is as far from the formula's as its one rounding to bf16 makes it
// (relative error 0.0017 over all; with the high term alone 0.0024, and a tenth faster with two tiles of pairs).  All else is fp32.
//
// Times on a B200, caches in HBM, 8 kv heads of 128 (its copy rate 6.56 TB/s, its bf16 rate 1670 TFLOP/s):
//   8 nodes of a sequence of 600 tokens, 32 heads       15 us   latency: start and plan 4, walk and epilogue 4, launches and join 7
//   64 nodes, 32 000 tokens, 32 heads                   55 us   131 MB: 2.4 TB/s; two tiles of pairs
//   32 x up to 25 nodes, 4 000 tokens, 32 heads        109 us   437 MB: 4.0 TB/s
//   4 x 256 nodes, 6 000 tokens, 40 heads              160 us   tensor cores 64 % of their cycles; two tiles of pairs
//   16 x 6 beams, 2 500 tokens, 64 heads, blocks of 16  55 us   133 MB: 2.4 TB/s (blocks of 128: 49)
// What bounds a step of the walk: with one tile of pairs 1330 cycles, which is the rate that keys and values arrive at; with two 1980, of which the MMAs take 1800 (scores read 6 KB of
// shared memory for 32 cycles of products, 48 cycles; weights have two terms).  Without products and softmax the cases take 8, 32, 82, 96 and 39 us.  64 tokens to a tile leave
// room in tensor memory for two tiles' scores of both groups beside O: the next scores are there when a softmax ends.
#include <algorithm>
#include <type_traits>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr int kMostWords = 32, kTreeThreads = 384, kTreeKeys = 64, kTreeSlots = 8;
constexpr int kTrQChunk = 128 * 128;            // [128 pairs][64 columns] bf16
constexpr int kTrChunk = kTreeKeys * 128;       // [64 keys][64 columns] bf16
constexpr int kTrTile = 2 * kTrChunk;
constexpr int kTrStage = 8 * 2048;              // output staging: 2 KiB per softmax warp
constexpr int kTrBad = 64;                      // tiles of an item for which it is known which keys' values are no numbers
// Items whose marks of such values are kept.  Of two tiles of pairs, a group may be two items with key tiles ahead of the other: the queries of item i + 2 wait for both groups' last scores of
// item i + 1, which, if it has one or two key tiles, are issued before any of its weights, while the other group may still be at the end of item i.  Not three: its last scores of item i + 2 come
// behind its weights of item i + 1, thus behind the end of item i
constexpr int kTrMarks = 3;
constexpr int kTrPart = kHeadDim + 2;           // floats of a pair in a part: sums, their maximum (of the products q . k), the denominator
constexpr int kTreeTable = 48;                  // units of a CTA in shared memory
constexpr int kMostRows = 4096;                 // of a step: the plan's lists fit where the tiles come to lie
constexpr int kMostTokens = 0x7fffffff - 4096;  // of a block table: places of a mask's last bit, and of tiles that are looked up ahead, are ints

// rows [row0, row0 + nrows) of one sequence; clear, end: tokens that all of them see, up to the last one that any sees
struct TreeItem {
  int row0, nrows, seq, clear, end;
};
// a CTA's walk over an item's tiles [tile0, tile1) of a kv head; parts > 1: other CTAs have the rest, each leaves its sums in a slot
struct alignas(16) TreeWork {
  TreeItem rows;
  int kvh, tile0, tile1, parts, slot, pad[2];
};

struct TreeParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t ldq, n_blocks;
  const int32_t *block_table, *row_to_seq, *ctx_lens;
  const uint32_t* masks;
  __nv_bfloat16* out;
  int64_t ldo;
  int bt_stride, words, T, hq, hkv, block_size;
  float scale;
  // workspace
  TreeWork* list;        // [item x kv head + CTA] the units of CTAs that have more than kTreeTable
  Kv8Cut* cuts;          // [CTA] its last item, where further CTAs have parts of it
  // [CTA][2]: of an item that began in an earlier CTA, of one that goes on in the next.  [32 x 4 columns][pairs][4], then [pairs][maximum, denominator]: neighbouring lanes own
  // neighbouring pairs (a row to a lane touches 32 lines with every store)
  float* part;
  int pairs;             // a multiple of 32
  uint32_t* status;
};

__host__ __device__ __forceinline__ int64_t tree_tokens(const TreeParams& p) { return (int64_t)p.bt_stride * p.block_size; }
__device__ __forceinline__ int tree_ctx(const TreeParams& p, int row) { return (int)min((int64_t)max(__ldg(p.ctx_lens + row), 0), tree_tokens(p)); }

constexpr int kTrSmem = 1024 + 4 * kTrQChunk + kTreeSlots * kTrTile + kTrStage + 2 * 128 * 8 + kTrMarks * kTrBad * 16 + (2 * kTreeSlots + 16) * 8 + 32 + kTreeTable * (int)sizeof(TreeWork) + 320;
static_assert(5 * kMostRows * 4 <= kTreeSlots * kTrTile, "the plan's lists");
static_assert(kTrSmem <= 232448, "shared memory");

// ---- plan -----------------------------------------------------------------------------------------------------------------------------
// Every CTA makes the step's items and finds its own share of them: 1 to 2 us for small steps, where a launch before this one took 6 and lists in global memory two more.  It reads all rows'
// contexts and masks: 4 096 rows without a token to see take 26 us in all with one mask word, 90 with 32 (8 rows 8 and 9).
//
// Units, an item's walk for a kv head, lie one after another on a line of costs, a unit's first tile at its front, tile t at gap + t x its cost behind that; CTA k has the
// tiles in [k share, (k + 1) share).  A share is no less than the widest distance of neighbouring tiles, so that every CTA between a unit's first and last tile has one of its tiles.
// Costs in halves of a key tile with one tile of pairs: with one, with two, and of an item's start and end (one tile of pairs 1300 cycles, two 2000).  Where units are few, they
// start at a CTA's share each (which costs a CTA a unit at most): a CTA with the end of one and the start of another would be 5 000 cycles later than the others.
constexpr int kCostOne = 2, kCostTwo = 3, kCostItem = 4, kFewUnits = kNumSMs / 4;

struct PlanShared {
  int starts[kTreeThreads / 32], costs[2][kTreeThreads / 32], counts[kTreeThreads / 32], first, units;
  Kv8Cut cut;
};
static_assert(sizeof(PlanShared) <= 320, "shared memory");

// Exclusive scan over the CTA, in two halves with a barrier between them: several go through one barrier, and a scan's shared memory is used once
template <typename F>
__device__ __forceinline__ int scan_warp(int x, F op, int* sh) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) >= o) x = op(x, u);
  }
  if ((threadIdx.x & 31) == 31) sh[threadIdx.x >> 5] = x;
  return __shfl_up_sync(0xffffffffu, x, 1);
}
template <typename F>
__device__ __forceinline__ int scan_cta(int left, int none, F op, const int* sh, int& all) {
  constexpr int kWarps = kTreeThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int t = lane < kWarps ? sh[lane] : none;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t = op(t, u);
  }
  all = __shfl_sync(0xffffffffu, t, kWarps - 1);
  const int before = __shfl_sync(0xffffffffu, t, max(warp - 1, 0));
  return op(warp ? before : none, lane ? left : none);
}

// the CTA's units -> table or, where there are more than it holds, p.list; returns their number, and the place of the first in p.list (-1: in the table).  Costs of all units are below
// 2^31 (tree_launch)
__device__ __forceinline__ int2 tree_plan(const TreeParams& p, int R, int cta, int* scratch, PlanShared* sh, TreeWork* table) {
  int *const ctx = scratch, *const end = scratch + kMostRows;   // of rows
  int *const clear_of = end + kMostRows, *const end_of = clear_of + kMostRows, *const count_of = end_of + kMostRows;   // of the item that starts with a row (count 0: none does)
  const int tid = threadIdx.x, lane = tid & 31, each_rows = (p.T + kTreeThreads - 1) / kTreeThreads, ra = min(p.T, tid * each_rows), rb = min(p.T, ra + each_rows);
  const int tokens = (int)tree_tokens(p);
  auto seq_of = [&](int r) { return p.row_to_seq ? __ldg(p.row_to_seq + r) : r; };
  auto most = [](int a, int b) { return max(a, b); };
  auto plus = [](int a, int b) { return a + b; };
  if (tid == 0) sh->first = 0x7fffffff, sh->units = 0, sh->cut = {0, 0, 0, 0};
  int start = -1;   // the last row here that starts a run of one sequence
#pragma unroll 1
  for (int r = ra; r < rb; ++r) {
    const int mine = seq_of(r), before = r > 0 ? seq_of(r - 1) : mine;
    int c = __ldg(p.ctx_lens + r), e = -1;
    const uint32_t* m = p.masks + (int64_t)r * p.words;
#pragma unroll 1
    for (int w = 0; w < p.words; w += 8) {
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = w + j < p.words ? __ldg(m + w + j) : 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x[j]) e = 32 * (w + j) + 31 - __clz(x[j]);
    }
    c = min(max(c, 0), tokens);
    ctx[r] = c, end[r] = min(c + e + 1, tokens);   // (tokens and a mask's bits: below 2^31 together)
    clear_of[r] = 0x7fffffff, end_of[r] = 0, count_of[r] = 0;
    if (r == 0 || mine != before) start = r;
  }
  int all;
  const int left = scan_warp(start, most, sh->starts);
  __syncthreads();
  int run = scan_cta(left, -1, most, sh->starts, all);
#pragma unroll 1
  for (int k = 0; k < each_rows; ++k) {
    const int r = ra + k;
    const bool in = r < rb;
    int r0 = -1, c = 0x7fffffff, e = 0;
    if (in) {
      if (each_rows == 1 ? start >= 0 : r == 0 || seq_of(r) != seq_of(r - 1)) run = r;
      r0 = r - (r - run) % (2 * R);   // its item's first row
      c = ctx[r], e = end[r];
    }
    if (__all_sync(0xffffffffu, r0 == __shfl_sync(0xffffffffu, r0, 0) || !in)) {   // a warp's rows are one item's
      c = __reduce_min_sync(0xffffffffu, c);
      e = __reduce_max_sync(0xffffffffu, e);
      const int n = __reduce_max_sync(0xffffffffu, in ? r - r0 + 1 : 0);
      if (lane == 0 && in) atomicMin(clear_of + r0, c), atomicMax(end_of + r0, e), atomicMax(count_of + r0, n);
    } else if (in) {
      atomicMin(clear_of + r0, c), atomicMax(end_of + r0, e), atomicMax(count_of + r0, r - r0 + 1);
    }
  }
  __syncthreads();
  auto tiles_of = [&](int r) { return (end_of[r] + kTreeKeys - 1) / kTreeKeys; };
  auto each_of = [&](int r) { return count_of[r] > R ? kCostTwo : kCostOne; };
  int cost = 0, items = 0, n_items, total;
#pragma unroll 1
  for (int r = ra; r < rb; ++r)
    if (count_of[r] > 0) cost += kCostItem + max(tiles_of(r), 1) * each_of(r), ++items;
  const int left_cost = scan_warp(cost, plus, sh->costs[0]), left_items = scan_warp(items, plus, sh->counts);
  __syncthreads();
  int mine = scan_cta(left_cost, 0, plus, sh->costs[0], total);
  const int item0 = scan_cta(left_items, 0, plus, sh->counts, n_items), n_units = n_items * p.hkv;
  const bool few = n_units <= kFewUnits;
  const int gap = few ? 0 : kCostItem;
  total *= p.hkv, mine *= p.hkv;
  int share = max(gap + (p.T > R ? kCostTwo : kCostOne), (total + kNumSMs - 1) / kNumSMs);
  auto whole_of = [&](int r) {
    const int c = gap + max(tiles_of(r), 1) * each_of(r);
    return few ? (c + share - 1) / share * share : c;
  };
  if (few) {
    total -= n_units * kCostItem;
    share = max(2 * kCostOne, (total + kNumSMs - n_units - 1) / (kNumSMs - n_units));   // (two groups of softmax warps: two key tiles at least)
    if (n_items > 1) {   // (the only one is at 0)
      cost = 0;
#pragma unroll 1
      for (int r = ra; r < rb; ++r)
        if (count_of[r] > 0) cost += whole_of(r) * p.hkv;
      const int left2 = scan_warp(cost, plus, sh->costs[1]);
      __syncthreads();
      mine = scan_cta(left2, 0, plus, sh->costs[1], total);
    }
  }
  const int lo = cta * share, hi = lo + share;
#pragma unroll 1
  for (int pass = 0;; ++pass) {   // the CTA's units: into the table, and once more, into the list, if they are too many
    int front = mine, item = item0;
#pragma unroll 1
    for (int r = ra; r < rb && front < hi; ++r) {
      if (count_of[r] == 0) continue;
      const int nt = tiles_of(r), each = each_of(r), behind = nt > 1 ? gap + (nt - 1) * each : 0, whole = whole_of(r);   // behind: of the last tile
      auto first_tile = [&](int x) {   // the first one, but for tile 0, at or behind this place of the unit's line
        const int y = x - gap;
        return y <= each ? 1 : min(nt, each == kCostTwo ? (y + kCostTwo - 1) / kCostTwo : (y + kCostOne - 1) / kCostOne);
      };
      int u = item++ * p.hkv;
      const int next = front + whole * p.hkv, skip = front < lo ? min(p.hkv, (lo - front) / whole) : 0;   // heads that end before the share
      front += skip * whole, u += skip;
#pragma unroll 1
      for (int h = skip; h < p.hkv && front < hi; ++h, front += whole, ++u) {
        const int last = front + behind;
        if (last < lo) continue;
        TreeWork w;
        w.rows = {r, count_of[r], seq_of(r), clear_of[r], end_of[r]};
        w.kvh = h;
        w.tile0 = front < lo ? first_tile(lo - front) : 0;
        w.tile1 = last < hi ? nt : first_tile(hi - front);
        w.parts = 1, w.slot = 0;
        if (front < lo || last >= hi) {
          const int back = front < lo ? (lo - front + share - 1) / share : 0, ahead = last >= hi ? (last - lo) / share : 0;   // CTAs before, behind
          w.parts = back + 1 + ahead;
          w.slot = 2 * cta + (back == 0);
          if (back == 0) sh->cut = {r, count_of[r], h, w.parts};
        }
        if (pass == 0) {
          const int place = atomicAdd(&sh->units, 1);
          if (place < kTreeTable) table[place] = w;
          atomicMin(&sh->first, u);
        } else {
          p.list[u + cta] = w;
        }
      }
      front = next;
    }
    __syncthreads();
    const int units = sh->units;
    if (units <= kTreeTable) return make_int2(units, -1);
    if (pass) return make_int2(units, sh->first + cta);
  }
}

// ---- the walk ---------------------------------------------------------------------------------------------------------------------------
struct TreeRow {   // what a pair sees
  const uint32_t* mask;
  int ctx, words, end;
  bool alive;
};
// of 64 tokens from k0 on, as bits
__device__ __forceinline__ void tree_bits(const TreeRow& r, int k0, uint32_t (&bits)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = k0 + 32 * h - r.ctx, left = r.end - k0 - 32 * h;   // place in the tail; tokens in front of the end
    uint32_t b;
    if (at <= -32) b = 0xffffffffu;
    else if (at < 0) b = (r.words > 0 ? __ldg(r.mask) << -at : 0u) | ((1u << -at) - 1u);
    else {
      const int w = at >> 5;
      b = __funnelshift_r(w < r.words ? __ldg(r.mask + w) : 0u, w + 1 < r.words ? __ldg(r.mask + w + 1) : 0u, at & 31);
    }
    if (left < 32) b &= left <= 0 ? 0u : (1u << left) - 1u;
    bits[h] = r.alive ? b : 0u;
  }
}

// Values that are no numbers, back into 32 sums of a pair (columns c..): those that were taken out of a tile, and in front of it infinities, whose products with weights' low
// terms of zero are not what the formula has (weights are above zero: the sum of such values is the result)
__device__ __noinline__ void tree_repair(const TreeParams& p, const TreeWork& w, const TreeRow& r, const uint32_t (*bad)[4], bool taken_out, float* o, int c) {
  const int first = max(w.tile0, w.rows.clear / kTreeKeys);   // the first tile that not all rows see
  auto add = [&](int key, float* to) {
    const int64_t blk = __ldg(p.block_table + (int64_t)w.rows.seq * p.bt_stride + key / p.block_size);
    if (blk < 0 || blk >= p.n_blocks) return;
    const __nv_bfloat16* v = p.v + ((blk * p.hkv + w.kvh) * p.block_size + key % p.block_size) * kHeadDim + c;
#pragma unroll 1
    for (int d = 0; d < 32; ++d) {
      const float x = __bfloat162float(v[d]);
      if (!(x - x == 0.f)) to[d] += x;
    }
  };
  bool nan = false;
#pragma unroll 1
  for (int d = 0; d < 32; ++d) nan |= o[d] != o[d];
  if (nan) {
    float s[32];
#pragma unroll 1
    for (int d = 0; d < 32; ++d) s[d] = 0.f;
    const int to = min(first, w.tile1) * kTreeKeys;
#pragma unroll 1
    for (int key = w.tile0 * kTreeKeys; key < to; ++key) add(key, s);
#pragma unroll 1
    for (int d = 0; d < 32; ++d)
      if (o[d] != o[d] && s[d] != 0.f) o[d] = s[d];
  }
  if (!taken_out) return;
#pragma unroll 1
  for (int t = first; t < w.tile1; ++t) {
    uint32_t bits[2];
    tree_bits(r, t * kTreeKeys, bits);
#pragma unroll 1
    for (int j = 0; j < kTreeKeys; ++j) {
      const bool known = t - first < kTrBad;
      if ((bits[j >> 5] >> (j & 31) & 1) && (!known || (bad[t - first][j >> 4] >> (2 * (j & 15)) & 3))) add(t * kTreeKeys + j, o);
    }
  }
}

__global__ void __launch_bounds__(kTreeThreads, 1)
attn_tree_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
  unsigned char* qs = smem;                        // two tiles of [2][128 pairs][64]
  unsigned char* ring = qs + 4 * kTrQChunk;        // [kTreeSlots][2][64 keys][64]: key and value tiles in turn
  unsigned char* ostage = ring + kTreeSlots * kTrTile;
  float2* exchange = reinterpret_cast<float2*>(ostage + kTrStage);                   // [group][pair] maximum, sum
  uint32_t(*bad_keys)[4] = reinterpret_cast<uint32_t(*)[4]>(exchange + 2 * 128);    // [item % kTrMarks][tile][16 keys]: two bits a key
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(bad_keys + kTrMarks * kTrBad);
  uint64_t* kv_free = kv_full + kTreeSlots;
  uint64_t* s_full = kv_free + kTreeSlots;         // [group][2] the scores of its even / odd key tile are there
  uint64_t* p_ready = s_full + 4;                  // [group][2] their weights are
  uint64_t* o_full = p_ready + 4;                  // [group][2] their second product has finished
  uint64_t* q_ready = o_full + 4;
  uint64_t* q_free = q_ready + 1;
  uint64_t* last = q_free + 1;                     // [group] the MMAs in flight when a wait ran out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last + 2);   // and, behind it, the mark of a wait that ran out
  int* taken_item = reinterpret_cast<int*>(tmem_slot + 2);       // [item % kTrMarks] the last one (counted from 1) with values that were taken out of a tile
  TreeWork* table = reinterpret_cast<TreeWork*>((reinterpret_cast<uintptr_t>(taken_item + kTrMarks) + 15) & ~(uintptr_t)15);
  PlanShared* plan = reinterpret_cast<PlanShared*>(table + kTreeTable);
  const Waits mbar_wait(tmem_slot + 1, p.status);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kTreeSlots; ++s) {
      mbar_init(kv_full + s, 1);
      mbar_init(kv_free + s, 2);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(p_ready + s, 4);
      mbar_init(o_full + s, 1);
    }
    mbar_init(q_ready, 1);
    mbar_init(q_free, 2);
    mbar_init(last, 1);
    mbar_init(last + 1, 1);
    tmem_slot[1] = 0;
    for (int s = 0; s < kTrMarks; ++s) taken_item[s] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int G = p.hq / p.hkv, R = 128 / G;
  pdl_wait();
  pdl_launch_dependents();
  const int2 units = tree_plan(p, R, cta, reinterpret_cast<int*>(ring), plan, table);
  fence_async_smem();   // (the plan's lists lie where tiles come)
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;   // per group 256 columns: scores of even, odd key tiles, O
  int unit = 0;
  auto next_work = [&](TreeWork& w) {
    if (unit >= units.x) return false;
    w = units.y < 0 ? table[unit] : p.list[units.y + unit];   // (written by this CTA)
    ++unit;
    return true;
  };

  if (warp == 8) {
    // ===== TMA: key tile, value tile, key tile, ... =====
    const bool issuer = elect_one();
    if (issuer) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    const int box = min(p.block_size, kTreeKeys), boxes = kTreeKeys / box, ahead = 32 / boxes;   // rows of a box; boxes of a tile; tiles whose rows are looked up at once
    const int none = (int)(p.n_blocks * p.hkv * p.block_size);   // behind the cache: zeros
    int slot = 0, row = 0;
    uint32_t ph = 1;
    bool stop = false;
    TreeWork w;
    while (!stop && next_work(w)) {
      const int32_t* bt = p.block_table + (int64_t)w.rows.seq * p.bt_stride;
      for (int i = w.tile0; i < w.tile1 && !(stop = mbar_wait.stop()); ++i) {
        const int k = (i - w.tile0) % ahead;
        if (k == 0) {   // lane: the row of box lane % boxes of tile i + lane / boxes
          const int tok = (i + lane / boxes) * kTreeKeys + lane % boxes * box, b = tok / p.block_size;
          const int blk = b < p.bt_stride && i + lane / boxes < w.tile1 ? __ldg(bt + b) : -1;
          row = blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + w.kvh) * p.block_size + (tok - b * p.block_size) : none;
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          mbar_wait(kv_free + slot, ph);
          if (issuer) mbar_expect_tx(kv_full + slot, kTrTile);
          __syncwarp();
          const int from = __shfl_sync(0xffffffffu, row, k * boxes + (lane >> 1) % boxes);
          if (lane < 2 * boxes)   // a lane a box and half of its columns
            tma_load_2d(ring + slot * kTrTile + (lane & 1) * kTrChunk + (lane >> 1) * box * 128, kv ? &map_v : &map_k, (lane & 1) * 64, from, kv_full + slot);
          __syncwarp();
          if (++slot == kTreeSlots) slot = 0, ph ^= 1;
        }
      }
    }
    if (mbar_wait.stop())   // the loads in flight: a slot's last one filled it in this round of the ring or in the one before
      for (int s = 0; s < kTreeSlots; ++s) mbar_wait.drain(kv_full + s, s < slot ? ph ^ 1 : ph);
  } else if (warp == 9 || warp == 11) {
    // ===== MMA, a warp for each group of softmax warps: its next key tile's scores, then this one's second product (one warp for both has its hands full: waits, commits and
    // the issue of 32 MMAs are as long as what it issues).  The whole warp walks the loop; bounds and addresses that come from memory are broadcast, so that they are uniform to the
    // compiler =====
    const int x = __shfl_sync(0xffffffffu, warp == 11 ? 1 : 0, 0);
    const uint32_t one = elect_one() ? 1u : 0u, tm = __shfl_sync(0xffffffffu, tmem, 0) + x * 256;
    const uint64_t desc_k = make_desc(smem_u32(ring), 16, 1024), desc_v = make_desc(smem_u32(ring), kTrChunk, 1024);
    const uint32_t id_s = idesc_bf16(kTreeKeys, 0), id_o = idesc_bf16(kHeadDim, 1);
    uint64_t *const s_done = s_full + 2 * x, *const weights = p_ready + 2 * x, *const o_done = o_full + 2 * x;
    uint32_t at_ring = 0, n = 0;   // places of the ring used up by the items before; key tiles of the group so far
    int active = 0;
    TreeWork w;
    while (__shfl_sync(0xffffffffu, next_work(w), 0)) {
      const int nt = __shfl_sync(0xffffffffu, w.tile1 - w.tile0, 0), two = __shfl_sync(0xffffffffu, w.rows.nrows > R ? 1 : 0, 0);
      if (nt <= 0) continue;
      // both tiles of pairs: every key tile, by either warp; one: every other one
      const int step = two ? 1 : 2, first = two ? 0 : x;
      const uint64_t desc_q = make_desc(smem_u32(qs + (two ? x : 0) * 2 * kTrQChunk), 16, 1024);
      auto arrived = [&](uint32_t place) {
        mbar_wait(kv_full + (place & (kTreeSlots - 1)), (place / kTreeSlots) & 1);
        fence_after();
        return place & (kTreeSlots - 1);
      };
      auto done_with = [&](uint32_t slot) {   // (two arrivals)
        if (!two && one) mbar_arrive(kv_free + slot);
        __syncwarp();
        commit(one, kv_free + slot);
      };
      auto scores = [&](int i, uint32_t nx) {   // of key tile i: places 2 i and 2 i + 1 of the item's part of the ring
        const uint32_t slot = arrived(at_ring + 2 * i);
        const uint64_t db = desc_k + (uint64_t)((slot * kTrTile) >> 4);
        const uint32_t d = tm + (nx & 1) * kTreeKeys;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          mma_ss(one, d, desc_q + ((j >> 2) * kTrQChunk + (j & 3) * 32) / 16, db + ((j >> 2) * kTrChunk + (j & 3) * 32) / 16, id_s, j ? 1u : 0u);
        commit(one, s_done + (nx & 1));
        done_with(slot);
        if (i + step >= nt) commit(one, q_free);   // the group's last scores are on their way
      };
      mbar_wait(q_ready, active & 1);
      if (first < nt) scores(first, n);
      else if (one) mbar_arrive(q_free);
      __syncwarp();
      for (int i = first; i < nt; i += step, ++n) {
        if (i + step < nt) scores(i + step, n + 1);
        const uint32_t slot = arrived(at_ring + 2 * i + 1);
        const uint64_t dv = desc_v + (uint64_t)((slot * kTrTile) >> 4);
        mbar_wait(weights + (n & 1), (n >> 1) & 1);
        fence_after();
        const uint32_t pa = tm + (n & 1) * kTreeKeys, d = tm + 128, more = i > first ? 1u : 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // 16 keys per step: 8 columns of weights, 16 further those of the second term
          mma_ts(one, d, pa + (j >> 1) * 32 + (j & 1) * 8, dv + (uint64_t)((j * 2048) >> 4), id_o, j ? 1u : more);
          mma_ts(one, d, pa + (j >> 1) * 32 + (j & 1) * 8 + 16, dv + (uint64_t)((j * 2048) >> 4), id_o, 1u);
        }
        commit(one, o_done + (n & 1));
        done_with(slot);
      }
      at_ring += 2 * nt;
      ++active;
    }
    if (mbar_wait.stop()) {
      commit(one, last + x);
      mbar_wait.drain(last + x, 0);
    }
  } else if (warp == 10) {
    // ===== queries -> the A operands: R rows of a kv head's G heads are R G rows of an operand (those behind them are never looked at) =====
    const bool issuer = elect_one();
    int active = 0;
    TreeWork w;
    if (lane == 0) p.cuts[cta] = plan->cut;
    while (next_work(w)) {
      if (w.tile1 <= w.tile0) continue;
      const int tiles = w.rows.nrows > R ? 2 : 1;
      if (active > 0) mbar_wait(q_free, (active - 1) & 1);
      if (mbar_wait.stop()) break;
      if (issuer) {
        mbar_expect_tx(q_ready, tiles * 2 * R * G * 128);
        for (int e = 0; e < 2 * tiles; ++e) tma_load_3d(qs + e * kTrQChunk, &map_q, (e & 1) * 64, w.kvh * G, w.rows.row0 + (e >> 1) * R, q_ready);
      }
      __syncwarp();
      ++active;
    }
    if (mbar_wait.stop() && active > 0) mbar_wait.drain(q_ready, (active - 1) & 1);
  } else if (warp < 8) {
    // ===== softmax and output: a thread owns a pair, of tile x of the item's, or with its fellow in the other group of the only one =====
    const int x = warp >> 2, quad = warp & 3, m = quad * 32 + lane;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16), own = base + x * 256;
    const int r = m / G, g = m % G;
    const float sc2 = p.scale * 1.4426950408889634f;   // scores in the log2 domain
    int n = 0, done = 0, item = 0, cleaned = 0;   // key tiles of this group so far; of all items before; items with key tiles; tiles cleaned by group 0 for both
    TreeWork w;
    while (next_work(w)) {
      if (w.tile1 > w.tile0) ++item;   // (nothing holds the groups together in the others, nor is anything marked)
      const int marks = item % kTrMarks;
      uint32_t(*const bad)[4] = bad_keys + marks * kTrBad;
      const bool two = w.rows.nrows > R;
      const int row = (two ? x * R : 0) + r, t = w.rows.row0 + row;
      const bool alive = r < R && row < w.rows.nrows, live = __any_sync(0xffffffffu, alive);   // a warp without a pair hands over whatever there is: its rows are never looked at
      const TreeRow see = {p.masks + (int64_t)t * p.words, alive ? tree_ctx(p, t) : 0, alive ? p.words : 0, w.rows.end, alive};
      const int masked = max(w.tile0, w.rows.clear / kTreeKeys);   // the first tile that not all rows see
      float mu = -INFINITY, l = 0.f;
      const int n0 = n;
      for (int i = w.tile0 + (two ? 0 : x); i < w.tile1; i += two ? 1 : 2, ++n) {
        mbar_wait(s_full + 2 * x + (n & 1), (n >> 1) & 1);
        fence_after();
        if (live) {
          const uint32_t s_addr = own + (n & 1) * kTreeKeys;
          uint32_t s[64];
          ld32(s_addr, s);
          ld32(s_addr + 32, s + 32);
          ld_wait<64>(s);
          if (i >= masked) {
            uint32_t bits[2];
            tree_bits(see, i * kTreeKeys, bits);
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (!(bits[j >> 5] >> (j & 31) & 1)) s[j] = 0xff800000u;   // -inf
          }
          const float mx = max64(s);
          const bool jump = alive && (mx - mu) * sc2 > 8.f;   // also the first live key (mu = -inf)
          if (__any_sync(0xffffffffu, jump)) {
            const float mn = jump ? mx : mu, f = jump && mu != -INFINITY ? exp2_fast((mu - mn) * sc2) : 1.f;
            if (n > n0 && __any_sync(0xffffffffu, f != 1.f)) {
              mbar_wait(o_full + 2 * x + ((n - 1) & 1), ((n - 1) >> 1) & 1);
              fence_after();
#pragma unroll 1
              for (int c = 0; c < kHeadDim; c += 16) {
                uint32_t o[16];
                ld16(own + 128 + c, o);
                ld_wait<16>(o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                st16(own + 128 + c, o);
              }
            }
            l *= f;
            mu = mn;
          }
          // exponents as (score - maximum) x scale: a product less a rounded one would be off by 2^-24 of either, which is more than the exponent itself where scores are large
          const uint64_t minus = f2::both(mu > -INFINITY ? -mu : 0.f), unit = f2::both(sc2);
          uint64_t sum2[2] = {0, 0};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint64_t e = f2::mul(f2::add(f2::pack(__uint_as_float(s[c * 32 + 2 * j]), __uint_as_float(s[c * 32 + 2 * j + 1])), minus), unit);
              const float p0 = exp2_fast(f2::lo(e)), p1 = exp2_fast(f2::hi(e));
              // the high term truncated, the rest rounded
              sum2[j & 1] = f2::add(sum2[j & 1], f2::pack(p0, p1));
              pk[j] = pack_bf16(p0, p1);
              const uint32_t h0 = pk[j] << 16, h1 = pk[j] & 0xffff0000u;
              const uint64_t rest = f2::add(f2::pack(p0, p1), f2::pack(-__uint_as_float(h0), -__uint_as_float(h1)));
              pk[16 + j] = pack_bf16(f2::lo(rest), f2::hi(rest));
            }
            st32(s_addr + c * 32, pk);
          }
          l += f2::sum(sum2[0]) + f2::sum(sum2[1]);
        }
        if (i >= masked && !(two && x)) {
          // 0 x NaN = NaN: what is no number leaves the value tile (two threads a key), everything behind the end does
          const int v_at = 2 * (done + i - w.tile0) + 1, vs = v_at % kTreeSlots, key = m >> 1;
          mbar_wait(kv_full + vs, (v_at / kTreeSlots) & 1);
          uint4* const vb = reinterpret_cast<uint4*>(ring + vs * kTrTile + (m & 1) * kTrChunk + key * 128);
          const bool behind = i * kTreeKeys + key >= w.rows.end;
          uint32_t found = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint4* const at16 = vb + ((k + key) & 7);
            uint4 v = *at16;
            uint32_t* const e = reinterpret_cast<uint32_t*>(&v);
            uint32_t no[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) no[q] = ((e[q] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;   // exponents of ones alone
            const uint32_t any = no[0] | no[1] | no[2] | no[3];
            if (behind || any) {
#pragma unroll
              for (int q = 0; q < 4; ++q) e[q] = behind ? 0u : e[q] & ~((no[q] >> 15) * 0xffffu);
              *at16 = v;
            }
            found |= any;
          }
          const uint32_t keys = __ballot_sync(0xffffffffu, found != 0 && !behind);
          if (lane == 0) {
            if (i - masked < kTrBad) bad[i - masked][quad] = keys;
            if (keys) reinterpret_cast<volatile int*>(taken_item)[marks] = item;
          }
          fence_async_smem();
        }
        if (two && i >= masked) {   // group 1's product waits for the clean values too (group 0 is at most three key tiles ahead: the ring)
          if (x) asm volatile("bar.sync %0, 256;" ::"r"(3 + (cleaned & 3)) : "memory");
          else asm volatile("bar.arrive %0, 256;" ::"r"(3 + (cleaned & 3)) : "memory");
          ++cleaned;
        }
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 2 * x + (n & 1));
      }
      done += w.tile1 - w.tile0;
      const bool any = n > n0;
      if (any) {
        mbar_wait(o_full + 2 * x + ((n - 1) & 1), ((n - 1) >> 1) & 1);
        fence_after();
      }
      // O of this group, or of both, times what brings them to one maximum
      float f_own = 1.f, f_other = 0.f;
      bool other = false;
      if (!two) {
        exchange[x * 128 + m] = make_float2(mu, l);
        fence_before();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        fence_after();
        const float2 o = exchange[(x ^ 1) * 128 + m];
        other = w.tile1 - w.tile0 > (x ? 0 : 1);
        const float mn = fmaxf(mu, o.x);
        f_own = mu == mn ? 1.f : exp2_fast((mu - mn) * sc2), f_other = o.x == mn ? 1.f : exp2_fast((o.x - mn) * sc2);
        l = l * f_own + o.y * f_other;
        mu = mn;
      }
      const bool taken = w.tile1 > w.tile0 && reinterpret_cast<volatile int*>(taken_item)[marks] == item;
      const int c0 = two ? 0 : x * 64, c1 = two ? kHeadDim : c0 + 64;
      const float inv = w.parts > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float4* const part = reinterpret_cast<float4*>(p.part + (int64_t)w.slot * p.pairs * kTrPart) + row * G + g;
      if (w.parts > 1 && alive && c0 == 0) reinterpret_cast<float2*>(p.part + (int64_t)w.slot * p.pairs * kTrPart + (int64_t)p.pairs * kHeadDim)[row * G + g] = make_float2(mu, l);
      unsigned char* const st = ostage + warp * 2048;
#pragma unroll 1
      for (int c = live ? c0 : c1; c < c1; c += 32) {
        uint32_t o[32];
        if (any) {
          ld32(own + 128 + c, o);
          ld_wait<32>(o);
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = any ? o[j] : 0u;
        if (other) {
          uint32_t o2[32];
          ld32(base + (x ^ 1) * 256 + 128 + c, o2);
          ld_wait<32>(o2);
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f_own + __uint_as_float(o2[j]) * f_other);
        }
        bool nan = false;
#pragma unroll
        for (int j = 0; j < 32; ++j) nan |= __uint_as_float(o[j]) != __uint_as_float(o[j]);
        if (alive && (taken || nan) && l == l) {
          float fix[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) fix[j] = __uint_as_float(o[j]);
          tree_repair(p, w, see, bad, taken, fix, c);
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(fix[j]);
        }
        __syncwarp();
        if (w.parts > 1) {
          if (alive) {
#pragma unroll
            for (int k = 0; k < 8; ++k) part[(c / 4 + k) * p.pairs] = *reinterpret_cast<const float4*>(o + 4 * k);
          }
        } else {
          // 32 columns at a time through shared memory: a row's 64 bytes leave from four neighbouring lanes
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = pack_bf16(__uint_as_float(o[8 * k + 2 * j]) * inv, __uint_as_float(o[8 * k + 2 * j + 1]) * inv);
            *reinterpret_cast<uint4*>(st + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int rr = k * 8 + (lane >> 2), mm = quad * 32 + rr, row2 = (two ? x * R : 0) + mm / G, col = c + (lane & 3) * 8;
            const uint4 v = *reinterpret_cast<const uint4*>(st + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
            if (mm / G < R && row2 < w.rows.nrows) *reinterpret_cast<uint4*>(p.out + (int64_t)(w.rows.row0 + row2) * p.ldo + (int64_t)(w.kvh * G + mm % G) * kHeadDim + col) = v;
          }
          __syncwarp();
        }
      }
      fence_before();
      // both groups have read either's O before one of them hands over the next item's first weights (whose product restarts O); a group of its own: the count of p_ready does it
      if (!two) asm volatile("bar.sync 2, 256;" ::: "memory");
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// ---- parts -> out -----------------------------------------------------------------------------------------------------------------------
// A job is 32 pairs of an item and eight columns: sum of a_i 2^(m_i - m) / sum of l_i 2^(m_i - m) over its parts, in their order.  Bound by latency, rounds of loads, for which four CTAs
// an SM have the warps (one: 4 x 256 rows over 6000 tokens 192 us in all, four 164).  Where there are fewer jobs than warps, two, four or eight warps share a job's parts (a
// tree of 30 nodes over 17 000 tokens, 4 heads over one, whose only item has 136 parts: 23 us in all, 65 with a warp a job; eight of 600 tokens, 32 over 8, 14.6 and 16.1; each part's loads of both rounds at once 15.4)
constexpr int kJoinThreads = 256, kJoinColumns = 8, kJoinCtas = 4;

// sums += a part's times what brings them to the maximum of all.  Weights are above zero: what is no number stays, however little of it fp32 has (0 x inf would make a NaN of an infinity)
__device__ __forceinline__ void join_part(float (&a)[8], const float (&x)[8], float f) {
  if (f > 0.f || f != f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] += x[j] * f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] += x[j] - x[j] == 0.f ? 0.f : x[j];
  }
}

__global__ void __launch_bounds__(kJoinThreads, kJoinCtas) tree_join_kernel(const __grid_constant__ TreeParams p) {
  __shared__ int front[kJoinThreads + 1], sh[kJoinThreads / 32];
  __shared__ Kv8Cut cuts[kNumSMs];
  __shared__ float sums[10][kJoinThreads];   // maximum, denominator, columns
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = p.hq / p.hkv;
  int n = 0;
  if (tid < kNumSMs) {
    const Kv8Cut cut = p.cuts[tid];
    cuts[tid] = cut;
    n = cut.parts < 2 ? 0 : (cut.nrows * G + 31) / 32 * (kHeadDim / kJoinColumns);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, n, o);
    if (lane >= o) n += u;
  }
  if (lane == 31) sh[warp] = n;
  __syncthreads();
  int t = lane < kJoinThreads / 32 && lane < warp ? sh[lane] : 0;
  n += __reduce_add_sync(0xffffffffu, t);
  front[tid + 1] = n;
  if (tid == 0) front[0] = 0;
  __syncthreads();
  const float unit = p.scale * 1.4426950408889634f;
  const int64_t slot = (int64_t)p.pairs * kTrPart;
  constexpr int kWarps = kJoinThreads / 32;
  const int jobs = front[kJoinThreads];
  int ways = 1;   // warps of a job
  while (2 * ways <= kWarps && (int64_t)jobs * 2 * ways <= (int64_t)gridDim.x * kWarps) ways *= 2;
  const int sub = warp % ways, step = gridDim.x * (kWarps / ways);
#pragma unroll 1
  for (int job0 = blockIdx.x * (kWarps / ways); job0 < jobs; job0 += step) {   // (the same in all warps; once, if several share a job)
    const int job = job0 + warp / ways;
    const bool in = job < jobs;
    int k = 0;   // the last with front[k] <= job
#pragma unroll
    for (int b = kJoinThreads / 2; b > 0; b >>= 1)
      if (front[k + b] <= job) k += b;
    const Kv8Cut cut = cuts[min(k, kNumSMs - 1)];
    const int at = job - front[k], c = at % (kHeadDim / kJoinColumns), pair = at / (kHeadDim / kJoinColumns) * 32 + lane;
    const float* part = p.part + (2 * k + 1) * slot;   // the first: behind it every other one
    auto part_of = [&](int i) { return part + (i ? 2 * i - 1 : 0) * slot; };
    auto ml = [&](int i) { return reinterpret_cast<const float2*>(part_of(i) + (int64_t)p.pairs * kHeadDim)[pair]; };
    float m = -INFINITY, l = 0.f, a[8] = {};
    const int each = (cut.parts + ways - 1) / ways, i0 = in ? sub * each : 0, i1 = in ? min(cut.parts, i0 + each) : 0;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) m = fmaxf(m, ml(i).x);
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
      const float2 t = ml(i);
      const float4 *v = reinterpret_cast<const float4*>(part_of(i)) + (int64_t)(2 * c) * p.pairs + pair, x = __ldcg(v), y = __ldcg(v + p.pairs);
      const float f = t.x == m ? 1.f : exp2_fast((t.x - m) * unit);
      l += t.y * f;
      join_part(a, {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}, f);
    }
    if (ways > 1) {
      sums[0][tid] = m, sums[1][tid] = l;
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[2 + j][tid] = a[j];
      __syncthreads();
      if (sub) return;
      for (int w = 1; w < ways; ++w) m = fmaxf(m, sums[0][tid + 32 * w]);
      l = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = 0.f;
      for (int w = 0; w < ways; ++w) {
        const float own = sums[0][tid + 32 * w], f = own == m ? 1.f : exp2_fast((own - m) * unit);
        l += sums[1][tid + 32 * w] * f;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = sums[2 + j][tid + 32 * w];
        join_part(a, x, f);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (in && pair < cut.nrows * G)
      *reinterpret_cast<uint4*>(p.out + (int64_t)(cut.row0 + pair / G) * p.ldo + (cut.kvh * G + pair % G) * kHeadDim + c * kJoinColumns) =
          make_uint4(pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv), pack_bf16(a[4] * inv, a[5] * inv), pack_bf16(a[6] * inv, a[7] * inv));
  }
}

// ---- workspace ----------------------------------------------------------------------------------------------------------------------------
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t tree_pairs(int T, int hq, int hkv) {   // of an item at most
  const int G = hq / hkv;
  return (std::min<int64_t>((int64_t)T * G, 2 * (128 / G) * G) + 31) / 32 * 32;
}
struct TreeSizes {
  int64_t cuts, part, list, all;
};
TreeSizes tree_sizes(int T, int hq, int hkv) {
  TreeSizes s = {};
  s.cuts = up256(kNumSMs * (int64_t)sizeof(Kv8Cut));
  s.part = up256(2 * kNumSMs * tree_pairs(T, hq, hkv) * kTrPart * 4);
  s.list = up256(((int64_t)T * hkv + kNumSMs) * (int64_t)sizeof(TreeWork));
  s.all = s.cuts + s.part + s.list;
  return s;
}

int tree_launch(TreeParams p, void* ws, cudaStream_t s) {
  if (const int e = wait_status()) return e;
  CUtensorMap mq, mk, mv;
  const int64_t rows = p.n_blocks * p.hkv * p.block_size;
  const int G = p.hq / p.hkv;
  if (const int rc = query_map_bf16(p.q, p.T, p.hq, p.ldq, G, 128 / G, &mq)) return rc;
  if (const int rc = rows_map_bf16(p.k, rows, std::min(p.block_size, kTreeKeys), &mk)) return rc;
  if (const int rc = rows_map_bf16(p.v, rows, std::min(p.block_size, kTreeKeys), &mv)) return rc;
  const TreeSizes z = tree_sizes(p.T, p.hq, p.hkv);
  char* const w = static_cast<char*>(ws);
  p.cuts = reinterpret_cast<Kv8Cut*>(w);
  p.part = reinterpret_cast<float*>(w + z.cuts);
  p.list = reinterpret_cast<TreeWork*>(w + z.cuts + z.part);
  p.pairs = (int)tree_pairs(p.T, p.hq, p.hkv);
  p.status = wait_status_word();
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(attn_tree_kernel, kTrSmem, done));
  B200_CUDA(launch(attn_tree_kernel, dim3(kNumSMs), dim3(kTreeThreads), (size_t)kTrSmem, s, mq, mk, mv, p));
  const PdlScope after;
  B200_CUDA(launch(tree_join_kernel, dim3(kJoinCtas * kNumSMs), dim3(kJoinThreads), (size_t)0, s, p));
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool tree_heads_ok(int hq, int hkv) { return hkv > 0 && hq > 0 && hq % hkv == 0; }

extern "C" int64_t b200_paged_attn_tree_workspace_bytes(int32_t T, int32_t hq, int32_t hkv) {
  return T > 0 && tree_heads_ok(hq, hkv) && hq / hkv <= 16 ? tree_sizes(T, hq, hkv).all : 0;
}

extern "C" int b200_paged_attn_tree(const void* q, int64_t ldq, const void* k_cache_layer, const void* v_cache_layer, int64_t n_blocks, const int32_t* block_table,
                                    int32_t bt_stride, const int32_t* row_to_seq, const int32_t* ctx_lens, const uint32_t* tree_masks, int32_t mask_words, void* out,
                                    int64_t ldo, int32_t T, int32_t hq, int32_t hkv, int32_t block_size, float scale, void* ws, int64_t ws_bytes, void* stream) {
  B200_REQUIRE(q && k_cache_layer && v_cache_layer && block_table && ctx_lens && out && (tree_masks || mask_words == 0), B200_ERR_INVALID, "paged_attn_tree: null");
  B200_REQUIRE(T >= 0 && tree_heads_ok(hq, hkv) && bt_stride > 0 && mask_words >= 0, B200_ERR_INVALID,
               "paged_attn_tree: %d rows, %d heads over %d, %d block-table columns, %d mask words", T, hq, hkv, bt_stride, mask_words);
  B200_REQUIRE(hq / hkv <= 16, B200_ERR_UNSUPPORTED, "paged_attn_tree: %d heads over %d (at most 16 to a kv head)", hq, hkv);
  B200_REQUIRE(mask_words <= kMostWords, B200_ERR_UNSUPPORTED, "paged_attn_tree: %d mask words (at most %d)", mask_words, kMostWords);
  B200_REQUIRE(kv8_block_ok(block_size), B200_ERR_UNSUPPORTED, "paged_attn_tree: block_size=%d (16, 32, 64 or a multiple of 128)", block_size);
  B200_REQUIRE(kv8_rows_ok(n_blocks, hkv, block_size), B200_ERR_INVALID, "paged_attn_tree: %lld blocks", (long long)n_blocks);
  B200_REQUIRE((int64_t)bt_stride * block_size <= kMostTokens, B200_ERR_UNSUPPORTED, "paged_attn_tree: block tables of %lld tokens", (long long)bt_stride * block_size);
  B200_REQUIRE(ldq >= (int64_t)hq * kHeadDim && ldq % 8 == 0 && ldo >= (int64_t)hq * kHeadDim && ldo % 8 == 0, B200_ERR_INVALID,
               "paged_attn_tree: ldq and ldo are multiples of 8 that hold a row");
  B200_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_cache_layer) && aligned16(v_cache_layer), B200_ERR_INVALID, "paged_attn_tree: tensors must be 16-byte aligned");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(tree_masks) & 3) == 0, B200_ERR_INVALID, "paged_attn_tree: masks must be 4-byte aligned");
  B200_REQUIRE(scale > 0.f && scale - scale == 0.f, B200_ERR_INVALID, "paged_attn_tree: scale must be positive and finite");
  if (T == 0) return B200_OK;
  const int64_t tiles = ((int64_t)bt_stride * block_size + kTreeKeys - 1) / kTreeKeys;
  B200_REQUIRE(T <= kMostRows && (int64_t)T * hkv * (kCostItem + kCostTwo * tiles) < 0x7fffffffll - 4 * kCostTwo * tiles, B200_ERR_UNSUPPORTED,
               "paged_attn_tree: %d rows of %d kv heads of up to %lld tokens (at most %d rows)", T, hkv, (long long)bt_stride * block_size, kMostRows);
  const int64_t need = b200_paged_attn_tree_workspace_bytes(T, hq, hkv);
  B200_REQUIRE(ws && aligned16(ws) && ws_bytes >= need, B200_ERR_INVALID, "paged_attn_tree: the workspace is 16-byte aligned and has at least %lld bytes (%lld)",
               (long long)need, (long long)ws_bytes);
  B200_REQUIRE(n_blocks * hkv * block_size <= 0x7fffffff - 256, B200_ERR_UNSUPPORTED, "paged_attn_tree: a cache of %lld rows", (long long)(n_blocks * hkv * block_size));
  TreeParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k_cache_layer);
  p.v = static_cast<const __nv_bfloat16*>(v_cache_layer);
  p.ldq = ldq;
  p.n_blocks = n_blocks;
  p.block_table = block_table;
  p.row_to_seq = row_to_seq;
  p.ctx_lens = ctx_lens;
  p.masks = tree_masks;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.bt_stride = bt_stride;
  p.words = mask_words;
  p.T = T;
  p.hq = hq;
  p.hkv = hkv;
  p.block_size = block_size;
  p.scale = scale;
  return tree_launch(p, ws, (cudaStream_t)stream);
}
