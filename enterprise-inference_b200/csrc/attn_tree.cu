// Attention over the paged cache with a mask per row (b200_paged_attn_tree): trees of drafted tokens, beams that share a prompt.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),  over the tokens j that the row sees: those in front of ctx_lens[t], and ctx_lens[t] + i for each
//   bit i of its mask.
//
// Three launches.  plan (one CTA): rows -> runs of one sequence -> items of up to two tiles of 128 (row, head) pairs of a kv head; the list of (item, kv head, tile of 64
// tokens) is cut into equal shares, one an SM.  The main kernel walks its share on tcgen05,
//   S = Q K^T (M = 128 pairs, N = 64 tokens), O += P V (N = 128),
// scores, weights (bf16 high and low terms: 16 bits) and O in tensor memory, keys and values by TMA through a ring of eight tiles.  An item of two tiles of pairs has a group of
// four softmax warps for each; one of a single tile lets the two groups take its key tiles in turn, each with a maximum, a sum and an O of its own, which are put together at its
// end.  Items that a cut goes through leave fp32 sums, which the last launch joins in the order of the cut.
// A tile that lies in front of every row's context is seen whole; in the others a thread (a pair) makes 64 bits of what it sees from its context and mask, and the values that
// are no numbers are taken out of the tile, since 0 x NaN would reach every row; rows that see them get them back at the end.
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
constexpr int kTrPart = 136;                    // floats of a pair in a part: 128 sums, their maximum (of the products q . k), the denominator; whole sectors
constexpr int kTrSmem = 1024 + 4 * kTrQChunk + kTreeSlots * kTrTile + kTrStage + 2 * 128 * 8 + 2 * kTrBad * 16 + (2 * kTreeSlots + 16) * 8 + 16;
static_assert(kTrSmem <= 232448, "shared memory");
constexpr int kPlanThreads = 1024, kPlanNear = 1024;   // rows of a step whose lists are in shared memory

// what an item's walk over the tiles [tile0, tile1) needs; parts > 1: further CTAs have the rest, each leaves its sums in a slot.  A CTA's items follow one another; cta -1: none
struct alignas(16) TreeWork {
  int row0, nrows, seq, clear, end, tile0, tile1, kvh, cta, parts, slot, pad;   // clear, end: tokens that all rows see, up to the last one that any sees
};
struct TreeItem {
  int row0, nrows, seq, clear, end;
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
  TreeWork* list;
  int* starts;           // [CTA] its first place of the list (-1: none)
  Kv8Cut* cuts;          // [CTA] its last item, where further CTAs have parts of it
  float* part;           // [CTA][2][pairs][kTrPart]: of an item that began in an earlier CTA, of one that goes on in the next
  int pairs;
  uint32_t* status;
};

__host__ __device__ __forceinline__ int64_t tree_tokens(const TreeParams& p) { return (int64_t)p.bt_stride * p.block_size; }
__device__ __forceinline__ int tree_ctx(const TreeParams& p, int row) { return (int)min((int64_t)max(__ldg(p.ctx_lens + row), 0), tree_tokens(p)); }

// ---- plan -----------------------------------------------------------------------------------------------------------------------------
// Costs, in units of a key tile with one tile of pairs: with two of them, and of an item's start and end
constexpr int kCostOne = 2, kCostTwo = 4, kCostItem = 2;

__device__ __forceinline__ int64_t scan64(int64_t& x, int64_t* sh) {   // exclusive over the CTA; returns the total
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t own = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += u;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  int64_t w = sh[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  const int64_t before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  x += (warp ? before : 0) - own;
  return __shfl_sync(0xffffffffu, w, 31);
}

struct PlanLists {   // of T entries each
  int *ctx, *end, *runs;
  TreeItem* items;
  int64_t* front;
};

__global__ void __launch_bounds__(kPlanThreads) tree_plan_kernel(const TreeParams p, int R, PlanLists far) {
  __shared__ int64_t sh[32];
  __shared__ int near_ctx[kPlanNear], near_end[kPlanNear], near_runs[kPlanNear];
  __shared__ TreeItem near_items[kPlanNear];
  __shared__ int64_t near_front[kPlanNear];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool near = p.T <= kPlanNear;
  int *const ctx = near ? near_ctx : far.ctx, *const end = near ? near_end : far.end, *const runs = near ? near_runs : far.runs;
  TreeItem* const items = near ? near_items : far.items;
  int64_t* const front = near ? near_front : far.front;
  const int64_t tokens = tree_tokens(p);
  auto seq_of = [&](int r) { return p.row_to_seq ? __ldg(p.row_to_seq + r) : r; };
  // rows: their context, and the end of what they see; the runs' first rows
  int n_runs = 0;
  for (int r0 = 0; r0 < p.T; r0 += kPlanThreads) {
    const int r = r0 + tid;
    int64_t at = 0;
    bool flag = false;
    if (r < p.T) {
      const int c = tree_ctx(p, r);
      int64_t e = c;
      const uint32_t* m = p.masks + (int64_t)r * p.words;
#pragma unroll 8
      for (int w = 0; w < p.words; ++w) {
        const uint32_t x = __ldg(m + w);
        if (x) e = (int64_t)c + 32 * w + 32 - __clz(x);
      }
      ctx[r] = c;
      end[r] = (int)min(e, tokens);
      flag = r == 0 || seq_of(r) != seq_of(r - 1);
    }
    at = flag;
    const int n = (int)scan64(at, sh);
    if (flag) runs[n_runs + at] = r;
    n_runs += n;
  }
  __syncthreads();
  // items: up to two tiles of pairs
  int n_items = 0;
  for (int i0 = 0; i0 < n_runs; i0 += kPlanThreads) {
    const int i = i0 + tid, first = i < n_runs ? runs[i] : 0, n = i < n_runs ? (i + 1 < n_runs ? runs[i + 1] : p.T) - first : 0, mine = (n + 2 * R - 1) / (2 * R);
    int64_t at = mine;
    const int all = (int)scan64(at, sh);
    for (int k = 0; k < mine; ++k) items[n_items + at + k] = {first + 2 * R * k, min(2 * R, n - 2 * R * k), seq_of(first), 0, 0};
    n_items += all;
  }
  __syncthreads();
  for (int i = warp; i < n_items; i += kPlanThreads / 32) {
    const int row0 = items[i].row0, n = items[i].nrows;
    int c = 0x7fffffff, e = 0;
    for (int r = lane; r < n; r += 32) c = min(c, ctx[row0 + r]), e = max(e, end[row0 + r]);
    c = __reduce_min_sync(0xffffffffu, c);
    e = __reduce_max_sync(0xffffffffu, e);
    if (lane == 0) items[i].clear = c, items[i].end = e;
  }
  const int n_units = n_items * p.hkv;
  for (int i = tid; i < n_units + kNumSMs + 1; i += kPlanThreads) p.list[i].cta = -1;
  if (tid < kNumSMs) p.starts[tid] = -1, p.cuts[tid].parts = 0;
  __syncthreads();
  // costs in front of an item (of one kv head)
  auto tiles_of = [&](const TreeItem& t) { return (t.end + kTreeKeys - 1) / kTreeKeys; };
  auto each_of = [&](const TreeItem& t) { return t.nrows > R ? kCostTwo : kCostOne; };
  int64_t total = 0;
  for (int i0 = 0; i0 < n_items; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t c = i < n_items ? kCostItem + (int64_t)max(tiles_of(items[i]), 1) * each_of(items[i]) : 0;
    const int64_t all = scan64(c, sh);
    if (i < n_items) front[i] = total + c;
    total += all;
  }
  __syncthreads();
  // Tile t of an item lies at its front + (t ? kCostItem : 0) + t x its cost on the line of all costs; CTA k has what lies in [k share, (k + 1) share).  A share is no less than the
  // widest gap, so none between the first and the last of an item is without a tile
  const int64_t share = max((int64_t)(kCostItem + kCostTwo), (total * p.hkv + kNumSMs - 1) / kNumSMs);
  auto at_line = [&](int u, int64_t& base, int64_t& last) {   // of an item's first and last tile
    const TreeItem& g = items[u / p.hkv];
    const int nt = tiles_of(g), each = each_of(g);
    base = front[u / p.hkv] * p.hkv + (int64_t)(u % p.hkv) * (kCostItem + (int64_t)max(nt, 1) * each);
    last = base + (nt > 1 ? kCostItem + (int64_t)(nt - 1) * each : 0);
  };
  for (int u = tid; u < n_units; u += kPlanThreads) {
    const TreeItem g = items[u / p.hkv];
    const int nt = tiles_of(g), each = each_of(g), h = u % p.hkv;
    int64_t base, last, base_before = 0, last_before = -share;
    at_line(u, base, last);
    if (u > 0) at_line(u - 1, base_before, last_before);
    const int k0 = (int)(base / share), k1 = (int)(last / share);
    auto first_tile = [&](int k) {   // the first one, but for the item's first, at or behind the start of share k
      const int64_t behind = k * share - base - kCostItem;
      return behind <= each ? 1 : (int)min((int64_t)nt, (behind + each - 1) / each);
    };
    for (int k = k0; k <= k1; ++k) {
      const int place = u + k;
      p.list[place] = {g.row0, g.nrows, g.seq, g.clear, g.end, k == k0 ? 0 : first_tile(k), k == k1 ? nt : first_tile(k + 1), h, k, k1 - k0 + 1, 2 * k + (k == k0 ? 1 : 0), 0};
      if (k > k0 || u == 0 || last_before / share < k) p.starts[k] = place;
    }
    if (k1 > k0) p.cuts[k0] = {g.row0, g.nrows, h, k1 - k0 + 1};
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
  const int first = max(w.tile0, w.clear / kTreeKeys);   // the first tile that not all rows see
  auto add = [&](int key, float* to) {
    const int64_t blk = __ldg(p.block_table + (int64_t)w.seq * p.bt_stride + key / p.block_size);
    if (blk < 0 || blk >= p.n_blocks) return;
    const __nv_bfloat16* v = p.v + ((blk * p.hkv + w.kvh) * p.block_size + key % p.block_size) * kHeadDim + c;
    for (int d = 0; d < 32; ++d) {
      const float x = __bfloat162float(v[d]);
      if (!(x - x == 0.f)) to[d] += x;
    }
  };
  bool nan = false;
  for (int d = 0; d < 32; ++d) nan |= o[d] != o[d];
  if (nan) {
    float s[32];
    for (int d = 0; d < 32; ++d) s[d] = 0.f;
    const int to = min(first, w.tile1) * kTreeKeys;
    for (int key = w.tile0 * kTreeKeys; key < to; ++key) add(key, s);
    for (int d = 0; d < 32; ++d)
      if (o[d] != o[d] && s[d] != 0.f) o[d] = s[d];
  }
  if (!taken_out) return;
  for (int t = first; t < w.tile1; ++t) {
    uint32_t bits[2];
    tree_bits(r, t * kTreeKeys, bits);
    for (int j = 0; j < kTreeKeys; ++j) {
      const bool known = t - first < kTrBad;
      if ((bits[j >> 5] >> (j & 31) & 1) && (!known || (bad[t - first][j >> 4] >> (2 * (j & 15)) & 3))) add(t * kTreeKeys + j, o);
    }
  }
}

__global__ void __launch_bounds__(kTreeThreads, 1)
attn_tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
  unsigned char* qs = smem;                        // two tiles of [2][128 pairs][64]
  unsigned char* ring = qs + 4 * kTrQChunk;        // [kTreeSlots][2][64 keys][64]: key and value tiles in turn
  unsigned char* ostage = ring + kTreeSlots * kTrTile;
  float2* exchange = reinterpret_cast<float2*>(ostage + kTrStage);                   // [group][pair] maximum, sum
  uint32_t(*bad_keys)[4] = reinterpret_cast<uint32_t(*)[4]>(exchange + 2 * 128);    // [item's parity][tile][16 keys]: two bits a key
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(bad_keys + 2 * kTrBad);
  uint64_t* kv_free = kv_full + kTreeSlots;
  uint64_t* s_full = kv_free + kTreeSlots;         // [group][2] the scores of its even / odd key tile are there
  uint64_t* p_ready = s_full + 4;                  // [group][2] their weights are
  uint64_t* o_full = p_ready + 4;                  // [group][2] their second product has finished
  uint64_t* q_ready = o_full + 4;
  uint64_t* q_first = q_ready + 1;                 // the CTA's first queries, staged by the softmax warps as well
  uint64_t* q_free = q_first + 1;
  uint64_t* last = q_free + 1;                     // the MMAs in flight when a wait ran out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last + 1);   // and, behind it, the mark of a wait that ran out
  int* taken_item = reinterpret_cast<int*>(tmem_slot + 2);       // [item's parity] the last one (counted from 1) with values that were taken out of a tile
  const Waits mbar_wait(tmem_slot + 1, p.status);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kTreeSlots; ++s) {
      mbar_init(kv_full + s, 1);
      mbar_init(kv_free + s, 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(p_ready + s, 4);
      mbar_init(o_full + s, 1);
    }
    mbar_init(q_ready, 2);
    mbar_init(q_first, 10);
    mbar_init(q_free, 1);
    mbar_init(last, 1);
    tmem_slot[1] = 0;
    taken_item[0] = taken_item[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  const int start = __ldcg(p.starts + cta);
  if (start < 0) return;
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int G = p.hq / p.hkv, R = 128 / G;
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;   // per group 256 columns: scores of even, odd key tiles, O
  auto next_work = [&](int& at, TreeWork& w) {
    const int4* src = reinterpret_cast<const int4*>(p.list + at);
    const int4 a = __ldcg(src), b = __ldcg(src + 1), c = __ldcg(src + 2);
    w = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
    ++at;
    return w.cta == cta;
  };
  // the A operands of an item, thread i of `threads`: 16-byte pieces of rows
  auto stage_q = [&](const TreeWork& w, int i, int threads) {
    const __nv_bfloat16* q0 = p.q + (int64_t)w.row0 * p.ldq + (int64_t)w.kvh * G * kHeadDim;
    const int pieces = (w.nrows > R ? 2 : 1) * 128 * 16;
    constexpr int U = 8;
#pragma unroll 1
    for (int e0 = i; e0 < pieces; e0 += U * threads) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = e0 + u * threads, m = e >> 4, chunk = e & 15, r = (m & 127) / G, g = (m & 127) % G, row = (m >> 7) * R + r;
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (e < pieces && r < R && row < w.nrows) v[u] = __ldg(reinterpret_cast<const uint4*>(q0 + (int64_t)row * p.ldq + g * kHeadDim + chunk * 8));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = e0 + u * threads, m = e >> 4, chunk = e & 15, mm = m & 127;
        if (e < pieces)
          *reinterpret_cast<uint4*>(qs + (2 * (m >> 7) + (chunk >> 3)) * kTrQChunk + (mm >> 3) * 1024 + (mm & 7) * 128 + (((chunk & 7) ^ (mm & 7)) << 4)) = v[u];
      }
    }
    fence_async_smem();
    __syncwarp();
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
    const int64_t tokens = tree_tokens(p);
    int slot = 0, row = 0;
    uint32_t ph = 1;
    bool stop = false;
    TreeWork w;
    for (int at = start; !stop && next_work(at, w);) {
      const int32_t* bt = p.block_table + (int64_t)w.seq * p.bt_stride;
      for (int i = w.tile0; i < w.tile1 && !(stop = mbar_wait.stop()); ++i) {
        const int k = (i - w.tile0) % ahead;
        if (k == 0) {   // lane: the row of box lane % boxes of tile i + lane / boxes
          const int64_t tok = (int64_t)(i + lane / boxes) * kTreeKeys + lane % boxes * box;
          const int blk = tok < tokens && i + lane / boxes < w.tile1 ? __ldg(bt + tok / p.block_size) : -1;
          row = blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + w.kvh) * p.block_size + (int)(tok % p.block_size) : none;
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          mbar_wait(kv_free + slot, ph);
          if (issuer) mbar_expect_tx(kv_full + slot, kTrTile);
          for (int b = 0; b < boxes; ++b) {
            const int from = __shfl_sync(0xffffffffu, row, k * boxes + b);
            if (issuer) {
              unsigned char* dst = ring + slot * kTrTile + b * box * 128;
              tma_load_2d(dst, kv ? &map_v : &map_k, 0, from, kv_full + slot);
              tma_load_2d(dst + kTrChunk, kv ? &map_v : &map_k, 64, from, kv_full + slot);
            }
          }
          __syncwarp();
          if (++slot == kTreeSlots) slot = 0, ph ^= 1;
        }
      }
    }
    if (mbar_wait.stop())   // the loads in flight: a slot's last one filled it in this round of the ring or in the one before
      for (int s = 0; s < kTreeSlots; ++s) mbar_wait.drain(kv_full + s, s < slot ? ph ^ 1 : ph);
  } else if (warp == 9) {
    // ===== MMA: per key tile the next one's scores, then this one's second product.  The whole warp walks the loop; bounds and addresses that come from memory are broadcast, so
    // that they are uniform to the compiler =====
    const uint32_t one = elect_one() ? 1u : 0u, tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t desc_q = make_desc(smem_u32(qs), 16, 1024), desc_k = make_desc(smem_u32(ring), 16, 1024), desc_v = make_desc(smem_u32(ring), kTrChunk, 1024);
    const uint32_t id_s = idesc_bf16(kTreeKeys, 0), id_o = idesc_bf16(kHeadDim, 1);
    int slot = 0, active = 0, n[2] = {0, 0};   // n: key tiles of either group so far
    uint32_t ph = 0;
    auto next_slot = [&]() {
      if (++slot == kTreeSlots) slot = 0, ph ^= 1;
    };
    auto scores = [&](int x, int tile, int nx, int k_slot) {   // group x, its tile of pairs
      const uint64_t da = desc_q + (uint64_t)((tile * 2 * kTrQChunk) >> 4), db = desc_k + (uint64_t)((k_slot * kTrTile) >> 4);
      const uint32_t d = tm + x * 256 + (nx & 1) * kTreeKeys;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        mma_ss(one, d, da + ((j >> 2) * kTrQChunk + (j & 3) * 32) / 16, db + ((j >> 2) * kTrChunk + (j & 3) * 32) / 16, id_s, j ? 1u : 0u);
      commit(one, s_full + 2 * x + (nx & 1));
    };
    auto product = [&](int x, int nx, int v_slot, uint32_t more) {
      const uint64_t dv = desc_v + (uint64_t)((v_slot * kTrTile) >> 4);
      mbar_wait(p_ready + 2 * x + (nx & 1), (nx >> 1) & 1);
      fence_after();
      const uint32_t pa = tm + x * 256 + (nx & 1) * kTreeKeys, d = tm + x * 256 + 128;
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // 16 keys per step: 8 columns of weights, 16 further those of the second term
        mma_ts(one, d, pa + (j >> 1) * 32 + (j & 1) * 8, dv + (uint64_t)((j * 2048) >> 4), id_o, j ? 1u : more);
        mma_ts(one, d, pa + (j >> 1) * 32 + (j & 1) * 8 + 16, dv + (uint64_t)((j * 2048) >> 4), id_o, 1u);
      }
    };
    // an item of nt key tiles with both tiles of pairs, or its key tiles by the groups in turn
    auto walk = [&](auto two_c, int nt) {
      constexpr bool TWO = decltype(two_c)::value;
      mbar_wait(kv_full + slot, ph);
      fence_after();
      int k_slot = slot;
      next_slot();
      scores(0, 0, n[0], k_slot);
      if (TWO) scores(1, 1, n[1], k_slot);
      commit(one, kv_free + k_slot);
      commit(nt == 1 ? one : 0u, q_free);
      auto step = [&](auto more_c, auto x_c, int i) {
        constexpr bool MORE = decltype(more_c)::value;
        [[maybe_unused]] constexpr int X = decltype(x_c)::value;   // (not TWO) the group of key tile i
        const int v_slot = slot;
        const uint32_t v_ph = ph;
        next_slot();
        if constexpr (MORE) {
          mbar_wait(kv_full + slot, ph);
          fence_after();
          k_slot = slot;
          next_slot();
        }
        if constexpr (TWO) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if constexpr (MORE) scores(x, x, n[x] + 1, k_slot);
            if (MORE && x == 1) {
              commit(one, kv_free + k_slot);
              commit(i + 2 == nt ? one : 0u, q_free);   // the item's last scores are on their way
            }
            if (x == 0) mbar_wait(kv_full + v_slot, v_ph);
            product(x, n[x], v_slot, i ? 1u : 0u);
            if (x == 1) commit(one, kv_free + v_slot);
            commit(one, o_full + 2 * x + (n[x] & 1));
            ++n[x];
          }
        } else {
          if constexpr (MORE) {
            scores(X ^ 1, 0, n[X ^ 1], k_slot);
            commit(one, kv_free + k_slot);
            commit(i + 2 == nt ? one : 0u, q_free);
          }
          mbar_wait(kv_full + v_slot, v_ph);
          product(X, n[X], v_slot, i > 1 ? 1u : 0u);
          commit(one, kv_free + v_slot);
          commit(one, o_full + 2 * X + (n[X] & 1));
          ++n[X];
        }
      };
      const std::integral_constant<int, 0> even;
      const std::integral_constant<int, 1> odd;
      if constexpr (TWO) {
        for (int i = 0; i + 1 < nt; ++i) step(std::true_type(), even, i);
        step(std::false_type(), even, nt - 1);
      } else {
        int i = 0;
        for (; i + 2 < nt; i += 2) {
          step(std::true_type(), even, i);
          step(std::true_type(), odd, i + 1);
        }
        if (i + 1 < nt) {
          step(std::true_type(), even, i);
          step(std::false_type(), odd, i + 1);
        } else {
          step(std::false_type(), even, i);
        }
      }
    };
    TreeWork w;
    for (int at = start; __shfl_sync(0xffffffffu, next_work(at, w), 0);) {
      const int nt = __shfl_sync(0xffffffffu, w.tile1 - w.tile0, 0), two = __shfl_sync(0xffffffffu, w.nrows > R ? 1 : 0, 0);
      if (nt <= 0) continue;
      if (active == 0) mbar_wait(q_first, 0);
      else mbar_wait(q_ready, (active - 1) & 1);
      if (two) walk(std::true_type(), nt);
      else walk(std::false_type(), nt);
      ++active;
    }
    if (mbar_wait.stop()) {
      commit(one, last);
      mbar_wait.drain(last, 0);
    }
  } else if (warp >= 10) {
    // ===== queries of the next item -> the A operands =====
    int active = 0;
    TreeWork w;
    for (int at = start; next_work(at, w);) {
      if (w.tile1 <= w.tile0) continue;
      if (active == 0) {
        stage_q(w, threadIdx.x - 64, 320);   // (beside the softmax warps' threads 0..255)
        if (lane == 0) mbar_arrive(q_first);
      } else {
        mbar_wait(q_free, (active - 1) & 1);
        stage_q(w, threadIdx.x - 320, 64);
        if (lane == 0) mbar_arrive(q_ready);
      }
      ++active;
    }
  } else {
    // ===== softmax and output: a thread owns a pair, of tile x of the item's, or with its fellow in the other group of the only one =====
    const int x = warp >> 2, quad = warp & 3, m = quad * 32 + lane;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16), own = base + x * 256;
    const int r = m / G, g = m % G;
    const float sc2 = p.scale * 1.4426950408889634f;   // scores in the log2 domain
    bool first = true;
    int n = 0, done = 0, item = 0;   // key tiles of this group so far; of all items before; items
    TreeWork w;
    for (int at = start; next_work(at, w);) {
      ++item;   // (a group is at most one item ahead of the other)
      uint32_t(*const bad)[4] = bad_keys + (item & 1) * kTrBad;
      if (first && w.tile1 > w.tile0) {
        stage_q(w, threadIdx.x, 320);   // (the stagers are threads 256..319 of this)
        if (lane == 0) mbar_arrive(q_first);
        first = false;
      }
      const bool two = w.nrows > R;
      const int row = (two ? x * R : 0) + r, t = w.row0 + row;
      const bool alive = r < R && row < w.nrows;
      const TreeRow see = {p.masks + (int64_t)t * p.words, alive ? tree_ctx(p, t) : 0, alive ? p.words : 0, w.end, alive};
      const int masked = max(w.tile0, w.clear / kTreeKeys);   // the first tile that not all rows see
      float mu = -INFINITY, l = 0.f;
      const int n0 = n;
      for (int i = w.tile0 + (two ? 0 : x); i < w.tile1; i += two ? 1 : 2, ++n) {
        mbar_wait(s_full + 2 * x + (n & 1), (n >> 1) & 1);
        fence_after();
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
        const bool jump = (mx - mu) * sc2 > 8.f;   // also the first live key (mu = -inf)
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
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint64_t e = f2::mul(f2::add(f2::pack(__uint_as_float(s[c * 32 + 2 * j]), __uint_as_float(s[c * 32 + 2 * j + 1])), minus), unit);
            const float p0 = exp2_fast(f2::lo(e)), p1 = exp2_fast(f2::hi(e));
            // the high term truncated, the rest rounded
            sum[j & 3] += p0 + p1;
            const uint32_t h0 = __float_as_uint(p0) & 0xffff0000u, h1 = __float_as_uint(p1) & 0xffff0000u;
            pk[j] = __byte_perm(h0, h1, 0x7632);
            pk[16 + j] = pack_bf16(p0 - __uint_as_float(h0), p1 - __uint_as_float(h1));
          }
          st32(s_addr + c * 32, pk);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (i >= masked && !(two && x)) {
          // 0 x NaN = NaN: what is no number leaves the value tile (two threads a key), everything behind the end does
          const int v_at = 2 * (done + i - w.tile0) + 1, vs = v_at % kTreeSlots, key = m >> 1;
          mbar_wait(kv_full + vs, (v_at / kTreeSlots) & 1);
          uint4* const vb = reinterpret_cast<uint4*>(ring + vs * kTrTile + (m & 1) * kTrChunk + key * 128);
          const bool behind = i * kTreeKeys + key >= w.end;
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
            if (keys) reinterpret_cast<volatile int*>(taken_item)[item & 1] = item;
          }
          fence_async_smem();
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
      const bool taken = reinterpret_cast<volatile int*>(taken_item)[item & 1] == item;
      const int c0 = two ? 0 : x * 64, c1 = two ? kHeadDim : c0 + 64;
      const float inv = w.parts > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float* const part = p.part + ((int64_t)w.slot * p.pairs + row * G + g) * kTrPart;
      if (w.parts > 1 && alive && c0 == 0) *reinterpret_cast<float2*>(part + kHeadDim) = make_float2(mu, l);
      unsigned char* const st = ostage + warp * 2048;
#pragma unroll 1
      for (int c = c0; c < c1; c += 32) {
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
            for (int k = 0; k < 4; ++k) store_sector(part + c + 8 * k, o + 8 * k);
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
            if (mm / G < R && row2 < w.nrows) *reinterpret_cast<uint4*>(p.out + (int64_t)(w.row0 + row2) * p.ldo + (int64_t)(w.kvh * G + mm % G) * kHeadDim + col) = v;
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
constexpr int kTreeManyParts = 4;

__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const Kv8Cut cut = p.cuts[blockIdx.x];
  if (cut.parts < 2) return;
  const int G = p.hq / p.hkv;
  const int64_t step = 2ll * p.pairs * kTrPart;
  auto join = [&](auto lanes_c) {
    constexpr int LANES = decltype(lanes_c)::value, EACH = 256 / LANES;
    for (int c = blockIdx.y * EACH + threadIdx.x / LANES; c < cut.nrows * G; c += EACH * gridDim.y) {
      const float* x = p.part + (2 * (int64_t)blockIdx.x * p.pairs + c) * kTrPart;
      join_parts<LANES>(x + p.pairs * kTrPart, x + step, step, cut.parts, p.out + (int64_t)(cut.row0 + c / G) * p.ldo + (cut.kvh * G + c % G) * kHeadDim, p.scale * 1.4426950408889634f);
    }
  };
  if (cut.parts > kTreeManyParts) join(std::integral_constant<int, 32>());
  else join(std::integral_constant<int, 8>());
}

// ---- workspace ----------------------------------------------------------------------------------------------------------------------------
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t tree_pairs(int T, int hq, int hkv) {   // of an item at most
  const int G = hq / hkv;
  return std::min<int64_t>((int64_t)T * G, 2 * (128 / G) * G);
}
struct TreeSizes {
  int64_t list, starts, cuts, part, rows, items, front, all;
};
TreeSizes tree_sizes(int T, int hq, int hkv) {
  TreeSizes s = {};
  s.list = up256(((int64_t)T * hkv + kNumSMs + 1) * (int64_t)sizeof(TreeWork));
  s.starts = up256(kNumSMs * 4);
  s.cuts = up256(kNumSMs * (int64_t)sizeof(Kv8Cut));
  s.part = up256(2 * kNumSMs * tree_pairs(T, hq, hkv) * kTrPart * 4);
  s.rows = up256((int64_t)T * 4);
  s.items = up256((int64_t)T * (int64_t)sizeof(TreeItem));
  s.front = up256((int64_t)T * 8);
  s.all = s.list + s.starts + s.cuts + s.part + 3 * s.rows + s.items + s.front;
  return s;
}

int tree_launch(TreeParams p, void* ws, cudaStream_t s) {
  if (const int e = wait_status()) return e;
  CUtensorMap mk, mv;
  const int64_t rows = p.n_blocks * p.hkv * p.block_size;
  if (const int rc = rows_map_bf16(p.k, rows, std::min(p.block_size, kTreeKeys), &mk)) return rc;
  if (const int rc = rows_map_bf16(p.v, rows, std::min(p.block_size, kTreeKeys), &mv)) return rc;
  const TreeSizes z = tree_sizes(p.T, p.hq, p.hkv);
  char* w = static_cast<char*>(ws);
  auto take = [&](int64_t n) {
    char* const at = w;
    w += n;
    return at;
  };
  p.list = reinterpret_cast<TreeWork*>(take(z.list));
  p.starts = reinterpret_cast<int*>(take(z.starts));
  p.cuts = reinterpret_cast<Kv8Cut*>(take(z.cuts));
  p.part = reinterpret_cast<float*>(take(z.part));
  p.pairs = (int)tree_pairs(p.T, p.hq, p.hkv);
  p.status = wait_status_word();
  PlanLists far;
  far.ctx = reinterpret_cast<int*>(take(z.rows));
  far.end = reinterpret_cast<int*>(take(z.rows));
  far.runs = reinterpret_cast<int*>(take(z.rows));
  far.items = reinterpret_cast<TreeItem*>(take(z.items));
  far.front = reinterpret_cast<int64_t*>(take(z.front));
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(attn_tree_kernel, kTrSmem, done));
  B200_CUDA(launch(tree_plan_kernel, dim3(1), dim3(kPlanThreads), (size_t)0, s, p, 128 / (p.hq / p.hkv), far));
  const PdlScope after;
  B200_CUDA(launch(attn_tree_kernel, dim3(kNumSMs), dim3(kTreeThreads), (size_t)kTrSmem, s, mk, mv, p));
  B200_CUDA(launch(tree_join_kernel, dim3(kNumSMs, 4), dim3(256), (size_t)0, s, p));
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
  B200_REQUIRE((int64_t)bt_stride * block_size <= 0x7fffffff - 256, B200_ERR_UNSUPPORTED, "paged_attn_tree: block tables of %lld tokens", (long long)bt_stride * block_size);
  B200_REQUIRE(ldq >= (int64_t)hq * kHeadDim && ldq % 8 == 0 && ldo >= (int64_t)hq * kHeadDim && ldo % 8 == 0, B200_ERR_INVALID,
               "paged_attn_tree: ldq and ldo are multiples of 8 that hold a row");
  B200_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_cache_layer) && aligned16(v_cache_layer), B200_ERR_INVALID, "paged_attn_tree: tensors must be 16-byte aligned");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(tree_masks) & 3) == 0, B200_ERR_INVALID, "paged_attn_tree: masks must be 4-byte aligned");
  B200_REQUIRE(scale > 0.f && scale - scale == 0.f, B200_ERR_INVALID, "paged_attn_tree: scale must be positive and finite");
  if (T == 0) return B200_OK;
  const int64_t need = b200_paged_attn_tree_workspace_bytes(T, hq, hkv);
  B200_REQUIRE(ws && aligned16(ws) && ws_bytes >= need, B200_ERR_INVALID, "paged_attn_tree: the workspace is 16-byte aligned and has at least %lld bytes (%lld)",
               (long long)need, (long long)ws_bytes);
  B200_REQUIRE(n_blocks * hkv * block_size <= 0x7fffffff - 256, B200_ERR_UNSUPPORTED, "paged_attn_tree: a cache of %lld rows", (long long)(n_blocks * hkv * block_size));
  B200_REQUIRE((int64_t)T * hkv <= 0x7fffffff - 2 * kNumSMs, B200_ERR_UNSUPPORTED, "paged_attn_tree: %d rows of %d kv heads", T, hkv);
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
