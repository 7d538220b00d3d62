// Paged attention of few (row, head) pairs over the 8-bit cache, on tcgen05 in e4m3: the 128 tokens of a tile fill the MMA's M, the pairs of a
// kv head are its columns (decode rows: the G heads; drafts: rows x G), at most 16.
//
//   S^T[128 tokens][2 NP] = K_tile . Q^T        (A = K as the cache has it, K-major)
//   O^T[128 dims][2 NP] = V_tile^T . W^T        (A = V as the cache has it, MN-major)
//
// The codes go to the tensor core as they are: nothing is widened.  Each column is there twice, as e4m3 and as 16 times what that rounding left: for a
// bf16 query scaled by a power of two both terms together are exact (4 + 4 significant bits), for a weight they have eight.  A token's exponents are
// applied in fp32: the key's to its scores, the value's to its weights.  What a column's codes hold is 2^(score + value exponent), relative to the tile's
// largest such one among the tokens that the column sees: a large value that a row does not see, or hardly weighs, takes no bits from the others, nor do small ones
// that take most of the weight.  The product of a tile is added to the running sums in registers, so that the 22 bits between the largest and the
// smallest code pair only have to span one tile (weights relative to a running maximum would lose a long context's small ones).
//
// The flattened list of (group, kv head, tile) is cut into equal shares, one per SM: contexts may differ as they like.  An item that a cut goes through
// leaves its sums as parts, joined by the next launch.
//
// Bound by the cache's bytes, 258 a token and kv head, where contexts are long: 8 rows of 32 k tokens, 64 heads over 8, 77 us, 5.0 TB/s.  A tile takes 1050 to 1300
// cycles there (the bytes alone 1020): the softmax warps' chain of scores, maximum, weights, and 950 for the warp that issues the MMAs.  In front of it 9000 cycles until the
// first load is asked for (groups, shares, table; much of it instructions fetched for the first time), and 2000 for every item that ends: 64 rows of 500 to
// 1000 tokens 34.5 us, 2.9 TB/s.
#include <algorithm>

#include "attn_kv8.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr int kSlotBytes = kKv8Tile * 128;   // a tile of keys or of values: 16 KiB
constexpr int kTable = 96;                   // items of a CTA that are described at a time
constexpr int kFacs = 2;                     // tiles whose factors are kept
constexpr int kFacBytes = kKv8Tile * 8 + 16; // a token's (key factor, value factor); the tile's factor, whether a token is dead
constexpr int kAhead = 8;                    // tiles ahead that the exponents are asked for (a power of two)
constexpr float kLowest = -3.402823466e38f;
constexpr int kStageWarps = 4;               // keys and values, MMA, queries, factors

struct Kv8Item {
  int row0, nrows, seq, kvh, tile0, tile1, ctx, ends;   // ends: 1 begins in an earlier CTA, 2 goes on in the next
};

template <int NC>
struct Cols {
  static constexpr int NP = NC < 8 ? 8 : NC;               // columns of either term: N = 2 NP is a multiple of 16
  // groups of four softmax warps that share the columns (two for eight columns: 8 rows of 32 k tokens 90 us instead of 81, 200 rows of 500 60 instead of 53; two sets
  // of two that take the tiles in turn: 108)
  static constexpr int CG = NC < 4 ? NC : 4;
  static constexpr int NCG = NC / CG;
  static constexpr int kThreads = (kStageWarps + 4 * CG) * 32;   // 640 at most: 96 registers a thread (a warp more would leave 80: 79 us instead of 74 for 8 rows of 32 k)
  static constexpr int kOperand = 2 * NP * 128;            // queries, or weights, of an item or tile
  static constexpr int kStages = 6;                        // tiles in flight, keys and values each
  static constexpr int kBars = (3 * kStages + 15 + kFacs + 1) & ~1;
  static constexpr uint32_t kTmem = 8 * NP;                // S, S, O, O
  static constexpr int kSmem = 1024 + 2 * kStages * kSlotBytes + 4 * kOperand + kFacs * kFacBytes + kTable * (int)sizeof(Kv8Item) +
                               kBars * 8 + (8 * kKv8Cols + CG * 2 * 4 * NCG + CG * 2 * 4 * NCG) * 4 + kAhead * 256 + 64;
  static_assert(kSmem + 8 * (kThreads + kThreads / 32) <= 232448, "shared memory");
};

// the first row of row i's run: few loads where runs are as short as the caller said, eight at a time where they are longer
__device__ __forceinline__ int run_start(const Kv8Params& p, int i) {
  const int seq = __ldg(p.row_to_seq + i);
  while (i > 0 && __ldg(p.row_to_seq + i - 1) == seq) {
    --i;
    if (i < 8) continue;
    bool same = true;
#pragma unroll
    for (int j = 1; j <= 8; ++j) same &= __ldg(p.row_to_seq + i - j) == seq;
    if (same) i -= 8;
  }
  return i;
}
// group i: of the plan, or (RUNS) the one that starts at row i (start: the first row of its run), or row i
template <bool RUNS>
__device__ __forceinline__ Kv8Group find_group(const Kv8Params& p, int i, int start) {
  if (!RUNS && p.groups) return p.groups[i];
  Kv8Group g = {i, 1, p.row_to_seq ? __ldg(p.row_to_seq + i) : i, kv8_ctx(p, i)};
  if constexpr (!RUNS) return g;
  if ((i - start) % p.group_rows) {
    g.nrows = g.ctx = 0;
    return g;
  }
  while (g.nrows < p.group_rows && i + g.nrows < p.T && __ldg(p.row_to_seq + i + g.nrows) == g.seq) g.ctx = max(g.ctx, kv8_ctx(p, i + g.nrows++));
  return g;
}
__device__ __forceinline__ int group_tiles(const Kv8Group& g) { return g.nrows > 0 && g.ctx > 0 ? (g.ctx + kKv8Tile - 1) / kKv8Tile : 0; }

// RUNS: runs of rows are found among the rows (at most group_rows to a group)
template <int NC, bool RUNS>
__global__ void __launch_bounds__(Cols<NC>::kThreads, 1)
kv8_cols_kernel(const __grid_constant__ Kv8Maps maps, const Kv8Params p) {
  using C = Cols<NC>;
  constexpr int NP = C::NP, CG = C::CG, NCG = C::NCG, kStages = C::kStages, kThreads = C::kThreads;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* qs = ring + 2 * kStages * kSlotBytes;          // [2] queries of an item
  unsigned char* ws = qs + 2 * C::kOperand;                // [2] weights of a tile
  unsigned char* facs = ws + 2 * C::kOperand;              // [kFacs]
  Kv8Item* table = reinterpret_cast<Kv8Item*>(facs + kFacs * kFacBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(table + kTable);   // [kStages]: a tile's keys and values are there
  uint64_t* freed = full + kStages;                        // [2 kStages]: keys, values, keys, ...
  uint64_t* s_full = freed + 2 * kStages;                  // [2]: the tile's scores, and its factors
  uint64_t* w_ready = s_full + 2;
  uint64_t* o_full = w_ready + 2;
  uint64_t* q_ready = o_full + 2;
  uint64_t* q_free = q_ready + 2;
  uint64_t* q_info = q_free + 2;                           // [4]: an item's scales, for the softmax warps (who may be three items behind)
  uint64_t* f_free = q_info + 4;                           // [kFacs]
  uint64_t* last = f_free + kFacs;
  float2* info = reinterpret_cast<float2*>(full + C::kBars);   // [4 items][pairs]: what undoes a query's scaling, the tokens that its row sees; from here on in whole 16 bytes
  float* x_sum = reinterpret_cast<float*>(info + 4 * kKv8Cols);                       // [CG][2][NCG][4 warps]
  float* x_max = x_sum + CG * 2 * NCG * 4;                 // [CG][2][NCG][4 warps]
  uint32_t* exps = reinterpret_cast<uint32_t*>(x_max + CG * 2 * NCG * 4);   // [kAhead][32 lanes][keys, values]
  int* shared_int = reinterpret_cast<int*>(exps + kAhead * 64);            // 0: tensor memory, 1: a wait ran out, 2, 3: the share's first and last item
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Waits wait(reinterpret_cast<uint32_t*>(shared_int + 1), p.status);
  if (p.groups) {
    pdl_wait();
    if (p.groups[-1].row0 == 0) {   // a plan without groups
      if (threadIdx.x == 0) p.cuts[blockIdx.x].parts = 0;
      pdl_launch_dependents();
      return;
    }
  }
  __shared__ uint64_t scan_warp[kThreads / 32], scan_thread[kThreads];

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(full + s, 1), mbar_init(freed + 2 * s, 1), mbar_init(freed + 2 * s + 1, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + s, 2);
      mbar_init(w_ready + s, 4 * CG);
      mbar_init(o_full + s, 1);
      mbar_init(q_ready + s, 1);
      mbar_init(q_free + s, 1);
    }
    for (int s = 0; s < 4; ++s) mbar_init(q_info + s, 1);
    for (int s = 0; s < kFacs; ++s) mbar_init(f_free + s, CG);
    mbar_init(last, 1);
    shared_int[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(shared_int)), "r"(C::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  for (int i = threadIdx.x; i < 4 * C::kOperand / 16; i += kThreads) reinterpret_cast<uint4*>(qs)[i] = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  pdl_wait();
  pdl_launch_dependents();

  // ---- the CTA's share of the tiles: a thread counts its groups' (32 bits hold them: the host's check) ----
  const int n_groups = p.groups ? p.groups[-1].row0 : p.T, each = (n_groups + kThreads - 1) / kThreads;
  const int g0 = min((int)threadIdx.x * each, n_groups), g1 = min(g0 + each, n_groups);
  const int start0 = RUNS && g0 < g1 ? run_start(p, g0) : g0;
  auto next_start = [&](int start, int i) { return RUNS && i > g0 && __ldg(p.row_to_seq + i) != __ldg(p.row_to_seq + i - 1) ? i : start; };
  Kv8Group own = {0, 0, 0, 0};
  uint64_t sum = 0;   // groups that see something << 32 | their tiles
#pragma unroll 1
  for (int i = g0, start = start0; i < g1; ++i) {
    start = next_start(start, i);
    own = find_group<RUNS>(p, i, start);
    const uint32_t nt = group_tiles(own);
    sum += (uint64_t)(nt > 0) << 32 | nt;
  }
  uint64_t before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) scan_warp[warp] = before;
  before -= sum;
  if (threadIdx.x == 0) p.cuts[blockIdx.x].parts = 0;
  __syncthreads();
  uint64_t warps = lane < kThreads / 32 ? scan_warp[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(0xffffffffu, warps, o);
    if (lane >= o) warps += v;
  }
  const uint64_t in_front = __shfl_sync(0xffffffffu, warps, max(warp - 1, 0));
  if (warp > 0) before += in_front;
  const uint32_t tiles = (uint32_t)__shfl_sync(0xffffffffu, warps, 31) * p.hkv, share = (tiles + gridDim.x - 1) / gridDim.x;
  const uint32_t begin = min(tiles, share * blockIdx.x), end = min(tiles, begin + share);
  scan_thread[threadIdx.x] = before;
  // the groups of this thread that the share touches: f(group, its first tile, tiles of a head, items in front of it)
  auto own_groups = [&](auto f) {
    uint64_t at = scan_thread[threadIdx.x];
#pragma unroll 1
    for (int i = g0, start = start0; i < g1; ++i) {
      start = next_start(start, i);
      const Kv8Group g = each == 1 ? own : find_group<RUNS>(p, i, start);
      const uint32_t nt = group_tiles(g), base = (uint32_t)at * p.hkv;
      if (nt > 0 && base < end && base + nt * p.hkv > begin) f(g, base, nt, (int)(at >> 32) * p.hkv);
      at += (uint64_t)(nt > 0) << 32 | nt;
    }
  };
  own_groups([&](const Kv8Group& g, uint32_t base, uint32_t nt, int items) {
    if (begin >= base) shared_int[2] = items + (int)((begin - base) / nt);                                  // the share's first item
    if (end <= base + nt * p.hkv) shared_int[3] = items + (int)((end - 1 - base) / nt);                     // its last
  });
  __syncthreads();
  const int first_item = shared_int[2], n_items = begin < end ? shared_int[3] - first_item + 1 : 0;
  // items [from, from + kTable) of the share, by all threads
  auto fill_table = [&](int from) {
    own_groups([&](const Kv8Group& g, uint32_t base, uint32_t nt, int items) {
      const int h1 = min(p.hkv, (int)((end - base + nt - 1) / nt));
      for (int h = begin > base ? (int)((begin - base) / nt) : 0; h < h1; ++h) {
        const int at = items + h - first_item - from;
        if (at < 0 || at >= kTable) continue;
        Kv8Item w = {g.row0, g.nrows, g.seq, h, 0, (int)nt, g.ctx, 0};
        const uint32_t b = base + h * nt;
        if (b < begin) w.tile0 = (int)(begin - b), w.ends |= 1;
        if (b + nt > end) {
          w.tile1 = (int)(end - b), w.ends |= 2;
          if (!(w.ends & 1)) p.cuts[blockIdx.x] = {g.row0, g.nrows, h, (int)((b + nt - 1) / share) - (int)blockIdx.x + 1};
        }
        table[at] = w;
      }
    });
  };
  if (n_items > 0) fill_table(0);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = (uint32_t)shared_int[0];
  // how many items the next table has (0: there is none); all threads come here
  int described = 0;
  auto next_table = [&]() {
    const int from = described;
    described += kTable;
    if (from > 0 && from < n_items) {
      __syncthreads();
      fill_table(from);
      __syncthreads();
    }
    return min(max(n_items - from, 0), kTable);
  };

  if (warp == 0) {
    // ===== TMA: keys and values =====
    const bool issuer = elect_one();
    if (issuer) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    const int box = min(p.block_size, kKv8Tile), per_tile = kKv8Tile / box;   // boxes of a tile
    const int cells = (int)(p.n_blocks * p.hkv * p.block_size);
    int stage = 0;
    uint32_t ph = 1;
    bool stop = false;
    // the first cell of an item's box number `at` (of those that hold something), a box to a lane
    auto cell_of = [&](const Kv8Item& w, int at) {
      const int tok = w.tile0 * kKv8Tile + at * box;
      if (tok >= min(w.ctx, w.tile1 * kKv8Tile)) return 0;
      const int blk = __ldg(p.block_table + (int64_t)w.seq * p.bt_stride + tok / p.block_size);
      return blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + w.kvh) * p.block_size + tok % p.block_size : cells;   // behind the cache: zeros
    };
    for (int count; (count = next_table()) > 0;) {
      int lead = cell_of(table[0], lane);   // the next item's first 32 boxes (asked for when its turn comes, they take 1000 cycles and more)
      for (int it = 0; it < count && !stop; ++it) {
        const Kv8Item w = table[it];
        const int boxes = (min(w.ctx, w.tile1 * kKv8Tile) - w.tile0 * kKv8Tile + box - 1) / box;
        int have = lead, next = 32 < boxes ? cell_of(w, 32 + lane) : 0;
        if (it + 1 < count) lead = cell_of(table[it + 1], lane);
        for (int b = 0; b < boxes && !(stop = wait.stop()); b += per_tile) {
          if (b && (b & 31) == 0) have = next, next = cell_of(w, b + 32 + lane);
          const int n = min(per_tile, boxes - b);
          unsigned char* const keys = ring + 2 * stage * kSlotBytes;
          int cell[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) cell[i] = __shfl_sync(0xffffffffu, have, (b + i) & 31);
          wait(freed + 2 * stage, ph);
          wait(freed + 2 * stage + 1, ph);
          if (issuer) {
            mbar_expect_tx(full + stage, 2 * n * box * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i < n) {
                tma_load_2d(keys + i * box * 128, &maps.k, 0, cell[i], full + stage);
                tma_load_2d(keys + kSlotBytes + i * box * 128, &maps.v, 0, cell[i], full + stage);
              }
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, ph ^= 1;
        }
      }
    }
    if (wait.stop())   // the loads in flight: a stage's last ones filled it in this round of the ring or in the one before
      for (int s = 0; s < kStages; ++s) wait.drain(full + s, s < stage ? ph ^ 1 : ph);
  } else if (warp == 1) {
    // ===== MMA: the scores of tile n + 1, of the next item if need be, then tile n's second product =====
    const uint32_t one = elect_one() ? 1u : 0u, tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t desc_ring = make_desc(smem_u32(ring), 16, 1024), desc_q = make_desc(smem_u32(qs), 16, 1024), desc_w = make_desc(smem_u32(ws), 16, 1024);
    constexpr uint32_t id_s = idesc_e4m3(2 * NP, 0), id_o = idesc_e4m3(2 * NP, 1);
    int stage = 0, prev = 0, n = 0, item = 0;   // stages of the next tile and of the one before
    uint32_t ph = 0;
    bool pending = false;
    auto product = [&](int m) {      // tile m's weights and values
      wait(w_ready + (m & 1), (m >> 1) & 1);
      fence_after();
      const uint64_t dv = desc_ring + (uint64_t)(((2 * prev + 1) * kSlotBytes) >> 4), dw = desc_w + (uint64_t)(((m & 1) * C::kOperand) >> 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_f8_ss(one, tm + 4 * NP + (m & 1) * 2 * NP, dv + (j * 4096) / 16, dw + (j * 32) / 16, id_o, j ? 1u : 0u);
      commit(one, freed + 2 * prev + 1);
      commit(one, o_full + (m & 1));
    };
    for (int count; (count = __shfl_sync(0xffffffffu, next_table(), 0)) > 0;) {
      for (int it = 0; it < count; ++it, ++item) {
        const int nt = __shfl_sync(0xffffffffu, table[it].tile1 - table[it].tile0, 0);
        // what is not there yet is not waited for before what is: the previous tile's product
        if (pending && !mbar_test(q_ready + (item & 1), (item >> 1) & 1)) product(n - 1), pending = false;
        wait(q_ready + (item & 1), (item >> 1) & 1);
        const uint64_t dq = desc_q + (uint64_t)(((item & 1) * C::kOperand) >> 4);
        for (int i = 0; i < nt; ++i, ++n) {
          if (pending && !mbar_test(full + stage, ph)) product(n - 1), pending = false;
          wait(full + stage, ph);
          fence_after();
          const uint64_t dk = desc_ring + (uint64_t)((2 * stage * kSlotBytes) >> 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_f8_ss(one, tm + (n & 1) * 2 * NP, dk + (j * 32) / 16, dq + (j * 32) / 16, id_s, j ? 1u : 0u);
          commit(one, freed + 2 * stage);
          commit(one, s_full + (n & 1));
          commit(i + 1 == nt ? one : 0u, q_free + (item & 1));
          if (pending) product(n - 1);
          pending = true;
          prev = stage;
          if (++stage == kStages) stage = 0, ph ^= 1;
        }
      }
      if (pending) product(n - 1);   // (the softmax warps finish a table's last item before they come to the next table)
      pending = false;
    }
    if (wait.stop()) {
      commit(one, last);
      wait.drain(last, 0);
    }
  } else if (warp == 2) {
    // ===== queries: 16 lanes a pair, scaled to [128, 256), in two terms =====
    const int G = p.hq / p.hkv;
    int item = 0;
    if (!p.groups)   // rows that see nothing: zeros, by the CTAs in turn
      for (int r = blockIdx.x; r < p.T; r += gridDim.x)
        if (__ldg(p.ctx_lens + r) <= 0)
          for (int i = lane; i < p.hq * kHeadDim / 8; i += 32) *reinterpret_cast<uint4*>(p.out + (int64_t)r * p.ldo + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
    for (int count; (count = next_table()) > 0;) {
      for (int it = 0; it < count; ++it, ++item) {
        const Kv8Item w = table[it];
        if (item >= 2) wait(q_free + (item & 1), ((item >> 1) - 1) & 1);
        unsigned char* qb = qs + (item & 1) * C::kOperand;
        const int ncol = w.nrows * G, d = (lane & 15) * 8;
        constexpr int U = NC < 8 ? (NC + 1) / 2 : 4;   // pairs of columns that are asked for at a time
        for (int c1 = 0; c1 < ncol; c1 += 2 * U) {
          uint4 v[U];
          int ctx[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c1 + 2 * u + (lane >> 4);
            v[u] = make_uint4(0u, 0u, 0u, 0u);
            ctx[u] = c < ncol && w.nrows > 1 ? kv8_ctx(p, w.row0 + c / G) : w.ctx;
            if (c < ncol) v[u] = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)(w.row0 + c / G) * p.ldq + (w.kvh * G + c % G) * kHeadDim + d));
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c1 + 2 * u + (lane >> 4);
            uint2 hi, lo;
            uint32_t m = query_max(v[u]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const uint32_t e = query_exponent(m);
            split_query<16>(v[u], e, hi, lo);
            if (c < ncol) {
              *reinterpret_cast<uint2*>(qb + operand_off(c, d)) = hi;
              *reinterpret_cast<uint2*>(qb + operand_off(NP + c, d)) = lo;
              if ((lane & 15) == 0) info[(item & 3) * kKv8Cols + c] = make_float2(query_back(e) * p.scale2, __int_as_float(ctx[u]));
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready + (item & 1)), mbar_arrive(q_info + (item & 3));
      }
    }
  } else if (warp == 3) {
    // ===== factors: a token's 2^key exponent, and 256 * 2^(value exponent - the tile's largest); four tokens a lane.  The exponents come by asynchronous copies kAhead tiles
    // ahead, each lane's own (as loads into registers they are waited for together with those of the tiles behind: 1100 cycles a tile; as bulk copies of 128 bytes
    // they took the issuing warp 400 each) =====
    const int box = min(p.block_size, kKv8Tile), per_tile = kKv8Tile / box, my_box = 4 * lane / box, my_cell = 4 * lane % box;
    int n = 0;
    for (int count; (count = next_table()) > 0;) {
      // the tiles in order: the first cells of 32 boxes (-1: behind the context, or outside the cache), of the 32 behind them, of the next item's first 32
      int it_c = -1, i_c = 0, first_c = 0, end_c = 0, ctx_c = 0, have = 0, next = 0;
      auto cell_of = [&](const Kv8Item& w, int at) {
        const int tok = w.tile0 * kKv8Tile + at * box;
        if (tok >= min(w.ctx, w.tile1 * kKv8Tile)) return -1;
        const int blk = __ldg(p.block_table + (int64_t)w.seq * p.bt_stride + tok / p.block_size);
        return blk >= 0 && blk < p.n_blocks ? (blk * p.hkv + w.kvh) * p.block_size + tok % p.block_size : -1;
      };
      int lead = cell_of(table[0], lane);
      auto ask = [&](int m) {   // tile m's
        if (i_c == end_c && it_c < count && ++it_c < count) {
          const Kv8Item w = table[it_c];
          i_c = w.tile0, end_c = w.tile1, ctx_c = min(w.ctx, w.tile1 * kKv8Tile), first_c = i_c * per_tile;
          have = lead, next = (w.tile1 - w.tile0) * per_tile > 32 ? cell_of(w, 32 + lane) : -1;
          if (it_c + 1 < count) lead = cell_of(table[it_c + 1], lane);
        }
        if (it_c < count) {
          const int b = i_c * per_tile - first_c;
          if (b && (b & 31) == 0) have = next, next = cell_of(table[it_c], b + 32 + lane);
          const int cell = __shfl_sync(0xffffffffu, have, (b & 31) + my_box);
          uint32_t* const at = exps + ((m & (kAhead - 1)) * 32 + lane) * 2;
          if (cell >= 0 && i_c * kKv8Tile + 4 * lane < ctx_c) f2::cp4(at, p.ke + cell + my_cell), f2::cp4(at + 1, p.ve + cell + my_cell);
          else at[0] = at[1] = 0u;
          ++i_c;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      for (int d = 0; d < kAhead; ++d) ask(n + d);
      for (int it = 0; it < count; ++it) {
        const int tile1 = table[it].tile1, ctx = table[it].ctx;
        for (int i = table[it].tile0; i < tile1; ++i, ++n) {
          const int left = ctx - i * kKv8Tile - 4 * lane;   // tokens of this lane's four
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
          const uint2 kv4 = *reinterpret_cast<const uint2*>(exps + ((n & (kAhead - 1)) * 32 + lane) * 2);
          // a value row that is not a number: the columns that see it are none either (its key's factor), the others must not meet it
          uint32_t ve[4], m = 1u;
          bool none = false;
          float kf[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ve[j] = (kv4.y >> (8 * j)) & 255u;
            kf[j] = __uint_as_float(j < left && ve[j] == 255u ? 0x7fffffffu : ((kv4.x >> (8 * j)) & 255u) << 23);   // (2^-127 counts as nothing)
            if (j >= left) ve[j] = 255u;
            if (ve[j] == 255u) none = true;
            else m = max(m, ve[j]);
          }
          m = __reduce_max_sync(0xffffffffu, m);
          ask(n + kAhead);   // (its place has been read)
          none = __any_sync(0xffffffffu, none);
          float vf[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[j] = ve[j] == 255u ? -0.f : __uint_as_float((uint32_t)max((int)(ve[j] - m) + 135, 0) << 23);
          if (n >= kFacs) wait(f_free + (n & (kFacs - 1)), (n / kFacs - 1) & 1);   // (that tile's scores have been waited for, too: s_full is in tile n's phase)
          float* f = reinterpret_cast<float*>(facs + (n & (kFacs - 1)) * kFacBytes);
          reinterpret_cast<float4*>(f)[2 * lane] = make_float4(kf[0], vf[0], kf[1], vf[1]);
          reinterpret_cast<float4*>(f)[2 * lane + 1] = make_float4(kf[2], vf[2], kf[3], vf[3]);
          if (lane == 0) {
            f[2 * kKv8Tile] = __uint_as_float((uint32_t)max((int)m - 8, 1) << 23);
            reinterpret_cast<int*>(f)[2 * kKv8Tile + 1] = none;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(s_full + (n & 1));
        }
      }
    }
  } else {
    // ===== softmax: a thread owns a token of the scores and an entry of the result; the columns are dealt to CG groups of four warps =====
    const int grp = (warp - kStageWarps) >> 2, quad = warp & 3, tau = quad * 32 + lane, G = p.hq / p.hkv, c0 = grp * NCG;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + c0;
    float* xm = x_max + grp * 2 * NCG * 4;
    float* xs = x_sum + grp * 2 * NCG * 4;
    int n = 0, item = 0, stage = 0;
    uint32_t ph = 0;
    float mu[NCG], l[NCG], acc[NCG], keep[NCG], take[NCG], keep0[NCG], take0[NCG];   // keep, take: what becomes of the sums, and of the previous tile's product; of that before it
    uint32_t oh[NCG], ol[NCG];                                 // a product on its way from tensor memory
    auto ask = [&](int m) {                                    // tile m's
      ld_cols<NCG>(base + 4 * NP + (m & 1) * 2 * NP, oh);
      ld_cols<NCG>(base + 4 * NP + (m & 1) * 2 * NP + NP, ol);
    };
    auto fold = [&](const float (&k)[NCG], const float (&t)[NCG]) {   // (it is there: ld_wait)
#pragma unroll
      for (int j = 0; j < NCG; ++j) {
        asm volatile("" : "+r"(oh[j]), "+r"(ol[j]));
        acc[j] = acc[j] * k[j] + fmaf(__uint_as_float(ol[j]), 0.0625f, __uint_as_float(oh[j])) * t[j];
      }
    };
    // an item's results: its last product, then the denominators (every token's share)
    auto finish = [&](const Kv8Item& w, const float (&mu0)[NCG], const float (&l0)[NCG], int last_tile) {
      float* xt = xs + (item & 1) * NCG * 4;
#pragma unroll
      for (int j = 0; j < NCG; ++j) {
        const float v = warp_sum(l0[j]);
        if (lane == 0) xt[j * 4 + quad] = v;
      }
      wait(o_full + (last_tile & 1), (last_tile >> 1) & 1);
      fence_after();
      ask(last_tile);
      ld_wait<NCG>(oh);
      fold(keep, take);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
      const int ncol = w.nrows * G;
#pragma unroll
      for (int j = 0; j < NCG; ++j) {
        const int c = c0 + j;
        if (c < ncol) {
          const float4 x = reinterpret_cast<const float4*>(xt)[j];
          const float sum_l = (x.x + x.y) + (x.z + x.w);
          if (w.ends == 0) {
            p.out[(int64_t)(w.row0 + c / G) * p.ldo + (w.kvh * G + c % G) * kHeadDim + tau] = __float2bfloat16_rn(sum_l == 0.f ? 0.f : __fdividef(acc[j], sum_l));
          } else {
            float* dst = p.part + ((int64_t)(2 * blockIdx.x + ((w.ends & 1) ? 0 : 1)) * kKv8Cols + c) * kKv8PartFloats;
            dst[tau] = acc[j];
            if (tau == 0) dst[128] = mu0[j], dst[129] = sum_l;
          }
        }
        acc[j] = 0.f;
      }
    };
#pragma unroll
    for (int j = 0; j < NCG; ++j) acc[j] = 0.f;
    for (int count; (count = next_table()) > 0;) {
      bool two = false;   // the last two products are to be added, both of one item
      for (int it = 0; it < count; ++it, ++item) {
        const Kv8Item w = table[it];
        const int ncol = w.nrows * G;
        int ctx[NCG];
        float qf[NCG], mu_before[NCG], l_before[NCG];
        wait(q_info + (item & 3), (item >> 2) & 1);
#pragma unroll
        for (int j = 0; j < NCG; ++j) {
          const float2 x = c0 + j < ncol ? info[(item & 3) * kKv8Cols + c0 + j] : make_float2(0.f, 0.f);
          qf[j] = x.x, ctx[j] = __float_as_int(x.y);
          mu_before[j] = mu[j], l_before[j] = l[j];
          mu[j] = kLowest;
          l[j] = 0.f;
        }
        for (int i = w.tile0; i < w.tile1; ++i, ++n) {
          const int tok = i * kKv8Tile + tau;
          float* xt = xm + (n & 1) * NCG * 4;
          wait(s_full + (n & 1), (n >> 1) & 1);
          fence_after();
          if (two) ask(n - 2);   // (scores of tile n are complete behind the product of tile n - 2)
          uint32_t hi[NCG], lo[NCG];
          ld_cols<NCG>(base + (n & 1) * 2 * NP, hi);
          ld_cols<NCG>(base + (n & 1) * 2 * NP + NP, lo);
          const float* f = reinterpret_cast<const float*>(facs + (n & (kFacs - 1)) * kFacBytes);
          const float2 kv = reinterpret_cast<const float2*>(f)[tau], vr = reinterpret_cast<const float2*>(f)[kKv8Tile];
          const float lv = fmaxf((float)(int)(__float_as_uint(kv.y) >> 23 & 255u) - 135.f, -(float)kKv8Span);   // the value's exponent below the tile's largest
          ld_wait<NCG>(hi);
          if (two) fold(keep0, take0);
          float s[NCG];   // score + lv
#pragma unroll
          for (int j = 0; j < NCG; ++j) {
            asm volatile("" : "+r"(lo[j]));
            s[j] = tok < ctx[j] ? fmaf(fmaf(__uint_as_float(lo[j]), 0.0625f, __uint_as_float(hi[j])), kv.x * qf[j], lv) : -INFINITY;
            const float m = warp_max_f32(s[j]);
            if (lane == 0) xt[j * 4 + quad] = m;
          }
          asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
          if (tau == 0) mbar_arrive(f_free + (n & (kFacs - 1)));
          float wt[NCG], keep1[NCG], take1[NCG];
#pragma unroll
          for (int j = 0; j < NCG; ++j) {
            const float4 x = reinterpret_cast<const float4*>(xt)[j];
            // (a column whose row does not see this tile: the lowest finite number stands for its maximum, and its scores are -inf)
            // the denominators are relative to this maximum too: e may be above 1 for tokens of smaller values, by 2^kKv8Span at most
            const float mt = fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), kLowest), mn = fmaxf(mu[j], mt);
            const float e = exp2_fast(s[j] - mt - lv), b = exp2_fast(mt - mn);
            keep1[j] = exp2_fast(mu[j] - mn);
            take1[j] = b * vr.x;
            l[j] = l[j] * keep1[j] + e * b;
            mu[j] = mn;
            wt[j] = e * kv.y;
          }
          unsigned char* wb = ws + (n & 1) * C::kOperand;
#pragma unroll
          for (int j = 0; j < NCG; j += 2) {   // (a weight that is not a number leaves its denominator so, whatever its codes)
            const float2 x = make_float2(wt[j], NCG > 1 ? wt[j + (NCG > 1)] : 0.f);
            const __nv_fp8x2_storage_t c = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
            const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3)));
            const __nv_fp8x2_storage_t d = __nv_cvt_float2_to_fp8x2(make_float2((x.x - back.x) * 16.f, (x.y - back.y) * 16.f), __NV_SATFINITE, __NV_E4M3);
            wb[operand_off(c0 + j, tau)] = (unsigned char)c;
            wb[operand_off(NP + c0 + j, tau)] = (unsigned char)d;
            if (NCG > 1) {
              wb[operand_off(c0 + j + 1, tau)] = (unsigned char)(c >> 8);
              wb[operand_off(NP + c0 + j + 1, tau)] = (unsigned char)(d >> 8);
            }
          }
          if (grp == 0 && __float_as_int(vr.y) != 0) {
            // value rows behind the context may hold anything, and 0 * NaN = NaN: zero them under their zero weights
            wait(full + stage, ph);
            if (__float_as_uint(kv.y) == 0x80000000u) {
              unsigned char* vb = ring + (2 * stage + 1) * kSlotBytes + tau * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vb + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_async_smem();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(w_ready + (n & 1));
          if (i == w.tile0 && it > 0) finish(table[it - 1], mu_before, l_before, n - 1);   // the item before, while this one's first product runs
          two = i > w.tile0;
#pragma unroll
          for (int j = 0; j < NCG; ++j) keep0[j] = keep[j], take0[j] = take[j], keep[j] = keep1[j], take[j] = take1[j];
          if (++stage == kStages) stage = 0, ph ^= 1;
        }
      }
      if (two) {
        wait(o_full + (n & 1), ((n - 2) >> 1) & 1);
        fence_after();
        ask(n - 2);
        ld_wait<NCG>(oh);
        fold(keep0, take0);
      }
      finish(table[count - 1], mu, l, n - 1);
    }
    fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem));
  }
}

template <int NC, bool RUNS>
int launch_cols(const Kv8Maps& m, const Kv8Params& p, int grid, cudaStream_t s) {
  static bool done[64] = {};
  B200_CUDA(ensure_dynamic_smem(kv8_cols_kernel<NC, RUNS>, Cols<NC>::kSmem, done));
  B200_CUDA(launch(kv8_cols_kernel<NC, RUNS>, dim3(grid), dim3(Cols<NC>::kThreads), (size_t)Cols<NC>::kSmem, s, m, p));
  return B200_OK;
}

}  // namespace

int kv8_cols_launch(const Kv8Maps& m, const Kv8Params& p, int cols, int grid, cudaStream_t s) {
  if (const int e = wait_status()) return e;
  if (!p.groups && p.group_rows > 1 && p.row_to_seq) {   // (of at most eight pairs)
    if (cols <= 2) return launch_cols<2, true>(m, p, grid, s);
    if (cols <= 4) return launch_cols<4, true>(m, p, grid, s);
    return launch_cols<8, true>(m, p, grid, s);
  }
  if (cols <= 2) return launch_cols<2, false>(m, p, grid, s);
  if (cols <= 4) return launch_cols<4, false>(m, p, grid, s);
  if (cols <= 8) return launch_cols<8, false>(m, p, grid, s);
  return launch_cols<16, false>(m, p, grid, s);
}

}  // namespace b200
